// The exponential of the router's softmax, in the top-k kernel and in the layer for a few tokens.
#pragma once
#include <cuda_runtime.h>

namespace rf {

// exp(x), x <= 0, as a fixed sequence of fp32 operations with no fused multiply-add, so a CPU
// restatement reproduces it bit for bit: t = max(x,-80)*log2e; n = rint(t); f = t-n; degree-7
// Horner for 2^f; exact scaling by 2^n.
__device__ __forceinline__ float det_exp(float x) {
    x = fmaxf(x, -80.0f);
    const float t = __fmul_rn(x, 1.4426950408889634f);
    const float n = rintf(t);
    const float f = __fsub_rn(t, n);
    float p = 1.5252733804059840e-05f;
    p = __fadd_rn(__fmul_rn(p, f), 0.0001540353039338161f);
    p = __fadd_rn(__fmul_rn(p, f), 0.0013333558146428443f);
    p = __fadd_rn(__fmul_rn(p, f), 0.009618129107628477f);
    p = __fadd_rn(__fmul_rn(p, f), 0.05550410866482158f);
    p = __fadd_rn(__fmul_rn(p, f), 0.2402265069591007f);
    p = __fadd_rn(__fmul_rn(p, f), 0.6931471805599453f);
    p = __fadd_rn(__fmul_rn(p, f), 1.0f);
    return __uint_as_float(__float_as_uint(p) + (static_cast<int>(n) << 23));   // p in [0.7, 1.42], result normal
}

}  // namespace rf
