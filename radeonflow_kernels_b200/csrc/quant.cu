// FP8 operands of the block-scaled GEMMs: e4m3fn values with one fp32 scale per 1 x 128 block of a row (activations) or per
// 128 x 128 block (weights).  No counterpart in the reference, whose operands arrive quantised.
//
//   a = max(largest magnitude of the block, 2^-100),  scale = a / 448,  q = e4m3(x * (448 / a)), to nearest, ties to even
//
// 448 is e4m3's largest value; the floor keeps 448 / a finite for blocks of zeros.  A NaN makes its whole block NaN, scale
// included, and an infinity makes the scale infinite: an overflow stays visible behind the product.
//
// All three are one pass over the data, held in registers between the block's maximum and its conversion.  HBM bounds them as long as
// the instructions per element stay few: with two IEEE divisions a lane, 64-bit index arithmetic and a modulo per block,
// 32768 x 7168 gathered bf16 rows took 146 us and SwiGLU of 32768 x 2048 fp16 81.
#include "ptx.cuh"
#include "host_util.h"
#include "launch.h"
#include "../../include/rf_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace rf {

namespace {

constexpr int kBlock = 128;
constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;      // 2^-100

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// max(|a|, |b|, c)
__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(c));
    return r;
}
// Four values to four e4m3 bytes, the first in the lowest.
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ __half zero_of(__half) { return __ushort_as_half(0); }
__device__ __forceinline__ __nv_bfloat16 zero_of(__nv_bfloat16) { return __ushort_as_bfloat16(0); }
__device__ __forceinline__ float zero_of(float) { return 0.f; }

// Eight consecutive elements, as they lie in memory: 16-byte loads (VEC: the address is a multiple of 16) or element by
// element, those from `n` on zero.
template <class T>
struct Eight {
    static constexpr int kVecs = sizeof(T) / 2;
    union {
        uint4 v[kVecs];
        T e[8];
    };
    __device__ __forceinline__ Eight() {}
    template <bool VEC>
    __device__ __forceinline__ void load(const T* p, int n = 8) {
        if (VEC && n >= 8) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) v[i] = ld_global_cg_v4(reinterpret_cast<const uint4*>(p) + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : zero_of(T());
        }
    }
    __device__ __forceinline__ float f(int i) const { return to_f32(e[i]); }
};

__device__ __forceinline__ float largest_of(const float (&x)[8]) {
    float a = max_nan(fabsf(x[0]), fabsf(x[1]));
#pragma unroll
    for (int i = 2; i < 8; i += 2) a = max_abs_nan(x[i], x[i + 1], a);
    return a;
}
// (magnitudes of 16-bit types two at a time, before they are widened)
__device__ __forceinline__ float largest_of(const Eight<float>& x) { return largest_of(x.e); }
__device__ __forceinline__ float largest_of(const Eight<__half>& x) {
    __half2 a = __habs2(__halves2half2(x.e[0], x.e[1]));
#pragma unroll
    for (int i = 2; i < 8; i += 2) a = __hmax2_nan(a, __habs2(__halves2half2(x.e[i], x.e[i + 1])));
    return max_nan(__low2float(a), __high2float(a));
}
__device__ __forceinline__ float largest_of(const Eight<__nv_bfloat16>& x) {
    __nv_bfloat162 a = __habs2(__halves2bfloat162(x.e[0], x.e[1]));
#pragma unroll
    for (int i = 2; i < 8; i += 2) a = __hmax2_nan(a, __habs2(__halves2bfloat162(x.e[i], x.e[i + 1])));
    return max_nan(__low2float(a), __high2float(a));
}

// The smallest of eight, NaN left out.
__device__ __forceinline__ float lowest_of(const Eight<float>& x) {
    float a = x.e[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) a = fminf(a, x.e[i]);
    return a;
}
__device__ __forceinline__ float lowest_of(const Eight<__half>& x) {
    __half2 a = __halves2half2(x.e[0], x.e[1]);
#pragma unroll
    for (int i = 2; i < 8; i += 2) a = __hmin2(a, __halves2half2(x.e[i], x.e[i + 1]));
    return fminf(__low2float(a), __high2float(a));
}
__device__ __forceinline__ float lowest_of(const Eight<__nv_bfloat16>& x) {
    __nv_bfloat162 a = __halves2bfloat162(x.e[0], x.e[1]);
#pragma unroll
    for (int i = 2; i < 8; i += 2) a = __hmin2(a, __halves2bfloat162(x.e[i], x.e[i + 1]));
    return fminf(__low2float(a), __high2float(a));
}

// The half warp's largest value (16 lanes hold one block of 128).
__device__ __forceinline__ float half_warp_max(float a) {
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, s));
    return a;
}

// Both factors of a block are quotients corrected by their remainder (Markstein): q0 within two units in the last place, then
// q0 + (numerator - q0 * divisor) / divisor in fused operations.
//
// 448 / a rounded to nearest for 2^-100 <= a, zero for an infinity; so values that lie on a tie of two e4m3 ones go where the
// formula sends them.  (On a scaled value: neither it nor its reciprocal leaves the range of normal numbers.  That one correction is
// enough for every a is tested: powers of two aside there are 2^23 of them.  A division costs the kernels for 16-bit rows, which have 32
// registers, a stack frame.)
__device__ __forceinline__ float steps_per_unit(float a) {
    constexpr float top = kE4m3Max * 0x1p-20f;
    const float b = a * 0x1p-20f;
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(b));
    const float q = y * top;
    return fmaf(fmaf(-q, fminf(b, 0x1p120f), top), y, q);         // (an infinity: 0 * finite)
}
// a / 448 rounded to nearest: here the divisor's reciprocal itself is.  An infinity stays one.
__device__ __forceinline__ float over_448(float a) {
    constexpr float inv = 1.0f / kE4m3Max;
    const float q = a * inv;
    return isinf(a) ? a : fmaf(fmaf(-q, kE4m3Max, a), inv, q);
}
// g / (1 + exp(-g)) for g >= kSiluLow, where the reciprocal is a normal number.  exp(-g) = 2^t exp(c) with t = fl(-g log2 e) and
// c = -g - t ln 2 what that left out, 2^-18 at most: 1 + c.  Off by 2^-20.7 at most: ten times 2^-24, of which 2^t has four and the
// reciprocal two.
constexpr float kSiluLow = -87.0f;
__device__ __forceinline__ float silu(float g) {
    constexpr float log2e = 1.44269504f, ln2 = 0.693147182f, ln2_rest = -1.90465421e-9f;
    const float t = -g * log2e, c = fmaf(-t, ln2_rest, fmaf(-t, ln2, -g));
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    // (where 2^t is no normal number, c may be none either)
    if (fabsf(t) < 126.0f) e = fmaf(e, c, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return g * r;
}
// SiLU(g) * u for every g.  Below kSiluLow 1 / (1 + exp(-g)) is exp(g), which leaves the normal numbers; its root does not before
// g u exp(g) does.
__device__ __forceinline__ float swiglu_far(float g, float u) {
    const float root = expf(0.5f * g);
    return g < kSiluLow ? (g * root) * (root * u) : silu(g) * u;
}

__device__ __forceinline__ uint2 to_e4m3x8(const float (&x)[8], float r) {
    return make_uint2(to_e4m3x4(x[0] * r, x[1] * r, x[2] * r, x[3] * r), to_e4m3x4(x[4] * r, x[5] * r, x[6] * r, x[7] * r));
}

// ------------------------------------------------------------------------------------------------- rows --
// 16 lanes per block of 128 columns, PER blocks in a row per half warp: all their loads are in flight before the first is used.
// PER is 4, or 1 where that fills the chip no more than twice over.  Row i of the result is row i of x, or row rows[i] mod n_src
// (as an unsigned number, so that no index leaves x).
//
// Memory and instructions bound it alike: a thread's 32 elements were 496 instructions when every lane reduced each of its blocks
// by itself, found its scale and checked each element for the end, and 32768 gathered rows of 7168 bf16 took 121 us.  So the four
// blocks are reduced together (lane l ends with block l / 4's maximum, by 5 shuffles instead of 16) and each quad of lanes finds one
// block's factors: 98 us.  What is left of a gather waits for memory, so that resident warps count: 91 to 96 us with 8 CTAs an SM
// (32 registers) where 6 fit by themselves; two units a thread, the second's loads ahead of the first's work, or a ring of bulk
// copies before a few warps, were slower (118 and 129), as were column panels that stay in L2 (95 beside 91, at best).
constexpr int kRowThreads = 256;
template <class T, bool VEC, bool SWIGLU, int PER>                   // resident, by registers: what fits without spills, elsewhere
constexpr int kRowCtas = PER == 1 || (VEC && !SWIGLU && sizeof(T) == 2) ? 8 : (SWIGLU && (!VEC || sizeof(T) == 4)) ? 3 : 5;

// SWIGLU: x is [gate | up], 2 k columns, and what is quantised is SiLU(gate) * up in fp32.
template <class T, bool VEC, bool SWIGLU, int PER>
__global__ void __launch_bounds__(kRowThreads, kRowCtas<T, VEC, SWIGLU, PER>)
quantize_rows_kernel(const T* x, long long row_stride, const int* rows, uint32_t n_src, uint32_t total, uint32_t kb, uint8_t* q,
                     float* scale) {
    static_assert(PER == 1 || PER == 4, "");
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 15;
    // (total < 2^31, and the last CTA reaches less than 64 beyond it)
    const uint32_t first = (blockIdx.x * (kRowThreads / 16) + (threadIdx.x >> 4)) * PER;
    if (first - (threadIdx.x & 16 ? PER : 0) >= total) return;       // whole warps leave: the shuffles need all lanes
    auto source = [&](uint32_t row) {
        if (rows == nullptr) return row;
        const uint32_t src = (uint32_t)ld_global_s32(rows + row);
        return src < n_src ? src : src % n_src;
    };
    Eight<T> g[PER], u[SWIGLU ? PER : 1];
    uint32_t at = min(first, total - 1), row = at / kb, col = at - row * kb;
    const T* p = x + (long long)source(row) * row_stride + col * kBlock + lane * 8;
    if (col + PER <= kb && first + PER <= total) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            g[i].template load<VEC>(p + i * kBlock);
            if (SWIGLU) u[i].template load<VEC>(p + (size_t)kb * kBlock + i * kBlock);
        }
    } else {                                                        // over the ends of rows; what lies behind the last repeats it
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            g[i].template load<VEC>(p);
            if (SWIGLU) u[i].template load<VEC>(p + (size_t)kb * kBlock);
            if (at + 1 < total) {
                ++at;
                p += kBlock;
                if (++col == kb) {
                    col = 0;
                    p = x + (long long)source(++row) * row_stride + lane * 8;
                }
            }
        }
    }
    float v[PER][8], a[PER];
    bool far = false;               // a gate that takes the long way: then all of the thread's do
    if (SWIGLU) {
        float low = lowest_of(g[0]);
#pragma unroll
        for (int i = 1; i < PER; ++i) low = fminf(low, lowest_of(g[i]));
        far = low < kSiluLow;
    }
    if (far) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = swiglu_far(g[i].f(j), u[SWIGLU ? i : 0].f(j));
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = SWIGLU ? silu(g[i].f(j)) * u[SWIGLU ? i : 0].f(j) : g[i].f(j);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) a[i] = SWIGLU ? largest_of(v[i]) : largest_of(g[i]);
    uint8_t* to = q + (size_t)first * kBlock + lane * 8;
    if (PER == 4) {
        const bool up8 = lane & 8, up4 = lane & 4;
        float b = max_nan(up8 ? a[PER / 2] : a[0], __shfl_xor_sync(0xffffffffu, up8 ? a[0] : a[PER / 2], 8));
        float c = max_nan(up8 ? a[PER - 1] : a[PER / 4], __shfl_xor_sync(0xffffffffu, up8 ? a[PER / 4] : a[PER - 1], 8));
        b = max_nan(up4 ? c : b, __shfl_xor_sync(0xffffffffu, up4 ? b : c, 4));
        b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, 2));
        b = max_nan(max_nan(b, __shfl_xor_sync(0xffffffffu, b, 1)), kAmaxFloor);
        const float steps = steps_per_unit(b);
        if ((lane & 3) == 0 && first + (lane >> 2) < total) scale[first + (lane >> 2)] = over_448(b);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float r = __shfl_sync(0xffffffffu, steps, 4 * i, 16);
            if (first + i < total) *reinterpret_cast<uint2*>(to + i * kBlock) = to_e4m3x8(v[i], r);
        }
    } else {
        const float b = max_nan(half_warp_max(a[0]), kAmaxFloor);
        const uint2 o = to_e4m3x8(v[0], steps_per_unit(b));
        if (first < total) {
            *reinterpret_cast<uint2*>(to) = o;
            if (lane == 0) scale[first] = over_448(b);
        }
    }
}

// ----------------------------------------------------------------------------------------------- blocks --
// One CTA per 128 x 128 block; element (n, k) of matrix e lies at w[e * stride_e + n * stride_n + k * stride_k].  A thread
// holds 64 values: with k contiguous (KMAJOR) eight runs of eight along k, written as they are read; with n contiguous two
// pieces of 4 k x 8 n, whose bytes, four along k to a word, are turned round in shared memory.  Word (n, k/4) lies at
// word n * 32 + (k/4 ^ 2 (n/8 mod 16)): conflict-free for the 16 x 2 pieces that a warp writes, and pairs of words stay together.
constexpr int kBlockThreads = 256;

template <class T, bool VEC, bool KMAJOR>
__global__ void __launch_bounds__(kBlockThreads)
quantize_blocks_kernel(const T* w, long long stride_e, long long stride_n, long long stride_k, int n, int kb, uint8_t* q,
                       float* scale) {
    __shared__ float warp_max[kBlockThreads / 32];
    __shared__ uint32_t turned[KMAJOR ? 1 : kBlock * kBlock / 4];
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, k0 = blockIdx.x * kBlock, nb = blockIdx.y, e = blockIdx.z, n0 = nb * kBlock;
    const int left = n - n0;                                   // rows of w that the block still has
    w += e * stride_e + (long long)n0 * stride_n + (long long)k0 * stride_k;
    const long long k = (long long)kb * kBlock;
    q += ((long long)e * n + n0) * k + k0;
    Eight<T> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (KMAJOR) {
            const int r = i * 16 + (tid >> 4);
            v[i].template load<VEC>(w + r * stride_n + (tid & 15) * 8, r < left ? 8 : 0);
        } else {
            // piece i / 4: k rows 4 (tid / 16 + 16 (i / 4)) + i % 4, columns 8 (tid % 16) ..
            const int r = 4 * ((tid >> 4) + 16 * (i >> 2)) + (i & 3), c = 8 * (tid & 15);
            v[i].template load<VEC>(w + r * stride_k + c, left - c);
        }
    }
    float a = kAmaxFloor;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) a = max_nan(a, fabsf(v[i].f(j)));
    a = half_warp_max(a);
    a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 16));
    if ((tid & 31) == 0) warp_max[tid >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBlockThreads / 32; ++i) a = max_nan(a, warp_max[i]);
    const float r = steps_per_unit(a);
    if (tid == 0) scale[((long long)e * gridDim.y + nb) * kb + blockIdx.x] = over_448(a);
    if (KMAJOR) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = i * 16 + (tid >> 4);
            if (row < left)
                *reinterpret_cast<uint2*>(q + row * k + (tid & 15) * 8) =
                    make_uint2(to_e4m3x4(v[i].f(0) * r, v[i].f(1) * r, v[i].f(2) * r, v[i].f(3) * r),
                               to_e4m3x4(v[i].f(4) * r, v[i].f(5) * r, v[i].f(6) * r, v[i].f(7) * r));
        }
    } else {
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                turned[(8 * (tid & 15) + j) * 32 + (((tid >> 4) + 16 * p) ^ (2 * (tid & 15)))] =
                    to_e4m3x4(v[4 * p].f(j) * r, v[4 * p + 1].f(j) * r, v[4 * p + 2].f(j) * r, v[4 * p + 3].f(j) * r);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = i * 16 + (tid >> 4), pair = (tid & 15) ^ (row >> 3);
            if (row < left)
                *reinterpret_cast<uint2*>(q + row * k + (tid & 15) * 8) =
                    *reinterpret_cast<const uint2*>(&turned[row * 32 + 2 * pair]);
        }
    }
}

template <class T, int PER>
cudaError_t launch_rows(bool vec, bool swiglu, const void* x, long long row_stride, const int* rows, int n_src, int m, int k,
                        void* q, float* scale, cudaStream_t stream) {
    auto kernel = swiglu ? (vec ? quantize_rows_kernel<T, true, true, PER> : quantize_rows_kernel<T, false, true, PER>)
                         : (vec ? quantize_rows_kernel<T, true, false, PER> : quantize_rows_kernel<T, false, false, PER>);
    const uint32_t kb = (uint32_t)(k / kBlock), total = (uint32_t)m * kb, per_cta = kRowThreads / 16 * PER;
    return launch_kernel(kernel, dim3((total + per_cta - 1) / per_cta), kRowThreads, 0, stream, true, static_cast<const T*>(x),
                         row_stride, rows, (uint32_t)n_src, total, kb, static_cast<uint8_t*>(q), scale);
}

template <class T>
cudaError_t launch_blocks(bool vec, bool k_major, const void* w, int e, int n, int k, long long stride_e, long long stride_n,
                          long long stride_k, void* q, float* scale, cudaStream_t stream) {
    auto kernel = k_major ? (vec ? quantize_blocks_kernel<T, true, true> : quantize_blocks_kernel<T, false, true>)
                          : (vec ? quantize_blocks_kernel<T, true, false> : quantize_blocks_kernel<T, false, false>);
    const dim3 grid((unsigned)(k / kBlock), (unsigned)((n + kBlock - 1) / kBlock), (unsigned)e);
    return launch_kernel(kernel, grid, kBlockThreads, 0, stream, true, static_cast<const T*>(w), stride_e, stride_n, stride_k, n,
                         k / kBlock, static_cast<uint8_t*>(q), scale);
}

int element_bytes(int dtype) { return dtype == RF_F16 || dtype == RF_BF16 ? 2 : dtype == RF_F32 ? 4 : 0; }

// x's rows can be read 16 bytes at a time
bool rows_aligned(const void* x, long long row_stride, int bytes) {
    return !misaligned({x}, 16) && (row_stride * bytes) % 16 == 0;
}

int quantize_rows(bool swiglu, const void* x, int dtype, long long row_stride, const int* rows, int n_src, int m, int k,
                  void* q, float* scale, rf_stream_t stream) {
    const int bytes = element_bytes(dtype);
    if (bytes == 0) return RF_ERR_UNSUPPORTED;
    if (m < 0 || k <= 0 || k % kBlock != 0 || (long long)m * (k / kBlock) > 0x7fffffffLL) return RF_ERR_BAD_SHAPE;
    if (rows != nullptr && n_src <= 0 && m > 0) return RF_ERR_BAD_SHAPE;
    if (m == 0) return RF_OK;
    if (!x || !q || !scale) return RF_ERR_NULL_POINTER;
    if (misaligned({q}, 16) || misaligned({scale, rows}, 4) || misaligned({x}, (unsigned)bytes)) return RF_ERR_MISALIGNED;
    DeviceState* st = device_state();
    if (!st) return RF_ERR_CUDA;
    const bool vec = rows_aligned(x, row_stride, bytes);
    // 24 x 7168: 1344 blocks on 84 CTAs instead of 21
    const bool few = (long long)m * (k / kBlock) <= 2LL * st->num_sms * (kRowThreads / 16);
    auto run = dtype == RF_F16    ? (few ? launch_rows<__half, 1> : launch_rows<__half, 4>)
               : dtype == RF_BF16 ? (few ? launch_rows<__nv_bfloat16, 1> : launch_rows<__nv_bfloat16, 4>)
                                  : (few ? launch_rows<float, 1> : launch_rows<float, 4>);
    return run(vec, swiglu, x, row_stride, rows, n_src, m, k, q, scale, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess
               ? RF_OK : RF_ERR_CUDA;
}

}  // namespace

}  // namespace rf

extern "C" {

int rf_fp8_quantize(const void* x, int dtype, long long row_stride, const int* rows, int n_src, int m, int k, void* q,
                    float* scale, rf_stream_t stream) {
    return rf::quantize_rows(false, x, dtype, row_stride, rows, n_src, m, k, q, scale, stream);
}

int rf_fp8_swiglu_quantize(const void* gate_up, int dtype, long long row_stride, int m, int f, void* q, float* scale,
                           rf_stream_t stream) {
    return rf::quantize_rows(true, gate_up, dtype, row_stride, nullptr, 0, m, f, q, scale, stream);
}

int rf_fp8_quantize_blocks(const void* w, int dtype, int e, int n, int k, long long stride_e, long long stride_n,
                           long long stride_k, void* q, float* scale, rf_stream_t stream) {
    const int bytes = rf::element_bytes(dtype);
    if (bytes == 0) return RF_ERR_UNSUPPORTED;
    // (the grid's second and third dimension hold 65535 blocks)
    if (e < 0 || e > 65535 || n < 0 || n > 65535 * 128 || k <= 0 || k % 128 != 0) return RF_ERR_BAD_SHAPE;
    if (stride_k != 1 && stride_n != 1) return RF_ERR_UNSUPPORTED;
    if (e == 0 || n == 0) return RF_OK;
    if (!w || !q || !scale) return RF_ERR_NULL_POINTER;
    if (rf::misaligned({q}, 16) || rf::misaligned({scale}, 4) || rf::misaligned({w}, (unsigned)bytes)) return RF_ERR_MISALIGNED;
    if (!rf::device_state()) return RF_ERR_CUDA;
    const bool k_major = stride_k == 1;
    const bool vec = rf::rows_aligned(w, k_major ? stride_n : stride_k, bytes) && (e == 1 || (stride_e * bytes) % 16 == 0);
    auto run = dtype == RF_F16 ? rf::launch_blocks<__half> : dtype == RF_BF16 ? rf::launch_blocks<__nv_bfloat16> : rf::launch_blocks<float>;
    return run(vec, k_major, w, e, n, k, stride_e, stride_n, stride_k, q, scale, reinterpret_cast<cudaStream_t>(stream)) ==
                   cudaSuccess ? RF_OK : RF_ERR_CUDA;
}

}  // extern "C"
