// A whole MoE layer for a few tokens (a decode step) in one kernel, sm_100a: router, softmax and top-k, SwiGLU experts, shared
// expert, weighted sum.
//
//   logits = fp16(x Wr^T + bias),  p = fp16(softmax(logits)),  the top_k largest p (equal ones: the lowest index)
//   h_e = (x Wg_e) / (1 + exp(-x Wg_e)) * (x Wu_e),  out = fp16(sum_i p_i h_i Wd_i + h_shared Wd_shared)
//
// What bounds it is the weight stream: each weight of every expert that a token chose is read once and used for a handful of
// multiplications.  So one persistent CTA per SM keeps a ring of TMA loads full from the first microsecond to the last, and all
// that depends on something else happens beside it.  The work is a list of items, dealt out by a ticket in this order:
//   router units   16 experts x 512 columns of the logits, partial sums
//   first product  64 columns of gate and the same of up x a chunk of K, the shared expert's first (they need no routing)
//   second product 128 columns of the result x a chunk of K
// An item depends on items with smaller tickets only, and a CTA works its tickets off in order, so whatever share of the grid is
// running makes progress, and the loads of an item never wait for its dependencies.  K chunks meet as fp32 partial sums in the
// workspace; who finishes the last chunk of a column tile adds them up, in the order of the chunks, and likewise the last item of
// a result tile adds the experts in rank order: results are the same bits whoever comes last.  Warps of a CTA:
//   0      draws tickets, issues the weight loads (16 KB stages)
//   1-3    the items' token rows (or, for the second product, h, once the expert's first is complete) into shared memory
//   4-11   mma.sync m16n8k16, weights as the 16-row operand, up to 8 tokens as the 8 columns: a warp owns 16 of the item's 128
//          columns.  (The legacy tensor path on purpose: the stream feeds one such MMA per 21 cycles and SM, and its
//          accumulators need no trip through TMEM.)  FP8 weights become fp16 on the way, their scale is applied per 128 of K.
//   12-15  publish finished items, add up what is complete
//   16-19  softmax, top-k and the experts' token lists, in every CTA for itself, once the logits are complete
// h is rounded to fp16, the type of the second product's operand; everything else is fp32.
#include "moe_few.h"
#include "launch.h"
#include "ptx.cuh"
#include "softmax_exp.cuh"

namespace rf {

namespace {

constexpr int WARP_X = 1, WARP_MMA = 4, WARP_PUB = 12, WARP_ROUTE = 16, WARPS = 20;
constexpr int X_WARPS = WARP_MMA - WARP_X, MMA_WARPS = WARP_PUB - WARP_MMA;
constexpr int THREADS = 32 * WARPS;
constexpr int BAR_MMA = 1, BAR_PUB = 2, BAR_ROUTE = 3;
constexpr int STAGE_BYTES = 16384, BOX_BYTES = 8192;
constexpr int ITEM_SLOTS = 8;
constexpr int DRAW_AHEAD = 4;           // stages before an item's last load at which the next ticket is drawn
constexpr int MAX_PAIRS = kFewMaxTokens * kFewMaxTopK;

enum ItemKind { kRouter = 0, kFirst = 1, kSecond = 2, kEnd = 3 };
// kind, expert slot (index into the active list, -1 = shared), column tile, K chunk
using Item = int4;

struct Routing {
    int n_active;
    int active[kFewMaxExperts];         // experts with tokens, ascending
    int base[kFewMaxExperts + 1];       // first pair of each of them; pairs are sorted by expert, then token
    int token[MAX_PAIRS];               // of a pair
    int expert[MAX_PAIRS];              // [token][rank]
    int pos[MAX_PAIRS];                 // pair of [token][rank]
    float weight[MAX_PAIRS];            // [token][rank]
    int sums[4];
    int last;                           // publishers: whether the item was the last of its tile
};

template <bool FP8, int NG>
struct Cfg {
    static constexpr int kStageK = FP8 ? 128 : 64;
    static constexpr int kRows = 8 * NG;
    static constexpr int kMaxChunk = NG == 4 ? 512 : 1024;
    // fp16 operands go through ldmatrix (rows 16 bytes apart modulo 128), those of FP8 through 8-byte loads (32 bytes)
    static constexpr int kPad = FP8 ? 32 : 16;
    static constexpr int kXStride = kMaxChunk * 2 + kPad;
    static constexpr int kXBytes = kRows * kXStride;
    static constexpr int kRedBytes = MMA_WARPS * 16 * kRows * 4;
    static constexpr int kStages = NG == 1 ? 11 : 8;
    static constexpr int kBars = 2 * kStages + 4 + 3 * ITEM_SLOTS + 1;
    static constexpr int kSmemBytes = kStages * STAGE_BYTES + 2 * kXBytes + kRedBytes + ITEM_SLOTS * 16 + kBars * 8 +
                                      (int)sizeof(Routing) + 1024;
    static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

__device__ __forceinline__ int ld_acquire_gpu_s32(const int* p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// Bounded wait for *p >= want (limit, status word and unwinding as in mbar_wait).
__device__ __forceinline__ bool counter_wait(const int* p, int want, int* status, int code, int tag) {
    unsigned long long t0 = 0;
    for (uint32_t it = 1;; ++it) {
        if (ld_acquire_gpu_s32(p) >= want) return true;
        if ((it & 0x3fu) == 0) {
            const int seen = *reinterpret_cast<volatile int*>(status);
            if (seen != 0 && (seen >> kStatusTagShift) == tag) return false;
            const unsigned long long now = globaltimer_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > wait_limit_ns(status)) {
                atomicCAS(status, 0, code | (tag << kStatusTagShift));
                return false;
            }
        }
    }
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
__device__ __forceinline__ float2 ld_cg_f2(const float* p) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float ld_cg_f(const float* p) {
    float v;
    asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}

// How the work divides: known once the routing is.
struct Shape {
    int tiles1, tiles1s;        // column tiles of the first product: of an expert, of the shared one
    int tiles2;
    int chunks1, chunks2, chunks2s;
    __device__ __forceinline__ explicit Shape(const MoeFewParams& p)
        : tiles1(p.f / 64), tiles1s(p.fs / 64), tiles2((p.d + 127) / 128), chunks1((p.d + p.kc1 - 1) / p.kc1),
          chunks2((p.f + p.kc2 - 1) / p.kc2), chunks2s((p.fs + p.kc2 - 1) / p.kc2) {}
};

// Tickets beyond the router's and the shared expert's first product (`r` counts from there) -> item.  Column tiles run fastest,
// so that the CTAs at work read neighbouring columns of the same rows.
__device__ __forceinline__ Item decode_routed(int r, const Shape& s, int n_active) {
    const int per1 = s.tiles1 * s.chunks1;
    if (r < n_active * per1) {
        const int e = r / per1, i = r - e * per1, c = i / s.tiles1;
        return make_int4(kFirst, e, i - c * s.tiles1, c);
    }
    r -= n_active * per1;
    if (r < s.tiles2 * s.chunks2s) {
        const int c = r / s.tiles2;
        return make_int4(kSecond, -1, r - c * s.tiles2, c);
    }
    r -= s.tiles2 * s.chunks2s;
    const int per2 = s.tiles2 * s.chunks2;
    if (r < n_active * per2) {
        const int e = r / per2, i = r - e * per2, c = i / s.tiles2;
        return make_int4(kSecond, e, i - c * s.tiles2, c);
    }
    return make_int4(kEnd, 0, 0, 0);
}

template <bool FP8, int NG>
__global__ void __launch_bounds__(THREADS, 1)
moe_few_kernel(const MoeFewParams p) {
    using C = Cfg<FP8, NG>;
    constexpr int STAGES = C::kStages;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t x_base = smem_base + STAGES * STAGE_BYTES;
    const uint32_t red_base = x_base + 2 * C::kXBytes;
    const uint32_t item_base = red_base + C::kRedBytes;
    const uint32_t bar_base = item_base + ITEM_SLOTS * 16;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto x_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto x_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
    auto item_bar = [&](uint32_t j) { return bar_base + 8u * (2 * STAGES + 4 + j % ITEM_SLOTS); };
    auto done_bar = [&](uint32_t j) { return bar_base + 8u * (2 * STAGES + 4 + ITEM_SLOTS + j % ITEM_SLOTS); };
    auto free_bar = [&](uint32_t j) { return bar_base + 8u * (2 * STAGES + 4 + 2 * ITEM_SLOTS + j % ITEM_SLOTS); };
    const uint32_t routed_bar = bar_base + 8u * (2 * STAGES + 4 + 3 * ITEM_SLOTS);
    auto at = [&](uint32_t addr) { return smem_raw + (addr - smem_u32(smem_raw)); };
    Routing& rt = *reinterpret_cast<Routing*>(at(bar_base + 8u * C::kBars));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    griddep_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), MMA_WARPS);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(x_full_bar(b), X_WARPS);
            mbar_init(x_empty_bar(b), MMA_WARPS);
        }
        for (int j = 0; j < ITEM_SLOTS; ++j) {
            mbar_init(item_bar(j), 1);
            mbar_init(done_bar(j), MMA_WARPS);
            mbar_init(free_bar(j), X_WARPS + MMA_WARPS + 1);
        }
        mbar_init(routed_bar, 1);
        mbar_fence_init();
    }
    griddep_wait();
    // A workspace in which an earlier call lost a wait holds counts that belong to nothing: no result then, and a code.
    const int bad = __syncthreads_or(ld_global_s32(p.head + kFewBad) != 0);
    if (bad) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0, kErrSchedWait | (p.launch_tag << kStatusTagShift));
        return;
    }

    const Shape shape(p);
    const int shared_first = shape.tiles1s * shape.chunks1;
    const int before_routed = p.router_units + shared_first;
    const int pairs = p.t * p.top_k;            // the shared expert's pairs come behind them, one per token
    int* const done1 = p.head + kFewHeadWords;
    auto wait_routed = [&](int code) { return mbar_wait(routed_bar, 0, p.status, code, p.launch_tag); };
    auto wait_item = [&](uint32_t j, int code) {
        return mbar_wait(item_bar(j), (j / ITEM_SLOTS) & 1, p.status, code, p.launch_tag);
    };
    auto get_item = [&](uint32_t j) {
        const uint4 v = ld_shared_v4(item_base + 16u * (j % ITEM_SLOTS));
        return make_int4((int)v.x, (int)v.y, (int)v.z, (int)v.w);
    };
    // K range of an item
    auto k_range = [&](const Item& it, int* k0, int* len) {
        const int kc = it.x == kFirst ? p.kc1 : p.kc2;
        const int k = it.x == kFirst ? p.d : it.y < 0 ? p.fs : p.f;
        *k0 = it.w * kc;
        *len = min(kc, k - *k0);
    };
    auto expert_of = [&](const Item& it) { return it.y < 0 ? p.experts : rt.active[it.y]; };
    auto first_pair = [&](const Item& it) { return it.y < 0 ? pairs : rt.base[it.y]; };
    auto pair_count = [&](const Item& it) { return it.y < 0 ? p.t : rt.base[it.y + 1] - rt.base[it.y]; };

    bool lost = false;          // this thread's role gave a wait up
    if (warp == 0) {
        // ------------------------------------------------------------------------------ tickets, weight loads
        if (lane == 0) {
            uint32_t st = 0, s = 0, ph = 1;
            bool ok = true, routed = false;
            int ticket = atomicAdd(p.head + kFewTicket, 1);
            for (uint32_t j = 0; ok; ++j) {
                Item it;
                if (ticket < p.router_units) {
                    it = make_int4(kRouter, 0, ticket, 0);
                } else if (ticket < before_routed) {
                    const int i = ticket - p.router_units, c = i / shape.tiles1s;
                    it = make_int4(kFirst, -1, i - c * shape.tiles1s, c);
                } else {
                    if (!routed) {
                        ok = wait_routed(kErrProducerWait);
                        if (!ok) break;
                        routed = true;
                    }
                    it = decode_routed(ticket - before_routed, shape, rt.n_active);
                }
                ok = mbar_wait(free_bar(j), ((j / ITEM_SLOTS) & 1) ^ 1, p.status, kErrProducerWait, p.launch_tag);
                if (!ok) break;
                st_shared_v4(item_base + 16u * (j % ITEM_SLOTS), it.x, it.y, it.z, it.w);
                mbar_arrive(item_bar(j));
                if (it.x == kEnd) break;
                if (it.x == kRouter) {
                    ticket = atomicAdd(p.head + kFewTicket, 1);
                    continue;
                }
                const int e = expert_of(it);
                int k0, len;
                k_range(it, &k0, &len);
                const CUtensorMap* m0 = p.maps + 3 * e + (it.x == kFirst ? 0 : 2);
                const CUtensorMap* m1 = it.x == kFirst ? m0 + 1 : m0;
                const int n0 = it.x == kFirst ? it.z * 64 : it.z * 128, n1 = it.x == kFirst ? n0 : n0 + 64;
                const int n_stages = len / C::kStageK;
                for (int i = 0; i < n_stages; ++i, ++st) {
                    if (i == max(n_stages - DRAW_AHEAD, 0)) ticket = atomicAdd(p.head + kFewTicket, 1);
                    ok = mbar_wait(empty_bar(s), ph, p.status, kErrProducerWait, p.launch_tag);
                    if (!ok) break;
                    const uint32_t dst = smem_base + s * STAGE_BYTES;
                    const int k = k0 + i * C::kStageK;
                    mbar_expect_tx(full_bar(s), STAGE_BYTES);
                    tma_load_2d(dst, m0, full_bar(s), FP8 ? k : n0, FP8 ? n0 : k);
                    tma_load_2d(dst + BOX_BYTES, m1, full_bar(s), FP8 ? k : n1, FP8 ? n1 : k);
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
            finish_producer(ok, st, STAGES, empty_bar(0), p.status, kErrProducerWait, p.launch_tag);
            lost = !ok;
        }
        __syncwarp();
    } else if (warp < WARP_MMA) {
        // ------------------------------------------------------------------------------ token rows
        const int tid = threadIdx.x - 32 * WARP_X;
        bool ok = true, routed = false;
        uint32_t n = 0;         // items with rows so far
        for (uint32_t j = 0; ok; ++j) {
            ok = __all_sync(0xffffffffu, wait_item(j, kErrMmaWaitFull));
            if (!ok) break;
            const Item it = get_item(j);
            __syncwarp();
            if (lane == 0) mbar_arrive(free_bar(j));
            if (it.x == kEnd) break;
            if (it.x == kRouter) continue;
            if (it.y >= 0 && !routed) {
                ok = __all_sync(0xffffffffu, wait_routed(kErrMmaWaitFull));
                if (!ok) break;
                routed = true;
            }
            int k0, len;
            k_range(it, &k0, &len);
            const uint32_t b = n & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(x_empty_bar(b), ((n >> 1) & 1) ^ 1, p.status, kErrMmaWaitFull, p.launch_tag));
            if (!ok) break;
            const int n_rows = pair_count(it), first = first_pair(it);
            const __half* src;
            size_t stride;
            if (it.x == kFirst) {
                src = static_cast<const __half*>(p.x) + k0;
                stride = p.d;
            } else {
                const int e = expert_of(it);
                if (lane == 0)
                    ok = counter_wait(done1 + e, it.y < 0 ? shape.tiles1s : shape.tiles1, p.status, kErrSchedWait, p.launch_tag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                src = static_cast<const __half*>(p.h) + (size_t)first * p.width + k0;
                stride = p.width;
            }
            const int vecs = len >> 3;
            const uint32_t dst = x_base + b * C::kXBytes;
            const bool gather = it.x == kFirst && it.y >= 0;
#pragma unroll 4
            for (int i = tid; i < n_rows * vecs; i += 32 * X_WARPS) {
                const int r = i / vecs, v = i - r * vecs;
                const int row = gather ? rt.token[first + r] : r;
                const uint4 q = ld_global_cg_v4(src + (size_t)row * stride + 8 * v);
                st_shared_v4(dst + r * C::kXStride + 16 * v, q.x, q.y, q.z, q.w);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(x_full_bar(b));
            ++n;
        }
        lost = !ok;
        // This CTA draws no ticket, and this warp waits for no counter any more: the last warp to come here clears them for the
        // next call.  (Where a wait was lost the workspace is marked below, and its next call refuses to run.)
        if (ok) {
            int last = 0;
            if (lane == 0) last = atomicAdd(p.head + kFewExits, 1) == (int)gridDim.x * X_WARPS - 1;
            if (__shfl_sync(0xffffffffu, last, 0)) {
                if (lane < 3) p.head[lane] = 0;             // ticket, router units done, exits
                for (int e = lane; e <= p.experts; e += 32) done1[e] = 0;
            }
        }
    } else if (warp < WARP_PUB) {
        // ------------------------------------------------------------------------------ MMA
        const int w = warp - WARP_MMA;
        const int g = lane >> 2, q = lane & 3;      // row (column) of the fragments, pair inside
        const uint32_t box = (w >> 2) * BOX_BYTES;
        bool ok = true, routed = false;
        uint32_t n = 0, s = 0, ph = 0;
        for (uint32_t j = 0;; ++j) {
            ok = ok && wait_item(j, kErrMmaWaitFull);
            Item it = get_item(j);
            if (ok && it.x != kRouter && it.x != kEnd && it.y >= 0 && !routed) {
                ok = wait_routed(kErrMmaWaitFull);
                routed = true;
            }
            ok = named_barrier_all(BAR_MMA, 32 * MMA_WARPS, ok);       // all of the group go on, or none: they meet at barriers below
            if (!ok) break;
            if (lane == 0) mbar_arrive(free_bar(j));
            if (it.x == kEnd) break;
            if (it.x == kRouter) {
                // 16 experts x 512 columns, 64 of them per warp.  A lane holds 16 consecutive k of its row (and token): the
                // order of k inside a fragment is free as long as both operands share it.
                const int e0 = it.z / p.router_chunks * 16, c = it.z % p.router_chunks;
                const int k = c * kFewRouterChunk + w * 64;
                float acc[NG][4] = {};
                if (k < p.d) {
                    uint4 a[2][2], b[NG][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const __half* row = static_cast<const __half*>(p.router) + (size_t)min(e0 + g + 8 * i, p.experts - 1) * p.d;
#pragma unroll
                        for (int v = 0; v < 2; ++v) a[i][v] = ld_global_cg_v4(row + k + 16 * q + 8 * v);
                    }
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const __half* row = static_cast<const __half*>(p.x) + (size_t)min(8 * i + g, p.t - 1) * p.d;
#pragma unroll
                        for (int v = 0; v < 2; ++v) b[i][v] = ld_global_cg_v4(row + k + 16 * q + 8 * v);
                    }
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const uint32_t lo[4] = {a[0][v].x, a[1][v].x, a[0][v].y, a[1][v].y};
                        const uint32_t hi[4] = {a[0][v].z, a[1][v].z, a[0][v].w, a[1][v].w};
#pragma unroll
                        for (int i = 0; i < NG; ++i) {
                            mma_f16(acc[i], lo, b[i][v].x, b[i][v].y);
                            mma_f16(acc[i], hi, b[i][v].z, b[i][v].w);
                        }
                    }
                }
                // [warp][expert][token]
                const uint32_t mine = red_base + w * (16 * C::kRows * 4);
#pragma unroll
                for (int i = 0; i < NG; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        st_shared_f32(mine + ((g + 8 * (v >> 1)) * C::kRows + 8 * i + 2 * q + (v & 1)) * 4, acc[i][v]);
                named_barrier(BAR_MMA, 32 * MMA_WARPS);
                for (int i = w * 32 + lane; i < 16 * C::kRows; i += 32 * MMA_WARPS) {
                    const int e = e0 + i / C::kRows, t = i % C::kRows;
                    float v = 0.f;
#pragma unroll
                    for (int o = 0; o < MMA_WARPS; ++o)
                        v += __uint_as_float(ld_shared_u32(red_base + (o * 16 * C::kRows + i) * 4));
                    if (e < p.experts && t < p.t) p.logits[((size_t)c * p.t + t) * p.experts + e] = v;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(done_bar(j));
                continue;
            }
            int k0, len;
            k_range(it, &k0, &len);
            const int n_rows = pair_count(it), first = first_pair(it);
            const uint32_t b = n & 1;
            float scale = 0.f;
            if (FP8) {
                // lane i holds the scale of the chunk's i-th 128 of K
                const int m = it.x == kFirst ? (w >> 2) : 2, k = it.x == kFirst ? p.d : it.y < 0 ? p.fs : p.f;
                const int block = it.x == kFirst ? it.z >> 1 : it.z;
                if (lane < len / 128)
                    scale = ld_global_f32(p.scales[3 * expert_of(it) + m] + (size_t)block * (k / 128) + k0 / 128 + lane);
            }
            ok = __all_sync(0xffffffffu, mbar_wait(x_full_bar(b), (n >> 1) & 1, p.status, kErrMmaWaitFull, p.launch_tag));
            const uint32_t xb = x_base + b * C::kXBytes;
            const int groups = (n_rows + 7) >> 3;
            float acc[NG][4] = {};
            const int n_stages = len / C::kStageK;
            for (int i = 0; i < n_stages && ok; ++i) {
                ok = __all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, p.status, kErrMmaWaitFull, p.launch_tag));
                if (!ok) break;
                const uint32_t wb = smem_base + s * STAGE_BYTES + box;
                if (FP8) {
                    // rows are output columns; a lane takes 4 consecutive k of its two rows per MMA
                    float part[NG][4] = {};
                    const int r0 = (w & 3) * 16 + g;
                    const uint32_t row = wb + r0 * 128 + 4 * q;
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t off = (uint32_t)((kk ^ (r0 & 7)) << 4);
                        const uint32_t lo = ld_shared_u32(row + off), hi = ld_shared_u32(row + 8 * 128 + off);
                        const uint32_t a[4] = {f16x2_of_e4m3x2((uint16_t)lo), f16x2_of_e4m3x2((uint16_t)hi),
                                               f16x2_of_e4m3x2((uint16_t)(lo >> 16)), f16x2_of_e4m3x2((uint16_t)(hi >> 16))};
#pragma unroll
                        for (int u = 0; u < NG; ++u) {
                            if (u >= groups) break;
                            const uint2 x = ld_shared_v2(xb + (8 * u + g) * C::kXStride + 2 * (i * 128 + kk * 16 + 4 * q));
                            mma_f16(part[u], a, x.x, x.y);
                        }
                    }
                    const float sc = __shfl_sync(0xffffffffu, scale, i);
#pragma unroll
                    for (int u = 0; u < NG; ++u)
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(sc, part[u][v], acc[u][v]);
                } else {
                    // rows are k; transposed 8 x 8 pieces give the weights as [column][k] fragments
                    const int kr = (lane & 7) + 8 * (lane >> 4), chunk = 2 * (w & 3) + ((lane >> 3) & 1);
                    const uint32_t wa = wb + kr * 128 + ((chunk ^ (kr & 7)) << 4);
                    const uint32_t xa = xb + (lane & 7) * C::kXStride + 2 * (i * 64 + 8 * (lane >> 3));
                    uint32_t x[2][NG][4];
#pragma unroll
                    for (int v = 0; v < 2; ++v)
#pragma unroll
                        for (int u = 0; u < NG; ++u)
                            if (u < groups) ldmatrix_x4(xa + u * 8 * C::kXStride + v * 64, x[v][u]);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        uint32_t a[4];
                        ldmatrix_x4_trans(wa + kk * 16 * 128, a);
#pragma unroll
                        for (int u = 0; u < NG; ++u)
                            if (u < groups) mma_f16(acc[u], a, x[kk >> 1][u][2 * (kk & 1)], x[kk >> 1][u][2 * (kk & 1) + 1]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty_bar(s));
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            if (ok) {
                float* dst;
                size_t stride;
                if (it.x == kFirst) {
                    stride = 2 * (size_t)p.width;
                    dst = p.part1 + ((size_t)it.w * (pairs + p.t) + first) * stride + it.z * 128 + w * 16;
                } else {
                    stride = p.d;
                    dst = p.part2 + ((size_t)it.w * (pairs + p.t) + first) * stride + it.z * 128 + w * 16;
                }
                const bool inside = it.x == kFirst || it.z * 128 + w * 16 < p.d;
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        const int r = 8 * u + 2 * q + (v & 1);
                        if (r < n_rows && inside) dst[r * stride + g + 8 * (v >> 1)] = acc[u][v];
                    }
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(x_empty_bar(b));
                mbar_arrive(done_bar(j));
            }
            ++n;
        }
        lost = !ok;
    } else if (warp < WARP_ROUTE) {
        // ------------------------------------------------------------------------------ finished items
        const int w = warp - WARP_PUB;
        bool ok = true;
        for (uint32_t j = 0;; ++j) {
            ok = ok && wait_item(j, kErrEpilogueWait);
            const Item it = get_item(j);
            if (ok && it.x != kEnd)
                ok = mbar_wait(done_bar(j), (j / ITEM_SLOTS) & 1, p.status, kErrEpilogueWait, p.launch_tag);
            if (ok && it.x == kSecond) ok = wait_routed(kErrEpilogueWait);
            ok = named_barrier_all(BAR_PUB, 128, ok);
            if (!ok || it.x == kEnd) break;
            if (it.x == kRouter) {
                if (w == 0 && lane == 0) {
                    __threadfence();
                    atomicAdd(p.head + kFewRouterDone, 1);
                }
            } else {
                const int e = it.x == kFirst ? expert_of(it) : 0;
                int* const count = it.x == kFirst ? p.count1 + e * p.tiles1_max + it.z : p.count2 + it.z;
                const int want = it.x == kFirst ? shape.chunks1 : rt.n_active * shape.chunks2 + shape.chunks2s;
                if (w == 0 && lane == 0) {
                    __threadfence();
                    const bool last = atomicAdd(count, 1) == want - 1;
                    if (last) *count = 0;       // for the next call; nobody else comes here in this one
                    __threadfence();
                    rt.last = last;
                }
                named_barrier(BAR_PUB, 128);
                if (rt.last) {
                    const size_t rows = pairs + p.t;
                    if (it.x == kFirst) {
                        const int n_rows = pair_count(it), first = first_pair(it);
                        for (int r = w; r < n_rows; r += 4) {
                            const float* src = p.part1 + (size_t)(first + r) * 2 * p.width + it.z * 128 + 2 * lane;
                            float2 gate = make_float2(0.f, 0.f), up = gate;
#pragma unroll 8
                            for (int c = 0; c < shape.chunks1; ++c) {
                                const float2 a = ld_cg_f2(src + c * rows * 2 * p.width), b = ld_cg_f2(src + c * rows * 2 * p.width + 64);
                                gate.x += a.x; gate.y += a.y;
                                up.x += b.x; up.y += b.y;
                            }
                            const float hx = gate.x / (1.0f + expf(-gate.x)) * up.x, hy = gate.y / (1.0f + expf(-gate.y)) * up.y;
                            *reinterpret_cast<uint32_t*>(static_cast<__half*>(p.h) + (size_t)(first + r) * p.width + it.z * 64 + 2 * lane) =
                                pack_f16x2(hx, hy);
                        }
                        named_barrier(BAR_PUB, 128);
                        if (w == 0 && lane == 0) {
                            __threadfence();
                            atomicAdd(done1 + e, 1);
                        }
                    } else {
                        const int col = it.z * 128 + 4 * lane;
                        for (int t = w; t < p.t && col < p.d; t += 4) {
                            float4 y[kFewMaxTopK];
#pragma unroll
                            for (int i = 0; i < kFewMaxTopK; ++i) y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                            for (int c = 0; c < shape.chunks2; ++c)
#pragma unroll
                                for (int i = 0; i < kFewMaxTopK; ++i)
                                    if (i < p.top_k) {
                                        const float4 v = ld_global_cg_v4_f32(p.part2 + (c * rows + rt.pos[t * p.top_k + i]) * p.d + col);
                                        y[i].x += v.x; y[i].y += v.y; y[i].z += v.z; y[i].w += v.w;
                                    }
                            float4 o = make_float4(0.f, 0.f, 0.f, 0.f), sh = o;
#pragma unroll
                            for (int i = 0; i < kFewMaxTopK; ++i)
                                if (i < p.top_k) {
                                    const float wt = rt.weight[t * p.top_k + i];
                                    o.x = fmaf(wt, y[i].x, o.x); o.y = fmaf(wt, y[i].y, o.y);
                                    o.z = fmaf(wt, y[i].z, o.z); o.w = fmaf(wt, y[i].w, o.w);
                                }
                            for (int c = 0; c < shape.chunks2s; ++c) {
                                const float4 v = ld_global_cg_v4_f32(p.part2 + (c * rows + pairs + t) * p.d + col);
                                sh.x += v.x; sh.y += v.y; sh.z += v.z; sh.w += v.w;
                            }
                            *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + (size_t)t * p.d + col) =
                                make_uint2(pack_f16x2(o.x + sh.x, o.y + sh.y), pack_f16x2(o.z + sh.z, o.w + sh.w));
                        }
                    }
                }
            }
            named_barrier(BAR_PUB, 128);        // rt.last has been read
            if (w == 0 && lane == 0) mbar_arrive(free_bar(j));
        }
        lost = !ok;
    } else {
        // ------------------------------------------------------------------------------ routing
        const int w = warp - WARP_ROUTE, tid = w * 32 + lane;
        bool ok = true;
        if (lane == 0) ok = counter_wait(p.head + kFewRouterDone, p.router_units, p.status, kErrSchedWait, p.launch_tag);
        ok = named_barrier_all(BAR_ROUTE, 128, ok);
        if (ok) {
            // softmax and top-k as topk_kernel (moe_route.cu) does them, on the same fp16 roundings: lane l owns experts
            // l * vpt ..; a key is an fp16 probability, then the complement of the expert's number
            const int vpt = p.experts <= 32 ? 1 : p.experts / 32, e0 = lane * vpt;
            const bool active = e0 < p.experts;
            for (int t = w; t < p.t; t += 4) {
                float l[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) l[i] = 0.f;
                for (int c = 0; c < p.router_chunks; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (active && i < vpt) l[i] += ld_cg_f(p.logits + ((size_t)c * p.t + t) * p.experts + e0 + i);
                float mx = -65504.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (active && i < vpt) {
                        if (p.router_bias != nullptr) l[i] += ld_global_f32(p.router_bias + e0 + i);
                        l[i] = __half2float(__float2half_rn(l[i]));
                        mx = fmaxf(mx, l[i]);
                    }
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
                float part = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < vpt) {
                        l[i] = active ? det_exp(__fsub_rn(l[i], mx)) : 0.f;
                        part = i == 0 ? l[0] : __fadd_rn(part, l[i]);
                    }
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) part = __fadd_rn(part, __shfl_xor_sync(0xffffffffu, part, s));
                const float recip = __fdiv_rn(1.0f, part);
                uint32_t key[8], mine = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    key[i] = active && i < vpt ? ((uint32_t)__half_as_ushort(__float2half_rn(__fmul_rn(l[i], recip))) << 16) |
                                                     (0xFFFFu - (uint32_t)(e0 + i))
                                               : 0u;
                for (int k = 0; k < p.top_k; ++k) {
                    uint32_t best = key[0];
#pragma unroll
                    for (int i = 1; i < 8; ++i) best = max(best, key[i]);
                    best = __reduce_max_sync(0xffffffffu, best);
                    if (lane == k) mine = best;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (key[i] == best) key[i] = 0u;
                }
                if (lane < p.top_k) {
                    rt.expert[t * p.top_k + lane] = (int)(0xFFFFu - (mine & 0xFFFFu));
                    rt.weight[t * p.top_k + lane] = __half2float(__ushort_as_half((unsigned short)(mine >> 16)));
                }
            }
            named_barrier(BAR_ROUTE, 128);
            // the experts' token lists: a thread counts for two experts
            int n[2] = {0, 0};
            for (int i = 0; i < pairs; ++i) {
                const int e = rt.expert[i];
                n[0] += e == 2 * tid;
                n[1] += e == 2 * tid + 1;
            }
            // pairs before (low half) and active experts before (high half)
            const int mine = n[0] + n[1] + ((n[0] > 0) << 16) + ((n[1] > 0) << 16);
            int incl = mine;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, incl, s);
                if (lane >= s) incl += o;
            }
            if (lane == 31) rt.sums[w] = incl;
            named_barrier(BAR_ROUTE, 128);
            int before = incl - mine;
            for (int i = 0; i < w; ++i) before += rt.sums[i];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (n[i] == 0) continue;
                const int slot = before >> 16;
                int pair = before & 0xFFFF;
                rt.active[slot] = 2 * tid + i;
                rt.base[slot] = pair;
                for (int o = 0; o < pairs; ++o)
                    if (rt.expert[o] == 2 * tid + i) {
                        rt.token[pair] = o / p.top_k;
                        rt.pos[o] = pair++;
                    }
                before += n[i] + (1 << 16);
            }
            if (tid == 127) {
                rt.n_active = before >> 16;
                rt.base[before >> 16] = pairs;
            }
            named_barrier(BAR_ROUTE, 128);
            if (tid == 0) mbar_arrive(routed_bar);
        }
        lost = !ok;
    }
    if (lost) *reinterpret_cast<volatile int*>(p.head + kFewBad) = 1;
    __syncthreads();
}

template <bool FP8, int NG>
cudaError_t launch_one(const MoeFewParams& p, int num_sms, cudaStream_t stream) {
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    auto kernel = moe_few_kernel<FP8, NG>;
    constexpr int smem = Cfg<FP8, NG>::kSmemBytes;
    if (dev < 64 && !attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        attr_set[dev] = true;
    }
    return launch_kernel(kernel, dim3((unsigned)num_sms), THREADS, smem, stream, true, p);
}

}  // namespace

cudaError_t moe_few_launch(const MoeFewParams& p, bool fp8, int num_sms, cudaStream_t stream) {
    switch (moe_few_groups(p.t)) {
        case 1: return fp8 ? launch_one<true, 1>(p, num_sms, stream) : launch_one<false, 1>(p, num_sms, stream);
        case 2: return fp8 ? launch_one<true, 2>(p, num_sms, stream) : launch_one<false, 2>(p, num_sms, stream);
        default: return fp8 ? launch_one<true, 4>(p, num_sms, stream) : launch_one<false, 4>(p, num_sms, stream);
    }
}

}  // namespace rf
