// A whole MoE layer for a few tokens (a decode step) in one kernel, sm_100a: router, softmax and top-k, SwiGLU experts, shared
// expert, weighted sum.
//
//   logits = fp16(x Wr^T + bias),  p = fp16(softmax(logits)),  the top_k largest p (equal ones: the lowest index)
//   h_e = (x Wg_e) / (1 + exp(-x Wg_e)) * (x Wu_e),  out = fp16(sum_i p_i h_i Wd_i + h_shared Wd_shared)
//
// What bounds it is the weight stream: each weight of every expert that a token chose is read once and used for a handful of
// multiplications.  So one persistent CTA per SM keeps a ring of TMA loads full from the first microsecond to the last, and all
// that depends on something else happens beside it.  The work is a list of items, dealt out by a ticket in this order:
//   router units   16 experts x a chunk of K of the logits, partial sums
//   routes         a token's top-k, from its logits
//   first product  64 columns of gate and the same of up x a chunk of K, the shared expert's first (they need no routing)
//   second product 128 columns of the result x a chunk of K
// An item depends on items with smaller tickets only, and a CTA works its tickets off in order, so whatever share of the grid is
// running makes progress, and the loads of an item never wait for its dependencies.
//
// What one CTA computes for another travels as 64-bit words, 32 bits of data beside the number of the call, which the reader
// polls for: no fence, no counter, one trip through L2.  (With partial sums behind fences and counters, each hand-over was four
// or five trips of 1.2 us under load: one token through 9 experts of 1024 x 512 took 25 us, through 5 of 7168 x 2048 98.)  The
// item with the last chunk of a column tile adds the chunks up in their order, and the last item of a result tile adds the
// experts in rank order: results are the same bits whoever comes last.  A token is routed by one CTA: every CTA for itself takes one
// hand-over less, and for 32 tokens through 128 or 256 experts 10 us more.
// One token through 9 fp16 experts of 1024 x 512 takes 18 us, through 5 of 7168 x 2048 71 to 75 (5.9 to 6.2 TB/s); 13 tokens through 86 of
// 256 FP8 experts 700 to 760 (5.1 to 5.5 TB/s), 32 through 164 1310 to 1395 (5.5).  What holds FP8 below fp16's rate: the MMA warps are busy for
// two thirds of the time, so that their waits and the stream's do not always overlap (the stream alone took 641 us of 729 for those 13
// tokens); a third group of four, at 96 registers, is slower.  Warps of a CTA:
//   0      draws tickets, issues the weight loads (16 KB stages)
//   1-3    the items' token rows (or, for the second product, h) into shared memory
//   4-11   mma.sync m16n8k16, weights as the 16-row operand, up to 8 tokens as the 8 columns: a warp owns 16 of the item's 128
//          columns.  (The legacy tensor path on purpose: the stream feeds one such MMA per 21 cycles and SM, and its
//          accumulators need no trip through TMEM.)  FP8 weights become fp16 on the way, their scale is applied per 128 of K.
//   12-15  softmax and top-k of a token (its ticket says whose), the experts' token lists (every CTA for itself), then the sums of
//          complete tiles
// h is rounded to fp16, the type of the second product's operand; everything else is fp32.
#include "moe_few.h"
#include "launch.h"
#include "ptx.cuh"
#include "softmax_exp.cuh"

namespace rf {

namespace {

constexpr int WARP_X = 1, WARP_MMA = 4, WARP_SUM = 12, WARPS = 16;
constexpr int X_WARPS = WARP_MMA - WARP_X, MMA_WARPS = WARP_SUM - WARP_MMA, SUM_WARPS = WARPS - WARP_SUM;
constexpr int THREADS = 32 * WARPS;
constexpr int STAGE_BYTES = 16384, BOX_BYTES = 8192;
constexpr int ITEM_SLOTS = 8, SUM_SLOTS = 8;
constexpr int DRAW_AHEAD = 4;           // stages before an item's last load at which the next ticket is drawn
constexpr int MAX_PAIRS = kFewMaxTokens * kFewMaxTopK;

enum ItemKind { kRouter = 0, kFirst = 1, kSecond = 2, kEnd = 3, kRoute = 4, kLists = 5 };
// kind, expert slot (index into the active list; the shared expert's are -1, -2), column tile, K chunk
using Item = int4;

struct Routing {
    int n_active;
    int active[MAX_PAIRS];              // experts with tokens, ascending, each once per kRows tokens
    int base[MAX_PAIRS + 1];            // first pair of each of them; pairs are sorted by expert, then token
    int token[MAX_PAIRS];               // of a pair
    int expert[MAX_PAIRS];              // [token][rank]
    int pos[MAX_PAIRS];                 // pair of [token][rank]
    float weight[MAX_PAIRS];            // [token][rank]
    int count[kFewMaxExperts];
    float logits[SUM_WARPS][kFewMaxExperts];
};

template <bool FP8, int NG>
struct Cfg {
    static constexpr int kStageK = FP8 ? 128 : 64;
    static constexpr int kRows = 8 * NG;
    // beside fp16 weights x goes through ldmatrix (rows 16 bytes apart modulo 128), beside FP8 through 16-byte loads (64 bytes)
    static constexpr int kPad = FP8 ? 64 : 16;
    static constexpr int kXStride = kFewMaxChunk * 2 + kPad;
    // ... and behind the rows the scales of the item's two boxes, one per 128 of K
    static constexpr int kXBytes = kRows * kXStride + (FP8 ? 64 : 0);
    // a router unit's partial sums of every MMA warp; later the sums that one group of them hands to the other
    static constexpr int kRedBytes = MMA_WARPS * 16 * kRows * 4;
    static_assert(kRedBytes == MMA_WARPS / 2 * 2 * NG * 4 * 128, "both uses");
    static constexpr int kStages = few_stages(FP8, NG);
    static_assert(!FP8 || kStages % 2 == 0, "two groups, each with slots of its own");
    static constexpr int kBars = 2 * kStages + 4 + 2 * ITEM_SLOTS + 2 * SUM_SLOTS + 3 + MMA_WARPS;
    static constexpr int kSmemBytes = kStages * STAGE_BYTES + 2 * kXBytes + kRedBytes + (ITEM_SLOTS + SUM_SLOTS) * 16 + kBars * 8 +
                                      (int)sizeof(Routing) + 1024;
    static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

// A word that travels between CTAs: data below, the number of the call above.  One 64-bit access each, so that data and number
// arrive together; two words at a time where they lie side by side.
__device__ __forceinline__ unsigned long long word_of(uint32_t data, uint32_t call) {
    return (unsigned long long)data | ((unsigned long long)call << 32);
}
__device__ __forceinline__ void st_word(unsigned long long* p, uint32_t data, uint32_t call) {
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(word_of(data, call)) : "memory");
}
__device__ __forceinline__ void st_words(unsigned long long* p, uint32_t a, uint32_t b, uint32_t call) {
    asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};" ::"l"(p), "l"(word_of(a, call)), "l"(word_of(b, call)) : "memory");
}
__device__ __forceinline__ unsigned long long ld_word(const unsigned long long* p) {
    unsigned long long v;
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ ulonglong2 ld_words(const unsigned long long* p) {
    ulonglong2 v;
    asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t call_of(unsigned long long w) { return (uint32_t)(w >> 32); }
__device__ __forceinline__ float float_of(unsigned long long w) { return __uint_as_float((uint32_t)w); }

// The limit of a polling loop (status word and unwinding as in mbar_wait): false = give up.
struct Patience {
    int* status;
    int tag;
    uint32_t polls = 0;
    unsigned long long t0 = 0;
    __device__ __forceinline__ Patience(int* s, int t) : status(s), tag(t) {}
    __device__ __forceinline__ bool more() {
        if ((++polls & 0x3fu) != 0) return true;
        const int seen = *reinterpret_cast<volatile int*>(status);
        if (seen != 0 && (seen >> kStatusTagShift) == tag) return false;
        const unsigned long long now = globaltimer_ns();
        if (t0 == 0) t0 = now;
        else if (now - t0 > wait_limit_ns(status)) {
            atomicCAS(status, 0, kErrSchedWait | (tag << kStatusTagShift));
            return false;
        }
        return true;
    }
};

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
// (no "volatile": a function of its operands alone)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}

// A warp's sums of n partial sums, `step` words apart, in their order: two neighbouring words at `a` and two at `b`.  Eight chunks are
// in flight together.
__device__ __forceinline__ bool sum_chunks(const unsigned long long* a, const unsigned long long* b, size_t step, int n,
                                           uint32_t call, Patience& patience, float2* sa, float2* sb) {
    float2 x = make_float2(0.f, 0.f), y = x;
    for (int c0 = 0; c0 < n; c0 += 8) {
        ulonglong2 u[8], v[8];
        for (;;) {
            bool here = true;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const size_t at = (size_t)min(c0 + i, n - 1) * step;
                u[i] = ld_words(a + at);
                v[i] = ld_words(b + at);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                here = here && call_of(u[i].x) == call && call_of(u[i].y) == call && call_of(v[i].x) == call && call_of(v[i].y) == call;
            if (__all_sync(0xffffffffu, here)) break;
            if (!__all_sync(0xffffffffu, patience.more())) return false;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i < n) {
                x.x += float_of(u[i].x); x.y += float_of(u[i].y);
                y.x += float_of(v[i].x); y.y += float_of(v[i].y);
            }
    }
    *sa = x;
    *sb = y;
    return true;
}

// mbar_wait for the roles that mostly wait: they sleep between polls, which would take issue slots and shared memory cycles from the
// MMA warps.
__device__ __forceinline__ bool idle_wait(uint32_t bar, uint32_t parity, int* status, int code, int tag) {
    for (int i = 0; i < 4; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    Patience patience(status, tag);
    while (!mbar_try_wait(bar, parity)) {
        __nanosleep(64);
        if (!patience.more()) return false;
    }
    (void)code;
    return true;
}

// How the work divides: known once the routing is.
struct Shape {
    int groups;                 // slots of the shared expert
    int tiles1, tiles1s;        // column tiles of the first product: of an expert, of the shared one
    int tiles2;
    int chunks1, chunks2, chunks2s;
    __device__ __forceinline__ Shape(const MoeFewParams& p, int rows)
        : groups((p.t + rows - 1) / rows), tiles1(p.f / 64), tiles1s(p.fs / 64), tiles2((p.d + 127) / 128), chunks1((p.d + p.kc1 - 1) / p.kc1),
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
    const int per2s = s.tiles2 * s.chunks2s;
    if (r < s.groups * per2s) {
        const int e = r / per2s, i = r - e * per2s, c = i / s.tiles2;
        return make_int4(kSecond, -1 - e, i - c * s.tiles2, c);
    }
    r -= s.groups * per2s;
    const int per2 = s.tiles2 * s.chunks2;
    if (r < n_active * per2) {
        const int e = r / per2, i = r - e * per2, c = i / s.tiles2;
        return make_int4(kSecond, e, i - c * s.tiles2, c);
    }
    return make_int4(kEnd, 0, 0, 0);
}

// One warp: a token's logits over the K chunks c, c + SUM_WARPS, ..., two experts side by side a lane (512 bytes a load).
template <int VPT>
__device__ __forceinline__ bool sum_logits(const MoeFewParams& p, int t, int c, uint32_t call, Patience& patience, float* row) {
    constexpr int BATCH = 32 / VPT < 4 ? 32 / VPT : 4;          // chunks whose loads are in flight together
    const int lane = threadIdx.x & 31;
    const unsigned long long* src = p.logits + (size_t)t * p.experts;
    const size_t step = (size_t)p.t * p.experts;
    float l[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) l[i] = 0.f;
    for (; c < p.router_chunks; c += BATCH * SUM_WARPS) {
        unsigned long long v[BATCH][VPT];
        for (;;) {
            bool here = true;
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int cb = c + b * SUM_WARPS;
                const unsigned long long* at = src + (size_t)(cb < p.router_chunks ? cb : c) * step;
                if (VPT == 1) {
                    v[b][0] = ld_word(at + min(lane, p.experts - 1));
                } else {
#pragma unroll
                    for (int i = 0; i < VPT / 2; ++i) {
                        const ulonglong2 w = ld_words(at + 64 * i + 2 * lane);
                        v[b][2 * i] = w.x;
                        v[b][VPT == 1 ? 0 : 2 * i + 1] = w.y;
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
#pragma unroll
                for (int i = 0; i < VPT; ++i) here = here && call_of(v[b][i]) == call;
            if (__all_sync(0xffffffffu, here)) break;
            if (!__all_sync(0xffffffffu, patience.more())) return false;
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
            if (c + b * SUM_WARPS < p.router_chunks)
#pragma unroll
                for (int i = 0; i < VPT; ++i) l[i] += float_of(v[b][i]);
    }
    if (VPT == 1) row[lane] = l[0];
#pragma unroll
    for (int i = 0; i < VPT / 2; ++i) *reinterpret_cast<float2*>(row + 64 * i + 2 * lane) = make_float2(l[2 * i], l[VPT == 1 ? 0 : 2 * i + 1]);
    return true;
}

// One warp: a token's softmax and top-k from its logits' partial sums, as topk_kernel (moe_route.cu) does them, on the same fp16
// roundings.  Lane l owns experts l * VPT ..; a key is an fp16 probability, then the complement of the expert's number, and
// lane k < top_k returns the k-th largest.
template <int VPT>
__device__ __forceinline__ uint32_t pick(const MoeFewParams& p, const float (&sums)[SUM_WARPS][kFewMaxExperts]) {
    const int lane = threadIdx.x & 31, e0 = lane * VPT;
    const bool active = e0 < p.experts;
    float l[VPT], mx = -65504.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) l[i] = 0.f;
    if (active)
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
#pragma unroll
            for (int w = 0; w < SUM_WARPS; ++w) l[i] += sums[w][e0 + i];
            if (p.router_bias != nullptr) l[i] += ld_global_f32(p.router_bias + e0 + i);
            l[i] = __half2float(__float2half_rn(l[i]));
            mx = fmaxf(mx, l[i]);
        }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        l[i] = active ? det_exp(__fsub_rn(l[i], mx)) : 0.f;
        part = i == 0 ? l[0] : __fadd_rn(part, l[i]);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) part = __fadd_rn(part, __shfl_xor_sync(0xffffffffu, part, s));
    const float recip = __fdiv_rn(1.0f, part);
    uint32_t key[VPT], mine = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        key[i] = active ? ((uint32_t)__half_as_ushort(__float2half_rn(__fmul_rn(l[i], recip))) << 16) | (0xFFFFu - (uint32_t)(e0 + i))
                        : 0u;
    for (int k = 0; k < p.top_k; ++k) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < VPT; ++i) best = max(best, key[i]);
        best = __reduce_max_sync(0xffffffffu, best);
        if (lane == k) mine = best;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (key[i] == best) key[i] = 0u;
    }
    return mine;
}

// The routing warps together: token t's top-k for everyone. `meet` is their barrier, with its parity.
template <int VPT, class Meet>
__device__ __forceinline__ bool route_token(const MoeFewParams& p, Routing& rt, int t, uint32_t call, Patience& patience, Meet meet) {
    const int w = (threadIdx.x >> 5) - WARP_SUM, lane = threadIdx.x & 31;
    if (!sum_logits<VPT>(p, t, w, call, patience, rt.logits[w]) || !meet(0)) return false;
    if (w == 0) {
        const uint32_t key = pick<VPT>(p, rt.logits);
        if (lane < p.top_k) st_word(p.routes + t * p.top_k + lane, key, call);
    }
    return meet(1);     // (the next token's sums go where these were)
}

// One warp: every token's top-k.
template <int BATCH>
__device__ __forceinline__ bool read_routes(const MoeFewParams& p, Routing& rt, uint32_t call, Patience& patience) {
    const int lane = threadIdx.x & 31, pairs = p.t * p.top_k;
    unsigned long long v[BATCH];
    for (;;) {
        bool here = true;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) v[i] = ld_word(p.routes + min(32 * i + lane, pairs - 1));
#pragma unroll
        for (int i = 0; i < BATCH; ++i) here = here && call_of(v[i]) == call;
        if (__all_sync(0xffffffffu, here)) break;
        if (!__all_sync(0xffffffffu, patience.more())) return false;
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
        if (32 * i + lane < pairs) {
            rt.expert[32 * i + lane] = (int)(0xFFFFu - ((uint32_t)v[i] & 0xFFFFu));
            rt.weight[32 * i + lane] = __half2float(__ushort_as_half((unsigned short)((uint32_t)v[i] >> 16)));
        }
    __syncwarp();
    return true;
}

// One warp: the experts' token lists, in an order that every CTA finds alike.  Ranks inside 32 pairs by match_any, pairs in order;
// then the experts' offsets, eight experts a lane.
template <int ROWS>
__device__ __forceinline__ void build_lists(const MoeFewParams& p, Routing& rt) {
    const int lane = threadIdx.x & 31, pairs = p.t * p.top_k;
    for (int e = lane; e < kFewMaxExperts; e += 32) rt.count[e] = 0;
    __syncwarp();
    for (int i0 = 0; i0 < pairs; i0 += 32) {
        const int i = i0 + lane, e = i < pairs ? rt.expert[i] : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        const int before = __popc(peers & ((1u << lane) - 1));
        if (e >= 0) rt.pos[i] = rt.count[e] + before;
        __syncwarp();
        if (e >= 0 && before == 0) rt.count[e] += __popc(peers);
        __syncwarp();
    }
    // pairs (low half) and slots (high half) in front of this lane's eight experts
    int n[8], mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        n[i] = rt.count[8 * lane + i];
        mine += n[i] + ((n[i] + ROWS - 1) / ROWS << 16);
    }
    int incl = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, s);
        if (lane >= s) incl += o;
    }
    int run = incl - mine;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rt.count[8 * lane + i] = run & 0xFFFF;          // now the expert's first pair
        for (int left = n[i]; left > 0; left -= ROWS) {
            rt.active[run >> 16] = 8 * lane + i;
            rt.base[run >> 16] = run & 0xFFFF;
            run += min(left, ROWS) + (1 << 16);
        }
    }
    if (lane == 31) {
        rt.n_active = run >> 16;
        rt.base[run >> 16] = pairs;
    }
    __syncwarp();
    for (int i = lane; i < pairs; i += 32) {
        const int at = rt.count[rt.expert[i]] + rt.pos[i];
        rt.pos[i] = at;
        rt.token[at] = i / p.top_k;
    }
    __syncwarp();
}

template <bool FP8, int NG>
__global__ void __launch_bounds__(THREADS, 1)
moe_few_kernel(const __grid_constant__ FewMaps even, const MoeFewParams p) {
    using C = Cfg<FP8, NG>;
    constexpr int STAGES = C::kStages;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t x_base = smem_base + STAGES * STAGE_BYTES;
    const uint32_t red_base = x_base + 2 * C::kXBytes;
    const uint32_t item_base = red_base + C::kRedBytes;
    const uint32_t sum_base = item_base + ITEM_SLOTS * 16;
    const uint32_t bar_base = sum_base + SUM_SLOTS * 16;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto x_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto x_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
    // rings of items: for the rows and MMA warps, and of those that end with a sum
    auto item_bar = [&](uint32_t j) { return bar_base + 8u * (2 * STAGES + 4 + j % ITEM_SLOTS); };
    auto free_bar = [&](uint32_t j) { return bar_base + 8u * (2 * STAGES + 4 + ITEM_SLOTS + j % ITEM_SLOTS); };
    auto sum_bar = [&](uint32_t j) { return bar_base + 8u * (2 * STAGES + 4 + 2 * ITEM_SLOTS + j % SUM_SLOTS); };
    auto sum_free_bar = [&](uint32_t j) { return bar_base + 8u * (2 * STAGES + 4 + 2 * ITEM_SLOTS + SUM_SLOTS + j % SUM_SLOTS); };
    const uint32_t routed_bar = bar_base + 8u * (2 * STAGES + 4 + 2 * ITEM_SLOTS + 2 * SUM_SLOTS);
    const uint32_t meet_bar = routed_bar + 8, sum_meet_bar = routed_bar + 16;
    auto merge_bar = [&](uint32_t i) { return routed_bar + 8u * (3 + i); };
    auto merge_free_bar = [&](uint32_t i) { return routed_bar + 8u * (3 + MMA_WARPS / 2 + i); };
    Routing& rt = *reinterpret_cast<Routing*>(smem_raw + (bar_base + 8u * C::kBars - smem_u32(smem_raw)));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    griddep_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), FP8 ? MMA_WARPS / 2 : MMA_WARPS);
        }
        for (int i = 0; i < MMA_WARPS / 2; ++i) {
            mbar_init(merge_bar(i), 1);
            mbar_init(merge_free_bar(i), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(x_full_bar(b), X_WARPS);
            mbar_init(x_empty_bar(b), MMA_WARPS);
        }
        for (int j = 0; j < ITEM_SLOTS; ++j) {
            mbar_init(item_bar(j), 1);
            mbar_init(free_bar(j), X_WARPS + MMA_WARPS);
        }
        for (int j = 0; j < SUM_SLOTS; ++j) {
            mbar_init(sum_bar(j), 1);
            mbar_init(sum_free_bar(j), SUM_WARPS);
        }
        mbar_init(routed_bar, 1);
        mbar_init(meet_bar, MMA_WARPS);
        mbar_init(sum_meet_bar, SUM_WARPS);
        mbar_fence_init();
    }
    griddep_wait();
    // The number of this call: zero, which fresh words hold, is left out.  (A word that no call has written for the 2^32 - 1 calls
    // before this one could pass for this call's.)
    uint32_t call = (uint32_t)ld_global_s32(p.head + kFewCalls) + 1;
    if (call == 0) call = 1;
    // A workspace in which an earlier call lost a wait holds a ticket that belongs to nothing: no result then, and a code.
    int ticket = threadIdx.x == 0 ? atomicAdd(p.head + kFewTicket, 1) : 0;
    const int bad = __syncthreads_or(ld_global_s32(p.head + kFewBad) != 0);
    if (bad) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0, kErrSchedWait | (p.launch_tag << kStatusTagShift));
        return;
    }

    const Shape shape(p, C::kRows);
    const int shared_first = shape.groups * shape.tiles1s * shape.chunks1;
    const int before_shared = p.router_units + p.t, before_routed = before_shared + shared_first;
    const int pairs = p.t * p.top_k;            // the shared expert's pairs come behind them, one per token
    const size_t rows = pairs + p.t;            // of h and the partial sums
    auto wait_routed = [&](int code) { return idle_wait(routed_bar, 0, p.status, code, p.launch_tag); };
    // A barrier of a role's warps with a limit: a warp that gave a wait up does not come.
    auto meet_at = [&](uint32_t bar, uint32_t parity, int code) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status, code, p.launch_tag)) != 0;
    };
    auto wait_item = [&](uint32_t j, int code) {
        return mbar_wait(item_bar(j), (j / ITEM_SLOTS) & 1, p.status, code, p.launch_tag);
    };
    const uint32_t zero = (uint32_t)p.t >> 16;
    // The item in a slot, which is free for the next.
    auto take = [&](uint32_t addr, uint32_t bar) {
        const uint4 v = ld_shared_v4(addr);
        __syncwarp();
        if (lane == 0) mbar_arrive_after(bar, v.x, zero);
        return make_int4((int)v.x, (int)v.y, (int)v.z, (int)v.w);
    };
    auto take_item = [&](uint32_t j) { return take(item_base + 16u * (j % ITEM_SLOTS), free_bar(j)); };
    // K range of an item
    auto k_range = [&](const Item& it, int* k0, int* len) {
        const int kc = it.x == kFirst ? p.kc1 : p.kc2;
        const int k = it.x == kFirst ? p.d : it.y < 0 ? p.fs : p.f;
        *k0 = it.w * kc;
        *len = min(kc, k - *k0);
    };
    auto expert_of = [&](const Item& it) { return it.y < 0 ? p.experts : rt.active[it.y]; };
    auto first_token = [&](const Item& it) { return (-1 - it.y) * C::kRows; };       // (the shared expert's)
    auto first_pair = [&](const Item& it) { return it.y < 0 ? pairs + first_token(it) : rt.base[it.y]; };
    auto pair_count = [&](const Item& it) {
        return it.y < 0 ? min(p.t - first_token(it), C::kRows) : rt.base[it.y + 1] - rt.base[it.y];
    };

    bool lost = false;          // this thread's role gave a wait up
    if (warp == 0) {
        // ------------------------------------------------------------------------------ tickets, weight loads
        if (lane == 0) {
            uint32_t st = 0, s = 0, ph = 1;
            bool ok = true, routed = false, lists = false;
            uint32_t sums = 0;
            const CUtensorMap* acquired = nullptr;
            auto push_sum = [&](const Item& it) {
                ok = idle_wait(sum_free_bar(sums), ((sums / SUM_SLOTS) & 1) ^ 1, p.status, kErrProducerWait, p.launch_tag);
                if (!ok) return;
                st_shared_v4(sum_base + 16u * (sums % SUM_SLOTS), it.x, it.y, it.z, it.w);
                mbar_arrive(sum_bar(sums++));
            };
            for (uint32_t j = 0; ok; ++j) {
                Item it;
                for (; ok && ticket >= p.router_units && ticket < before_shared; ticket = atomicAdd(p.head + kFewTicket, 1))
                    push_sum(make_int4(kRoute, 0, ticket - p.router_units, 0));
                if (ok && ticket >= before_shared && !lists) {
                    push_sum(make_int4(kLists, 0, 0, 0));
                    lists = true;
                }
                if (!ok) break;
                if (ticket < p.router_units) {
                    it = make_int4(kRouter, 0, ticket, 0);
                } else if (ticket < before_routed) {
                    const int per = shape.tiles1s * shape.chunks1, r = ticket - before_shared, e = r / per, i = r - e * per;
                    const int c = i / shape.tiles1s;
                    it = make_int4(kFirst, -1 - e, i - c * shape.tiles1s, c);
                } else {
                    if (!routed) {
                        ok = wait_routed(kErrProducerWait);
                        if (!ok) break;
                        routed = true;
                    }
                    it = decode_routed(ticket - before_routed, shape, rt.n_active);
                }
                ok = idle_wait(free_bar(j), ((j / ITEM_SLOTS) & 1) ^ 1, p.status, kErrProducerWait, p.launch_tag);
                if (!ok) break;
                st_shared_v4(item_base + 16u * (j % ITEM_SLOTS), it.x, it.y, it.z, it.w);
                mbar_arrive(item_bar(j));
                // the last chunk of a column tile, the last item of a result tile
                if (it.x == kEnd || (it.x == kFirst && it.w == shape.chunks1 - 1) ||
                    (it.x == kSecond && it.y == rt.n_active - 1 && it.w == shape.chunks2 - 1)) {
                    push_sum(it);
                    if (!ok) break;
                }
                if (it.x == kEnd) break;
                if (it.x == kRouter) {
                    ticket = atomicAdd(p.head + kFewTicket, 1);
                    continue;
                }
                int k0, len;
                k_range(it, &k0, &len);
                const int which = it.x == kFirst ? 0 : 2, e = expert_of(it);
                const CUtensorMap* m0 = p.maps != nullptr ? p.maps + 3 * e + which : even.m + (it.y < 0 ? 3 : 0) + which;
                const CUtensorMap* m1 = it.x == kFirst ? m0 + 1 : m0;
                if (p.maps != nullptr && m0 != acquired) {
                    tma_acquire_desc(m0);
                    if (m1 != m0) tma_acquire_desc(m1);
                    acquired = m0;
                }
                // columns; and the rows in front of the expert's matrix in its stack
                const int n0 = it.x == kFirst ? it.z * 64 : it.z * 128, n1 = it.x == kFirst ? n0 : n0 + 64;
                const int in_stack = p.maps == nullptr && it.y >= 0 ? e : 0;
                const int r0 = in_stack * even.rows[which], r1 = it.x == kFirst ? in_stack * even.rows[1] : r0;
                const int n_stages = len / C::kStageK;
                for (int i = 0; i < n_stages; ++i, ++st) {
                    if (i == max(n_stages - DRAW_AHEAD, 0)) ticket = atomicAdd(p.head + kFewTicket, 1);
                    ok = idle_wait(empty_bar(s), ph, p.status, kErrProducerWait, p.launch_tag);
                    if (!ok) break;
                    const uint32_t dst = smem_base + s * STAGE_BYTES;
                    const int k = k0 + i * C::kStageK;
                    mbar_expect_tx(full_bar(s), STAGE_BYTES);
                    tma_load_2d(dst, m0, full_bar(s), FP8 ? k : n0, r0 + (FP8 ? n0 : k));
                    tma_load_2d(dst + BOX_BYTES, m1, full_bar(s), FP8 ? k : n1, r1 + (FP8 ? n1 : k));
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
            ok = __all_sync(0xffffffffu, idle_wait(item_bar(j), (j / ITEM_SLOTS) & 1, p.status, kErrMmaWaitFull, p.launch_tag));
            if (!ok) break;
            const Item it = take_item(j);
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
            ok = __all_sync(0xffffffffu, idle_wait(x_empty_bar(b), ((n >> 1) & 1) ^ 1, p.status, kErrMmaWaitFull, p.launch_tag));
            if (!ok) break;
            const int n_rows = pair_count(it), first = first_pair(it);
            const uint32_t dst = x_base + b * C::kXBytes;
            float scale = 0.f;
            if (FP8 && warp == WARP_X && lane < 16 && (lane & 7) < len / 128) {
                const int m = it.x == kFirst ? lane >> 3 : 2, k = it.x == kFirst ? p.d : it.y < 0 ? p.fs : p.f;
                scale = ld_global_f32(p.scales[3 * expert_of(it) + m] +
                                      (size_t)(it.x == kFirst ? it.z >> 1 : it.z) * (k / 128) + k0 / 128 + (lane & 7));
            }
            if (it.x == kFirst) {
                // one bulk copy per row, all by the first of the warps
                if (warp == WARP_X) {
                    if (lane == 0) mbar_expect_tx_only(x_full_bar(b), (uint32_t)(n_rows * len * 2));
                    __syncwarp();
                    if (lane < n_rows) {
                        const int row = it.y >= 0 ? rt.token[first + lane] : first_token(it) + lane;
                        bulk_load(dst + lane * C::kXStride, static_cast<const __half*>(p.x) + (size_t)row * p.d + k0, (uint32_t)len * 2,
                                  x_full_bar(b));
                    }
                }
            } else {
                // h comes as words of two values: two of them make 8 bytes of a row
                const int vecs = len >> 2, total = n_rows * vecs;
                const unsigned long long* src = p.h + (size_t)first * (p.width / 2) + k0 / 2;
                Patience patience(p.status, p.launch_tag);
                constexpr int BATCH = 8;
                for (int i0 = 0; i0 < total && ok; i0 += BATCH * 32 * X_WARPS) {
                    ulonglong2 v[BATCH];
                    for (;;) {
                        bool here = true;
#pragma unroll
                        for (int i = 0; i < BATCH; ++i) {
                            const int at = min(i0 + i * 32 * X_WARPS + tid, total - 1), r = at / vecs;
                            v[i] = ld_words(src + (size_t)r * (p.width / 2) + 2 * (at - r * vecs));
                        }
#pragma unroll
                        for (int i = 0; i < BATCH; ++i) here = here && call_of(v[i].x) == call && call_of(v[i].y) == call;
                        if (__all_sync(0xffffffffu, here)) break;
                        ok = __all_sync(0xffffffffu, patience.more());
                        if (!ok) break;
                    }
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < BATCH; ++i) {
                        const int at = i0 + i * 32 * X_WARPS + tid, r = at / vecs;
                        if (at < total) st_shared_v2(dst + r * C::kXStride + 8 * (at - r * vecs), (uint32_t)v[i].x, (uint32_t)v[i].y);
                    }
                }
                if (!ok) break;
            }
            if (FP8 && warp == WARP_X && lane < 16) st_shared_f32(dst + C::kRows * C::kXStride + lane * 4, scale);
            __syncwarp();
            if (lane == 0) mbar_arrive(x_full_bar(b));
            ++n;
        }
        lost = !ok;
        // This CTA draws no ticket any more: the last warp to come here gives the next call its ticket and its number.  (Where a wait
        // was lost the workspace is marked below, and its next call refuses to run.)
        if (ok && lane == 0 && atomicAdd(p.head + kFewExits, 1) == (int)gridDim.x * X_WARPS - 1) {
            p.head[kFewTicket] = p.head[kFewExits] = 0;
            p.head[kFewCalls] = (int)call;
        }
    } else if (warp < WARP_SUM) {
        // ------------------------------------------------------------------------------ MMA
        const int w = warp - WARP_MMA;
        const int g = lane >> 2, q = lane & 3;      // row (column) of the fragments, pair inside
        const uint32_t box = (w >> 2) * BOX_BYTES;      // (fp16: 16 columns a warp)
        bool ok = true, routed = false;
        uint32_t n = 0, s = 0, ph = 0, met = 0;
        auto meet = [&] { return meet_at(meet_bar, met++ & 1, kErrMmaWaitFull); };
        for (uint32_t j = 0;; ++j) {
            ok = ok && __all_sync(0xffffffffu, wait_item(j, kErrMmaWaitFull));
            if (!ok) break;
            const Item it = take_item(j);
            if (it.x == kEnd) break;
            if (it.x != kRouter && it.y >= 0 && !routed) {
                ok = __all_sync(0xffffffffu, wait_routed(kErrMmaWaitFull));
                if (!ok) break;
                routed = true;
            }
            if (it.x == kRouter) {
                // 16 experts x a chunk of K, 64 columns per warp and round.  A lane holds 16 consecutive k of its row (and token): the
                // order of k inside a fragment is free as long as both operands share it.
                const int c = it.z % p.router_chunks, et = it.z / p.router_chunks, e_tiles = (p.experts + 15) / 16;
                const int e0 = et % e_tiles * 16, t0 = et / e_tiles * C::kRows;
                float acc[NG][4] = {};
#pragma unroll 1
                for (int k = c * p.router_kc + w * 64; k < min((c + 1) * p.router_kc, p.d); k += MMA_WARPS * 64) {
                    uint4 a[2][2], b[NG][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const __half* row = static_cast<const __half*>(p.router) + (size_t)min(e0 + g + 8 * i, p.experts - 1) * p.d;
#pragma unroll
                        for (int v = 0; v < 2; ++v) a[i][v] = ld_global_cg_v4(row + k + 16 * q + 8 * v);
                    }
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const __half* row = static_cast<const __half*>(p.x) + (size_t)min(t0 + 8 * i + g, p.t - 1) * p.d;
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
                // (met: all have written; met again: all have read, and the next unit may write)
                ok = meet();
                if (!ok) break;
                for (int i = w * 32 + lane; i < 16 * C::kRows; i += 32 * MMA_WARPS) {
                    const int e = e0 + i / C::kRows, t = t0 + i % C::kRows;
                    float v = 0.f;
#pragma unroll
                    for (int o = 0; o < MMA_WARPS; ++o)
                        v += __uint_as_float(ld_shared_u32(red_base + (o * 16 * C::kRows + i) * 4));
                    if (e < p.experts && t < p.t) st_word(p.logits + ((size_t)c * p.t + t) * p.experts + e, __float_as_uint(v), call);
                }
                ok = meet();
                continue;
            }
            int k0, len;
            k_range(it, &k0, &len);
            const int n_rows = pair_count(it), first = first_pair(it);
            const uint32_t b = n & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(x_full_bar(b), (n >> 1) & 1, p.status, kErrMmaWaitFull, p.launch_tag));
            const uint32_t xb = x_base + b * C::kXBytes;
            const int groups = (n_rows + 7) >> 3;
            float acc[FP8 ? 2 * NG : NG][4] = {};       // FP8: two tiles of 16 columns for each 8 tokens
            const int n_stages = len / C::kStageK;
            // A stage is free when what it held has become a sum.  (Freed when its loads had been issued, one call in twenty with 24
            // tokens multiplied some of the next weights: those that come from L2 are there before the loads.)
            auto give_back = [&](uint32_t bar, float sum) {
                __syncwarp();
                if (lane == 0) mbar_arrive_after(bar, __float_as_uint(sum), zero);
            };
            auto next_stage = [&] {
                const bool here = __all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, p.status, kErrMmaWaitFull, p.launch_tag));
                return here;
            };
            if (FP8) {
                // Two groups of four warps take the item's stages in turn (by their slots of the ring, few_first_stage), 32 columns a
                // warp: while one group waits and loads, the other multiplies, and a row of x is read by half as many warps.  (All eight on every stage, 16 columns each:
                // barrier, loads, conversions and MMAs of a stage come one after the other, 540 cycles; so 360.)  Which of the
                // MMA's 16 rows is which column, and the order of k inside it, are free as long as both operands and the result
                // agree: rows g and g + 8 are columns 2g and 2g + 1 (their 8-byte pieces lie in banks of their own), a lane
                // takes 8 consecutive k for two MMAs.  Rows of x that hold no token repeat the last one (nobody takes their sums), and x
                // is read ahead of the stage's barrier: a group spends 1050 cycles on a stage between waits without either, 860 with both.  Four
                // chains of MMAs instead of two, and scales and h read before their buffer is free, changed nothing.
                const int group = w >> 2, c0 = (w & 3) * 32 + 2 * g;
                const uint32_t w_lo = smem_base + c0 * 128 + (((q >> 1) ^ (c0 & 7)) << 4) + 8 * (q & 1);
                const uint32_t scales = xb + C::kRows * C::kXStride + ((w >> 1) & 1) * 32;
                const uint32_t x_row = xb + min(g, n_rows - 1) * C::kXStride + 16 * q;
                for (int i = few_first_stage(group, (int)s); i < n_stages; i += 2) {
                    const bool wrap = s + i >= (uint32_t)STAGES;
                    const uint32_t si = s + i - (wrap ? STAGES : 0);
                    uint4 x[4];
                    auto load_x = [&](int u) {
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            x[b] = ld_shared_v4((u == 0 ? x_row : xb + min(8 * u + g, n_rows - 1) * C::kXStride + 16 * q) + 2 * (i * 128 + b * 32));
                    };
                    load_x(0);
                    ok = __all_sync(0xffffffffu, mbar_wait(full_bar(si), ph ^ (wrap ? 1u : 0u), p.status, kErrMmaWaitFull, p.launch_tag));
                    if (!ok) break;
                    uint2 l[2][4], h[2][4];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        // (64 columns to a box of 8 KB; 16-byte pieces are swizzled by their column modulo 8)
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            l[t][b] = ld_shared_v2(((w_lo + si * STAGE_BYTES) ^ (b << 5)) + t * 2048);
                            h[t][b] = ld_shared_v2((((w_lo + si * STAGE_BYTES) ^ (b << 5)) ^ 16) + 128 + t * 2048);
                        }
                    }
                    const float sc = __uint_as_float(ld_shared_u32(scales + i * 4));
#pragma unroll
                    for (int u = 0; u < NG; ++u) {
                        if (u >= groups) break;
                        float part[2][4] = {};
                        if (u > 0) load_x(u);
                        auto convert = [](uint32_t lo, uint32_t hi, uint32_t (&a)[4]) {
                            a[0] = f16x2_of_e4m3x2((uint16_t)lo);
                            a[1] = f16x2_of_e4m3x2((uint16_t)hi);
                            a[2] = f16x2_of_e4m3x2((uint16_t)(lo >> 16));
                            a[3] = f16x2_of_e4m3x2((uint16_t)(hi >> 16));
                        };
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            uint32_t a[4];
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                convert(l[t][b].x, h[t][b].x, a);
                                mma_f16(part[t], a, x[b].x, x[b].y);
                            }
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                convert(l[t][b].y, h[t][b].y, a);
                                mma_f16(part[t], a, x[b].z, x[b].w);
                            }
                        }
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int v = 0; v < 4; ++v) acc[2 * u + t][v] = fmaf(sc, part[t][v], acc[2 * u + t][v]);
                        if (u == 0) give_back(empty_bar(si), part[0][0] + part[1][0]);
                    }
                }
                s += n_stages;
                if (s >= (uint32_t)STAGES) {
                    s -= STAGES;
                    ph ^= 1;
                }
                // the second group's sums join the first's
                const uint32_t mine = red_base + (w & 3) * (2 * NG * 4 * 128) + lane * 4;
                if (group == 1) {
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(merge_free_bar(w & 3), (n & 1) ^ 1, p.status, kErrMmaWaitFull, p.launch_tag));
                    if (ok) {
#pragma unroll
                        for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
                            for (int v = 0; v < 4; ++v) st_shared_f32(mine + (4 * i + v) * 128, acc[i][v]);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(merge_bar(w & 3));
                    }
                } else {
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(merge_bar(w & 3), n & 1, p.status, kErrMmaWaitFull, p.launch_tag));
                    if (ok) {
                        uint32_t seen = 0;
#pragma unroll
                        for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                const uint32_t other = ld_shared_u32(mine + (4 * i + v) * 128);
                                acc[i][v] += __uint_as_float(other);
                                seen |= other;
                            }
                        __syncwarp();
                        if (lane == 0) mbar_arrive_after(merge_free_bar(w & 3), seen, zero);
                    }
                }
            } else {
                // rows are k; transposed 8 x 8 pieces give the weights as [column][k] fragments
                const int kr = (lane & 7) + 8 * (lane >> 4), chunk = 2 * (w & 3) + ((lane >> 3) & 1);
                const uint32_t w_off = box + kr * 128 + ((chunk ^ (kr & 7)) << 4);
                for (int i = 0; i < n_stages && ok; ++i) {
                    ok = next_stage();
                    if (!ok) break;
                    const uint32_t wa = smem_base + s * STAGE_BYTES + w_off;
                    const uint32_t xa = xb + (lane & 7) * C::kXStride + 2 * (i * 64 + 8 * (lane >> 3));
                    uint32_t a[4][4], x[2][NG][4];
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) ldmatrix_x4_trans(wa + kk * 16 * 128, a[kk]);
#pragma unroll
                    for (int v = 0; v < 2; ++v)
#pragma unroll
                        for (int u = 0; u < NG; ++u)
                            if (u < groups) ldmatrix_x4(xa + u * 8 * C::kXStride + v * 64, x[v][u]);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                        for (int u = 0; u < NG; ++u)
                            if (u < groups) mma_f16(acc[u], a[kk], x[kk >> 1][u][2 * (kk & 1)], x[kk >> 1][u][2 * (kk & 1) + 1]);
                    give_back(empty_bar(s), acc[0][0]);
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
            if (ok && (!FP8 || w < 4)) {
                const size_t stride = it.x == kFirst ? 2 * (size_t)p.width : (size_t)p.d;
                const int col0 = it.z * 128 + (FP8 ? (w & 3) * 32 : w * 16);
                unsigned long long* dst = (it.x == kFirst ? p.part1 : p.part2) + ((size_t)it.w * rows + first) * stride + col0;
                const bool inside = it.x == kFirst || col0 < p.d;
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int r = 8 * u + 2 * q + v;
                        if (r >= n_rows || !inside) continue;
                        if (FP8) {
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                st_words(dst + r * stride + 16 * t + 2 * g, __float_as_uint(acc[FP8 ? 2 * u + t : 0][v]),
                                         __float_as_uint(acc[FP8 ? 2 * u + t : 0][v + 2]), call);
                        } else {
                            st_word(dst + r * stride + g, __float_as_uint(acc[u][v]), call);
                            st_word(dst + r * stride + g + 8, __float_as_uint(acc[u][v + 2]), call);
                        }
                    }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(x_empty_bar(b));
            ++n;
        }
        lost = !ok;
    } else {
        // ------------------------------------------------------------------------------ routing, sums of complete tiles
        const int w = warp - WARP_SUM;
        bool ok = true;
        auto meet = [&](uint32_t parity) { return meet_at(sum_meet_bar, parity, kErrEpilogueWait); };
        for (uint32_t j = 0; ok; ++j) {
            ok = __all_sync(0xffffffffu, idle_wait(sum_bar(j), (j / SUM_SLOTS) & 1, p.status, kErrEpilogueWait, p.launch_tag));
            if (!ok) break;
            const Item it = take(sum_base + 16u * (j % SUM_SLOTS), sum_free_bar(j));
            if (it.x == kEnd) break;
            if (it.x == kRoute) {
                Patience wait(p.status, p.launch_tag);
                if (p.experts <= 32) ok = route_token<1>(p, rt, it.z, call, wait, meet);
                else if (p.experts == 64) ok = route_token<2>(p, rt, it.z, call, wait, meet);
                else if (p.experts == 128) ok = route_token<4>(p, rt, it.z, call, wait, meet);
                else ok = route_token<8>(p, rt, it.z, call, wait, meet);
            } else if (it.x == kLists) {
                if (w == 0) {
                    Patience wait(p.status, p.launch_tag);
                    ok = pairs <= 32 ? read_routes<1>(p, rt, call, wait) : read_routes<MAX_PAIRS / 32>(p, rt, call, wait);
                    if (ok) build_lists<C::kRows>(p, rt);
                    if (ok && lane == 0) mbar_arrive(routed_bar);
                } else {
                    ok = __all_sync(0xffffffffu, wait_routed(kErrEpilogueWait));
                }
            } else if (it.x == kFirst) {
                // a warp per row, two columns a lane
                Patience wait(p.status, p.launch_tag);
                const int n_rows = pair_count(it), first = first_pair(it);
                for (int r = w; r < n_rows && ok; r += SUM_WARPS) {
                    const unsigned long long* src = p.part1 + (size_t)(first + r) * 2 * p.width + it.z * 128 + 2 * lane;
                    float2 gate, up;
                    ok = sum_chunks(src, src + 64, rows * 2 * p.width, shape.chunks1, call, wait, &gate, &up);
                    if (!ok) break;
                    const float hx = gate.x / (1.0f + expf(-gate.x)) * up.x, hy = gate.y / (1.0f + expf(-gate.y)) * up.y;
                    st_word(p.h + (size_t)(first + r) * (p.width / 2) + it.z * 32 + lane, pack_f16x2(hx, hy), call);
                }
            } else {
                // two warps per token, two columns a lane; the words of two chunks of every expert and of the shared one are in flight
                const int col = it.z * 128 + (w & 1) * 64 + 2 * lane;
                const size_t step = rows * p.d;
                Patience wait(p.status, p.launch_tag);
                for (int t = w >> 1; t < p.t && it.z * 128 + (w & 1) * 64 < p.d && ok; t += SUM_WARPS / 2) {
                    float2 y[kFewMaxTopK + 1];
#pragma unroll
                    for (int i = 0; i <= kFewMaxTopK; ++i) y[i] = make_float2(0.f, 0.f);
                    for (int c0 = 0; c0 < max(shape.chunks2, shape.chunks2s) && ok; c0 += 2) {
                        ulonglong2 v[kFewMaxTopK + 1][2];
                        for (;;) {
                            bool here = true;
#pragma unroll
                            for (int i = 0; i <= kFewMaxTopK; ++i)
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    v[i][c] = make_ulonglong2(word_of(0, call), word_of(0, call));
                                    const bool wanted = i < kFewMaxTopK ? i < p.top_k && c0 + c < shape.chunks2 : c0 + c < shape.chunks2s;
                                    const int pair = i < kFewMaxTopK ? rt.pos[t * p.top_k + min(i, p.top_k - 1)] : pairs + t;
                                    if (wanted) v[i][c] = ld_words(p.part2 + (size_t)(c0 + c) * step + (size_t)pair * p.d + col);
                                }
#pragma unroll
                            for (int i = 0; i <= kFewMaxTopK; ++i)
#pragma unroll
                                for (int c = 0; c < 2; ++c) here = here && call_of(v[i][c].x) == call && call_of(v[i][c].y) == call;
                            if (__all_sync(0xffffffffu, here)) break;
                            ok = __all_sync(0xffffffffu, wait.more());
                            if (!ok) break;
                        }
#pragma unroll
                        for (int i = 0; i <= kFewMaxTopK; ++i)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                y[i].x += float_of(v[i][c].x);
                                y[i].y += float_of(v[i][c].y);
                            }
                    }
                    float2 o = make_float2(0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < kFewMaxTopK; ++i)
                        if (i < p.top_k) {
                            const float wt = rt.weight[t * p.top_k + i];
                            o.x = fmaf(wt, y[i].x, o.x);
                            o.y = fmaf(wt, y[i].y, o.y);
                        }
                    if (ok)
                        *reinterpret_cast<uint32_t*>(static_cast<__half*>(p.out) + (size_t)t * p.d + col) =
                            pack_f16x2(o.x + y[kFewMaxTopK].x, o.y + y[kFewMaxTopK].y);
                }
            }
        }
        lost = !ok;
    }
    if (lost) *reinterpret_cast<volatile int*>(p.head + kFewBad) = 1;
    __syncthreads();
}

template <bool FP8, int NG>
cudaError_t launch_one(const FewMaps& maps, const MoeFewParams& p, int num_sms, cudaStream_t stream) {
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
    return launch_kernel(kernel, dim3((unsigned)num_sms), THREADS, smem, stream, true, maps, p);
}

}  // namespace

cudaError_t moe_few_launch(const MoeFewParams& p, const FewMaps& maps, bool fp8, int num_sms, cudaStream_t stream) {
    if (moe_few_rows(p.t) == 8)
        return fp8 ? launch_one<true, 1>(maps, p, num_sms, stream) : launch_one<false, 1>(maps, p, num_sms, stream);
    return fp8 ? launch_one<true, 2>(maps, p, num_sms, stream) : launch_one<false, 2>(maps, p, num_sms, stream);
}

}  // namespace rf
