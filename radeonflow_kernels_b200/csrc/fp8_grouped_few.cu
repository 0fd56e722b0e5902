// Grouped FP8 block-scaled product for groups of few rows (a decode step's experts), sm_100a.
//
//   c[r, n] = sum_kb a_s[r, kb] b_s[g, n/128, kb] sum_{j < 128} a[r, 128 kb + j] b[g, n, 128 kb + j],   r in group g
//
// The product is computed transposed: 128 rows of a group's weight are the MMA's M, the group's rows (up to 64 in a tile) its N in
// steps of 16, so that a dozen rows cost a 16-wide MMA beside the weight stream, which bounds the kernel: 512 rows in 32 groups,
// n 7168, k 2048 take 79 us, 6.0 TB/s of what cannot be left out.  Scales differ per accumulator column then (one product a_s * b_s
// per row of a), and a scale warp leaves them in shared memory, from where they are broadcast to the promotion's FMAs.  (Those
// reads are what larger tiles fail at: 256 rows a tile, 32768 rows of k 7168, 1.33 ms where fp8_grouped.cu takes 0.92.)
// Warps of the one persistent CTA per SM:
//   warp 0      TMA producer: 16 KB of weights and 64 rows of a, 128 deep, per stage
//   warp 1      MMA issuer: 4 x tcgen05.mma (M 128) per K block into one of four accumulator buffers
//   warp 2      scales of the next K blocks
//   warps 4-11  epilogue, two per lane quadrant with half of the columns each: fp32 promotion in registers, direct stores
// Tiles of 16 and 32 rows were measured beside those of 64 (us, 16 / 32 / 64): 512 rows in 32 groups as above 82 / 80 / 79; 128
// rows in 32 groups, n 4096, k 7168 145 / 143 / 140; 1777 rows in 64 uneven groups, n 1472, k 1024 33 / 26 / 24; 8 rows in 8
// groups, n 4096, k 2048 12.4 / 13.0 / 13.5.
#include "fp8_grouped.cuh"
#include "launch.h"

namespace rf {

namespace {

constexpr int BK = 128;
constexpr int UMMA_K = 32;
constexpr int W_BYTES = 128 * BK;
constexpr int NB = 4;                       // accumulator buffers
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (4 + EPI_WARPS);

constexpr int NT = kGroupedFewRows;
constexpr int HALF = NT / 2;                // columns of one epilogue warp: one TMEM load
static_assert(HALF == 32, "tmem_ld32");
constexpr int X_BYTES = NT * BK;
constexpr int STAGE_BYTES = W_BYTES + X_BYTES;
constexpr int STAGES = 8;
constexpr int TMEM_COLS = NB * NT;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + NB * NT * 4 + (2 * STAGES + 2 * NB) * 8 + 16 + (int)sizeof(GroupTable) + 1024;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");

__global__ void __launch_bounds__(THREADS, 1)
fp8_grouped_few_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x,
                       const GroupedParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t scale_base = smem_base + STAGES * STAGE_BYTES;
    const uint32_t bar_base = scale_base + NB * NT * 4;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto tmem_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };
    auto tmem_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + NB + b); };
    const uint32_t tmem_slot = bar_base + 8u * (2 * STAGES + 2 * NB);
    GroupTable& table = *reinterpret_cast<GroupTable*>(smem_raw + (tmem_slot + 16 - smem_u32(smem_raw)));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    griddep_launch_dependents();
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tma_w);
        tma_prefetch_desc(&tma_x);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < NB; ++b) {
            mbar_init(tmem_full_bar(b), 2);                // the MMAs' commit and the scale warp
            mbar_init(tmem_empty_bar(b), EPI_WARPS);
        }
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    griddep_wait();
    build_group_table(table, p, NT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - smem_u32(smem_raw)));

    const int kb_total = p.k / BK;
    const int tiles_n = (p.n + 127) / 128;
    const int total = table.start[p.groups] * tiles_n;

    if (warp == 0) {
        if (elect_one()) {
            uint32_t it = 0, s = 0, ph = 1;
            bool ok = true;
            for (int w = blockIdx.x; ok && w < total; w += gridDim.x) {
                const GroupedTile t = decode_grouped(table, p, w, tiles_n);
                const int x_row = table.lo[t.group] + t.m_blk * NT, w_row = t.group * p.n + t.n_blk * 128;
                for (int kb = 0; kb < kb_total; ++kb, ++it) {
                    ok = mbar_wait(empty_bar(s), ph, p.status, kErrProducerWait, p.launch_tag);
                    if (!ok) break;
                    const uint32_t st = smem_base + s * STAGE_BYTES;
                    mbar_expect_tx(full_bar(s), STAGE_BYTES);
                    tma_load_2d(st, &tma_w, full_bar(s), kb * BK, w_row);
                    tma_load_2d(st + W_BYTES, &tma_x, full_bar(s), kb * BK, x_row);
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
            finish_producer(ok, it, STAGES, empty_bar(0), p.status, kErrProducerWait, p.launch_tag);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            const uint64_t desc0 = smem_desc_kmajor_sw128(smem_base);
            uint32_t it = 0, s = 0, ph = 0;
            bool ok = true;
            for (int w = blockIdx.x; ok && w < total; w += gridDim.x) {
                const GroupedTile t = decode_grouped(table, p, w, tiles_n);
                const int rows = min(table.hi[t.group] - table.lo[t.group] - t.m_blk * NT, NT);
                const uint32_t idesc = make_idesc(128, (rows + 15) & ~15, /*e4m3*/ 0, /*e4m3*/ 0, 0, 0);
                for (int kb = 0; kb < kb_total; ++kb, ++it) {
                    const uint32_t buf = it % NB;
                    ok = mbar_wait(full_bar(s), ph, p.status, kErrMmaWaitFull, p.launch_tag) &&
                         mbar_wait(tmem_empty_bar(buf), ((it / NB) & 1) ^ 1, p.status, kErrMmaWaitTmem, p.launch_tag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t wdesc = desc0 + s * (STAGE_BYTES / 16), xdesc = wdesc + W_BYTES / 16;
#pragma unroll
                    for (int j = 0; j < BK / UMMA_K; ++j)
                        umma_f8(tmem_base + buf * NT, wdesc + 2 * j, xdesc + 2 * j, idesc, j > 0 ? 1u : 0u);
                    umma_commit(tmem_full_bar(buf));
                    umma_commit(empty_bar(s));
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        // The products a_s * b_s of the tile's rows, K block by K block; loads run PF K blocks ahead inside a tile.
        // (Rows behind the group's end take the matrix's last row's: what they are multiplied with is not stored.)
        constexpr int PER = NT / 32;
        constexpr int PF = 4;
        uint32_t it = 0;
        bool ok = true;
        for (int w = blockIdx.x; ok && w < total; w += gridDim.x) {
            const GroupedTile t = decode_grouped(table, p, w, tiles_n);
            const int row0 = table.lo[t.group] + t.m_blk * NT;
            const float* as[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) as[i] = p.a_scale + (size_t)min(row0 + i * 32 + lane, p.m - 1) * kb_total;
            const float* bs = p.b_scale + ((size_t)t.group * tiles_n + t.n_blk) * kb_total;
            float qa[PF][PER], qb[PF];
            auto load = [&](int d, int kb) {
                if (kb >= kb_total) return;
#pragma unroll
                for (int i = 0; i < PER; ++i) qa[d][i] = ld_global_f32(as[i] + kb);
                qb[d] = ld_global_f32(bs + kb);
            };
#pragma unroll
            for (int d = 0; d < PF; ++d) load(d, d);
            for (int kb0 = 0; ok && kb0 < kb_total; kb0 += PF) {
#pragma unroll
                for (int d = 0; d < PF; ++d) {
                    const int kb = kb0 + d;
                    if (kb >= kb_total || !ok) break;
                    const uint32_t buf = it % NB;
                    // (the epilogue's arrivals say that it has read the slot too)
                    ok = __all_sync(0xffffffffu, mbar_wait(tmem_empty_bar(buf), ((it / NB) & 1) ^ 1, p.status, kErrSchedWait,
                                                           p.launch_tag));
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < PER; ++i) st_shared_f32(scale_base + (buf * NT + i * 32 + lane) * 4, qa[d][i] * qb[d]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tmem_full_bar(buf));
                    load(d, kb + PF);
                    ++it;
                }
            }
        }
    } else if (warp >= 4) {
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * HALF;
        uint32_t it = 0;
        for (int w = blockIdx.x; w < total; w += gridDim.x) {
            float2 acc[HALF / 2];
#pragma unroll
            for (int j = 0; j < HALF / 2; ++j) acc[j] = make_float2(0.f, 0.f);
            bool ok = true;
#pragma unroll 1
            for (int kb = 0; kb < kb_total; ++kb, ++it) {
                const uint32_t buf = it % NB;
                ok = mbar_wait(tmem_full_bar(buf), (it / NB) & 1, p.status, kErrEpilogueWait, p.launch_tag);
                if (!ok) break;
                tc_fence_after();
                float v[HALF];
                tmem_ld32(lane_addr + buf * NT, v);
                const uint32_t sc = scale_base + (buf * NT + half * HALF) * 4;
                uint32_t seen = 0;
#pragma unroll
                for (int j = 0; j < HALF / 4; ++j) {
                    const uint4 s = ld_shared_v4(sc + 16 * j);
                    seen |= s.x;
                    acc[2 * j] = __ffma2_rn(make_float2(v[4 * j], v[4 * j + 1]),
                                            make_float2(__uint_as_float(s.x), __uint_as_float(s.y)), acc[2 * j]);
                    acc[2 * j + 1] = __ffma2_rn(make_float2(v[4 * j + 2], v[4 * j + 3]),
                                                make_float2(__uint_as_float(s.z), __uint_as_float(s.w)), acc[2 * j + 1]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_after(tmem_empty_bar(buf), seen, (uint32_t)p.groups >> 16);
            }
            if (!ok) break;
            const GroupedTile t = decode_grouped(table, p, w, tiles_n);
            const int row0 = table.lo[t.group] + t.m_blk * NT + half * HALF;
            const int rows = min(table.hi[t.group] - row0, HALF);
            const int col = t.n_blk * 128 + quad * 32 + lane;
            if (t.n_blk * 128 + quad * 32 < p.n) {
                uint16_t* c = static_cast<uint16_t*>(p.c) + (size_t)row0 * p.n + col;
#pragma unroll
                for (int j = 0; j < HALF; ++j) {
                    if (j >= rows) break;
                    const float v = j & 1 ? acc[j / 2].y : acc[j / 2].x;
                    c[(size_t)j * p.n] = p.out_f16 ? __half_as_ushort(__float2half_rn(v))
                                                   : __bfloat16_as_ushort(__float2bfloat16_rn(v));
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

}  // namespace

cudaError_t fp8_grouped_few_launch(const CUtensorMap& tma_w, const CUtensorMap& tma_x, const GroupedParams& p, int num_sms,
                                   cudaStream_t stream) {
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && !attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(fp8_grouped_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
        if (e != cudaSuccess) return e;
        attr_set[dev] = true;
    }
    return launch_kernel(fp8_grouped_few_kernel, dim3((unsigned)num_sms), THREADS, SMEM_BYTES, stream, true, tma_w, tma_x, p);
}

}  // namespace rf
