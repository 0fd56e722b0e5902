// Grouped FP8 block-scaled product for groups of many rows, sm_100a; and the C-ABI entry.
//
// The formula is that of fp8_grouped_few.cu.  Here a tile is 128 rows of a group x 256 columns.  As in fp8_gemm_pair.cu the columns are
// two halves of 128 = one scale block, whose MMAs alternate, each with accumulator buffers and four epilogue warps of its own:
// one half's epilogue works while the other's waits for its next K block; two warps multiply the scales ahead.  What differs is
// where a tile lies and how it leaves: row ranges come from the device, and a warp's 32 rows x 64 columns go out by TMA where they
// are all of the group, else row by row up to the group's end.
//
// What bounds it: as the plain product the power cap and the epilogue's K block, and here the rows that tiles hold beyond their
// groups' ends, half a tile a group.  32768 rows, n 4096, k 7168: one group 0.89 ms (the plain product's CTA pairs 0.81 to 0.90 on
// that box), 32 uneven groups, which need a ninth tile every other time, 0.97 to 1.14 between runs.  The same on CTA pairs with
// 256 x 256 tiles: 1.01 to 1.19; 8192 rows in 32 groups 368 us, here 331; they win in one group only, 870 / 887.
#include "fp8_grouped.cuh"
#include "host_util.h"
#include "launch.h"
#include "../../include/rf_b200.h"

#include <cstdio>

namespace rf {

namespace {

constexpr int BM = 128;          // rows per CTA
constexpr int BK = 128;
constexpr int UMMA_K = 32;
constexpr int HN = 128;          // columns of a half
constexpr int BN = 2 * HN;
constexpr int NB = 512 / BN;     // accumulator buffers of each half
constexpr int NUM_NON_EPI_WARPS = 4;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (NUM_NON_EPI_WARPS + EPI_WARPS);
// 128 * lo + 256 * hi is at most what the CTA was launched with (168 each).  TMEM is read 16 columns at a time: with 32, as in the
// plain product, the K loop spills (CTA pairs, 32768 x 4096 x 7168 in 32 groups: 1.40 ms, so 1.04 to 1.11).
constexpr int kRegsLo = 112, kRegsHi = 192;
static_assert(128 * kRegsLo + 256 * kRegsHi <= 64512, "register split");

constexpr int A_BYTES = BM * BK;
constexpr int CHUNKS = HN / 64;
constexpr int SLAB_BYTES = 32 * 128;
constexpr int SCALE_BYTES = 2 * NB * BM * 4;

constexpr int B_HALF_BYTES = HN * BK;
constexpr int STAGE_BYTES = A_BYTES + 2 * B_HALF_BYTES;
constexpr int STAGES = 3;
constexpr int BAR_BYTES = (2 * STAGES + 4 * NB) * 8 + 16;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * CHUNKS * SLAB_BYTES + SCALE_BYTES + BAR_BYTES +
                           (int)sizeof(GroupTable) + 1024;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");

using F32x2 = unsigned long long;
__device__ __forceinline__ float lo_f32(F32x2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_f32(F32x2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ void fma_f32x2(F32x2& acc, float x, float y, float s) {
    const float2 r = __ffma2_rn(make_float2(x, y), make_float2(s, s), make_float2(lo_f32(acc), hi_f32(acc)));
    acc = (F32x2)__float_as_uint(r.x) | ((F32x2)__float_as_uint(r.y) << 32);
}

__global__ void __launch_bounds__(THREADS, 1)
fp8_grouped_many_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                        const __grid_constant__ CUtensorMap tma_c, const GroupedParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t slab_base = smem_base + STAGES * STAGE_BYTES;
    const uint32_t scale_base = slab_base + EPI_WARPS * CHUNKS * SLAB_BYTES;
    const uint32_t bar_base = scale_base + SCALE_BYTES;
    auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (STAGES + s); };
    auto tmem_full_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + b); };           // b = half * NB + i
    auto tmem_empty_bar = [&](uint32_t b) { return bar_base + 8u * (2 * STAGES + 2 * NB + b); };
    const uint32_t tmem_slot = bar_base + 8u * (2 * STAGES + 4 * NB);
    GroupTable& table = *reinterpret_cast<GroupTable*>(smem_raw + (tmem_slot + 16 - smem_u32(smem_raw)));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    griddep_launch_dependents();
    const int unit = (int)blockIdx.x;
    const int n_units = (int)gridDim.x;

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tma_a);
        tma_prefetch_desc(&tma_b);
        tma_prefetch_desc(&tma_c);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2 * NB; ++b) {
            mbar_init(tmem_full_bar(b), 2);                // the MMAs' commit and the scale warp
            mbar_init(tmem_empty_bar(b), EPI_WARPS / 2);   // the half's four warps
        }
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    griddep_wait();
    build_group_table(table, p, BM);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - smem_u32(smem_raw)));

    const int kb_total = p.k / BK;
    const int tiles_n = (p.n + BN - 1) / BN;
    const int total = table.start[p.groups] * tiles_n;

    if (warp < NUM_NON_EPI_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kRegsLo));
        if (warp == 0) {
            if (elect_one()) {
                // -------------------------------------------------- TMA producer
                uint32_t it = 0, s = 0, ph = 1;
                bool ok = true;
                for (int w = unit; ok && w < total; w += n_units) {
                    const GroupedTile t = decode_grouped(table, p, w, tiles_n);
                    const int a_row0 = table.lo[t.group] + t.m_blk * BM;
                    const int b_row0 = t.group * p.n + t.n_blk * BN;
                    int x = 0;
                    for (const uint32_t end = it + kb_total; it != end; ++it, x += BK) {
                        ok = mbar_wait(empty_bar(s), ph, p.status, kErrProducerWait, p.launch_tag);
                        if (!ok) break;
                        const uint32_t sa = smem_base + s * STAGE_BYTES;
                        mbar_expect_tx(full_bar(s), STAGE_BYTES);
                        tma_load_2d(sa, &tma_a, full_bar(s), x, a_row0);
                        tma_load_2d(sa + A_BYTES, &tma_b, full_bar(s), x, b_row0);       // both halves' rows
                        if (++s == STAGES) { s = 0; ph ^= 1; }
                    }
                }
                finish_producer(ok, it, STAGES, empty_bar(0), p.status, kErrProducerWait, p.launch_tag);
            }
            __syncwarp();
        } else if (warp == 1) {
            if (elect_one()) {
                // ---------------------------------------------------- MMA issuer
                constexpr uint32_t idesc = make_idesc(BM, HN, /*e4m3*/ 0, /*e4m3*/ 0, 0, 0);
                const uint64_t desc0 = smem_desc_kmajor_sw128(smem_base);
                uint32_t it = 0, s = 0, ph = 0;
                bool ok = true;
                for (int w = unit; ok && w < total; w += n_units) {
                    const GroupedTile t = decode_grouped(table, p, w, tiles_n);
                    const bool both = t.n_blk * BN + HN < p.n;        // else the second half has no columns to compute
                    for (const uint32_t end = it + kb_total; it != end; ++it) {
                        const uint32_t buf = it % NB;
                        const uint32_t bph = ((it / NB) & 1) ^ 1;
                        const uint64_t adesc = desc0 + s * (STAGE_BYTES / 16);
                        const uint32_t d = tmem_base + buf * HN;
                        ok = mbar_wait(full_bar(s), ph, p.status, kErrMmaWaitFull, p.launch_tag);
                        if (!ok) break;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            ok = mbar_wait(tmem_empty_bar(h * NB + buf), bph, p.status, kErrMmaWaitTmem, p.launch_tag);
                            if (!ok) break;
                            tc_fence_after();
                            const uint64_t bdesc = adesc + (A_BYTES + h * B_HALF_BYTES) / 16;
                            if (h == 0 || both) {
#pragma unroll
                                for (int j = 0; j < BK / UMMA_K; ++j)
                                    umma_f8(d + h * (NB * HN), adesc + 2 * j, bdesc + 2 * j, idesc, j > 0 ? 1u : 0u);
                            }
                            umma_commit(tmem_full_bar(h * NB + buf));
                        }
                        if (!ok) break;
                        umma_commit(empty_bar(s));
                        if (++s == STAGES) { s = 0; ph ^= 1; }
                    }
                }
            }
            __syncwarp();
        } else {
            // ------------------------------------------------------ scales
            // One warp per half: the products a_s * b_s of the tile's 128 rows, one K block at a time, into the slot of the
            // block's accumulator buffer.  Its loads run PF K blocks ahead, across tiles.  (Rows behind the group's end take
            // the last row's scales: what they are multiplied with is not stored.)
            const int half = warp - 2;
            constexpr int PF = 4;
            int w = unit - n_units;
            uint32_t ar[4], br = 0;            // element offsets of the rows' and the column block's next scales
            int left = 0;
            auto next_tile = [&] {
                w += n_units;
                if (w >= total) return false;
                const GroupedTile t = decode_grouped(table, p, w, tiles_n);
                const int col0 = t.n_blk * BN + half * HN;
                const int row0 = table.lo[t.group] + t.m_blk * BM + 4 * lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) ar[i] = (uint32_t)min(row0 + i, p.m - 1) * (uint32_t)kb_total;
                br = ((uint32_t)t.group * (uint32_t)((p.n + HN - 1) / HN) + (uint32_t)(col0 < p.n ? col0 / HN : 0)) *
                     (uint32_t)kb_total;
                left = kb_total;
                return true;
            };
            bool more = next_tile();
            float qa[PF][4], qb[PF];
            uint32_t n_loaded = 0;
            auto load = [&](int d) {
                if (!more) return;
#pragma unroll
                for (int i = 0; i < 4; ++i) qa[d][i] = ld_global_f32(p.a_scale + ar[i]++);
                qb[d] = ld_global_f32(p.b_scale + br++);
                ++n_loaded;
                if (--left == 0) more = next_tile();
            };
#pragma unroll
            for (int d = 0; d < PF; ++d) load(d);
            bool ok = true;
            for (uint32_t q = 0; ok && q < n_loaded;) {
#pragma unroll
                for (int d = 0; d < PF; ++d) {
                    if (q >= n_loaded) break;
                    // (the epilogue gives accumulator and slot back together)
                    const uint32_t buf = half * NB + q % NB;
                    if (q >= NB) {
                        ok = __all_sync(0xffffffffu, mbar_wait(tmem_empty_bar(buf), (q / NB - 1) & 1, p.status,
                                                               kErrSchedWait, p.launch_tag));
                        if (!ok) break;
                    }
                    const uint32_t slot = scale_base + buf * (BM * 4);
                    st_shared_v4(slot + lane * 16, __float_as_uint(qa[d][0] * qb[d]), __float_as_uint(qa[d][1] * qb[d]),
                                 __float_as_uint(qa[d][2] * qb[d]), __float_as_uint(qa[d][3] * qb[d]));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tmem_full_bar(buf));
                    load(d);
                    ++q;
                }
            }
        }
    } else {
        // ---------------------------------------------------------- epilogue
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kRegsHi));
        const int ew = warp - NUM_NON_EPI_WARPS;
        const int quad = warp & 3;            // TMEM lane quadrant this warp may access
        const int half = ew >> 2;
        const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * (NB * HN);
        const uint32_t slab0 = slab_base + ew * CHUNKS * SLAB_BYTES;
        const uint32_t my_scale = scale_base + half * NB * (BM * 4) + (quad * 32 + lane) * 4;
        uint32_t it = 0;
        F32x2 acc[HN / 2];
#pragma unroll
        for (int j = 0; j < HN / 2; ++j) acc[j] = 0;
        for (int w = unit; w < total; w += n_units) {
            bool ok = true;
#pragma unroll 1
            for (uint32_t end = it + kb_total; it != end; ++it) {
                const uint32_t buf = half * NB + it % NB;
                if (!mbar_wait(tmem_full_bar(buf), (it / NB) & 1, p.status, kErrEpilogueWait, p.launch_tag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t taddr = lane_addr + (it % NB) * HN;
                float v[2][16];
                tmem_ld16_async(taddr, v[0]);
                const float s = __uint_as_float(ld_shared_u32(my_scale + (it % NB) * (BM * 4)));
                // (the scales' slot goes back with the accumulator: behind this load, mbar_arrive_after's rule.  Made at the arrival itself
                // the address cost 4 % of 32768 rows, here 1)
                const uint32_t back = tmem_empty_bar(buf) + (__float_as_uint(s) & ((uint32_t)p.groups >> 16));
#pragma unroll
                for (int c = 0; c < HN / 16; ++c) {
                    tmem_ld16_fence(v[c % 2]);
                    if (c + 1 < HN / 16) tmem_ld16_async(taddr + (c + 1) * 16, v[(c + 1) % 2]);
                    if (c + 1 == HN / 16) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(back);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        fma_f32x2(acc[c * 8 + j], v[c % 2][2 * j], v[c % 2][2 * j + 1], s);
                }
            }
            if (!ok) break;
            // Tile store: 32 rows x 128 bytes slabs, swizzled
            if (lane == 0) tma_store_wait_read<0>();       // (issued a tile ago)
            __syncwarp();
            const bool f16 = p.out_f16 != 0;
#pragma unroll
            for (int ch = 0; ch < CHUNKS; ++ch) {
                const uint32_t my_row = slab0 + ch * SLAB_BYTES + lane * 128;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const F32x2 a = acc[ch * 32 + j * 4 + i];
                        o[i] = f16 ? pack_f16x2(lo_f32(a), hi_f32(a)) : pack_bf16x2(lo_f32(a), hi_f32(a));
                    }
                    st_shared_v4(my_row + ((j ^ (lane & 7)) << 4), o[0], o[1], o[2], o[3]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            const GroupedTile t = decode_grouped(table, p, w, tiles_n);
            const int col0 = t.n_blk * BN + half * HN;
            const int row0 = table.lo[t.group] + t.m_blk * BM + quad * 32;
            const int rows = table.hi[t.group] - row0;
            if (rows >= 32) {
                if (lane == 0) {
                    for (int ch = 0; ch < CHUNKS; ++ch)
                        if (col0 + ch * 64 < p.n) tma_store_2d(&tma_c, slab0 + ch * SLAB_BYTES, col0 + ch * 64, row0);
                    tma_store_commit();
                }
            } else {
                for (int ch = 0; ch < CHUNKS; ++ch) {
                    if (col0 + ch * 64 >= p.n) break;
                    for (int r = lane >> 3; r < rows; r += 4) {
                        const uint4 o = ld_shared_v4(slab0 + ch * SLAB_BYTES + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.c) + (size_t)(row0 + r) * p.n + col0 + ch * 64 +
                                                  (lane & 7) * 8) = o;
                    }
                }
                __syncwarp();
            }
#pragma unroll
            for (int j = 0; j < HN / 2; ++j) acc[j] = 0;
        }
        if (lane == 0) tma_store_wait_read<0>();
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

}  // namespace

cudaError_t fp8_grouped_many_launch(const CUtensorMap& tma_a, const CUtensorMap& tma_b, const CUtensorMap& tma_c,
                                    const GroupedParams& p, int num_sms, cudaStream_t stream) {
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && !attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(fp8_grouped_many_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
        if (e != cudaSuccess) return e;
        attr_set[dev] = true;
    }
    return launch_kernel(fp8_grouped_many_kernel, dim3((unsigned)num_sms), THREADS, SMEM_BYTES, stream, true, tma_a, tma_b, tma_c, p);
}

}  // namespace rf

extern "C" {

int rf_fp8_grouped_gemm(const void* a, const void* b, const float* as, const float* bs, const int* offsets, void* c,
                        int c_dtype, int m, int n_groups, int n, int k, rf_stream_t stream) {
    if (c_dtype != RF_F16 && c_dtype != RF_BF16) return RF_ERR_UNSUPPORTED;
    // (row and scale indices of a and b are 32-bit)
    if (m < 0 || n_groups < 1 || n_groups > rf::kGroupedMaxGroups || n <= 0 || n % 64 != 0 || k <= 0 || k % 128 != 0 ||
        (long long)n_groups * n > 0x7fffffffLL || (long long)m * (k / 128) > 0x7fffffffLL ||
        (long long)n_groups * ((n + 127) / 128) * (k / 128) > 0x7fffffffLL ||
        ((long long)m / 16 + n_groups) * ((n + 127) / 128) > 0x7fffffffLL)
        return RF_ERR_BAD_SHAPE;
    if (m == 0) return RF_OK;
    if (!a || !b || !as || !bs || !offsets || !c) return RF_ERR_NULL_POINTER;
    if (rf::misaligned({a, b, c}, 16) || rf::misaligned({as, bs, offsets}, 4)) return RF_ERR_MISALIGNED;
    rf::DeviceState* st = rf::device_state();
    if (!st) return RF_ERR_CUDA;
    rf::GroupedParams p;
    p.a_scale = as;
    p.b_scale = bs;
    p.offsets = offsets;
    p.c = c;
    p.status = st->status;
    p.launch_tag = rf::next_launch_tag();
    p.m = m; p.n = n; p.k = k; p.groups = n_groups;
    p.out_f16 = c_dtype == RF_F16;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // Few rows a group, or too few tiles of 128 x 256 for the chip, run transposed (us, transposed / not): 1536 rows in 32 groups, n 4096,
    // k 2048 50 / 56, 2048 rows 55 / 57, 4096 rows of k 7168 278 / 230; 1777 rows in 8 groups, n 576, k 2048 12.8 / 13.6.  The counts
    // are on the device: the rule goes by the mean.
    const bool few = m <= 64LL * n_groups || ((long long)m / 128 + n_groups) * ((n + 255) / 256) <= st->num_sms;
    cudaError_t e;
    CUtensorMap ta, tb, tc;
    if (few) {
        if (!rf::encode_tma_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, b, (uint64_t)n_groups * n, (uint64_t)k, (uint64_t)k, 128, 128, true) ||
            !rf::encode_tma_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a, (uint64_t)m, (uint64_t)k, (uint64_t)k, rf::kGroupedFewRows, 128, true))
            return RF_ERR_CUDA;
        e = rf::fp8_grouped_few_launch(tb, ta, p, st->num_sms, s);
    } else {
        if (!rf::encode_tma_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a, (uint64_t)m, (uint64_t)k, (uint64_t)k, 128, 128, true) ||
            !rf::encode_tma_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, b, (uint64_t)n_groups * n, (uint64_t)k, (uint64_t)k, 256, 128, true) ||
            !rf::encode_tma_2d(&tc, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, c, (uint64_t)m, (uint64_t)n, (uint64_t)n * 2, 32, 64, true))
            return RF_ERR_CUDA;
        e = rf::fp8_grouped_many_launch(ta, tb, tc, p, st->num_sms, s);
    }
    if (e != cudaSuccess) {
        fprintf(stderr, "rf_b200: grouped fp8 gemm launch failed: %s\n", cudaGetErrorString(e));
        return RF_ERR_CUDA;
    }
    return RF_OK;
}

}  // extern "C"
