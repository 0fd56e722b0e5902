// What the two kernels of the grouped FP8 product share: parameters and the table of groups.
#pragma once
#include "ptx.cuh"

namespace rf {

constexpr int kGroupedMaxGroups = 1024;

struct GroupedParams {
    const float* a_scale;       // [m, k/128]
    const float* b_scale;       // [groups, ceil(n/128), k/128]
    const int* offsets;         // [groups + 1], device
    void* c;                    // [m, n], bf16 or fp16
    int* status;                // device status area (status_words.h)
    int launch_tag;
    int m, n, k, groups;
    int out_f16;                // c is fp16, else bf16
};

// Row ranges of the groups and the number of tiles in front of each, in shared memory.
struct GroupTable {
    int lo[kGroupedMaxGroups], hi[kGroupedMaxGroups];
    int start[kGroupedMaxGroups + 1];       // [groups] = all tiles
    int sums[33];
};

__device__ __forceinline__ int clipped_offset(const GroupedParams& p, int g) {
    return min(max(ld_global_s32(p.offsets + g), 0), p.m);
}

// Every thread of the CTA calls it (the caller synchronises behind it).  A group's rows are cut into tiles of `tile_rows`.
// Offsets are clipped to 0 .. m, and one below an earlier one counts as that: no table leads outside the matrices, no row is in two
// groups, and there are m / tile_rows + groups tiles at most.
__device__ __forceinline__ void build_group_table(GroupTable& t, const GroupedParams& p, int tile_rows) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_warps = blockDim.x >> 5;
    const int per = (p.groups + blockDim.x - 1) / blockDim.x;
    const int g0 = min(tid * per, p.groups), g1 = min(g0 + per, p.groups);
    int mine = 0;
    bool descends = false;
    for (int g = g0; g < g1; ++g) {
        const int lo = clipped_offset(p, g), hi = clipped_offset(p, g + 1);
        descends = descends || hi < lo;
        t.lo[g] = lo;
        t.hi[g] = hi;
        mine += (hi - lo + tile_rows - 1) / tile_rows;
    }
    int incl = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, s);
        if (lane >= s) incl += o;
    }
    if (lane == 31) t.sums[warp] = incl;
    if (__syncthreads_or(descends)) {           // no table that a permutation makes: one thread takes its time
        if (tid == 0) {
            int at = clipped_offset(p, 0), run = 0;
            for (int g = 0; g < p.groups; ++g) {
                const int end = max(at, clipped_offset(p, g + 1));
                t.lo[g] = at;
                t.hi[g] = end;
                t.start[g] = run;
                run += (end - at + tile_rows - 1) / tile_rows;
                at = end;
            }
            t.start[p.groups] = run;
        }
        return;
    }
    int before = 0, all = 0;
    for (int w = 0; w < n_warps; ++w) {
        if (w < warp) before += t.sums[w];
        all += t.sums[w];
    }
    int run = before + incl - mine;
    for (int g = g0; g < g1; ++g) {
        t.start[g] = run;
        run += (t.hi[g] - t.lo[g] + tile_rows - 1) / tile_rows;
    }
    if (tid == 0) t.start[p.groups] = all;
}

// Work item -> group, tile of the group, block of columns.  A group's items stand together, row tiles first inside bands of
// eight, so that the CTAs at work share weight columns (and, across columns, the band's rows) in L2.
struct GroupedTile {
    int group, m_blk, n_blk;
};
__device__ __forceinline__ GroupedTile decode_grouped(const GroupTable& t, const GroupedParams& p, int w, int tiles_n) {
    const int tile = w / tiles_n;
    int lo = 0, hi = p.groups;                      // the last group that starts at or before the tile (one without tiles
    while (hi - lo > 1) {                           // starts where the next one does)
        const int mid = (lo + hi) >> 1;
        if (t.start[mid] <= tile) lo = mid;
        else hi = mid;
    }
    const int first = t.start[lo], tiles_m = t.start[lo + 1] - first, r = w - first * tiles_n;
    const int band = r / (8 * tiles_n), first_m = band * 8, rows = min(8, tiles_m - first_m);
    const int in_band = r - band * 8 * tiles_n;
    const int n_blk = in_band / rows;
    return GroupedTile{lo, first_m + in_band - n_blk * rows, n_blk};
}

// tma_w: boxes of 128 weight rows, tma_x: of kGroupedFewRows rows of a
constexpr int kGroupedFewRows = 64;
cudaError_t fp8_grouped_few_launch(const CUtensorMap& tma_w, const CUtensorMap& tma_x, const GroupedParams& p, int num_sms,
                                   cudaStream_t stream);
// tma_a: boxes of 128 rows of a, tma_b: of 256 weight rows, tma_c: 32 x 64
cudaError_t fp8_grouped_many_launch(const CUtensorMap& tma_a, const CUtensorMap& tma_b, const CUtensorMap& tma_c,
                                    const GroupedParams& p, int num_sms, cudaStream_t stream);

}  // namespace rf
