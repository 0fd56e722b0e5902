// Internal interface of the MoE layer for a few tokens (moe_few.cu, moe_few_api.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>

namespace rf {

constexpr int kFewMaxTokens = 32;
constexpr int kFewMaxExperts = 256;
constexpr int kFewMaxTopK = 8;

// Words in front of the workspace (128 bytes apart: the ticket is drawn while the others are read)
enum { kFewTicket = 0, kFewExits = 32, kFewBad = 64, kFewCalls = 96, kFewHeadWords = 128 };

// Tensor maps of weights that lie whole rows apart at even distances, as those of one stack do: gate, up, down of all experts one
// below the other, then of the shared one.  As kernel parameters they need no fence.  Where the experts lie anywhere, a table has a
// map for each of their matrices, which the proxy's fence has to be run on at every change of expert: 1.5 % of the time of 1
// token through 4 fp16 experts of 7168 x 2048, 4 % with 13 tokens through 86 of 256 FP8 experts, 6 % with 32 through 8 of 128 of
// 2048 x 768.  (One 3-D map of a stack instead of a 2-D one is 1 % slower for those 13 tokens.)
struct FewMaps {
    CUtensorMap m[6];
    int rows[3];                    // from an expert's matrix to the next one's
};

struct MoeFewParams {
    const void* x;                  // fp16 [t, d]
    const void* router;             // fp16 [experts, d]
    const float* router_bias;       // fp32 [experts] or nullptr
    const CUtensorMap* maps;        // device: gate, up, down of every expert, then of the shared one; or nullptr: FewMaps
    const float* const* scales;     // device: the same order (FP8 weights)
    void* out;                      // fp16 [t, d]
    // workspace: words of 32 bits of data and the call's number
    int* head;                      // kFewHeadWords
    unsigned long long* logits;     // [router_chunks][t][experts] partial sums
    unsigned long long* routes;     // [t][top_k] fp16 probability | 0xFFFF - expert
    unsigned long long* part1;      // [chunks1][pairs][2 * width] partial sums of gate | up, 64 + 64 columns per tile
    unsigned long long* h;          // [pairs][width / 2] two fp16 values each
    unsigned long long* part2;      // [chunks2][pairs][d] partial sums
    int t, d, f, fs;                // fs: the shared expert's width, 0 = none
    int experts, top_k;
    int width;                      // max(f, fs)
    int kc1, kc2;                   // K of an item of the first and the second product
    int router_kc, router_chunks, router_units;
    int* status;
    int launch_tag;
};

// Token rows of an item: 8, or 16.  An expert with more tokens than that (and the shared one) takes several items a tile, of which the
// later find the weights in L2.  (Items of 32 rows leave room for chunks of 512 and an accumulator that spills: 32 tokens through
// 8 of 256 FP8 experts of 7168 x 2048 took 1835 us so.)
inline int moe_few_rows(int t) { return t <= 8 ? 8 : 16; }
inline int moe_few_token_groups(int t) { return (t + 15) / 16; }
// Largest K chunk: its two operand buffers leave room for the weight stages.
constexpr int kFewMaxChunk = 1024;
// K of a router unit: a round of the eight MMA warps.
constexpr int kFewRouterChunk = 512;

// The ring of weight stages, for items of 8 * ng token rows: what fits beside the operand buffers.  FP8 stages are taken in turn by two
// groups of MMA warps, and a group waits for its own stages only.  A wait on a stage's barrier knows odd phases from even ones
// and nothing else: whoever has not seen the phase before would take "not yet there" for "there".  So a slot of the ring
// belongs to one group for good, which an even number of slots makes possible.
__host__ __device__ constexpr int few_stages(bool fp8, int ng) { return ng > 1 ? 8 : fp8 ? 10 : 11; }
// The first stage of an item that is `group`'s, where stage 0 lies in slot s; from there every other one is.
__host__ __device__ constexpr int few_first_stage(int group, int s) { return (group ^ s) & 1; }

cudaError_t moe_few_launch(const MoeFewParams& p, const FewMaps& maps, bool fp8, int num_sms, cudaStream_t stream);

}  // namespace rf
