// C-ABI of the MoE layer for a few tokens: one object per layer holds what every call needs of its weights (tensor maps,
// addresses of the scales) on the device; the caller holds the workspace.
#include "../../include/rf_b200.h"
#include "host_util.h"
#include "moe_few.h"

#include <atomic>
#include <cstdint>
#include <cstdio>
#include <new>
#include <vector>

struct RfMoeFew {
    RfMoeFewConfig cfg;
    int device;
    const void* router;
    const float* router_bias;
    void* tables;               // device: maps (if there are any), scales
    CUtensorMap* maps;          // nullptr: the experts lie at even distances
    const float** scales;
    rf::FewMaps even;
};

namespace {

size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

// What a call of t tokens needs: K chunks, and where the parts of the workspace lie.
struct Plan {
    int kc1, kc2, router_kc, router_chunks;
    size_t logits, routes, part1, h, part2, bytes;
};

// The K chunk for `tiles` column tiles: least rounds of items over the SMs x (chunk + what an item costs beside its weights, about
// 120 of K).  A call whose weights fit one round takes the longest chunk that still gives every SM an item: all its loads are then
// in flight at once (9 experts of 1024 x 512: 18.2 us with 288 and 144 items, two rounds and one).
int choose_chunk(int tiles, int k, int most, int num_sms) {
    int best = most;
    long long least = -1;
    for (int kc = most; kc >= 256; kc /= 2) {
        const long long items = (long long)tiles * ((k + kc - 1) / kc);
        const long long cost = ((items + num_sms - 1) / num_sms) * ((kc < k ? kc : k) + 120);
        if (least < 0 || cost < least) {
            least = cost;
            best = kc;
        }
    }
    return best;
}

Plan make_plan(const RfMoeFewConfig& c, int t) {
    const int num_sms = 148;        // a B200's: a workspace's size needs no device (with another count the plan is less even)
    const int fs = c.d_expert * c.n_shared_experts, width = fs > c.d_expert ? fs : c.d_expert;
    const int hit = c.n_routed_experts < t * c.n_experts_per_token ? c.n_routed_experts : t * c.n_experts_per_token;
    const size_t pairs = (size_t)t * (c.n_experts_per_token + 1), d = c.d_hidden;
    Plan p;
    p.kc1 = choose_chunk((hit * c.d_expert + fs) / 64, c.d_hidden, rf::kFewMaxChunk, num_sms);
    p.kc2 = choose_chunk((hit + (fs > 0)) * ((c.d_hidden + 127) / 128), c.d_expert, rf::kFewMaxChunk, num_sms);
    p.router_kc = rf::kFewRouterChunk;
    p.router_chunks = (c.d_hidden + p.router_kc - 1) / p.router_kc;
    const size_t chunks1 = (d + p.kc1 - 1) / p.kc1, chunks2 = ((size_t)width + p.kc2 - 1) / p.kc2;
    size_t b = rf::kFewHeadWords * sizeof(int);
    auto take = [&](size_t words) { const size_t at = b; b += align_up(words * 8); return at; };
    p.logits = take((size_t)p.router_chunks * t * c.n_routed_experts);
    p.routes = take((size_t)t * c.n_experts_per_token);
    p.part1 = take(chunks1 * pairs * 2 * width);
    p.h = take(pairs * width / 2);
    p.part2 = take(chunks2 * pairs * d);
    p.bytes = b;
    return p;
}

int check_config(const RfMoeFewConfig& c) {
    if (c.weight_type != RF_MOE_FEW_F16 && c.weight_type != RF_MOE_FEW_E4M3) return RF_ERR_UNSUPPORTED;
    const int step = c.weight_type == RF_MOE_FEW_E4M3 ? 128 : 64;
    if (c.d_hidden <= 0 || c.d_hidden % step != 0 || c.d_expert <= 0 || c.d_expert % step != 0) return RF_ERR_BAD_SHAPE;
    if (c.n_shared_experts < 0 || c.n_shared_experts > 64 || c.d_hidden > (1 << 20) || c.d_expert > (1 << 20)) return RF_ERR_BAD_SHAPE;
    const int e = c.n_routed_experts;
    if (e < 1 || e > rf::kFewMaxExperts || (e & (e - 1)) != 0) return RF_ERR_UNSUPPORTED;
    if (c.n_experts_per_token < 1 || c.n_experts_per_token > rf::kFewMaxTopK || c.n_experts_per_token > e) return RF_ERR_UNSUPPORTED;
    return RF_OK;
}

// Memory that belongs to a captured graph (a CUDA user object of it, which its executables own too).  When the last of them has gone,
// the object's destructor runs on a thread of CUDA's that may call nothing of CUDA: it only says so, and a later call frees.
struct GraphMemory {
    void* ptr;
    size_t bytes;
    GraphMemory* next;
};
std::atomic<GraphMemory*> g_left{nullptr};
std::atomic<size_t> g_with_graphs{0};

void CUDART_CB graph_gone(void* p) {
    GraphMemory* m = static_cast<GraphMemory*>(p);
    m->next = g_left.load(std::memory_order_relaxed);
    while (!g_left.compare_exchange_weak(m->next, m, std::memory_order_release, std::memory_order_relaxed)) {
    }
}

// (in relaxed capture mode)
cudaError_t free_left() {
    cudaError_t e = cudaSuccess;
    for (GraphMemory* m = g_left.exchange(nullptr, std::memory_order_acquire); m != nullptr;) {
        GraphMemory* next = m->next;
        const cudaError_t f = cudaFree(m->ptr);
        if (f != cudaSuccess) e = f;
        g_with_graphs -= m->bytes;
        delete m;
        m = next;
    }
    return e;
}

// While a stream of this thread is being captured: what runs inside touches none that is.
class Relaxed {
public:
    Relaxed() { ok_ = cudaThreadExchangeStreamCaptureMode(&mode_) == cudaSuccess; }
    ~Relaxed() {
        if (ok_) cudaThreadExchangeStreamCaptureMode(&mode_);
    }
    bool ok() const { return ok_; }

private:
    cudaStreamCaptureMode mode_ = cudaStreamCaptureModeRelaxed;
    bool ok_;
};

cudaError_t zeroed(size_t bytes, void** out) {
    void* p = nullptr;
    cudaError_t e = cudaMalloc(&p, bytes);
    if (e == cudaSuccess) e = rf::upload_zeroes(p, bytes);
    if (e != cudaSuccess) {
        cudaGetLastError();
        if (p) cudaFree(p);
        p = nullptr;
    }
    *out = p;
    return e;
}

// Weights of k x n; `below`: rows that the map reaches beyond them
bool encode(CUtensorMap* m, bool fp8, const void* base, int k, int n, long long below) {
    return fp8 ? rf::encode_tma_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, (uint64_t)(n + below), (uint64_t)k, (uint64_t)k, 64, 128, true)
               : rf::encode_tma_2d(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, (uint64_t)(k + below), (uint64_t)n, (uint64_t)n * 2, 64, 64,
                                   true);
}

// Rows from one matrix of `rows` rows to the next, where all lie evenly and a coordinate reaches the last one; else 0.
int rows_apart(const void* const* p, int count, long long rows, long long row_bytes) {
    const long long apart = count > 1 ? (long long)((uintptr_t)p[1] - (uintptr_t)p[0]) : rows * row_bytes;
    for (int i = 2; i < count; ++i)
        if ((long long)((uintptr_t)p[i] - (uintptr_t)p[i - 1]) != apart) return 0;
    return apart >= rows * row_bytes && apart % row_bytes == 0 && apart / row_bytes <= 0x7fffffffLL / count ? (int)(apart / row_bytes) : 0;
}

}  // namespace

extern "C" {

int rf_moe_few_create(const RfMoeFewConfig* config, const void* router_weight, const float* router_bias,
                      const void* const* expert_gate, const void* const* expert_up, const void* const* expert_down,
                      const float* const* gate_scale, const float* const* up_scale, const float* const* down_scale,
                      RfMoeFew** out) {
    if (!config || !out) return RF_ERR_NULL_POINTER;
    *out = nullptr;
    const int rc = check_config(*config);
    if (rc != RF_OK) return rc;
    const RfMoeFewConfig& c = *config;
    const bool fp8 = c.weight_type == RF_MOE_FEW_E4M3;
    if (!router_weight || !expert_gate || !expert_up || !expert_down || (fp8 && (!gate_scale || !up_scale || !down_scale)))
        return RF_ERR_NULL_POINTER;
    const int sets = c.n_routed_experts + (c.n_shared_experts > 0 ? 1 : 0);
    for (int e = 0; e < sets; ++e) {
        if (!expert_gate[e] || !expert_up[e] || !expert_down[e]) return RF_ERR_NULL_POINTER;
        if (rf::misaligned({expert_gate[e], expert_up[e], expert_down[e]}, 16)) return RF_ERR_MISALIGNED;
        if (!fp8) continue;
        if (!gate_scale[e] || !up_scale[e] || !down_scale[e]) return RF_ERR_NULL_POINTER;
        if (rf::misaligned({gate_scale[e], up_scale[e], down_scale[e]}, 4)) return RF_ERR_MISALIGNED;
    }
    if (rf::misaligned({router_weight}, 16) || rf::misaligned({router_bias}, 4)) return RF_ERR_MISALIGNED;
    if (!rf::device_state()) return RF_ERR_CUDA;
    const int experts = c.n_routed_experts, d = c.d_hidden, f = c.d_expert, fs = f * c.n_shared_experts;
    const void* const* const mats[3] = {expert_gate, expert_up, expert_down};
    const float* const* const mat_scales[3] = {gate_scale, up_scale, down_scale};
    rf::FewMaps even_maps = {};
    std::vector<CUtensorMap> maps;
    std::vector<const float*> scales;
    bool even = true;
    for (int i = 0; i < 3; ++i) {
        const int k = i < 2 ? d : f, n = i < 2 ? f : d;            // (FP8 rows are the n of a matrix, fp16 ones its k)
        even_maps.rows[i] = rows_apart(mats[i], experts, fp8 ? n : k, fp8 ? k : 2LL * n);
        even = even && even_maps.rows[i] != 0;
    }
    try {
        if (!even) maps.resize((size_t)3 * sets);
        scales.resize((size_t)3 * sets, nullptr);
    } catch (const std::bad_alloc&) {
        return RF_ERR_CUDA;
    }
    for (int i = 0; i < 3; ++i) {
        auto one = [&](CUtensorMap* m, const void* base, int width, long long below) {
            return i < 2 ? encode(m, fp8, base, d, width, below) : encode(m, fp8, base, width, d, below);
        };
        if (even && !one(&even_maps.m[i], mats[i][0], f, (experts - 1LL) * even_maps.rows[i])) return RF_ERR_CUDA;
        if (even && fs > 0 && !one(&even_maps.m[3 + i], mats[i][experts], fs, 0)) return RF_ERR_CUDA;
        for (int e = 0; e < sets; ++e) {
            if (!even && !one(&maps[3 * e + i], mats[i][e], e < experts ? f : fs, 0)) return RF_ERR_CUDA;
            if (fp8) scales[3 * e + i] = mat_scales[i][e];
        }
    }
    RfMoeFew* few = new (std::nothrow) RfMoeFew();
    if (!few) return RF_ERR_CUDA;
    few->cfg = c;
    few->router = router_weight;
    few->router_bias = router_bias;
    few->even = even_maps;
    cudaGetDevice(&few->device);
    const size_t map_bytes = maps.size() * sizeof(CUtensorMap), scale_bytes = scales.size() * sizeof(float*);
    char* dev = nullptr;
    if (cudaMalloc(&dev, map_bytes + scale_bytes) != cudaSuccess) {
        cudaGetLastError();
        delete few;
        return RF_ERR_CUDA;
    }
    few->tables = dev;
    few->maps = even ? nullptr : reinterpret_cast<CUtensorMap*>(dev);
    few->scales = reinterpret_cast<const float**>(dev + map_bytes);
    if ((!even && rf::upload(dev, maps.data(), map_bytes) != cudaSuccess) ||
        rf::upload(dev + map_bytes, scales.data(), scale_bytes) != cudaSuccess) {
        cudaFree(dev);
        delete few;
        return RF_ERR_CUDA;
    }
    *out = few;
    return RF_OK;
}

int rf_moe_few_destroy(RfMoeFew* few) {
    if (!few) return RF_OK;
    const int rc = rf_moe_few_workspace_free(few->tables);       // (may come from a garbage collector during a capture)
    delete few;
    return rc;
}

size_t rf_moe_few_workspace_bytes(const RfMoeFewConfig* config, int n_tokens) {
    if (!config || check_config(*config) != RF_OK || n_tokens < 1 || n_tokens > rf::kFewMaxTokens) return 0;
    return make_plan(*config, n_tokens).bytes;
}

int rf_moe_few_workspace_alloc(size_t bytes, void** out) {
    if (!out) return RF_ERR_NULL_POINTER;
    *out = nullptr;
    if (!rf::device_state()) return RF_ERR_CUDA;
    Relaxed relaxed;
    if (!relaxed.ok()) return RF_ERR_CUDA;
    free_left();
    return zeroed(bytes, out) == cudaSuccess ? RF_OK : RF_ERR_CUDA;
}

int rf_moe_few_workspace_alloc_captured(rf_stream_t stream, size_t bytes, void** out) {
    if (!out) return RF_ERR_NULL_POINTER;
    *out = nullptr;
    if (!rf::device_state()) return RF_ERR_CUDA;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    cudaGraph_t graph = nullptr;
    if (cudaStreamGetCaptureInfo_v2(reinterpret_cast<cudaStream_t>(stream), &status, nullptr, &graph) != cudaSuccess)
        return RF_ERR_CUDA;
    if (status != cudaStreamCaptureStatusActive || graph == nullptr) return RF_ERR_UNSUPPORTED;
    GraphMemory* m = new (std::nothrow) GraphMemory{nullptr, bytes, nullptr};
    if (!m) return RF_ERR_CUDA;
    Relaxed relaxed;
    if (relaxed.ok()) free_left();
    if (!relaxed.ok() || zeroed(bytes, &m->ptr) != cudaSuccess) {
        delete m;
        return RF_ERR_CUDA;
    }
    cudaUserObject_t object = nullptr;
    if (cudaUserObjectCreate(&object, m, graph_gone, 1, cudaUserObjectNoDestructorSync) != cudaSuccess) {
        cudaFree(m->ptr);
        delete m;
        return RF_ERR_CUDA;
    }
    g_with_graphs += bytes;
    if (cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove) != cudaSuccess) {
        cudaUserObjectRelease(object, 1);
        return RF_ERR_CUDA;
    }
    *out = m->ptr;
    return RF_OK;
}

int rf_moe_few_workspace_free(void* workspace) {
    Relaxed relaxed;
    if (!relaxed.ok()) return RF_ERR_CUDA;
    const cudaError_t left = free_left(), e = cudaFree(workspace);
    return left == cudaSuccess && e == cudaSuccess ? RF_OK : RF_ERR_CUDA;
}

int rf_moe_few_workspace_reap(size_t* bytes) {
    cudaError_t e = cudaSuccess;
    if (g_left.load(std::memory_order_relaxed) != nullptr) {
        Relaxed relaxed;
        if (!relaxed.ok()) return RF_ERR_CUDA;
        e = free_left();
    }
    if (bytes) *bytes = g_with_graphs.load(std::memory_order_relaxed);
    return e == cudaSuccess ? RF_OK : RF_ERR_CUDA;
}

int rf_stream_capture_id(rf_stream_t stream, unsigned long long* id) {
    if (!id) return RF_ERR_NULL_POINTER;
    *id = 0;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long n = 0;
    if (cudaStreamGetCaptureInfo(reinterpret_cast<cudaStream_t>(stream), &status, &n) != cudaSuccess) return RF_ERR_CUDA;
    if (status != cudaStreamCaptureStatusNone) *id = n + 1;
    return RF_OK;
}

int rf_moe_few_forward(RfMoeFew* few, const void* x, int n_tokens, void* out, void* workspace, size_t workspace_bytes,
                       rf_stream_t stream) {
    if (!few) return RF_ERR_NULL_POINTER;
    if (n_tokens < 0 || n_tokens > rf::kFewMaxTokens) return RF_ERR_BAD_SHAPE;
    if (n_tokens == 0) return RF_OK;
    if (!x || !out || !workspace) return RF_ERR_NULL_POINTER;
    if (rf::misaligned({x, out}, 16) || rf::misaligned({workspace}, 256)) return RF_ERR_MISALIGNED;
    // (x is read until the kernel's end)
    const uintptr_t xa = reinterpret_cast<uintptr_t>(x), oa = reinterpret_cast<uintptr_t>(out);
    if ((xa < oa ? oa - xa : xa - oa) < (uintptr_t)n_tokens * few->cfg.d_hidden * 2) return RF_ERR_UNSUPPORTED;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev != few->device) return RF_ERR_UNSUPPORTED;
    const RfMoeFewConfig& c = few->cfg;
    const Plan plan = make_plan(c, n_tokens);
    if (workspace_bytes < plan.bytes) return RF_ERR_WORKSPACE;
    rf::DeviceState* st = rf::device_state();
    if (!st) return RF_ERR_CUDA;
    char* ws = static_cast<char*>(workspace);
    rf::MoeFewParams p;
    p.x = x;
    p.router = few->router;
    p.router_bias = few->router_bias;
    p.maps = few->maps;
    p.scales = few->scales;
    p.out = out;
    p.head = reinterpret_cast<int*>(ws);
    p.logits = reinterpret_cast<unsigned long long*>(ws + plan.logits);
    p.routes = reinterpret_cast<unsigned long long*>(ws + plan.routes);
    p.part1 = reinterpret_cast<unsigned long long*>(ws + plan.part1);
    p.h = reinterpret_cast<unsigned long long*>(ws + plan.h);
    p.part2 = reinterpret_cast<unsigned long long*>(ws + plan.part2);
    p.t = n_tokens;
    p.d = c.d_hidden;
    p.f = c.d_expert;
    p.fs = c.d_expert * c.n_shared_experts;
    p.experts = c.n_routed_experts;
    p.top_k = c.n_experts_per_token;
    p.width = p.fs > p.f ? p.fs : p.f;
    p.kc1 = plan.kc1;
    p.kc2 = plan.kc2;
    p.router_kc = plan.router_kc;
    p.router_chunks = plan.router_chunks;
    p.router_units = (p.experts + 15) / 16 * p.router_chunks * rf::moe_few_token_groups(p.t);
    p.status = st->status;
    p.launch_tag = rf::next_launch_tag();
    const cudaError_t e = rf::moe_few_launch(p, few->even, c.weight_type == RF_MOE_FEW_E4M3, st->num_sms, reinterpret_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
        fprintf(stderr, "rf_b200: launch of the layer for a few tokens failed: %s\n", cudaGetErrorString(e));
        return RF_ERR_CUDA;
    }
    return RF_OK;
}

}  // extern "C"
