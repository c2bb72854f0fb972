// C entry points of the paged key/value cache (declared in include/mlq_hip.h).
// Every check runs on the host before any launch: the batch's lengths and page
// ids when it is set (kv_plan.cpp), buffers and layers at each call.

#include "abi.h"
#include "kv_layout.h"
#include "kv_plan.h"

#include "../../include/mlq_hip.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <string>
#include <vector>

namespace {

constexpr int64_t kMost = int64_t(1) << 30;

struct KvMemory {
    int device = 0, qtype = 0, n_layers = 0, n_pages = 0, page_size = 0, n_kv = 0, head_dim = 0, nb = 0;
    size_t layer_bytes = 0;
    uint8_t* mem = nullptr;

    size_t bytes() const { return layer_bytes * n_layers; }
    ~KvMemory() {
        if (mem == nullptr) return;
        (void)hipSetDevice(device);
        (void)hipFree(mem);
    }
};

}  // namespace

struct mlq_kv_cache_s {
    std::shared_ptr<KvMemory> kv;
};

struct mlq_kv_plan_s {
    std::shared_ptr<KvMemory> kv;
    mlq::KvPlanShape shape{};
    float scale = 0.0f;
    int n_heads = 0;
    // Lists in device memory, each with room for the largest batch, and the pinned
    // blocks they are uploaded from: one may still be read while the next is filled.
    size_t list_bytes = 0, at[mlq::kKvParts] = {};
    uint8_t* lists = nullptr;
    uint8_t* pinned[2] = {nullptr, nullptr};
    hipEvent_t uploaded[2] = {nullptr, nullptr};
    int turn = 0;
    // Partial results and arrival counters of split work, narrow list then wide.
    float* partial[2] = {nullptr, nullptr};
    unsigned* arrived[2] = {nullptr, nullptr};
    void* work = nullptr;
    // The batch.
    bool set = false;
    int n_tokens = 0, n_positions = 0;
    int counts[mlq::kKvCounts] = {};
    // Turns per position of the last theta.
    float theta = 0.0f;
    mlq::KvRope rope{};

    mlq::KvLists device_lists() const {
        mlq::KvLists l;
        l.counts = reinterpret_cast<const int*>(lists + at[0]);
        l.fresh = reinterpret_cast<const mlq::KvTileItem*>(lists + at[1]);
        l.pages = reinterpret_cast<const mlq::KvPage*>(lists + at[2]);
        l.items[0] = reinterpret_cast<const mlq::KvAttnItem*>(lists + at[3]);
        l.items[1] = reinterpret_cast<const mlq::KvAttnItem*>(lists + at[4]);
        return l;
    }
    mlq::KvView view(int layer) const {
        return mlq::KvView{kv->mem + kv->layer_bytes * layer, kv->qtype, kv->nb, kv->head_dim, kv->n_kv,
                           kv->page_size / mlq::kKvTile};
    }
    ~mlq_kv_plan_s() {
        if (kv) (void)hipSetDevice(kv->device);
        for (int i = 0; i < 2; ++i) {
            if (uploaded[i] != nullptr) {
                (void)hipEventSynchronize(uploaded[i]);
                (void)hipEventDestroy(uploaded[i]);
            }
            if (pinned[i] != nullptr) (void)hipHostFree(pinned[i]);
        }
        if (lists != nullptr) (void)hipFree(lists);
        if (work != nullptr) (void)hipFree(work);
    }
};

namespace {

using mlq::abi_fail;
using mlq::abi_hip_fail;

#define MLQ_KV_HIP(expr)                                              \
    do {                                                              \
        hipError_t mlq_e_ = (expr);                                   \
        if (mlq_e_ != hipSuccess) return abi_hip_fail(mlq_e_, #expr); \
    } while (0)

// Runs a C entry's body: nothing may be thrown across it.
template <typename F>
int entry(const char* caller, F&& body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return abi_fail(MLQ_ERR_LIMIT, std::string(caller) + ": out of host memory");
    } catch (const std::exception& e) {
        return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": " + e.what());
    }
}

// A call's plan, layer and stream.
int check_call(mlq_kv_plan_t p, int layer, const char* caller) {
    if (p == nullptr) return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": null plan");
    if (layer < 0 || layer >= p->kv->n_layers) {
        return abi_fail(MLQ_ERR_SHAPE, std::string(caller) + ": layer " + std::to_string(layer) + " out of " +
                                           std::to_string(p->kv->n_layers));
    }
    if (!p->set) return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": the plan holds no batch");
    return mlq::abi_device(p->kv->device);
}

int check_rows(const void* ptr, mlq_kv_plan_t p, const char* caller, const char* what, int64_t rows, int heads) {
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) {
        return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": " + what + " is not 16-byte aligned");
    }
    return mlq::abi_device_ptr(ptr, p->kv->device, caller, what,
                               static_cast<size_t>(rows) * heads * p->kv->head_dim * sizeof(float));
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

}  // namespace

extern "C" {

int mlq_hip_kv_cache_create(int device, int type, int n_layers, int n_pages, int page_size, int n_kv_heads, int head_dim,
                            mlq_kv_cache_t* out) {
    const char* caller = "hip_kv_cache_create";
    if (out == nullptr) return abi_fail(MLQ_ERR_INVALID, "hip_kv_cache_create: null output handle");
    *out = nullptr;
    return entry(caller, [&]() -> int {
        const std::string who(caller);
        if (type < MLQ_F32 || type > MLQ_Q4_1) {
            return abi_fail(MLQ_ERR_INVALID, who + ": unsupported type " + std::to_string(type));
        }
        if (n_layers <= 0 || n_pages <= 0 || n_kv_heads <= 0 || head_dim <= 0) {
            return abi_fail(MLQ_ERR_SHAPE, who + ": empty caches are not supported");
        }
        if (page_size < mlq::kKvTile || page_size > 65536 || (page_size & (page_size - 1)) != 0) {
            return abi_fail(MLQ_ERR_SHAPE, who + ": page size " + std::to_string(page_size) +
                                               " is not a power of two from 32 to 65536");
        }
        if (head_dim % 8 != 0 || head_dim > mlq::kKvMaxHeadDim) {
            return abi_fail(MLQ_ERR_SHAPE, who + ": head_dim " + std::to_string(head_dim) +
                                               " is not a multiple of 8 up to " + std::to_string(mlq::kKvMaxHeadDim));
        }
        if (n_kv_heads > 65536) return abi_fail(MLQ_ERR_LIMIT, who + ": more than 65536 KV heads");
        auto kv = std::make_shared<KvMemory>();
        kv->device = device, kv->qtype = type, kv->n_layers = n_layers, kv->n_pages = n_pages;
        kv->page_size = page_size, kv->n_kv = n_kv_heads, kv->head_dim = head_dim;
        kv->nb = (head_dim + mlq::kQK - 1) / mlq::kQK;
        if (kv->nb == 5 || kv->nb == 7) ++kv->nb;  // the attention is built for 1, 2, 3, 4, 6 and 8 blocks
        const double bytes = static_cast<double>(mlq::kv_tile_bytes(type, kv->nb)) * (page_size / mlq::kKvTile) * n_kv_heads *
                             static_cast<double>(n_pages) * n_layers;
        if (bytes > 9e15) return abi_fail(MLQ_ERR_LIMIT, who + ": the cache is too large");
        kv->layer_bytes = mlq::kv_tile_bytes(type, kv->nb) * (page_size / mlq::kKvTile) * n_kv_heads * n_pages;
        const int rc = mlq::abi_device(device);
        if (rc != MLQ_OK) return rc;
        const hipStream_t s = mlq::abi_stream(device, nullptr);
        if (mlq::abi_capturing(s)) return abi_fail(MLQ_ERR_INVALID, who + ": not under graph capture");
        void* mem = nullptr;
        MLQ_KV_HIP(hipMalloc(&mem, kv->bytes()));
        kv->mem = static_cast<uint8_t*>(mem);
        // Zeros: a slot that nothing has been written to holds finite values.
        MLQ_KV_HIP(hipMemsetAsync(mem, 0, kv->bytes(), s));
        MLQ_KV_HIP(hipStreamSynchronize(s));
        *out = new mlq_kv_cache_s{std::move(kv)};
        return MLQ_OK;
    });
}

int mlq_hip_kv_cache_info(mlq_kv_cache_t cache, int* type, int* n_layers, int* n_pages, int* page_size, int* n_kv_heads,
                          int* head_dim, size_t* bytes) {
    if (cache == nullptr) return abi_fail(MLQ_ERR_INVALID, "hip_kv_cache_info: null cache");
    const KvMemory& kv = *cache->kv;
    if (type) *type = kv.qtype;
    if (n_layers) *n_layers = kv.n_layers;
    if (n_pages) *n_pages = kv.n_pages;
    if (page_size) *page_size = kv.page_size;
    if (n_kv_heads) *n_kv_heads = kv.n_kv;
    if (head_dim) *head_dim = kv.head_dim;
    if (bytes) *bytes = kv.bytes();
    return MLQ_OK;
}

int mlq_hip_kv_cache_destroy(mlq_kv_cache_t cache) {
    delete cache;
    return MLQ_OK;
}

int mlq_hip_kv_plan_create(mlq_kv_cache_t cache, int n_heads, int window, int sinks, float scale, int max_seqs,
                           int max_tokens, int max_pages, mlq_kv_plan_t* out) {
    const char* caller = "hip_kv_plan_create";
    if (out == nullptr) return abi_fail(MLQ_ERR_INVALID, "hip_kv_plan_create: null output handle");
    *out = nullptr;
    return entry(caller, [&]() -> int {
        const std::string who(caller);
        if (cache == nullptr) return abi_fail(MLQ_ERR_INVALID, who + ": null cache");
        const KvMemory& kv = *cache->kv;
        if (n_heads <= 0 || n_heads % kv.n_kv != 0) {
            return abi_fail(MLQ_ERR_SHAPE, who + ": " + std::to_string(n_heads) + " heads over " + std::to_string(kv.n_kv) +
                                               " KV heads");
        }
        if (window < 0 || sinks < 0) return abi_fail(MLQ_ERR_INVALID, who + ": negative window or sinks");
        if (sinks > 0 && window == 0) return abi_fail(MLQ_ERR_INVALID, who + ": sinks need a window");
        if (!(scale == 0.0f || (std::fabs(scale) >= 0x1p-100f && std::fabs(scale) <= 0x1p100f))) {
            return abi_fail(MLQ_ERR_INVALID, who + ": scale is neither 0 nor of magnitude 2^-100 to 2^100");
        }
        if (max_seqs <= 0 || max_tokens <= 0 || max_pages <= 0) {
            return abi_fail(MLQ_ERR_SHAPE, who + ": empty plans are not supported");
        }
        if (static_cast<int64_t>(max_tokens) * n_heads > kMost || static_cast<int64_t>(max_pages) * kv.page_size > kMost ||
            max_seqs > 1 << 20) {
            return abi_fail(MLQ_ERR_LIMIT, who + ": more than 2^30 token heads or positions, or 2^20 sequences");
        }
        auto p = std::make_unique<mlq_kv_plan_s>();
        p->kv = cache->kv;
        p->n_heads = n_heads;
        p->scale = scale != 0.0f ? scale : static_cast<float>(1.0 / std::sqrt(static_cast<double>(kv.head_dim)));
        p->shape = mlq::KvPlanShape{kv.page_size, kv.n_pages, kv.n_kv, n_heads / kv.n_kv, mlq::kv_wide_rows(kv.nb),
                                    window, sinks, max_seqs, max_tokens, max_pages};
        const mlq::KvPlanLimits lim = mlq::kv_plan_limits(p->shape);
        const size_t sizes[mlq::kKvParts] = {
            mlq::kKvCounts * sizeof(int), static_cast<size_t>(lim.fresh) * sizeof(mlq::KvTileItem),
            static_cast<size_t>(max_pages) * sizeof(mlq::KvPage), static_cast<size_t>(lim.items[0]) * sizeof(mlq::KvAttnItem),
            static_cast<size_t>(lim.items[1]) * sizeof(mlq::KvAttnItem)};
        for (int i = 0; i < mlq::kKvParts; ++i) {
            p->at[i] = p->list_bytes;
            p->list_bytes += (sizes[i] + 255) / 256 * 256;
        }
        const int rc = mlq::abi_device(kv.device);
        if (rc != MLQ_OK) return rc;
        const hipStream_t s = mlq::abi_stream(kv.device, nullptr);
        if (mlq::abi_capturing(s)) return abi_fail(MLQ_ERR_INVALID, who + ": not under graph capture");
        void* mem = nullptr;
        MLQ_KV_HIP(hipMalloc(&mem, p->list_bytes));
        p->lists = static_cast<uint8_t*>(mem);
        for (int i = 0; i < 2; ++i) {
            void* host = nullptr;
            MLQ_KV_HIP(hipHostMalloc(&host, p->list_bytes, hipHostMallocDefault));
            p->pinned[i] = static_cast<uint8_t*>(host);
            MLQ_KV_HIP(hipEventCreateWithFlags(&p->uploaded[i], hipEventDisableTiming));
        }
        size_t floats[2], words[2];
        for (int i = 0; i < 2; ++i) {
            words[i] = (static_cast<size_t>(lim.slots[i]) * kv.n_kv + 63) / 64 * 64;
            floats[i] = static_cast<size_t>(lim.slots[i]) * kv.n_kv * mlq::kv_partial_floats(kv.nb, i);
        }
        MLQ_KV_HIP(hipMalloc(&p->work, (words[0] + words[1] + floats[0] + floats[1]) * 4));
        p->arrived[0] = static_cast<unsigned*>(p->work);
        p->arrived[1] = p->arrived[0] + words[0];
        p->partial[0] = reinterpret_cast<float*>(p->arrived[1] + words[1]);
        p->partial[1] = p->partial[0] + floats[0];
        MLQ_KV_HIP(hipMemsetAsync(p->work, 0, (words[0] + words[1]) * 4, s));
        MLQ_KV_HIP(hipStreamSynchronize(s));
        *out = p.release();
        return MLQ_OK;
    });
}

int mlq_hip_kv_plan_set(mlq_kv_plan_t p, int n_seqs, const int* new_tokens, const int* kv_len, const int* pages,
                        void* stream) {
    const char* caller = "hip_kv_plan_set";
    return entry(caller, [&]() -> int {
        if (p == nullptr) return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": null plan");
        mlq::KvBatch b;
        const std::string wrong = mlq::kv_plan_build(p->shape, n_seqs, new_tokens, kv_len, pages, &b);
        if (!wrong.empty()) return abi_fail(MLQ_ERR_SHAPE, std::string(caller) + ": " + wrong);
        const int rc = mlq::abi_device(p->kv->device);
        if (rc != MLQ_OK) return rc;
        const hipStream_t s = mlq::abi_stream(p->kv->device, stream);
        if (mlq::abi_capturing(s)) {
            return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": a batch cannot be set under graph capture");
        }
        int counts[mlq::kKvCounts];
        counts[mlq::kKvCountFresh] = static_cast<int>(b.fresh.size());
        counts[mlq::kKvCountPages] = static_cast<int>(b.pages.size());
        counts[mlq::kKvCountNarrow] = static_cast<int>(b.items[0].size());
        counts[mlq::kKvCountWide] = static_cast<int>(b.items[1].size());
        const void* from[mlq::kKvParts] = {counts, b.fresh.data(), b.pages.data(), b.items[0].data(), b.items[1].data()};
        const size_t bytes[mlq::kKvParts] = {sizeof counts, b.fresh.size() * sizeof b.fresh[0],
                                             b.pages.size() * sizeof b.pages[0], b.items[0].size() * sizeof b.items[0][0],
                                             b.items[1].size() * sizeof b.items[1][0]};
        const int t = p->turn;
        MLQ_KV_HIP(hipEventSynchronize(p->uploaded[t]));  // the block's last upload (none yet: done)
        mlq::KvParts parts;
        for (int i = 0; i < mlq::kKvParts; ++i) {
            if (p->at[i] + bytes[i] > (i + 1 < mlq::kKvParts ? p->at[i + 1] : p->list_bytes)) {
                return abi_fail(MLQ_ERR_LIMIT, std::string(caller) + ": a work list is longer than the plan holds");
            }
            if (bytes[i] > 0) std::memcpy(p->pinned[t] + p->at[i], from[i], bytes[i]);
            parts.src[i] = reinterpret_cast<const uint32_t*>(p->pinned[t] + p->at[i]);
            parts.dst[i] = reinterpret_cast<uint32_t*>(p->lists + p->at[i]);
            parts.words[i] = static_cast<int>(bytes[i] / 4);
        }
        const hipError_t e = mlq::launch_kv_upload(parts, s);
        if (e != hipSuccess) return abi_hip_fail(e, caller);
        MLQ_KV_HIP(hipEventRecord(p->uploaded[t], s));
        p->turn ^= 1;
        std::copy(counts, counts + mlq::kKvCounts, p->counts);
        p->n_tokens = b.n_tokens;
        p->n_positions = b.n_positions;
        p->set = true;
        return MLQ_OK;
    });
}

int mlq_hip_kv_plan_destroy(mlq_kv_plan_t p) {
    delete p;
    return MLQ_OK;
}

int mlq_hip_kv_write(mlq_kv_plan_t p, int layer, const float* k, const float* v, const float* q, float* q_out, float theta,
                     int neox, void* stream) {
    const char* caller = "hip_kv_write";
    return entry(caller, [&]() -> int {
        int rc = check_call(p, layer, caller);
        if (rc != MLQ_OK) return rc;
        if (!(theta >= 0.0f) || std::isinf(theta)) {
            return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": theta is negative or not finite");
        }
        if ((q == nullptr) != (q_out == nullptr)) {
            return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": q and q_out come together");
        }
        if (q != nullptr && theta == 0.0f) {
            return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": q without a rotation");
        }
        const hipStream_t s = mlq::abi_stream(p->kv->device, stream);
        const bool recorded = mlq::abi_capturing(s);
        const int64_t rows = recorded ? p->shape.max_tokens : p->n_tokens;
        if (rows == 0) return MLQ_OK;
        const int n_kv = p->kv->n_kv;
        if ((rc = check_rows(k, p, caller, "k", rows, n_kv)) != MLQ_OK) return rc;
        if ((rc = check_rows(v, p, caller, "v", rows, n_kv)) != MLQ_OK) return rc;
        if (q != nullptr) {
            if ((rc = check_rows(q, p, caller, "q", rows, p->n_heads)) != MLQ_OK) return rc;
            if ((rc = check_rows(q_out, p, caller, "q_out", rows, p->n_heads)) != MLQ_OK) return rc;
            const size_t nq = static_cast<size_t>(rows) * p->n_heads * p->kv->head_dim * 4;
            const size_t nk = static_cast<size_t>(rows) * n_kv * p->kv->head_dim * 4;
            if ((q_out != q && overlap(q, nq, q_out, nq)) || overlap(k, nk, q_out, nq) || overlap(v, nk, q_out, nq)) {
                return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": q_out overlaps an input");
            }
        }
        if (theta != p->theta) {
            for (int r = 0; 2 * r < p->kv->head_dim; ++r) {
                p->rope.turns[r] = std::pow(static_cast<double>(theta), -2.0 * r / p->kv->head_dim) / (2.0 * M_PI);
            }
            p->theta = theta;
        }
        p->rope.on = theta > 0.0f;
        p->rope.neox = neox != 0;
        const hipError_t e = mlq::launch_kv_write(p->view(layer), p->device_lists(), recorded ? 0 : p->counts[mlq::kKvCountFresh],
                                                  static_cast<int>(rows), k, v, q, q_out, p->n_heads, p->rope, s);
        return e == hipSuccess ? MLQ_OK : abi_hip_fail(e, caller);
    });
}

int mlq_hip_kv_read(mlq_kv_plan_t p, int layer, int new_only, float* k, float* v, void* stream) {
    const char* caller = "hip_kv_read";
    return entry(caller, [&]() -> int {
        int rc = check_call(p, layer, caller);
        if (rc != MLQ_OK) return rc;
        const hipStream_t s = mlq::abi_stream(p->kv->device, stream);
        const bool recorded = mlq::abi_capturing(s);
        const int64_t most = new_only != 0 ? p->shape.max_tokens
                                           : static_cast<int64_t>(p->shape.max_pages) * p->shape.page_size;
        const int64_t rows = recorded ? most : new_only != 0 ? p->n_tokens : p->n_positions;
        if (rows == 0) return MLQ_OK;
        if ((rc = check_rows(k, p, caller, "k", rows, p->kv->n_kv)) != MLQ_OK) return rc;
        if ((rc = check_rows(v, p, caller, "v", rows, p->kv->n_kv)) != MLQ_OK) return rc;
        const size_t bytes = static_cast<size_t>(rows) * p->kv->n_kv * p->kv->head_dim * 4;
        if (overlap(k, bytes, v, bytes)) return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": k overlaps v");
        const int count = p->counts[new_only != 0 ? mlq::kKvCountFresh : mlq::kKvCountPages];
        const hipError_t e = mlq::launch_kv_read(p->view(layer), p->device_lists(), new_only != 0, recorded ? 0 : count, k, v, s);
        return e == hipSuccess ? MLQ_OK : abi_hip_fail(e, caller);
    });
}

int mlq_hip_kv_attention(mlq_kv_plan_t p, int layer, const float* q, float* out, void* stream) {
    const char* caller = "hip_kv_attention";
    return entry(caller, [&]() -> int {
        int rc = check_call(p, layer, caller);
        if (rc != MLQ_OK) return rc;
        const hipStream_t s = mlq::abi_stream(p->kv->device, stream);
        const bool recorded = mlq::abi_capturing(s);
        const int64_t rows = recorded ? p->shape.max_tokens : p->n_tokens;
        if (rows == 0) return MLQ_OK;
        if ((rc = check_rows(q, p, caller, "q", rows, p->n_heads)) != MLQ_OK) return rc;
        if ((rc = check_rows(out, p, caller, "out", rows, p->n_heads)) != MLQ_OK) return rc;
        const size_t bytes = static_cast<size_t>(rows) * p->n_heads * p->kv->head_dim * 4;
        if (overlap(q, bytes, out, bytes)) return abi_fail(MLQ_ERR_INVALID, std::string(caller) + ": out overlaps q");
        for (int kind = 0; kind < 2; ++kind) {
            const int count = p->counts[mlq::kKvCountNarrow + kind];
            if (count == 0 && !recorded) continue;
            const mlq::KvAttention a{p->view(layer), p->device_lists(), p->shape.group, p->shape.window, p->shape.sinks,
                                     static_cast<float>(p->scale * 1.4426950408889634), p->partial[kind], p->arrived[kind]};
            const hipError_t e = mlq::launch_kv_attention(a, kind, recorded ? 0 : count, q, out, s);
            if (e != hipSuccess) return abi_hip_fail(e, caller);
        }
        return MLQ_OK;
    });
}

}  // extern "C"
