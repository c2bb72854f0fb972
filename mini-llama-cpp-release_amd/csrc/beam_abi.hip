// C entry points of the beam selection (declared in include/mlq_hip.h).

#include "abi.h"
#include "beam.h"

#include "../../include/mlq_hip.h"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <memory>
#include <new>
#include <string>

struct mlq_beam_s {
    int device = 0, max_groups = 0, max_beams = 0, max_vocab = 0, max_keep = 0;
    void* work = nullptr;

    ~mlq_beam_s() {
        if (work == nullptr) return;
        (void)hipSetDevice(device);
        (void)hipFree(work);
    }
};

namespace {

using mlq::abi_fail;
using mlq::abi_hip_fail;

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

size_t part_count(const mlq_beam_s& h) {
    return mlq::beam_parts(static_cast<long long>(h.max_groups) * h.max_beams, h.max_vocab);
}

struct Buffer {
    const void* ptr;
    const char* what;
    size_t words;
};

}  // namespace

extern "C" {

int mlq_hip_beam_create(int device, int max_groups, int max_beams, int max_vocab, int max_keep, mlq_beam_t* out) {
    const char* caller = "hip_beam_create";
    if (out == nullptr) return abi_fail(MLQ_ERR_INVALID, "hip_beam_create: null output handle");
    *out = nullptr;
    return entry(caller, [&]() -> int {
        const std::string who(caller);
        if (max_groups <= 0 || max_beams <= 0 || max_vocab <= 0 || max_keep <= 0) {
            return abi_fail(MLQ_ERR_SHAPE, who + ": empty searches are not supported");
        }
        if (max_beams > mlq::kBeamMostBeams || max_keep > mlq::kBeamMostKeep) {
            return abi_fail(MLQ_ERR_LIMIT, who + ": more than 64 beams of a group, or 64 continuations");
        }
        if (max_vocab > mlq::kBeamMostVocab) return abi_fail(MLQ_ERR_LIMIT, who + ": more than 2^30 tokens");
        auto h = std::make_unique<mlq_beam_s>();
        h->device = device, h->max_groups = max_groups, h->max_beams = max_beams, h->max_vocab = max_vocab, h->max_keep = max_keep;
        if (static_cast<double>(max_groups) * max_beams * (max_vocab / mlq::kBeamPart + 1) > 0x1p28) {
            return abi_fail(MLQ_ERR_LIMIT, who + ": more than 2^28 parts of rows of logits");
        }
        const int rc = mlq::abi_device(device);
        if (rc != MLQ_OK) return rc;
        if (mlq::abi_capturing(mlq::abi_stream(device, nullptr))) {
            return abi_fail(MLQ_ERR_INVALID, who + ": not under graph capture");
        }
        const hipError_t e = hipMalloc(&h->work, part_count(*h) * (sizeof(mlq::BeamPart) + sizeof(unsigned long long) * max_keep));
        if (e != hipSuccess) return abi_hip_fail(e, caller);
        *out = h.release();
        return MLQ_OK;
    });
}

int mlq_hip_beam_destroy(mlq_beam_t h) {
    delete h;
    return MLQ_OK;
}

int mlq_hip_beam_select(mlq_beam_t h, const float* logits, const float* scores, const int32_t* ended, int end_token, int groups,
                        int beams, int vocab, int keep, int32_t* parents, int32_t* tokens, float* out_scores, void* stream) {
    const char* caller = "hip_beam_select";
    return entry(caller, [&]() -> int {
        const std::string who(caller);
        if (h == nullptr) return abi_fail(MLQ_ERR_INVALID, who + ": null handle");
        if (groups < 0 || beams <= 0 || vocab <= 0 || keep <= 0 || groups > h->max_groups || beams > h->max_beams ||
            vocab > h->max_vocab || keep > h->max_keep) {
            return abi_fail(MLQ_ERR_SHAPE, who + ": " + std::to_string(groups) + " groups, " + std::to_string(beams) + " beams, " +
                                               std::to_string(vocab) + " tokens, " + std::to_string(keep) +
                                               " continuations, the handle holds " + std::to_string(h->max_groups) + ", " +
                                               std::to_string(h->max_beams) + ", " + std::to_string(h->max_vocab) + ", " +
                                               std::to_string(h->max_keep));
        }
        if (ended != nullptr && (end_token < 0 || end_token >= vocab)) {
            return abi_fail(MLQ_ERR_SHAPE, who + ": end token " + std::to_string(end_token) + " of " + std::to_string(vocab));
        }
        int rc = mlq::abi_device(h->device);
        if (rc != MLQ_OK || groups == 0) return rc;
        const size_t rows = static_cast<size_t>(groups) * beams, found = static_cast<size_t>(groups) * keep;
        const Buffer all[6] = {{logits, "logits", rows * vocab}, {scores, "scores", rows},  {ended, "ended", ended != nullptr ? rows : 0},
                               {parents, "parents", found},      {tokens, "tokens", found}, {out_scores, "out_scores", found}};
        for (int i = 0; i < 6; ++i) {
            const Buffer& b = all[i];
            if (b.words == 0) continue;
            if (reinterpret_cast<uintptr_t>(b.ptr) % 4 != 0) {
                return abi_fail(MLQ_ERR_INVALID, who + ": " + b.what + " is not 4-byte aligned");
            }
            if ((rc = mlq::abi_device_ptr(b.ptr, h->device, caller, b.what, b.words * 4)) != MLQ_OK) return rc;
            for (int j = 0; i >= 3 && j < i; ++j) {
                const uintptr_t x = reinterpret_cast<uintptr_t>(b.ptr), y = reinterpret_cast<uintptr_t>(all[j].ptr);
                if (x < y + all[j].words * 4 && y < x + b.words * 4) {
                    return abi_fail(MLQ_ERR_INVALID, who + ": " + b.what + " overlaps " + all[j].what);
                }
            }
        }
        const size_t parts = part_count(*h);
        const mlq::BeamCall c{logits, scores, ended, end_token, groups, beams, vocab, keep, parents, tokens, out_scores,
                              static_cast<mlq::BeamPart*>(h->work),
                              reinterpret_cast<unsigned long long*>(static_cast<mlq::BeamPart*>(h->work) + parts)};
        const hipError_t e = mlq::launch_beam_select(c, mlq::abi_stream(h->device, stream));
        return e == hipSuccess ? MLQ_OK : abi_hip_fail(e, caller);
    });
}

}  // extern "C"
