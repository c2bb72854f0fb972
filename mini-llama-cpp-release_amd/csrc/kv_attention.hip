// Attention over the paged cache: which type's kernels a call runs (kv_attention.h).

#include "kv_layout.h"

namespace mlq {

// One translation unit a type.
hipError_t launch_kv_attention_f32(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_attention_q8_0(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_attention_q4_0(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_attention_q4_1(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);

hipError_t launch_kv_tree_attention_f32(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_tree_attention_q8_0(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_tree_attention_q4_0(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_tree_attention_q4_1(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);

size_t kv_partial_floats(int nb, int kind) {
    return static_cast<size_t>(kind == 0 ? 1 : kv_wide_rows(nb) / 16) * 64 * (8 * nb + 2);
}

hipError_t launch_kv_attention(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    switch (a.kv.qtype) {
        case 0: return launch_kv_attention_f32(a, kind, count, q, out, s);
        case 1: return launch_kv_attention_q8_0(a, kind, count, q, out, s);
        case 2: return launch_kv_attention_q4_0(a, kind, count, q, out, s);
        case 3: return launch_kv_attention_q4_1(a, kind, count, q, out, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_kv_tree_attention(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    switch (a.kv.qtype) {
        case 0: return launch_kv_tree_attention_f32(a, kind, count, q, out, s);
        case 1: return launch_kv_tree_attention_q8_0(a, kind, count, q, out, s);
        case 2: return launch_kv_tree_attention_q4_0(a, kind, count, q, out, s);
        case 3: return launch_kv_tree_attention_q4_1(a, kind, count, q, out, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mlq
