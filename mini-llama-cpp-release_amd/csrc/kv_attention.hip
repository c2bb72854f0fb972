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

int kv_wide_rows(int nb) { return nb <= 4 ? 128 : 64; }

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

// Measured, us by the kernel for few rows and the one for many (8 KV heads of 128, rows a KV head and sequence x
// sequences x positions): Q8_0 64 x 1 x 4000 17 and 45, 256 x 1 x 4000 31 and 49, 32 x 32 x 2000 48 and 121, 96 x 16 x 3000
// 106 and 105, 256 x 16 x 2000 182 and 127; Q4_1 96 x 16 x 3000 134 and 113; f32 128 x 4 x 3000 93 and 62, 256 x 16 x 2000
// 446 and 171.  Per tile that is about as much a block of 32 elements.
KvTreeCost kv_tree_cost(int qtype, int nb) {
    constexpr float kFew[4] = {0.74f, 0.33f, 0.32f, 0.40f}, kMany[4] = {2.0f, 1.3f, 1.25f, 1.5f};
    // Above 128 elements (f32: 64) a SIMD has one wave of the kernel for few rows, so more workgroups than CUs are two rounds:
    // 4 x 8 nodes after 1500 positions of f32, 32 heads over 8 of 128, in 512 33 us, in 256 24; 16 after 4000 of Q4_1 of
    // 192 elements 41 and 32.  (A workgroup of the other has half the rows above 128.)
    return KvTreeCost{kFew[qtype] * nb * (nb > 4 ? 1.3f : 1.0f), kMany[qtype] * nb, 14000.0f + 4000.0f * nb,
                      nb > (qtype == 0 ? 2 : 4) ? 256 : 512};
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
