// Attention over pages of Q4_0 keys and values (kv_attention.h, kv_attention_rows.h).

#include "kv_attention_rows.h"

namespace mlq {

hipError_t launch_kv_attention_q4_0(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    return kv::launch<2>(a, kind, count, q, out, s);
}

}  // namespace mlq
