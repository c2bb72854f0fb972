// Attention of drafted trees over pages of Q4_1 keys and values (kv_attention_tree.h).

#include "kv_attention_tree.h"

namespace mlq {

hipError_t launch_kv_tree_attention_q4_1(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    return kv::launch_tree<3>(a, kind, count, q, out, s);
}

}  // namespace mlq
