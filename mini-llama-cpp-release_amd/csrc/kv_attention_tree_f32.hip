// Attention of drafted trees over pages of f32 keys and values (kv_attention_tree.h).

#include "kv_attention_tree.h"

namespace mlq {

hipError_t launch_kv_tree_attention_f32(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    return kv::launch_tree<0>(a, kind, count, q, out, s);
}

}  // namespace mlq
