// How the paged key/value cache lies in memory, and what its kernels are launched with.
//
// [layer][page][KV head][tile of the page], a tile holding 32 positions of one
// head: keys, their scales, values, their scales.  Codes lie as the MFMA operands
// of the attention read them, so its waves load them from memory straight into
// registers, 16 bytes a lane where the width allows, with no transposition:
//
//   keys    A operand of S^T = K Q^T (v_mfma_f32_16x16x32_f16), one block of 32
//           elements its depth: lane i + 16 g of half kt holds key 16 kt + i,
//           elements 8 g .. 8 g + 7 of every block;
//   values  A operand of O^T = V^T P^T, the tile's 32 keys its depth: lane i + 16 g
//           holds dimensions i and 16 + i of every block, keys 4 g .. 4 g + 3 and
//           16 + 4 g .. 16 + 4 g + 3 -- the keys whose scores the lane has in S^T.
//
// A lane's bytes are cut into units of 16 (8, 4 where they are no multiple) and
// unit u of all lanes lies together.  Q8_0 codes are stored plus 128, two 4-bit
// codes share a byte (keys: elements j and 4 + j of the lane's eight; values:
// dimensions i and 16 + i).  Scales are binary16 (Q4_1: scales, then minima), in
// the order of the lanes that use them.  F32 elements are stored as they are; per
// block there is a power of two (f32) that brings them into fp16's range, Inf
// where a block holds something that is not finite or reaches 2^80.
#pragma once

#include "kv_plan.h"
#include "mlq_kernels.h"

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace mlq {

constexpr int kKvMaxHeadDim = 256;

// Sizes of a tile of heads of nb blocks, in bytes.
template <int QT>
struct KvForm {
    static constexpr int kElemBits = QT == 0 ? 32 : QT == 1 ? 8 : 4;
    static constexpr int kPlanes = QT == 3 ? 2 : 1;           // scale planes
    static constexpr int kScaleBytes = QT == 0 ? 4 : 2;
    static constexpr int kBlockBytes = kKvTile * 4 * kElemBits;  // codes of a block of all positions (32 x 32 elements)
    __host__ __device__ static constexpr int codes(int nb) { return nb * kBlockBytes; }
    __host__ __device__ static constexpr int plane(int nb) { return nb * kKvTile * kScaleBytes; }
    __host__ __device__ static constexpr int half(int nb) { return codes(nb) + kPlanes * plane(nb); }  // keys or values
    __host__ __device__ static constexpr int tile(int nb) { return 2 * half(nb); }
    // A lane's bytes of one half tile of keys / of the values, and their unit.
    __host__ __device__ static constexpr int key_lane(int nb) { return nb * kElemBits; }
    __host__ __device__ static constexpr int value_lane(int nb) { return nb * 2 * kElemBits; }
    __host__ __device__ static constexpr int unit(int lane_bytes) {
        return lane_bytes % 16 == 0 ? 16 : lane_bytes % 8 == 0 ? 8 : 4;
    }
    // Byte x of lane `lane`.
    __host__ __device__ static constexpr int at(int lane_bytes, int lane, int x) {
        const int u = unit(lane_bytes);
        return x / u * 64 * u + lane * u + x % u;
    }
    // Index of the scale of (key, block b) in its plane.
    __host__ __device__ static constexpr int key_scale(int nb, int key, int b) {
        return ((key >> 2) * nb + b) * 4 + (key & 3);  // [kt][g][b][4 keys]
    }
    __host__ __device__ static constexpr int value_scale(int nb, int key, int b) {
        return (((key & 15) >> 2) * nb + b) * 8 + (key >> 4) * 4 + (key & 3);  // [g][b][8 keys]
    }
};

inline size_t kv_tile_bytes(int qtype, int nb) {
    switch (qtype) {
        case 0: return KvForm<0>::tile(nb);
        case 1: return KvForm<1>::tile(nb);
        case 2: return KvForm<2>::tile(nb);
        default: return KvForm<3>::tile(nb);
    }
}

// One layer of a cache.
struct KvView {
    uint8_t* base;
    int qtype, nb, head_dim, n_kv, page_tiles;  // tiles per page: a power of two
};

// The lists of a plan in device memory.
struct KvLists {
    const int* counts;  // kKvCount*
    const KvTileItem* fresh;
    const KvPage* pages;
    const KvAttnItem* items[2];
};
enum { kKvCountFresh, kKvCountPages, kKvCountNarrow, kKvCountWide, kKvCounts };

// RoPE of a write: turns per position of pair r, and how elements pair.
struct KvRope {
    double turns[kKvMaxHeadDim / 2];
    int on, neox;
};

// Copies `n` parts of pinned host memory to the lists (one launch, any stream).
constexpr int kKvParts = 5;
struct KvParts {
    const uint32_t* src[kKvParts];
    uint32_t* dst[kKvParts];
    int words[kKvParts];
};
hipError_t launch_kv_upload(const KvParts& parts, hipStream_t s);

// `count`: the items of the list in use (0: as many as the device says, for launches
// that are recorded and replayed with other lists); `tokens`: new tokens of the batch.
hipError_t launch_kv_write(const KvView& kv, const KvLists& lists, int count, int tokens, const float* k, const float* v,
                           const float* q, float* q_out, int n_heads, const KvRope& rope, hipStream_t s);
hipError_t launch_kv_read(const KvView& kv, const KvLists& lists, bool fresh, int count, float* k, float* v, hipStream_t s);

struct KvAttention {
    KvView kv;
    KvLists lists;
    int group;          // query heads per KV head
    int window, sinks;
    float scale;        // of the scores, times log2(e)
    float* partial;     // [slot][KV head][kv_partial_floats]
    unsigned* arrived;  // [first slot of a split][KV head], zero between launches
};
// Query rows of a workgroup of the kernel for many rows, and a part's floats in `partial` by list (0 narrow, 1 wide).
int kv_wide_rows(int nb);
size_t kv_partial_floats(int nb, int kind);
// count: items of the narrow (kind 0) or wide list, 0 as above.
hipError_t launch_kv_attention(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);

}  // namespace mlq
