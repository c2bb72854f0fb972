// Positions and pages of the paged key/value cache moved within it, in every layer at once
// (kv_layout.h says how a tile lies in memory).  The lists travel as launch arguments: no upload, and no
// memory that a later call could overwrite.

#include "kv_layout.h"

#include <algorithm>

namespace mlq {
namespace {

constexpr int kThreads = 256;
constexpr int kCopies = 360, kMoves = 240;  // of a launch: its arguments stay below 4 KB
constexpr int kTogether = 8;                // moves of a path that are read before one is written

struct CopyArgs {
    int from[kCopies], to[kCopies];
    uint16_t tiles[kCopies];
};
struct MoveArgs {
    KvMove move[kMoves];
    uint16_t end[kMoves];  // of each path, in moves
};

// Bound: memory.  A workgroup copies the tiles of one page, head and layer, which lie together (256 pages of 64 positions,
// 8 KV heads of 128 in Q8_0, 4 layers: 75 us, 3.8 TB/s read and written; three pages of a small model 5 us).  Eight
// 16-byte loads in flight a thread are no faster than four.
__global__ __launch_bounds__(kThreads) void kv_copy_kernel(KvView kv, int n_layers, size_t layer_bytes, int tile_bytes, CopyArgs args,
                                                           int n) {
    const long long total = static_cast<long long>(n) * n_layers * kv.n_kv;
    for (long long w = blockIdx.x; w < total; w += gridDim.x) {
        const int head = static_cast<int>(w % kv.n_kv);
        const long long rest = w / kv.n_kv;
        const int i_copy = static_cast<int>(rest % n);
        const KvCopy c{args.from[i_copy], args.to[i_copy], args.tiles[i_copy]};
        uint8_t* const layer = kv.base + layer_bytes * (rest / n);
        const size_t page_bytes = static_cast<size_t>(kv.page_tiles) * tile_bytes;
        const uint4* const from = reinterpret_cast<const uint4*>(layer + (static_cast<size_t>(c.from) * kv.n_kv + head) * page_bytes);
        uint4* const to = reinterpret_cast<uint4*>(layer + (static_cast<size_t>(c.to) * kv.n_kv + head) * page_bytes);
        const int units = c.tiles * (tile_bytes / 16);
        int i = threadIdx.x;
        for (; i + 3 * kThreads < units; i += 4 * kThreads) {
            uint4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = from[i + k * kThreads];
#pragma unroll
            for (int k = 0; k < 4; ++k) to[i + k * kThreads] = x[k];
        }
        for (; i < units; i += kThreads) to[i] = from[i];
    }
}

// The pieces of one slot in its tile, in the order of `piece`: keys (eight elements each), their scales, values (an
// element, or the byte of two), their scales.  Every piece is the slot's alone.
template <int QT>
struct Slot {
    using F = KvForm<QT>;
    int nb;
    __device__ int keys() const { return 4 * nb; }
    __device__ int values() const { return (QT >= 2 ? 16 : 32) * nb; }
    __device__ int scales() const { return F::kPlanes * nb; }
    __device__ int pieces() const { return keys() + values() + 2 * scales(); }
    static constexpr int kPiece = QT == 0 ? 32 : QT == 1 ? 8 : 4;  // bytes of the largest piece

    // Offset and bytes of piece i.
    __device__ int at(int slot, int i, int* bytes) const {
        if (i < keys()) {
            const int b = i >> 2, g = i & 3, lb = F::key_lane(nb);
            *bytes = kPiece;
            return (slot >> 4) * 64 * lb + F::at(lb, 16 * g + (slot & 15), b * F::kElemBits);
        }
        i -= keys();
        if (i < values()) {
            const int lb = F::value_lane(nb), per = QT >= 2 ? 16 : 32, b = i / per, d = i % per;
            const int j = (slot >> 4) * 4 + (slot & 3), lane = 16 * ((slot & 15) >> 2) + (d & 15);
            *bytes = QT == 0 ? 4 : 1;
            const int x = QT == 0 ? b * 64 + (d >> 4) * 32 + j * 4 : QT == 1 ? b * 16 + (d >> 4) * 8 + j : b * 8 + j;
            return F::half(nb) + F::at(lb, lane, x);
        }
        i -= values();
        const bool of_values = i >= scales();
        if (of_values) i -= scales();
        const int plane = i / nb, b = i % nb;
        *bytes = F::kScaleBytes;
        return (of_values ? F::half(nb) : 0) + F::codes(nb) + plane * F::plane(nb) +
               (of_values ? F::value_scale(nb, slot, b) : F::key_scale(nb, slot, b)) * F::kScaleBytes;
    }
};

__device__ __forceinline__ void move_piece(uint8_t* to, const uint8_t* from, int bytes) {
    switch (bytes) {
        case 1: *to = *from; break;
        case 2: *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from); break;
        case 4: *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from); break;
        case 8: *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from); break;
        default: break;
    }
}

// Bound: the lines of memory that a slot's pieces lie in, some ten of 128 bytes for the 150 bytes of a Q4_0 head of 128,
// read and written back (paths of four nodes of 64 sequences, 16 layers, 8 heads: 19 us); few paths by latency (4 us).
// A path a wave, without barriers, takes 17 and 6, pieces in registers 27, a move by whole waves 22 (its addresses are
// then the waves', not the lanes').  A workgroup takes one path in one head and layer: reads up to kTogether slots into
// LDS, then writes them where they go, piece by piece, so that what else lies in their tiles is never rewritten.  A
// path's sources ascend and lie at or behind their destinations: none is one of an earlier move, so it is read before
// anything has been written there.
template <int QT>
__global__ __launch_bounds__(kThreads) void kv_moves_kernel(KvView kv, int n_layers, size_t layer_bytes, MoveArgs args, int n_ends) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    using F = KvForm<QT>;
    const Slot<QT> form{kv.nb};
    const int pieces = form.pieces();
    constexpr int kPiece = Slot<QT>::kPiece;
    const long long total = static_cast<long long>(n_ends) * n_layers * kv.n_kv;
    for (long long w = blockIdx.x; w < total; w += gridDim.x) {
        const int head = static_cast<int>(w % kv.n_kv);
        const long long rest = w / kv.n_kv;
        const int path = static_cast<int>(rest % n_ends);
        uint8_t* const layer = kv.base + layer_bytes * (rest / n_ends);
        auto tile_of = [&](int page, int slot) {
            return layer + ((static_cast<size_t>(page) * kv.n_kv + head) * kv.page_tiles + slot / kKvTile) * F::tile(kv.nb);
        };
        const int end = args.end[path];
        for (int m0 = path > 0 ? args.end[path - 1] : 0; m0 < end; m0 += kTogether) {
            const int tasks = min(kTogether, end - m0) * pieces;
            __syncthreads();  // the last ones' readers are done
            for (int t = threadIdx.x; t < tasks; t += kThreads) {
                const KvMove m = args.move[m0 + t / pieces];
                int bytes;
                const int off = form.at(m.from_slot % kKvTile, t % pieces, &bytes);
                const uint8_t* const from = tile_of(m.from_page, m.from_slot) + off;
                if (QT == 0 && bytes == 32) {  // elements 0 .. 3 and 4 .. 7 lie in units of their own
                    *reinterpret_cast<uint4*>(lds + t * kPiece) = *reinterpret_cast<const uint4*>(from);
                    *reinterpret_cast<uint4*>(lds + t * kPiece + 16) = *reinterpret_cast<const uint4*>(from + 1024);
                } else {
                    move_piece(lds + t * kPiece, from, bytes);
                }
            }
            __syncthreads();
            for (int t = threadIdx.x; t < tasks; t += kThreads) {
                const KvMove m = args.move[m0 + t / pieces];
                int bytes;
                const int off = form.at(m.to_slot % kKvTile, t % pieces, &bytes);
                uint8_t* const to = tile_of(m.to_page, m.to_slot) + off;
                if (QT == 0 && bytes == 32) {
                    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(lds + t * kPiece);
                    *reinterpret_cast<uint4*>(to + 1024) = *reinterpret_cast<const uint4*>(lds + t * kPiece + 16);
                } else {
                    move_piece(to, lds + t * kPiece, bytes);
                }
            }
        }
    }
}

template <int QT>
hipError_t moves(const KvView& kv, int n_layers, size_t layer_bytes, const MoveArgs& args, int n_ends, hipStream_t s) {
    const int pieces = (4 + (QT >= 2 ? 16 : 32) + 2 * KvForm<QT>::kPlanes) * kv.nb;
    const int lds = kTogether * pieces * Slot<QT>::kPiece;
    if (lds > 64 << 10) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kv_moves_kernel<QT>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    const long long groups = static_cast<long long>(n_ends) * n_layers * kv.n_kv;
    kv_moves_kernel<QT><<<static_cast<unsigned>(std::min<long long>(groups, 1 << 20)), kThreads, lds, s>>>(kv, n_layers, layer_bytes,
                                                                                                          args, n_ends);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_copy(const KvView& kv, int n_layers, size_t layer_bytes, const KvCopy* copies, int n, hipStream_t s) {
    const int tile_bytes = static_cast<int>(kv_tile_bytes(kv.qtype, kv.nb));
    for (int at = 0; at < n; at += kCopies) {
        CopyArgs args;
        const int now = std::min(kCopies, n - at);
        for (int i = 0; i < now; ++i) {
            args.from[i] = copies[at + i].from;
            args.to[i] = copies[at + i].to;
            args.tiles[i] = static_cast<uint16_t>(copies[at + i].tiles);
        }
        const long long groups = static_cast<long long>(now) * n_layers * kv.n_kv;
        kv_copy_kernel<<<static_cast<unsigned>(std::min<long long>(groups, 1 << 20)), kThreads, 0, s>>>(kv, n_layers, layer_bytes,
                                                                                                      tile_bytes, args, now);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_kv_moves(const KvView& kv, int n_layers, size_t layer_bytes, const KvMove* list, const int* ends, int n_ends,
                           hipStream_t s) {
    const int n = n_ends > 0 ? ends[n_ends - 1] : 0;
    int path = 0;
    for (int at = 0; at < n;) {
        // (a path may be cut anywhere: its launches follow each other)
        MoveArgs args;
        const int now = std::min(kMoves, n - at);
        std::copy(list + at, list + at + now, args.move);
        int paths = 0;
        for (; path < n_ends && ends[path] <= at + now; ++path) args.end[paths++] = static_cast<uint16_t>(ends[path] - at);
        if (paths == 0 || args.end[paths - 1] < now) args.end[paths++] = static_cast<uint16_t>(now);
        hipError_t e = hipErrorInvalidValue;
        switch (kv.qtype) {
            case 0: e = moves<0>(kv, n_layers, layer_bytes, args, paths, s); break;
            case 1: e = moves<1>(kv, n_layers, layer_bytes, args, paths, s); break;
            case 2: e = moves<2>(kv, n_layers, layer_bytes, args, paths, s); break;
            case 3: e = moves<3>(kv, n_layers, layer_bytes, args, paths, s); break;
            default: break;
        }
        if (e != hipSuccess) return e;
        at += now;
    }
    return hipSuccess;
}

}  // namespace mlq
