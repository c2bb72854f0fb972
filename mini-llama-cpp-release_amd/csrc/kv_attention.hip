// Attention of a batch's new tokens over the paged cache (kv_layout.h), straight from
// the formulas: out = softmax_j(scale q . k_j) v over the positions j that a token
// at position i sees, j <= i and, with a window of w, j > i - w or j < sinks.  A
// workgroup takes the rows of one item one after the other, 256 positions at a time
// (a thread a score, then a thread an output element) with a running maximum and sum.
// Each element is decoded where it is used: 34 GFLOP of a 2048-token prompt, 32
// heads of 128, take tens of milliseconds.

#include "kv_device.h"
#include "kv_layout.h"

#include <algorithm>
#include <cmath>

namespace mlq {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float fold(float v, bool max, float* part) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float u = __shfl_xor(v, o, 64);
        v = max ? fmaxf(v, u) : v + u;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return max ? fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) : part[0] + part[1] + part[2] + part[3];
}

// An element as the attention takes it: NaN in a block marked as not finite.
template <int QT>
__device__ __forceinline__ float element(const uint8_t* tile, int nb, bool values, int key, int e) {
    using F = KvForm<QT>;
    const float y = kv_element<QT>(tile, nb, values, key, e);
    if (QT != 0) return y;
    const float* scale = reinterpret_cast<const float*>(tile + (values ? F::half(nb) : 0) + F::codes(nb));
    return scale[values ? F::value_scale(nb, key, e >> 5) : F::key_scale(nb, key, e >> 5)] == INFINITY ? NAN : y;
}

template <int QT>
__global__ __launch_bounds__(kThreads) void kv_attention_kernel(KvAttention a, int kind, int count, int rows_per_wave,
                                                                const float* __restrict__ q, float* __restrict__ out) {
    __shared__ float qs[kKvMaxHeadDim], ps[kThreads], part[4];
    const int hd = a.kv.head_dim, nb = a.kv.nb, heads = a.kv.n_kv * a.group;
    const int tile_bytes = KvForm<QT>::tile(nb);
    const int total = (count > 0 ? count : a.lists.counts[kKvCountNarrow + kind]) * a.kv.n_kv;
    for (int w = blockIdx.x; w < total; w += gridDim.x) {
        const KvAttnItem it = a.lists.items[kind][w / a.kv.n_kv];
        const int head = w % a.kv.n_kv;
        if (it.split != 0) continue;
        const int rows = min(it.new_tokens * a.group, it.row0 + rows_per_wave * (it.stride == 1 ? kKvWaves : 1));
        for (int r = it.row0; r < rows; ++r) {
            const int token = r / a.group, pos = it.len - it.new_tokens + token;
            const size_t row = (static_cast<size_t>(it.token0 + token) * heads + head * a.group + r % a.group) * hd;
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < hd) qs[threadIdx.x] = q[row + threadIdx.x];
            float m = -INFINITY, l = 0.0f, o = 0.0f;
            for (int j0 = 0; j0 <= pos; j0 += kThreads) {
                __syncthreads();
                const int j = j0 + threadIdx.x;
                float t = -INFINITY;
                if (j <= pos && (a.window == 0 || j > pos - a.window || j < a.sinks)) {
                    const int page = a.lists.pages[it.page0 + j / (a.kv.page_tiles * kKvTile)].page;
                    const uint8_t* tile = a.kv.base + ((static_cast<size_t>(page) * a.kv.n_kv + head) * a.kv.page_tiles +
                                                       j / kKvTile % a.kv.page_tiles) * tile_bytes;
                    float s = 0.0f;
                    for (int e = 0; e < hd; ++e) s += qs[e] * element<QT>(tile, nb, false, j % kKvTile, e);
                    t = s * a.scale;
                }
                const float top = fmaxf(m, fold(t, true, part));
                const float base = top == -INFINITY ? 0.0f : top;
                const float p = exp2f(t - base), old = exp2f(m - base);
                ps[threadIdx.x] = p;
                l = l * old + fold(p, false, part);
                o *= old;
                m = top;
                if (static_cast<int>(threadIdx.x) < hd) {
                    for (int i = 0; i < min(kThreads, pos + 1 - j0); ++i) {
                        if (ps[i] == 0.0f) continue;
                        const int page = a.lists.pages[it.page0 + (j0 + i) / (a.kv.page_tiles * kKvTile)].page;
                        const uint8_t* tile = a.kv.base + ((static_cast<size_t>(page) * a.kv.n_kv + head) * a.kv.page_tiles +
                                                           (j0 + i) / kKvTile % a.kv.page_tiles) * tile_bytes;
                        o += ps[i] * element<QT>(tile, nb, true, (j0 + i) % kKvTile, threadIdx.x);
                    }
                }
            }
            if (static_cast<int>(threadIdx.x) < hd) out[row + threadIdx.x] = o / l;
        }
    }
}

template <int QT>
hipError_t launch(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    const unsigned grid = count > 0 ? static_cast<unsigned>(count) * a.kv.n_kv : 1024u;
    kv_attention_kernel<QT><<<grid, kThreads, 0, s>>>(a, kind, count, kind == 0 ? kKvNarrowRows : kv_wide_rows(a.kv.nb), q, out);
    return hipGetLastError();
}

}  // namespace

int kv_wide_rows(int nb) { return nb <= 4 ? 32 : 16; }

size_t kv_partial_floats(int nb, int kind) { return static_cast<size_t>(kind == 0 ? 1 : kv_wide_rows(nb) / 16) * 64 * (8 * nb + 2); }

hipError_t launch_kv_attention(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    switch (a.kv.qtype) {
        case 0: return launch<0>(a, kind, count, q, out, s);
        case 1: return launch<1>(a, kind, count, q, out, s);
        case 2: return launch<2>(a, kind, count, q, out, s);
        case 3: return launch<3>(a, kind, count, q, out, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mlq
