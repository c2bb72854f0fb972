// Paged key/value cache: new tokens quantized into their pages (with the rotary
// embedding of keys and queries), and positions read back as f32.  kv_layout.h says
// how a tile lies in memory, kv_plan.h how the work lists come about.
//
// Scales and codes are those of quantize.hip's kernels bit for bit: the same f32
// steps, none of them contracted.  The rotation is in 64 bits and rounded to f32
// once, angles reduced to a fraction of a turn first, so a far position's angle
// costs no digits and a code next to a border falls as the definition says.

#include "kv_layout.h"
#include "quant_device.h"

#include <algorithm>

namespace mlq {
namespace {

constexpr int kWriteThreads = 512;  // at the most
constexpr int kReadThreads = 256;
constexpr int kRecordedGroups = 1024;  // workgroups of a recorded launch: four a CU

__global__ __launch_bounds__(256) void kv_upload_kernel(KvParts p) {
    for (int k = 0; k < kKvParts; ++k) {
        for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < p.words[k]; i += gridDim.x * blockDim.x) {
            p.dst[k][i] = p.src[k][i];
        }
    }
}

// Where the codes and scales of one tile go: the tile's image in LDS, or its memory.
template <int QT>
struct TileOut {
    uint8_t* p;
    int nb;

    // A lane's eight codes of (key, block b, elements 8 g ..).
    __device__ void key(int slot, int b, int g, const float* y, const int* code) const {
        using F = KvForm<QT>;
        const int lb = F::key_lane(nb);
        uint8_t* half = p + (slot >> 4) * 64 * lb;
        const int lane = 16 * g + (slot & 15);
        if (QT == 0) {
            float4* o = reinterpret_cast<float4*>(half + F::at(lb, lane, b * 32));
            o[0] = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4*>(half + F::at(lb, lane, b * 32 + 16)) = make_float4(y[4], y[5], y[6], y[7]);
        } else if (QT == 1) {
            uint32_t w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[h] = static_cast<uint32_t>(code[4 * h]) | static_cast<uint32_t>(code[4 * h + 1]) << 8 |
                       static_cast<uint32_t>(code[4 * h + 2]) << 16 | static_cast<uint32_t>(code[4 * h + 3]) << 24;
            }
            *reinterpret_cast<uint2*>(half + F::at(lb, lane, b * 8)) = make_uint2(w[0], w[1]);
        } else {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) w |= static_cast<uint32_t>(code[j] | code[4 + j] << 4) << (8 * j);
            *reinterpret_cast<uint32_t*>(half + F::at(lb, lane, b * 4)) = w;
        }
    }

    // The same of values.  4-bit codes: `code` holds the byte of dimensions d and 16 + d
    // (lanes g of 0 and 1).
    __device__ void value(int slot, int b, int g, const float* y, const int* code) const {
        using F = KvForm<QT>;
        const int lb = F::value_lane(nb);
        uint8_t* o = p + F::half(nb);
        const int j = (slot >> 4) * 4 + (slot & 3);
        const int gk = 16 * ((slot & 15) >> 2);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = 8 * (g & 1) + e;
            if (QT == 0) {
                *reinterpret_cast<float*>(o + F::at(lb, gk + d, b * 64 + (g >> 1) * 32 + j * 4)) = y[e];
            } else if (QT == 1) {
                o[F::at(lb, gk + d, b * 16 + (g >> 1) * 8 + j)] = static_cast<uint8_t>(code[e]);
            } else if (g < 2) {
                o[F::at(lb, gk + d, b * 8 + j)] = static_cast<uint8_t>(code[e]);
            }
        }
    }

    __device__ void scale(bool values, int slot, int b, uint32_t d, uint32_t m) const {
        using F = KvForm<QT>;
        uint8_t* o = p + (values ? F::half(nb) : 0) + F::codes(nb);
        const int i = values ? F::value_scale(nb, slot, b) : F::key_scale(nb, slot, b);
        if (QT == 0) {
            reinterpret_cast<uint32_t*>(o)[i] = d;
        } else {
            reinterpret_cast<uint16_t*>(o)[i] = static_cast<uint16_t>(d);
            if (QT == 3) reinterpret_cast<uint16_t*>(o + F::plane(nb))[i] = static_cast<uint16_t>(m);
        }
    }
};

// Scale (and minimum) of a block whose 32 elements a quad of lanes holds, eight in
// element order each, `here`: whether the lane's lie in the row; codes as stored.
template <int QT>
__device__ __forceinline__ void quantize_block(const float* y, bool here, int g, uint32_t* d, uint32_t* m, int* code) {
#pragma clang fp contract(off)
    *m = 0;
    if (QT == 0) {
        // 2^e with the block's largest element in [2^e, 2^(e+1)), e at least -80; Inf from 2^80 on (sums of
        // products of such elements and their powers of two stay in f32's range)
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, f32_bits(y[i]) & 0x7fffffffu);
        top = max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0xB1, 0xf, 0xf, true)));
        top = max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0x4E, 0xf, 0xf, true)));
        const uint32_t e = top >> 23;
        *d = e >= 127 + 80 ? 0x7f800000u : max(e, 127u - 80u) << 23;
        return;
    }
    if (QT == 3) {
        // the reference's minimum and maximum: the first of equal values stays, NaN never enters
        float lo = __builtin_inff(), hi = -__builtin_inff();
        if (here) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                lo = (y[i] < lo) ? y[i] : lo;
                hi = (hi < y[i]) ? y[i] : hi;
            }
        }
        lo = quad_first_min(lo, g);
        const float range = quad_max(hi) - lo;
        const bool some = range > 0.0f;
        *d = some ? half_round_up(range / 15.0f) : 0;
        *m = half_round_up((!some && lo == __builtin_inff()) ? 0.0f : lo);
        const float dq = half_value(static_cast<uint16_t>(*d)), mq = half_value(static_cast<uint16_t>(*m));
        const float inv = (dq == 0.0f) ? 0.0f : 1.0f / dq;
#pragma unroll
        for (int i = 0; i < 8; ++i) code[i] = some && here ? max(0, min(15, round_int((y[i] - mq) * inv))) : 0;
        return;
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(y[i]);
        amax = (a > amax) ? a : amax;
    }
    amax = quad_max(amax);
    const bool some = amax > 0.0f;
    *d = some ? half_round_up(amax / (QT == 1 ? 127.0f : 7.0f)) : 0;
    const float dq = half_value(static_cast<uint16_t>(*d));
    const float inv = (dq == 0.0f) ? 0.0f : 1.0f / dq;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (QT == 1) {
            code[i] = (some ? max(-127, min(127, round_int(y[i] * inv))) : 0) + 128;
        } else {
            code[i] = some ? max(0, min(15, round_int(y[i] * inv + 8.0f))) : 0;
        }
    }
}

__device__ __forceinline__ void load8(const float* p, float* x) {
    const float4 a = reinterpret_cast<const float4*>(p)[0];
    const float4 b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// Elements e .. e + 7 of a row at x, rotated; turn: the row's (cos, sin) by pair.
__device__ __forceinline__ void load8_rotated(const float* x, int e, int half, int neox, const double2* turn, float* y) {
    float a[8];
    load8(x + e, a);
    if (neox) {
        // four elements at a time lie on one side of the middle
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool low = e + 4 * h < half;
            const int r = low ? e + 4 * h : e + 4 * h - half;
            const float4 o = *reinterpret_cast<const float4*>(x + (low ? r + half : r));
            const float b[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double2 t = turn[r + i];
                const double self = a[4 * h + i], other = low ? -static_cast<double>(b[i]) : static_cast<double>(b[i]);
                y[4 * h + i] = static_cast<float>(self * t.x + other * t.y);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double2 t = turn[e / 2 + i];
            const double x0 = a[2 * i], x1 = a[2 * i + 1];
            y[2 * i] = static_cast<float>(x0 * t.x - x1 * t.y);
            y[2 * i + 1] = static_cast<float>(x0 * t.y + x1 * t.x);
        }
    }
}

// One KV head of an item's tokens: keys (rotated) and values, quantized, to `out`.
template <int QT, typename Tile>
__device__ __forceinline__ void write_kv_head(const KvTileItem& it, int head, const Tile& out, const KvView& kv,
                                              const float* __restrict__ k, const float* __restrict__ v, int rope, int neox,
                                              const double2* turn) {
    const int nb = kv.nb, hd = kv.head_dim, half = hd / 2;
    const int per = 4 * nb;  // tasks of a row: (block, eight elements), a quad of lanes a block
    const int tasks = it.n * per;
    // every quad is whole: `per` and the workgroup are multiples of four
    for (int t = threadIdx.x; t < tasks; t += blockDim.x) {
        const int s = t / per, b = t % per >> 2, g = t & 3;
        const int e = 32 * b + 8 * g;
        const bool here = e < hd;
        const size_t row = (static_cast<size_t>(it.row + s) * kv.n_kv + head) * hd;
        float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        int code[8];
        uint32_t d, m;
        if (here) {
            if (rope) load8_rotated(k + row, e, half, neox, turn + s * half, y);
            else load8(k + row + e, y);
        }
        quantize_block<QT>(y, here, g, &d, &m, code);
        out.key(it.slot + s, b, g, y, code);
        if (g == 0) out.scale(false, it.slot + s, b, d, m);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = 0.0f;
        if (here) load8(v + row + e, y);
        quantize_block<QT>(y, here, g, &d, &m, code);
        if (QT >= 2) {
            // a byte's other nibble is sixteen dimensions on: two lanes of the quad
#pragma unroll
            for (int i = 0; i < 8; ++i) code[i] |= __builtin_amdgcn_mov_dpp(code[i], 0x4E, 0xf, 0xf, true) << 4;
        }
        out.value(it.slot + s, b, g, y, code);
        if (g == 0) out.scale(true, it.slot + s, b, d, m);
    }
}

// Bound: memory (4-byte elements in, cache bytes and rotated queries out: 2048 tokens of
// 32 + 32 heads of 128 in Q8_0 50 us, 3.0 TB/s), for single tokens launch and a chain of
// loads, angles and stores (5 us for one, 10.8 for 64 sequences of 32 + 8 heads).  115
// registers, 16 waves a CU; 80 (some spilled) took as long, 64 up to a third longer.  A
// workgroup takes `per_group` heads of one tile's new tokens; the pairs' cosines and
// sines, in 64 bits, are computed once for them.  A tile that is written whole
// gathers in LDS and leaves as 16-byte stores; of others the new slots are
// stored where they belong, values byte by byte, so that slots of other
// sequences or earlier tokens in the same words are never rewritten.
template <int QT>
__global__ __launch_bounds__(kWriteThreads) void kv_write_kernel(KvView kv, const KvTileItem* __restrict__ items,
                                                              const int* __restrict__ counts, int count,
                                                              const float* __restrict__ k, const float* __restrict__ v,
                                                              const float* q, float* q_out, int n_heads, int per_group,
                                                              KvRope rope) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    double2* const turn = reinterpret_cast<double2*>(lds);  // [token][pair]
    const int hd = kv.head_dim, half = hd / 2;
    uint8_t* const image = lds + (rope.on ? kKvTile * half * sizeof(double2) : 0);
    const int heads = kv.n_kv + (q != nullptr ? n_heads : 0);
    const int chunks = (heads + per_group - 1) / per_group;
    const int total = (count > 0 ? count : counts[kKvCountFresh]) * chunks;
    const int tile_bytes = KvForm<QT>::tile(kv.nb);
    for (int w = blockIdx.x; w < total; w += gridDim.x) {
        const KvTileItem it = items[w / chunks];
        const int h0 = w % chunks * per_group, h1 = min(heads, h0 + per_group);
        if (rope.on) {
            __syncthreads();  // the last item's readers are done
            for (int i = threadIdx.x; i < it.n * half; i += blockDim.x) {
                const double a = static_cast<double>(it.pos + i / half) * rope.turns[i % half];
                double2 t;
                sincospi(2.0 * (a - rint(a)), &t.y, &t.x);
                turn[i] = t;
            }
            __syncthreads();
        }
        for (int h = h0; h < min(h1, kv.n_kv); ++h) {
            uint8_t* tile = kv.base + ((static_cast<size_t>(it.page) * kv.n_kv + h) * kv.page_tiles + it.tile) * tile_bytes;
            if (it.n == kKvTile) {
                write_kv_head<QT>(it, h, TileOut<QT>{image, kv.nb}, kv, k, v, rope.on, rope.neox, turn);
                __syncthreads();
                for (int i = threadIdx.x * 16; i < tile_bytes; i += blockDim.x * 16) {
                    *reinterpret_cast<uint4*>(tile + i) = *reinterpret_cast<const uint4*>(image + i);
                }
                __syncthreads();
            } else {
                write_kv_head<QT>(it, h, TileOut<QT>{tile, kv.nb}, kv, k, v, rope.on, rope.neox, turn);
            }
        }
        // Query heads: a thread rotates four pairs, both members, so q_out may be q.
        const int q0 = max(h0, kv.n_kv) - kv.n_kv, nq = h1 - kv.n_kv - q0;
        const int per = hd / 8;
        for (int t = threadIdx.x; t < nq * it.n * per; t += blockDim.x) {
            const int r = t % per * 4, s = t / per % it.n, h = q0 + t / per / it.n;
            const size_t row = (static_cast<size_t>(it.row + s) * n_heads + h) * hd;
            const int e0 = rope.neox ? r : 2 * r, e1 = rope.neox ? r + half : 2 * r + 4;
            const float4 a = *reinterpret_cast<const float4*>(q + row + e0);
            const float4 b = *reinterpret_cast<const float4*>(q + row + e1);
            const float x0[4] = {a.x, rope.neox ? a.y : a.z, rope.neox ? a.z : b.x, rope.neox ? a.w : b.z};
            const float x1[4] = {rope.neox ? b.x : a.y, rope.neox ? b.y : a.w, rope.neox ? b.z : b.y, b.w};
            float y0[4], y1[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double2 c = turn[s * half + r + i];
                y0[i] = static_cast<float>(x0[i] * c.x - x1[i] * c.y);
                y1[i] = static_cast<float>(x0[i] * c.y + x1[i] * c.x);
            }
            float4 o0 = make_float4(y0[0], y0[1], y0[2], y0[3]), o1 = make_float4(y1[0], y1[1], y1[2], y1[3]);
            if (!rope.neox) {
                o0 = make_float4(y0[0], y1[0], y0[1], y1[1]);
                o1 = make_float4(y0[2], y1[2], y0[3], y1[3]);
            }
            *reinterpret_cast<float4*>(q_out + row + e0) = o0;
            *reinterpret_cast<float4*>(q_out + row + e1) = o1;
        }
    }
}

// Byte i of a word of codes (4-bit: its low nibble) times its scale, exactly.
template <int QT>
__device__ __forceinline__ float value_of(uint32_t w, int i, float d, float m) {
    const int c = static_cast<int>((w >> (8 * i)) & (QT == 1 ? 0xffu : 0xfu));
    const float y = static_cast<float>(c - (QT == 1 ? 128 : QT == 2 ? 8 : 0)) * d;
    return QT == 3 ? y + m : y;
}

// Bound: memory (cache bytes in, 4-byte elements out: 8 sequences of up to 4000 positions,
// 8 KV heads of 128 in Q8_0, 46 us, 4.7 TB/s).  A workgroup brings one tile to LDS with
// 16-byte loads and writes its positions' rows; a thread decodes what shares a word.
template <int QT>
__global__ __launch_bounds__(kReadThreads) void kv_read_kernel(KvView kv, KvLists lists, bool fresh, int count,
                                                             float* __restrict__ k, float* __restrict__ v) {
    using F = KvForm<QT>;
    extern __shared__ __attribute__((aligned(16))) uint8_t image[];
    const int nb = kv.nb, hd = kv.head_dim;
    const int tile_bytes = F::tile(nb);
    const int entries = count > 0 ? count : lists.counts[fresh ? kKvCountFresh : kKvCountPages];
    const int per_entry = (fresh ? 1 : kv.page_tiles) * kv.n_kv;
    const long long total = static_cast<long long>(entries) * per_entry;
    for (long long w = blockIdx.x; w < total; w += gridDim.x) {
        const int entry = static_cast<int>(w / per_entry), part = static_cast<int>(w % per_entry);
        const int head = part % kv.n_kv;
        int page, tile, slot = 0, n, row;
        if (fresh) {
            const KvTileItem it = lists.fresh[entry];
            page = it.page, tile = it.tile, slot = it.slot, n = it.n, row = it.row;
        } else {
            const KvPage p = lists.pages[entry];
            page = p.page, tile = part / kv.n_kv;
            n = min(kKvTile, p.n - tile * kKvTile), row = p.row + tile * kKvTile;
        }
        if (n <= 0) continue;
        const uint8_t* src = kv.base + ((static_cast<size_t>(page) * kv.n_kv + head) * kv.page_tiles + tile) * tile_bytes;
        __syncthreads();  // the last tile's readers are done
        for (int i = threadIdx.x * 16; i < tile_bytes; i += kReadThreads * 16) {
            *reinterpret_cast<uint4*>(image + i) = *reinterpret_cast<const uint4*>(src + i);
        }
        __syncthreads();
        // Keys: four elements of a position a thread, which share a word of codes and a scale.
        const size_t first = (static_cast<size_t>(row) * kv.n_kv + head) * hd, step = static_cast<size_t>(kv.n_kv) * hd;
        const int per = hd / 4, at_once = kReadThreads / per;
        const uint16_t* scale = reinterpret_cast<const uint16_t*>(image + F::codes(nb));
        const uint16_t* minimum = reinterpret_cast<const uint16_t*>(image + F::codes(nb) + F::plane(nb));
        {
            const int e = threadIdx.x % per * 4, b = e >> 5, r = e & 31;
            const int lb = F::key_lane(nb);
            for (int s = threadIdx.x / per; s < n; s += at_once) {
                if (static_cast<int>(threadIdx.x) >= at_once * per) break;
                const int key = slot + s, lane = 16 * (r >> 3) + (key & 15);
                const uint8_t* p = image + (key >> 4) * 64 * lb;
                float4 y;
                if (QT == 0) {
                    y = *reinterpret_cast<const float4*>(p + F::at(lb, lane, (b * 8 + (r & 7)) * 4));
                } else {
                    const int si = F::key_scale(nb, key, b);
                    const float d = half_value(scale[si]), m = QT == 3 ? half_value(minimum[si]) : 0.0f;
                    uint32_t w;
                    if (QT == 1) w = *reinterpret_cast<const uint32_t*>(p + F::at(lb, lane, b * 8 + (r & 7)));
                    else w = *reinterpret_cast<const uint32_t*>(p + F::at(lb, lane, b * 4)) >> (r & 4);
                    y = make_float4(value_of<QT>(w, 0, d, m), value_of<QT>(w, 1, d, m), value_of<QT>(w, 2, d, m), value_of<QT>(w, 3, d, m));
                }
                *reinterpret_cast<float4*>(k + first + s * step + e) = y;
            }
        }
        // Values: a thread takes the four positions of one dimension that share a word.
        scale = reinterpret_cast<const uint16_t*>(image + F::half(nb) + F::codes(nb));
        minimum = reinterpret_cast<const uint16_t*>(image + F::half(nb) + F::codes(nb) + F::plane(nb));
        const int lb = F::value_lane(nb);
        for (int t = threadIdx.x; t < 8 * hd; t += kReadThreads) {
            const int d = t % hd, quad = t / hd;  // positions 4 quad ..
            if (4 * quad + 3 < slot || 4 * quad >= slot + n) continue;
            const int b = d >> 5, r = d & 31, lane = 16 * (quad & 3) + (r & 15), x = (r >> 4) * 8 + (quad >> 2) * 4;
            const uint8_t* p = image + F::half(nb);
            float y[4];
            if (QT == 0) {
                const float4 f = *reinterpret_cast<const float4*>(p + F::at(lb, lane, (b * 16 + x) * 4));
                y[0] = f.x, y[1] = f.y, y[2] = f.z, y[3] = f.w;
            } else {
                uint32_t w;
                if (QT == 1) w = *reinterpret_cast<const uint32_t*>(p + F::at(lb, lane, b * 16 + x));
                else w = *reinterpret_cast<const uint32_t*>(p + F::at(lb, lane, b * 8 + (x & 7))) >> (r >> 4 << 2);
                const int si = F::value_scale(nb, 4 * quad, b);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[i] = value_of<QT>(w, i, half_value(scale[si + i]), QT == 3 ? half_value(minimum[si + i]) : 0.0f);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int s = 4 * quad + i - slot;
                if (s >= 0 && s < n) v[first + s * step + d] = y[i];
            }
        }
    }
}

template <typename K>
hipError_t allow_lds(K kernel, int bytes) {
    if (bytes <= 64 << 10) return hipSuccess;
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int QT>
hipError_t write(const KvView& kv, const KvLists& lists, int count, int tokens, const float* k, const float* v, const float* q,
                 float* q_out, int n_heads, const KvRope& rope, hipStream_t s) {
    const int heads = kv.n_kv + (q != nullptr ? n_heads : 0);
    // Heads a workgroup takes: the angles are computed once for them, as long as there are workgroups
    // enough (2048 tokens, 64 heads, 1 / 2 / 4 / 8 a workgroup: 75 / 71 / 64 / 62 us with the read
    // back; 903 tokens 29 / 31 / 33 / 42).
    const int per_group = std::max(1, std::min(8, static_cast<int>(static_cast<long long>(count) * heads / kRecordedGroups)));
    const long long groups = static_cast<long long>(count) * ((heads + per_group - 1) / per_group);
    const int lds = KvForm<QT>::tile(kv.nb) +
                    (rope.on ? kKvTile * (kv.head_dim / 2) * static_cast<int>(sizeof(double2)) : 0);
    // Whole tiles keep 512 threads busy (2048 tokens, 32 + 32 heads of 128: 62 us with the read back, 92
    // with 256); a token or two do not (64 sequences: 14 us, 17 with 512).
    const unsigned threads = tokens > 4ll * count ? kWriteThreads : kWriteThreads / 2;
    const hipError_t e = allow_lds(kv_write_kernel<QT>, lds);
    if (e != hipSuccess) return e;
    const unsigned grid = count > 0 ? static_cast<unsigned>(std::min<long long>(groups, 1 << 20)) : kRecordedGroups;
    kv_write_kernel<QT><<<grid, threads, lds, s>>>(kv, lists.fresh, lists.counts, count, k, v, q, q_out, n_heads,
                                                      count > 0 ? per_group : 4, rope);
    return hipGetLastError();
}

template <int QT>
hipError_t read(const KvView& kv, const KvLists& lists, bool fresh, int count, float* k, float* v, hipStream_t s) {
    const long long groups = static_cast<long long>(count) * (fresh ? 1 : kv.page_tiles) * kv.n_kv;
    const int lds = KvForm<QT>::tile(kv.nb);
    const hipError_t e = allow_lds(kv_read_kernel<QT>, lds);
    if (e != hipSuccess) return e;
    const unsigned grid = count > 0 ? static_cast<unsigned>(std::min<long long>(groups, 1 << 20)) : kRecordedGroups;
    kv_read_kernel<QT><<<grid, kReadThreads, lds, s>>>(kv, lists, fresh, count, k, v);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_upload(const KvParts& parts, hipStream_t s) {
    int most = 1;
    for (int w : parts.words) most = std::max(most, w);
    kv_upload_kernel<<<std::min((most + 255) / 256, 256), 256, 0, s>>>(parts);
    return hipGetLastError();
}

hipError_t launch_kv_write(const KvView& kv, const KvLists& lists, int count, int tokens, const float* k, const float* v,
                           const float* q, float* q_out, int n_heads, const KvRope& rope, hipStream_t s) {
    switch (kv.qtype) {
        case 0: return write<0>(kv, lists, count, tokens, k, v, q, q_out, n_heads, rope, s);
        case 1: return write<1>(kv, lists, count, tokens, k, v, q, q_out, n_heads, rope, s);
        case 2: return write<2>(kv, lists, count, tokens, k, v, q, q_out, n_heads, rope, s);
        case 3: return write<3>(kv, lists, count, tokens, k, v, q, q_out, n_heads, rope, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_kv_read(const KvView& kv, const KvLists& lists, bool fresh, int count, float* k, float* v, hipStream_t s) {
    switch (kv.qtype) {
        case 0: return read<0>(kv, lists, fresh, count, k, v, s);
        case 1: return read<1>(kv, lists, fresh, count, k, v, s);
        case 2: return read<2>(kv, lists, fresh, count, k, v, s);
        case 3: return read<3>(kv, lists, fresh, count, k, v, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mlq
