// Attention of a batch's new tokens over the paged cache (kv_layout.h) on MFMA.
//
// out = softmax_j(scale q . k_j) v over the positions j that a token at position i
// sees: j <= i and, with a window of w, j > i - w or j < sinks.
//
// A wave walks tiles of 32 positions of one KV head for up to 32 query rows (row =
// token * group + query head of the group, so grouped heads fill the tile and share
// what is read).  Per tile, in v_mfma_f32_16x16x32_f16 with operands that come
// from memory as they lie there:
//
//   S^T = K Q^T   per block b of 32 elements: the codes are whole numbers (exact in
//                 fp16), the queries pairs of fp16 parts hi + lo relative to the row's
//                 largest (2^-22 of it is lost), so a product is exact and the sum
//                 f32; times the block's scale it goes into the score.  A Q4_1 block adds
//                 its minimum times the queries' sum.  f32 keys are split the same way,
//                 relative to the block's power of two: three products.
//   O^T += V^T P^T   the value scale d_jb belongs to key and block, so it goes into the
//                 weights: P_b = p_j d_jb, split into hi + lo, times the codes.
//
// The running maximum m of a row is that of t_j + e_j, t the score in base 2 and 2^e_j
// (nearly) the largest value scale of position j: then no P_b passes 2^15 and what is
// large in the sum is what keeps all its digits, whatever the values' size; a value of
// zero takes no digits from the others.  It moves only when t + e passes it by 6, so the
// accumulators are seldom rescaled.  The sum of the weights is f32 in the same frame.
//
// Where few rows share a KV head (up to 8: decode), the hi parts are columns 0 .. 7 of
// the query operand and the lo parts columns 8 .. 15, of the weights as well: one product
// where there would be two, the halves added at the end.
//
// What a row does not see gets weight 0, and 0 times a scale that is Inf or NaN is 0
// (v_mul_legacy_f32); codes are finite always.
#pragma once

#include "kv_layout.h"

#include <hip/hip_runtime.h>

#include <cmath>

namespace mlq {
namespace kv {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef unsigned short us2_t __attribute__((ext_vector_type(2)));

constexpr int kThreads = 64 * kKvWaves;
constexpr int kCoherent = 16;   // sc1: through to / from the point of coherence
constexpr float kSlack = 6.0f;  // a row's maximum moves when it is passed by this

template <typename T>
__device__ __forceinline__ T bits(uint32_t v) { return __builtin_bit_cast(T, v); }

// Reads of the work lists, through the scalar cache: uniform, constant for the launch.
__device__ __forceinline__ int uniform(const int* p) { return *(const __attribute__((address_space(4))) int*)(p); }
__device__ __forceinline__ KvAttnItem uniform(const KvAttnItem* p) {
    constexpr int N = sizeof(KvAttnItem) / sizeof(int);
    struct Words {
        int v[N];
    } w;
#pragma unroll
    for (int i = 0; i < N; ++i) w.v[i] = uniform(reinterpret_cast<const int*>(p) + i);
    return __builtin_bit_cast(KvAttnItem, w);
}

__device__ __forceinline__ float max_quarters(float v) {  // over the lanes of equal lane % 16
    auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = fmaxf(bits<float>(r[0]), bits<float>(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(bits<float>(r[0]), bits<float>(r[1]));
}
__device__ __forceinline__ float sum_quarters(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = bits<float>(r[0]) + bits<float>(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return bits<float>(r[0]) + bits<float>(r[1]);
}
// a * b, and 0 where either is 0, whatever the other is (Inf and NaN too).
// (The compiler's intrinsic by its name, as there is no builtin of it; not inline asm, whose
// operands the compiler does not keep apart from the transcendental unit's results.)
__device__ __attribute__((const)) float mul_or_zero(float a, float b) __asm("llvm.amdgcn.fmul.legacy");
// The lane 8 columns on (row_ror:8): the other half of a stacked row.
__device__ __forceinline__ float other_half(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));
}

// A lane's LB bytes, unit by unit.
template <int LB>
__device__ __forceinline__ void load_units(const uint8_t* p, int lane, uint32_t* w) {
    constexpr int U = KvForm<0>::unit(LB);
#pragma unroll
    for (int x = 0; x < LB; x += U) {
        const uint8_t* at = p + x * 64 + lane * U;
        if (U == 16) {
            const u4_t v = *reinterpret_cast<const u4_t*>(at);
            w[x / 4] = v.x, w[x / 4 + 1] = v.y, w[x / 4 + 2] = v.z, w[x / 4 + 3] = v.w;
        } else if (U == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            w[x / 4] = v.x, w[x / 4 + 1] = v.y;
        } else {
            w[x / 4] = *reinterpret_cast<const uint32_t*>(at);
        }
    }
}
// N consecutive bytes.
template <int N>
__device__ __forceinline__ void load_run(const uint8_t* p, uint32_t* w) {
    constexpr int U = KvForm<0>::unit(N);
#pragma unroll
    for (int x = 0; x < N; x += U) {
        if (U == 16) {
            const u4_t v = *reinterpret_cast<const u4_t*>(p + x);
            w[x / 4] = v.x, w[x / 4 + 1] = v.y, w[x / 4 + 2] = v.z, w[x / 4 + 3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(p + x);
            w[x / 4] = v.x, w[x / 4 + 1] = v.y;
        }
    }
}

// Four unsigned bytes minus `off`, as fp16: the bytes become the low bits of 1024 + byte.
__device__ __forceinline__ void bytes_f16(uint32_t w, _Float16 off, h2_t* out) {
    const _Float16 base = static_cast<_Float16>(1024.0f) + off;
    const h2_t sub{base, base};
    out[0] = bits<h2_t>(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - sub;
    out[1] = bits<h2_t>(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - sub;
}
__device__ __forceinline__ h8_t join(h2_t a, h2_t b, h2_t c, h2_t d) {
    return h8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// Eight bytes (two words); eight nibbles, low ones first (one word); one nibble of eight bytes.
__device__ __forceinline__ h8_t codes8(uint32_t w0, uint32_t w1, _Float16 off) {
    h2_t a[2], b[2];
    bytes_f16(w0, off, a);
    bytes_f16(w1, off, b);
    return join(a[0], a[1], b[0], b[1]);
}
// v = hi + lo, both fp16, for |v| < 65504: 2^-22 of v (or 2^-25) is lost.
__device__ __forceinline__ void split8(const float* v, h8_t* hi, h8_t* lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const _Float16 h = static_cast<_Float16>(v[j]);
        (*hi)[j] = h;
        (*lo)[j] = static_cast<_Float16>(v[j] - static_cast<float>(h));
    }
}
// 1 / s for a power of two s from 2^-90 on; 0 for Inf.
__device__ __forceinline__ float inverse_power(uint32_t s) {
    return bits<float>(static_cast<uint32_t>(max(static_cast<int>(0x7f000000u) - static_cast<int>(s), 0)));
}

__device__ __forceinline__ f4_t mfma(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

template <int QT, int NB, int ROWS>
__global__ __launch_bounds__(kThreads) void attention_kernel(KvAttention a, int kind, int count,
                                                                const float* __restrict__ q, float* __restrict__ out) {
    using F = KvForm<QT>;
    constexpr bool STACK = ROWS == kKvNarrowRows;
    constexpr int NQ = ROWS == 32 ? 2 : 1;  // query tiles of 16 columns
    constexpr int SB = F::kScaleBytes;
    constexpr int KL = F::key_lane(NB), VL = F::value_lane(NB);
    constexpr int KW = KL / 4, VW = VL / 4;
    constexpr int KS = NB * SB, VS = 2 * NB * SB;  // words of a lane's scales: 4 keys a half tile, 8 keys
    constexpr int QUADS = NQ * 2 * NB;             // accumulators
    constexpr int STATE = (QUADS * 4 + 2 * NQ) * 64;  // floats of a wave's state
    __shared__ float merge[2 * STATE];
    __shared__ unsigned last;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i16 = lane & 15, g = lane >> 4;
    const int n_kv = a.kv.n_kv, hd = a.kv.head_dim, heads = n_kv * a.group;
    const int page_tiles = a.kv.page_tiles, tile_shift = __builtin_ctz(page_tiles);
    const int total = (count > 0 ? count : uniform(a.lists.counts + kKvCountNarrow + kind)) * n_kv;

    for (int w = blockIdx.x; w < total; w += gridDim.x) {
        const int head = w % n_kv;
        const KvAttnItem it = uniform(a.lists.items[kind] + w / n_kv);
        const bool together = it.stride == 1;
        const int rows = it.new_tokens * a.group, start = it.len - it.new_tokens;
        const int row0 = it.row0 + (together ? wave * ROWS : 0);
        const bool idle = row0 >= rows;
        const int row1 = min(rows, row0 + ROWS);
        const int pos_lo = start + min(row0, rows - 1) / a.group, pos_hi = start + (max(row1, 1) - 1) / a.group;

        // Queries: row's elements relative to its largest, which becomes 2^13 .. 2^14.
        h8_t qh[NQ][NB], ql[NQ][NB];
        float qsum[NQ][NB], to_t[NQ];
        int pos[NQ];
        size_t out_row[NQ];
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            const int r = min(row0 + 16 * u + (STACK ? i16 & 7 : i16), rows - 1);
            const int token = r / a.group;
            pos[u] = start + token;
            out_row[u] = (static_cast<size_t>(it.token0 + token) * heads + head * a.group + r % a.group) * hd;
            float v[NB][8];
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int e = 32 * b + 8 * g;
                float4 x = make_float4(0, 0, 0, 0), y = x;
                if (e < hd) {
                    x = *reinterpret_cast<const float4*>(q + out_row[u] + e);
                    y = *reinterpret_cast<const float4*>(q + out_row[u] + e + 4);
                }
                v[b][0] = x.x, v[b][1] = x.y, v[b][2] = x.z, v[b][3] = x.w;
                v[b][4] = y.x, v[b][5] = y.y, v[b][6] = y.z, v[b][7] = y.w;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[b][j]));
            }
            top = max_quarters(top);
            // exponent, kept where 2^(13 - e) and its inverse are normal
            const int e = min(max(static_cast<int>(__builtin_bit_cast(uint32_t, top) >> 23) - 127, -100), 127);
            const float up = ldexpf(1.0f, 13 - e);
            to_t[u] = ldexpf(a.scale, e - 13);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[b][j] *= up;
                    sum += v[b][j];
                }
                h8_t hi, lo;
                split8(v[b], &hi, &lo);
                qh[u][b] = STACK && i16 >= 8 ? lo : hi;
                ql[u][b] = lo;
                if (QT == 3) qsum[u][b] = STACK && i16 >= 8 ? 0.0f : sum_quarters(sum);
            }
        }

        f4_t o[NQ][2 * NB];
        float om[NQ][NB];  // Q4_1: this lane's part of the sum of weights times minima
        float m[NQ], l[NQ];
        const f4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            m[u] = -3.402823466e38f;
            l[u] = 0.0f;
#pragma unroll
            for (int t = 0; t < 2 * NB; ++t) o[u][t] = zero;
#pragma unroll
            for (int b = 0; b < NB; ++b) om[u][b] = 0.0f;
        }

        // This wave's tiles: every it.stride-th of the item's, those past its last row left out.
        const int past = pos_hi / kKvTile + 1;  // tiles up to here have something to see
        int end = it.first + it.count;
        if (past - it.shift < end) end = max(past - it.shift, it.sinks);
        if (idle) end = 0;
        int at = it.first + (together ? 0 : wave);
        auto tile_of = [&](int i) { return i < it.sinks ? i : i + it.shift; };
        auto page_of = [&](int i) { return uniform(&a.lists.pages[it.page0 + (tile_of(i) >> tile_shift)].page); };
        auto base_of = [&](int i, int page) {
            return a.kv.base + ((static_cast<size_t>(page) * n_kv + head) * page_tiles + (tile_of(i) & (page_tiles - 1))) * F::tile(NB);
        };

        uint32_t kw[2][KW], ks[2][KS], km[2][QT == 3 ? KS : 1];
        uint32_t kp[2][QT == 0 ? NB : 1];  // f32: the scales of the lane's own key (ks: of the keys of its scores)
        uint32_t vw[VW], vs[VS], vm[QT == 3 ? VS : 1];
        auto load_keys = [&](const uint8_t* tile) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                load_units<KL>(tile + h * 64 * KL, lane, kw[h]);
                load_run<4 * KS>(tile + F::codes(NB) + (4 * h + g) * 4 * KS, ks[h]);
                if (QT == 3) load_run<4 * KS>(tile + F::codes(NB) + F::plane(NB) + (4 * h + g) * 4 * KS, km[h]);
                if (QT == 0) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        kp[h][b] = reinterpret_cast<const uint32_t*>(tile + F::codes(NB))[F::key_scale(NB, 16 * h + i16, b)];
                    }
                }
            }
        };
        auto load_values = [&](const uint8_t* tile) {
            load_units<VL>(tile + F::half(NB), lane, vw);
            load_run<4 * VS>(tile + F::half(NB) + F::codes(NB) + g * 4 * VS, vs);
            if (QT == 3) load_run<4 * VS>(tile + F::half(NB) + F::codes(NB) + F::plane(NB) + g * 4 * VS, vm);
        };
        // f16 scale i of an array of words (f32: word i)
        auto scale_at = [&](const uint32_t* s, int i) -> float {
            if (QT == 0) return bits<float>(s[i]);
            const h2_t p = bits<h2_t>(s[i / 2]);
            return static_cast<float>(i % 2 == 0 ? p.x : p.y);
        };

        int next_page = 0;
        if (at < end) {
            const uint8_t* tile = base_of(at, page_of(at));
            load_keys(tile);
            load_values(tile);
            if (at + it.stride < end) next_page = page_of(at + it.stride);
        }
        for (; at < end; at += it.stride) {
            const int first = tile_of(at) * kKvTile;
            const bool more = at + it.stride < end;
            const uint8_t* next = base_of(more ? at + it.stride : at, next_page);
            if (at + 2 * it.stride < end) next_page = page_of(at + 2 * it.stride);

            // Scores.
            f4_t s[NQ][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int u = 0; u < NQ; ++u) s[u][h] = zero;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    f4_t acc[NQ];
                    if (QT == 0) {
                        h8_t hi, lo;
                        float v[8];
                        const float inv = inverse_power(kp[h][b]);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = mul_or_zero(bits<float>(kw[h][8 * b + j]), inv);
                        split8(v, &hi, &lo);
#pragma unroll
                        for (int u = 0; u < NQ; ++u) {
                            acc[u] = mfma(hi, qh[u][b], zero);
                            if (!STACK) acc[u] = mfma(hi, ql[u][b], acc[u]);
                            acc[u] = mfma(lo, qh[u][b], acc[u]);
                        }
                    } else {
                        h8_t k;
                        if (QT == 1) {
                            k = codes8(kw[h][2 * b], kw[h][2 * b + 1], static_cast<_Float16>(128.0f));
                        } else {
                            const uint32_t x = kw[h][b];
                            k = codes8(x & 0x0f0f0f0fu, (x >> 4) & 0x0f0f0f0fu, static_cast<_Float16>(QT == 2 ? 8.0f : 0.0f));
                        }
#pragma unroll
                        for (int u = 0; u < NQ; ++u) {
                            acc[u] = mfma(k, qh[u][b], zero);
                            if (!STACK) acc[u] = mfma(k, ql[u][b], acc[u]);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < NQ; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[u][h][i] = fmaf(scale_at(ks[h], 4 * b + i), acc[u][i], s[u][h][i]);
                            if (QT == 3) s[u][h][i] = fmaf(scale_at(km[h], 4 * b + i), qsum[u][b], s[u][h][i]);
                        }
                }
            }
            if (more) load_keys(next);

            // Weights.
            float e[8];  // log2 of a position's largest value scale, plus a constant
            {
                uint32_t top[8];
                if (QT == 0) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        top[j] = vs[j];
#pragma unroll
                        for (int b = 1; b < NB; ++b) top[j] = max(top[j], vs[8 * b + j]);
                        e[j] = static_cast<float>(top[j]) * 0x1p-23f;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        us2_t t = bits<us2_t>(vs[j / 2]);
#pragma unroll
                        for (int b = 1; b < NB; ++b) t = __builtin_elementwise_max(t, bits<us2_t>(vs[4 * b + j / 2]));
                        e[j] = static_cast<float>(t.x) * 0x1p-10f;
                        e[j + 1] = static_cast<float>(t.y) * 0x1p-10f;
                    }
                }
            }
            constexpr float kBias = (QT == 0 ? 127.0f : 15.0f) + 8.0f;
            const bool full = first + kKvTile - 1 <= pos_lo &&
                              (a.window == 0 || first > pos_hi - a.window || first + kKvTile <= a.sinks);
            float p[NQ][8];
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float x = s[u][j >> 2][j & 3];
                    if (STACK) x += other_half(x);
                    x *= to_t[u];
                    // an infinite scale (minimum) with codes that are not 0: NaN like the sum of its elements
                    if (QT >= 2) x = fmaf(x, 0.0f, x);
                    if (!full) {
                        const int key = first + (j >> 2) * 16 + 4 * g + (j & 3);
                        const bool seen = key <= pos[u] && (a.window == 0 || key > pos[u] - a.window || key < a.sinks);
                        x = seen ? x : -INFINITY;
                    }
                    p[u][j] = x;
                    top = fmaxf(top, x + e[j]);
                }
                top = max_quarters(top);
                if (__any(top > m[u] + kSlack)) {
                    const float to = top > m[u] + kSlack ? top : m[u];
                    const float c = __builtin_amdgcn_exp2f(m[u] - to);
                    m[u] = to;
                    l[u] *= c;
#pragma unroll
                    for (int t = 0; t < 2 * NB; ++t) o[u][t] *= c;
                    if (QT == 3) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) om[u][b] *= c;
                    }
                }
                const float frame = m[u] - kBias;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[u][j] = __builtin_amdgcn_exp2f(p[u][j] - frame);
                    l[u] += p[u][j];
                }
            }

            // Values.
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                h8_t ph[NQ], pl[NQ];
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = mul_or_zero(p[u][j], scale_at(vs, 8 * b + j));
                    h8_t hi, lo;
                    split8(v, &hi, &lo);
                    ph[u] = STACK && i16 >= 8 ? lo : hi;
                    pl[u] = lo;
                    if (QT == 3) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) om[u][b] += mul_or_zero(p[u][j], scale_at(vm, 8 * b + j));
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    h8_t c, lo;
                    if (QT == 0) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            v[j] = mul_or_zero(bits<float>(vw[16 * b + 8 * t + j]), inverse_power(vs[8 * b + j]));
                        }
                        split8(v, &c, &lo);
                    } else if (QT == 1) {
                        c = codes8(vw[4 * b + 2 * t], vw[4 * b + 2 * t + 1], static_cast<_Float16>(128.0f));
                    } else {
                        const uint32_t x = vw[2 * b], y = vw[2 * b + 1];
                        c = codes8((t == 0 ? x : x >> 4) & 0x0f0f0f0fu, (t == 0 ? y : y >> 4) & 0x0f0f0f0fu,
                                   static_cast<_Float16>(QT == 2 ? 8.0f : 0.0f));
                    }
#pragma unroll
                    for (int u = 0; u < NQ; ++u) {
                        f4_t& acc = o[u][2 * b + t];
                        acc = mfma(c, ph[u], acc);
                        if (!STACK) acc = mfma(c, pl[u], acc);
                        if (QT == 0) acc = mfma(lo, ph[u], acc);
                    }
                }
            }
            if (more) load_values(next);
        }

        // The lanes' sums, the stacked halves and the minima's part together.
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            l[u] = sum_quarters(l[u]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float add = QT == 3 ? sum_quarters(om[u][b]) : 0.0f;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = o[u][2 * b + t][i];
                        if (STACK) x += other_half(x);
                        o[u][2 * b + t][i] = QT == 3 ? x + add : x;
                    }
            }
        }
        // Takes in another state of the same rows.
        auto fold = [&](int u, float m1, float l1, float* w0, float* w1) {
            const float to = fmaxf(m[u], m1);
            *w0 = __builtin_amdgcn_exp2f(m[u] - to);
            *w1 = __builtin_amdgcn_exp2f(m1 - to);
            m[u] = to;
            l[u] = l[u] * *w0 + l1 * *w1;
        };
        auto leave = [&](float* to) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
#pragma unroll
                for (int t = 0; t < 2 * NB; ++t) *reinterpret_cast<f4_t*>(to + ((u * 2 * NB + t) * 64 + lane) * 4) = o[u][t];
                to[QUADS * 256 + (2 * u) * 64 + lane] = m[u];
                to[QUADS * 256 + (2 * u + 1) * 64 + lane] = l[u];
            }
        };
        auto take = [&](const float* from) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                float w0, w1;
                fold(u, from[QUADS * 256 + (2 * u) * 64 + lane], from[QUADS * 256 + (2 * u + 1) * 64 + lane], &w0, &w1);
#pragma unroll
                for (int t = 0; t < 2 * NB; ++t) {
                    const f4_t x = *reinterpret_cast<const f4_t*>(from + ((u * 2 * NB + t) * 64 + lane) * 4);
                    o[u][t] = o[u][t] * w0 + x * w1;
                }
            }
        };
        // The four waves' states into wave 0, in a fixed order.
        auto merge_waves = [&] {
            __syncthreads();
            if (wave >= 2) leave(merge + (wave - 2) * STATE);
            __syncthreads();
            if (wave < 2) take(merge + wave * STATE);
            __syncthreads();
            if (wave == 1) leave(merge);
            __syncthreads();
            if (wave == 0) take(merge);
        };
        if (!together) merge_waves();

        if (it.nsplit > 1) {
            // This part's state to memory; the workgroup that arrives last merges all parts.
            const size_t each = static_cast<size_t>(STATE) * sizeof(float);
            uint8_t* const parts = reinterpret_cast<uint8_t*>(a.partial);
            auto rsrc_of = [&](int split) {
                return __builtin_amdgcn_make_buffer_rsrc(
                    parts + (static_cast<size_t>(it.slot + split) * n_kv + head) * each, static_cast<short>(0),
                    static_cast<int>(each), 0x00020000);
            };
            if (wave == 0) {
                const __amdgpu_buffer_rsrc_t rs = rsrc_of(it.split);
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
#pragma unroll
                    for (int t = 0; t < 2 * NB; ++t) {
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, o[u][t]), rs,
                                                               ((u * 2 * NB + t) * 64 + lane) * 16, 0, kCoherent);
                    }
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, m[u]), rs,
                                                          (QUADS * 256 + (2 * u) * 64 + lane) * 4, 0, kCoherent);
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, l[u]), rs,
                                                          (QUADS * 256 + (2 * u + 1) * 64 + lane) * 4, 0, kCoherent);
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the state is in memory
                if (lane == 0) {
                    unsigned* const c = a.arrived + static_cast<size_t>(it.slot) * n_kv + head;
                    const unsigned before = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    last = before + 1 == static_cast<unsigned>(it.nsplit) ? 1u : 0u;
                    if (last != 0u) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
            __syncthreads();
            const bool mine = last != 0u;
            __syncthreads();
            if (!mine) continue;
            // Wave w takes parts w, w + 4, ...
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                m[u] = -3.402823466e38f;
                l[u] = 0.0f;
#pragma unroll
                for (int t = 0; t < 2 * NB; ++t) o[u][t] = zero;
            }
            for (int part = wave; part < it.nsplit; part += kKvWaves) {
                const __amdgpu_buffer_rsrc_t rs = rsrc_of(part);
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    const float m1 = bits<float>(__builtin_amdgcn_raw_buffer_load_b32(rs, (QUADS * 256 + (2 * u) * 64 + lane) * 4, 0, kCoherent));
                    const float l1 = bits<float>(__builtin_amdgcn_raw_buffer_load_b32(rs, (QUADS * 256 + (2 * u + 1) * 64 + lane) * 4, 0, kCoherent));
                    f4_t x[2 * NB];
#pragma unroll
                    for (int t = 0; t < 2 * NB; ++t) {
                        x[t] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, ((u * 2 * NB + t) * 64 + lane) * 16, 0, kCoherent));
                    }
                    float w0, w1;
                    fold(u, m1, l1, &w0, &w1);
#pragma unroll
                    for (int t = 0; t < 2 * NB; ++t) o[u][t] = o[u][t] * w0 + x[t] * w1;
                }
            }
            merge_waves();
        }

        if (!idle && (together || wave == 0)) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                if (row0 + 16 * u + i16 >= row1 || (STACK && i16 >= 8)) continue;
                const float inv = 1.0f / l[u];
#pragma unroll
                for (int t = 0; t < 2 * NB; ++t) {
                    const int d = 16 * t + 4 * g;
                    if (d < hd) *reinterpret_cast<f4_t*>(out + out_row[u] + d) = o[u][t] * inv;
                }
            }
        }
    }
}

template <int QT, int NB, int ROWS>
hipError_t launch_rows(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    // recorded launches walk whatever list is set by then: four workgroups a CU
    const unsigned grid = count > 0 ? static_cast<unsigned>(count) * a.kv.n_kv : 1024u;
    attention_kernel<QT, NB, ROWS><<<grid, kThreads, 0, s>>>(a, kind, count, q, out);
    return hipGetLastError();
}

template <int QT, int NB>
hipError_t launch_blocks(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    return kind == 0 ? launch_rows<QT, NB, kKvNarrowRows>(a, kind, count, q, out, s)
                     : launch_rows<QT, NB, NB <= 4 ? 32 : 16>(a, kind, count, q, out, s);
}

template <int QT>
hipError_t launch(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    switch (a.kv.nb) {
        case 1: return launch_blocks<QT, 1>(a, kind, count, q, out, s);
        case 2: return launch_blocks<QT, 2>(a, kind, count, q, out, s);
        case 3: return launch_blocks<QT, 3>(a, kind, count, q, out, s);
        case 4: return launch_blocks<QT, 4>(a, kind, count, q, out, s);
        case 6: return launch_blocks<QT, 6>(a, kind, count, q, out, s);
        case 8: return launch_blocks<QT, 8>(a, kind, count, q, out, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace kv

// One translation unit a type.
hipError_t launch_kv_attention_f32(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_attention_q8_0(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_attention_q4_0(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);
hipError_t launch_kv_attention_q4_1(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s);

}  // namespace mlq
