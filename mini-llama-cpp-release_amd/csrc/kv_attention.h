// Attention of a batch's new tokens over the paged cache (kv_layout.h) on MFMA: what its two
// kernels share, and the one for up to eight query rows a KV head (decode).
//
// out = softmax_j(scale q . k_j) v over the positions j that a token at position i
// sees: j <= i and, with a window of w, j > i - w or j < sinks.
//
// A wave walks tiles of 32 positions of one KV head for up to eight query rows (row =
// token * group + query head of the group, so grouped heads share what is read), the
// four waves of a workgroup every fourth tile each, and workgroups parts of a long context; the
// states are merged in a fixed order, the last workgroup to arrive merging the parts.  Per tile,
// in v_mfma_f32_16x16x32_f16 with operands that come from memory as they lie there:
//
//   S^T = K Q^T   per block b of 32 elements: the codes are whole numbers (exact in
//                 fp16), the queries pairs of fp16 parts hi + lo relative to the block's
//                 largest (2^-22 of it is lost), so a product is exact and the sum
//                 f32; times the block's scale it goes into the score.  A Q4_1 block adds
//                 its minimum times the queries' sum.  f32 keys are split the same way,
//                 relative to the block's power of two: three products.
//   O^T += V^T P^T   the value scale d_jb belongs to key and block, so it goes into the
//                 weights: P_b = p_j d_jb f_b, split into hi + lo, times the codes.
//
// p_j = 2^(t_j - m), t the score in base 2 and m a running maximum of it, a whole number that moves
// only when t passes it by 6; the sum of the weights is f32.  f_b, a power of two of every row and
// block, takes the block's largest p_j d_jb so far to 2^9 .. 2^15: what is large in a block's sum keeps
// all its digits in fp16 (2^-34 of it is lost of a small weight), whatever the values' size and
// whatever other blocks of the head or positions with values of zero hold.  When m moves, f_b takes the
// step up and the accumulators stay; they are rescaled when a weight passes 2^15.
//
// The hi parts are columns 0 .. 7 of the query operand and the lo parts columns 8 .. 15, of
// the weights as well: one product where there would be two, the halves added at the end.
//
// What a row does not see gets weight 0, and 0 times a scale that is Inf or NaN is 0
// (v_mul_legacy_f32); codes are finite always.  A weight that is not 0 times such a scale (or minimum)
// ends as NaN; one that a row sees but that is below f32's range is looked for (`spoilt`).
//
// Bound: memory where the rows of a KV head are few and the contexts fill the chip (64
// sequences of up to 4000 positions, Q8_0, 8 KV heads of 128, four query heads each: 75 us,
// 4.7 TB/s of cache); with 4-bit codes half the bytes take about as many instructions, some
// 625 a tile (75 of them for the blocks' frames and factors).  100 000 positions, Q4_0: 51 us, 2.2 TB/s;
// a wave lives for 31 of them, and vector instructions issue in four fifths of its cycles at two waves a SIMD;
// the rest is the launch and the merge of 64 parts, which takes each wave of the last workgroup 16 trips
// to memory one after the other.  Short contexts: launch, a chain of four trips to
// memory (list, page, tile, parts) and the merge (700 positions 11.4 us).  Two workgroups a CU up to a
// head_dim of 128 (f32: 64), one above; a third (fewer registers, Q4_0, 128) was no faster, and parts beyond one
// round of them slower.
//
// Measured and no faster: a branch that skips the blocks' factors where a query needs none (Q8_0, 64 sequences
// 78 us), the largest scale of a walk kept in a register (84), the first tile's frames found for all blocks at
// once.
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
constexpr int kMostFrame = 126;  // f_b is at most 2^this: what is lost by it is below f32's range
constexpr int kFirstUp = 1000;   // steps of a maximum beyond this are as good as infinite, the first one is
constexpr float kElementLift = 8192.0f;  // f32 elements are split times this over their block's power of two

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
    typedef float f2_t __attribute__((ext_vector_type(2)));
    h2_t h[4], r[4];
    // v - hi as a product with 1, one instruction that takes the fp16 operand as it is
    // (v_fma_mix_f32); a 1 that the compiler knows would make it a conversion and a subtraction.
    float one = 1.0f;
    asm("" : "+s"(one));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = __builtin_convertvector((f2_t{v[2 * j], v[2 * j + 1]}), h2_t);
        const f2_t rest{fmaf(-static_cast<float>(h[j].x), one, v[2 * j]), fmaf(-static_cast<float>(h[j].y), one, v[2 * j + 1])};
        r[j] = __builtin_convertvector(rest, h2_t);
    }
    *hi = join(h[0], h[1], h[2], h[3]);
    *lo = join(r[0], r[1], r[2], r[3]);
}
// The one part a lane has: hi where `low` is 0, lo where it is 1.
__device__ __forceinline__ h8_t split8_one(const float* v, float low) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    h2_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const h2_t h = __builtin_convertvector((f2_t{v[2 * j], v[2 * j + 1]}), h2_t);
        const f2_t rest{fmaf(-static_cast<float>(h.x), low, v[2 * j]), fmaf(-static_cast<float>(h.y), low, v[2 * j + 1])};
        r[j] = __builtin_convertvector(rest, h2_t);
    }
    return join(r[0], r[1], r[2], r[3]);
}
// 1 / s for a power of two s from 2^-80 on; 0 for Inf.
__device__ __forceinline__ float inverse_power(uint32_t s) {
    return bits<float>(static_cast<uint32_t>(max(static_cast<int>(0x7f000000u) - static_cast<int>(s), 0)));
}
// e of a positive v in [2^e, 2^(e+1)); 128 for Inf.
__device__ __forceinline__ int exponent(float v) { return static_cast<int>(__builtin_bit_cast(uint32_t, v) >> 23) - 127; }

__device__ __forceinline__ f4_t mfma(h8_t a, h8_t b, f4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// A lane's part of a query row (elements 8 g .. of every block), relative to the row's largest (EACH: to
// the block's), which becomes 2^13 .. 2^14; the blocks' sums; what takes a score (EACH: a block's part of
// it) to base 2.
// Whether a block of the row is far below the largest (2^-13 of it, and not zeros).
template <int NB, bool EACH>
__device__ __forceinline__ bool load_query(const float* q, int hd, int g, float scale, float (*v)[8], float* sum, float* to_t) {
    float tops[NB], top = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int e = 32 * b + 8 * g;
        float4 x = make_float4(0, 0, 0, 0), y = x;
        if (e < hd) {
            x = *reinterpret_cast<const float4*>(q + e);
            y = *reinterpret_cast<const float4*>(q + e + 4);
        }
        v[b][0] = x.x, v[b][1] = x.y, v[b][2] = x.z, v[b][3] = x.w;
        v[b][4] = y.x, v[b][5] = y.y, v[b][6] = y.z, v[b][7] = y.w;
        tops[b] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) tops[b] = fmaxf(tops[b], fabsf(v[b][j]));
        top = fmaxf(top, tops[b]);
    }
    if (!EACH) top = max_quarters(top);
    bool apart = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        if (!EACH) {
            tops[b] = max_quarters(tops[b]);
            apart = apart || (tops[b] > 0.0f && exponent(tops[b]) < exponent(top) - 13);
        }
        // exponent, kept where 2^(13 - e) is finite and to_t is 2^-112 or more (a row of zeros or nearly: its
        // scores are then as near to 0 as to_t says, and what is taken over to_t stays finite)
        const int log_scale = exponent(fabsf(scale));
        const int e = min(max(exponent(EACH ? max_quarters(tops[b]) : top), max(-110, -99 - log_scale)), 127);
        // a negative scale turns the queries; a score's factor is positive, so that -inf stays -inf
        const float up = ldexpf(scale < 0.0f ? -1.0f : 1.0f, 13 - e);
        if (b == 0 || EACH) to_t[b] = ldexpf(fabsf(scale), e - 13);
        sum[b] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[b][j] *= up;
            sum[b] += v[b][j];
        }
    }
    return apart;
}

// The state of a wave's rows (accumulators, running maximum, sum) in memory, for parts
// of a split that other workgroups merge: written through, read past the caches.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t state_rsrc(float* states, size_t index, int floats) {
    return __builtin_amdgcn_make_buffer_rsrc(states + index * floats, static_cast<short>(0), floats * 4, 0x00020000);
}
template <int NQ, int NB>
__device__ __forceinline__ void leave_state(__amdgpu_buffer_rsrc_t rs, int lane, const f4_t (*o)[2 * NB], const float* m,
                                            const float* l) {
    constexpr int QUADS = NQ * 2 * NB;
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, o[u][t]), rs, ((u * 2 * NB + t) * 64 + lane) * 16, 0,
                                                   kCoherent);
        }
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, m[u]), rs, (QUADS * 256 + 2 * u * 64 + lane) * 4, 0,
                                              kCoherent);
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, l[u]), rs,
                                              (QUADS * 256 + (2 * u + 1) * 64 + lane) * 4, 0, kCoherent);
    }
}
// l 2^d, in halves: d is a difference of scores *and* of f32 values' exponents, and a sum of weights whose
// values are small may be far above 1, so it counts where 2^d itself is below what f32 holds.
__device__ __forceinline__ float down(float l, float d, float* w) {
    const float half = __builtin_amdgcn_exp2f(0.5f * d);
    *w = half * half;
    return l * half * half;
}
// Takes another state of the same rows into one's own.
__device__ __forceinline__ void fold(float& m, float& l, float m1, float l1, float* w0, float* w1) {
    const float to = fmaxf(m, m1);
    l = down(l, m - to, w0) + down(l1, m1 - to, w1);
    m = to;
}
template <int NQ, int NB>
__device__ __forceinline__ void take_state(__amdgpu_buffer_rsrc_t rs, int lane, f4_t (*o)[2 * NB], float* m, float* l) {
    constexpr int QUADS = NQ * 2 * NB;
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        const float m1 = bits<float>(__builtin_amdgcn_raw_buffer_load_b32(rs, (QUADS * 256 + 2 * u * 64 + lane) * 4, 0, kCoherent));
        const float l1 =
            bits<float>(__builtin_amdgcn_raw_buffer_load_b32(rs, (QUADS * 256 + (2 * u + 1) * 64 + lane) * 4, 0, kCoherent));
        f4_t x[2 * NB];
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t) {
            x[t] = __builtin_bit_cast(f4_t,
                                      __builtin_amdgcn_raw_buffer_load_b128(rs, ((u * 2 * NB + t) * 64 + lane) * 16, 0, kCoherent));
        }
        float w0, w1;
        fold(m[u], l[u], m1, l1, &w0, &w1);
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t) o[u][t] = o[u][t] * w0 + x[t] * w1;
    }
}
// One arrival of `parts`: whether it is the last, which leaves the counter at zero.
__device__ __forceinline__ unsigned arrive(unsigned* counter, int parts) {
    const unsigned before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before + 1 != static_cast<unsigned>(parts)) return 0u;
    __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return 1u;
}
// A lane's elements of an output row: 4 g .. of every sixteen.
template <int NB>
__device__ __forceinline__ void store_row(float* out, int hd, int g, const f4_t* o, float inv) {
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t) {
        const int d = 16 * t + 4 * g;
        if (d < hd) *reinterpret_cast<f4_t*>(out + d) = o[t] * inv;
    }
}

template <int QT, int NB>
__global__ __launch_bounds__(kThreads, (QT == 0 ? NB <= 2 : NB <= 4) ? 2 : 1) void attention_kernel(
    KvAttention a, int count, const float* __restrict__ q, float* __restrict__ out) {
    using F = KvForm<QT>;
    constexpr int SB = F::kScaleBytes;
    constexpr int KL = F::key_lane(NB), VL = F::value_lane(NB);
    constexpr int KW = KL / 4, VW = VL / 4;
    constexpr int KS = NB * SB, VS = 2 * NB * SB;  // words of a lane's scales: 4 keys a half tile, 8 keys
    constexpr int STATE = (8 * NB + 2) * 64;       // floats of a wave's state
    __shared__ float merge[2 * STATE];
    __shared__ unsigned last;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const bool low = i16 >= 8;  // the lane's column holds low parts
    const int n_kv = a.kv.n_kv, hd = a.kv.head_dim, heads = n_kv * a.group;
    const int page_tiles = a.kv.page_tiles, tile_shift = __builtin_ctz(page_tiles);
    const int total = (count > 0 ? count : uniform(a.lists.counts + kKvCountNarrow)) * n_kv;

    for (int w = blockIdx.x; w < total; w += gridDim.x) {
        const int head = w % n_kv;
        const KvAttnItem it = uniform(a.lists.items[0] + w / n_kv);
        const int rows = it.new_tokens * a.group, start = it.len - it.new_tokens;
        const int row1 = min(rows, it.row0 + kKvNarrowRows);
        const int pos_lo = start + it.row0 / a.group, pos_hi = start + (row1 - 1) / a.group;
        const int row = min(it.row0 + (i16 & 7), rows - 1);
        const int pos = start + row / a.group;
        const size_t out_row =
            (static_cast<size_t>(it.token0 + row / a.group) * heads + head * a.group + row % a.group) * hd;

        h8_t qs[NB];
        float qsum[NB], to_t[NB];
        {
            float v[NB][8];
            load_query<NB, true>(q + out_row, hd, g, a.scale * (QT == 0 ? 1.0f / kElementLift : 1.0f), v, qsum, to_t);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                h8_t hi, lo;
                split8(v[b], &hi, &lo);
                qs[b] = low ? lo : hi;
                if (QT == 3) qsum[b] = low ? 0.0f : sum_quarters(qsum[b]) * to_t[b];
            }
        }

        const f4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
        f4_t o[1][2 * NB];
        float om[NB];  // Q4_1: this lane's part of the sum of weights times minima
        int frame[NB];  // log2 f_b
        uint32_t spoilt = 0;  // bit b: this lane's part of the row sees a block that is not finite with a weight of 0
        float m = -3.402823466e38f, l = 0.0f;
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t) o[0][t] = zero;
#pragma unroll
        for (int b = 0; b < NB; ++b) om[b] = 0.0f, frame[b] = kMostFrame - kFirstUp;

        // This wave's tiles: every fourth of the item's.
        const int end = it.first + it.count;
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

        // The next tile's loads are under way during this one's work, unless its registers are not enough for both:
        // f32 heads of 256 would keep 2.6 KB a lane in scratch (32 sequences of 4000, 8 KV heads: 1015 us, 399 so).
        constexpr bool AHEAD = QT != 0 || NB <= 4;
        int at = it.first + wave;
        int next_page = 0;
        if (AHEAD && at < end) {
            const uint8_t* tile = base_of(at, page_of(at));
            load_keys(tile);
            load_values(tile);
            if (at + kKvWaves < end) next_page = page_of(at + kKvWaves);
        }
        for (; at < end; at += kKvWaves) {
            const int first = tile_of(at) * kKvTile;
            const bool more = AHEAD && at + kKvWaves < end;
            if (!AHEAD) next_page = page_of(at);
            const uint8_t* next = base_of(more ? at + kKvWaves : at, next_page);
            if (AHEAD && at + 2 * kKvWaves < end) next_page = page_of(at + 2 * kKvWaves);
            if (!AHEAD) load_keys(next);

            // Scores, halves apart.
            float t[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f4_t s = zero;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    f4_t acc;
                    if (QT == 0) {
                        h8_t hi, lo;
                        float v[8];
                        const float inv = inverse_power(kp[h][b]) * kElementLift;
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = mul_or_zero(bits<float>(kw[h][8 * b + j]), inv);
                        split8(v, &hi, &lo);
                        acc = mfma(lo, qs[b], mfma(hi, qs[b], zero));  // (times kElementLift, which to_t takes back)
                    } else if (QT == 1) {
                        acc = mfma(codes8(kw[h][2 * b], kw[h][2 * b + 1], static_cast<_Float16>(128.0f)), qs[b], zero);
                    } else {
                        const uint32_t x = kw[h][b];
                        acc = mfma(codes8(x & 0x0f0f0f0fu, (x >> 4) & 0x0f0f0f0fu, static_cast<_Float16>(QT == 2 ? 8.0f : 0.0f)),
                                   qs[b], zero);
                    }
                    acc *= to_t[b];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[i] = fmaf(scale_at(ks[h], 4 * b + i), acc[i], s[i]);
                        if (QT == 3) s[i] = fmaf(scale_at(km[h], 4 * b + i), qsum[b], s[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) t[4 * h + i] = s[i];
            }
            if (more) load_keys(next);
            if (!AHEAD) load_values(next);

            // Weights.
            const bool full = first + kKvTile - 1 <= pos_lo &&
                              (a.window == 0 || first > pos_hi - a.window || first + kKvTile <= a.sinks);
            auto seen = [&](int j) {
                const int key = first + (j >> 2) * 16 + 4 * g + (j & 3);
                return (key <= pos) & ((a.window == 0) | (key > pos - a.window) | (key < a.sinks));
            };
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                t[j] += other_half(t[j]);
                // an infinite scale (minimum) with codes that are not 0: NaN like the sum of its elements
                if (QT >= 2) t[j] = fmaf(t[j], 0.0f, t[j]);
            }
            if (!full) {
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = seen(j) ? t[j] : -INFINITY;
            }
            float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
            top = max_quarters(top);
            if (__any(top > m + kSlack)) {
                const bool moves = top > m + kSlack;
                const float to = ceilf(top);
                const int up = moves ? static_cast<int>(fminf(to - m, static_cast<float>(kFirstUp))) : 0;
                m = moves ? to : m;
                l = ldexpf(l, -up);
                int over = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    frame[b] += up;
                    over = max(over, frame[b] - kMostFrame);
                    if (QT == 3) om[b] = ldexpf(om[b], -up);
                }
                if (__builtin_expect(__any(over > 0), 0)) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const int less = max(frame[b] - kMostFrame, 0);
                        frame[b] -= less;
#pragma unroll
                        for (int x = 0; x < 2; ++x)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[0][2 * b + x][i] = ldexpf(o[0][2 * b + x][i], -less);
                    }
                }
            }
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = __builtin_amdgcn_exp2f(t[j] - m);
                l += p[j];
            }
            if (__builtin_expect(__any(fminf(fminf(fminf(p[0], p[1]), fminf(p[2], p[3])), fminf(fminf(p[4], p[5]), fminf(p[6], p[7]))) == 0.0f), 0)) {
                // (the largest of all scales and minima tells whether there is anything to look for)
                uint32_t any_bad;
                if (QT == 0) {
                    uint32_t x = vs[0];
#pragma unroll
                    for (int i = 1; i < VS; ++i) x = max(x, vs[i]);
                    any_bad = x >= 0x7f800000u;
                } else {
                    us2_t x{0, 0};
#pragma unroll
                    for (int i = 0; i < VS; ++i) {
                        x = __builtin_elementwise_max(x, bits<us2_t>(vs[i]));
                        if (QT == 3) x = __builtin_elementwise_max(x, bits<us2_t>(vm[QT == 3 ? i : 0] & 0x7fff7fffu));
                    }
                    any_bad = max(x.x, x.y) >= 0x7c00;
                }
                if (__builtin_expect(__any(any_bad != 0), 0)) {
                    auto bad_at = [&](const uint32_t* s, int i) {
                        return QT == 0 ? s[i] >= 0x7f800000u : ((s[i / 2] >> (i % 2 * 16)) & 0x7fffu) >= 0x7c00u;
                    };
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool lost = p[j] == 0.0f && seen(j);
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const bool bad = bad_at(vs, 8 * b + j) || (QT == 3 && bad_at(vm, QT == 3 ? 8 * b + j : 0));
                            spoilt |= (lost && bad ? 1u : 0u) << b;
                        }
                    }
                }
            }

            // Values.
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float v[8];
                h8_t hi, lo;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = mul_or_zero(p[j], scale_at(vs, 8 * b + j));
                float most = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
                if (__builtin_expect(__any(ldexpf(most, frame[b]) > 0x1p15f), 0)) {
                    most = max_quarters(most);
                    const int to = ldexpf(most, frame[b]) > 0x1p15f ? 9 - exponent(most) : frame[b];
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[0][2 * b + x][i] = ldexpf(o[0][2 * b + x][i], to - frame[b]);
                    frame[b] = to;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = ldexpf(v[j], frame[b]);
                const h8_t ps = split8_one(v, low ? 1.0f : 0.0f);
                if (QT == 3) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) om[b] += mul_or_zero(p[j], scale_at(vm, 8 * b + j));
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    f4_t& acc = o[0][2 * b + x];
                    if (QT == 0) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            v[j] = mul_or_zero(bits<float>(vw[16 * b + 8 * x + j]), inverse_power(vs[8 * b + j]) * kElementLift);
                        }
                        split8(v, &hi, &lo);
                        acc = mfma(lo, ps, mfma(hi, ps, acc));
                    } else if (QT == 1) {
                        acc = mfma(codes8(vw[4 * b + 2 * x], vw[4 * b + 2 * x + 1], static_cast<_Float16>(128.0f)), ps, acc);
                    } else {
                        const uint32_t y = vw[2 * b], z = vw[2 * b + 1];
                        acc = mfma(codes8((x == 0 ? y : y >> 4) & 0x0f0f0f0fu, (x == 0 ? z : z >> 4) & 0x0f0f0f0fu,
                                          static_cast<_Float16>(QT == 2 ? 8.0f : 0.0f)), ps, acc);
                    }
                }
            }
            if (more) load_values(next);
        }

        // The lanes' sums, the halves and the minima's part together, out of the blocks' frames.
        l = sum_quarters(l);
        const bool any_spoilt = __any(spoilt != 0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float add = QT == 3 ? sum_quarters(om[b]) : 0.0f;
            add = fmaf(add, 0.0f, add);  // an infinite minimum: NaN
            if (__builtin_expect(any_spoilt, 0)) add += sum_quarters((spoilt >> b) & 1u ? NAN : 0.0f);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = o[0][2 * b + x][i];
                    o[0][2 * b + x][i] = ldexpf(y + other_half(y), -frame[b] - (QT == 0 ? 13 : 0)) + add;
                }
        }
        // The four waves' states into wave 0, in a fixed order.
        auto leave = [&](float* to) {
#pragma unroll
            for (int x = 0; x < 2 * NB; ++x) *reinterpret_cast<f4_t*>(to + (x * 64 + lane) * 4) = o[0][x];
            to[2 * NB * 256 + lane] = m;
            to[2 * NB * 256 + 64 + lane] = l;
        };
        auto take = [&](const float* from) {
            float w0, w1;
            fold(m, l, from[2 * NB * 256 + lane], from[2 * NB * 256 + 64 + lane], &w0, &w1);
#pragma unroll
            for (int x = 0; x < 2 * NB; ++x) {
                o[0][x] = o[0][x] * w0 + *reinterpret_cast<const f4_t*>(from + (x * 64 + lane) * 4) * w1;
            }
        };
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
        merge_waves();

        if (it.nsplit > 1) {
            // This part's state to memory; the workgroup that arrives last merges all parts, wave w
            // taking w, w + 4, ...
            auto rsrc_of = [&](int split) {
                return state_rsrc(a.partial, static_cast<size_t>(it.slot + split) * n_kv + head, STATE);
            };
            const bool live = !low && it.row0 + i16 < row1;  // the lane's column is a row's
            if (wave == 0) {
                if (live) leave_state<1, NB>(rsrc_of(it.split), lane, o, &m, &l);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the state is in memory
                if (lane == 0) last = arrive(a.arrived + static_cast<size_t>(it.slot) * n_kv + head, it.nsplit);
            }
            __syncthreads();
            const bool mine = last != 0u;
            __syncthreads();
            if (!mine) continue;
            m = -3.402823466e38f;
            l = 0.0f;
#pragma unroll
            for (int x = 0; x < 2 * NB; ++x) o[0][x] = zero;
            for (int part = wave; live && part < it.nsplit; part += kKvWaves) take_state<1, NB>(rsrc_of(part), lane, o, &m, &l);
            merge_waves();
        }

        if (wave == 0 && !low && it.row0 + i16 < row1) store_row<NB>(out + out_row, hd, g, o[0], 1.0f / l);
    }
}

}  // namespace kv
}  // namespace mlq
