// The paged attention for many query rows a KV head: chunks of a prompt, whole prompts
// (kv_attention.h has the formula and the kernel for few rows).
//
// A workgroup of four waves takes 4 x 16 NQ rows of one KV head, a wave 16 NQ of them, and walks
// tiles of 32 positions that its waves convert for each other: a tile's keys and values are
// decoded once, and lie in LDS as the MFMA operands they are, split into two fp16 parts
// (hi + lo; 2^-22 of a block's largest is lost, nothing of a Q8_0 or Q4_0 element, which is a code times a
// binary16 scale: at most 19 bits).  Then, all in v_mfma_f32_16x16x32_f16, three products a pair (low parts
// times low parts, 2^-22 of an element, are left out):
//
//   S^T = K Q^T      A from LDS, B (queries, relative to the row's largest) in registers;
//   O^T += V^T P^T   A from LDS, B the weights: a lane's eight scores are its eight weights.
//
// A value block is taken over a power of two of its own for the whole item, and a position's elements over
// one where they are still far from 1, which comes back in the score (2^ek) and in the weight (P_j = p_j 2^ev_j);
// the running maximum is that of t_j + ev_j.  The weights are one operand for all blocks of a head, so this
// holds what the few-row kernel's frames do as long as a position's blocks do not differ too much
// (make_scales); rows that see one where they do become NaN and are done again in plain f32 (plain_rows).
//
// One step a tile and one barrier: products of the last tile's values and this one's keys (96 at
// head_dim 128), then the conversion of the next tile, the loads ahead and the softmax.  Two
// workgroups fit a CU.  Bound: issue and LDS.  A wave's step issues 1540 cycles of products, about
// 290 vector instructions and reads 32 KB of operands from LDS; the matrix cores are busy 37 % of the
// time.  512 tokens of 32 heads after 3500 positions (Q8_0, 8 KV heads of 128): 105 us, 300 TFLOP/s of
// the formula's operations (900 with the parts); a prompt of 2048 in f32, 32 heads: 170 us, 204.
// At head_dim 128 all 256 registers are in use and 35 to 49 more lie in scratch, all but one or two outside of
// the main loop (two there, before one wait for all loads, cost 9 %).
// Keys far from 1 take a sixth longer (125 -> 150 us a call).  Rows in plain f32 take 12 to 30 times as long
// (2.7 ms): one of the last positions' value blocks 1000 times below its others is enough.
// Measured and no faster: those rows by the kernel for few rows' steps, inline (three times the time of all
// rows, for want of registers), in a function (127 us) or in a launch behind (4 us a call); eight waves that
// share a conversion; halves of them in turn on the products and the rest; the products' fences left out;
// several parts of a split in flight in the merge (spills).
#pragma once

#include "kv_attention.h"
#include "quant_device.h"

#include <algorithm>
#include <type_traits>

namespace mlq {
namespace kv {

// Scales of a tile in LDS: what a code (f32: an element) is multiplied by, and, for f32
// arithmetic on quantized codes, what is added then.
template <int QT, int NB>
struct TileScales {
    static constexpr bool kPacked = QT == 1 || QT == 2;  // decoded in packed fp16
    typename std::conditional<kPacked, _Float16, float>::type scale[2][QT == 3 ? 2 : 1][NB][kKvTile];  // keys, values
    float key_up[kKvTile];      // 2^ek
    float value_log[kKvTile];   // ev
    float value_down[kKvTile];  // 2^-ev
    uint8_t bad[NB][kKvTile];   // whether a position's value block is not finite
    uint32_t flags[kKvWaves];   // of the wave's part: kBad, some of `bad`; kFar, some power of two is not 1
};
constexpr uint32_t kBad = 1, kFar = 2;
constexpr float kLift = 256.0f;  // operands lie in LDS times this
constexpr float kWeightLift = 9.0f;  // log2 of what weights are split times, at the running maximum
constexpr int kLeastLog = -90;  // of a position's values over their blocks' powers of two, zeros too (sums of 2^-ev stay finite)
constexpr float kFloor = 0x1p-80f;  // f32: the power of two of a block of zeros, or of elements this small

template <int QT, int NB>
constexpr int rows_lds_bytes() {
    return 2 * 8 * NB * 1024 + 3 * static_cast<int>(sizeof(TileScales<QT, NB>));
}

// Element `i` of a word of codes, times its scale.
template <int QT>
__device__ __forceinline__ float element(uint32_t w, int i, float d, float add) {
    const float c = static_cast<float>(static_cast<int>((w >> (8 * i)) & (QT == 1 ? 0xffu : 0xfu)) - (QT == 1 ? 128 : QT == 2 ? 8 : 0));
    return QT == 3 ? fmaf(c, d, add) : c * d;
}

// Rows of one wave of an item (those of the mask `which`, from row_base on), in plain f32: what a wave of
// attention_rows_kernel does where blocks of a position that the row sees or of its query differ too much in size for
// its operands.  Four rows at a time; a lane takes one position's half of every block for the scores, every 64th dimension for
// the values.  In few registers: the kernel's own are not touched by it.  lds: the wave's, 4 (32 NB + 32) floats.
template <int QT, int NB, int NQ>
__device__ __forceinline__ void plain_rows(const KvAttention& a, const KvAttnItem& it, int head, int row_base, uint32_t which, int wave,
                                           int lane, const float* __restrict__ q, float* __restrict__ out, float* lds) {
    using F = KvForm<QT>;
    constexpr int KL = F::key_lane(NB), VL = F::value_lane(NB), HD = 32 * NB, DIMS = (HD + 63) / 64;
    constexpr int QUADS = NQ * 2 * NB, STATE = (QUADS * 4 + 2 * NQ) * 64;
    const int hd = a.kv.head_dim, n_kv = a.kv.n_kv, heads = n_kv * a.group;
    const int rows = it.new_tokens * a.group, start = it.len - it.new_tokens;
    const int page_tiles = a.kv.page_tiles, tile_shift = __builtin_ctz(page_tiles);
    // (opaque here, or what depends on it would be computed ahead of the kernel's loop, in registers that it needs)
    asm volatile("" : "+v"(lane));
    float* const weights = lds + 4 * HD;  // [position][row]
    auto over_lanes = [](float x, auto two) {  // of 32: both halves of the wave have the same
#pragma unroll
        for (int s = 1; s < 32; s *= 2) x = two(x, __shfl_xor(x, s));
        return x;
    };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto plus = [](float x, float y) { return x + y; };
    auto in_order = [] {  // what the wave has written to LDS is there for all its lanes
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    auto scale_of = [](const uint8_t* plane, int i) {
        return QT == 0 ? reinterpret_cast<const float*>(plane)[i] : half_value(reinterpret_cast<const uint16_t*>(plane)[i]);
    };
#pragma unroll 1
    for (int r = 0; r < 16 * NQ; r += 4) {
        if ((which >> r & 15u) == 0) continue;
        // Queries over the power of two of the row's largest; a score's factor to base 2.
        float to_t[4], m[4], l[4], acc[DIMS][4];
        int pos[4];
        size_t at[4];
        in_order();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int row = min(row_base + r + k, rows - 1);
            pos[k] = start + row / a.group;
            at[k] = (static_cast<size_t>(it.token0 + row / a.group) * heads + head * a.group + row % a.group) * hd;
            float x[DIMS], top = 0.0f;
#pragma unroll
            for (int c = 0; c < DIMS; ++c) {
                const int e = lane + 64 * c;
                x[c] = e < hd ? q[at[k] + e] : 0.0f;
                top = fmaxf(top, fabsf(x[c]));
            }
            top = over_lanes(top, larger);
            top = fmaxf(top, __shfl_xor(top, 32));
            const int e = min(max(exponent(top), -120), 127);
            to_t[k] = ldexpf(a.scale, e);
#pragma unroll
            for (int c = 0; c < DIMS; ++c) {
                if (lane + 64 * c < HD) lds[k * HD + lane + 64 * c] = ldexpf(x[c], -e);
                acc[c][k] = 0.0f;
            }
            m[k] = -3.402823466e38f;
            l[k] = 0.0f;
        }
        in_order();
#pragma unroll 1
        for (int i = it.first; i < it.first + it.count; ++i) {
            const int t = i < it.sinks ? i : i + it.shift;
            const int page = uniform(&a.lists.pages[it.page0 + (t >> tile_shift)].page);
            const uint8_t* const tile =
                a.kv.base + ((static_cast<size_t>(page) * n_kv + head) * page_tiles + (t & (page_tiles - 1))) * F::tile(NB);
            // Scores: this lane's position, half of every block's elements.
            const int slot = lane & 31, key = t * kKvTile + slot;
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            bool bad_value = false;
#pragma unroll 1
            for (int x = 0; x < 2 * NB; ++x) {
                const int b = x >> 1, g = (lane >> 5) * 2 + (x & 1);
                const uint8_t* const from = tile + (slot >> 4) * 64 * KL;
                const int of_lane = 16 * g + (slot & 15);
                float d = scale_of(tile + F::codes(NB), F::key_scale(NB, slot, b)), y[8];
                if (QT == 0) {
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const f4_t four = *reinterpret_cast<const f4_t*>(from + F::at(KL, of_lane, b * 32 + 16 * z));
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[4 * z + e] = d < INFINITY ? four[e] : NAN;
                    }
                } else {
                    const float add = QT == 3 ? scale_of(tile + F::codes(NB) + F::plane(NB), F::key_scale(NB, slot, b)) : 0.0f;
                    const uint8_t* const p = from + F::at(KL, of_lane, b * F::kElemBits);
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const uint32_t w = QT == 1 ? reinterpret_cast<const uint32_t*>(p)[z] : *reinterpret_cast<const uint32_t*>(p) >> (4 * z);
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[4 * z + e] = element<QT>(w, e, d, add);
                    }
                }
                d = scale_of(tile + F::half(NB) + F::codes(NB), F::value_scale(NB, slot, b));
                bad_value = bad_value || !(d < INFINITY);
                if (QT == 3) {
                    d = scale_of(tile + F::half(NB) + F::codes(NB) + F::plane(NB), F::value_scale(NB, slot, b));
                    bad_value = bad_value || !(fabsf(d) < INFINITY);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f4_t* const of_row = reinterpret_cast<const f4_t*>(lds + k * HD + 32 * b + 8 * g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[k] = fmaf(of_row[e >> 2][e & 3], y[e], s[k]);
                }
            }
            // Weights.
            f4_t p;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float x = (s[k] + __shfl_xor(s[k], 32)) * to_t[k];
                x = fmaf(x, 0.0f, x);  // an infinite scale: NaN
                const bool seen = key <= pos[k] && (a.window == 0 || key > pos[k] - a.window || key < a.sinks);
                x = seen ? x : -INFINITY;
                const float to = fmaxf(m[k], over_lanes(x, larger)), c = __builtin_amdgcn_exp2f(m[k] - to);
                m[k] = to;
                p[k] = __builtin_amdgcn_exp2f(x - to);
                l[k] = l[k] * c + over_lanes(p[k], plus);
                // (a block that is not finite counts however small its weight)
                if (bad_value && seen) p[k] = fmaxf(p[k], 0x1p-126f);
#pragma unroll
                for (int z = 0; z < DIMS; ++z) acc[z][k] *= c;
            }
            in_order();
            if (lane < 32) *reinterpret_cast<f4_t*>(weights + 4 * slot) = p;
            in_order();
            // Values: four positions of a dimension share a word.
#pragma unroll
            for (int c = 0; c < DIMS; ++c) {
                const int dim = min(lane + 64 * c, HD - 1), b = dim >> 5, side = (dim >> 4) & 1;
#pragma unroll 1
                for (int quad = 0; quad < 8; ++quad) {
                    const uint8_t* const from = tile + F::half(NB);
                    const int of_lane = 16 * (quad & 3) + (dim & 15), x = side * 8 + (quad >> 2) * 4;
                    const int first_scale = F::value_scale(NB, 4 * quad, b);
                    f4_t y;
                    uint32_t w = 0;
                    if (QT == 0) y = *reinterpret_cast<const f4_t*>(from + F::at(VL, of_lane, (b * 16 + x) * 4));
                    else if (QT == 1) w = *reinterpret_cast<const uint32_t*>(from + F::at(VL, of_lane, b * 16 + x));
                    else w = *reinterpret_cast<const uint32_t*>(from + F::at(VL, of_lane, b * 8 + (x & 7))) >> (4 * side);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float d = scale_of(from + F::codes(NB), first_scale + e);
                        const float add = QT == 3 ? scale_of(from + F::codes(NB) + F::plane(NB), first_scale + e) : 0.0f;
                        float v = QT == 0 ? y[e] : element<QT>(w, e, d, add);
                        if (!(d < INFINITY) || !(fabsf(add) < INFINITY)) v = NAN;
                        const f4_t of_rows = *reinterpret_cast<const f4_t*>(weights + 4 * (4 * quad + e));
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[c][k] += mul_or_zero(of_rows[k], v);
                    }
                }
            }
        }
        // The output, or the state as leave_state lays it out, in the units of the others (weights times 2^kWeightLift,
        // values times kLift).
        const __amdgpu_buffer_rsrc_t rs =
            state_rsrc(a.partial, (static_cast<size_t>(it.slot + it.split) * n_kv + head) * kKvWaves + wave, STATE);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if ((which >> (r + k) & 1u) == 0) continue;
            const int u = (r + k) >> 4, column = (r + k) & 15;
#pragma unroll
            for (int c = 0; c < DIMS; ++c) {
                const int dim = lane + 64 * c;
                if (it.nsplit == 1) {
                    if (dim < hd) out[at[k] + dim] = acc[c][k] / l[k];
                } else if (dim < HD) {
                    const int of_lane = column + 16 * ((dim & 15) >> 2);
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, acc[c][k] * kLift), rs,
                                                          ((u * 2 * NB + (dim >> 4)) * 64 + of_lane) * 16 + (dim & 3) * 4, 0, kCoherent);
                }
            }
            if (it.nsplit > 1 && lane < 4) {
                const int of_lane = column + 16 * lane;
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, m[k] + kWeightLift), rs,
                                                      (QUADS * 256 + 2 * u * 64 + of_lane) * 4, 0, kCoherent);
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, l[k]), rs,
                                                      (QUADS * 256 + (2 * u + 1) * 64 + of_lane) * 4, 0, kCoherent);
            }
        }
    }
}

template <int QT, int NB, int NQ>
__global__ __launch_bounds__(kThreads, 2) void attention_rows_kernel(KvAttention a, int count, const float* __restrict__ q,
                                                                      float* __restrict__ out) {
    using F = KvForm<QT>;
    using Scales = TileScales<QT, NB>;
    constexpr int KL = F::key_lane(NB), VL = F::value_lane(NB);
    constexpr int FRAGS = 2 * NB;                          // operands of keys, of values (hi or lo) a tile
    constexpr int TASKS = (FRAGS + kKvWaves - 1) / kKvWaves;  // of either, per wave
    constexpr int RAW_K = QT == 0 ? 8 : QT == 1 ? 2 : 1, RAW_V = QT == 0 ? 8 : 2;  // words a lane loads for an operand
    constexpr int QUADS = NQ * 2 * NB, STATE = (QUADS * 4 + 2 * NQ) * 64;
    constexpr int ROWS = 16 * NQ;
    constexpr int PER = NB <= 4 ? 4 : 8, PASSES = 2 * kKvTile * PER / (kThreads);  // threads a position's scales, rounds of them
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // [buffer][key hi, key lo, value hi, value lo][operand][lane] of 16 bytes, then the scales
    h8_t* const operands = reinterpret_cast<h8_t*>(lds);
    Scales* const scales = reinterpret_cast<Scales*>(lds + 2 * 8 * NB * 1024);
    auto operand = [&](int buffer, int part, int f) { return operands + ((buffer * 4 + part) * FRAGS + f) * 64; };
    __shared__ unsigned last;
    __shared__ float block_tops[kKvWaves][PER];  // the largest of the first tile's values, by wave that looked
    __shared__ int item_range[2];  // positions of the item's rows (in LDS, as few tiles ask for them)

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int n_kv = a.kv.n_kv, hd = a.kv.head_dim, heads = n_kv * a.group;
    const int page_tiles = a.kv.page_tiles, tile_shift = __builtin_ctz(page_tiles);
    const int total = (count > 0 ? count : uniform(a.lists.counts + kKvCountWide)) * n_kv;

    // What this thread loads of a tile: a task is one operand of keys and one of values, both parts.
    auto mine = [&](int x) { return FRAGS % kKvWaves == 0 || wave + kKvWaves * (x >> 1) < FRAGS; };
    // (Task k's offsets are those of task 0 and a constant, for keys where the waves share out whole halves: a register each.)
    constexpr bool WHOLE = NB % kKvWaves == 0;
    uint32_t key_off[WHOLE ? 1 : TASKS], scale_off[PASSES];
#pragma unroll
    for (int k = 0; k < (WHOLE ? 1 : TASKS); ++k) {
        const int f = wave + kKvWaves * k, h = f / NB, b = f % NB;
        key_off[k] = WHOLE ? F::at(KL, lane, wave * F::kElemBits) : h * 64 * KL + F::at(KL, lane, b * F::kElemBits);
    }
    auto key_at = [&](const uint8_t* tile, int k) {
        const int b = kKvWaves * k;  // of task k, less the wave
        return WHOLE ? tile + key_off[0] + (b / NB * 64 * KL + F::at(KL, 0, b % NB * F::kElemBits)) : tile + key_off[WHOLE ? 0 : k];
    };
    const uint32_t value_off = F::half(NB) + F::at(VL, lane, (QT < 2 ? wave : wave & ~1) * F::kElemBits);
    auto value_at = [&](const uint8_t* tile, int k) { return tile + value_off + F::at(VL, 0, kKvWaves * k * F::kElemBits); };
#pragma unroll
    for (int z = 0; z < PASSES; ++z) {
        const int block = min(static_cast<int>(threadIdx.x % PER), NB - 1), item = (threadIdx.x + z * (kThreads)) / PER;
        const int key = item % kKvTile;
        scale_off[z] = (item >= kKvTile ? F::half(NB) : 0) + F::codes(NB) +
                       (item >= kKvTile ? F::value_scale(NB, key, block) : F::key_scale(NB, key, block)) * F::kScaleBytes;
    }

    for (int w = blockIdx.x; w < total; w += gridDim.x) {
        const int head = w % n_kv;
        const KvAttnItem it = uniform(a.lists.items[1] + w / n_kv);
        const int rows = it.new_tokens * a.group, start = it.len - it.new_tokens;
        const int row0 = it.row0 + wave * ROWS, row1 = min(rows, row0 + ROWS);
        const bool idle = row0 >= rows;
        const int pos_lo = start + min(row0, rows - 1) / a.group, pos_hi = start + (row1 - 1) / a.group;

        h8_t qh[NQ][NB], ql[NQ][NB];
        float to_t[NQ];
        int pos[NQ];
        // This lane's row u of the batch, and where its elements start.
        auto token_of = [&](int u) { return min(row0 + 16 * u + i16, rows - 1) / a.group; };
        auto element_of = [&](int u) {
            const int r = min(row0 + 16 * u + i16, rows - 1);
            return (static_cast<size_t>(it.token0 + r / a.group) * heads + head * a.group + r % a.group) * hd;
        };
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            pos[u] = start + token_of(u);
            float v[NB][8], sum[NB];
            const bool apart = load_query<NB, false>(q + element_of(u), hd, g, a.scale * (1.0f / kLift), v, sum, &to_t[u]);
            if (apart) to_t[u] = NAN;  // (the row is done in plain f32: below)
#pragma unroll
            for (int b = 0; b < NB; ++b) split8(v[b], &qh[u][b], &ql[u][b]);
        }

        f4_t o[NQ][2 * NB];
        float m[NQ], l[NQ];
        const f4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            m[u] = -3.402823466e38f;
            l[u] = 0.0f;
#pragma unroll
            for (int t = 0; t < 2 * NB; ++t) o[u][t] = zero;
        }

        // Tiles counted from the item's first; those past the end repeat the last one: loads stay in
        // bounds, nothing uses them.
        auto tile_of = [&](int i) {
            const int k = it.first + min(i, it.count - 1);
            return k < it.sinks ? k : k + it.shift;
        };
        // (A vector load: one through the scalar cache would make every wait for LDS a wait for all of it.)
        auto page_of = [&](int i) { return a.lists.pages[it.page0 + (tile_of(i) >> tile_shift)].page; };
        // (And the address by vector arithmetic: there is no other wave to hide a chain of scalar steps.)
        const uint8_t* const head_base = a.kv.base + static_cast<size_t>(head) * page_tiles * F::tile(NB);
        const uint32_t page_bytes = static_cast<uint32_t>(page_tiles) * F::tile(NB);
        auto address_of = [&](int i, int page) -> const uint8_t* {
            const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(page) * static_cast<uint64_t>(n_kv)) * page_bytes;
            return head_base + at + static_cast<uint32_t>((tile_of(i) & (page_tiles - 1)) * F::tile(NB));
        };

        // Loads of a tile: this wave's operands, and the scale of one (keys or values, position, block)
        // a thread.
        uint32_t raw_k[TASKS][RAW_K], raw_v[TASKS][RAW_V];
        uint32_t raw_s[PASSES][F::kPlanes];
        auto load_keys = [&](const uint8_t* tile) {
#pragma unroll
            for (int k = 0; k < TASKS; ++k) {
                if (!mine(2 * k)) continue;
                const uint8_t* p = key_at(tile, k);
                if (QT == 0) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {  // the lane's two units
                        const u4_t k4 = *reinterpret_cast<const u4_t*>(p + x * 1024);
#pragma unroll
                        for (int i = 0; i < 4; ++i) raw_k[k][(4 * x + i) & (RAW_K - 1)] = k4[i];
                    }
                } else if (QT == 1) {
                    const uint2 k2 = *reinterpret_cast<const uint2*>(p);
                    raw_k[k][0] = k2.x, raw_k[k][RAW_K - 1] = k2.y;
                } else {
                    raw_k[k][0] = *reinterpret_cast<const uint32_t*>(p);
                }
            }
        };
        auto load_values = [&](const uint8_t* tile) {
#pragma unroll
            for (int k = 0; k < TASKS; ++k) {
                if (!mine(2 * k)) continue;
                const uint8_t* p = value_at(tile, k);
                if (QT == 0) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const u4_t v4 = *reinterpret_cast<const u4_t*>(p + x * 1024);
#pragma unroll
                        for (int i = 0; i < 4; ++i) raw_v[k][(4 * x + i) & (RAW_V - 1)] = v4[i];
                    }
                } else {
                    const uint2 v2 = *reinterpret_cast<const uint2*>(p);
                    raw_v[k][0] = v2.x, raw_v[k][1] = v2.y;
                }
            }
        };
        auto load_scales = [&](const uint8_t* tile) {
#pragma unroll
            for (int z = 0; z < PASSES; ++z)
#pragma unroll
                for (int x = 0; x < F::kPlanes; ++x) {
                    const uint8_t* p = tile + scale_off[z] + x * F::plane(NB);
                    raw_s[z][x] = QT == 0 ? *reinterpret_cast<const uint32_t*>(p) : *reinterpret_cast<const uint16_t*>(p);
                }
        };
        auto over_blocks = [&](float x, auto two) {  // over a position's blocks, PER lanes in a row
            x = two(x, quad_peer<0xB1>(x));
            x = two(x, quad_peer<0x4E>(x));
            if (PER == 8) x = two(x, quad_peer<0x141>(x));  // (the mirror of eight lanes)
            return x;
        };
        auto slot_of = [](int i) { return i % 3; };  // of tile i's scales
        // log2 of a block's power of two for values: of its largest in the first tile, -20 .. 20 (what is beyond that,
        // in f32's range, stays so over it).  A block of zeros there beside others (`asleep`: padded heads) is taken to stay so.
        // (In f32 it may hold elements up to kFloor: over 2^-74 they are operands up to 2^3 (times 2^-ev), and 2^-100 is far
        // above what operands lose, 2^-25.)
        constexpr float kZeros = QT == 0 ? kFloor : 0.0f;  // a block of zeros, or nearly
        auto first_top = [&](int b) {
            return fmaxf(fmaxf(block_tops[0][b], block_tops[1][b]), fmaxf(block_tops[2][b], block_tops[3][b]));
        };
        auto block_exponent = [&](float top, bool block_asleep) {
            return block_asleep ? (QT == 0 ? -74 : 0) : top > 0.0f ? min(max(exponent(top), -20), 20) : 0;
        };
        float value_unit;  // one over it, of the block whose scales this thread makes
        bool asleep;
        // A position, a block and a bound of the block's elements, within a factor of 3; whether a row of the item sees it.
        auto size_of = [&](float d, float add) {
            return QT == 0 ? d : QT == 3 ? fmaf(16.0f, d, fabsf(add)) : (QT == 1 ? 128.0f : 8.0f) * d;
        };
        auto scale_in = [&](const uint32_t* raw, int plane) {
            return QT == 0 ? bits<float>(raw[0]) : half_value(static_cast<uint16_t>(raw[F::kPlanes == 2 ? plane : 0]));
        };
        auto seen_by_some = [&](int i, int key) {
            const int at = tile_of(i) * kKvTile + key;
            return at <= item_range[1] && (a.window == 0 || at > item_range[0] - a.window || at < a.sinks);
        };
        // Scales to LDS.  Operands lie there times 2^8 and over a power of two per position, so that what they lose,
        // 2^-25, is 2^-22 of every block's largest, and none reaches 2^15.  Keys: 1 where all blocks are of sizes from
        // 2^-10 to 2^7, else what brings the largest to [2^5, 2^6), which serves blocks from 2^-14 of it on; a block of
        // zeros adds nothing and loses nothing.  Values are first taken over the block's own power of two, that of its
        // largest in the item's first tile; then 1 where all blocks are from 2^-7 to 2^3, else
        // what brings the largest to [2^2, 2^3), which serves blocks from 2^-9 of it on.  (The range is narrow as a weight
        // keeps 2^-34 of the row's largest: a position that has that one then has values of at least 2^-10 of any
        // other's.)  What else there is, a value's block of zeros beside others too unless it is asleep, leaves the rows
        // that see it to plain_rows.
        // Positions that no row of the item sees are zeros.
        auto make_scales = [&](int i) {
            Scales* const s = scales + slot_of(i);
            using T = typename std::remove_reference<decltype(s->scale[0][0][0][0])>::type;
            uint32_t flags = 0;
#pragma unroll
            for (int z = 0; z < PASSES; ++z) {
                const int block = threadIdx.x % PER, item = (threadIdx.x + z * (kThreads)) / PER;
                const bool values = (wave * 64 + z * (kThreads)) / PER >= kKvTile;  // a wave has one or the other
                const int key = item % kKvTile;
                const float d = scale_in(raw_s[z], 0), add = QT == 3 ? scale_in(raw_s[z], 1) : 0.0f;
                const float unit = values ? value_unit : 1.0f;
                const float size = size_of(d, add) * unit;  // (lanes past the last block repeat it)
                float lift = kLift * unit;
                int e = 0;
                bool bad = false, nothing = false, uneven = false;
                const float high = values ? 0x1p3f : 0x1p7f, low = values ? 0x1p-7f : 0x1p-10f;
                const bool quiet = 32 * block >= hd || (QT != 0 && size == 0.0f && (!values || asleep));
                if (__builtin_expect(!__all((size >= low && size < high) || quiet), 0)) {
                    nothing = !seen_by_some(i, key);
                    bad = !nothing && !(size_of(d, add) < INFINITY);
                    const bool zeros = size_of(d, add) <= kZeros, rests = values && asleep;
                    const bool real = !nothing && !bad && 32 * block < hd, counts = real && !rests;
                    const float top = over_blocks(counts ? size : 0.0f, [](float x, float y) { return fmaxf(x, y); });
                    // 1: a block is asleep, 2: and wakes, which makes the position uneven
                    const float sleeps = over_blocks(real && rests ? (zeros ? 1.0f : 2.0f) : 0.0f, [](float x, float y) { return fmaxf(x, y); });
                    const float least = over_blocks(counts && !zeros ? size : INFINITY, [](float x, float y) { return fminf(x, y); });
                    const float any_zeros = over_blocks(counts && zeros ? 1.0f : 0.0f, [](float x, float y) { return fmaxf(x, y); });
                    // (no block that counts leaves the infinity; where all are zeros the power of two is far below the others')
                    const bool all_zeros = least == INFINITY && any_zeros != 0.0f;
                    const bool near = values ? least >= low && top < high && any_zeros == 0.0f
                                             : top == 0.0f || (least >= low && top < high && !(QT == 0 && all_zeros));
                    const bool even = least >= top * (values ? 0x1p-9f : 0x1p-14f) && (!values || any_zeros == 0.0f || all_zeros);
                    e = near ? 0 : values ? max(exponent(top) - 2, kLeastLog) : exponent(top) - 5;
                    // (elements up to kFloor of a block asleep: below 2^15 from 2^-12 on, held to 2^-100 up to 2^6)
                    uneven = !(near || even) || sleeps == 2.0f || (QT == 0 && sleeps != 0.0f && (e < -12 || e > 6));
                    if (uneven) e = 0;
                    lift = ldexpf(kLift * unit, -e);
                    flags |= (__any(e != 0 || bad || uneven) ? kFar : 0u) | (values && __any(bad) ? kBad : 0u);
                }
                if (block == 0) {
                    // (the scores of an uneven position are NaN)
                    (values ? s->value_down : s->key_up)[key] = uneven && !values ? NAN : ldexpf(1.0f, values ? -e : e);
                    if (values) s->value_log[key] = uneven ? NAN : static_cast<float>(e);
                }
                if (block < NB) {
                    // keys: NaN through to the score; values: zero here, NaN for the rows that see it (`bad`)
                    const bool other = bad || nothing || uneven || !(lift < INFINITY);
                    const float instead = values || !bad ? 0.0f : NAN;
                    if (values) s->bad[block][key] = bad;
                    s->scale[values][0][block][key] = static_cast<T>(other ? instead : QT == 0 ? lift : d * lift);
                    if (QT == 3) s->scale[values][QT == 3 ? 1 : 0][block][key] = static_cast<T>(other ? instead : add * lift);
                }
            }
            if (lane == 0) s->flags[wave] = flags;
        };
        // Eight codes as fp16 (minus the stored offset): keys, values (`t`: which nibbles).
        auto codes_of = [&](const uint32_t* raw, bool values, int t) -> h8_t {
            if (QT == 1) return codes8(raw[0], raw[RAW_K - 1], static_cast<_Float16>(128.0f));
            const _Float16 off = static_cast<_Float16>(QT == 2 ? 8.0f : 0.0f);
            if (values) return codes8((raw[0] >> (4 * t)) & 0x0f0f0f0fu, (raw[1] >> (4 * t)) & 0x0f0f0f0fu, off);
            return codes8(raw[0] & 0x0f0f0f0fu, (raw[0] >> 4) & 0x0f0f0f0fu, off);
        };
        // A tile's conversion in SLICES steps, two an operand pair (task): keys, values.  `begin` reads
        // a step's scales, `finish` decodes, splits and stores.
        constexpr int SLICES = 2 * TASKS;
        typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
        struct SliceScales {
            _Float16 d16;
            h4_t v16[2];
            float d, add;
            f4_t v[2], vadd[2];
        };
        auto begin = [&](int x, const Scales* s, SliceScales& c) {
            if (!mine(x)) return;
            const int f = wave + kKvWaves * (x >> 1);
            const int h = f / NB, b = f % NB, bv = f >> 1;
            if (x % 2 == 0) {
                if constexpr (Scales::kPacked) {
                    c.d16 = s->scale[0][0][b][16 * h + i16];
                } else {
                    c.d = s->scale[0][0][b][16 * h + i16];
                    if (QT == 3) c.add = s->scale[0][QT == 3 ? 1 : 0][b][16 * h + i16];
                }
            } else {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    if constexpr (Scales::kPacked) {
                        c.v16[y] = *reinterpret_cast<const h4_t*>(s->scale[1][0][bv] + 16 * y + 4 * g);
                    } else {
                        c.v[y] = *reinterpret_cast<const f4_t*>(s->scale[1][0][bv] + 16 * y + 4 * g);
                        if (QT == 3) c.vadd[y] = *reinterpret_cast<const f4_t*>(s->scale[1][QT == 3 ? 1 : 0][bv] + 16 * y + 4 * g);
                    }
                }
            }
        };
        auto finish = [&](int x, int buffer, const SliceScales& c) {
            if (!mine(x)) return;
            const int k = x >> 1, f = wave + kKvWaves * k, t = f & 1;
            const bool values = x % 2 != 0;
            h8_t hi, lo;
            if constexpr (Scales::kPacked) {
                // code times scale: at most 19 bits, so hi and what is left of it are exact
                const h8_t d = values ? __builtin_shufflevector(c.v16[0], c.v16[1], 0, 1, 2, 3, 4, 5, 6, 7)
                                      : h8_t{c.d16, c.d16, c.d16, c.d16, c.d16, c.d16, c.d16, c.d16};
                const h8_t code = values ? codes_of(raw_v[k], true, t) : codes_of(raw_k[k], false, 0);
                hi = code * d;
                lo = __builtin_elementwise_fma(code, d, -hi);
            } else {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (QT == 0) {
                        y[j] = values ? mul_or_zero(bits<float>(raw_v[k][j & (RAW_V - 1)]), c.v[j >> 2][j & 3])
                                      : bits<float>(raw_k[k][j & (RAW_K - 1)]) * c.d;
                    } else {
                        const uint32_t nibbles = values ? raw_v[k][(j >> 2) & (RAW_V - 1)] >> (4 * t) : raw_k[k][0] >> (4 * (j >> 2));
                        const float code = static_cast<float>(((nibbles & 0x0f0f0f0fu) >> (8 * (j & 3))) & 0xffu);
                        y[j] = values ? fmaf(code, c.v[j >> 2][j & 3], c.vadd[j >> 2][j & 3]) : fmaf(code, c.d, c.add);
                    }
                }
                split8(y, &hi, &lo);
            }
            operand(buffer, values ? 2 : 0, f)[lane] = hi;
            operand(buffer, values ? 3 : 1, f)[lane] = lo;
        };

        auto barrier = [] {
            __builtin_amdgcn_sched_barrier(0);  // a step's vector work stays out of the other's
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
            __builtin_amdgcn_sched_barrier(0);
        };
        // Converts the keys of tile i + 1 and the values of tile i, and loads those of the next.
        auto convert_begin = [&](int i, SliceScales* c) {
#pragma unroll
            for (int x = 0; x < SLICES; ++x) begin(x, scales + slot_of(x % 2 == 0 ? i + 1 : i), c[x]);
        };
        auto convert_finish = [&](int i, const SliceScales* c, int page1, int page2) {
#pragma unroll
            for (int x = 0; x < SLICES; ++x) finish(x, x % 2 == 0 ? (i + 1) & 1 : i & 1, c[x]);
            load_keys(address_of(i + 2, page2));
            load_values(address_of(i + 1, page1));
        };

        // Fill the pipeline: scales of tiles 0 and 1 (counted from the item's first), keys of 0.
        if (threadIdx.x == 0) {
            item_range[0] = start + it.row0 / a.group;
            item_range[1] = start + (min(rows, it.row0 + kKvWaves * ROWS) - 1) / a.group;
        }
        __syncthreads();  // the last item's readers are done
        load_scales(address_of(0, page_of(0)));
        load_keys(address_of(0, page_of(0)));
        // The blocks' powers of two for values.
        {
            float top = 0.0f;
#pragma unroll
            for (int z = 0; z < PASSES; ++z) {
                const int block = threadIdx.x % PER, item = (threadIdx.x + z * (kThreads)) / PER;
                const float size = size_of(scale_in(raw_s[z], 0), QT == 3 ? scale_in(raw_s[z], 1) : 0.0f);
                if (item >= kKvTile && 32 * block < hd && size < INFINITY && seen_by_some(0, item % kKvTile)) top = fmaxf(top, size);
            }
            // over the wave's positions (row_ror)
            if (PER == 4) top = fmaxf(top, quad_peer<0x124>(top));
            top = max_quarters(fmaxf(top, quad_peer<0x128>(top)));
            if (lane < PER) block_tops[wave][lane] = top;
        }
        __syncthreads();
        {
            const float top = first_top(threadIdx.x % PER);
            const float any = over_blocks(top, [](float x, float y) { return fmaxf(x, y); });
            asleep = top <= kZeros && any > kZeros;
            value_unit = ldexpf(1.0f, -block_exponent(top, asleep));
        }
        // what the first step takes for the values of a tile before the first
        for (int f = wave; f < 2 * FRAGS; f += kKvWaves) operand(1, 2 + f / FRAGS, f % FRAGS)[lane] = h8_t{0, 0, 0, 0, 0, 0, 0, 0};
        make_scales(0);
        load_scales(address_of(1, page_of(1)));
        make_scales(1);
        load_scales(address_of(2, page_of(2)));
        __syncthreads();
#pragma unroll
        for (int x = 0; x < SLICES; x += 2) {
            SliceScales c;
            begin(x, scales + 0, c);
            finish(x, 0, c);
        }
        load_keys(address_of(1, page_of(1)));
        load_values(address_of(0, page_of(0)));
        __syncthreads();

        f4_t sc[NQ][2];
        h8_t ph[NQ], pl[NQ];
        uint32_t spoilt = 0;  // this lane's part: bit u NB + b
#pragma unroll
        for (int u = 0; u < NQ; ++u) ph[u] = pl[u] = h8_t{0, 0, 0, 0, 0, 0, 0, 0};
        // The products of a step: NB blocks of values of tile i - 1 (in the first step zeros times zeros) and, if
        // `keys`, NB of keys of tile i; a block's operands are read a block ahead (the fences keep it so).
        auto products = [&](bool keys, int i) {
            h8_t frag[2][4];
            auto read = [&](int x) {  // x: 0 .. NB - 1 values, NB .. 2 NB - 1 keys
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    frag[x & 1][y] = x < NB ? operand((i + 1) & 1, 2 + (y >> 1), 2 * x + (y & 1))[lane]
                                            : operand(i & 1, y >> 1, (y & 1) * NB + x - NB)[lane];
                }
            };
            __builtin_amdgcn_s_setprio(1);
            read(0);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b + 1 < NB || keys) read(b + 1);
                __builtin_amdgcn_sched_barrier(0);
                const h8_t* v = frag[b & 1];
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    o[u][2 * b] = mfma(v[0], ph[u], o[u][2 * b]), o[u][2 * b + 1] = mfma(v[1], ph[u], o[u][2 * b + 1]);
                }
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    o[u][2 * b] = mfma(v[0], pl[u], o[u][2 * b]), o[u][2 * b + 1] = mfma(v[1], pl[u], o[u][2 * b + 1]);
                }
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    o[u][2 * b] = mfma(v[2], ph[u], o[u][2 * b]), o[u][2 * b + 1] = mfma(v[3], ph[u], o[u][2 * b + 1]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (keys) {
#pragma unroll
                for (int u = 0; u < NQ; ++u) sc[u][0] = sc[u][1] = zero;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (b + 1 < NB) read(NB + b + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    const h8_t* k = frag[(NB + b) & 1];
#pragma unroll
                    for (int u = 0; u < NQ; ++u) sc[u][0] = mfma(k[0], qh[u][b], sc[u][0]), sc[u][1] = mfma(k[1], qh[u][b], sc[u][1]);
#pragma unroll
                    for (int u = 0; u < NQ; ++u) sc[u][0] = mfma(k[0], ql[u][b], sc[u][0]), sc[u][1] = mfma(k[1], ql[u][b], sc[u][1]);
#pragma unroll
                    for (int u = 0; u < NQ; ++u) sc[u][0] = mfma(k[2], qh[u][b], sc[u][0]), sc[u][1] = mfma(k[3], qh[u][b], sc[u][1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        };
        // The weights of tile i's scores.
        auto softmax = [&](int i) {
            const Scales* const s = scales + slot_of(i);
            float x_[NQ][8];
#pragma unroll
            for (int u = 0; u < NQ; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) x_[u][j] = sc[u][j >> 2][j & 3];
            const int first = tile_of(i) * kKvTile;
            const bool full = first + kKvTile - 1 <= pos_lo &&
                              (a.window == 0 || first > pos_hi - a.window || first + kKvTile <= a.sinks);
            const u4_t all = *reinterpret_cast<const u4_t*>(s->flags);
            const uint32_t flags = __builtin_amdgcn_readfirstlane(all.x | all.y | all.z | all.w);
            // (a lane's positions are 4 g .. and 16 + 4 g ..)
            auto of_tile = [&](const float* x) {
                const f4_t lo = *reinterpret_cast<const f4_t*>(x + 4 * g), hi = *reinterpret_cast<const f4_t*>(x + 16 + 4 * g);
                return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            };
            if (__builtin_expect((flags & kFar) != 0, 0)) {
                // (a value's power of two goes into the score here: P_j = p_j 2^ev_j; its sum is set right below)
                const auto up = of_tile(s->key_up), log = of_tile(s->value_log);
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    const float inv = 1.0f / to_t[u];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x_[u][j] = fmaf(log[j], inv, x_[u][j] * up[j]);
                }
            }
            if (!full) {
#pragma unroll
                for (int u = 0; u < NQ; ++u)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int k = first + (j >> 2) * 16 + 4 * g + (j & 3);
                        const bool seen = k <= pos[u] && (a.window == 0 || k > pos[u] - a.window || k < a.sinks);
                        x_[u][j] = seen ? x_[u][j] : -INFINITY;
                    }
            }
            // The maximum moves when it is passed by kSlack.
            float top[NQ];
            bool passed = false;
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                const float* x = x_[u];
                top[u] = max_quarters(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                            fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])))) * to_t[u];
                passed = passed || top[u] > m[u] + kSlack;
            }
            if (__any(passed)) {
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    const float to = top[u] > m[u] + kSlack ? top[u] : m[u];
                    float c;
                    l[u] = down(l[u], m[u] - to, &c);
                    m[u] = to;
#pragma unroll
                    for (int x = 0; x < 2 * NB; ++x) o[u][x] *= c;
                }
            }
            if (__builtin_expect((flags & kBad) != 0, 0)) {
                // rows that see a value block that is not finite: NaN in its dimensions, in the end
#pragma unroll 1
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t bit = s->bad[b][(j >> 2) * 16 + 4 * g + (j & 3)];  // 0 or 1
#pragma unroll
                        for (int u = 0; u < NQ; ++u) spoilt |= (x_[u][j] != -INFINITY ? bit : 0u) << (u * NB + b);
                    }
            }

            // P_j, up to 2^15
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                const float frame = m[u] - kWeightLift;
                float p[8], sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = __builtin_amdgcn_exp2f(fmaf(x_[u][j], to_t[u], -frame));
                    sum += p[j];
                }
                if (__builtin_expect((flags & kFar) != 0, 0)) {
                    // p_j = P_j 2^-ev_j, which may count where P_j is below what f32 holds
                    const auto down = of_tile(s->value_down);
                    sum = 0.0f;
                    bool deep = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        sum = fmaf(p[j], down[j], sum);
                        deep = deep || (p[j] < 0x1p-60f && down[j] > 1.0f && x_[u][j] != -INFINITY);
                    }
                    if (__builtin_expect(__any(deep), 0)) {
                        sum = 0.0f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float y = fmaf(x_[u][j], to_t[u], -frame);
                            const bool far = y < -60.0f;
                            sum = fmaf(__builtin_amdgcn_exp2f(far ? y + 100.0f : y), far ? down[j] * 0x1p-100f : down[j], sum);
                        }
                    }
                }
                l[u] += sum;
                split8(p, &ph[u], &pl[u]);
            }
        };

        const int n = it.count;
        int page1 = page_of(1), page2 = page_of(2), page3 = page_of(3);
        for (int i = 0; i < n; ++i) {
            products(true, i);
            __builtin_amdgcn_sched_barrier(0);
            // All that a tile loads is used a tile later: its own waits are for loads long done.
            // (The pages are opaque until then, or their products would be computed as they arrive.)
            asm volatile("" : "+v"(page1), "+v"(page2), "+v"(page3));
            SliceScales c[SLICES];
            convert_begin(i, c);
            make_scales(i + 2);
            convert_finish(i, c, page1, page2);
            load_scales(address_of(i + 3, page3));
            page1 = page2;
            page2 = page3;
            page3 = page_of(i + 4);
            __builtin_amdgcn_sched_barrier(0);
            softmax(i);
            barrier();
        }
        products(false, n);

        float any_first = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) any_first = fmaxf(any_first, first_top(b));
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            l[u] = sum_quarters(l[u]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float add = sum_quarters((spoilt >> (u * NB + b)) & 1u ? NAN : 0.0f);
                const int e = block_exponent(first_top(b), first_top(b) <= kZeros && any_first > kZeros);
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[u][2 * b + x][i] = ldexpf(o[u][2 * b + x][i], e) + add;
            }
        }

        // Rows that are NaN: for what they are made of, or for blocks that differ too much in size, and then done again.
        uint32_t again = 0;
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            const uint64_t lanes = __ballot(l[u] != l[u] && row0 + 16 * u + i16 < row1);
            again |= static_cast<uint32_t>((lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) & 0xffffu) << (16 * u);
        }
        auto plain = [&] {
            // (in the LDS of the first keys' operands, which no wave reads any more)
            plain_rows<QT, NB, NQ>(a, it, head, row0, again, wave, lane, q, out, reinterpret_cast<float*>(lds) + wave * 4 * (32 * NB + 32));
        };

        if (it.nsplit > 1) {
            // Every wave's state to memory; the workgroup that arrives last merges the parts, each wave its rows.
            auto rsrc_of = [&](int split) {
                return state_rsrc(a.partial, (static_cast<size_t>(it.slot + split) * n_kv + head) * kKvWaves + wave, STATE);
            };
            leave_state<NQ, NB>(rsrc_of(it.split), lane, o, m, l);
            if (__builtin_expect(again != 0, 0)) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                plain();
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the state is in memory
            __syncthreads();
            if (threadIdx.x == 0) last = arrive(a.arrived + static_cast<size_t>(it.slot) * n_kv + head, it.nsplit);
            __syncthreads();
            const bool mine = last != 0u;
            if (!mine) continue;
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                m[u] = -3.402823466e38f;
                l[u] = 0.0f;
#pragma unroll
                for (int t = 0; t < 2 * NB; ++t) o[u][t] = zero;
            }
            for (int part = 0; part < it.nsplit; ++part) take_state<NQ, NB>(rsrc_of(part), lane, o, m, l);
        }

        if (!idle) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                if (row0 + 16 * u + i16 >= row1) continue;
                store_row<NB>(out + element_of(u), hd, g, o[u], 1.0f / (l[u] * kLift));
            }
            if (__builtin_expect(it.nsplit == 1 && again != 0, 0)) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                plain();
            }
        }
    }
}

// Workgroups of a recorded launch, which walks whatever list is set by then.
constexpr unsigned kRecorded = 1024;
constexpr long long kMostGroups = 1 << 20;

template <int QT, int NB>
hipError_t launch_blocks(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    // (a launch holds less than 2^32 threads; the kernels walk their lists whatever the grid)
    const unsigned grid =
        count > 0 ? static_cast<unsigned>(std::min<long long>(static_cast<long long>(count) * a.kv.n_kv, kMostGroups)) : kRecorded;
    if (kind == 0) {
        attention_kernel<QT, NB><<<grid, kThreads, 0, s>>>(a, count, q, out);
    } else {
        constexpr int NQ = NB <= 4 ? 2 : 1;
        constexpr int lds = rows_lds_bytes<QT, NB>();
        const auto kernel = attention_rows_kernel<QT, NB, NQ>;
        if (lds > 64 << 10) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<grid, kThreads, lds, s>>>(a, count, q, out);
    }
    return hipGetLastError();
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
}  // namespace mlq
