// The paged attention for more than eight query rows a KV head: chunks of a prompt,
// whole prompts (kv_attention.h has the formula and the kernel for few rows).
//
// A workgroup takes 4 x 16 NQ rows of one KV head, a wave 16 NQ of them, and walks tiles of 32
// positions that its waves convert for each other: a tile's keys and values are
// decoded to f32 once, brought into fp16's range by a power of two per position and
// split into two fp16 parts (hi + lo, 2^-22 is lost; the decoded product of a code and a
// binary16 scale has at most 19 bits and is exact), and lie in LDS as the MFMA
// operands they are.  Then, all in v_mfma_f32_16x16x32_f16, three products a pair:
//
//   S^T = K Q^T      A from LDS, B (queries, relative to the row's largest) in registers;
//   O^T += V^T P^T   A from LDS, B the weights: a lane's eight scores are its eight weights.
//
// The powers of two come back per position: 2^ek into the score, 2^ev into the weight
// (P_j = p_j 2^ev_j); the running maximum is that of t_j + ev_j, as in the kernel for few
// rows, so what a row does not see cannot cost it a digit.
//
// The loop is a pipeline over tiles i: compute on i, convert i + 1 into the other LDS buffer,
// scales of i + 2, loads ahead of both; one barrier a tile.
#pragma once

#include "kv_attention.h"
#include "quant_device.h"

#include <type_traits>

namespace mlq {
namespace kv {

// Scales of a tile in LDS: what a code (f32: an element) is multiplied by, and, for f32
// arithmetic on quantized codes, what is added then.
template <int QT, int NB>
struct TileScales {
    static constexpr bool kPacked = QT == 1 || QT == 2;  // decoded in packed fp16
    typename std::conditional<kPacked, _Float16, float>::type scale[2][QT == 3 ? 2 : 1][NB][kKvTile];  // keys, values
    float key_up[kKvTile];     // 2^ek
    float value_log[kKvTile];  // ev
    float value_up[kKvTile];   // 2^ev
    uint32_t bad[NB];          // positions whose value block is not finite
    uint32_t flags;            // kBad: any of `bad`; kFar: some power of two is not 1
};
constexpr uint32_t kBad = 1, kFar = 2;
constexpr float kLift = 256.0f;  // operands lie in LDS times this

template <int QT, int NB>
constexpr int rows_lds_bytes() {
    return 2 * 8 * NB * 1024 + 3 * static_cast<int>(sizeof(TileScales<QT, NB>));
}

template <int QT, int NB, int NQ>
__global__ __launch_bounds__(kThreads, NB <= 4 ? 2 : 1) void attention_rows_kernel(KvAttention a, int count, const float* __restrict__ q,
                                                                      float* __restrict__ out) {
    using F = KvForm<QT>;
    using Scales = TileScales<QT, NB>;
    constexpr int KL = F::key_lane(NB), VL = F::value_lane(NB);
    constexpr int FRAGS = 2 * NB;                          // operands of keys, of values (hi or lo) a tile
    constexpr int TASKS = (FRAGS + kKvWaves - 1) / kKvWaves;  // of either, per wave
    constexpr int RAW_K = QT == 0 ? 8 : QT == 1 ? 2 : 1, RAW_V = QT == 0 ? 8 : 2;  // words a lane loads for an operand
    constexpr int QUADS = NQ * 2 * NB, STATE = (QUADS * 4 + 2 * NQ) * 64;
    constexpr int ROWS = 16 * NQ;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // [buffer][key hi, key lo, value hi, value lo][operand][lane] of 16 bytes, then the scales
    h8_t* const operands = reinterpret_cast<h8_t*>(lds);
    Scales* const scales = reinterpret_cast<Scales*>(lds + 2 * 8 * NB * 1024);
    auto operand = [&](int buffer, int part, int f) { return operands + ((buffer * 4 + part) * FRAGS + f) * 64; };
    __shared__ unsigned last;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int n_kv = a.kv.n_kv, hd = a.kv.head_dim, heads = n_kv * a.group;
    const int page_tiles = a.kv.page_tiles, tile_shift = __builtin_ctz(page_tiles);
    const int total = (count > 0 ? count : uniform(a.lists.counts + kKvCountWide)) * n_kv;

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
        size_t out_row[NQ];
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            const int r = min(row0 + 16 * u + i16, rows - 1);
            const int token = r / a.group;
            pos[u] = start + token;
            out_row[u] = (static_cast<size_t>(it.token0 + token) * heads + head * a.group + r % a.group) * hd;
            float v[NB][8], sum[NB];
            load_query<NB>(q + out_row[u], hd, g, a.scale * (1.0f / kLift), v, sum, &to_t[u]);
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

        const int end = it.first + it.count;
        auto tile_of = [&](int i) { return i < it.sinks ? i : i + it.shift; };
        // Tiles past the end repeat the last one: loads stay in bounds, nothing uses them.
        auto base_of = [&](int i) -> const uint8_t* {
            const int t = tile_of(min(i, end - 1));
            const int page = uniform(&a.lists.pages[it.page0 + (t >> tile_shift)].page);
            return a.kv.base + ((static_cast<size_t>(page) * n_kv + head) * page_tiles + (t & (page_tiles - 1))) * F::tile(NB);
        };

        // Loads of a tile: this wave's operands, and (wave 0) lane's scales: keys' by
        // lanes 0 .. 31, values' by lanes 32 .. 63.
        uint32_t raw_k[TASKS][RAW_K], raw_v[TASKS][RAW_V];
        uint32_t raw_s[F::kPlanes][NB];
        auto load_raw = [&](const uint8_t* tile) {
#pragma unroll
            for (int k = 0; k < TASKS; ++k) {
                const int f = wave + kKvWaves * k;
                if (f >= FRAGS) continue;
                const int h = f / NB, b = f % NB;  // keys: half tile, block
                const uint8_t* p = tile + h * 64 * KL;
                const uint8_t* pv = tile + F::half(NB);
                const int bv = f >> 1, t = f & 1;  // values: block, half of its dimensions
                if (QT == 0) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const u4_t k4 = *reinterpret_cast<const u4_t*>(p + F::at(KL, lane, b * 32 + 16 * x));
                        const u4_t v4 = *reinterpret_cast<const u4_t*>(pv + F::at(VL, lane, bv * 64 + t * 32 + 16 * x));
#pragma unroll
                        for (int i = 0; i < 4; ++i) raw_k[k][4 * x + i] = k4[i], raw_v[k][4 * x + i] = v4[i];
                    }
                } else {
                    if (QT == 1) {
                        const uint2 k2 = *reinterpret_cast<const uint2*>(p + F::at(KL, lane, b * 8));
                        raw_k[k][0] = k2.x, raw_k[k][RAW_K - 1] = k2.y;
                    } else {
                        raw_k[k][0] = *reinterpret_cast<const uint32_t*>(p + F::at(KL, lane, b * 4));
                    }
                    const uint2 v2 = *reinterpret_cast<const uint2*>(pv + F::at(VL, lane, QT == 1 ? bv * 16 + t * 8 : bv * 8));
                    raw_v[k][0] = v2.x, raw_v[k][1] = v2.y;
                }
            }
        };
        const int key = lane & 31;
        auto load_scales = [&](const uint8_t* tile) {
            if (wave != 0) return;
            const uint8_t* p = tile + (lane >= 32 ? F::half(NB) : 0) + F::codes(NB);
#pragma unroll
            for (int x = 0; x < F::kPlanes; ++x)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int at = lane >= 32 ? F::value_scale(NB, key, b) : F::key_scale(NB, key, b);
                    raw_s[x][b] = QT == 0 ? reinterpret_cast<const uint32_t*>(p)[at]
                                          : reinterpret_cast<const uint16_t*>(p + x * F::plane(NB))[at];
                }
        };
        // Scales to LDS.  Operands lie there times 2^8 and over a power of two per position: 1 where the
        // position's largest element is from 2^-10 to 2^7 (the parts then lose what they do at 1,
        // 2^-22, and none reaches 2^15), else what brings it to [1, 2).
        auto make_scales = [&](Scales* s) {
            if (wave != 0) return;
            float d[NB], add[NB];
            float top = 0.0f;
            bool bad[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                d[b] = QT == 0 ? bits<float>(raw_s[0][b]) : half_value(static_cast<uint16_t>(raw_s[0][b]));
                add[b] = QT == 3 ? half_value(static_cast<uint16_t>(raw_s[F::kPlanes - 1][b])) : 0.0f;
                bad[b] = !(fabsf(d[b]) < INFINITY) || !(fabsf(add[b]) < INFINITY);
                const float most = QT == 0 ? d[b] : QT == 3 ? fmaf(16.0f, d[b], fabsf(add[b])) : (QT == 1 ? 128.0f : 8.0f) * d[b];
                if (!bad[b]) top = fmaxf(top, most);
            }
            int e = static_cast<int>(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
            e = top == 0.0f || (e >= -10 && e < 7) ? 0 : max(e, -90);
            const float down = ldexpf(kLift, -e);
            uint32_t any = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                // keys: NaN through to the score; values: zero here, NaN for the rows that see it (`bad`)
                const float nothing = lane >= 32 ? 0.0f : NAN;
                using T = typename std::remove_reference<decltype(s->scale[0][0][0][0])>::type;
                s->scale[lane >> 5][0][b][key] = static_cast<T>(bad[b] ? nothing : QT == 0 ? down : d[b] * down);
                if (QT == 3) s->scale[lane >> 5][QT == 3 ? 1 : 0][b][key] = static_cast<T>(bad[b] ? nothing : add[b] * down);
                const uint32_t mask = static_cast<uint32_t>(__ballot(bad[b]) >> 32);
                any |= mask;
                if (lane == 0) s->bad[b] = mask;
            }
            if (lane < 32) {
                s->key_up[key] = ldexpf(1.0f, e);
            } else {
                s->value_log[key] = static_cast<float>(e);
                s->value_up[key] = ldexpf(1.0f, e);
            }
            const bool far = __any(e != 0);
            if (lane == 0) s->flags = (any != 0 ? kBad : 0u) | (far ? kFar : 0u);
        };
        // Eight codes as fp16 (minus the stored offset): keys, values (`t`: which nibbles).
        auto codes_of = [&](const uint32_t* raw, bool values, int t) -> h8_t {
            if (QT == 1) return codes8(raw[0], raw[RAW_K - 1], static_cast<_Float16>(128.0f));
            const _Float16 off = static_cast<_Float16>(QT == 2 ? 8.0f : 0.0f);
            if (values) return codes8((raw[0] >> (4 * t)) & 0x0f0f0f0fu, (raw[1] >> (4 * t)) & 0x0f0f0f0fu, off);
            return codes8(raw[0] & 0x0f0f0f0fu, (raw[0] >> 4) & 0x0f0f0f0fu, off);
        };
        auto convert = [&](int buffer, const Scales* s) {
#pragma unroll
            for (int k = 0; k < TASKS; ++k) {
                const int f = wave + kKvWaves * k;
                if (FRAGS % kKvWaves != 0 && f >= FRAGS) continue;
                const int h = f / NB, b = f % NB, bv = f >> 1, t = f & 1;
                h8_t hi, lo;
                if constexpr (Scales::kPacked) {
                    // code times scale: at most 19 bits, so hi and what is left of it are exact
                    const _Float16 d = s->scale[0][0][b][16 * h + i16];
                    const h8_t d8{d, d, d, d, d, d, d, d};
                    h8_t c = codes_of(raw_k[k], false, 0);
                    hi = c * d8;
                    lo = __builtin_elementwise_fma(c, d8, -hi);
                    operand(buffer, 0, f)[lane] = hi;
                    operand(buffer, 1, f)[lane] = lo;
                    typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
                    const h4_t x = *reinterpret_cast<const h4_t*>(s->scale[1][0][bv] + 4 * g);
                    const h4_t y = *reinterpret_cast<const h4_t*>(s->scale[1][0][bv] + 16 + 4 * g);
                    const h8_t dv = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                    c = codes_of(raw_v[k], true, t);
                    hi = c * dv;
                    lo = __builtin_elementwise_fma(c, dv, -hi);
                } else {
                    float x[8];
                    const float d = s->scale[0][0][b][16 * h + i16];
                    const float add = QT == 3 ? s->scale[0][QT == 3 ? 1 : 0][b][16 * h + i16] : 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        x[j] = QT == 0 ? bits<float>(raw_k[k][j & (RAW_K - 1)]) * d
                                       : fmaf(static_cast<float>((raw_k[k][0] >> (8 * (j & 3) + 4 * (j >> 2))) & 0xfu), d, add);
                    }
                    split8(x, &hi, &lo);
                    operand(buffer, 0, f)[lane] = hi;
                    operand(buffer, 1, f)[lane] = lo;
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const f4_t d4 = *reinterpret_cast<const f4_t*>(s->scale[1][0][bv] + 16 * y + 4 * g);
                        const f4_t a4 = *reinterpret_cast<const f4_t*>(s->scale[1][QT == 3 ? 1 : 0][bv] + 16 * y + 4 * g);
                        const uint32_t nibbles = (raw_v[k][y] >> (4 * t)) & 0x0f0f0f0fu;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[4 * y + i] = QT == 0 ? mul_or_zero(bits<float>(raw_v[k][(4 * y + i) & (RAW_V - 1)]), d4[i])
                                                   : fmaf(static_cast<float>((nibbles >> (8 * i)) & 0xffu), d4[i], a4[i]);
                        }
                    }
                    split8(x, &hi, &lo);
                }
                operand(buffer, 2, f)[lane] = hi;
                operand(buffer, 3, f)[lane] = lo;
            }
        };

        // Fill the pipeline: tile `first` converted, `first + 1` loaded, scales of both.
        const uint8_t* tile0 = base_of(it.first);
        const uint8_t* tile1 = base_of(it.first + 1);
        __syncthreads();  // the last item's readers are done
        load_scales(tile0);
        load_raw(tile0);
        make_scales(scales + 0);
        load_scales(tile1);
        make_scales(scales + 1);
        __syncthreads();
        convert(0, scales + 0);
        load_raw(tile1);
        load_scales(base_of(it.first + 2));
        __syncthreads();

        int slot = 0;  // of tile i's scales
        for (int i = it.first; i < end; ++i) {
            const int buffer = (i - it.first) & 1;
            const int slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot1 == 2 ? 0 : slot1 + 1;
            const Scales* const s = scales + slot;

            f4_t sc[NQ][2];
#pragma unroll
            for (int u = 0; u < NQ; ++u) sc[u][0] = sc[u][1] = zero;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const h8_t k0 = operand(buffer, 0, b)[lane], k1 = operand(buffer, 0, NB + b)[lane];
                const h8_t l0 = operand(buffer, 1, b)[lane], l1 = operand(buffer, 1, NB + b)[lane];
#pragma unroll
                for (int u = 0; u < NQ; ++u) sc[u][0] = mfma(k0, qh[u][b], sc[u][0]), sc[u][1] = mfma(k1, qh[u][b], sc[u][1]);
#pragma unroll
                for (int u = 0; u < NQ; ++u) sc[u][0] = mfma(k0, ql[u][b], sc[u][0]), sc[u][1] = mfma(k1, ql[u][b], sc[u][1]);
#pragma unroll
                for (int u = 0; u < NQ; ++u) sc[u][0] = mfma(l0, qh[u][b], sc[u][0]), sc[u][1] = mfma(l1, qh[u][b], sc[u][1]);
            }
            // Ahead: convert i + 1, scales of i + 2, loads of i + 2 (raw) and i + 3 (scales).
            convert(buffer ^ 1, scales + slot1);
            make_scales(scales + slot2);
            load_raw(base_of(i + 2));
            load_scales(base_of(i + 3));

            const int first = tile_of(i) * kKvTile;
            const bool full = first + kKvTile - 1 <= pos_lo &&
                              (a.window == 0 || first > pos_hi - a.window || first + kKvTile <= a.sinks);
            const uint32_t flags = __builtin_amdgcn_readfirstlane(s->flags);
            h8_t ph[NQ], pl[NQ];
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                float t[8], top;
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = sc[u][j >> 2][j & 3] * to_t[u];
                if (flags & kFar) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[j] *= s->key_up[(j >> 2) * 16 + 4 * g + (j & 3)];
                }
                if (!full) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int k = first + (j >> 2) * 16 + 4 * g + (j & 3);
                        const bool seen = k <= pos[u] && (a.window == 0 || k > pos[u] - a.window || k < a.sinks);
                        t[j] = seen ? t[j] : -INFINITY;
                    }
                }
                if (flags & kFar) {
                    top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, t[j] + s->value_log[(j >> 2) * 16 + 4 * g + (j & 3)]);
                } else {
                    top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
                }
                top = max_quarters(top);
                if (__any(top > m[u] + kSlack)) {
                    const float to = top > m[u] + kSlack ? top : m[u];
                    const float c = __builtin_amdgcn_exp2f(m[u] - to);
                    m[u] = to;
                    l[u] *= c;
#pragma unroll
                    for (int x = 0; x < 2 * NB; ++x) o[u][x] *= c;
                }
                // P_j = p_j 2^ev_j up to 2^(6 + 8)
                const float frame = m[u] - 8.0f;
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = __builtin_amdgcn_exp2f(t[j] - frame);
                    l[u] += p[j];
                }
                if (flags & kBad) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t mask = s->bad[b];
                        bool hit = false;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            hit = hit || (((mask >> ((j >> 2) * 16 + 4 * g + (j & 3))) & 1u) != 0 && !(p[j] == 0.0f));
                        }
                        const float add = sum_quarters(hit ? NAN : 0.0f);
                        o[u][2 * b] += add;
                        o[u][2 * b + 1] += add;
                    }
                }
                if (flags & kFar) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[j] *= s->value_up[(j >> 2) * 16 + 4 * g + (j & 3)];
                }
                split8(p, &ph[u], &pl[u]);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const h8_t v0 = operand(buffer, 2, 2 * b)[lane], v1 = operand(buffer, 2, 2 * b + 1)[lane];
                const h8_t l0 = operand(buffer, 3, 2 * b)[lane], l1 = operand(buffer, 3, 2 * b + 1)[lane];
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    o[u][2 * b] = mfma(v0, ph[u], o[u][2 * b]), o[u][2 * b + 1] = mfma(v1, ph[u], o[u][2 * b + 1]);
                }
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    o[u][2 * b] = mfma(v0, pl[u], o[u][2 * b]), o[u][2 * b + 1] = mfma(v1, pl[u], o[u][2 * b + 1]);
                }
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    o[u][2 * b] = mfma(l0, ph[u], o[u][2 * b]), o[u][2 * b + 1] = mfma(l1, ph[u], o[u][2 * b + 1]);
                }
            }
            __syncthreads();
            slot = slot1;
        }

#pragma unroll
        for (int u = 0; u < NQ; ++u) l[u] = sum_quarters(l[u]);

        if (it.nsplit > 1) {
            // Every wave's state to memory; the workgroup that arrives last merges the parts, each wave its rows.
            auto rsrc_of = [&](int split) {
                return state_rsrc(a.partial, (static_cast<size_t>(it.slot + split) * n_kv + head) * kKvWaves + wave, STATE);
            };
            leave_state<NQ, NB>(rsrc_of(it.split), lane, o, m, l);
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
                store_row<NB>(out + out_row[u], hd, g, o[u], 1.0f / (l[u] * kLift));
            }
        }
    }
}

// Workgroups of a recorded launch, which walks whatever list is set by then.
constexpr unsigned kRecorded = 1024;

template <int QT, int NB>
hipError_t launch_blocks(const KvAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    const unsigned grid = count > 0 ? static_cast<unsigned>(count) * a.kv.n_kv : kRecorded;
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
