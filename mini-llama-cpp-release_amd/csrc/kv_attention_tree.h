// Attention of drafted trees over the paged cache (kv_layout.h) on MFMA.
//
// A sequence's new tokens are the nodes of a tree, in an order that has parents first; node i lies in slot
// start + i and has position start + depth.  It sees what came before the tree (within the window, and the first
// positions), its ancestors and itself:
//
//   out = softmax_j(scale q . k_j) v   over these j.
//
// Who sees whom among the nodes is a bit a slot, laid out by tiles when the batch is set (kv_plan.cpp), so a tile of
// nodes costs a lane one word; tiles before the tree are as in kv_attention.h, whose arithmetic this is: codes as they
// lie, queries split in two fp16 parts over their block's largest, value scales in the weights, which are split over a
// power of two of every row and block that keeps its largest at 2^9 .. 2^15.  There eight rows stand beside their own
// low parts in an operand's sixteen columns; a tree has more rows than that, so here the sixteen columns are sixteen
// rows and a block takes two products (f32: three, as low parts times low parts, 2^-22 of an element, are left out).
// Batches with rows enough to fill its workgroups many times over run the kernel of kv_attention_rows.h instead, in
// its form for trees (kv_tree_cost says which; a batch runs one of them, as two launches would follow each other).
//
// Bound: issue.  A tile takes a wave 500 vector instructions and 32 products, and the two waves of a SIMD issue vector
// instructions 78 % of their time (64 nodes after 4000 positions, Q8_0, 32 heads over 8 KV heads of 128: 32 us, 20 of them
// tiles; the cache is read 16 times, from L2); small batches by the launch, four dependent trips to memory and the merge
// (8 nodes after 700 positions, 14 heads over 2 of 64: 8.3 us).  24 nodes of 16 sequences, Q4_1, 80 elements, a window of 1024:
// 40 us, in two rounds, as its 528 workgroups are more than the 512 that the chip holds and whole items are not split then.
// Measured and no faster: 32 rows a wave (one wave a SIMD: 46 us for the 64 nodes, 57 for the 16 sequences), weights
// times scales as one mixed-precision instruction each (33 us), with one look at a tile's frames as well (33),
// s_setprio around the products, 256 and 1024 workgroups (34 and 36); one power of two for a row's queries in place of one
// a block saves 2 % but needs a second form for queries whose blocks lie far apart.
#pragma once

#include "kv_attention_rows.h"

#include <algorithm>

namespace mlq {
namespace kv {

// Waves a SIMD: two at the least up to 128 elements (f32: 64), where 256 registers are enough but for Q4_1 of four blocks,
// which keeps 76 bytes a lane in scratch; above, one with all 512 (the compiler would rather have two that spill).
template <int QT, int NB>
constexpr int tree_waves() {
    return (QT == 0 ? NB <= 2 : NB <= 4) ? 2 : 1;
}

template <int QT, int NB>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(tree_waves<QT, NB>(), NB <= 4 ? 8 : 1))) void attention_tree_kernel(
    KvTreeAttention a, int count, const float* __restrict__ q, float* __restrict__ out) {
    using F = KvForm<QT>;
    constexpr int SB = F::kScaleBytes;
    constexpr int KL = F::key_lane(NB), VL = F::value_lane(NB);
    constexpr int KW = KL / 4, VW = VL / 4;
    constexpr int KS = NB * SB, VS = 2 * NB * SB;  // words of a lane's scales: 4 keys a half tile, 8 keys
    constexpr int STATE = (8 * NB + 2) * 64;       // floats of a wave's state of sixteen rows
    __shared__ float merge[2 * STATE];
    __shared__ unsigned last;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int n_kv = a.kv.n_kv, hd = a.kv.head_dim, heads = n_kv * a.group;
    const int page_tiles = a.kv.page_tiles, tile_shift = __builtin_ctz(page_tiles);
    const int total = (count > 0 ? count : uniform(a.lists.counts + kKvCountNarrow)) * n_kv;

    for (int w = blockIdx.x; w < total; w += gridDim.x) {
        const int head = w % n_kv;
        const KvTreeItem it = uniform(a.lists.items[0] + w / n_kv);
        const int rows = it.new_tokens * a.group, start = it.len - it.new_tokens;
        const int first_node_tile = start / kKvTile;

        // The lane's row: its token's position (only a window asks for it), where its bits and its elements start.
        const int row = min(it.row0 + i16, rows - 1), token = row / a.group;
        const int pos = a.window > 0 ? a.lists.pos[it.token0 + token] : 0;
        const uint32_t* const mask = a.lists.masks + (it.mask0 + token * it.words - first_node_tile);
        const size_t out_row = (static_cast<size_t>(it.token0 + token) * heads + head * a.group + row % a.group) * hd;
        h8_t qh[NB], ql[NB];
        float qsum[NB], to_t[NB];
        {
            float v[NB][8];
            load_query<NB, true>(q + out_row, hd, g, a.scale * (QT == 0 ? 1.0f / kElementLift : 1.0f), v, qsum, to_t);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                split8(v[b], &qh[b], &ql[b]);
                if (QT == 3) qsum[b] = sum_quarters(qsum[b]) * to_t[b];
            }
        }

        const f4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
        f4_t o[2 * NB];
        float om[NB];   // Q4_1: this lane's part of the sum of weights times minima
        int frame[NB];  // log2 f_b
        uint32_t spoilt = 0;  // bit b: this lane's part of the row sees a block that is not finite with a weight of 0
        float m = -3.402823466e38f, l = 0.0f;
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t) o[t] = zero;
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

        // The next tile's loads are under way during this one's work, unless its registers are not enough for both.
        constexpr bool AHEAD = QT == 0 ? NB <= 4 : QT != 3 || NB <= 6;
        int at = it.first + wave;
        int next_page = 0;
        if (AHEAD && at < end) {
            const uint8_t* tile = base_of(at, page_of(at));
            load_keys(tile);
            load_values(tile);
            if (at + kKvWaves < end) next_page = page_of(at + kKvWaves);
        }
        for (; at < end; at += kKvWaves) {
            const int tile_index = tile_of(at), first = tile_index * kKvTile;
            const bool more = AHEAD && at + kKvWaves < end;
            if (!AHEAD) next_page = page_of(at);
            const uint8_t* next = base_of(more ? at + kKvWaves : at, next_page);
            if (AHEAD && at + 2 * kKvWaves < end) next_page = page_of(at + 2 * kKvWaves);
            if (!AHEAD) load_keys(next);
            const bool nodes = tile_index >= first_node_tile;
            const bool full = !nodes && (a.window == 0 || first > it.far - a.window || first + kKvTile <= a.sinks);
            uint32_t word = 0;  // a tile of nodes: the row's bits
            if (nodes) word = mask[tile_index];

            // Scores.
            float t[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f4_t s = zero;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    h8_t hi, lo;
                    if (QT == 0) {
                        float v[8];
                        const float inv = inverse_power(kp[h][b]) * kElementLift;
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = mul_or_zero(bits<float>(kw[h][8 * b + j]), inv);
                        split8(v, &hi, &lo);
                    } else if (QT == 1) {
                        hi = codes8(kw[h][2 * b], kw[h][2 * b + 1], static_cast<_Float16>(128.0f));
                    } else {
                        const uint32_t x = kw[h][b];
                        hi = codes8(x & 0x0f0f0f0fu, (x >> 4) & 0x0f0f0f0fu, static_cast<_Float16>(QT == 2 ? 8.0f : 0.0f));
                    }
                    f4_t acc = mfma(hi, ql[b], mfma(hi, qh[b], zero));
                    if (QT == 0) acc = mfma(lo, qh[b], acc);  // (times kElementLift, which to_t takes back)
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
            auto key_in_tile = [&](int j) { return (j >> 2) * 16 + 4 * g + (j & 3); };
            float p[8];
            auto seen = [&](int j) -> bool {
                const int k = key_in_tile(j), key = first + k;
                return nodes ? (word >> k & 1u) != 0 : (a.window == 0) | (key > pos - a.window) | (key < a.sinks);
            };
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // an infinite scale (minimum) with codes that are not 0: NaN like the sum of its elements
                if (QT >= 2) t[j] = fmaf(t[j], 0.0f, t[j]);
            }
            if (!full) {
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = seen(j) ? t[j] : -INFINITY;
            }
            float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])),
                              fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
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
                            for (int i = 0; i < 4; ++i) o[2 * b + x][i] = ldexpf(o[2 * b + x][i], -less);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = __builtin_amdgcn_exp2f(t[j] - m);
                l += p[j];
            }
            const float least = fminf(fminf(fminf(p[0], p[1]), fminf(p[2], p[3])),
                                      fminf(fminf(p[4], p[5]), fminf(p[6], p[7])));
            if (__builtin_expect(__any(least == 0.0f), 0)) {
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
                h8_t vh[2], vl[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (QT == 0) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            v[j] = mul_or_zero(bits<float>(vw[16 * b + 8 * x + j]), inverse_power(vs[8 * b + j]) * kElementLift);
                        }
                        split8(v, &vh[x], &vl[x]);
                    } else if (QT == 1) {
                        vh[x] = codes8(vw[4 * b + 2 * x], vw[4 * b + 2 * x + 1], static_cast<_Float16>(128.0f));
                    } else {
                        const uint32_t y = vw[2 * b], z = vw[2 * b + 1];
                        vh[x] = codes8((x == 0 ? y : y >> 4) & 0x0f0f0f0fu, (x == 0 ? z : z >> 4) & 0x0f0f0f0fu,
                                       static_cast<_Float16>(QT == 2 ? 8.0f : 0.0f));
                    }
                }
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = mul_or_zero(p[j], scale_at(vs, 8 * b + j));
                float most = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
                if (__builtin_expect(__any(ldexpf(most, frame[b]) > 0x1p15f), 0)) {
                    most = max_quarters(most);
                    const int to = ldexpf(most, frame[b]) > 0x1p15f ? 9 - exponent(most) : frame[b];
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[2 * b + x][i] = ldexpf(o[2 * b + x][i], to - frame[b]);
                    frame[b] = to;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = ldexpf(v[j], frame[b]);
                if (QT == 3) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) om[b] += mul_or_zero(p[j], scale_at(vm, 8 * b + j));
                }
                h8_t ph, pl;
                split8(v, &ph, &pl);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    f4_t& acc = o[2 * b + x];
                    acc = mfma(vh[x], pl, mfma(vh[x], ph, acc));
                    if (QT == 0) acc = mfma(vl[x], ph, acc);
                }
            }
            if (more) load_values(next);
        }

        // The lanes' sums and the minima's part, out of the blocks' frames.
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
                    o[2 * b + x][i] = ldexpf(o[2 * b + x][i], -frame[b] - (QT == 0 ? 13 : 0)) + add;
                }
        }
        // The four waves' states into wave 0, in a fixed order.
        auto leave = [&](float* to) {
#pragma unroll
            for (int x = 0; x < 2 * NB; ++x) *reinterpret_cast<f4_t*>(to + (x * 64 + lane) * 4) = o[x];
            to[2 * NB * 256 + lane] = m;
            to[2 * NB * 256 + 64 + lane] = l;
        };
        auto take = [&](const float* from) {
            float w0, w1;
            fold(m, l, from[2 * NB * 256 + lane], from[2 * NB * 256 + 64 + lane], &w0, &w1);
#pragma unroll
            for (int x = 0; x < 2 * NB; ++x) {
                o[x] = o[x] * w0 + *reinterpret_cast<const f4_t*>(from + (x * 64 + lane) * 4) * w1;
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
            if (wave == 0) {
                leave_state<1, NB>(rsrc_of(it.split), lane, &o, &m, &l);
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
            for (int x = 0; x < 2 * NB; ++x) o[x] = zero;
            for (int part = wave; part < it.nsplit; part += kKvWaves) take_state<1, NB>(rsrc_of(part), lane, &o, &m, &l);
            merge_waves();
        }

        if (wave == 0 && it.row0 + i16 < rows) store_row<NB>(out + out_row, hd, g, o, 1.0f / l);
    }
}

template <int QT, int NB>
hipError_t launch_tree_blocks(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    if (kind != 0) return launch_rows<QT, NB, true>(a, count, q, out, s);
    attention_tree_kernel<QT, NB><<<grid_of(a.kv, count), kThreads, 0, s>>>(a, count, q, out);
    return hipGetLastError();
}

template <int QT>
hipError_t launch_tree(const KvTreeAttention& a, int kind, int count, const float* q, float* out, hipStream_t s) {
    switch (a.kv.nb) {
        case 1: return launch_tree_blocks<QT, 1>(a, kind, count, q, out, s);
        case 2: return launch_tree_blocks<QT, 2>(a, kind, count, q, out, s);
        case 3: return launch_tree_blocks<QT, 3>(a, kind, count, q, out, s);
        case 4: return launch_tree_blocks<QT, 4>(a, kind, count, q, out, s);
        case 6: return launch_tree_blocks<QT, 6>(a, kind, count, q, out, s);
        case 8: return launch_tree_blocks<QT, 8>(a, kind, count, q, out, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace kv
}  // namespace mlq
