// Beam selection: the best continuations over the beams of a group and the vocabulary.
//
//   value(b, t) = score_b + (x_bt - log sum_t exp x_bt)      in 64 bits
//
// over the tokens t whose logit x_bt is above -Inf of the beams whose score is; an ended beam has the one
// continuation (b, end_token) at score_b.  The `keep` largest values, largest first; of equal ones the lower
// beam, in a beam the larger logit, then the lower token.
//
// Two launches.  Parts of a row (kBeamPart logits, in registers from one pass): the largest logit, the sum of the
// exponentials in 64 bits, and the best `keep` logits.  A logit among a part's best is at least the keep-th
// largest of the threads' own largest, so few pass that bar, and those few are ranked by counting.  Then a
// workgroup a group: the rows' sums, and the best of the parts' best by the same bar.  Sums are taken in a fixed
// order: equal rows have equal sums, and the same call gives the same bits.
//
// Measured: 32 groups of 8 beams over 128011 tokens, 16 kept, 48 us (40 + 9 of kernels, 3.3 TB/s of logits in the first), with a
// quarter of the beams ended 44 (48 while their rows were read); 4 beams over 32000 tokens 11 us.  In one launch, the last part of a group to arrive selecting, 55 and 11.

#include "beam.h"

#include <algorithm>

namespace mlq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Unsigned numbers in the order of the values (-0 is 0), and back.
__device__ __forceinline__ uint32_t order_of(float v) {
    uint32_t b = __builtin_bit_cast(uint32_t, v);
    b = b == 0x80000000u ? 0u : b;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __builtin_bit_cast(float, (order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
// Orders by value, then by lower index.
__device__ __forceinline__ unsigned long long key_of(float v, uint32_t index) {
    return static_cast<unsigned long long>(order_of(v)) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float logit_of(unsigned long long key) { return value_of(static_cast<uint32_t>(key >> 32)); }
__device__ __forceinline__ uint32_t index_of(unsigned long long key) { return ~static_cast<uint32_t>(key); }
constexpr unsigned long long kNoKey = 0;  // below every logit's key, -Inf's too
// From this magnitude on the neighbours of a row's largest logit are 512 and more away, so that exp(logit - largest) is
// nothing beside 1 for all but its equals; below, largest - 800 is at least 288 smaller in f32 too.
constexpr float kFarTop = 0x1p33f;

// exp(d) for d <= 0 in 64 bits, 2^-39 of it off at the most: 2^n times a polynomial of the rest, at most 0.3466 (of
// degree 8, through exp at the Chebyshev points; 1.1e-12 off, the series to degree 9 6.9e-12).  n is rounded by a sum
// whose last places are whole numbers: its low word is n.  d is far above -2^31.
__device__ __forceinline__ double exp64(double d) {
    constexpr double kWhole = 6755399441055744.0;  // 1.5 x 2^52
    const double t = fma(d, 1.4426950408889634, kWhole);
    const double r = fma(t - kWhole, -0.6931471805599453, d);
    double y = 2.4876178959085513e-05;
    y = fma(y, r, 0.00019915881871396035);
    y = fma(y, r, 0.001388882165071769);
    y = fma(y, r, 0.008333266071022454);
    y = fma(y, r, 0.0416666668910917);
    y = fma(y, r, 0.16666666891180545);
    y = fma(y, r, 0.49999999999797773);
    y = fma(y, r, 0.999999999979769);
    y = fma(y, r, 1.0);
    return ldexp(y, static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(unsigned long long, t))));
}

// Over a wave, by lane permutations of the vector unit: rows of sixteen turned by 8, 4, 2 and 1, then the rows.
template <int ROR>
__device__ __forceinline__ float turned(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x120 + ROR, 0xf, 0xf, true));
}
template <int ROR>
__device__ __forceinline__ double turned(double v) {
    const uint2 w = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_mov_dpp(static_cast<int>(w.x), 0x120 + ROR, 0xf, 0xf, true),
                                                 __builtin_amdgcn_mov_dpp(static_cast<int>(w.y), 0x120 + ROR, 0xf, 0xf, true)));
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, turned<8>(v));
    v = fmaxf(v, turned<4>(v));
    v = fmaxf(v, turned<2>(v));
    v = fmaxf(v, turned<1>(v));
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ double wave_sum(double v) {
    v += turned<8>(v);
    v += turned<4>(v);
    v += turned<2>(v);
    v += turned<1>(v);
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// The r-th largest of the wave's values, r from 1 to 64 (the order of their bits, bit by bit).
__device__ __forceinline__ uint32_t wave_rth_largest(uint32_t v, int r) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = t | 1u << bit;
        t = __builtin_popcountll(__ballot(v >= c)) >= r ? c : t;
    }
    return t;
}

// Bound: issue and what it waits for, in turn.  Of the 36 us over the 192 live of the 256 rows above the vector units issue
// for 20 (by counters: 32 instructions a logit, 16 of them the exponential in 64 bits, which run at about the rate of 32);
// a wave spends 36 % of its life waiting for memory or at barriers and 37 % for its turn to issue.  3072 live workgroups
// share 1280 places, and each loads its part, then computes, then ranks, so that only other workgroups' work hides its loads.
// Five waves a SIMD (four: 42 us for the 256 rows); parts of 4096 logits 47 us.
template <int E>
__global__ __launch_bounds__(kThreads, 5) void beam_part_kernel(BeamCall c, int parts) {
    constexpr int kMost = kBeamMostKeep * E;
    __shared__ unsigned long long list[kMost];
    __shared__ float top_of[kWaves];
    __shared__ uint32_t bar_of[kWaves];
    __shared__ double sum_of[kWaves];
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const long long total = static_cast<long long>(c.groups) * c.beams * parts;
    for (long long w = blockIdx.x; w < total; w += gridDim.x) {
        const int lo = static_cast<int>(w % parts) * (E * kThreads), n = min(c.vocab - lo, E * kThreads);
        const size_t row = static_cast<size_t>(w / parts);
        // (rows without continuations of their own, and those of groups that come out as NaN: nothing is read of them here)
        const float score = c.scores[row];
        if (!(fabsf(score) < __builtin_inff()) || (c.ended != nullptr && c.ended[row] != 0)) continue;
        const float* const from = c.logits + row * c.vocab + lo;
        float x[E];
        if (n == E * kThreads) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = from[e * kThreads + tid];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = e * kThreads + tid < n ? from[e * kThreads + tid] : -__builtin_inff();
        }
        float mine = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < E; ++e) mine = fmaxf(mine, x[e]);
        // Enough of the wave's threads have a logit from here on.
        const uint32_t wave_bar = wave_rth_largest(order_of(mine), (c.keep + kWaves - 1) / kWaves);
        float top = wave_max(mine);
        __syncthreads();  // the last part's readers are done
        if (lane == 0) top_of[wave] = top, bar_of[wave] = wave_bar;
        if (tid == 0) found = 0;
        __syncthreads();
        uint32_t lowest = bar_of[0];
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            top = fmaxf(top, top_of[k]);
            lowest = min(lowest, bar_of[k]);
        }
        // The keys of what passes the bar.
        const float bar = fmaxf(value_of(lowest), -3.402823466e38f);  // (-Inf is no continuation)
        int index = lo + tid;
        asm("" : "+v"(index));  // (or all of them would be computed ahead)
        unsigned long long who[E];
        int passing = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            who[e] = __ballot(x[e] >= bar);
            passing += __builtin_popcountll(who[e]);
        }
        int base = 0;
        if (lane == 0) base = atomicAdd(&found, passing);
        base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (who[e] == 0) continue;
            const int at = base + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who[e] >> 32),
                                                            __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who[e]), 0));
            if (x[e] >= bar && at < kMost) list[at] = key_of(x[e], static_cast<uint32_t>(index + e * kThreads));
            base += __builtin_popcountll(who[e]);
        }
        // (a logit that is NaN, or +Inf and so minus itself, makes the sum NaN)
        double sum = 0.0;
        if (top > -__builtin_inff()) {
            const double top64 = top;
            const float least = top - 800.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                sum += exp64(static_cast<double>(__builtin_elementwise_maximum(x[e], least)) - top64);
                if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (few of them at a time: registers)
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) sum += x[e] != x[e] ? static_cast<double>(x[e]) : 0.0;
        }
        if (__builtin_expect(fabsf(top) >= kFarTop && top > -__builtin_inff(), 0)) {
            sum = 0.0;
            int first = tid;
            asm("" : "+v"(first));  // (as above: no addresses ahead)
#pragma unroll 1
            for (int i = first; i < n; i += kThreads) {  // (read again: rare, and the registers are the others')
                const float v = from[i];
                sum += v != v || v == __builtin_inff() ? __builtin_nan("") : v == top ? 1.0 : 0.0;
            }
        }
        sum = wave_sum(sum);
        if (lane == 0) sum_of[wave] = sum;
        __syncthreads();
        int m = found;
        if (__builtin_expect(m > kMost, 0)) {
            // As many equal logits: the bar is that of the threads' best keys, which differ.
            __shared__ unsigned long long key[kThreads], key_bar;
            unsigned long long best = kNoKey;
#pragma unroll 1
            for (int i = tid; i < n; i += kThreads) {
                const float v = from[i];
                const unsigned long long k = key_of(v, static_cast<uint32_t>(lo + i));
                if (v > -__builtin_inff() && k > best) best = k;
            }
            key[tid] = best;
            __syncthreads();
            int rank = 0;
            for (int k = 0; k < kThreads; ++k) rank += key[k] > best || (key[k] == best && k < tid) ? 1 : 0;
            if (rank == c.keep - 1) key_bar = best;
            if (tid == 0) found = 0;
            __syncthreads();
            // (of keep threads: at most all their logits)
#pragma unroll 1
            for (int i = tid; i < n; i += kThreads) {
                const float v = from[i];
                const unsigned long long k = key_of(v, static_cast<uint32_t>(lo + i));
                if (v > -__builtin_inff() && k >= key_bar) list[atomicAdd(&found, 1)] = k;
            }
            __syncthreads();
            m = found;
        }
        // (a group's lists lie side by side, best ones first)
        const int lists = c.beams * parts;
        unsigned long long* const best = c.best + static_cast<size_t>(w / lists) * lists * c.keep + w % lists;
        for (int i = tid; i < m; i += kThreads) {
            const unsigned long long k = list[i];
            int at = 0;
#pragma unroll 8
            for (int j = 0; j < m; ++j) at += list[j] > k ? 1 : 0;
            if (at < c.keep) best[static_cast<size_t>(at) * lists] = k;
        }
        for (int i = m + tid; i < c.keep; i += kThreads) best[static_cast<size_t>(i) * lists] = kNoKey;
        if (tid == 0) {
            double all = sum_of[0];
#pragma unroll
            for (int k = 1; k < kWaves; ++k) all += sum_of[k];
            c.parts[w] = BeamPart{all, all != all ? __builtin_nanf("") : top, 0};
        }
    }
}

// A continuation; better ones first.
struct Candidate {
    double value;
    unsigned long long key;
    int beam;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
    return a.value != b.value ? a.value > b.value : a.beam != b.beam ? a.beam < b.beam : a.key > b.key;
}

constexpr int kGroupEach = 8;  // candidates a thread and round
constexpr int kLanes = 16;     // that take a beam's parts

__global__ __launch_bounds__(kThreads) void beam_group_kernel(BeamCall c, int parts) {
    constexpr int E = kGroupEach, kMost = kBeamMostKeep * E;
    __shared__ double largest[kBeamMostBeams], sums[kBeamMostBeams], score[kBeamMostBeams];  // (the sums' logarithms)
    __shared__ int state[kBeamMostBeams];  // 0: no continuations, 1: of the logits, 2: ended
    __shared__ Candidate list[kMost + kBeamMostKeep], best[kBeamMostKeep];
    __shared__ double value[kMost + kBeamMostKeep];  // of the list
    __shared__ uint32_t bar_of[kWaves];
    __shared__ int found, bad;
    const int tid = threadIdx.x, wave = tid / 64, keep = c.keep;
    const double none = -__builtin_inf();
    for (int group = blockIdx.x; group < c.groups; group += gridDim.x) {
        // Candidates as they lie: the best of every part, the second best of every part ...
        const int lists = c.beams * parts, n = lists * keep;
        const unsigned long long* const keys = c.best + static_cast<size_t>(group) * n;
        // Four neighbours go to the four waves, from place to place in another order, so that each has its part of few
        // candidates and of every list: the waves' bars are then alike, whatever the beams' scores.
        const int shift = 31 - __builtin_clz(lists);  // (a place is about as many candidates)
        auto candidate = [&](int first, int e) {
            const int four = first + e * kThreads + tid % 64 * kWaves;
            return four + (wave + (four >> shift)) % kWaves;
        };
        unsigned long long key[E];
        auto load = [&](int first) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = candidate(first, e);
                key[e] = i < n ? keys[i] : kNoKey;
            }
        };
        load(0);
        __syncthreads();  // the last group's readers are done
        if (tid == 0) bad = 0;
        __syncthreads();
        // The beams' sums: the parts' over their largest logit, lanes and then pairs of lanes in order.
        for (int b = tid / kLanes; b < (c.beams + 3) / 4 * 4; b += kThreads / kLanes) {  // (whole waves)
            const bool there = b < c.beams;
            const size_t row = static_cast<size_t>(group) * c.beams + min(b, c.beams - 1);
            const float s = c.scores[row];
            int what = !(s < __builtin_inff()) ? -1 : s == -__builtin_inff() ? 0 : c.ended != nullptr && c.ended[row] != 0 ? 2 : 1;
            const BeamPart* const p = c.parts + row * parts;
            float top = -__builtin_inff();
            int wrong = 0;
            for (int k = tid % kLanes; k < parts; k += kLanes) {
                const float x = p[k].largest;
                wrong |= x != x ? 1 : 0;
                top = fmaxf(top, x);
            }
#pragma unroll
            for (int k = kLanes / 2; k > 0; k /= 2) {
                top = fmaxf(top, __shfl_xor(top, k));
                wrong |= __shfl_xor(wrong, k);
            }
            double sum = 0.0;
            for (int k = tid % kLanes; k < parts; k += kLanes) {
                const BeamPart x = p[k];
                if (x.largest == top) {
                    sum += x.sum;
                } else if (x.largest > -__builtin_inff() && fabsf(top) < kFarTop) {
                    sum += x.sum * exp64(static_cast<double>(fmaxf(x.largest, top - 800.0f)) - static_cast<double>(top));
                }
            }
#pragma unroll
            for (int k = kLanes / 2; k > 0; k /= 2) sum += __shfl_xor(sum, k);
            if (there && tid % kLanes == 0) {
                if (what == 1) what = wrong != 0 ? -1 : top == -__builtin_inff() ? 0 : 1;
                largest[b] = what == 1 ? static_cast<double>(top) : 0.0;
                sums[b] = what == 1 ? log(sum) : 0.0;
                score[b] = static_cast<double>(s);
                state[b] = what;
                if (what < 0) bad = 1;
            }
        }
        __syncthreads();
        const size_t out = static_cast<size_t>(group) * keep;
        if (bad != 0) {
            for (int i = tid; i < keep; i += kThreads) {
                c.parents[out + i] = c.tokens[out + i] = -1;
                c.out_scores[out + i] = __builtin_nanf("");
            }
            continue;
        }
        // Rounds: what is best so far, and the next candidates, until a candidate of every list has been too small.
        int have = 0, small = 0;
        for (int first = 0; first < n && small < lists; first += E * kThreads) {
            Candidate x[E];
            float mine = -__builtin_inff();  // of the thread's, rounded down
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = candidate(first, e), list_of = i % lists, b = list_of / parts;
                x[e] = Candidate{none, key[e], b};
                if (i < n) {
                    const float logit = logit_of(key[e]);
                    if (state[b] == 1 && key[e] != kNoKey) {
                        x[e].value = score[b] + (static_cast<double>(logit) - largest[b] - sums[b]);
                    } else if (state[b] == 2 && i < lists && list_of % parts == 0) {
                        x[e].value = score[b];
                        x[e].key = key_of(0.0f, static_cast<uint32_t>(c.end_token));
                    }
                }
                mine = fmaxf(mine, __double2float_rd(x[e].value));
            }
            if (first + E * kThreads < n) load(first + E * kThreads);
            const int each = (keep + kWaves - 1) / kWaves;
            // To the list goes what passes the waves' bars, as many as have to and more.
            auto gather = [&](uint32_t wave_bar) {
                if (tid % 64 == 0) bar_of[wave] = wave_bar;
                if (tid == 0) found = 0;
                __syncthreads();
                uint32_t lowest = bar_of[0];
#pragma unroll
                for (int k = 1; k < kWaves; ++k) lowest = min(lowest, bar_of[k]);
                double bar = static_cast<double>(value_of(lowest));
                if (have == keep) bar = fmax(bar, best[keep - 1].value);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (x[e].value >= bar && x[e].value > none) {
                        const int at = atomicAdd(&found, 1);
                        if (at < kMost) list[at] = x[e];
                    }
                }
                __syncthreads();
                return found;
            };
            int m = gather(wave_rth_largest(order_of(mine), each));
            if (m > kThreads) {
                // (many of a thread's: the bar is that of all the wave's)
                uint32_t order[E], t = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) order[e] = order_of(__double2float_rd(x[e].value));
#pragma unroll 1
                for (int bit = 31; bit >= 0; --bit) {
                    const uint32_t c = t | 1u << bit;
                    int above = 0;
#pragma unroll
                    for (int e = 0; e < E; ++e) above += __builtin_popcountll(__ballot(order[e] >= c));
                    t = above >= each ? c : t;
                }
                __syncthreads();  // (all have read what was found)
                m = gather(t);
            }
            if (__builtin_expect(m > kMost, 0)) {
                // As many values that f32 does not tell apart: the bar is that of the threads' best, which differ.
                __shared__ Candidate of_thread[kThreads], exact_bar;
                Candidate top{none, kNoKey, c.beams};
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (x[e].value > none && before(x[e], top)) top = x[e];
                }
                of_thread[tid] = top;
                __syncthreads();
                int rank = 0;
                for (int k = 0; k < kThreads; ++k) {
                    const Candidate other = of_thread[k];
                    rank += before(other, top) || (k < tid && !before(top, other)) ? 1 : 0;
                }
                if (rank == keep - 1) exact_bar = top;
                if (tid == 0) found = 0;
                __syncthreads();
                const Candidate least = exact_bar;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (x[e].value > none && !before(least, x[e])) list[atomicAdd(&found, 1)] = x[e];
                }
                __syncthreads();
                m = found;
            }
            small = m > 0 ? 0 : small + E * kThreads;
            if (m > 0) {
                for (int i = tid; i < have; i += kThreads) list[m + i] = best[i];
                m += have;
                __syncthreads();
                for (int i = tid; i < m; i += kThreads) value[i] = list[i].value;
                __syncthreads();
                for (int i = tid; i < m; i += kThreads) {
                    const Candidate k = list[i];
                    int at = 0, equal = 0;
#pragma unroll 8
                    for (int j = 0; j < m; ++j) {
                        const double v = value[j];
                        at += v > k.value ? 1 : 0;
                        equal += v == k.value ? 1 : 0;
                    }
                    if (equal > 1) {
                        for (int j = 0; j < m; ++j) at += value[j] == k.value && before(list[j], k) ? 1 : 0;
                    }
                    if (at < keep) best[at] = k;
                }
                have = min(m, keep);
            }
            __syncthreads();
        }
        for (int i = tid; i < keep; i += kThreads) {
            const bool some = i < have;
            c.parents[out + i] = some ? best[i].beam : -1;
            c.tokens[out + i] = some ? static_cast<int>(index_of(best[i].key)) : -1;
            c.out_scores[out + i] = some ? static_cast<float>(best[i].value) : -__builtin_inff();
        }
    }
}

}  // namespace

hipError_t launch_beam_select(const BeamCall& c, hipStream_t s) {
    const int each = beam_part(static_cast<long long>(c.groups) * c.beams, c.vocab), parts = (c.vocab + each - 1) / each;
    const long long groups = static_cast<long long>(c.groups) * c.beams * parts;
    const unsigned grid = static_cast<unsigned>(std::min<long long>(groups, 1 << 20));
    if (each == kBeamPart) beam_part_kernel<kBeamPart / kThreads><<<grid, kThreads, 0, s>>>(c, parts);
    else beam_part_kernel<kBeamSmallPart / kThreads><<<grid, kThreads, 0, s>>>(c, parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    beam_group_kernel<<<std::min(c.groups, 1 << 20), kThreads, 0, s>>>(c, parts);
    return hipGetLastError();
}

}  // namespace mlq
