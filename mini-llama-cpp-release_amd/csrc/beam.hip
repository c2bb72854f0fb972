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

#include "beam.h"

#include <algorithm>

namespace mlq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Orders by value, then by lower index.
__device__ __forceinline__ unsigned long long key_of(float v, uint32_t index) {
    uint32_t b = __builtin_bit_cast(uint32_t, v);
    b = b == 0x80000000u ? 0u : b;
    const uint32_t order = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return static_cast<unsigned long long>(order) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float logit_of(unsigned long long key) {
    const uint32_t order = static_cast<uint32_t>(key >> 32);
    return __builtin_bit_cast(float, (order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint32_t index_of(unsigned long long key) { return ~static_cast<uint32_t>(key); }
constexpr unsigned long long kNoKey = 0;  // below every logit's key, -Inf's too

// exp(d) for d <= 0 in 64 bits, 2^-36 of it off at the most: 2^n times the series to degree 9 of the rest, at most
// 0.35 (0.35^10 / 10! = 7.6e-12).  0 below -700.
__device__ __forceinline__ double exp64(double d) {
    const double n = rint(d * 1.4426950408889634);
    const double r = fma(n, -0.6931471805599453, d);
    double y = 1.0 / 362880;
    y = fma(y, r, 1.0 / 40320);
    y = fma(y, r, 1.0 / 5040);
    y = fma(y, r, 1.0 / 720);
    y = fma(y, r, 1.0 / 120);
    y = fma(y, r, 1.0 / 24);
    y = fma(y, r, 1.0 / 6);
    y = fma(y, r, 0.5);
    y = fma(y, r, 1.0);
    y = fma(y, r, 1.0);
    return d < -700.0 ? 0.0 : ldexp(y, static_cast<int>(n));
}

template <int E>
__global__ __launch_bounds__(kThreads) void beam_part_kernel(BeamCall c, int parts) {
    __shared__ unsigned long long key[kThreads];
    __shared__ unsigned long long list[kBeamMostKeep * E];
    __shared__ float top_of[kWaves];
    __shared__ int bad_of[kWaves];
    __shared__ double sum_of[kWaves];
    __shared__ unsigned long long bar;
    __shared__ int found;
    const int tid = threadIdx.x, wave = tid / 64;
    const long long total = static_cast<long long>(c.groups) * c.beams * parts;
    for (long long w = blockIdx.x; w < total; w += gridDim.x) {
        const int part = static_cast<int>(w % parts);
        const long long row = w / parts;
        const int lo = static_cast<int>(static_cast<long long>(c.vocab) * part / parts);
        const int n = static_cast<int>(static_cast<long long>(c.vocab) * (part + 1) / parts) - lo;  // E * kThreads at the most
        const float* const from = c.logits + static_cast<size_t>(row) * c.vocab + lo;
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = e * kThreads + tid;
            x[e] = i < n ? from[i] : -__builtin_inff();
        }
        float top = -__builtin_inff();
        bool bad = false;
        unsigned long long mine = kNoKey;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            bad = bad || !(x[e] < __builtin_inff());
            top = fmaxf(top, x[e]);
            const int i = e * kThreads + tid;
            if (i < n) {
                const unsigned long long k = key_of(x[e], static_cast<uint32_t>(lo + i));
                mine = k > mine ? k : mine;
            }
        }
#pragma unroll
        for (int s = 32; s > 0; s /= 2) top = fmaxf(top, __shfl_xor(top, s));
        const bool wave_bad = __any(bad);
        __syncthreads();  // the last part's readers are done
        key[tid] = mine;
        if (tid % 64 == 0) top_of[wave] = top, bad_of[wave] = wave_bad;
        if (tid == 0) found = 0;
        __syncthreads();
        bad = false;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) top = fmaxf(top, top_of[k]), bad = bad || bad_of[k] != 0;
        // The sum, and where this thread's largest stands among the threads'.
        double sum = 0.0;
        if (top > -__builtin_inff()) {
#pragma unroll
            for (int e = 0; e < E; ++e) sum += x[e] > -__builtin_inff() ? exp64(static_cast<double>(x[e]) - static_cast<double>(top)) : 0.0;
        }
#pragma unroll
        for (int s = 32; s > 0; s /= 2) sum += __shfl_xor(sum, s);
        if (tid % 64 == 0) sum_of[wave] = sum;
        int rank = 0;
        for (int k = 0; k < kThreads; ++k) rank += key[k] > mine || (key[k] == mine && k < tid) ? 1 : 0;
        if (rank == c.keep - 1) bar = mine;
        __syncthreads();
        // (a thread without logits has kNoKey; with a bar of that all logits pass, which are then fewer than keep * E)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = e * kThreads + tid;
            if (i < n) {
                const unsigned long long k = key_of(x[e], static_cast<uint32_t>(lo + i));
                if (k >= bar) list[atomicAdd(&found, 1)] = k;
            }
        }
        __syncthreads();
        const int m = found;
        unsigned long long* const best = c.best + static_cast<size_t>(w) * c.keep;
        for (int i = tid; i < m; i += kThreads) {
            const unsigned long long k = list[i];
            int at = 0;
            for (int j = 0; j < m; ++j) at += list[j] > k ? 1 : 0;
            if (at < c.keep) best[at] = k;
        }
        for (int i = m + tid; i < c.keep; i += kThreads) best[i] = kNoKey;
        if (tid == 0) {
            double all = sum_of[0];
#pragma unroll
            for (int k = 1; k < kWaves; ++k) all += sum_of[k];
            c.parts[w] = BeamPart{all, bad ? __builtin_nanf("") : top, 0};
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

__global__ __launch_bounds__(kThreads) void beam_group_kernel(BeamCall c, int parts) {
    constexpr int E = 4;  // candidates a thread and round
    __shared__ double sums[kBeamMostBeams], score[kBeamMostBeams];
    __shared__ int state[kBeamMostBeams];  // 0: no continuations, 1: of the logits, 2: ended
    __shared__ Candidate of_thread[kThreads], bar, list[kBeamMostKeep * (E + 1)], best[kBeamMostKeep];
    __shared__ int found, have, bad;
    const int tid = threadIdx.x, keep = c.keep;
    const double none = -__builtin_inf();
    for (int group = blockIdx.x; group < c.groups; group += gridDim.x) {
        __syncthreads();
        if (tid == 0) have = 0, bad = 0;
        __syncthreads();
        for (int b = tid; b < c.beams; b += kThreads) {
            const size_t row = static_cast<size_t>(group) * c.beams + b;
            const float s = c.scores[row];
            int what = !(s < __builtin_inff()) ? -1 : s == -__builtin_inff() ? 0 : c.ended != nullptr && c.ended[row] != 0 ? 2 : 1;
            sums[b] = 0.0;
            if (what == 1) {
                const BeamPart* const p = c.parts + row * parts;
                float top = -__builtin_inff();
                bool wrong = false;
                for (int k = 0; k < parts; ++k) {
                    const float x = p[k].largest;
                    wrong = wrong || x != x;
                    top = fmaxf(top, x);
                }
                double sum = 0.0;
                for (int k = 0; k < parts; ++k) {
                    if (p[k].largest > -__builtin_inff()) sum += p[k].sum * exp64(static_cast<double>(p[k].largest) - static_cast<double>(top));
                }
                sums[b] = static_cast<double>(top) + log(sum);
                what = wrong ? -1 : top == -__builtin_inff() ? 0 : 1;
            }
            score[b] = static_cast<double>(s);
            state[b] = what;
            if (what < 0) bad = 1;
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
        // Rounds: what is best so far, and the next candidates.
        const int per = parts * keep, n = c.beams * per;
        const unsigned long long* const keys = c.best + static_cast<size_t>(group) * n;
        for (int first = 0; first < n; first += E * kThreads) {
            Candidate mine{none, kNoKey, c.beams}, x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = first + e * kThreads + tid;
                x[e] = Candidate{none, kNoKey, c.beams};
                if (i < n) {
                    const int b = i / per;
                    if (state[b] == 1) {
                        const unsigned long long k = keys[i];
                        const float logit = logit_of(k);
                        if (k != kNoKey && logit > -__builtin_inff()) {
                            x[e] = Candidate{score[b] + (static_cast<double>(logit) - sums[b]), k, b};
                        }
                    } else if (state[b] == 2 && i % per == 0) {
                        x[e] = Candidate{score[b], key_of(0.0f, static_cast<uint32_t>(c.end_token)), b};
                    }
                }
                if (before(x[e], mine)) mine = x[e];
            }
            of_thread[tid] = mine;
            if (tid == 0) found = 0;
            __syncthreads();
            int rank = 0;
            for (int k = 0; k < kThreads; ++k) {
                const Candidate other = of_thread[k];
                rank += before(other, mine) || (k < tid && !before(mine, other)) ? 1 : 0;
            }
            if (rank == keep - 1) bar = mine;
            __syncthreads();
            const Candidate least = bar;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (x[e].beam < c.beams && !before(least, x[e])) list[atomicAdd(&found, 1)] = x[e];
            }
            for (int i = tid; i < have; i += kThreads) list[atomicAdd(&found, 1)] = best[i];
            __syncthreads();
            const int m = found;
            for (int i = tid; i < m; i += kThreads) {
                const Candidate k = list[i];
                int at = 0;
                for (int j = 0; j < m; ++j) at += before(list[j], k) ? 1 : 0;
                if (at < keep) best[at] = k;
            }
            __syncthreads();
            if (tid == 0) have = min(m, keep);
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
    const int parts = beam_parts(c.vocab);
    const long long groups = static_cast<long long>(c.groups) * c.beams * parts;
    beam_part_kernel<kBeamPart / kThreads><<<static_cast<unsigned>(std::min<long long>(groups, 1 << 20)), kThreads, 0, s>>>(c, parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    beam_group_kernel<<<std::min(c.groups, 1 << 20), kThreads, 0, s>>>(c, parts);
    return hipGetLastError();
}

}  // namespace mlq
