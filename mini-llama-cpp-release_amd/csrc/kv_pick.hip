// Greedy picks of a batch of drafted trees, and the paths of nodes that they confirm.
//
// pick of a node = first index of the largest of its logits, -1 where one is not finite.  A sequence's path
// starts at its first node and goes on to the lowest child whose token is the last node's pick.
//
// Two launches: the picks, as the largest key of every part of a row (pick_key.h orders by value, then by lower
// index, so the order of the parts has no say), and the paths, a workgroup a sequence.

#include "kv_layout.h"
#include "pick_key.h"

#include <algorithm>

namespace mlq {
namespace {

constexpr int kThreads = 256;
constexpr int kLeastPart = 2048;  // logits

// Parts of a row: workgroups enough for the chip where the rows are few.
__host__ __device__ inline int parts_of(int rows, int vocab) {
    const int most = kKvPickParts / (rows > 0 ? rows : 1), useful = (vocab + kLeastPart - 1) / kLeastPart;
    const int parts = most < useful ? most : useful;
    return parts > 1 ? parts : 1;
}

__device__ __forceinline__ unsigned long long larger(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

__device__ __forceinline__ unsigned long long wave_largest(unsigned long long k) {
#pragma unroll
    for (int s = 32; s > 0; s /= 2) k = larger(k, __shfl_xor(k, s));
    return k;
}

// Bound: memory (the logits once).
__global__ __launch_bounds__(kThreads) void kv_pick_kernel(KvPick p, int tokens) {
    __shared__ unsigned long long of_wave[kThreads / 64];
    const int rows = tokens > 0 ? tokens : p.lists.counts[kKvCountTokens], vocab = p.vocab;
    const int parts = parts_of(rows, vocab);
    const long long total = static_cast<long long>(rows) * parts;
    for (long long w = blockIdx.x; w < total; w += gridDim.x) {
        const int part = static_cast<int>(w % parts);
        const float* const row = p.logits + static_cast<size_t>(w / parts) * vocab;
        const int lo = static_cast<int>(static_cast<long long>(vocab) * part / parts);
        const int hi = static_cast<int>(static_cast<long long>(vocab) * (part + 1) / parts);
        float best = -__builtin_inff();
        int at = lo;
        bool bad = false;
        auto take = [&](float x, int i) {
            bad = bad || !(fabsf(x) < __builtin_inff());
            at = x > best ? i : at;
            best = x > best ? x : best;
        };
        int i = lo + threadIdx.x;
        for (; i + 7 * kThreads < hi; i += 8 * kThreads) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = row[i + k * kThreads];
#pragma unroll
            for (int k = 0; k < 8; ++k) take(x[k], i + k * kThreads);
        }
        for (; i < hi; i += kThreads) take(row[i], i);
        // (a thread without logits has no say)
        unsigned long long key = bad ? ~0ull : best > -__builtin_inff() ? pick_key(best, at) : 0ull;
        key = wave_largest(key);
        __syncthreads();
        if (threadIdx.x % 64 == 0) of_wave[threadIdx.x / 64] = key;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int k = 1; k < kThreads / 64; ++k) key = larger(key, of_wave[k]);
            p.keys[w] = key;
        }
    }
}

// Bound: latency.  The picks of a sequence's nodes, then, in one wave, its path, node by node.
__global__ __launch_bounds__(kThreads) void kv_path_kernel(KvPick p, int tokens, int seqs) {
    __shared__ int parent[kKvMostNodes], token[kKvMostNodes], pick[kKvMostNodes], path[kKvMostNodes];
    const int rows = tokens > 0 ? tokens : p.lists.counts[kKvCountTokens];
    const int total = seqs > 0 ? seqs : p.lists.counts[kKvCountSeqs];
    const int parts = parts_of(rows, p.vocab);
    for (int s = blockIdx.x; s < total; s += gridDim.x) {
        const KvTreeSeq q = p.lists.seqs[s];
        __syncthreads();  // the last sequence's reader is done
        for (int i = threadIdx.x; i < q.nodes; i += kThreads) {
            unsigned long long key = 0;
            for (int k = 0; k < parts; ++k) key = larger(key, p.keys[static_cast<size_t>(q.token0 + i) * parts + k]);
            pick[i] = pick_token(key);
            p.picks[q.token0 + i] = pick[i];
            parent[i] = p.lists.parents[q.token0 + i];
            token[i] = p.tokens[q.token0 + i];
        }
        __syncthreads();
        if (threadIdx.x >= 64) continue;
        const int lane = threadIdx.x;
        int here = q.nodes > 0 ? 0 : -1, n = 0, next = -1;
        while (here >= 0) {
            if (lane == 0) path[n] = here;
            ++n;
            next = pick[here];
            int child = -1;
            // (children come after their parent)
            for (int i = here + 1; next >= 0 && child < 0 && i < q.nodes; i += 64) {
                const bool fits = i + lane < q.nodes && parent[i + lane] == here && token[i + lane] == next;
                const unsigned long long found = __ballot(fits);
                if (found != 0) child = i + __builtin_ctzll(found);
            }
            here = child;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int i = lane; i < q.nodes; i += 64) p.kept[q.token0 + i] = i < n ? path[i] : -1;
        if (lane == 0) {
            p.n_kept[s] = n;
            p.next[s] = next;
        }
    }
}

}  // namespace

hipError_t launch_kv_pick(const KvPick& p, int tokens, int seqs, hipStream_t s) {
    const long long groups = static_cast<long long>(tokens) * parts_of(tokens, p.vocab);
    if (tokens >= 0 && groups > 0) {
        kv_pick_kernel<<<static_cast<unsigned>(std::min<long long>(groups, 1 << 20)), kThreads, 0, s>>>(p, tokens);
    } else if (tokens < 0) {
        kv_pick_kernel<<<kKvPickParts, kThreads, 0, s>>>(p, 0);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    kv_path_kernel<<<seqs > 0 ? std::min(seqs, 1 << 20) : kKvPickParts / 4, kThreads, 0, s>>>(p, std::max(tokens, 0), std::max(seqs, 0));
    return hipGetLastError();
}

}  // namespace mlq
