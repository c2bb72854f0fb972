// Greedy picks of a batch of drafted trees, and the paths of nodes that they confirm.
//
// pick of a node = first index of the largest of its logits, -1 where one is not finite.  A sequence's path
// starts at its first node and goes on to the lowest child whose token is the last node's pick.
//
// One launch: a workgroup finds the largest key of a part of a row (pick_key.h orders by value, then by lower index, so
// the order of the parts has no say), and the one that is last to have done so for a sequence walks its tree.

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

struct Walk {
    unsigned long long key[kKvMostNodes];
    int parent[kKvMostNodes], token[kKvMostNodes], pick[kKvMostNodes], path[kKvMostNodes];
};

// The picks of a sequence's nodes from their parts' keys, then, in one wave, its path, node by node.
__device__ __forceinline__ void walk(const KvPick& p, int seq, const KvTreeSeq& q, int parts, Walk& w) {
    for (int i = threadIdx.x; i < q.nodes; i += kThreads) {
        w.key[i] = 0;
        w.parent[i] = p.lists.parents[q.token0 + i];
        w.token[i] = p.tokens[q.token0 + i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < q.nodes * parts; i += kThreads) {
        const unsigned long long* const from = p.keys + static_cast<size_t>(q.token0) * parts + i;
        atomicMax(&w.key[i / parts], __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < q.nodes; i += kThreads) p.picks[q.token0 + i] = w.pick[i] = pick_token(w.key[i]);
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x;
    int here = 0, n = 0, next = -1;
    while (here >= 0) {
        if (lane == 0) w.path[n] = here;
        ++n;
        next = w.pick[here];
        int child = -1;
        // (children come after their parent)
        for (int i = here + 1; next >= 0 && child < 0 && i < q.nodes; i += 64) {
            const bool fits = i + lane < q.nodes && w.parent[i + lane] == here && w.token[i + lane] == next;
            const unsigned long long found = __ballot(fits);
            if (found != 0) child = i + __builtin_ctzll(found);
        }
        here = child;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int i = lane; i < q.nodes; i += 64) p.kept[q.token0 + i] = i < n ? w.path[i] : -1;
    if (lane == 0) {
        p.n_kept[seq] = n;
        p.next[seq] = next;
    }
}

// Bound: memory (the logits once: 315 rows of 152000, 32 us, 6 TB/s, part of it from the last-level cache); of few rows, launch, a trip for the logits, one for the arrival, one for the keys and
// the walk.
__global__ __launch_bounds__(kThreads) void kv_pick_kernel(KvPick p, int tokens, int seqs) {
    __shared__ unsigned long long of_wave[kThreads / 64];
    __shared__ unsigned last;
    __shared__ Walk tree;
    const int rows = tokens >= 0 ? tokens : p.lists.counts[kKvCountTokens], vocab = p.vocab;
    const int parts = parts_of(rows, vocab);
    const long long total = static_cast<long long>(rows) * parts;
    for (long long w = blockIdx.x; w < total; w += gridDim.x) {
        const int part = static_cast<int>(w % parts), row_index = static_cast<int>(w / parts);
        const int seq = p.lists.seq_of[row_index];
        const float* const row = p.logits + static_cast<size_t>(row_index) * vocab;
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
        __syncthreads();  // the last part's readers are done
        if (threadIdx.x % 64 == 0) of_wave[threadIdx.x / 64] = key;
        __syncthreads();
        const KvTreeSeq q = p.lists.seqs[seq];
        if (threadIdx.x == 0) {
#pragma unroll
            for (int k = 1; k < kThreads / 64; ++k) key = larger(key, of_wave[k]);
            // Through to the point of coherence, as other workgroups' are read from there.
            __hip_atomic_store(&p.keys[w], key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            unsigned* const arrived = p.arrived + static_cast<size_t>(seq) * kKvPickApart;
            const unsigned all = static_cast<unsigned>(q.nodes) * parts;
            last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == all ? 1u : 0u;
            if (last != 0u) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (last != 0u) walk(p, seq, q, parts, tree);
    }
    // Empty trees.
    const int all = seqs >= 0 ? seqs : p.lists.counts[kKvCountSeqs];
    for (int s = blockIdx.x * kThreads + threadIdx.x; s < all; s += gridDim.x * kThreads) {
        if (p.lists.seqs[s].nodes == 0) {
            p.n_kept[s] = 0;
            p.next[s] = -1;
        }
    }
}

}  // namespace

hipError_t launch_kv_pick(const KvPick& p, int tokens, int seqs, hipStream_t s) {
    const long long groups = tokens >= 0 ? static_cast<long long>(tokens) * parts_of(tokens, p.vocab) : kKvPickParts;
    kv_pick_kernel<<<static_cast<unsigned>(std::max(1ll, std::min<long long>(groups, 1 << 20))), kThreads, 0, s>>>(p, tokens, seqs);
    return hipGetLastError();
}

}  // namespace mlq
