// Host side of a batch over the paged key/value cache: checks what the caller
// describes and lays out the work lists that the kernels walk.  Plain C++
// without HIP, so it is tested on the CPU.
#pragma once

#include <cstdint>
#include <string>
#include <vector>

namespace mlq {

constexpr int kKvTile = 32;       // positions per tile: the depth of one MFMA over keys
constexpr int kKvNarrowRows = 8;  // query rows of a workgroup of the kernel for few rows (fp16 hi and lo parts side by side)
// Rows of a sequence up to which it runs them.  64 rows over 4000 positions (Q8_0) 21 us, 45 in the
// kernel for many rows; 128 rows 30 and 46; 16 such sequences of 2000 85 and 77, 150 and 78.  (The number of
// sequences has no say, so one of 128 rows takes the slower kernel.)
constexpr int kKvNarrowMost = 64;
constexpr int kKvWaves = 4;       // waves of an attention workgroup

// New tokens in one tile: positions pos .. pos + n - 1 at slots slot .. of tile
// `tile` of page `page`, rows row .. of the caller's token buffers.
struct KvTileItem {
    int page, tile, slot, n, row, pos;
};

// An entry of the page list: the page, how many of its slots the sequence holds, and
// the row of the first among all positions of the batch.
struct KvPage {
    int page, n, row;
};

// One workgroup's share of the attention, for every KV head: query rows row0 ..
// (row = token * group + query head of the group) of one sequence over `count` of
// its tiles.  The tiles a row can see are numbered without the gap between the
// first tiles that stay visible (`sinks` of them) and the window: tile i is i
// below `sinks` and i + shift from there.
struct KvAttnItem {
    int token0, new_tokens, len, page0;  // the sequence: first row in q, new tokens, positions, first entry in the page list
    int row0, first, count;
    int sinks, shift;
    int split, nsplit, slot;  // part `split` of nsplit; the parts' first slot in the partial results
};

struct KvPlanShape {
    int page_size, n_pages, n_kv_heads;
    int group;      // query heads per KV head
    int wide_rows;  // query rows of a workgroup of the kernel for many rows
    int window, sinks;
    int max_seqs, max_tokens, max_pages;
};

// What a set of a plan of this shape can need at the most.
struct KvPlanLimits {
    int fresh;     // tiles with new tokens
    int items[2];  // narrow, wide
    int slots[2];  // partial results
};
KvPlanLimits kv_plan_limits(const KvPlanShape& s);

struct KvBatch {
    int n_tokens = 0, n_positions = 0;
    std::vector<KvTileItem> fresh;     // tiles with new tokens
    std::vector<KvPage> pages;
    std::vector<KvAttnItem> items[2];  // narrow, wide
};

// Checks a batch and builds its lists.  Returns "" or what is wrong with it;
// `out` is complete only on "".
std::string kv_plan_build(const KvPlanShape& s, int n_seqs, const int* new_tokens, const int* kv_len, const int* pages,
                          KvBatch* out);

}  // namespace mlq
