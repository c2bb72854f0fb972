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

// The same of a batch of trees (kv_attention_tree.h).  The sequence's nodes see each other by bits: those of its
// node i start at word mask0 + i * words of the masks, a word a tile from that of the first node on.
struct KvTreeItem {
    int token0, new_tokens, len, page0;
    int row0, first, count;
    int sinks, shift;
    int split, nsplit, slot;
    int mask0, words;
    int near, far;  // the smallest and the largest position of the item's rows
};

// A sequence of a batch of trees: its first row in the token buffers, and its nodes.
struct KvTreeSeq {
    int token0, nodes;
};

// Query rows of a workgroup of the trees' first list: the columns of an MFMA operand.
constexpr int kKvTreeRows = 16;
constexpr int kKvMostNodes = 1024;

// What the trees' two kernels take, in ns: for a tile by a workgroup of the one for few rows (16 at a time) and of the one
// for many (wide_rows at a time), what the second takes longer for filling its pipeline and merging, and what a workgroup
// of the first takes beside its tiles.  A batch runs the one that takes less.
struct KvTreeCost {
    float few = 1.0f, many = 5.0f, fill = 30000.0f;
    int groups = 512;  // workgroups of the first that the chip holds at once
    float each = 0.0f;
};
KvTreeCost kv_tree_cost(int qtype, int nb);  // of heads of nb blocks of 32 elements
// Query rows of a workgroup of the kernel for many rows.
int kv_wide_rows(int nb);

struct KvPlanShape {
    int page_size, n_pages, n_kv_heads;
    int group;      // query heads per KV head
    int wide_rows;  // query rows of a workgroup of the kernel for many rows
    int window, sinks;
    int max_seqs, max_tokens, max_pages;
    int max_nodes = 0;  // of a sequence's tree; 0: batches of plain sequences
    KvTreeCost tree_cost = {};
};

// What a set of a plan of this shape can need at the most.
struct KvPlanLimits {
    int fresh;     // tiles with new tokens
    int items[2];  // narrow, wide (of trees: few rows, many)
    int slots[2];  // partial results
    int64_t masks = 0;  // words of the trees' bits
};
KvPlanLimits kv_plan_limits(const KvPlanShape& s);

struct KvBatch {
    int n_tokens = 0, n_positions = 0;
    std::vector<KvTileItem> fresh;     // tiles with new tokens
    std::vector<KvPage> pages;
    std::vector<KvAttnItem> items[2];  // narrow, wide
    // Of trees, in place of `items`.
    std::vector<KvTreeItem> trees[2];
    std::vector<KvTreeSeq> seqs;
    std::vector<int> starts, first_page;  // of each sequence: positions before its tree, first entry in `pages`
    std::vector<int> pos, parents, seq_of;  // of each token: its position, the parent among its sequence's nodes, the sequence
    std::vector<uint32_t> masks;
    std::vector<int> holds;  // which of its tree's nodes lies in each token's slot (moves change it)
};

// Checks a batch and builds its lists.  Returns "" or what is wrong with it;
// `out` is complete only on "".  parents: of shapes with max_nodes, each new token's
// parent among its sequence's new tokens, an earlier one, or -1 (null: chains).
std::string kv_plan_build(const KvPlanShape& s, int n_seqs, const int* new_tokens, const int* kv_len, const int* pages,
                          const int* parents, KvBatch* out);
inline std::string kv_plan_build(const KvPlanShape& s, int n_seqs, const int* new_tokens, const int* kv_len, const int* pages,
                                 KvBatch* out) {
    return kv_plan_build(s, n_seqs, new_tokens, kv_len, pages, nullptr, out);
}

// Moves of a path's tokens behind what came before the tree: slots of the cache's pages.
struct KvMove {
    int from_page, to_page;
    uint16_t from_slot, to_slot;  // (a page has 65536 at the most)
};
// Checks what is kept of a batch (of each sequence n_kept[s] of its new tokens, each the child of the one before)
// and lists the moves, one sequence's after the other's, `ends` the list's length after each sequence that has some.
std::string kv_keep_build(const KvPlanShape& s, const KvBatch& b, const int* n_kept, const int* kept, std::vector<KvMove>* moves,
                          std::vector<int>* ends);
// Notes what its moves have left in the slots.
void kv_keep_done(const int* n_kept, const int* kept, KvBatch* b);

}  // namespace mlq
