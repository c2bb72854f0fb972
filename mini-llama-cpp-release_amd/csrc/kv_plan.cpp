// Batches over the paged key/value cache: checks and work lists (kv_plan.h).

#include "kv_plan.h"

#include <algorithm>

namespace mlq {
namespace {

// A split makes workgroups until there are this many, two a CU, and no more.  Measured at a head_dim of
// 128, where either kernel's registers allow two: one token over 100000 positions (Q4_0, 8 KV heads), 256 /
// 512 / 1024 of them: 48 / 46 / 57 us; 8 sequences of 4000 (Q8_0) 21 / 21 / 26.  (Above 128 one fits a CU and
// these are two rounds, at 64 three or four fit: not tuned.)
constexpr int kTargetGroups = 512;
// Fewer tiles than this are not split further, as the parts' merge would cost more.  One token over
// 4000 positions, at least 4 / 8 / 16 tiles: 14.9 / 12.8 / 13.8 us; over 700 9.6 / 10.3 / 11.6; 128 rows
// over 4000 53 / 46 / 54.
constexpr int kLeastTiles = 8;
// Few rows of trees: a tile a wave where that makes no more workgroups than there are CUs and a merge of a few parts.
// At least 8 and 4 tiles, us with the write: 16 nodes after 700 positions (Q4_0, 32 heads over 8 of 128, 192
// workgroups) 17.5 and 16.5, after 1500 (384) 18.2 and 19.5; 4 nodes after 1500 (Q8_0, 14 heads over 2 of 64, 12
// parts) 13.6 and 13.3, after 4000 (32) 14.5 and 15.4; 4 x 8 nodes after 300 (f32, 32 heads of 128) 19.2 and 17.0.
constexpr int kFewTiles = 4, kFewParts = 16, kFewGroups = 256;

int ceil_div(int a, int b) { return a / b + (a % b != 0); }  // (sinks go up to the largest int)

// Tiles that query rows at positions lo .. hi can see, in the numbering of KvAttnItem.
struct Seen {
    int sinks, shift, count;
};

// (`most`: of a position in the first tile of the window.)
Seen seen_tiles(const KvPlanShape& s, int lo, int hi, int most) {
    const int last = hi / kKvTile;
    const int first = s.window > 0 ? std::max(0, std::min(most, lo - s.window + 1)) / kKvTile : 0;
    // the sinks are first positions: below `first` they are whole tiles of their own
    const int sinks = s.window > 0 ? std::min(first, ceil_div(s.sinks, kKvTile)) : 0;
    return Seen{sinks, first - sinks, sinks + last - first + 1};
}

// Adds the items of `whole` to `list`, split along their tiles where there are too few: parts of at most
// `most` tiles, as even as they come: the fewest tiles that do not make more items than `target`, since those
// beyond one round of workgroups would take a second one.
// Where there is a round without splits, only items of twice the average are split if `lone` (64 ragged
// sequences of up to 4000: 79 us, 85 with those over the average split).
// (Not a prompt's row groups, whose lengths are spread: 2048 tokens, 32 heads: 167 us, 193 unsplit.)
// few: the items are few rows of trees.
template <typename Item>
void split_items(const std::vector<Item>& whole, int n_kv_heads, bool lone, bool few, int groups, std::vector<Item>& list) {
    int64_t tiles = 0;
    for (const Item& w : whole) tiles += w.count;
    const int target = std::max(1, groups / n_kv_heads);
    auto items_of = [&](int64_t most) {
        int64_t n = 0;
        for (const Item& w : whole) n += (w.count + most - 1) / most;
        return n;
    };
    const bool enough = static_cast<int>(whole.size()) >= target;
    int longest = 0;
    for (const Item& w : whole) longest = std::max(longest, w.count);
    few = few && longest <= kFewParts * kFewTiles && items_of(kFewTiles) * n_kv_heads <= kFewGroups;
    int64_t lo = std::max<int64_t>(few ? kFewTiles : kLeastTiles, (enough && lone ? 2 : 1) * ((tiles + target - 1) / target)), hi = lo;
    hi = std::max<int64_t>(hi, longest);
    while (lo < hi && !enough) {
        const int64_t mid = (lo + hi) / 2;
        if (items_of(mid) <= target) hi = mid;
        else lo = mid + 1;
    }
    const int most = static_cast<int>(std::max<int64_t>(1, lo));
    int slot = 0;
    for (const Item& w : whole) {
        const int parts = ceil_div(w.count, most);
        for (int p = 0; p < parts; ++p) {
            Item it = w;
            it.first = static_cast<int>(static_cast<int64_t>(w.count) * p / parts);
            it.count = static_cast<int>(static_cast<int64_t>(w.count) * (p + 1) / parts) - it.first;
            it.split = p;
            it.nsplit = parts;
            it.slot = slot;
            list.push_back(it);
        }
        if (parts > 1) slot += parts;
    }
    // The longest first: what starts last is short.
    std::stable_sort(list.begin(), list.end(), [](const Item& x, const Item& y) { return x.count > y.count; });
}

// The tree of one sequence, n nodes after `start` positions: checks `parents` (null: a chain) and adds positions,
// parents and bits to the batch.  Bit k of node i's word w: whether it sees position 32 (start / 32 + w) + k,
// counted in slots.
std::string add_tree(const KvPlanShape& s, const std::string& who, int n, int start, const int* parents, KvBatch& b) {
    const int t0 = start / kKvTile, words = (start + n - 1) / kKvTile - t0 + 1, base = start % kKvTile;
    const size_t first = b.masks.size(), pos0 = b.pos.size();
    b.masks.resize(first + static_cast<size_t>(n) * words, 0);
    for (int i = 0; i < n; ++i) {
        const int parent = parents != nullptr ? parents[i] : i - 1;
        if (parent < -1 || parent >= i) {
            return who + ": node " + std::to_string(i) + " has parent " + std::to_string(parent) + ", not -1 or an earlier node";
        }
        b.parents.push_back(parent);
        b.holds.push_back(i);
        const int pos = parent < 0 ? start : b.pos[pos0 + parent] + 1;
        b.pos.push_back(pos);
        uint32_t* const mask = &b.masks[first + static_cast<size_t>(i) * words];
        const int lo = s.window > 0 ? pos - s.window : -1;  // positions up to here are seen as sinks only
        auto set = [&](int bit) { mask[bit / kKvTile] |= 1u << (bit % kKvTile); };
        if (lo < start && parent >= 0) {
            // all nodes of the path are seen
            const uint32_t* const of_parent = &b.masks[first + static_cast<size_t>(parent) * words];
            std::copy(of_parent, of_parent + words, mask);
            mask[0] &= ~((1u << base) - 1u);
        } else {
            for (int p = parent; p >= 0; p = b.parents[pos0 + p]) {
                if (b.pos[pos0 + p] > lo || b.pos[pos0 + p] < s.sinks) set(base + p);
            }
        }
        for (int k = 0; k < base; ++k) {
            const int p = t0 * kKvTile + k;
            if (p > lo || p < s.sinks) set(k);
        }
        set(base + i);
    }
    return "";
}

}  // namespace

int kv_wide_rows(int nb) { return nb <= 4 ? 128 : 64; }

// Measured, us by the kernel for few rows and the one for many (8 KV heads of 128, rows a KV head and sequence x
// sequences x positions): Q8_0 64 x 1 x 4000 17 and 45, 256 x 1 x 4000 31 and 49, 32 x 32 x 2000 48 and 121, 96 x 16 x 3000
// 106 and 105, 256 x 16 x 2000 182 and 127; Q4_1 96 x 16 x 3000 134 and 113; f32 128 x 4 x 3000 93 and 62, 256 x 16 x 2000
// 446 and 171.  Per tile that is about as much a block of 32 elements.  Beside its tiles, which a window may leave few of,
// a workgroup of the first holds its place for 3 us (launch, trips to memory, the waves' merge), for 8 where it has its CU
// to itself.  Of 1400 random batches of all types, 32 to 256 elements, with and without windows, the chosen kernel takes
// 1.0 % longer than the better one on average, 3.9 % without those, 5.4 % where tiles outside the windows count as well.
KvTreeCost kv_tree_cost(int qtype, int nb) {
    constexpr float kFew[4] = {0.74f, 0.33f, 0.32f, 0.40f}, kMany[4] = {2.0f, 1.3f, 1.25f, 1.5f};
    // Above 128 elements (f32: 64) a SIMD has one wave of the kernel for few rows, so more workgroups than CUs are two rounds:
    // 4 x 8 nodes after 1500 positions of f32, 32 heads over 8 of 128, in 512 33 us, in 256 24; 16 after 4000 of Q4_1 of
    // 192 elements 41 and 32.  (A workgroup of the other has half the rows above 128.)
    const int groups = nb > (qtype == 0 ? 2 : 4) ? 256 : 512;
    return KvTreeCost{kFew[qtype] * nb * (nb > 4 ? 1.3f : 1.0f), kMany[qtype] * nb, 14000.0f + 4000.0f * nb, groups,
                      groups == 256 ? 30.0f : 6.0f};
}

KvPlanLimits kv_plan_limits(const KvPlanShape& s) {
    const int64_t rows = static_cast<int64_t>(s.max_tokens) * s.group;
    const int64_t narrow = std::min(rows / kKvNarrowRows, static_cast<int64_t>(s.max_seqs) * (kKvNarrowMost / kKvNarrowRows - 1));
    int whole[2] = {static_cast<int>(narrow) + s.max_seqs, static_cast<int>(rows / s.wide_rows) + s.max_seqs};
    KvPlanLimits l;
    if (s.max_nodes > 0) {
        whole[0] = static_cast<int>(rows / kKvTreeRows) + s.max_seqs;
        // (a node's bits begin inside a tile at the most)
        l.masks = static_cast<int64_t>(s.max_tokens) * (s.max_nodes / kKvTile + 2);
    }
    // a sequence's new tokens begin and end inside a tile at the most
    l.fresh = static_cast<int>(std::min<int64_t>(s.max_tokens, s.max_tokens / kKvTile + 2ll * s.max_seqs));
    for (int kind = 0; kind < 2; ++kind) {
        // Only an item of n parts adds to the list, n - 1 items, and all parts take slots: at
        // most twice what is added.
        const int groups = s.max_nodes > 0 ? std::max(kTargetGroups, s.tree_cost.groups) : kTargetGroups;
        const int extra = ceil_div(groups, s.n_kv_heads);
        l.items[kind] = whole[kind] + extra;
        l.slots[kind] = 2 * extra;
    }
    return l;
}

std::string kv_plan_build(const KvPlanShape& s, int n_seqs, const int* new_tokens, const int* kv_len, const int* pages,
                          const int* parents, KvBatch* out) {
    if (n_seqs < 0 || n_seqs > s.max_seqs) {
        return std::to_string(n_seqs) + " sequences, the plan holds " + std::to_string(s.max_seqs);
    }
    if (n_seqs > 0 && (new_tokens == nullptr || kv_len == nullptr)) return "null lengths";
    int64_t tokens = 0, entries = 0, positions = 0;
    for (int i = 0; i < n_seqs; ++i) {
        const std::string who = "sequence " + std::to_string(i);
        if (new_tokens[i] < 0) return who + ": negative token count";
        if (kv_len[i] < new_tokens[i]) {
            return who + ": " + std::to_string(new_tokens[i]) + " new tokens in a length of " + std::to_string(kv_len[i]);
        }
        if (s.max_nodes > 0 && new_tokens[i] > s.max_nodes) {
            return who + ": " + std::to_string(new_tokens[i]) + " nodes, the plan's trees hold " + std::to_string(s.max_nodes);
        }
        tokens += new_tokens[i];
        positions += kv_len[i];
        entries += kv_len[i] / s.page_size + (kv_len[i] % s.page_size != 0);
    }
    if (tokens > s.max_tokens) {
        return std::to_string(tokens) + " new tokens, the plan holds " + std::to_string(s.max_tokens);
    }
    if (entries > s.max_pages) {
        return std::to_string(entries) + " page entries, the plan holds " + std::to_string(s.max_pages);
    }
    if (entries > 0 && pages == nullptr) return "null page list";
    for (int64_t e = 0; e < entries; ++e) {
        if (pages[e] < 0 || pages[e] >= s.n_pages) {
            return "page entry " + std::to_string(e) + " is " + std::to_string(pages[e]) + ", the cache has " +
                   std::to_string(s.n_pages) + " pages";
        }
    }

    KvBatch& b = *out;
    b = KvBatch();
    b.n_tokens = static_cast<int>(tokens);
    b.n_positions = static_cast<int>(positions);

    // Pages, tiles, and the slots new tokens go to (page, first and last slot in the page).
    struct Written {
        int page, lo, hi;
    };
    std::vector<Written> written;
    std::vector<KvAttnItem> base[2];
    std::vector<KvTreeItem> of_trees[2];
    int token0 = 0, row0 = 0, page0 = 0;
    std::vector<int> mask0;  // of each sequence's tree
    for (int i = 0; i < n_seqs; ++i) {
        const int len = kv_len[i], n = new_tokens[i], start = len - n;
        for (int p = 0; p < len; p += s.page_size) {
            b.pages.push_back(KvPage{pages[page0 + p / s.page_size], std::min(s.page_size, len - p), row0 + p});
        }
        for (int p = start; p < len;) {
            const int end = std::min(len, (p / kKvTile + 1) * kKvTile);
            b.fresh.push_back(KvTileItem{pages[page0 + p / s.page_size], p % s.page_size / kKvTile, p % kKvTile, end - p,
                                         token0 + p - start, p});
            p = end;
        }
        for (int p = start; p < len;) {
            const int end = std::min(len, (p / s.page_size + 1) * s.page_size);
            written.push_back(Written{pages[page0 + p / s.page_size], p % s.page_size, (end - 1) % s.page_size});
            p = end;
        }
        if (s.max_nodes > 0) {
            mask0.push_back(static_cast<int>(b.masks.size()));
            if (n > 0) {
                const std::string wrong =
                    add_tree(s, "sequence " + std::to_string(i), n, start, parents != nullptr ? parents + token0 : nullptr, b);
                if (!wrong.empty()) return wrong;
            }
            b.seqs.push_back(KvTreeSeq{token0, n});
            b.seq_of.insert(b.seq_of.end(), n, i);
            b.starts.push_back(start);
            b.first_page.push_back(page0);
        } else if (n > 0) {
            const int rows = n * s.group;
            const int kind = rows <= kKvNarrowMost ? 0 : 1;
            base[kind].push_back(KvAttnItem{token0, n, len, page0, 0, 0, 0, 0, 0, 0, 1, 0});
        }
        token0 += n;
        row0 += len;
        page0 += len / s.page_size + (len % s.page_size != 0);
    }
    std::sort(written.begin(), written.end(), [](const Written& x, const Written& y) {
        return x.page != y.page ? x.page < y.page : x.lo < y.lo;
    });
    for (size_t k = 1; k < written.size(); ++k) {
        if (written[k].page == written[k - 1].page && written[k].lo <= written[k - 1].hi) {
            return "page " + std::to_string(written[k].page) + " takes two new tokens in slot " + std::to_string(written[k].lo);
        }
    }

    if (s.max_nodes > 0) {
        // The row groups of either kernel, and the kernel that takes less for all of them, by the tiles that they visit (two
        // launches would follow each other).  256 nodes after 8000 positions with a window of 64 (Q8_0, 32 heads over 8 of
        // 128): 13 us by the kernel for few rows, 32 by the other, which takes less where all positions are seen.
        double cost[2] = {0.0, s.tree_cost.fill};
        for (int kind = 0; kind < 2; ++kind) {
            if (cost[0] <= cost[1] && kind == 1) break;  // (whatever the second visits)
            const int step = kind == 0 ? kKvTreeRows : s.wide_rows;
            of_trees[kind].reserve(static_cast<size_t>(b.n_tokens) * s.group / step + n_seqs);
            for (int i = 0; i < n_seqs; ++i) {
                const int n = new_tokens[i], start = kv_len[i] - n, rows = n * s.group, token = b.seqs[i].token0;
                const int words = n > 0 ? (kv_len[i] - 1) / kKvTile - start / kKvTile + 1 : 0;
                for (int r = 0; r < rows; r += step) {
                    const int last = (std::min(rows, r + step) - 1) / s.group;
                    int near = b.pos[token + r / s.group], far = near;
                    for (int t = r / s.group; t <= last; ++t) {
                        near = std::min(near, b.pos[token + t]);
                        far = std::max(far, b.pos[token + t]);
                    }
                    // (from the tree's first tile at the latest: a node may be seen as a sink wherever it lies)
                    const Seen t = seen_tiles(s, near, start + last, start);
                    of_trees[kind].push_back(KvTreeItem{token, n, kv_len[i], b.first_page[i], r, 0, t.count, t.sinks, t.shift, 0, 1, 0,
                                                        mask0[i], words, near, far});
                    cost[kind] += s.n_kv_heads * (kind == 0 ? s.tree_cost.few * static_cast<double>(t.count) + s.tree_cost.each
                                                            : s.tree_cost.many * static_cast<double>(t.count));
                }
            }
        }
        of_trees[cost[0] <= cost[1] ? 1 : 0].clear();
    }
    for (int kind = 0; kind < 2; ++kind) {
        split_items(of_trees[kind], s.n_kv_heads, true, kind == 0, kind == 0 ? s.tree_cost.groups : kTargetGroups, b.trees[kind]);
        const int step = kind == 0 ? kKvNarrowRows : s.wide_rows;
        std::vector<KvAttnItem> whole;
        for (const KvAttnItem& q : base[kind]) {
            const int rows = q.new_tokens * s.group, start = q.len - q.new_tokens;
            for (int r = 0; r < rows; r += step) {
                const Seen t = seen_tiles(s, start + r / s.group, start + (std::min(rows, r + step) - 1) / s.group, q.len);
                KvAttnItem it = q;
                it.row0 = r;
                it.count = t.count;
                it.sinks = t.sinks;
                it.shift = t.shift;
                whole.push_back(it);
            }
        }
        split_items(whole, s.n_kv_heads, kind == 0, false, kTargetGroups, b.items[kind]);
    }
    return "";
}

std::string kv_keep_build(const KvPlanShape& s, const KvBatch& b, const int* n_kept, const int* kept, std::vector<KvMove>* moves,
                          std::vector<int>* ends) {
    moves->clear();
    ends->clear();
    if (!b.seqs.empty() && n_kept == nullptr) return "null counts";
    size_t at = 0;
    int64_t total = 0;
    for (size_t i = 0; i < b.seqs.size(); ++i) {
        const std::string who = "sequence " + std::to_string(i);
        if (n_kept[i] < 0 || n_kept[i] > b.seqs[i].nodes) {
            return who + ": " + std::to_string(n_kept[i]) + " of " + std::to_string(b.seqs[i].nodes) + " nodes kept";
        }
        total += n_kept[i];
    }
    if (total > 0 && kept == nullptr) return "null list";
    for (size_t i = 0; i < b.seqs.size(); ++i) {
        const KvTreeSeq& q = b.seqs[i];
        for (int j = 0; j < n_kept[i]; ++j) {
            const int node = kept[at + j], before = j > 0 ? kept[at + j - 1] : -1;
            if (node < 0 || node >= q.nodes || b.parents[q.token0 + node] != before) {
                return "sequence " + std::to_string(i) + ": kept node " + std::to_string(node) + " is not a child of " +
                       (j > 0 ? "node " + std::to_string(before) : "what came before the tree");
            }
            if (b.holds[q.token0 + node] != node) {
                return "sequence " + std::to_string(i) + ": kept node " + std::to_string(node) + " has been moved over by node " +
                       std::to_string(b.holds[q.token0 + node]);
            }
            // A path's nodes ascend, so node j lies at slot j or later.
            if (node != j) {
                const int from = b.starts[i] + node, to = b.starts[i] + j;
                moves->push_back(KvMove{b.pages[b.first_page[i] + from / s.page_size].page, b.pages[b.first_page[i] + to / s.page_size].page,
                                        static_cast<uint16_t>(from % s.page_size), static_cast<uint16_t>(to % s.page_size)});
            }
        }
        at += n_kept[i];
        if (!moves->empty() && (ends->empty() || ends->back() != static_cast<int>(moves->size()))) {
            ends->push_back(static_cast<int>(moves->size()));
        }
    }
    return "";
}

void kv_keep_done(const int* n_kept, const int* kept, KvBatch* b) {
    for (size_t i = 0; i < b->seqs.size(); ++i) {
        std::copy(kept, kept + n_kept[i], b->holds.begin() + b->seqs[i].token0);
        kept += n_kept[i];
    }
}

}  // namespace mlq
