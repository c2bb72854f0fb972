// The work lists of batches of drafted trees and the moves of what is kept of them (csrc/kv_plan.h)
// against what they have to cover, over random shapes and trees, and every refusal.  No GPU.

#include "../../mini-llama-cpp-release_amd/csrc/kv_plan.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <string>
#include <vector>

namespace {

#define CHECK(cond, ...)                                      \
    do {                                                      \
        if (!(cond)) {                                        \
            std::printf("FAIL %s:%d %s: ", __FILE__, __LINE__, #cond); \
            std::printf(__VA_ARGS__);                         \
            std::printf("\n");                                \
            std::exit(1);                                     \
        }                                                     \
    } while (0)

using mlq::KvBatch;
using mlq::KvPlanShape;
using mlq::KvTreeItem;

int pick(std::mt19937& rng, std::initializer_list<int> of) { return *(of.begin() + rng() % of.size()); }

// A sequence's tree: parents and depths of its nodes.
struct Tree {
    std::vector<int> parent, depth;
};

Tree grow(std::mt19937& rng, int n) {
    Tree t;
    const int back = pick(rng, {1, 2, 5, 1000}), roots = pick(rng, {1, 1, 3});
    for (int i = 0; i < n; ++i) {
        const int p = i < roots ? -1 : i - 1 - static_cast<int>(rng() % std::min(i, back));
        t.parent.push_back(p);
        t.depth.push_back(p < 0 ? 0 : t.depth[p] + 1);
    }
    return t;
}

// Whether node i of a tree after `start` positions sees slot j.
bool sees(const KvPlanShape& s, const Tree& t, int start, int i, int j) {
    const int pos = start + t.depth[i];
    int at = j;
    if (j >= start) {
        int p = i;
        while (p >= 0 && p != j - start) p = t.parent[p];
        if (p < 0) return false;
        at = start + t.depth[j - start];
    }
    return s.window == 0 || at > pos - s.window || at < s.sinks;
}

void one(std::mt19937& rng, int trial) {
    KvPlanShape s;
    s.page_size = pick(rng, {32, 64, 256});
    s.n_kv_heads = pick(rng, {1, 2, 8, 32});
    s.group = pick(rng, {1, 2, 7, 8, 16});
    s.wide_rows = 128;
    s.window = pick(rng, {0, 0, 1, 3, 20, 33, 100, 2147483647});
    s.sinks = s.window ? pick(rng, {0, 1, 4, 40, 2147483647}) : 0;
    s.tree_cost.fill = static_cast<float>(pick(rng, {0, 100, 30000, 1000000}));
    const int n_seqs = rng() % 5;
    std::vector<int> nodes(n_seqs), len(n_seqs), parents, pages;
    std::vector<Tree> trees;
    int tokens = 0, entries = 0, most = 1;
    for (int i = 0; i < n_seqs; ++i) {
        nodes[i] = pick(rng, {0, 1, 2, 17, 40, 65, 130});
        len[i] = nodes[i] + pick(rng, {0, 0, 1, 31, 32, 33, 500, 2000});
        trees.push_back(grow(rng, nodes[i]));
        parents.insert(parents.end(), trees.back().parent.begin(), trees.back().parent.end());
        tokens += nodes[i];
        most = std::max(most, nodes[i]);
        entries += (len[i] + s.page_size - 1) / s.page_size;
    }
    s.n_pages = entries + 3;
    for (int i = 0; i < s.n_pages; ++i) pages.push_back(i);
    std::shuffle(pages.begin(), pages.end(), rng);
    pages.resize(entries);
    s.max_seqs = std::max(1, n_seqs);
    s.max_tokens = std::max(1, tokens);
    s.max_pages = std::max(1, entries);
    s.max_nodes = most;

    KvBatch b;
    const std::string wrong = mlq::kv_plan_build(s, n_seqs, nodes.data(), len.data(), pages.data(), parents.data(), &b);
    CHECK(wrong.empty(), "trial %d: %s", trial, wrong.c_str());
    const mlq::KvPlanLimits lim = mlq::kv_plan_limits(s);
    CHECK(static_cast<int64_t>(b.masks.size()) <= lim.masks, "trial %d", trial);
    CHECK(b.items[0].empty() && b.items[1].empty(), "trial %d", trial);
    CHECK(static_cast<int>(b.seqs.size()) == n_seqs && static_cast<int>(b.pos.size()) == tokens && b.parents == parents, "trial %d", trial);

    // Every (row, slot it sees) in exactly one item, and no other slot of a node's tiles.
    std::map<std::pair<int, int>, int> covered;  // (token * group + head, tile)
    std::map<int, std::set<int>> parts;
    for (int kind = 0; kind < 2; ++kind) {
        CHECK(static_cast<int>(b.trees[kind].size()) <= lim.items[kind], "trial %d: %d items", trial, static_cast<int>(b.trees[kind].size()));
        const int step = kind == 0 ? mlq::kKvTreeRows : s.wide_rows;
        for (const KvTreeItem& it : b.trees[kind]) {
            CHECK(it.count > 0 && it.first >= 0 && it.split < it.nsplit, "trial %d", trial);
            if (it.nsplit > 1) {
                CHECK(it.slot >= 0 && it.slot + it.nsplit <= lim.slots[kind], "trial %d", trial);
                CHECK(parts[2 * it.slot + kind].insert(it.split).second, "trial %d", trial);
            }
            int seq = 0;
            while (b.seqs[seq].token0 != it.token0 || b.seqs[seq].nodes == 0) ++seq;
            const Tree& t = trees[seq];
            const int start = it.len - it.new_tokens, rows = it.new_tokens * s.group;
            CHECK(it.row0 < rows && it.row0 % step == 0 && it.len == len[seq], "trial %d", trial);
            CHECK(it.words == (it.len - 1) / 32 - start / 32 + 1, "trial %d", trial);
            for (int r = it.row0; r < std::min(rows, it.row0 + step); ++r) {
                const int node = r / s.group;
                CHECK(b.pos[it.token0 + node] == start + t.depth[node] && it.far >= start + t.depth[node], "trial %d", trial);
                for (int k = it.first; k < it.first + it.count; ++k) {
                    const int tile = k < it.sinks ? k : k + it.shift;
                    CHECK(tile * 32 < it.len, "trial %d: tile %d of a length of %d", trial, tile, it.len);
                    ++covered[{it.token0 * s.group + r, tile}];
                    if (tile < start / 32) continue;
                    const uint32_t word = b.masks[it.mask0 + node * it.words + tile - start / 32];
                    for (int j = 0; j < 32; ++j) {
                        const int slot = tile * 32 + j;
                        const bool want = slot < it.len && sees(s, t, start, node, slot);
                        CHECK(((word >> j & 1u) != 0) == want, "trial %d: node %d slot %d of %d, start %d", trial, node, slot, it.len, start);
                    }
                }
            }
        }
    }
    for (const auto& c : covered) CHECK(c.second == 1, "trial %d: row %d tile %d", trial, c.first.first, c.first.second);
    for (int i = 0; i < n_seqs; ++i) {
        const int start = len[i] - nodes[i];
        for (int k = 0; k < nodes[i]; ++k) {
            for (int j = 0; j < len[i]; ++j) {
                if (!sees(s, trees[i], start, k, j)) continue;
                for (int h = 0; h < s.group; ++h) {
                    CHECK(covered.count({(b.seqs[i].token0 + k) * s.group + h, j / 32}) == 1, "trial %d: node %d slot %d", trial, k, j);
                }
            }
        }
    }

    // What is kept: the path to a node of each tree.
    std::vector<int> n_kept, kept;
    std::map<std::pair<int, int>, std::pair<int, int>> want;  // destination -> source (page, slot)
    int page0 = 0;
    for (int i = 0; i < n_seqs; ++i) {
        std::vector<int> path;
        if (nodes[i] > 0 && rng() % 4 != 0) {
            for (int p = static_cast<int>(rng() % nodes[i]); p >= 0; p = trees[i].parent[p]) path.insert(path.begin(), p);
        }
        n_kept.push_back(static_cast<int>(path.size()));
        kept.insert(kept.end(), path.begin(), path.end());
        auto at = [&](int slot) { return std::make_pair(pages[page0 + slot / s.page_size], slot % s.page_size); };
        for (size_t j = 0; j < path.size(); ++j) {
            if (path[j] != static_cast<int>(j)) want[at(len[i] - nodes[i] + static_cast<int>(j))] = at(len[i] - nodes[i] + path[j]);
        }
        page0 += (len[i] + s.page_size - 1) / s.page_size;
    }
    std::vector<mlq::KvMove> moves;
    std::vector<int> ends;
    const std::string bad = mlq::kv_keep_build(s, b, n_kept.data(), kept.data(), &moves, &ends);
    CHECK(bad.empty(), "trial %d: %s", trial, bad.c_str());
    CHECK(moves.size() == want.size() && (moves.empty() ? ends.empty() : ends.back() == static_cast<int>(moves.size())), "trial %d", trial);
    std::set<std::pair<int, int>> written;
    int before = 0;
    for (int e : ends) {
        CHECK(e > before, "trial %d", trial);
        written.clear();
        for (int k = before; k < e; ++k) {
            const mlq::KvMove& m = moves[k];
            const std::pair<int, int> from{m.from_page, m.from_slot}, to{m.to_page, m.to_slot};
            CHECK(want.count(to) == 1 && want[to] == from, "trial %d", trial);
            // a source is never what an earlier move of the path has written
            CHECK(written.count(from) == 0, "trial %d", trial);
            written.insert(to);
        }
        before = e;
    }
}

KvBatch batch;

void refused(const KvPlanShape& s, std::vector<int> nodes, std::vector<int> len, std::vector<int> parents, const char* what) {
    const int pages[6] = {0, 1, 2, 3, 4, 5};
    const std::string wrong =
        mlq::kv_plan_build(s, static_cast<int>(nodes.size()), nodes.data(), len.data(), pages, parents.data(), &batch);
    CHECK(wrong.find(what) != std::string::npos, "\"%s\" in \"%s\"", what, wrong.c_str());
}

void not_kept(const KvPlanShape& s, std::vector<int> n_kept, std::vector<int> kept, const char* what) {
    std::vector<mlq::KvMove> moves;
    std::vector<int> ends;
    const std::string wrong = mlq::kv_keep_build(s, batch, n_kept.data(), kept.data(), &moves, &ends);
    CHECK(wrong.find(what) != std::string::npos, "\"%s\" in \"%s\"", what, wrong.c_str());
}

}  // namespace

int main() {
    std::mt19937 rng(11);
    for (int t = 0; t < 300; ++t) one(rng, t);
    KvPlanShape s{64, 10, 2, 4, 256, 0, 0, 3, 100, 6, 8, {}};
    refused(s, {9}, {9}, {-1, 0, 1, 2, 3, 4, 5, 6, 7}, "sequence 0: 9 nodes, the plan's trees hold 8");
    refused(s, {2}, {5}, {-1, 1}, "sequence 0: node 1 has parent 1");
    refused(s, {1, 3}, {5, 3}, {-1, -1, 0, 5}, "sequence 1: node 2 has parent 5");
    refused(s, {2}, {5}, {0, 0}, "node 0 has parent 0");
    refused(s, {2}, {5}, {-2, 0}, "node 0 has parent -2");
    // two roots, and a chain where there are no parents
    const int n2[2] = {4, 3}, l2[2] = {4, 70}, p2[3] = {1, 2, 3}, up[7] = {-1, -1, 0, 2, -1, 0, 0};
    CHECK(mlq::kv_plan_build(s, 2, n2, l2, p2, nullptr, &batch) == "" && batch.parents == std::vector<int>({-1, 0, 1, 2, -1, 0, 1}), "chains");
    CHECK(mlq::kv_plan_build(s, 2, n2, l2, p2, up, &batch) == "", "two trees");
    not_kept(s, {5, 0}, {0, 2, 3, 3, 3}, "sequence 0: 5 of 4 nodes kept");
    not_kept(s, {-1, 0}, {}, "sequence 0: -1 of 4 nodes kept");
    not_kept(s, {2, 0}, {0, 1}, "sequence 0: kept node 1 is not a child of node 0");
    not_kept(s, {1, 0}, {2}, "sequence 0: kept node 2 is not a child of what came before the tree");
    not_kept(s, {0, 2}, {0, 3}, "sequence 1: kept node 3 is not a child of node 0");
    not_kept(s, {0, 2}, {0, -1}, "sequence 1: kept node -1");
    not_kept(s, {2, 1}, {1, 0, 0}, "sequence 0: kept node 0 is not a child of node 1");
    std::vector<mlq::KvMove> moves;
    std::vector<int> ends;
    CHECK(mlq::kv_keep_build(s, batch, nullptr, nullptr, &moves, &ends) == "null counts", "null counts");
    const int some[2] = {0, 1}, none[2] = {0, 0};
    CHECK(mlq::kv_keep_build(s, batch, some, nullptr, &moves, &ends) == "null list", "null list");
    CHECK(mlq::kv_keep_build(s, batch, none, nullptr, &moves, &ends) == "" && moves.empty() && ends.empty(), "nothing kept");
    // What has been moved over is not kept any more; what lies in place, or has not been moved over, is.
    const int path_n[2] = {3, 2}, path[5] = {0, 2, 3, 0, 2};
    CHECK(mlq::kv_plan_build(s, 2, n2, l2, p2, up, &batch) == "", "two trees");
    CHECK(mlq::kv_keep_build(s, batch, path_n, path, &moves, &ends) == "" && moves.size() == 3, "a path");
    mlq::kv_keep_done(path_n, path, &batch);
    CHECK(batch.holds == std::vector<int>({0, 2, 3, 3, 0, 2, 2}), "what the slots hold");
    not_kept(s, {3, 2}, {0, 2, 3, 0, 2}, "sequence 0: kept node 2 has been moved over by node 3");
    not_kept(s, {1, 0}, {1}, "sequence 0: kept node 1 has been moved over by node 2");
    not_kept(s, {0, 2}, {0, 1}, "sequence 1: kept node 1 has been moved over by node 2");
    const int again_n[2] = {1, 2}, again[3] = {0, 0, 2};
    CHECK(mlq::kv_keep_build(s, batch, again_n, again, &moves, &ends) == "" && moves.size() == 1, "a path that can be moved again");
    std::printf("PASS kv_tree\n");
    return 0;
}
