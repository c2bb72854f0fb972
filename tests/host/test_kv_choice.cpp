// Which of its two kernels a batch of drafted trees runs (csrc/kv_plan.h): by the tiles that each kernel's workgroups
// visit, counted here from who sees what.  And the smallest and largest positions that the items name.  No GPU.
//   test_kv_choice         random batches and three long ones
//   test_kv_choice kind    the kernel ("few" or "many") of batches on stdin:
//                          type head_dim heads kv window sinks sequences, then of each: nodes, positions before, parents

#include "../../mini-llama-cpp-release_amd/csrc/kv_plan.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <numeric>
#include <random>
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

struct Tree {
    int before;
    std::vector<int> parent;
};

int blocks(int head_dim) {
    const int nb = (head_dim + 31) / 32;
    return nb == 5 || nb == 7 ? nb + 1 : nb;
}

struct Call {
    int type, head_dim, heads, kv, window, sinks;
    std::vector<Tree> trees;

    KvPlanShape shape() const {
        KvPlanShape s;
        s.page_size = 64;
        s.n_kv_heads = kv;
        s.group = heads / kv;
        s.wide_rows = mlq::kv_wide_rows(blocks(head_dim));
        s.window = window;
        s.sinks = sinks;
        s.max_seqs = std::max<int>(1, trees.size());
        s.max_tokens = s.max_pages = s.max_nodes = 1;
        for (const Tree& t : trees) {
            const int n = t.parent.size();
            s.max_tokens += n;
            s.max_pages += (t.before + n + 63) / 64;
            s.max_nodes = std::max(s.max_nodes, n);
        }
        s.n_pages = s.max_pages;
        s.tree_cost = mlq::kv_tree_cost(type, blocks(head_dim));
        return s;
    }
    KvBatch build() const {
        const KvPlanShape s = shape();
        std::vector<int> nodes, len, parents, pages(s.max_pages);
        for (const Tree& t : trees) {
            nodes.push_back(t.parent.size());
            len.push_back(t.before + t.parent.size());
            parents.insert(parents.end(), t.parent.begin(), t.parent.end());
        }
        std::iota(pages.begin(), pages.end(), 0);
        KvBatch b;
        const std::string wrong = mlq::kv_plan_build(s, trees.size(), nodes.data(), len.data(), pages.data(), parents.data(), &b);
        CHECK(wrong.empty(), "%s", wrong.c_str());
        return b;
    }
};

// The workgroups' tiles and the workgroups, for every KV head.
struct Work {
    double tiles, groups;
};

// What the kernel whose workgroups take `step` rows visits: of each group of rows the tiles from the window of its
// first position (or from the tree's first tile) to its last node's, and whole tiles of first positions below those.
Work work(const Call& c, int step) {
    Work sum{0, 0};
    const int group = c.heads / c.kv;
    for (const Tree& t : c.trees) {
        std::vector<int> pos;
        for (int p : t.parent) pos.push_back(p < 0 ? t.before : pos[p] + 1);
        const int rows = t.parent.size() * group;
        for (int r = 0; r < rows; r += step) {
            const int first = r / group, last = (std::min(rows, r + step) - 1) / group;
            const int near = *std::min_element(pos.begin() + first, pos.begin() + last + 1);
            for (int tile = 0; 32 * tile <= t.before + last; ++tile) {
                const bool windowed = c.window == 0 || 32 * tile + 31 > near - c.window || 32 * tile + 31 >= t.before;
                sum.tiles += windowed || 32 * tile < c.sinks ? c.kv : 0;
            }
            sum.groups += c.kv;
        }
    }
    return sum;
}

// Checks the choice, and returns it.
int check(const Call& c, const char* what) {
    const KvBatch b = c.build();
    const KvPlanShape s = c.shape();
    const Work by[2] = {work(c, mlq::kKvTreeRows), work(c, s.wide_rows)};
    const double few = by[0].tiles * s.tree_cost.few + by[0].groups * s.tree_cost.each;
    const double many = by[1].tiles * s.tree_cost.many + s.tree_cost.fill;
    CHECK(b.trees[0].empty() || b.trees[1].empty(), "%s: both kernels", what);
    const int kind = b.trees[1].empty() ? 0 : 1;
    double visited = 0;
    for (const KvTreeItem& it : b.trees[kind]) {
        visited += it.count;
        const int step = kind == 0 ? mlq::kKvTreeRows : s.wide_rows;
        const int* const pos = b.pos.data() + it.token0;
        const int first = it.row0 / s.group, last = (std::min(it.new_tokens * s.group, it.row0 + step) - 1) / s.group;
        CHECK(it.near == *std::min_element(pos + first, pos + last + 1), "%s: near %d", what, it.near);
        CHECK(it.far == *std::max_element(pos + first, pos + last + 1), "%s: far %d", what, it.far);
    }
    CHECK(visited * c.kv == by[kind].tiles, "%s: %.0f tiles", what, visited);
    // (sums of products of floats: equal ones may fall either way)
    if (std::abs(few - many) > 1e-6 * many) {
        CHECK(kind == (few <= many ? 0 : 1), "%s: few rows %.1f us, many %.1f, runs %s", what, few / 1e3, many / 1e3, kind == 0 ? "few" : "many");
    }
    return kind;
}

Tree tree(std::mt19937& rng, int nodes, int before) {
    Tree t{before, {}};
    const int back = 1 + static_cast<int>(rng() % 6);
    for (int i = 0; i < nodes; ++i) t.parent.push_back(i == 0 ? -1 : i - 1 - static_cast<int>(rng() % std::min(i, back)));
    return t;
}

int of(std::mt19937& rng, std::initializer_list<int> x) { return *(x.begin() + rng() % x.size()); }

}  // namespace

int main(int argc, char** argv) {
    if (argc > 1 && std::strcmp(argv[1], "kind") == 0) {
        Call c;
        int seqs;
        while (std::scanf("%d %d %d %d %d %d %d", &c.type, &c.head_dim, &c.heads, &c.kv, &c.window, &c.sinks, &seqs) == 7) {
            c.trees.assign(seqs, Tree{});
            for (Tree& t : c.trees) {
                int nodes;
                if (std::scanf("%d %d", &nodes, &t.before) != 2) return 1;
                t.parent.resize(nodes);
                for (int& p : t.parent) {
                    if (std::scanf("%d", &p) != 1) return 1;
                }
            }
            std::puts(check(c, "batch") == 0 ? "few" : "many");
        }
        return 0;
    }
    std::mt19937 rng(5);
    int kinds[2] = {0, 0};
    for (int trial = 0; trial < 1800; ++trial) {
        Call c;
        c.type = rng() % 4;
        c.head_dim = of(rng, {32, 64, 80, 128, 192, 256});
        c.kv = of(rng, {1, 2, 8});
        c.heads = c.kv * of(rng, {1, 2, 4, 7});
        c.window = of(rng, {0, 1, 40, 64, 300, 1024, 2147483647});
        c.sinks = c.window ? of(rng, {0, 1, 40, 500, 2147483647}) : 0;
        const int seqs = of(rng, {1, 3, 16}), nodes = of(rng, {1, 8, 24, 100, 256}), before = of(rng, {0, 31, 700, 3000, 9000});
        for (int i = 0; i < seqs; ++i) c.trees.push_back(tree(rng, nodes - i % 2 * (nodes / 3), before + 7 * i));
        ++kinds[check(c, ("trial " + std::to_string(trial)).c_str())];
    }
    CHECK(kinds[0] > 50 && kinds[1] > 50, "%d and %d batches", kinds[0], kinds[1]);
    // Long contexts: all of it takes the kernel for many rows, a window the other.
    struct {
        int type, head_dim, heads, kv, seqs, nodes, before, window;
    } const cases[] = {{1, 128, 32, 8, 1, 256, 8000, 64}, {1, 128, 32, 8, 8, 64, 8000, 256}, {3, 80, 32, 8, 16, 24, 3000, 1024},
                       {0, 128, 32, 8, 4, 32, 8000, 512}};
    for (const auto& k : cases) {
        Call c{k.type, k.head_dim, k.heads, k.kv, 0, 0, {}};
        for (int i = 0; i < k.seqs; ++i) c.trees.push_back(tree(rng, k.nodes, k.before));
        CHECK(check(c, "without a window") == 1, "type %d: %d nodes after %d", k.type, k.nodes, k.before);
        c.window = k.window;
        CHECK(check(c, "with a window") == 0, "type %d: %d nodes after %d, window %d", k.type, k.nodes, k.before, k.window);
    }
    std::printf("PASS kv_choice\n");
    return 0;
}
