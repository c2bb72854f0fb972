// The work lists of the paged cache (csrc/kv_plan.h) against what they have to
// cover, over random shapes and batches, and every refusal.  No GPU.

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

using mlq::KvAttnItem;
using mlq::KvBatch;
using mlq::KvPlanShape;

int pick(std::mt19937& rng, std::initializer_list<int> of) { return *(of.begin() + rng() % of.size()); }

bool sees(const KvPlanShape& s, int pos, int j) {
    return j <= pos && (s.window == 0 || j > pos - s.window || j < s.sinks);
}

void one(std::mt19937& rng, int trial) {
    KvPlanShape s;
    s.page_size = pick(rng, {32, 64, 256, 4096});
    s.n_kv_heads = pick(rng, {1, 2, 8, 32});
    s.group = pick(rng, {1, 2, 7, 8, 16});
    s.wide_rows = pick(rng, {128, 256});
    s.window = pick(rng, {0, 0, 1, 20, 32, 33, 100, 1000, 2147483647});
    s.sinks = s.window ? pick(rng, {0, 1, 4, 32, 40, 3000, 2147483647}) : 0;
    const int n_seqs = rng() % 6;
    std::vector<int> fresh(n_seqs), len(n_seqs), pages;
    int tokens = 0, entries = 0;
    const int longest = pick(rng, {1, 40, 700, 5000});
    for (int i = 0; i < n_seqs; ++i) {
        len[i] = rng() % (longest + 1);
        fresh[i] = len[i] == 0 ? 0 : pick(rng, {0, 1, 1, 2, static_cast<int>(rng() % len[i]) + 1});
        if (fresh[i] > len[i]) fresh[i] = len[i];
        tokens += fresh[i];
        entries += (len[i] + s.page_size - 1) / s.page_size;
    }
    s.n_pages = entries + 3;
    std::vector<int> ids(s.n_pages);
    for (int i = 0; i < s.n_pages; ++i) ids[i] = i;
    std::shuffle(ids.begin(), ids.end(), rng);
    pages.assign(ids.begin(), ids.begin() + entries);
    s.max_seqs = std::max(1, n_seqs);
    s.max_tokens = std::max(1, tokens);
    s.max_pages = std::max(1, entries);

    KvBatch b;
    const std::string wrong = mlq::kv_plan_build(s, n_seqs, fresh.data(), len.data(), pages.data(), &b);
    CHECK(wrong.empty(), "trial %d: %s", trial, wrong.c_str());
    const mlq::KvPlanLimits lim = mlq::kv_plan_limits(s);
    CHECK(static_cast<int>(b.fresh.size()) <= lim.fresh && lim.fresh <= s.max_tokens, "trial %d", trial);
    CHECK(static_cast<int>(b.pages.size()) == entries, "trial %d", trial);
    CHECK(b.n_tokens == tokens, "trial %d", trial);

    // Pages and new tokens.
    std::vector<std::pair<int, int>> want, got;  // (page * page_size + slot, position) by token row
    int e = 0, row = 0;
    for (int i = 0; i < n_seqs; ++i) {
        const int first = e;
        for (int p = 0; p < len[i]; p += s.page_size, ++e) {
            CHECK(b.pages[e].page == pages[e] && b.pages[e].row == row + p &&
                      b.pages[e].n == std::min(s.page_size, len[i] - p), "trial %d entry %d", trial, e);
        }
        for (int p = len[i] - fresh[i]; p < len[i]; ++p) want.push_back({pages[first + p / s.page_size] * s.page_size + p % s.page_size, p});
        row += len[i];
    }
    got.resize(want.size(), {-1, -1});
    for (const mlq::KvTileItem& t : b.fresh) {
        CHECK(t.n > 0 && t.slot >= 0 && t.slot + t.n <= mlq::kKvTile && t.tile < s.page_size / mlq::kKvTile, "trial %d", trial);
        for (int k = 0; k < t.n; ++k) {
            CHECK(t.row + k < tokens && got[t.row + k].first == -1, "trial %d", trial);
            got[t.row + k] = {t.page * s.page_size + t.tile * mlq::kKvTile + t.slot + k, t.pos + k};
        }
    }
    CHECK(want == got, "trial %d", trial);

    // Attention: every (row, tile it sees) in exactly one place; other tiles may come along.
    std::map<std::pair<int, int>, int> covered;  // (token row * group + head, tile)
    std::map<int, std::set<int>> parts;
    for (int kind = 0; kind < 2; ++kind) {
        CHECK(static_cast<int>(b.items[kind].size()) <= lim.items[kind], "trial %d", trial);
        const int step = kind == 0 ? mlq::kKvNarrowRows : s.wide_rows;
        for (const KvAttnItem& it : b.items[kind]) {
            CHECK(it.count > 0 && it.first >= 0 && it.split < it.nsplit, "trial %d", trial);
            if (it.nsplit > 1) {
                CHECK(it.slot >= 0 && it.slot + it.nsplit <= lim.slots[kind], "trial %d: slot %d of %d", trial, it.slot, lim.slots[kind]);
                CHECK(parts[2 * it.slot + kind].insert(it.split).second, "trial %d", trial);
            }
            const int rows = it.new_tokens * s.group;
            CHECK(it.row0 < rows && it.row0 % step == 0, "trial %d", trial);
            for (int k = it.first; k < it.first + it.count; ++k) {
                const int tile = k < it.sinks ? k : k + it.shift;
                CHECK(tile * mlq::kKvTile < it.len, "trial %d: tile %d of a length of %d", trial, tile, it.len);
                for (int r = it.row0; r < std::min(rows, it.row0 + step); ++r) ++covered[{it.token0 * s.group + r, tile}];
            }
        }
    }
    for (const auto& c : covered) CHECK(c.second == 1, "trial %d: row %d tile %d", trial, c.first.first, c.first.second);
    int token = 0;
    for (int i = 0; i < n_seqs; ++i) {
        for (int k = 0; k < fresh[i]; ++k, ++token) {
            const int pos = len[i] - fresh[i] + k;
            for (int t = 0; t * mlq::kKvTile <= pos; ++t) {
                bool any = false;
                for (int j = t * mlq::kKvTile; j < (t + 1) * mlq::kKvTile && !any; ++j) any = sees(s, pos, j);
                if (!any) continue;
                for (int h = 0; h < s.group; ++h) {
                    CHECK(covered.count({token * s.group + h, t}) == 1, "trial %d: token %d tile %d", trial, token, t);
                }
            }
        }
    }
}

void refused(const KvPlanShape& s, std::vector<int> fresh, std::vector<int> len, std::vector<int> pages, const char* what) {
    KvBatch b;
    const std::string wrong = mlq::kv_plan_build(s, static_cast<int>(fresh.size()), fresh.data(), len.data(), pages.data(), &b);
    CHECK(wrong.find(what) != std::string::npos, "\"%s\" in \"%s\"", what, wrong.c_str());
}

}  // namespace

int main() {
    std::mt19937 rng(7);
    for (int t = 0; t < 200; ++t) one(rng, t);
    const KvPlanShape s{64, 10, 2, 4, 256, 0, 0, 3, 100, 6};
    refused(s, {1, 1, 1, 1}, {1, 1, 1, 1}, {0, 1, 2, 3}, "4 sequences, the plan holds 3");
    refused(s, {-1}, {4}, {0}, "negative token count");
    refused(s, {5}, {4}, {0}, "5 new tokens in a length of 4");
    refused(s, {0}, {-3}, {}, "0 new tokens in a length of -3");
    refused(s, {101}, {101}, {0, 1}, "101 new tokens, the plan holds 100");
    refused(s, {1}, {400}, {0, 1, 2, 3, 4, 5, 6}, "7 page entries, the plan holds 6");
    refused(s, {1}, {2147483647}, {0}, "page entries, the plan holds 6");
    refused(s, {1}, {65}, {0, 10}, "page entry 1 is 10, the cache has 10 pages");
    refused(s, {1}, {65}, {-1, 1}, "page entry 0 is -1");
    refused(s, {2, 1}, {66, 1}, {3, 4, 4}, "page 4 takes two new tokens in slot 0");
    refused(s, {70}, {70}, {5, 5}, "page 5 takes two new tokens in slot 0");
    KvBatch b;
    CHECK(mlq::kv_plan_build(s, -1, nullptr, nullptr, nullptr, &b) != "", "negative count");
    CHECK(mlq::kv_plan_build(s, 1, nullptr, nullptr, nullptr, &b) == "null lengths", "null lengths");
    const int one_new = 1, four = 4;
    CHECK(mlq::kv_plan_build(s, 1, &one_new, &four, nullptr, &b) == "null page list", "null pages");
    CHECK(mlq::kv_plan_build(s, 0, nullptr, nullptr, nullptr, &b) == "", "an empty batch");
    // A page may be read by several sequences, and written in slots of their own.
    const int n2[2] = {1, 1}, l2[2] = {70, 72}, p2[4] = {1, 2, 1, 2};
    CHECK(mlq::kv_plan_build(s, 2, n2, l2, p2, &b) == "", "shared pages");
    std::printf("PASS kv_plan\n");
    return 0;
}
