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

int ceil_div(int a, int b) { return a / b + (a % b != 0); }  // (sinks go up to the largest int)

// Tiles that query rows at positions lo .. hi can see, in the numbering of KvAttnItem.
struct Seen {
    int sinks, shift, count;
};

Seen seen_tiles(const KvPlanShape& s, int lo, int hi) {
    const int last = hi / kKvTile;
    const int first = s.window > 0 ? std::max(0, lo - s.window + 1) / kKvTile : 0;
    // the sinks are first positions: below `first` they are whole tiles of their own
    const int sinks = s.window > 0 ? std::min(first, ceil_div(s.sinks, kKvTile)) : 0;
    return Seen{sinks, first - sinks, sinks + last - first + 1};
}

}  // namespace

KvPlanLimits kv_plan_limits(const KvPlanShape& s) {
    const int64_t rows = static_cast<int64_t>(s.max_tokens) * s.group;
    const int64_t narrow = std::min(rows / kKvNarrowRows, static_cast<int64_t>(s.max_seqs) * (kKvNarrowMost / kKvNarrowRows - 1));
    const int whole[2] = {static_cast<int>(narrow) + s.max_seqs, static_cast<int>(rows / s.wide_rows) + s.max_seqs};
    KvPlanLimits l;
    // a sequence's new tokens begin and end inside a tile at the most
    l.fresh = static_cast<int>(std::min<int64_t>(s.max_tokens, s.max_tokens / kKvTile + 2ll * s.max_seqs));
    for (int kind = 0; kind < 2; ++kind) {
        // Only an item of n parts adds to the list, n - 1 items, and all parts take slots: at
        // most twice what is added.
        const int extra = ceil_div(kTargetGroups, s.n_kv_heads);
        l.items[kind] = whole[kind] + extra;
        l.slots[kind] = 2 * extra;
    }
    return l;
}

std::string kv_plan_build(const KvPlanShape& s, int n_seqs, const int* new_tokens, const int* kv_len, const int* pages,
                          KvBatch* out) {
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
    int token0 = 0, row0 = 0, page0 = 0;
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
        if (n > 0) {
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

    for (int kind = 0; kind < 2; ++kind) {
        const int step = kind == 0 ? kKvNarrowRows : s.wide_rows;
        std::vector<KvAttnItem> whole;
        int64_t tiles = 0;
        for (const KvAttnItem& q : base[kind]) {
            const int rows = q.new_tokens * s.group, start = q.len - q.new_tokens;
            for (int r = 0; r < rows; r += step) {
                const Seen t = seen_tiles(s, start + r / s.group, start + (std::min(rows, r + step) - 1) / s.group);
                KvAttnItem it = q;
                it.row0 = r;
                it.count = t.count;
                it.sinks = t.sinks;
                it.shift = t.shift;
                tiles += t.count;
                whole.push_back(it);
            }
        }
        // Parts of at most `most` tiles, as even as they come: the fewest tiles that do not make more
        // items than `target`, since those beyond one round of workgroups would take a second one.
        std::vector<KvAttnItem>& list = b.items[kind];
        const int target = std::max(1, kTargetGroups / s.n_kv_heads);
        auto items_of = [&](int64_t most) {
            int64_t n = 0;
            for (const KvAttnItem& w : whole) n += (w.count + most - 1) / most;
            return n;
        };
        // Where there is a round without splits, only items of twice the average are split (64 ragged
        // sequences of up to 4000: 79 us, 85 with those over the average split).
        // (Not a prompt's row groups, whose lengths are spread: 2048 tokens, 32 heads: 167 us, 193 unsplit.)
        const bool enough = static_cast<int>(whole.size()) >= target;
        int64_t lo = std::max<int64_t>(kLeastTiles, (enough && kind == 0 ? 2 : 1) * ((tiles + target - 1) / target)), hi = lo;
        for (const KvAttnItem& w : whole) hi = std::max<int64_t>(hi, w.count);
        while (lo < hi && !enough) {
            const int64_t mid = (lo + hi) / 2;
            if (items_of(mid) <= target) hi = mid;
            else lo = mid + 1;
        }
        const int most = static_cast<int>(std::max<int64_t>(1, lo));
        int slot = 0;
        for (const KvAttnItem& w : whole) {
            const int parts = ceil_div(w.count, most);
            for (int p = 0; p < parts; ++p) {
                KvAttnItem it = w;
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
        std::stable_sort(list.begin(), list.end(),
                         [](const KvAttnItem& x, const KvAttnItem& y) { return x.count > y.count; });
    }
    return "";
}

}  // namespace mlq
