// paged_joins.cu — the division of paged attention calls into shares, followed
// on the host with the kernels' own arithmetic: which ticket words and which
// places of the workspace every row tile uses.  Two row tiles of one call may
// share neither, whatever the lengths.
//
// Input: one call a line, "ctas kernel causal kv_heads group n_seq" (kernel 0:
// mma.sync, 1: tcgen05) and n_seq pairs "new_tokens kv_len".  Output, a line
// each: cut tiles, the most parts of one, tiles joined in groups, groups of one
// part, tiles whose last CTA starts the next cut tile behind a group of one,
// words or places that two tiles use, parts that hold no unit.
#include <algorithm>
#include <cstdio>
#include <set>
#include <vector>

#include "../../p100_b200/csrc/fa_paged_tc.cuh"

using namespace p100b;

namespace {

struct Tile {
    long long first;
    int units;
};

template <int ROWS, int KEYS, int OVER>
std::vector<Tile> tiles_of(const paged::Desc& d, const std::vector<int>& lens, long long* total) {
    std::vector<Tile> tiles;
    long long at = 0;
    for (int s = 0; s < d.n_seq; ++s)
        for (int h = 0; h < d.n_head_kv; ++h)
            for (int t = 0; t < paged::row_tiles<ROWS>(d, lens[2 * s]); ++t) {
                tiles.push_back({at, paged::tile_units<ROWS, KEYS>(d, lens[2 * s], lens[2 * s + 1], t)});
                at += tiles.back().units + OVER;
            }
    *total = at;
    return tiles;
}

struct Result {
    int cut = 0, most = 0, grouped = 0, ones = 0, followed = 0, shared = 0, empty = 0;
};

Result follow(const std::vector<Tile>& tiles, long long total, int parts, int ctas, bool mma) {
    Result r;
    std::set<long long> words, places;
    int one_at = -1;   // the CTA of the last tile's group of one
    for (const Tile& t : tiles) {
        const int c0 = paged::share_of(t.first, total, parts), c1 = paged::share_of(t.first + t.units - 1, total, parts);
        if (c0 == c1) continue;   // whole
        ++r.cut;
        const int np = c1 - c0 + 1;
        r.most = std::max(r.most, np);
        if (one_at == c0) ++r.followed;
        one_at = -1;
        for (int c = c0; c <= c1; ++c) {
            const long long lo = std::max(t.first, paged::share_begin(total, c, parts));
            const long long hi = std::min(t.first + t.units, paged::share_begin(total, c + 1, parts));
            if (lo >= hi) ++r.empty;
            if (!places.insert(2 * c + (lo == t.first)).second) ++r.shared;
        }
        if (!mma) {
            if (!words.insert(c0).second) ++r.shared;
            continue;
        }
        const fap::Joins joins(np);
        for (int first = 0; first < np; first += joins.per) {
            if (joins.size_of(first) == 1) {
                ++r.ones;
                if (c0 + first == c1) one_at = c1;
            }
            if (joins.counts(first) && !words.insert(c0 + first).second) ++r.shared;
        }
        if (joins.groups > 1) {
            ++r.grouped;
            if (!words.insert(ctas + c0).second) ++r.shared;
        }
    }
    return r;
}

}  // namespace

int main() {
    int ctas, kernel, causal, kv_heads, group, n_seq;
    while (std::scanf("%d %d %d %d %d %d", &ctas, &kernel, &causal, &kv_heads, &group, &n_seq) == 6) {
        std::vector<int> lens(2 * n_seq);
        for (int& v : lens)
            if (std::scanf("%d", &v) != 1) return 1;
        paged::Desc d = {};
        d.n_seq = n_seq;
        d.n_head_kv = kv_heads;
        d.group = group;
        d.causal = causal;
        long long total;
        Result r;
        if (kernel == 0) {
            const auto tiles = tiles_of<fap::kRows, fap::kKeys, fap::kOver>(d, lens, &total);
            r = follow(tiles, total, fap::shares(total, ctas), ctas, true);
        } else {
            const auto tiles = tiles_of<fatc::kRows, fatc::kKeys, fatc::kOver>(d, lens, &total);
            r = follow(tiles, total, int(std::min<long long>(ctas, total)), ctas, false);
        }
        std::printf("%d %d %d %d %d %d %d\n", r.cut, r.most, r.grouped, r.ones, r.followed, r.shared, r.empty);
    }
    return 0;
}
