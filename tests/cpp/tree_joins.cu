// tree_joins.cu — the division of tree attention calls into shares, followed on
// the host with the kernel's own arithmetic: which place of the workspace every
// part of a cut row tile uses, and which CTA notes the cut for the joining kernel.
//
// Input: one call a line, "ctas kv_heads group n_seq" and n_seq pairs "new_tokens
// kv_len".  Output, a line each: cut tiles, the most parts of one, places or
// notes that two tiles use, parts that hold no unit, shares without a unit.
#include <algorithm>
#include <cstdio>
#include <set>
#include <vector>

#include "../../p100_b200/csrc/fa_tree.cuh"

using namespace p100b;

int main() {
    int ctas, kv_heads, group, n_seq;
    while (std::scanf("%d %d %d %d", &ctas, &kv_heads, &group, &n_seq) == 4) {
        paged::Desc d = {};
        d.n_seq = n_seq;
        d.n_head_kv = kv_heads;
        d.group = group;
        std::vector<int> lens(2 * n_seq);
        for (int& v : lens)
            if (std::scanf("%d", &v) != 1) return 1;
        struct Tile {
            long long first;
            int units;
        };
        std::vector<Tile> tiles;
        long long total = 0;
        for (int s = 0; s < n_seq; ++s)
            for (int h = 0; h < kv_heads; ++h)
                for (int t = 0; t < paged::row_tiles<fatr::kRows>(d, lens[2 * s]); ++t) {
                    tiles.push_back({total, paged::tile_units<fatr::kRows, fatr::kKeys>(d, lens[2 * s], lens[2 * s + 1], t)});
                    total += tiles.back().units + fatr::kOver;
                }
        const int parts = fatr::shares(total, ctas);
        int cut = 0, most = 0, shared = 0, empty = 0, thin = 0;
        std::set<long long> places;
        std::set<int> notes;
        for (const Tile& t : tiles) {
            const int c0 = paged::share_of(t.first, total, parts), c1 = paged::share_of(t.first + t.units - 1, total, parts);
            if (c0 == c1) continue;   // whole
            ++cut;
            most = std::max(most, c1 - c0 + 1);
            if (!notes.insert(c0).second) ++shared;
            for (int c = c0; c <= c1; ++c) {
                const long long lo = std::max(t.first, paged::share_begin(total, c, parts));
                const long long hi = std::min(t.first + t.units, paged::share_begin(total, c + 1, parts));
                if (lo >= hi) ++empty;
                if (!places.insert(2LL * c + (lo == t.first)).second) ++shared;
            }
        }
        for (int c = 0; c < parts; ++c)
            if (paged::share_begin(total, c + 1, parts) - paged::share_begin(total, c, parts) < 1) ++thin;
        std::printf("%d %d %d %d %d\n", cut, most, shared, empty, thin);
    }
    return 0;
}
