// fa_tree.cuh — attention of drafted trees over a paged cache on the
// 5th-generation tensor cores (the formulas are fa_paged.cuh's; which of the new
// tokens' keys a row sees is a row of bits).
//
// A tree of n tokens is n x (query heads of a kv head) rows, a few dozen, over a
// long context: the cache's bytes bound it, and what a unit (128 rows x 128 keys)
// computes has to stay behind them.  fa_paged_tc.cuh's two row tiles of 128 that
// take turns leave one softmax warpgroup idle here and the other waiting for
// its products.  So the two warpgroups share one row tile and take its key
// tiles in turn, each with a running maximum, sum and accumulator of its own:
//
//   warps 0-3, 4-7  softmax of the even and the odd key tiles (thread = row =
//                   tensor-memory lane); warps without a row only keep step
//   warp 8          issues S_w = Q K^T and O_w += P_w V (w: the key tile's
//                   parity), the next scores of a warpgroup behind its product
//   warp 9          hands out the items and loads K and V by TMA in the order
//                   the products take them: K0 K1 V0 K2 V1 ...
//   warps 10, 11    load them instead, by gathered 16-byte copies, where a page is
//                   no multiple of 16 tokens
//
// At the end of an item the warpgroups exchange their statistics and each joins
// one half of the accumulators' columns.  Parts of a row tile cut by the shares
// are left in the workspace, and a second kernel joins them.
//
// The probabilities are rounded once to the cache's 16-bit type, as fa_paged_tc.cuh
// does and for its reason: a second part (what the rounding left) would be half as
// many products again, and both the products and the energy they take count here
// (48 trees of 8 over 8192 tokens, 64 / 8 heads: 143 to 150 us, 0.83 to 0.87 of measured bandwidth,
// at the 1000 W cap that streaming the cache alone comes near; two parts took a
// fifth more).  Calls of at most 16 rows a kv head carry them in two (TWO), as
// fa_paged.cuh does for as many rows: a short draft keeps the digits that its
// tokens have one by one (one sequence of 4096, 32 / 8 heads, 4 tokens: 17.7 us, with
// one part 16.4).  Both parts take the scores' place in tensor memory.
#pragma once
#include "fa_paged_tc.cuh"

namespace p100b {
namespace fatr {

using fatc::Cap;
using fatc::Job;
using fatc::kJobs;
using fatc::kSub;
using fatc::tile_bytes;
using fatc::warp_wait;
using paged::Desc;
using paged::Item;
using paged::Lengths;
using paged::add2;
using paged::fma2;
using paged::pair;
using paged::unpair;

constexpr int kRows = 128, kKeys = 128;
constexpr int kOver = 4;                  // what a row tile costs beyond its keys, in units (48 trees of 8: 145 us, with 2 152)
constexpr int kMinUnits = 2;              // of a share: a tile for each warpgroup
// Row tiles per CTA from which they are dealt out whole.  64 / 8 heads, trees of 8:
// 5.4 of up to 2048 tokens 106 us either way, of 512 55 (cut 66); 3.5 of 2048 82 (cut
// 72), of 512 38 (cut 43).
constexpr int kWholeFrom = 4;
constexpr int kThreads = fatc::kThreads;
constexpr int kMmaWarp = fatc::kMmaWarp, kLoadWarp = fatc::kLoadWarp, kGatherWarp = fatc::kGatherWarp;

template <int D>
__host__ __device__ constexpr int slots() { return D == 128 ? 5 : 8; }

// The row tile that a CTA begins and others end, as the joining kernel gets it.
struct Cut {
    int last;                    // CTA of the last part; the CTA itself: none
    int q0, row0, rows, head;    // the sequence's first token; first row, rows of the tile; kv head
    int pad[3];
};

struct Params {
    Desc d;
    const void* q;
    void* o;
    int o_f32;
    float* lse;
    float* ws_o;        // [CTAs][2][D / 4][128] float4
    float* ws_ml;       // [CTAs][2][128] float2
    Cut* cuts;          // [CTAs]
    float scale, softcap;
    int box;            // rows of a TMA box, 0: gathered rows
    const void *k, *v;
    const unsigned* mask;   // [n_tokens][words]
    int words;
};

struct Barriers {
    uint64_t full[8], empty[8], q_full, s_full[2], p_full[2][2], stats, o_free, job_full[kJobs], job_empty[kJobs], drain;
    uint32_t tmem;
    int abort;
    Job jobs[kJobs];
    float2 ml[2][kRows];   // the warpgroups' maxima and sums
};
using Units = paged::Share<kRows, kKeys, kOver>;

// Without the lengths.
template <int D>
constexpr size_t smem_bytes() {
    return 1024 + (1 + slots<D>()) * tile_bytes<D>() + sizeof(Barriers) + 64;
}

__host__ __device__ __forceinline__ int shares(long long total, int ctas) {
    const long long most = (total + kMinUnits - 1) / kMinUnits;
    return most < ctas ? int(most) : ctas;
}

// The place of an item's key tile t (of count) among its loads.
__device__ __forceinline__ unsigned k_at(int t) { return t == 0 ? 0 : 2 * t - 1; }
__device__ __forceinline__ unsigned v_at(int t, int count) { return t + 1 < count ? 2 * t + 2 : 2 * count - 1; }

// ------------------------------------------------------------ roles
template <int D>
__device__ __forceinline__ void load_role(const Params& p, const CUtensorMap* tmk, const CUtensorMap* tmv, const Lengths& len,
                                          Barriers& bars, uint8_t* ring, Units share) {
    constexpr int NS = slots<D>();
    const Desc& d = p.d;
    const int lane = threadIdx.x & 31;
    const int boxes = p.box ? kKeys / p.box : 1;     // of a tile, at most 8
    const int i = lane & (boxes - 1), half = lane / boxes;
    const bool mine = half < D / 64;
    const uint32_t at = uint32_t(half) * kSub + uint32_t(i) * p.box * 128;
    unsigned used = 0;                               // slots filled so far
    bool ok = true;
    struct Box {
        int page, off;   // off -1: nothing to read
    };
    for (unsigned j = 0; ok; ++j) {
        Item it;
        const bool more = share.next(d, len, it);
        if (j >= kJobs) ok = warp_wait(&bars.job_empty[j % kJobs], (j / kJobs - 1) & 1, &bars.abort);
        if (!ok) break;
        const int end = more ? it.kv : 0;
        if (lane == 0) {
            Job& job = bars.jobs[j % kJobs];
            job.count = more ? it.count : 0;
            if (more) {
                job.seq = it.seq;
                job.key_tile = it.key_tile;
                job.row0 = it.tile * kRows;
                job.q0 = len.q0[it.seq];
                job.n = it.n;
                job.kv = it.kv;
                job.end = end;
                job.head = it.head;
                job.whole = it.count == it.units;
                job.units = it.units;
                job.first = it.tile_first;
            }
            mbar_arrive(&bars.job_full[j % kJobs]);
        }
        if (!more) break;
        if (p.box == 0) continue;   // the gathering warps load
        const int* table = d.block_table + (long long)it.seq * d.max_pages;
        // Where a box lies; its table entry is looked at two tiles later, so that the loop does not wait for it.
        auto find = [&](int t) {
            Box b = {0, -1};
            if (!mine || t >= it.count) return b;
            const int key = (it.key_tile + t) * kKeys + i * p.box;
            if (key < end) {
                const int n = key / d.page_size;
                b.off = key - n * d.page_size;
                b.page = table[n];
            }
            return b;
        };
        auto load = [&](const CUtensorMap* map, const Box& b) {
            const int slot = used % NS;
            const bool known = b.page >= 0 && b.page < d.n_pages, there = b.off >= 0 && known;
            if (b.off >= 0 && !known) paged::flag_input();
            const uint32_t bytes = uint32_t(__popc(__ballot_sync(0xffffffffu, there))) * p.box * 128;
            if (used >= NS) ok = warp_wait(&bars.empty[slot], (used / NS - 1) & 1, &bars.abort);
            if (!ok) return;
            if (lane == 0) {
                if (bytes) mbar_arrive_expect_tx(&bars.full[slot], bytes);
                else mbar_arrive(&bars.full[slot]);
            }
            __syncwarp();
            if (there)
                asm volatile(
                    "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                    " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(ring) + uint32_t(slot) * tile_bytes<D>() + at),
                    "l"(map), "r"(half * 64), "r"(b.off), "r"(it.head), "r"(b.page), "r"(smem_addr(&bars.full[slot]))
                    : "memory");
            ++used;
        };
        Box now = find(0), next = find(1);
        load(tmk, now);
        for (int t = 0; ok && t < it.count; ++t) {
            const Box later = find(t + 2);
            if (t + 1 < it.count) load(tmk, next);
            if (ok) load(tmv, now);
            now = next;
            next = later;
        }
    }
    if (!ok)   // leave only when the copies in flight have landed
        for (unsigned u = used > NS ? used - NS : 0; u < used; ++u) mbar_wait(&bars.full[u % NS], (u / NS) & 1);
}

// The tiles of pages of any size: each of two warps gathers 64 keys' rows, in the
// order of load_role.  A slot's barrier takes the copies' own arrivals, and the
// issuing warp puts the fence between them and its products (a gathering warp's
// fence waits for the next slot's copies, too: 16 trees of 5 over 8192, pages of
// 24, 91 us, with it 94).  What bounds it are the copies of 16 bytes: boxes take 63.
// A third gathering warp, the one that hands out the items, made it 119.
template <typename T, int D>
__device__ __forceinline__ void gather_role(const Params& p, Barriers& bars, uint32_t ring) {
    constexpr int NS = slots<D>();
    constexpr int kChunks = D / 8, kStep = 32 / kChunks;   // 16-byte chunks of a row; rows of a copy of the warp
    const Desc& d = p.d;
    const int lane = threadIdx.x & 31, first = int((threadIdx.x >> 5) - kGatherWarp) * 64;
    const int chunk = lane % kChunks, sub = lane / kChunks;
    unsigned used = 0;
    bool ok = true;
    struct Rows {   // of keys `lane` and `lane + 32`
        int page[2], off[2];   // off -1: not read
    };
    for (unsigned j = 0;; ++j) {
        if (!warp_wait(&bars.job_full[j % kJobs], (j / kJobs) & 1, &bars.abort)) break;
        const Job& job = bars.jobs[j % kJobs];
        const int count = job.count, end = job.end, key0 = job.key_tile * kKeys + first + lane;
        if (count == 0) break;
        const int* table = d.block_table + (long long)job.seq * d.max_pages;
        const long long head = job.head * d.head_stride + chunk * 8;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.job_empty[j % kJobs]);
        // (the table entries are looked at two tiles later, as in load_role)
        auto find = [&](int t) {
            Rows r = {{0, 0}, {-1, -1}};
            if (t >= count) return r;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = key0 + t * kKeys + h * 32;
                if (key < end && key >= 0) {
                    const int n = key / d.page_size;
                    r.off[h] = key - n * d.page_size;
                    r.page[h] = table[n];
                }
            }
            return r;
        };
        auto load = [&](const void* pages, const Rows& r) {
            if (used >= NS && !warp_wait(&bars.empty[used % NS], (used / NS - 1) & 1, &bars.abort)) {
                ok = false;
                return;
            }
            long long at[2];   // where the rows begin, -1: not read
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool known = r.page[h] >= 0 && r.page[h] < d.n_pages;
                if (r.off[h] >= 0 && !known) paged::flag_input();
                at[h] = r.off[h] >= 0 && known ? r.page[h] * d.page_stride + r.off[h] * d.token_stride : -1;
            }
            const T* from = static_cast<const T*>(pages) + head;
            const uint32_t slot = ring + (used % NS) * tile_bytes<D>() + (chunk >> 3) * kSub;
            // eight rows' places first, then their copies
#pragma unroll 1
            for (int i = 0; i < 64; i += 8 * kStep) {
                long long o[8];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    o[u] = __shfl_sync(0xffffffffu, i + u * kStep < 32 ? at[0] : at[1], (i + u * kStep & 31) + sub);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int row = first + i + u * kStep + sub;
                    fap::cp_async16(slot + row * 128 + (((chunk & 7) ^ (row & 7)) << 4), from + (o[u] < 0 ? 0 : o[u]), o[u] >= 0);
                }
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_addr(&bars.full[used % NS])) : "memory");
            ++used;
        };
        Rows now = find(0), next = find(1);
        load(p.k, now);
        for (int t = 0; ok && t < count; ++t) {
            const Rows later = find(t + 2);
            if (t + 1 < count) load(p.k, next);
            if (ok) load(p.v, now);
            now = next;
            next = later;
        }
        if (!ok) break;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Issues the products; false when a wait was given up.
template <typename T, int D, bool TWO>
__device__ __forceinline__ bool mma_role(const Desc& d, float scale, bool gathered, Barriers& bars, uint32_t q_smem,
                                         uint32_t ring, uint32_t tmem) {
    constexpr int NS = slots<D>();
    // a negative scale turns the scores' sign here, so that the softmax has a positive one
    const uint32_t idesc_s = fatc::idesc_f16<T>(kKeys, false) | (scale < 0.f ? fatc::kNegateA : 0u);
    constexpr uint32_t kIdescO = fatc::idesc_f16<T>(D, true);
    const int lane = threadIdx.x & 31;
    unsigned used = 0, items = 0, tiles[2] = {0, 0};
    auto slot_of = [&](unsigned at) { return (used + at) % NS; };
    auto landed = [&](unsigned at) {
        const bool ok = warp_wait(&bars.full[slot_of(at)], ((used + at) / NS) & 1, &bars.abort);
        if (gathered) fatc::fence_async();
        return ok;
    };
    auto qk = [&](int w, unsigned slot) {   // S_w = Q K^T
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = uint32_t(k >> 2) * kSub + uint32_t(k & 3) * 32;
            fatc::mma_ss(tmem + w * 128, fatc::sw128_desc(q_smem + off, 16, 1024),
                         fatc::sw128_desc(ring + slot * tile_bytes<D>() + off, 16, 1024), idesc_s, k > 0);
        }
        fatc::mma_commit(&bars.s_full[w]);
        fatc::mma_commit(&bars.empty[slot]);
    };
    auto pv = [&](int w, int half, unsigned slot, bool add) {   // O_w += P_w V over half of the keys
#pragma unroll
        for (int part = 0; part < (TWO ? 2 : 1); ++part)
#pragma unroll
            for (int k = half * (kKeys / 32); k < (half + 1) * (kKeys / 32); ++k)
                fatc::mma_ts(tmem + 256 + w * D, tmem + w * 128 + part * 64 + k * 8,
                             fatc::sw128_desc(ring + slot * tile_bytes<D>() + uint32_t(k) * 2048, kSub, 1024), kIdescO,
                             add || part > 0 || k > 0);
    };
    for (unsigned j = 0;; ++j) {
        if (!warp_wait(&bars.job_full[j % kJobs], (j / kJobs) & 1, &bars.abort)) return false;
        const int count = int(fatc::uniform(bars.jobs[j % kJobs].count));
        if (count == 0) return true;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.job_empty[j % kJobs]);
        if (!warp_wait(&bars.q_full, items & 1, &bars.abort)) return false;
        for (int t = 0; t < 2 && t < count; ++t) {
            if (!landed(k_at(t))) return false;
            fatc::fence_after();
            qk(t, slot_of(k_at(t)));
        }
        for (int t = 0; t < count; ++t) {
            const int w = t & 1;
            const unsigned v = v_at(t, count);
            if (!landed(v)) return false;
            // the accumulators of the item before have been read
            if (t == 0 && items > 0 && !warp_wait(&bars.o_free, (items - 1) & 1, &bars.abort)) return false;
            if (!warp_wait(&bars.p_full[w][0], tiles[w] & 1, &bars.abort)) return false;
            fatc::fence_after();
            pv(w, 0, slot_of(v), t > 1);
            if (!warp_wait(&bars.p_full[w][1], tiles[w]++ & 1, &bars.abort)) return false;
            fatc::fence_after();
            pv(w, 1, slot_of(v), true);
            fatc::mma_commit(&bars.empty[slot_of(v)]);
            if (t + 2 < count) {
                if (!landed(k_at(t + 2))) return false;
                qk(w, slot_of(k_at(t + 2)));
            }
        }
        fatc::mma_commit(&bars.s_full[0]);
        fatc::mma_commit(&bars.s_full[1]);
        used += 2 * count;
        ++items;
    }
}

// The row of a thread in an item.
struct Row {
    int tok, g;   // token of the sequence, query head of the group
    bool live;
    __device__ __forceinline__ Row(const Desc& d, const Job& job, int row) {
        const int r = job.row0 + row;
        tok = r / d.group;
        g = r - tok * d.group;
        live = r < job.n * d.group;
    }
    __device__ __forceinline__ long long at(const Desc& d, const Job& job, long long stride, int D) const {
        return (long long)(job.q0 + tok) * stride + (long long)(job.head * d.group + g) * D;
    }
};

// The queries on their way into shared memory (zeros for rows that are none):
// each warpgroup brings half of the rows, two threads a row.
template <typename T, int D>
__device__ __forceinline__ void load_queries(const Params& p, const Job& job, uint32_t q_smem) {
    const int row = threadIdx.x >> 1, part = threadIdx.x & 1;
    const Row r(p.d, job, row);
    const T* src = static_cast<const T*>(p.q) + (r.live ? r.at(p.d, job, p.d.q_stride, D) : 0);
    const uint32_t dst = q_smem + row * 128;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        const int i = part * (D / 16) + c;
        fap::cp_async16(dst + (i >> 3) * kSub + (((i & 7) ^ (row & 7)) << 4), src + i * 8, r.live);
    }
}

// Which of 32 keys from `key` on a row sees, ctx keys before the tree's: bit i
// for key + i.  row: its words of the mask, nothing seen from `limit` on.
__device__ __forceinline__ uint32_t seen32(const unsigned* row, int words, int key, int ctx, int limit) {
    const int left = limit - key, node = key - ctx;   // the node of bit 0, negative in the context
    if (left <= 0) return 0u;
    uint32_t bits = 0xffffffffu;
    if (node > -32) {
        const int k = node >> 5;
        const uint32_t lo = k < 0 ? 0xffffffffu : k < words ? row[k] : 0u, hi = k + 1 < words ? row[k + 1] : 0u;
        bits = __funnelshift_r(lo, hi, node & 31);
    }
    return left < 32 ? bits & ((1u << left) - 1) : bits;
}

// Values of a row over their sum, to o.
template <typename T, int N>
__device__ __forceinline__ void write_row(const Params& p, const float (&o)[N], long long at, float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (p.o_f32) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.o) + at);
#pragma unroll
        for (int e = 0; e < N; e += 4) dst[e / 4] = make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
    } else if constexpr (N == 4) {
        *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + at) =
            make_uint2(paged::pack2<T>(o[0] * inv, o[1] * inv), paged::pack2<T>(o[2] * inv, o[3] * inv));
    } else {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + at);
#pragma unroll
        for (int e = 0; e < N; e += 8)
            dst[e / 8] = make_uint4(paged::pack2<T>(o[e] * inv, o[e + 1] * inv), paged::pack2<T>(o[e + 2] * inv, o[e + 3] * inv),
                                    paged::pack2<T>(o[e + 4] * inv, o[e + 5] * inv), paged::pack2<T>(o[e + 6] * inv, o[e + 7] * inv));
    }
}
__device__ __forceinline__ void write_lse(const Params& p, int token, int head, float top, float sum) {
    if (p.lse)
        p.lse[(long long)token * p.d.n_head_q + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) / 1.4426950408889634f;
}

template <typename T, int D, bool CAP, bool TWO>
__device__ __forceinline__ void softmax_role(const Params& p, Barriers& bars, uint32_t q_smem, uint8_t* ring, uint32_t tmem,
                                             long long total_units, int parts) {
    constexpr int NS = slots<D>();
    constexpr float kLog2e = 1.4426950408889634f;
    const Desc& d = p.d;
    const int w = threadIdx.x >> 7, row = threadIdx.x & 127;
    const uint32_t lanes = uint32_t(row & ~31) << 16;
    const uint32_t t_s = tmem + w * 128 + lanes, t_o = tmem + 256 + lanes;
    const float c = fabsf(p.scale) * kLog2e;   // of the scores to units of log2
    const Cap cap(fabsf(p.scale), CAP ? p.softcap : 1.f);
    unsigned done = 0, used = 0;   // phases of s_full passed; loads of the CTA before this item
    bool loaded = false;           // the item's queries are on their way
    for (unsigned j = 0;; ++j) {
        if (!warp_wait(&bars.job_full[j % kJobs], (j / kJobs) & 1, &bars.abort)) return;
        const Job& job = bars.jobs[j % kJobs];
        const int count = job.count;
        if (count == 0) return;
        auto queries_ready = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            fatc::fence_async();
            fatc::fence_before();
            mbar_arrive(&bars.q_full);
        };
        if (!loaded) {
            load_queries<T, D>(p, job, q_smem);
            queries_ready();
        }
        const Row r(d, job, row);
        // (a row that is none takes the first one's mask: its results go nowhere)
        const int ctx = job.kv - job.n, limit = job.kv;
        const unsigned* bits = p.mask + (long long)(job.q0 + (r.live ? r.tok : 0)) * p.words;
        const bool any_row = (row & ~31) < job.n * d.group - job.row0;   // of the warp
        float m = -INFINITY, l = 0.f;
        // Zeroes the rows of V behind the last key, before the products of tile t.
        auto clear_v = [&](int t, int key0) {
            if (job.end - key0 >= kKeys) return true;
            const unsigned u = used + v_at(t, count);
            if (!warp_wait(&bars.full[u % NS], (u / NS) & 1, &bars.abort)) return false;
            if (row >= job.end - key0) {
                uint8_t* v = ring + (u % NS) * tile_bytes<D>() + row * 128;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    *reinterpret_cast<uint4*>(v + (i >> 3) * kSub + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fatc::fence_async();
            return true;
        };
        for (int t = w; t < count; t += 2) {
            const int key0 = (job.key_tile + t) * kKeys;   // key0 + kKeys may pass 2^31
            if (!warp_wait(&bars.s_full[w], done++ & 1, &bars.abort)) return;
            fatc::fence_after();
            if (!any_row) {   // the products of these rows go nowhere
                if (!clear_v(t, key0)) return;
                mbar_arrive(&bars.p_full[w][0]);
                mbar_arrive(&bars.p_full[w][1]);
                continue;
            }
            float s[128];
#pragma unroll
            for (int i = 0; i < 4; ++i) fatc::ld32(t_s + i * 32, s + i * 32);
            fatc::wait_ld();
            const bool masked = __any_sync(0xffffffffu, limit - key0 < kKeys || ctx - key0 < kKeys);
            float hidden = -INFINITY, k[5];
            uint32_t seen[4];
            if (masked) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    seen[i] = limit - key0 > 32 * i ? seen32(bits, p.words, key0 + 32 * i, ctx, limit) : 0u;
            }
            if (CAP) {
                if (masked) {   // whatever stands there must not look large
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = seen[i >> 5] >> (i & 31) & 1u ? s[i] : 0.f;
                }
                float far4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 128; i += 8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) far4[e] = fmaxf(fmaxf(far4[e], fabsf(s[i + e])), fabsf(s[i + 4 + e]));
                }
                const float largest = fmaxf(fmaxf(far4[0], far4[1]), fmaxf(far4[2], far4[3]));
                const bool far = !__all_sync(0xffffffffu, largest <= cap.most);
                if (far) {
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = fap::cap_score(s[i], cap.near, cap.out);
                }
#pragma unroll
                for (int i = 0; i < 5; ++i) k[i] = far ? float(i == 0) : cap.k[i];
                hidden = cap.hidden(far);
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 128; ++i) s[i] = seen[i >> 5] >> (i & 31) & 1u ? s[i] : hidden;
            }
            float mx4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < 128; i += 8) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mx4[e] = i + 4 + e < 128 ? fmaxf(fmaxf(mx4[e], s[i + e]), s[i + 4 + e]) : fmaxf(mx4[e], s[i + e]);
            }
            float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));   // then in units of log2
            if (CAP) {
                const float z = mx * mx;
                mx = mx == hidden ? -INFINITY : mx * fmaf(z, fmaf(z, fmaf(z, fmaf(z, k[4], k[3]), k[2]), k[1]), k[0]);
            } else {
                mx *= c;
            }
            mx -= fatc::kLift<T>;
            if (t < 2) {
                m = mx;
            } else {
                const bool rise = mx - m > fatc::kRise;
                if (__any_sync(0xffffffffu, rise)) {
                    const float a = rise ? paged::exp2_approx(m - mx) : 1.f;
                    if (rise) m = mx;
                    l *= a;
#pragma unroll 1
                    for (int i = 0; i < D / 16; ++i) {   // few registers: the scores stay in theirs
                        float o[16];
                        fatc::ld16(t_o + w * D + i * 16, o);
                        fatc::wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] *= a;
                        fatc::st16(t_o + w * D + i * 16, reinterpret_cast<const uint32_t*>(o));
                    }
                }
            }
            const float base = m == -INFINITY ? 0.f : m;
            const uint64_t c2 = pair(c, c), b2 = pair(-base, -base);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int half = 0; half < 2; ++half) {   // the products with the first half start while the second is computed
#pragma unroll
                for (int i = 4 * half; i < 4 * half + 4; ++i) {
                    uint32_t pk[8], rest[8];
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const uint64_t x = pair(s[i * 16 + e], s[i * 16 + e + 1]);
                        uint64_t f = c2;
                        if (CAP) {
                            const uint64_t z = paged::mul2(x, x);
                            f = pair(k[4], k[4]);
#pragma unroll
                            for (int n = 3; n >= 0; --n) f = fma2(z, f, pair(k[n], k[n]));
                        }
                        float a, b;
                        unpair(fma2(x, f, b2), a, b);
                        a = paged::exp2_approx(a);
                        b = paged::exp2_approx(b);
                        sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pair(a, b));
                        pk[e >> 1] = paged::pack2<T>(a, b);
                        if (TWO) {
                            float high_a, high_b;
                            paged::unpack2<T>(pk[e >> 1], high_a, high_b);
                            rest[e >> 1] = paged::pack2<T>(a - high_a, b - high_b);
                        }
                    }
                    fatc::st8(t_s + i * 8, pk);
                    if (TWO) fatc::st8(t_s + 64 + i * 8, rest);
                }
                fatc::wait_st();
                if (half == 0 && !clear_v(t, key0)) return;
                fatc::fence_before();
                mbar_arrive(&bars.p_full[w][half]);
            }
            {
                float a, b;
                unpair(add2(sum[0], sum[1]), a, b);
                l += a + b;
            }
        }
        used += 2 * count;
        if (!warp_wait(&bars.s_full[w], done++ & 1, &bars.abort)) return;   // every product of the item is complete
        fatc::fence_after();
        // the queries' place is free for the next item's
        if (!warp_wait(&bars.job_full[(j + 1) % kJobs], ((j + 1) / kJobs) & 1, &bars.abort)) return;
        loaded = bars.jobs[(j + 1) % kJobs].count != 0;
        if (loaded) load_queries<T, D>(p, bars.jobs[(j + 1) % kJobs], q_smem);
        bars.ml[w][row] = make_float2(m, l);
        mbar_arrive(&bars.stats);
        if (!warp_wait(&bars.stats, j & 1, &bars.abort)) return;
        const float2 st0 = bars.ml[0][row], st1 = bars.ml[1][row];
        const float top = fmaxf(st0.x, st1.x), safe = top == -INFINITY ? 0.f : top;
        const float f0 = paged::exp2_approx(st0.x - safe), f1 = paged::exp2_approx(st1.x - safe);
        const float total = fmaf(f0, st0.y, f1 * st1.y);
        constexpr int kCols = D / 2;   // of this warpgroup's half
        float o[kCols];
#pragma unroll
        for (int i = 0; i < kCols / 32; ++i) fatc::ld32(t_o + w * kCols + i * 32, o + i * 32);
        fatc::wait_ld();
#pragma unroll
        for (int e = 0; e < kCols; ++e) o[e] *= f0;
        if (count > 1) {
#pragma unroll
            for (int i = 0; i < kCols / 32; ++i) {
                float x[32];
                fatc::ld32(t_o + D + w * kCols + i * 32, x);
                fatc::wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[i * 32 + e] = fmaf(f1, x[e], o[i * 32 + e]);
            }
        }
        fatc::fence_before();
        mbar_arrive(&bars.o_free);
        if (loaded) queries_ready();   // the next item's scores are computed while this one's results are written
        const long long o_at = r.at(d, job, d.o_stride, D) + w * kCols;
        if (job.whole) {
            if (r.live) {
                write_row<T>(p, o, o_at, total);
                if (w == 0) write_lse(p, job.q0 + r.tok, job.head * d.group + r.g, top, total);
            }
        } else if (r.live) {   // a part for fa_tree_join_kernel
            const long long slot = blockIdx.x * 2 + (job.key_tile == 0);
            float4* dst = reinterpret_cast<float4*>(p.ws_o) + (slot * (D / 4) + w * (kCols / 4)) * kRows + row;
#pragma unroll
            for (int e = 0; e < kCols / 4; ++e)
                __stcg(dst + e * kRows, make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]));
            if (w == 0) __stcg(reinterpret_cast<float2*>(p.ws_ml) + slot * kRows + row, make_float2(top, total));
        }
        if (threadIdx.x == 0 && !job.whole && job.key_tile == 0)
            p.cuts[blockIdx.x] = {paged::share_of(job.first + job.units - 1, total_units, parts), job.q0, job.row0,
                                  min(kRows, job.n * d.group - job.row0), job.head, {}};
        __syncwarp();
        if ((row & 31) == 0) mbar_arrive(&bars.job_empty[j % kJobs]);
    }
}

template <typename T, int D, bool CAP, bool TWO>
__global__ void __launch_bounds__(kThreads, 1)
    fa_tree_kernel(const Params p, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_smem = smem;
    uint8_t* ring = q_smem + tile_bytes<D>();
    Barriers& bars = *reinterpret_cast<Barriers*>(ring + slots<D>() * tile_bytes<D>());
    const Lengths len(reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(&bars + 1) + 15) & ~uintptr_t(15)), p.d.n_seq);
    const int warp = threadIdx.x >> 5;

    pdl_allow_dependents();   // the joining kernel, which waits for this one's end
    if (threadIdx.x == 0) p.cuts[blockIdx.x].last = blockIdx.x;
    if (threadIdx.x == kLoadWarp * 32 && p.box) {
        prefetch_tensormap(&tmk);
        prefetch_tensormap(&tmv);
    }
    paged::read_lengths<kRows, kKeys, kOver, kThreads, true>(p.d, len, (long long)kWholeFrom * gridDim.x);
    // whole row tiles are dealt out over all CTAs, cut ones in shares of some units
    const int parts = !len.head->ok ? 0 : len.head->whole ? int(gridDim.x) : shares(len.head->total, int(gridDim.x));
    if (int(blockIdx.x) >= parts) return;
    // what the first copies wait for, side by side: the barriers, tensor memory
    // and the load warp's place in the work
    if (threadIdx.x < 8) {
        mbar_init(&bars.full[threadIdx.x], p.box ? 1 : 64);
        mbar_init(&bars.empty[threadIdx.x], 1);
    } else if (threadIdx.x < 10) {
        const int w = threadIdx.x - 8;
        mbar_init(&bars.s_full[w], 1);
        mbar_init(&bars.p_full[w][0], 128);
        mbar_init(&bars.p_full[w][1], 128);
    } else if (threadIdx.x < 10 + kJobs) {
        mbar_init(&bars.job_full[threadIdx.x - 10], 1);
        mbar_init(&bars.job_empty[threadIdx.x - 10], p.box ? 9 : 11);   // the softmax warps, the issuing one, the gathering ones
    } else if (threadIdx.x == 30) {
        mbar_init(&bars.q_full, 256);
        mbar_init(&bars.stats, 256);
        mbar_init(&bars.o_free, 256);
    } else if (threadIdx.x == 31) {
        mbar_init(&bars.drain, 1);
        bars.abort = 0;
    }
    if (warp == 0) fence_barrier_init();
    Units share;
    if (warp == kLoadWarp) share.begin(p.d, len, blockIdx.x, parts);
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&bars.tmem)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fatc::fence_before();
    __syncthreads();
    fatc::fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem);
    if (warp < kMmaWarp) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(fatc::kSoftmaxRegs));
        softmax_role<T, D, CAP, TWO>(p, bars, smem_addr(q_smem), ring, tmem, len.head->total, parts);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(fatc::kIssueRegs));
        if (warp == kLoadWarp) {
            load_role<D>(p, &tmk, &tmv, len, bars, ring, share);
        } else if (warp == kMmaWarp) {
            if (!mma_role<T, D, TWO>(p.d, p.scale, p.box == 0, bars, fatc::uniform(smem_addr(q_smem)),
                                     fatc::uniform(smem_addr(ring)), fatc::uniform(tmem))) {
                // leave only when the products in flight are done
                fatc::mma_commit(&bars.drain);
                __syncwarp();
                mbar_wait(&bars.drain, 0);
            }
        } else if (p.box == 0) {
            gather_role<T, D>(p, bars, smem_addr(ring));
        }
    }

    fatc::fence_before();
    __syncthreads();
    fatc::fence_after();
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ------------------------------------------------------------ join
// Row tiles cut by the shares: 32 rows x 4 COLS columns of the parts are a warp's
// item, joined in share order, and the items of all cuts are dealt out over the
// warps of all CTAs.  (The last CTA of a row tile to finish would read its parts
// at one SM's rate: those of one tree over 4096 keys, 19 of 32 KB, in 10 us.)
// What it costs is a few round trips to the L2: the cuts, then PARTS parts in
// each; a cut of few parts has wider items instead.
constexpr int kJoinThreads = 512, kFewParts = 3;
template <typename T, int D, int COLS, int PARTS>
__device__ __forceinline__ void join_item(const Params& p, const Cut& cut, int c0, int row, int col) {
    const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + row;
    const float4* po = reinterpret_cast<const float4*>(p.ws_o) + col * kRows + row;
    const bool live = row < cut.rows;
    float top = -INFINITY, sum = 0.f, o[COLS][4] = {};
    for (int q0 = c0; q0 <= cut.last; q0 += PARTS) {
        float2 st[PARTS];
        float4 x[PARTS][COLS];
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
            const long long part = (long long)(q0 + k) * 2 + (q0 + k == c0);
            const bool in = live && q0 + k <= cut.last;
            st[k] = in ? __ldcg(ml + part * kRows) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < COLS; ++i)
                x[k][i] = in ? __ldcg(po + (part * (D / 4) + i) * kRows) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const float before = top;
#pragma unroll
        for (int k = 0; k < PARTS; ++k) top = fmaxf(top, st[k].x);
        const float safe = top == -INFINITY ? 0.f : top, a = paged::exp2_approx(before - safe);
        sum *= a;
#pragma unroll
        for (int i = 0; i < COLS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] *= a;
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
            const float f = paged::exp2_approx(st[k].x - safe);
            sum = fmaf(f, st[k].y, sum);
#pragma unroll
            for (int i = 0; i < COLS; ++i) {
                o[i][0] = fmaf(f, x[k][i].x, o[i][0]);
                o[i][1] = fmaf(f, x[k][i].y, o[i][1]);
                o[i][2] = fmaf(f, x[k][i].z, o[i][2]);
                o[i][3] = fmaf(f, x[k][i].w, o[i][3]);
            }
        }
    }
    if (!live) return;
    const Desc& d = p.d;
    const int r = cut.row0 + row, tok = r / d.group, head = cut.head * d.group + (r - tok * d.group), token = cut.q0 + tok;
#pragma unroll
    for (int i = 0; i < COLS; ++i)
        write_row<T>(p, o[i], (long long)token * d.o_stride + (long long)head * D + (col + i) * 4, sum);
    if (col == 0) write_lse(p, token, head, top, sum);
}

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) fa_tree_join_kernel(const Params p, int ctas) {
    __shared__ int s_first[kJoinThreads];   // items before a CTA's cut
    __shared__ int s_warp[kJoinThreads / 32];
    constexpr int kWide = 4;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait_prior_grid();
    int own = 0;
    if (tid < ctas && p.cuts[tid].last != tid)
        own = (p.cuts[tid].rows + 31) / 32 * (D / 4) / (p.cuts[tid].last - tid < kFewParts ? kWide : 1);
    int v = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += u;
    }
    if (lane == 31) s_warp[warp] = v;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) {
        if (i < warp) v += s_warp[i];
        total += s_warp[i];
    }
    s_first[tid] = v - own;
    __syncthreads();
    for (int item = warp * gridDim.x + blockIdx.x; item < total; item += gridDim.x * (kJoinThreads / 32)) {
        int c0 = 0, hi = ctas - 1;   // the last CTA whose first item is at or before this one
        while (c0 < hi) {
            const int mid = (c0 + hi + 1) >> 1;
            if (s_first[mid] <= item) c0 = mid; else hi = mid - 1;
        }
        const Cut cut = p.cuts[c0];
        const int at = item - s_first[c0];
        if (cut.last - c0 < kFewParts)
            join_item<T, D, kWide, kFewParts>(p, cut, c0, at / (D / 4 / kWide) * 32 + lane, at % (D / 4 / kWide) * kWide);
        else
            join_item<T, D, 1, 10>(p, cut, c0, at / (D / 4) * 32 + lane, at % (D / 4));
    }
}

}  // namespace fatr
}  // namespace p100b
