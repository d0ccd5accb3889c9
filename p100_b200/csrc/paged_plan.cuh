// paged_plan.cuh — the small kernels around a step over a paged cache: the plan
// (pages taken and given back, starts, slots and positions of the new tokens
// from the requests' lengths), the masks and positions of drafted trees, and
// the move of the accepted tokens' rows.  Each is a few KB of work: what bounds
// them is the launch and a chain of dependent loads, which the kernels keep
// short.
#pragma once
#include "paged.cuh"

namespace p100b {
namespace paged {

// ------------------------------------------------------------ plan
// kv = length + new, need = ceil(kv / page); a request holds its first `held`
// table entries.  Entries [need, held) go back to the pool, [held, need) are
// filled from it.  With R entries given back, in order of the requests and of
// their entries, and `count` free pages on the stack, the r-th lies at stack
// place count + R - 1 - r, and the k-th entry taken gets place count + R - 1 - k:
// what a call gives back, the same call reversed takes again.
//
// The whole is exclusive sums over at most 1024 requests, one a thread, which
// every CTA of the (one) cluster does for itself, and then loops over the
// entries and tokens, found again by bisection of the sums.  All stack places
// are written before any is read: one meeting of the cluster in between.
struct PlanParams {
    int n_seq, n_tokens, page_size, n_pages, max_pages;
    const int *length, *n_new;   // [n_seq]
    int* pool;                   // [2 + n_pages]: free pages, missing ones, the stack
    int* held;                   // [n_seq]
    int* block_table;            // [n_seq][max_pages]
    int* q_start;                // [n_seq + 1]
    int* kv_len;                 // [n_seq]
    long long* slot;             // [n_tokens] or null
    int* position;               // [n_tokens] or null
};
constexpr int kPlanSmall = 256, kPlanThreads = 1024;

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_size() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// A meeting of the cluster's threads: what one wrote before it, global memory
// too, the others see behind it.
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// The last i < n with first[i] <= x, first ascending from 0.
__device__ __forceinline__ int last_at(const int* first, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanParams p) {
    __shared__ int s_q0[kMaxSeq + 1], s_len[kMaxSeq], s_held[kMaxSeq], s_need[kMaxSeq], s_give[kMaxSeq], s_take[kMaxSeq];
    __shared__ long long s_part[3][32];
    __shared__ int s_count;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
    const int rank = int(cluster_rank()), all = int(cluster_size() * blockDim.x), me = rank * int(blockDim.x) + tid;

    int len = 0, fresh = 0, held = 0, need = 0;
    bool good = true;
    if (tid == 0) s_count = p.pool[0];
    if (tid < p.n_seq) {   // the host gives every request a thread
        len = p.length[tid];
        fresh = p.n_new[tid];
        held = p.held[tid];
        const long long kv = (long long)len + fresh;
        good = len >= 0 && fresh >= 0 && held >= 0 && held <= p.max_pages && kv <= (long long)p.max_pages * p.page_size;
        need = good ? int((kv + p.page_size - 1) / p.page_size) : held;
    }
    // exclusive sums of the new tokens, the entries given back and those taken
    long long v[3] = {fresh, max(held - need, 0), max(need - held, 0)};
    const long long own[3] = {v[0], v[1], v[2]};
#pragma unroll
    for (int off = 1; off < 32; off <<= 1)
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const long long u = __shfl_up_sync(0xffffffffu, v[k], off);
            if (lane >= off) v[k] += u;
        }
    if (lane == 31)
        for (int k = 0; k < 3; ++k) s_part[k][warp] = v[k];
    good = __syncthreads_and(good);
    long long total[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        long long part = lane < warps ? s_part[k][lane] : 0, before = lane < warp ? part : 0;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            part += __shfl_xor_sync(0xffffffffu, part, off);
            before += __shfl_xor_sync(0xffffffffu, before, off);
        }
        total[k] = part;
        v[k] += before - own[k];
    }
    const int count = s_count;
    good = good && total[0] <= p.n_tokens && count >= 0 && total[1] <= (long long)p.n_pages - count;
    const long long missing = good ? max(total[2] - total[1] - count, 0LL) : -1;
    if (tid < p.n_seq) {   // the sums fit where the call is not refused
        s_q0[tid] = int(v[0]);
        s_len[tid] = len;
        s_held[tid] = held;
        s_need[tid] = need;
        s_give[tid] = int(v[1]);
        s_take[tid] = int(v[2]);
    }
    cluster_meet();   // every CTA has read the pool's count, the lengths (kv_len may be their place) and `held`
    if (missing != 0) {   // refused: no pages move and no request has new tokens
        if (rank == 0) {
            if (tid < p.n_seq) p.kv_len[tid] = len;
            if (tid < p.n_seq) p.q_start[tid] = 0;
            if (tid == 0) {
                p.q_start[p.n_seq] = 0;
                p.pool[1] = int(min(missing, 0x7fffffffLL));
                if (missing < 0) flag_input();
            }
        }
        for (unsigned t = me; t < unsigned(p.n_tokens); t += all) {
            if (p.slot) p.slot[t] = -1;
            if (p.position) p.position[t] = -1;
        }
        return;
    }
    const int tokens = int(total[0]), give = int(total[1]), take = int(total[2]), top = count + give - 1;
    int* stack = p.pool + 2;
    // (the counters pass 2^31 - 1 behind the last of as many rows or pages)
    for (unsigned i = me; i < unsigned(give); i += all) {
        const int r = int(i);
        const int s = last_at(s_give, p.n_seq, r);
        int* entry = p.block_table + (long long)s * p.max_pages + s_need[s] + (r - s_give[s]);
        stack[top - r] = *entry;
        *entry = -1;
    }
    cluster_meet();
    for (unsigned i = me; i < unsigned(take); i += all) {
        const int k = int(i);
        const int s = last_at(s_take, p.n_seq, k);
        p.block_table[(long long)s * p.max_pages + s_held[s] + (k - s_take[s])] = stack[top - k];
    }
    for (unsigned i = me; i < unsigned(p.n_tokens); i += all) {
        const int t = int(i);
        int pos = -1;
        long long slot = -1;
        if (t < tokens) {
            const int s = last_at(s_q0, p.n_seq, t);
            pos = s_len[s] + (t - s_q0[s]);
            if (p.slot) {
                const int e = pos / p.page_size;
                const int page = e < s_held[s] ? p.block_table[(long long)s * p.max_pages + e]
                                               : stack[top - (s_take[s] + e - s_held[s])];
                slot = (long long)page * p.page_size + (pos - e * p.page_size);
            }
        }
        if (p.slot) p.slot[t] = slot;
        if (p.position) p.position[t] = pos;
    }
    if (rank == 0) {
        if (tid < p.n_seq) {
            p.q_start[tid] = int(v[0]);
            p.kv_len[tid] = len + fresh;
            p.held[tid] = need;
        }
        if (tid == 0) {
            p.q_start[p.n_seq] = tokens;
            p.pool[0] = top + 1 - take;
            p.pool[1] = 0;
        }
    }
}

// An empty pool of all pages, the first on top, and requests that hold none.
__global__ void paged_pool_kernel(int n_seq, int n_pages, int max_pages, int* pool, int* held, int* block_table) {
    const long long all = (long long)gridDim.x * blockDim.x, me = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    for (long long i = me; i < n_pages; i += all) pool[2 + i] = int(n_pages - 1 - i);
    for (long long i = me; i < (long long)n_seq * max_pages; i += all) block_table[i] = -1;
    for (long long i = me; i < n_seq; i += all) held[i] = 0;
    if (me == 0) pool[0] = n_pages, pool[1] = 0;
}

// ------------------------------------------------------------ trees
// M_i = {i} and M_parent(i), depth |M_i| - 1.  A CTA per sequence, a thread per
// token: it walks to the root through parents in shared memory.  A parent comes
// before its child, so the bits fall from the highest word to the lowest and
// each word is written once, without a read.  The longest walk bounds it: 64 trees
// of 250 of depth 60 5.5 us, chains of 250 38 us and of 1024 433.
struct TreeParams {
    int n_seq, n_tokens, words;
    const int *parent, *q_start, *kv_len;
    unsigned* mask;     // [n_tokens][words]
    int* position;      // [n_tokens] or null
};
constexpr int kTreeThreads = 256, kTreeNodes = 32 * P100_TREE_MAX_WORDS;

__global__ void __launch_bounds__(kTreeThreads) tree_mask_kernel(const TreeParams p) {
    __shared__ short s_parent[kTreeNodes];
    const int tid = threadIdx.x;
    const int q0 = p.q_start[blockIdx.x], n = p.q_start[blockIdx.x + 1] - q0, kv = p.kv_len[blockIdx.x];
    if (q0 < 0 || n < 0 || n > 32 * p.words || q0 > p.n_tokens - n || kv < n) {
        if (tid == 0) flag_input();
        return;
    }
    for (int i = tid; i < n; i += kTreeThreads) {
        int up = p.parent[q0 + i];
        if (up < -1 || up >= i) {
            flag_input();
            up = -1;
        }
        s_parent[i] = short(up);
    }
    __syncthreads();
    for (int i = tid; i < n; i += kTreeThreads) {
        unsigned* row = p.mask + (long long)(q0 + i) * p.words;
        int word = p.words - 1, depth = 0;
        for (; word > i >> 5; --word) row[word] = 0;
        unsigned bits = 1u << (i & 31);
        for (int up = s_parent[i]; up >= 0; up = s_parent[up]) {
            ++depth;
            for (; word > up >> 5; --word, bits = 0) row[word] = bits;
            bits |= 1u << (up & 31);
        }
        for (; word >= 0; --word, bits = 0) row[word] = bits;
        if (p.position) p.position[q0 + i] = kv - n + depth;
    }
}

// ------------------------------------------------------------ keep
// Row ctx + keep[i] to row ctx + i for i < keep_len, in the pages' place: a
// thread owns 16 bytes of a row (of K or V, one head) and takes the kept rows in
// their order, kKeepRows loads ahead of as many stores.  keep rises, so keep[i]
// >= i and no row is read after it was written.  The lanes look up the pages of
// 32 rows at a time for each other.
struct KeepParams {
    Desc d;
    uint4 *k, *v;
    const int *keep, *keep_len;
    int* length;            // [n_seq] or null
};
constexpr int kKeepThreads = 128, kKeepRows = 8;

__global__ void __launch_bounds__(kKeepThreads) paged_keep_kernel(const KeepParams p, int chunks) {
    const Desc& d = p.d;
    const int s = blockIdx.y, lane = threadIdx.x & 31;
    const int q0 = d.q_start[s], n = d.q_start[s + 1] - q0, kv = d.kv_len[s], asked = p.keep_len[s];
    const bool usable = q0 >= 0 && n >= 0 && q0 <= d.n_tokens - n && kv >= n && kv <= (long long)d.max_pages * d.page_size;
    const bool counted = asked >= 0 && asked <= n;
    const int kept = usable && counted ? asked : 0;
    // every sequence gets a length that the next plan can take; one without new
    // tokens (a step that lacked pages has none) keeps its own, whatever was asked
    if (p.length && blockIdx.x == 0 && threadIdx.x == 0) p.length[s] = usable ? kv - n + kept : kv;
    if (threadIdx.x == 0 && (!usable || (!counted && n > 0))) flag_input();
    const int column = blockIdx.x * kKeepThreads + threadIdx.x, per = d.n_head_kv * chunks;
    const bool mine = column < 2 * per;
    const int c = column % per;
    uint4* base = (column < per ? p.k : p.v) + (c / chunks) * (d.head_stride / 8) + c % chunks;
    const int* table = d.block_table + (long long)s * d.max_pages;
    for (unsigned at0 = 0; at0 < unsigned(kept); at0 += 32) {   // (at0 may pass 2^31 - 1)
        const int i0 = int(at0);
        long long from = -1, to = -1;   // of row i0 + lane, in 16 bytes; -1: stays
        if (i0 + lane < kept) {
            const int j = p.keep[q0 + i0 + lane], before = i0 + lane ? p.keep[q0 + i0 + lane - 1] : -1;
            const bool rising = j > before && j >= i0 + lane && j < n;
            if (rising && j != i0 + lane) {
                const int a = kv - n + j, b = kv - n + i0 + lane;
                const int pa = table[a / d.page_size], pb = table[b / d.page_size];
                if (pa >= 0 && pa < d.n_pages && pb >= 0 && pb < d.n_pages) {
                    from = (pa * d.page_stride + a % d.page_size * d.token_stride) / 8;
                    to = (pb * d.page_stride + b % d.page_size * d.token_stride) / 8;
                } else {
                    flag_input();
                }
            }
            if (!rising) flag_input();
        }
        const int rows = min(32, kept - i0);
        for (int i = 0; i < rows; i += kKeepRows) {
            uint4 x[kKeepRows];
#pragma unroll
            for (int u = 0; u < kKeepRows; ++u) {
                const long long at = __shfl_sync(0xffffffffu, from, i + u);
                if (mine && at >= 0) x[u] = base[at];
            }
#pragma unroll
            for (int u = 0; u < kKeepRows; ++u) {
                const long long at = __shfl_sync(0xffffffffu, to, i + u);
                if (mine && at >= 0) base[at] = x[u];
            }
        }
    }
}

}  // namespace paged
}  // namespace p100b
