// paged_append.cuh — a chunk of new tokens into a paged cache: the norms of
// the query and key heads, their rotation and the write to the pages in one
// pass over the fused q|k|v rows.
//
// Per head x of a token at position p: x' = x w / sqrt(mean(x^2) + eps) (with
// norm weights), then for each pair (a, b): (a cos - b sin, a sin + b cos)
// with the table's angle of p; pairs are adjacent values, or value i with
// value i + D/2.  All in FP32; the one rounding is the store to 16 bits.
//
// Bytes bound it: every value is read once and written once.  A lane takes the
// E consecutive values of one 16-byte load (pairs of adjacent values stay in
// the lane, the halves' partner sits D / 2E lanes away), a warp 32 E / D heads
// of one kind in a step, a few steps together with the next ones on their way.  The token's sequence, page and angles are looked up once a warp; how
// many warps share a token follows from the number of tokens, so a single
// token's heads are spread over SMs and a prompt's lookups are not repeated.
// Measured: 8192 tokens of 64 / 8 heads of 128 from fp32 97 us, 0.80 of measured
// bandwidth; 2,900 tokens of 32 / 8 heads from bf16 with norms 22.5 us.
#pragma once
#include "paged.cuh"

namespace p100b {
namespace paged {

constexpr int kAppendThreads = 256;
// Warps of an SM, at least, before a token's heads share a warp (2,900 tokens of
// 24 steps: 22.5 us with 16 or 32, 23.1 with 64, 26.6 with 128, 36.9 with 256),
// and steps of a warp at most (8,192 tokens of 80 steps: 96 us in two warps,
// 103 in one or four).
constexpr int kAppendWarps = 32;
constexpr int kAppendMost = 40;
template <typename S>
__host__ __device__ constexpr int append_values() { return 16 / int(sizeof(S)); }   // of a lane in a step
template <typename S>
__host__ __device__ constexpr int append_steps() { return sizeof(S) == 4 ? 4 : 2; }   // of a warp at a time

struct AppendParams {
    Desc d;
    const void* qkv;
    long long qkv_stride;
    const float* q_norm;    // [D] or null
    const float* k_norm;
    float eps;
    const float2* rope;     // [max_pos][D/2] or null
    int max_pos, half;
    int warps;              // that share a token
    void *q, *k, *v;
};

// E values rounded to 16 bits.
template <typename T, int E>
__device__ __forceinline__ void store_values(T* p, const float (&x)[E]) {
    if constexpr (E == 4)
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    else
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

// The steps of a token: its q heads, then k, then v, `at_once` of a kind in each.
struct Steps {
    int q, kv;   // of the q heads, of the k (or v) heads
    __host__ __device__ Steps(int n_head_q, int n_head_kv, int at_once) {
        q = (n_head_q + at_once - 1) / at_once;
        kv = (n_head_kv + at_once - 1) / at_once;
    }
    __host__ __device__ int all() const { return q + 2 * kv; }
};

// The sequence of token t, or -1: the last s with q_start[s] <= t, found 32
// candidates at a time, if t also lies before q_start[s + 1]; q0, q1 its first
// token and the one behind its last, kv its length.
__device__ __forceinline__ int find_seq(const Desc& d, int t, int& q0, int& q1, int& kv) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = d.n_seq;   // the answer lies in [lo, lo + len)
    while (len > 32) {
        const int step = (len + 31) / 32;
        const bool at = lane * step < len && d.q_start[lo + lane * step] <= t;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, at) | 1u);
        lo += k * step;
        len = min(step, len - k * step);
    }
    const int i = lo + min(lane, len - 1);
    const int a = d.q_start[i], b = d.q_start[i + 1], c = d.kv_len[i];
    const int k = 31 - __clz(__ballot_sync(0xffffffffu, lane < len && a <= t) | 1u);
    q0 = __shfl_sync(0xffffffffu, a, k);
    q1 = __shfl_sync(0xffffffffu, b, k);
    kv = __shfl_sync(0xffffffffu, c, k);
    return q0 <= t && t < q1 ? lo + k : -1;
}

template <typename S, typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
    constexpr int E = append_values<S>();
    constexpr int kLanes = D / E;              // of a head
    constexpr int kHeads = 32 / kLanes;        // of a step
    constexpr int U = append_steps<S>();
    const int lane = threadIdx.x & 31, in_head = lane % kLanes;
    const Steps steps(p.d.n_head_q, p.d.n_head_kv, kHeads);
    const long long item = (long long)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
    const int t = int(item / p.warps);
    if (t >= p.d.n_tokens) return;
    const int part = int(item - (long long)t * p.warps);
    const int begin = int((long long)part * steps.all() / p.warps);
    const int end = int((long long)(part + 1) * steps.all() / p.warps);

    // the steps of kind 0 (q), 1 (k), 2 (v) are [first_of(kind), first_of(kind + 1))
    auto first_of = [&](int kind) { return kind == 0 ? 0 : steps.q + (kind - 1) * steps.kv; };
    const int own = lane / kLanes;             // this lane's head of a step
    const S* row = static_cast<const S*>(p.qkv) + t * p.qkv_stride + own * D + in_head * E;
    uint4 x[U];
    // the first U steps from step `at` of a kind whose heads start at `src`
    auto load = [&](const S* src, int at, int stop, int heads) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at + u < stop && (at + u) * kHeads + own < heads)
                x[u] = __ldcs(reinterpret_cast<const uint4*>(src + (long long)(at + u) * kHeads * D));
    };
    int kind = begin < first_of(1) ? 0 : begin < first_of(2) ? 1 : 2;
    auto source = [&](int k) { return row + (long long)((k > 0 ? p.d.n_head_q : 0) + (k > 1 ? p.d.n_head_kv : 0)) * D; };
    load(source(kind), begin - first_of(kind), min(end, first_of(kind + 1)) - first_of(kind),
         kind == 0 ? p.d.n_head_q : p.d.n_head_kv);

    int q0, q1, kv;
    const int seq = find_seq(p.d, t, q0, q1, kv);
    if (seq < 0) return;   // a padding token
    const int pos = kv - (q1 - q0) + (t - q0);
    const int page_at = pos / p.d.page_size;
    if (pos < 0 || page_at >= p.d.max_pages || (p.rope && pos >= p.max_pos)) {
        if (lane == 0) flag_input();
        return;
    }
    // pairs of the lane's values: adjacent ones (cs[0 .. E / 2)), or with the partner lane's
    const bool second = in_head >= kLanes / 2;
    float2 cs[E];
    if (p.rope) {
        const float2* c = p.rope + (long long)pos * (D / 2);
        if (p.half) {
#pragma unroll
            for (int i = 0; i < E; ++i) cs[i] = c[in_head % (kLanes / 2) * E + i];
        } else {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) cs[i] = c[in_head * (E / 2) + i];
        }
    }
    long long dst = 0;
    bool has_page = true;
    if (end > steps.q) {
        const int page = p.d.block_table[(long long)seq * p.d.max_pages + page_at];
        has_page = page >= 0 && page < p.d.n_pages;
        if (!has_page && lane == 0) flag_input();
        dst = page * p.d.page_stride + (pos - page_at * p.d.page_size) * p.d.token_stride;
    }
    for (int at = begin; at < end; ++kind) {
        const int base = first_of(kind), stop = min(end, first_of(kind + 1)) - base, from = at - base;
        const int heads = kind == 0 ? p.d.n_head_q : p.d.n_head_kv;
        const float* norm = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
        const bool turn = p.rope && kind < 2;
        const S* src = source(kind);
        if (at != begin) load(src, from, stop, heads);
        T* to = kind == 0 ? static_cast<T*>(p.q) + t * p.d.q_stride : static_cast<T*>(kind == 2 ? p.v : p.k) + dst;
        const long long stride = kind == 0 ? D : p.d.head_stride;   // between heads
        to += own * stride + in_head * E;
        float w[E];
        if (norm) {
#pragma unroll
            for (int i = 0; i < E; ++i) w[i] = norm[in_head * E + i];
        }
        for (int step = from; step < stop; step += U) {
            uint4 now[U];
#pragma unroll
            for (int u = 0; u < U; ++u) now[u] = x[u];
            load(src, step + U, stop, heads);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (step + u >= stop) break;
                float y[E];
#pragma unroll
                for (int i = 0; i < E; ++i) y[i] = to_float<S>(reinterpret_cast<const S*>(&now[u])[i]);
                if (norm) {
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < E; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
                    for (int off = 1; off < kLanes; off <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
                    const float r = rsqrtf(fmaf(ss, 1.0f / float(D), p.eps));
#pragma unroll
                    for (int i = 0; i < E; ++i) y[i] = y[i] * r * w[i];
                }
                if (turn) {
                    if (p.half) {
#pragma unroll
                        for (int i = 0; i < E; ++i) {
                            const float o = __shfl_xor_sync(0xffffffffu, y[i], kLanes / 2);
                            y[i] = second ? o * cs[i].y + y[i] * cs[i].x : y[i] * cs[i].x - o * cs[i].y;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < E / 2; ++i) {
                            const float a = y[2 * i], b = y[2 * i + 1];
                            y[2 * i] = a * cs[i].x - b * cs[i].y;
                            y[2 * i + 1] = a * cs[i].y + b * cs[i].x;
                        }
                    }
                }
                if ((step + u) * kHeads + own < heads && (kind == 0 || has_page))
                    store_values<T, E>(to + (step + u) * kHeads * stride, y);
            }
        }
        at = base + stop;
    }
}

}  // namespace paged
}  // namespace p100b
