// paged_append.cuh — a chunk of new tokens into a paged cache: the norms of
// the query and key heads, their rotation and the write to the pages in one
// pass over the fused q|k|v rows.
//
// Per head x of a token at position p: x' = x w / sqrt(mean(x^2) + eps) (with
// norm weights), then for each pair (a, b): (a cos - b sin, a sin + b cos)
// with the table's angle of p; pairs are adjacent values, or value i with
// value i + D/2.  All in FP32; the one rounding is the store to 16 bits.
//
// Bytes bound it: every value is read once and written once.  A warp takes
// four heads of one token (a lane the D/32 consecutive values that one vector
// load gives), so four loads are in flight before the first reduction, the
// token's sequence is searched once and its angles are read once for four
// heads; adjacent pairs stay inside a lane and the halves' partner sits 16
// lanes away.
#pragma once
#include "paged.cuh"

namespace p100b {
namespace paged {

constexpr int kAppendThreads = 256;
constexpr int kAppendHeads = 4;   // heads of a warp

struct AppendParams {
    Desc d;
    const void* qkv;
    long long qkv_stride;
    const float* q_norm;    // [D] or null
    const float* k_norm;
    float eps;
    const float2* rope;     // [max_pos][D/2] or null
    int max_pos, half;
    void *q, *k, *v;
};

// E consecutive values at p (aligned to their size) as floats.
template <typename S, int E>
__device__ __forceinline__ void load_values(const S* p, float (&x)[E]) {
    if constexpr (sizeof(S) * E == 16) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p));
        const S* s = reinterpret_cast<const S*>(&w);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_float<S>(s[i]);
    } else if constexpr (sizeof(S) * E == 8) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2*>(p));
        const S* s = reinterpret_cast<const S*>(&w);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_float<S>(s[i]);
    } else {
        const uint32_t w = __ldcs(reinterpret_cast<const unsigned*>(p));
        const S* s = reinterpret_cast<const S*>(&w);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_float<S>(s[i]);
    }
}

template <typename T, int E>
__device__ __forceinline__ void store_values(T* p, const float (&x)[E]) {
    if constexpr (E == 4)
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    else
        *reinterpret_cast<uint32_t*>(p) = pack2<T>(x[0], x[1]);
}

// The sequence of token t, or -1: the last s with q_start[s] <= t, found 32
// candidates at a time, if t also lies before q_start[s + 1].
__device__ __forceinline__ int find_seq(const Desc& d, int t, int& q0, int& q1) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = d.n_seq;   // the answer lies in [lo, lo + len)
    while (len > 1) {
        const int step = (len + 31) / 32;
        const int i = lo + lane * step;
        const bool at = lane * step < len && d.q_start[i] <= t;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, at) | 1u);
        lo += k * step;
        len = min(step, len - k * step);
    }
    q0 = d.q_start[lo];
    q1 = d.q_start[lo + 1];
    return q0 <= t && t < q1 ? lo : -1;
}

template <typename S, typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int heads = p.d.n_head_q + 2 * p.d.n_head_kv;
    const int groups = (heads + kAppendHeads - 1) / kAppendHeads;
    const long long item = (long long)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
    const int t = int(item / groups);
    if (t >= p.d.n_tokens) return;
    const int h0 = int(item - (long long)t * groups) * kAppendHeads;
    const int nh = min(kAppendHeads, heads - h0);

    const S* row = static_cast<const S*>(p.qkv) + t * p.qkv_stride + (long long)h0 * D + lane * E;
    float x[kAppendHeads][E];
#pragma unroll
    for (int h = 0; h < kAppendHeads; ++h)
        if (h < nh) load_values<S, E>(row + h * D, x[h]);

    int q0, q1;
    const int seq = find_seq(p.d, t, q0, q1);
    if (seq < 0) return;   // a padding token
    const int pos = p.d.kv_len[seq] - (q1 - q0) + (t - q0);
    const int page_at = pos / p.d.page_size;
    if (pos < 0 || page_at >= p.d.max_pages || (p.rope && pos >= p.max_pos)) {
        if (lane == 0) flag_input();
        return;
    }
    float2 cs[E];
    if (p.rope) {
        const float2* c = p.rope + (long long)pos * (D / 2);
        if (p.half) {
#pragma unroll
            for (int i = 0; i < E; ++i) cs[i] = c[(lane & 15) * E + i];
        } else {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) cs[i] = c[lane * (E / 2) + i];
        }
    }
    long long dst = 0;
    bool has_page = true;
    if (h0 + nh > p.d.n_head_q) {
        const int page = p.d.block_table[(long long)seq * p.d.max_pages + page_at];
        has_page = page >= 0 && page < p.d.n_pages;
        if (!has_page && lane == 0) flag_input();
        dst = page * p.d.page_stride + (pos - page_at * p.d.page_size) * p.d.token_stride;
    }
#pragma unroll
    for (int h = 0; h < kAppendHeads; ++h) {
        if (h >= nh) break;
        const int head = h0 + h;
        const bool is_q = head < p.d.n_head_q, is_v = head >= p.d.n_head_q + p.d.n_head_kv;
        float y[E];
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = x[h][i];
        const float* w = is_v ? nullptr : is_q ? p.q_norm : p.k_norm;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) ss = fmaf(y[i], y[i], ss);
            const float r = 1.0f / sqrtf(warp_sum(ss) / float(D) + p.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] = y[i] * r * w[lane * E + i];
        }
        if (p.rope && !is_v) {
            if (p.half) {   // lanes 0-15 hold the first values of the pairs, lanes 16-31 the second
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float o = __shfl_xor_sync(0xffffffffu, y[i], 16);
                    y[i] = lane < 16 ? y[i] * cs[i].x - o * cs[i].y : o * cs[i].y + y[i] * cs[i].x;
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
        if (is_q) {
            store_values<T, E>(static_cast<T*>(p.q) + t * p.d.q_stride + (long long)head * D + lane * E, y);
        } else if (has_page) {
            const int kh = is_v ? head - p.d.n_head_q - p.d.n_head_kv : head - p.d.n_head_q;
            store_values<T, E>(static_cast<T*>(is_v ? p.v : p.k) + dst + kh * p.d.head_stride + lane * E, y);
        }
    }
}

}  // namespace paged
}  // namespace p100b
