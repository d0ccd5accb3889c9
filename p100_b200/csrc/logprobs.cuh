// logprobs.cuh — the scoring of logit rows in one read: log probability and
// rank of a given token, entropy, and the top alternatives.
//
// With m = max x, s = sum e^(x-m), u = sum e^(x-m) (x-m):
//   lse = m + ln s,  logprob = x_tok - lse,  entropy = ln s - u / s.
// Every thread keeps a running (m, s, u) in FP32 (in units of log2 e) and
// rescales them when a vector of logits raises its maximum; the threads' and
// the parts' triples are joined at the end.  -inf and NaN count as masked.
//
// The top alternatives need no second read of the row: the k-th largest of
// the threads' maxima is a lower bound of the row's k-th largest value, and
// only threads whose own maximum reaches it can hold one of the k.  On random
// rows barely more than k threads do, so the block reads just their vectors
// again (from L2), keeps the values that reach the bound and ranks them by
// (value, lowest index).  Rows with more such values than the buffer holds
// (long runs of equal logits) take k passes over the part instead, each
// finding the largest key below the previous one.
//
// Bytes bound it (the logits are read once).  Few rows are split over
// several CTAs; the last one of a row (an atomic ticket, no waiting) joins the
// parts.
#pragma once
#include "paged.cuh"

namespace p100b {
namespace lp {

constexpr int kThreads = 512;
constexpr int kMaxTop = 32;
constexpr int kCand = 2048;       // candidates kept in shared memory
constexpr int kMaxParts = 64;     // parts x top <= kCand
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
    const void* x;
    long long stride;     // between rows, in elements
    int n, rows, parts, part_len;   // part_len: a multiple of a vector's elements
    int top;
    const int* token;     // [rows] or null
    float *logprob, *entropy;
    int *rank, *top_index;
    float* top_logprob;
    float4* ws_sums;                // [rows][parts] {m, s, u, count as int bits}
    unsigned long long* ws_keys;    // [rows][parts][top]
    unsigned* tickets;              // [rows]
};

// Larger value first, then lower index: one unsigned order.  -0 equals 0.
__device__ __forceinline__ unsigned long long make_key(float v, unsigned idx) {
    unsigned b = __float_as_uint(v + 0.0f);
    b = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((unsigned long long)b << 32) | (~idx);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
    const unsigned b = unsigned(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ unsigned key_index(unsigned long long k) { return ~unsigned(k); }

// (m, s, u) of the union of two disjoint sets.
__device__ __forceinline__ void join(float& m, float& s, float& u, float m2, float s2, float u2) {
    const float mm = fmaxf(m, m2);
    const float d1 = fmaxf((m - mm) * kLog2e, -1e4f), d2 = fmaxf((m2 - mm) * kLog2e, -1e4f);
    const float a = paged::exp2_approx(d1), b = paged::exp2_approx(d2);
    u = a * fmaf(d1, s, u) + b * fmaf(d2, s2, u2);
    s = a * s + b * s2;
    m = mm;
}

template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    __device__ static __forceinline__ void load(const T* p, float (&f)[N]) { unpack(*reinterpret_cast<const uint4*>(p), f); }
    __device__ static __forceinline__ void unpack(const uint4& w, float (&f)[N]) {
        const T* s = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = paged::to_float<T>(s[i]);
    }
};

struct Running {
    float m = -3.402823466e38f, s = 0.f, u = 0.f;
    int above = 0;

    // ge: a value counts above the token if it is >= ge.
    template <int N>
    __device__ __forceinline__ void add(const float (&f)[N], float ge) {
        float c = f[0];
#pragma unroll
        for (int i = 1; i < N; ++i) c = fmaxf(c, f[i]);
        if (c > m) {
            const float d = fmaxf((m - c) * kLog2e, -1e4f);
            const float a = paged::exp2_approx(d);
            u = a * fmaf(d, s, u);
            s *= a;
            m = c;
        }
        // the difference first: m log2 e would overflow for a row of the type's lowest value
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = fmaxf((f[i] - m) * kLog2e, -1e4f);
            const float e = paged::exp2_approx(d);
            s += e;
            u = fmaf(e, d, u);
            above += f[i] >= ge;
        }
    }
};

// The keys in s_key[0, count) ranked: the best `top` into best[0, top), zeros
// behind them.  Every thread of the block calls it.
__device__ __forceinline__ void rank_keys(const unsigned long long* s_key, int count, int top,
                                          unsigned long long* best) {
    for (int i = threadIdx.x; i < top; i += kThreads) best[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const unsigned long long k = s_key[i];
        int r = 0;
        for (int j = 0; j < count; ++j) r += s_key[j] > k;
        if (r < top) best[r] = k;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const Params p) {
    constexpr int N = Vec<T>::N;
    constexpr int W = kThreads / 32;
    __shared__ unsigned long long s_key[kCand];
    __shared__ unsigned long long s_best[kMaxTop];
    __shared__ float s_max[kThreads];
    __shared__ float s_m[W], s_s[W], s_u[W];
    __shared__ int s_above[W];
    __shared__ int s_hit[kThreads];
    __shared__ int s_count, s_hits, s_last;
    __shared__ unsigned long long s_word[W];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts;
    const T* x = static_cast<const T*>(p.x) + row * p.stride;
    // elements [lo, hi) of the row are this part's; vectors start at the row's
    // first 16-byte boundary, `head` elements in
    const int head = min(p.n, int(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    const long long part_lo = part ? (long long)head + (long long)part * p.part_len : 0;
    const int lo = int(min((long long)p.n, part_lo));
    const int hi = part + 1 == p.parts ? p.n : int(min((long long)p.n, (long long)head + (long long)(part + 1) * p.part_len));
    const int vlo = part ? lo : head;                 // first vector element
    const int nvec = max(0, hi - vlo) / N;
    const int tail = vlo + nvec * N;                  // elements behind the vectors

    // the token's logit: values >= it count before its index, > it behind
    int tok = -1;
    float xt = -INFINITY, gt = INFINITY;
    if (p.token) {
        tok = p.token[row];
        if (tok < 0 || tok >= p.n) {
            if (tok != -1 && part == 0 && tid == 0) paged::flag_input();
            tok = -1;
        } else {
            xt = paged::to_float<T>(x[tok]);
            if (isnan(xt)) xt = -INFINITY;
        }
    }
    gt = xt == INFINITY ? __int_as_float(0x7fc00000) : nextafterf(xt, INFINITY);
    if (tok < 0) gt = __int_as_float(0x7fc00000);
    const float ge = tok < 0 ? gt : xt;

    Running r;
    const uint4* v = reinterpret_cast<const uint4*>(x + vlo);
    constexpr int U = 4;   // vectors in flight a thread
    int i = tid;
    for (; i + (U - 1) * kThreads < nvec; i += U * kThreads) {
        uint4 w[U];
#pragma unroll
        for (int j = 0; j < U; ++j) w[j] = v[i + j * kThreads];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float f[N];
            Vec<T>::unpack(w[j], f);
            r.add(f, vlo + (i + j * kThreads) * N < tok ? ge : gt);
        }
    }
    for (; i < nvec; i += kThreads) {
        float f[N];
        Vec<T>::unpack(v[i], f);
        r.add(f, vlo + i * N < tok ? ge : gt);
    }
    // single elements in front of and behind the vectors
    const int nfront = vlo - lo, nback = hi - tail;
    if (tid < nfront + nback) {
        const int idx = tid < nfront ? lo + tid : tail + tid - nfront;
        float f[1] = {paged::to_float<T>(x[idx])};
        r.add(f, idx < tok ? ge : gt);
    }
    // the vector that holds the token counted its equals as if all were in
    // front of it (it starts before the token) : take those behind it out
    if (tok >= vlo && tok < tail && tid == 0) {
        const int base = vlo + (tok - vlo) / N * N;
        if (base < tok)
            for (int e = tok; e < base + N; ++e) r.above -= paged::to_float<T>(x[e]) == xt;
    }

    // join the threads
    s_max[tid] = r.m;
    float m = r.m, s = r.s, u = r.u;
    int above = r.above;
    if (s == 0.f && m != INFINITY) s_max[tid] = -INFINITY;   // nothing but masked logits
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off),
                    u2 = __shfl_xor_sync(0xffffffffu, u, off);
        join(m, s, u, m2, s2, u2);
    }
    above = __reduce_add_sync(0xffffffffu, above);
    if (lane == 0) s_m[warp] = m, s_s[warp] = s, s_u[warp] = u, s_above[warp] = above;
    if (tid == 0) s_count = s_hits = 0;
    __syncthreads();
    m = s_m[0], s = s_s[0], u = s_u[0], above = s_above[0];
#pragma unroll 1
    for (int j = 1; j < W; ++j) {
        join(m, s, u, s_m[j], s_s[j], s_u[j]);
        above += s_above[j];
    }

    const int top = p.top;
    if (top > 0) {
        // the top-th largest of the threads' maxima, by a search over the
        // ordered bits (the largest t with at least `top` maxima >= t)
        const unsigned mine = unsigned(make_key(s_max[tid], 0) >> 32);
        unsigned t = 0;
#pragma unroll 1
        for (int b = 31; b >= 0; --b) {
            const unsigned c = t | (1u << b);
            if (__syncthreads_count(mine >= c) >= top) t = c;
        }
        const float bound = __uint_as_float(t & 0x80000000u ? t & 0x7fffffffu : ~t);
        if (s_max[tid] >= bound && s_max[tid] > -INFINITY) s_hit[atomicAdd(&s_hits, 1)] = tid;
        __syncthreads();
        // the hit threads' vectors, shared out over the block
        const int per = (nvec + kThreads - 1) / kThreads;
        const long long work = (long long)s_hits * per;
        for (long long k = tid; k < work; k += kThreads) {
            const int h = int(k / per);
            const int at = s_hit[h] + int(k - (long long)h * per) * kThreads;
            if (at >= nvec) continue;
            float f[N];
            Vec<T>::unpack(v[at], f);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (f[e] >= bound && f[e] > -INFINITY) {
                    const int c = atomicAdd(&s_count, 1);
                    if (c < kCand) s_key[c] = make_key(f[e], unsigned(vlo + at * N + e));
                }
        }
        if (tid < nfront + nback) {
            const int idx = tid < nfront ? lo + tid : tail + tid - nfront;
            const float f = paged::to_float<T>(x[idx]);
            if (f >= bound && f > -INFINITY) {
                const int c = atomicAdd(&s_count, 1);
                if (c < kCand) s_key[c] = make_key(f, unsigned(idx));
            }
        }
        __syncthreads();
        if (s_count <= kCand) {
            rank_keys(s_key, s_count, top, s_best);
        } else {
            unsigned long long below = ~0ull;
#pragma unroll 1
            for (int k = 0; k < top; ++k) {
                unsigned long long best = 0;
                for (int e = lo + tid; e < hi; e += kThreads) {
                    const float f = paged::to_float<T>(x[e]);
                    if (f > -INFINITY) {
                        const unsigned long long key = make_key(f, unsigned(e));
                        if (key < below && key > best) best = key;
                    }
                }
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) {
                    const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, off);
                    if (o > best) best = o;
                }
                if (lane == 0) s_word[warp] = best;
                __syncthreads();
                best = s_word[0];
                for (int j = 1; j < W; ++j)
                    if (s_word[j] > best) best = s_word[j];
                if (tid == 0) s_best[k] = best;
                below = best;
                __syncthreads();
            }
        }
    }

    if (p.parts > 1) {
        const long long at = (long long)row * p.parts + part;
        if (tid < top) p.ws_keys[at * top + tid] = s_best[tid];
        if (tid == 0) p.ws_sums[at] = make_float4(m, s, u, __int_as_float(above));
        __threadfence();
        __syncthreads();
        if (tid == 0) s_last = atomicAdd(p.tickets + row, 1u) == unsigned(p.parts - 1);
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        if (tid == 0) p.tickets[row] = 0;   // ready for the next call
        const long long first = (long long)row * p.parts;
        if (tid < p.parts) {
            const float4 w = __ldcg(p.ws_sums + first + tid);
            s_max[tid] = w.x;
            s_max[kMaxParts + tid] = w.y;
            s_max[2 * kMaxParts + tid] = w.z;
            s_hit[tid] = __float_as_int(w.w);
        }
        for (int k = tid; k < p.parts * top; k += kThreads) s_key[k] = __ldcg(p.ws_keys + first * top + k);
        __syncthreads();
        m = s_max[0], s = s_max[kMaxParts], u = s_max[2 * kMaxParts], above = s_hit[0];
        for (int j = 1; j < p.parts; ++j) {
            join(m, s, u, s_max[j], s_max[kMaxParts + j], s_max[2 * kMaxParts + j]);
            above += s_hit[j];
        }
        if (top > 0) {
            // keys of absent alternatives are 0 and equal: they rank behind every other
            rank_keys(s_key, p.parts * top, top, s_best);
        }
    }

    const bool infinite = m == INFINITY;   // a row with +inf has no finite log probabilities
    const bool empty = s == 0.f && !infinite;
    const float ls = kLn2 * log2f(s);
    const float nan = __int_as_float(0x7fc00000);
    if (tid == 0) {
        if (p.logprob) p.logprob[row] = tok < 0 ? 0.f : infinite ? nan : empty ? -INFINITY : (xt - m) - ls;
        if (p.rank) p.rank[row] = tok < 0 ? -1 : above;
        if (p.entropy) p.entropy[row] = infinite ? nan : empty ? 0.f : ls - kLn2 * (u / s);
    }
    if (tid < top) {
        const unsigned long long k = s_best[tid];
        const long long at = (long long)row * top + tid;
        p.top_index[at] = k ? int(key_index(k)) : -1;
        p.top_logprob[at] = !k ? -INFINITY : infinite ? nan : (key_value(k) - m) - ls;
    }
}

}  // namespace lp
}  // namespace p100b
