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
// the maxima of 64 groups of threads is a lower bound of the row's k-th
// largest value, and only a thread's eighth of the row whose maximum reaches it
// can hold one of the k.  On random rows that is one to two times k eighths,
// so the block reads just their vectors again (from L2), keeps the values that
// reach the bound and ranks them by (value, lowest index).  Where many do (long
// runs of equal logits) k passes over them, or over the part where they are
// more than the buffer holds, each find the largest key below the previous one.
//
// Bytes bound it (the logits are read once); next come the exponentials, one a
// logit, 0.7 of the time that 16-bit logits take to read.  So the rest is kept
// small: 16-bit logits are masked, compared and counted two at a time before
// their conversion, the sums run on pairs of FP32.  Few rows are split over
// several CTAs; the last one of a row (an atomic ticket, no waiting) joins the
// parts.  Measured: 2048 rows of 128256 bf16 with 8 alternatives 116 to 126 us
// (4.2 to 4.5 TB/s), the loads alone 88; one fp32 row with 20 alternatives 12 us; 333 rows
// of 32003 fp32 with 32 alternatives 22.6 us.  128 threads and 8 CTAs an SM: 118
// us against 131 of 256 threads and 4.
#pragma once
#include <type_traits>

#include "paged.cuh"

namespace p100b {
namespace lp {

constexpr int kThreads = 128;
constexpr int kCtas = 8;           // of an SM
constexpr int kSpans = 8;          // parts of a thread's vectors with a maximum of their own
constexpr int kAhead = 4;          // vectors a thread has on their way
constexpr int kGroups = 64, kGroup = kThreads / kGroups;   // groups of threads, each with a maximum
constexpr int kMaxTop = 32;
constexpr int kCand = 2048;       // candidates kept in shared memory, twice kMaxParts x kMaxTop
constexpr int kRanked = 32;       // rounds of comparisons that ranking may take for each alternative
constexpr int kMaxLogits = 1 << 24;
constexpr int kMaxParts = 32;     // a lane each; parts x top <= kCand
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

// The unsigned order of values.  -0 equals 0.
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float ordered_value(unsigned b) {
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
// Larger value first, then lower index: one unsigned order.
__device__ __forceinline__ unsigned long long make_key(float v, unsigned idx) {
    return ((unsigned long long)ordered(v) << 32) | (~idx);
}
__device__ __forceinline__ float key_value(unsigned long long k) { return ordered_value(unsigned(k >> 32)); }
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

// Logits at or below the floor of their type count as masked in the first
// pass; a part whose largest is not above it, or not below `ceil` (where
// (floor - m) log2 e nears FP32's range), is summed again logit by logit.
template <typename T>
struct Range {
    static constexpr float floor = -8.507059173023462e37f, ceil = 8.507059173023462e37f;   // 2^126, of FP32 and bfloat16
};
template <>
struct Range<__half> {
    static constexpr float floor = -65504.f, ceil = 3.402823466e38f;
};

// ------------------------------------------------------------ 16 bytes of logits
// N logits: keep() replaces NaN and what lies below the floor by it, largest()
// is their maximum, count() how many reach `ge`, get() the logits in FP32.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int N = 4;
    float f[4];
    __device__ __forceinline__ explicit Vec(const uint4& w) {
        f[0] = __uint_as_float(w.x);
        f[1] = __uint_as_float(w.y);
        f[2] = __uint_as_float(w.z);
        f[3] = __uint_as_float(w.w);
    }
    using Bound = float;
    __device__ static __forceinline__ Bound bound(float ge) { return ge; }
    __device__ __forceinline__ void count(Bound ge, unsigned& n) const {
        n += (f[0] >= ge) + (f[1] >= ge) + (f[2] >= ge) + (f[3] >= ge);
    }
    __device__ static __forceinline__ int counted(unsigned n) { return int(n); }
    __device__ __forceinline__ void keep() {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = fmaxf(f[i], Range<float>::floor);
    }
    __device__ __forceinline__ float largest() const { return fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])); }
    __device__ __forceinline__ void get(float (&o)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = f[i];
    }
};
template <typename T, typename T2>
struct Vec16 {
    static constexpr int N = 8;
    T2 h[4];
    __device__ __forceinline__ explicit Vec16(const uint4& w) {
        const unsigned v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const T2*>(&v[i]);
    }
    // Each pair's comparison is 0xffff in the half that holds; added up as one
    // word, lo and hi of them make 65535 lo - 65536 hi modulo 2^32.  counted()
    // needs lo, hi < 2^16: a span has an eighth of that at most (a thread's whole
    // row, 2^16 of each at kMaxLogits, would be too many).
    using Bound = T2;
    __device__ __forceinline__ void count(Bound ge, unsigned& n) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) n += __hge2_mask(h[i], ge);
    }
    __device__ static __forceinline__ int counted(unsigned n) {
        const unsigned lo = -n & 0xffffu;
        return int(lo + ((lo - ((n + lo) >> 16)) & 0xffffu));
    }
    __device__ __forceinline__ void keep(T2 lowest) {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __hmax2(h[i], lowest);
    }
    __device__ __forceinline__ float largest() const {
        const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(paged::to_float<T>(m.x), paged::to_float<T>(m.y));
    }
    __device__ __forceinline__ void get(float (&o)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = paged::to_float<T>(h[i].x);
            o[2 * i + 1] = paged::to_float<T>(h[i].y);
        }
    }
};
template <>
struct Vec<__half> : Vec16<__half, __half2> {
    using Vec16::Vec16;
    __device__ static __forceinline__ Bound bound(float ge) { return __float2half2_rn(ge); }
    __device__ __forceinline__ void keep() { Vec16::keep(__half2half2(__ushort_as_half(0xfbff))); }
};
template <>
struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16, __nv_bfloat162> {
    using Vec16::Vec16;
    __device__ static __forceinline__ Bound bound(float ge) { return __float2bfloat162_rn(ge); }
    __device__ __forceinline__ void keep() { Vec16::keep(__bfloat162bfloat162(__ushort_as_bfloat16(0xfe80))); }
};
// The next larger value of T (`ge` of the logits behind the token).
template <typename T>
__device__ __forceinline__ float next_above(float x);
template <>
__device__ __forceinline__ float next_above<float>(float x) { return nextafterf(x, INFINITY); }
__device__ __forceinline__ unsigned short next_bits(unsigned short b) {   // of a 16-bit float below +inf
    return (b & 0x7fff) == 0 ? 1 : b & 0x8000 ? b - 1 : b + 1;
}
template <>
__device__ __forceinline__ float next_above<__half>(float x) {
    return __half2float(__ushort_as_half(next_bits(__half_as_ushort(__float2half_rn(x)))));
}
template <>
__device__ __forceinline__ float next_above<__nv_bfloat16>(float x) {
    return __bfloat162float(__ushort_as_bfloat16(next_bits(__bfloat16_as_ushort(__float2bfloat16_rn(x)))));
}

// A thread's running sums, relative to a logit m of the row that none of the
// thread's exceeds.  (A lower reference would be cheaper to keep but costs the
// entropy of rows with one dominant logit its last digits.)
struct Running {
    float m = -3.402823466e38f;
    float top = -3.402823466e38f;   // the largest logit
    uint64_t s2 = 0, u2 = 0;        // the sums, in two halves

    __device__ __forceinline__ void rise(float c) {
        const float d = fmaxf((m - c) * kLog2e, -1e4f);
        const float a = paged::exp2_approx(d);
        u2 = paged::mul2(paged::pair(a, a), paged::fma2(paged::pair(d, d), s2, u2));
        s2 = paged::mul2(paged::pair(a, a), s2);
        m = c;
    }
    // The largest of the logits that add() gets next.
    __device__ __forceinline__ void reach(float c) {
        top = fmaxf(top, c);
        if (c > m) rise(c);
    }
    // N logits within the range of their type.  The difference comes first, exact
    // or nearly: x log2 e - m log2 e in one fma would save an operation (2 us of
    // 2048 rows' 120) but puts the rounding of m log2 e, up to 2^-24 |m|,
    // into every term, which large or sharply peaked rows show.
    template <int N>
    __device__ __forceinline__ void add(const float (&f)[N]) {
        const uint64_t l2 = paged::pair(kLog2e, kLog2e), minus_m2 = paged::pair(-m, -m);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint64_t d2 = paged::mul2(paged::add2(paged::pair(f[i], f[i + 1]), minus_m2), l2);
            float a, b;
            paged::unpair(d2, a, b);
            const uint64_t e2 = paged::pair(paged::exp2_approx(a), paged::exp2_approx(b));
            s2 = paged::add2(s2, e2);
            u2 = paged::fma2(e2, d2, u2);
        }
    }
    // One logit of any size but -inf.
    __device__ __forceinline__ void add_one(float f) {
        reach(f);
        const float d = fmaxf((f - m) * kLog2e, -1e4f);
        const float e = paged::exp2_approx(d);
        s2 = paged::add2(s2, paged::pair(e, 0.f));
        u2 = paged::add2(u2, paged::pair(e * d, 0.f));
    }
    __device__ __forceinline__ float sum() const {
        float a, b;
        paged::unpair(s2, a, b);
        return a + b;
    }
    __device__ __forceinline__ float weighted() const {
        float a, b;
        paged::unpair(u2, a, b);
        return a + b;
    }
};

// The best `top` keys of those that each(take) gives to take() on every thread,
// one after the other, into best[0, top), zeros behind them.  Every thread of
// the block calls it.
template <typename Each>
__device__ __forceinline__ void pick_keys(int top, unsigned long long* best, unsigned long long* word, Each each) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned long long below = ~0ull;
#pragma unroll 1
    for (int k = 0; k < top; ++k) {
        unsigned long long most = 0;
        each([&](unsigned long long key) {
            if (key < below && key > most) most = key;
        });
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            const unsigned long long o = __shfl_xor_sync(0xffffffffu, most, off);
            if (o > most) most = o;
        }
        if (lane == 0) word[warp] = most;
        __syncthreads();
        most = word[0];
        for (int j = 1; j < kThreads / 32; ++j)
            if (word[j] > most) most = word[j];
        if (threadIdx.x == 0) best[k] = most;
        below = most;
        __syncthreads();
    }
}
// The same of the keys in s_key[0, count): ranked, every pair compared, or
// picked where they are many (1000 keys, top 20: 62 us ranked, 17 picked).
__device__ __forceinline__ void best_keys(const unsigned long long* s_key, int count, int top, unsigned long long* best,
                                          unsigned long long* word) {
    if (count * ((count + kThreads - 1) / kThreads) <= kRanked * top) {
        for (int i = threadIdx.x; i < top; i += kThreads) best[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += kThreads) {
            const unsigned long long k = s_key[i];
            int r = 0;
            for (int j = 0; j < count; ++j) r += s_key[j] > k;
            if (r < top) best[r] = k;
        }
        __syncthreads();
    } else {
        pick_keys(top, best, word, [&](auto take) {
            for (int i = threadIdx.x; i < count; i += kThreads) take(s_key[i]);
        });
    }
}

// One part of a row, and where its vectors lie.
template <typename T>
struct Part {
    int row, part;
    const T* x;
    int lo, hi;       // its logits
    int vlo, nvec;    // first logit and number of its vectors
    int tok;          // the row's token, -1 for none
    float given;      // its logit

    __device__ __forceinline__ Part(const Params& p, int item) {
        constexpr int N = Vec<T>::N;
        row = item / p.parts;
        part = item - row * p.parts;
        x = static_cast<const T*>(p.x) + row * p.stride;
        // vectors start at the row's first 16-byte boundary, `head` logits in
        const int head = min(p.n, int(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
        lo = part ? int(min((long long)p.n, (long long)head + (long long)part * p.part_len)) : 0;
        hi = part + 1 == p.parts ? p.n : int(min((long long)p.n, (long long)head + (long long)(part + 1) * p.part_len));
        vlo = part ? lo : head;
        nvec = max(0, hi - vlo) / N;
    }
    __device__ __forceinline__ void load_token(const Params& p) {
        tok = p.token ? p.token[row] : -1;
        given = -INFINITY;
        if (tok >= 0 && tok < p.n) given = paged::to_float<T>(x[tok]);
    }
    __device__ __forceinline__ void fetch(uint4 (&w)[kAhead]) const {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (int(threadIdx.x) + j * kThreads < nvec)
                w[j] = reinterpret_cast<const uint4*>(x + vlo)[threadIdx.x + j * kThreads];
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, kCtas) logprobs_kernel(const Params p) {
    constexpr int N = Vec<T>::N;
    constexpr int W = kThreads / 32;
    __shared__ unsigned long long s_key[kCand];
    __shared__ unsigned long long s_best[kMaxTop];
    __shared__ unsigned long long s_word[W];
    __shared__ float s_m[W], s_s[W], s_u[W];
    __shared__ float s_group[kGroups];
    __shared__ __align__(16) unsigned s_rank[kGroups];
    __shared__ float s_bound;
    __shared__ float s_span[kSpans][kThreads];
    uint64_t(*s_save)[kThreads] = reinterpret_cast<uint64_t(*)[kThreads]>(s_key);   // a thread's state before a span
    float* s_back = reinterpret_cast<float*>(s_key + 2 * kThreads);
    __shared__ int s_above[W];
    __shared__ int s_count, s_hits, s_last;
    int* s_hit = reinterpret_cast<int*>(s_key + kCand / 2);   // spans to read again: kSpans x kThreads
    static_assert(kGroups == 64 && W == 4 && kMaxTop <= 32 && kMaxParts <= 32, "a lane for each alternative and part, 16 groups a warp");
    static_assert(kMaxLogits / kThreads / kSpans / 2 < 1 << 16, "counts of a span");
    static_assert(kSpans * kThreads * sizeof(int) <= kCand / 2 * sizeof(unsigned long long), "spans beside half of the keys");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint4 w[kAhead];
    Part<T> it(p, blockIdx.x);
    it.fetch(w);
    it.load_token(p);
    const int row = it.row, part = it.part, lo = it.lo, hi = it.hi, vlo = it.vlo, nvec = it.nvec;
    const T* x = it.x;
    const int tail = vlo + nvec * N;                  // logits behind the vectors
    const int nfront = vlo - lo, nsingle = nfront + hi - tail;   // logits outside the vectors, a thread each
    const int single = tid < nfront ? lo + tid : tail + tid - nfront;

    // the token's logit: values >= it count before its index, > it behind
    const float nan = __int_as_float(0x7fc00000);
    int tok = it.tok;
    float xt = -INFINITY, ge = nan, gt = nan;
    if (tok < 0 || tok >= p.n) {
        if (tok != -1 && part == 0 && tid == 0) paged::flag_input();
        tok = -1;
    } else {
        xt = isnan(it.given) ? -INFINITY : it.given;
        ge = xt;
        if (xt < INFINITY) gt = next_above<T>(xt);
    }

    Running r;
    unsigned reached = 0;   // of the span
    int above = 0;
    const typename Vec<T>::Bound bge = Vec<T>::bound(ge), bgt = Vec<T>::bound(gt);
    const uint4* v = reinterpret_cast<const uint4*>(x + vlo);
    auto take = [&](const uint4& q4, int i) {
        Vec<T> q(q4);
        q.count(vlo + i * N < tok ? bge : bgt, reached);
        q.keep();
        float f[N];
        q.get(f);
        r.reach(q.largest());
        r.add(f);
    };
    bool masked;   // the row seems to hold masked logits
    {
        // The block's first vectors give every thread its first reference:
        // their maximum, which few of the later logits exceed.
        float c = -3.402823466e38f;
        bool low = false;
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (tid + j * kThreads < nvec) {
                Vec<T> q(w[j]);
                float f[N];
                q.get(f);
#pragma unroll
                for (int e = 0; e < N; ++e) low = low || !(f[e] > Range<T>::floor);
                q.keep();
                c = fmaxf(c, q.largest());
            }
        c = warp_max(c);
        if (lane == 0) s_m[warp] = c;
        masked = __syncthreads_or(low);
        c = s_m[0];
        for (int j = 1; j < W; ++j) c = fmaxf(c, s_m[j]);
        if (c > r.m) r.rise(c);
    }
    // a span: `per` vectors of every thread, a multiple of kAhead
    const int rounds = (nvec + kAhead * kThreads - 1) / (kAhead * kThreads);
    const int per = (rounds + kSpans - 1) / kSpans * kAhead;
    float best = r.top;   // the thread's largest logit
    auto run = [&](int k, int end, auto mask, bool loaded) {
#pragma unroll 1
        for (; k < end && (k + kAhead) * kThreads <= nvec; k += kAhead) {   // nobody's vectors end here
            const int i = tid + k * kThreads;
            if (!loaded) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) w[j] = v[i + j * kThreads];
            }
            loaded = false;
            float c = -3.402823466e38f;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                Vec<T> q(w[j]);
                q.count(vlo + (i + j * kThreads) * N < tok ? bge : bgt, reached);
                if (decltype(mask)::value) q.keep();
                c = fmaxf(c, q.largest());
            }
            r.reach(c);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                Vec<T> q(w[j]);
                if (decltype(mask)::value) q.keep();
                float f[N];
                q.get(f);
                r.add(f);
            }
        }
#pragma unroll 1
        for (; k < end; ++k)
            if (tid + k * kThreads < nvec) take(v[tid + k * kThreads], tid + k * kThreads);
    };
    for (int span = 0; span < kSpans; ++span) {
        r.top = -3.402823466e38f;
        const int begin = min(span * per, rounds * kAhead), end = min(begin + per, rounds * kAhead);
        if (begin < end) {
            if (!masked) {
                s_save[0][tid] = r.s2;
                s_save[1][tid] = r.u2;
                s_back[tid] = r.m;
                run(begin, end, std::false_type(), begin == 0);
            }
            if (masked || isnan(r.weighted())) {
                if (!masked) {
                    r.s2 = s_save[0][tid];
                    r.u2 = s_save[1][tid];
                    r.m = s_back[tid];
                    r.top = -3.402823466e38f;
                    reached = 0;
                }
                run(begin, end, std::true_type(), false);
            }
        }
        s_span[span][tid] = r.top;
        best = fmaxf(best, r.top);
        above += Vec<T>::counted(reached);
        reached = 0;
    }
    r.top = best;
    if (tid < nsingle) {
        const float f = paged::to_float<T>(x[single]);
        above += f >= (single < tok ? ge : gt);
        if (f > Range<T>::floor) r.add_one(f);
    }
    // the vector that holds the token counted its equals as if all were in
    // front of it (it starts before the token): take those behind it out
    if (tok >= vlo && tok < tail && tid == 0) {
        const int base = vlo + (tok - vlo) / N * N;
        if (base < tok)
            for (int e = tok; e < base + N; ++e) above -= paged::to_float<T>(x[e]) == xt;
    }
    // join the threads
    above = __reduce_add_sync(0xffffffffu, above);
    if (lane == 0) s_above[warp] = above;
    if (tid == 0) s_count = s_hits = 0;
    __syncthreads();   // s_m has been read
    float m, s, u, most;   // most: the part's largest logit
    auto join_threads = [&]() {
        m = r.m, s = r.sum(), u = r.weighted();
        float group = r.top;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            if (off < kGroup) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, off));
            const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off),
                        u2 = __shfl_xor_sync(0xffffffffu, u, off);
            join(m, s, u, m2, s2, u2);
        }
        if (lane % kGroup == 0) {
            s_group[tid / kGroup] = group;
            s_rank[tid / kGroup] = ordered(group) / kGroups * kGroups + tid / kGroup;
        }
        if (lane == 0) s_m[warp] = m, s_s[warp] = s, s_u[warp] = u;
        __syncthreads();
        m = s_m[lane % W], s = s_s[lane % W], u = s_u[lane % W];
        most = fmaxf(s_group[lane], s_group[lane + 32]);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
#pragma unroll
        for (int off = 1; off < W; off <<= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off),
                        u2 = __shfl_xor_sync(0xffffffffu, u, off);
            join(m, s, u, m2, s2, u2);
        }
    };
    join_threads();
    above = __reduce_add_sync(0xffffffffu, lane < W ? s_above[lane] : 0);
    float bottom = Range<T>::floor;   // maxima not above it are of masked logits
    if (!(most > Range<T>::floor && most < Range<T>::ceil)) {
        bottom = -INFINITY;
        r = Running();
        bool any = false;
        auto again = [&](float f) {
            if (f > -INFINITY) {
                r.add_one(f);
                any = true;
            }
        };
        float best = -INFINITY;
#pragma unroll 1
        for (int span = 0; span < kSpans; ++span) {   // the thread's own vectors, as before
            r.top = -INFINITY;
#pragma unroll 1
            for (int k = span * per; k < (span + 1) * per && tid + k * kThreads < nvec; ++k)
#pragma unroll 1
                for (int e = 0; e < N; ++e) again(paged::to_float<T>(x[vlo + (tid + k * kThreads) * N + e]));
            s_span[span][tid] = r.top;
            best = fmaxf(best, r.top);
        }
        r.top = best;
        if (tid < nsingle) again(paged::to_float<T>(x[single]));
        if (!any) r.top = -INFINITY;
        __syncthreads();   // everyone has read the first sums
        join_threads();
    }

    const int top = p.top;
    if (top > 0) {
        // the top-th largest of the groups' maxima, without their last bits,
        // which tell equals apart: a warp ranks 16 of them, two lanes each
        {
            const unsigned own = s_rank[warp * 16 + lane % 16];
            const uint4* others = reinterpret_cast<const uint4*>(s_rank) + lane / 16 * (kGroups / 8);
            int better = 0;
#pragma unroll 2
            for (int j = 0; j < kGroups / 8; ++j) {
                const uint4 o = others[j];
                better += (o.x > own) + (o.y > own) + (o.z > own) + (o.w > own);
            }
            better += __shfl_xor_sync(0xffffffffu, better, 16);
            if (better == top - 1 && lane < 16) {
                const float b = ordered_value(own / kGroups * kGroups);
                s_bound = b > bottom ? b : -INFINITY;
            }
        }
        __syncthreads();
        const float bound = s_bound;
        for (int span = 0; span < kSpans; ++span) {
            const float t = s_span[span][tid];
            if (bound > -INFINITY ? t >= bound : t > -INFINITY) s_hit[atomicAdd(&s_hits, 1)] = span * kThreads + tid;
        }
        __syncthreads();
        // the hit spans' vectors, shared out over the block
        const int hits = s_hits;
        auto keep = [&](float f, int idx) {
            if (f >= bound && f > -INFINITY) {
                const int c = atomicAdd(&s_count, 1);
                if (c < kCand / 2) s_key[c] = make_key(f, unsigned(idx));
            }
        };
        for (int k = tid; k < hits * per; k += kThreads) {
            const int h = k / per, hit = s_hit[h];
            const int at = hit % kThreads + (hit / kThreads * per + k - h * per) * kThreads;
            if (at >= nvec) continue;
            float f[N];
            Vec<T>(v[at]).get(f);
#pragma unroll
            for (int e = 0; e < N; ++e) keep(f[e], vlo + at * N + e);
        }
        if (tid < nsingle) keep(paged::to_float<T>(x[single]), single);
        __syncthreads();
        if (s_count <= kCand / 2) {
            best_keys(s_key, s_count, top, s_best, s_word);
        } else {
            pick_keys(top, s_best, s_word, [&](auto take) {
                for (int e = lo + tid; e < hi; e += kThreads) {
                    const float f = paged::to_float<T>(x[e]);
                    if (f > -INFINITY) take(make_key(f, unsigned(e)));
                }
            });
        }
    }

    if (p.parts > 1) {
        const int at = row * p.parts + part;
        if (tid < top) p.ws_keys[at * top + tid] = s_best[tid];
        if (tid == 0) {
            p.ws_sums[at] = make_float4(m, s, u, __int_as_float(above));
            s_count = 0;
        }
        __threadfence();
        __syncthreads();
        if (tid == 0) s_last = atomicAdd(p.tickets + row, 1u) == unsigned(p.parts - 1);
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        if (tid == 0) p.tickets[row] = 0;   // ready for the next call
        const int first = row * p.parts;
        for (int k = tid; k < p.parts * top; k += kThreads) s_key[k] = __ldcg(p.ws_keys + first * top + k);
        // a part a lane, in every warp
        const float4 w = lane < p.parts ? __ldcg(p.ws_sums + first + lane) : make_float4(-3.402823466e38f, 0.f, 0.f, 0.f);
        m = w.x, s = w.y, u = w.z;
        above = __reduce_add_sync(0xffffffffu, __float_as_int(w.w));
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off),
                        u2 = __shfl_xor_sync(0xffffffffu, u, off);
            join(m, s, u, m2, s2, u2);
        }
        if (top > 0) {
            __syncthreads();
            // a lower bound of the top-th key: the top-th of the parts' best
            // ones, or, of fewer parts, the least of the parts' j-th ones,
            // j x parts >= top; absent keys are 0
            unsigned long long bound = 0;
            if (p.parts >= top) {
                const unsigned long long own = lane < p.parts ? s_key[lane * top] : 0;
                int better = 0;
                for (int j = 0; j < p.parts; ++j) {
                    const unsigned long long o = s_key[j * top];
                    better += o > own || (o == own && j < lane);
                }
                bound = __shfl_sync(0xffffffffu, own, __ffs(__ballot_sync(0xffffffffu, lane < p.parts && better == top - 1)) - 1);
            } else {
                bound = lane < p.parts ? s_key[lane * top + (top - 1) / p.parts] : ~0ull;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const unsigned long long o = __shfl_xor_sync(0xffffffffu, bound, off);
                    if (o < bound) bound = o;
                }
            }
            unsigned long long* kept = s_key + kMaxParts * kMaxTop;
            for (int k = tid; k < p.parts * top; k += kThreads)
                if (s_key[k] != 0 && s_key[k] >= bound) kept[atomicAdd(&s_count, 1)] = s_key[k];
            __syncthreads();
            best_keys(kept, s_count, top, s_best, s_word);
        }
    }

    const bool infinite = m == INFINITY;   // a row with +inf has no finite log probabilities
    const bool empty = s == 0.f && !infinite;
    const float ls = kLn2 * log2f(s);
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
