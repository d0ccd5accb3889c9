// fa_paged.cuh — attention of new tokens over a paged cache on mma.sync: the
// kernel for single tokens (16 query rows of a kv head or fewer).
//
//   s_ij = scale q_i k_j  (then cap tanh(s / cap)),  j < limit_i
//   o_i = sum_j e^(s_ij - m_i) v_j / sum_j e^(s_ij - m_i),  lse_i = m_i + ln sum
//
// A CTA walks its share of units (paged.cuh): 16 rows x 64 keys.  The four
// warps of a CTA split every key tile, 16 keys each, with a running maximum,
// sum and 16 x D accumulator of their own in registers, joined once per item:
// no exchange per tile.  K and V rows are gathered by 16-byte asynchronous
// copies (any page size; a row's page is looked up two tiles ahead), swizzled
// so that ldmatrix reads without bank conflicts; rows behind kv_len are filled
// with zeros, so what a page holds there never reaches a product.  Statistics
// and accumulators are FP32.
//
// The tensor cores take 16-bit probabilities.  Each goes in two parts, rounded
// to nearest: the probability and what that rounding left of it, so a product
// loses 2^-16 (bfloat16) or 2^-22 of it and an FP32 output has the digits of
// FP32 probabilities.  Where a kv head has 8 rows or fewer (SPARE) the second
// parts are the upper 8 rows of the same products and are added to the lower
// ones at the end, at no cost (64 sequences up to 8192 tokens: 0.997 of the time
// with one part); else they take products of their own (1.03 of it with 16
// rows).  In FP16 the largest probability is 2^15, see kLift.
//
// HBM bytes bound it: K and V are read once per row tile.  A row tile cut by
// the shares leaves its partials {m, l, unnormalised o} in the workspace and
// its last CTA (an atomic ticket, no waiting) joins them in share order; more
// than kDirect parts are joined in groups first, each by its last CTA, so that
// no CTA reads more than about the square root of their number.  Measured: 64
// sequences up to 8192 tokens (64 / 8 heads of 128) 190 us in graph replays, 0.98
// of measured bandwidth (293 us with one CTA an SM); one of 4096 tokens (32 / 8
// heads) 14 us, of which the copies take 2.
#pragma once
#include <type_traits>

#include "paged.cuh"

namespace p100b {
namespace fap {

using paged::Desc;
using paged::Item;
using paged::Lengths;

constexpr int kThreads = 128;
constexpr int kRows = 16, kKeys = 64;
constexpr int kOver = 1;   // what a row tile costs beyond its keys, in units
constexpr int kStages = 3;
constexpr int kOffs = 5;   // tiles whose row offsets are held
constexpr int kDirect = 48;   // parts that one CTA joins (two levels cost 2.4 us more than one of 37 parts)
constexpr int kMaxJoin = 48;  // at most so many in one join
constexpr int kMinUnits = 2;  // of a share, where there is less work than CTAs (one of 4096: 18.4 us, with 4 or 8 20.5)

// log2 of the largest probability before the normalisation: FP16 holds nothing
// below 2^-25, and the many keys that a long context has there can weigh more
// than a rounding of the output.  The statistics m are that much below the
// maximum.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.f : 0.f;

struct Params {
    Desc d;
    const void *q, *k, *v;
    void* o;
    int o_f32;
    float* lse;        // [n_tokens][n_head_q] or null
    float* ws_o;       // [CTAs][2][kRows][D]
    float* ws_ml;      // [CTAs][2][kRows][2], m in units of log2
    unsigned* tickets; // [2][CTAs]
    float scale, softcap;
};

// Shares of a call's units on so many CTAs.  Every share has a unit, so every
// CTA between a cut tile's first and last holds a part of it.
__host__ __device__ __forceinline__ int shares(long long total, int ctas) {
    const long long most = (total + kMinUnits - 1) / kMinUnits;
    return most < ctas ? int(most) : ctas;
}

// How the parts of a row tile cut over the CTAs c0 .. c0 + np - 1 are joined: up
// to kDirect of them by the last one to finish, more in groups of `per`, each by
// its last one, and the groups by the last group's.  The parts of a group count
// on the ticket of the CTA of its first part.  No other tile counts on that word:
// a tile that is cut starts in c0, or has its first part in a CTA strictly
// between this tile's first and last one, and those hold nothing else.  Hence a
// group of one part takes no ticket: its CTA can be the tile's last, in which
// the next cut tile may start.
struct Joins {
    int np, per, groups;
    __host__ __device__ explicit Joins(int n) : np(n), per(n) {
        if (np > kDirect) {
            per = int(ceilf(sqrtf(float(np))));
            if (per > kMaxJoin) per = kMaxJoin;
        }
        groups = (np + per - 1) / per;
    }
    __host__ __device__ int first_of(int part) const { return part / per * per; }
    __host__ __device__ int size_of(int first) const { return per < np - first ? per : np - first; }
    __host__ __device__ bool counts(int first) const { return size_of(first) > 1; }
};

// Without the lengths, which lie behind.
template <int D>
constexpr size_t smem_bytes() {
    return size_t(kStages) * 2 * kKeys * D * 2 + kOffs * kKeys * sizeof(long long);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// out tanh(y), y = near x.  For |y| <= 1/2 tanh(y) / y is a polynomial of degree
// 4 in y^2, fitted to the least relative error (7e-8 with FP32's roundings), so
// that a cap far above the scores costs them nothing; beyond, 1 - 2 / (e^(2y) +
// 1) takes two approximate operations, absolute error a few 1e-7.
__device__ constexpr float kTanh[5] = {1.0f, -0.3333306908607483f, 0.13324779272079468f, -0.052986063063144684f,
                                       0.017134996131062508f};
__device__ __forceinline__ float cap_score(float x, float near, float out) {
    const float y = x * near, z = y * y;
    const float small = y * fmaf(z, fmaf(z, fmaf(z, fmaf(z, kTanh[4], kTanh[3]), kTanh[2]), kTanh[1]), kTanh[0]);
    const float large = fmaf(-2.f, paged::rcp_approx(paged::exp2_approx(y * 2.8853900817779268f) + 1.f), 1.f);
    return out * (fabsf(y) <= 0.5f ? small : large);
}
// scale / cap, finite where the cap is tiny.
__device__ __forceinline__ float cap_near(float scale, float cap) { return fmaxf(-3e38f, fminf(scale / cap, 3e38f)); }

// Row r (token r / group of the sequence, query head r % group of the kv
// head) of an item's query or output tensor, in elements.
__device__ __forceinline__ long long row_offset(const Desc& d, int q0, int head, int r, long long stride, int D) {
    const int tok = r / d.group, g = r - tok * d.group;
    return (long long)(q0 + tok) * stride + (long long)(head * d.group + g) * D;
}

// Where a finished row goes.
struct Out {
    int q0, head, row0, rows;
    template <typename T, int D>
    __device__ __forceinline__ void write4(const Params& p, int r, int c, float4 o, float sum) const {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const long long at = row_offset(p.d, q0, head, row0 + r, p.d.o_stride, D) + c;
        if (p.o_f32)
            *reinterpret_cast<float4*>(static_cast<float*>(p.o) + at) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        else
            *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + at) =
                make_uint2(paged::pack2<T>(o.x * inv, o.y * inv), paged::pack2<T>(o.z * inv, o.w * inv));
    }
    __device__ __forceinline__ void write_lse(const Params& p, int r, float m, float sum) const {
        if (!p.lse) return;
        const int tok = (row0 + r) / p.d.group;
        p.lse[(long long)(q0 + tok) * p.d.n_head_q + head * p.d.group + (row0 + r - tok * p.d.group)] =
            sum == 0.f ? -INFINITY : (m + log2f(sum)) / 1.4426950408889634f;
    }
};

// Joins the partials of parts first, first + step, ... (n <= kMaxJoin of them)
// of the row tile whose part 0 belongs to CTA c0, in that order: into the
// output, or back into the first one's place.  Every thread of the CTA calls
// it; scratch: (2 kMaxJoin + 1) x kRows floats.  Its loops stay rolled up to
// a few loads in flight: it runs once a CTA, and straight-line code costs more
// to fetch than it saves.
template <typename T, int D>
__device__ __forceinline__ void join_parts(const Params& p, const Out& out, int c0, int first, int step, int n, bool final,
                                           float* scratch) {
    constexpr int kLanes = kThreads / kRows;   // threads of a row's statistics
    const int tid = threadIdx.x;
    float* s_w = scratch;                      // [n][kRows] m, then the weight
    float* s_l = s_w + kMaxJoin * kRows;       // [n][kRows]
    float* s_sum = s_l + kMaxJoin * kRows;     // [kRows]
    auto slot = [&](int i) { return 2 * (c0 + first + i * step) + (first + i * step == 0); };
    {
        const int r = tid / kLanes, q = tid % kLanes;
        float top = -INFINITY;
#pragma unroll 2
        for (int i = q; i < n; i += kLanes) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.ws_ml) + slot(i) * kRows + r);
            s_w[i * kRows + r] = ml.x;
            s_l[i * kRows + r] = ml.y;
            top = fmaxf(top, ml.x);
        }
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll 1
        for (int i = q; i < n; i += kLanes) {
            const float w = paged::exp2_approx(s_w[i * kRows + r] - base);
            s_w[i * kRows + r] = w;
            sum = fmaf(w, s_l[i * kRows + r], sum);
        }
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (q == 0) {
            s_sum[r] = sum;
            if (final && r < out.rows) out.write_lse(p, r, top, sum);
            if (!final) reinterpret_cast<float2*>(p.ws_ml)[slot(0) * kRows + r] = make_float2(top, sum);
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int e = tid; e < out.rows * (D / 4); e += kThreads) {
        const int r = e / (D / 4), c = (e - r * (D / 4)) * 4;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const float4 o = __ldcg(reinterpret_cast<const float4*>(p.ws_o + (slot(i) * kRows + r) * D + c));
            const float w = s_w[i * kRows + r];
            a.x = fmaf(w, o.x, a.x);
            a.y = fmaf(w, o.y, a.y);
            a.z = fmaf(w, o.z, a.z);
            a.w = fmaf(w, o.w, a.w);
        }
        if (final) out.write4<T, D>(p, r, c, a, s_sum[r]);
        else *reinterpret_cast<float4*>(p.ws_o + (slot(0) * kRows + r) * D + c) = a;
    }
}

template <typename T, int D, bool SPARE>
__global__ void __launch_bounds__(kThreads, 2) fa_paged_kernel(const Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kRowBytes = D * 2;
    constexpr int kTileBytes = kKeys * kRowBytes;
    constexpr int kChunks = D / 8;            // 16-byte chunks of a row
    constexpr float kLog2e = 1.4426950408889634f;
    uint8_t* s_kv = smem;
    long long* s_off = reinterpret_cast<long long*>(s_kv + size_t(kStages) * 2 * kTileBytes);   // [kOffs][kKeys]
    const Lengths len(s_off + kOffs * kKeys, p.d.n_seq);
    __shared__ int s_last;
    const Desc& d = p.d;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    paged::read_lengths<kRows, kKeys, kOver, kThreads, false>(d, len, 0);
    if (!len.head->ok) return;
    const int parts = shares(len.head->total, int(gridDim.x));
    if (int(blockIdx.x) >= parts) return;
    paged::Share<kRows, kKeys, kOver> share;
    share.begin(d, len, blockIdx.x, parts);
    Item it;
    const float to_log2 = p.scale * kLog2e;
    const float cap_in = p.softcap != 0.f ? cap_near(p.scale, p.softcap) : 0.f;

    while (share.next(d, len, it)) {
        const int q0 = len.q0[it.seq], n = it.n, kv = it.kv;
        const int rows = min(kRows, n * d.group - it.tile * kRows);
        const int row0 = it.tile * kRows;
        const int end = paged::key_end<kRows>(d, n, kv, it.tile);   // keys any row sees
        const int* table = d.block_table + (long long)it.seq * d.max_pages;
        const long long head_off = it.head * d.head_stride;

        // The element offset of key row `key`, or -1 where it is not read.
        auto find = [&](int key) -> long long {
            if (key >= end) return -1;
            const int at = key / d.page_size;
            const int page = table[at];
            if (page < 0 || page >= d.n_pages) {
                paged::flag_input();
                return -1;
            }
            return page * d.page_stride + head_off + (long long)(key - at * d.page_size) * d.token_stride;
        };
        // Copies of tile t (counted from the item's first) into its stage.
        auto issue = [&](int t) {
            if (t < it.count) {
                const long long* off = s_off + (t % kOffs) * kKeys;
                uint8_t* ks = s_kv + size_t(t % kStages) * 2 * kTileBytes;
                const int c = tid % kChunks;
#pragma unroll
                for (int r = tid / kChunks; r < kKeys; r += kThreads / kChunks) {
                    const long long o = off[r];
                    const uint32_t dst = smem_addr(ks) + r * kRowBytes + ((c ^ (r & 7)) << 4);
                    const long long from = (o < 0 ? 0 : o) + c * 8;
                    cp_async16(dst, static_cast<const T*>(p.k) + from, o >= 0);
                    cp_async16(dst + kTileBytes, static_cast<const T*>(p.v) + from, o >= 0);
                }
            }
            cp_commit();
        };

        // Offsets of the first kOffs - 1 tiles, the first copies.
        for (int i = tid; i < (kOffs - 1) * kKeys; i += kThreads)
            s_off[i] = i / kKeys < it.count ? find((it.key_tile + i / kKeys) * kKeys + i % kKeys) : -1;
        __syncthreads();
        for (int t = 0; t < kStages - 1; ++t) issue(t);

        // Query fragments: rows g and g + 8 of the tile (zero past the rows).
        const int g = lane >> 2, cq = (lane & 3) * 2;
        uint32_t qf[D / 16][4];
        {
            const T* qa = nullptr;
            const T* qb = nullptr;
            if (g < rows) qa = static_cast<const T*>(p.q) + row_offset(d, q0, it.head, row0 + g, d.q_stride, D);
            if (g + 8 < rows) qb = static_cast<const T*>(p.q) + row_offset(d, q0, it.head, row0 + g + 8, d.q_stride, D);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qf[k][0] = qa ? *reinterpret_cast<const uint32_t*>(qa + k * 16 + cq) : 0u;
                qf[k][1] = qb ? *reinterpret_cast<const uint32_t*>(qb + k * 16 + cq) : 0u;
                qf[k][2] = qa ? *reinterpret_cast<const uint32_t*>(qa + k * 16 + cq + 8) : 0u;
                qf[k][3] = qb ? *reinterpret_cast<const uint32_t*>(qb + k * 16 + cq + 8) : 0u;
            }
        }
        // Keys [0, limit) of rows g and g + 8.
        int limit[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h;
            limit[h] = r >= rows ? 0 : d.causal ? min(kv, kv - n + (row0 + r) / d.group + 1) : kv;
        }
        float acc[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        for (int t = 0; t < it.count; ++t) {
            cp_wait<kStages - 2>();
            __syncthreads();   // tile t has landed; everyone is done with tile t - 1
            long long next_off = -1;
            const int ahead = t + kOffs - 1;
            if (tid < kKeys && ahead < it.count) next_off = find((it.key_tile + ahead) * kKeys + tid);
            issue(t + kStages - 1);
            const uint32_t ks = smem_addr(s_kv) + (t % kStages) * 2 * kTileBytes;
            const uint32_t vs = ks + kTileBytes;
            float s[2][4] = {};
            {
                // matrices 0/1: keys 0-7, low and high half of the 16 dims; 2/3: keys 8-15
                const int key = warp * 16 + (lane & 7) + ((lane >> 4) << 3);
                const uint32_t row = ks + key * kRowBytes;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t b[4];
                    ldsm4(row + (((2 * k + ((lane >> 3) & 1)) ^ (key & 7)) << 4), b);
                    mma16<T>(s[0], qf[k], b[0], b[1]);
                    mma16<T>(s[1], qf[k], b[2], b[3]);
                }
            }
            const int key0 = (it.key_tile + t) * kKeys + warp * 16 + cq;   // this lane's first column
            // Row g + 8 h: its probabilities, rounded (high, of both blocks of 8
            // keys) and what the rounding left (rest); the factor of its sums so far.
            auto softmax = [&](int h, uint32_t (&high)[2], uint32_t (&rest)[2]) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 2 * h; e < 2 * h + 2; ++e) {
                        float x = p.softcap != 0.f ? cap_score(s[j][e], cap_in, p.softcap * kLog2e) : s[j][e] * to_log2;
                        s[j][e] = key0 + j * 8 + (e & 1) < limit[h] ? x : -INFINITY;
                    }
                float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[h], mx - kLift<T>);
                const float base = mn == -INFINITY ? 0.f : mn;
                const float a = paged::exp2_approx(m[h] - base);
                m[h] = mn;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float p0 = paged::exp2_approx(s[j][2 * h] - base), p1 = paged::exp2_approx(s[j][2 * h + 1] - base);
                    sum += p0;
                    sum += p1;
                    float h0, h1;
                    high[j] = paged::pack2<T>(p0, p1);
                    paged::unpack2<T>(high[j], h0, h1);
                    rest[j] = paged::pack2<T>(p0 - h0, p1 - h1);
                }
                l[h] = l[h] * a + sum;
                return a;
            };
            uint32_t pf[4], pr[4];   // probabilities of rows g and g + 8, what their rounding left
            float a[2];
            {
                uint32_t high[2], rest[2];
                a[0] = a[1] = softmax(0, high, rest);
                pf[0] = high[0], pf[2] = high[1];
                if (SPARE) {
                    pf[1] = rest[0], pf[3] = rest[1];
                } else {
                    pr[0] = rest[0], pr[2] = rest[1];
                    a[1] = softmax(1, high, rest);
                    pf[1] = high[0], pf[3] = high[1];
                    pr[1] = rest[0], pr[3] = rest[1];
                }
            }
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] *= a[e >> 1];
            {
                // matrices 0/1: dims 0-7 of keys 0-7 and 8-15; 2/3: dims 8-15
                const int key = warp * 16 + (lane & 7) + (((lane >> 3) & 1) << 3);
                const uint32_t row = vs + key * kRowBytes;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    uint32_t b[4];
                    ldsm4_t(row + (((2 * i + (lane >> 4)) ^ (key & 7)) << 4), b);
                    mma16<T>(acc[2 * i], pf, b[0], b[1]);
                    mma16<T>(acc[2 * i + 1], pf, b[2], b[3]);
                    if (!SPARE) {
                        mma16<T>(acc[2 * i], pr, b[0], b[1]);
                        mma16<T>(acc[2 * i + 1], pr, b[2], b[3]);
                    }
                }
            }
            if (tid < kKeys) s_off[(ahead % kOffs) * kKeys + tid] = next_off;
        }

        if (SPARE) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) acc[i][0] += acc[i][2], acc[i][1] += acc[i][3];
        }
        // Join the warps: statistics, then the accumulators added in warp order.
        cp_wait<0>();
        __syncthreads();
        float* s_m = reinterpret_cast<float*>(s_kv);          // [4][16]
        float* s_l = s_m + 4 * kRows;                         // [4][16]
        float* s_o = s_l + 4 * kRows;                         // [4][16][D + 4]
        constexpr int kLd = D + 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if ((lane & 3) == 0) {
                s_m[warp * kRows + g + 8 * h] = m[h];
                s_l[warp * kRows + g + 8 * h] = l[h];
            }
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<float2*>(s_o + (warp * kRows + g + 8 * h) * kLd + i * 8 + cq) =
                    make_float2(acc[i][2 * h], acc[i][2 * h + 1]);
        __syncthreads();
        const bool whole = it.count == it.units;
        const Out out = {q0, it.head, row0, rows};
        const int slot = blockIdx.x * 2 + (it.key_tile == 0);   // 0: a tile begun by another CTA, 1: begun here
        for (int e = tid; e < rows * (D / 4); e += kThreads) {
            const int r = e / (D / 4), c = (e - r * (D / 4)) * 4;
            float mx = s_m[r];
#pragma unroll
            for (int w = 1; w < 4; ++w) mx = fmaxf(mx, s_m[w * kRows + r]);
            const float base = mx == -INFINITY ? 0.f : mx;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = paged::exp2_approx(s_m[w * kRows + r] - base);
                const float4 o = *reinterpret_cast<const float4*>(s_o + (w * kRows + r) * kLd + c);
                a.x = fmaf(f, o.x, a.x);
                a.y = fmaf(f, o.y, a.y);
                a.z = fmaf(f, o.z, a.z);
                a.w = fmaf(f, o.w, a.w);
                sum = fmaf(f, s_l[w * kRows + r], sum);
            }
            if (whole) {
                out.write4<T, D>(p, r, c, a, sum);
                if (c == 0) out.write_lse(p, r, mx, sum);
            } else {
                *reinterpret_cast<float4*>(p.ws_o + ((long long)slot * kRows + r) * D + c) = a;
                if (c == 0)
                    *reinterpret_cast<float2*>(p.ws_ml + ((long long)slot * kRows + r) * 2) = make_float2(mx, sum);
            }
        }
        if (!whole) {
            const int c0 = paged::share_of(it.tile_first, len.head->total, parts);
            const Joins joins(paged::share_of(it.tile_first + it.units - 1, len.head->total, parts) - c0 + 1);
            const int first = joins.first_of(int(blockIdx.x) - c0), n = joins.size_of(first);
            __threadfence();
            __syncthreads();
            bool last = true;
            if (joins.counts(first)) {
                if (tid == 0) s_last = atomicAdd(p.tickets + c0 + first, 1u) == unsigned(n - 1);
                __syncthreads();
                last = s_last;
                if (last) {
                    __threadfence();
                    if (tid == 0) p.tickets[c0 + first] = 0;   // ready for the next call
                    join_parts<T, D>(p, out, c0, first, 1, n, joins.groups == 1, reinterpret_cast<float*>(s_kv));
                    __threadfence();
                }
            }
            if (last && joins.groups > 1) {
                __syncthreads();
                if (tid == 0) s_last = atomicAdd(p.tickets + gridDim.x + c0, 1u) == unsigned(joins.groups - 1);
                __syncthreads();
                if (s_last) {
                    __threadfence();
                    if (tid == 0) p.tickets[gridDim.x + c0] = 0;
                    join_parts<T, D>(p, out, c0, 0, joins.per, joins.groups, true, reinterpret_cast<float*>(s_kv));
                }
            }
        }
        __syncthreads();   // shared memory is free for the next item
    }
}

}  // namespace fap
}  // namespace p100b
