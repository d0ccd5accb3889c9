// fa_paged_tc.cuh — attention of a chunk of new tokens over a paged cache on
// the 5th-generation tensor cores (the formulas are fa_paged.cuh's).
//
// A CTA walks its share of units (paged.cuh): 256 query rows x 128 keys, the
// rows of a kv head being (token, query head of its group) pairs, so a K/V
// tile serves every query head that reads it.  The 256 rows are two tiles of
// 128, one thread per row in two softmax warpgroups that take turns: while one
// works on its scores, the tensor cores multiply for the other.
//
//   warps 0-3, 4-7  softmax of row tiles 0 and 1 (thread = row = tensor-memory
//                   lane): the query rows into shared memory; per key tile the
//                   128 scores of the row from tensor memory into registers,
//                   running maximum and sum in FP32, the probabilities rounded
//                   to the cache's 16-bit type into tensor memory, in the
//                   scores' place; at the end the accumulator, normalised
//   warp 8          one lane issues every tcgen05.mma: S = Q K^T (both from
//                   shared memory, K-major, 128-byte swizzle) and O += P V (P
//                   from tensor memory, V as it lies, N-major), M = 128 rows
//   warp 9          TMA: K and V tiles into a ring, one box per page or the
//                   largest power of two of rows that divides a page (so pages
//                   of any multiple of 8 tokens may end inside a tile)
//
// The accumulator is rescaled only when a row's maximum has risen by more
// than 2^8 since the reference it uses (the probabilities then stay below 2^8,
// exact in scale in either 16-bit type); the row's thread does it in place,
// between the product that the scores' arrival proves finished and the next.
// Rows of V behind the last visible key are zeroed in shared memory before
// their product, so what a page holds there reaches nothing.
//
// Tensor work bounds it: 4 x 128 x 128 x D MACs a unit.  One exponential per
// score on the special-function units takes as many cycles as the products.
// Every wait is bounded; a role that gives up raises the device flag and the
// CTA's abort word, the others see it and leave.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "fa_paged.cuh"

namespace p100b {
namespace fatc {

using paged::Desc;
using paged::Item;
using paged::Lengths;

constexpr int kRows = 256, kKeys = 128;
constexpr int kThreads = 320;
constexpr int kMmaWarp = 8, kLoadWarp = 9;
constexpr int kSub = 128 * 128;           // bytes of 128 rows x 64 values
constexpr float kRise = 8.0f;             // log2 of the rise that forces a rescale

template <int D>
__host__ __device__ constexpr int slots() { return D == 128 ? 4 : 6; }
template <int D>
__host__ __device__ constexpr int tile_bytes() { return kSub * (D / 64); }

struct Params {
    Desc d;
    const void* q;
    void* o;
    int o_f32;
    float* lse;
    float* ws_o;        // [CTAs][2][2 row tiles][D / 4][128] float4
    float* ws_ml;       // [CTAs][2][2][128] float2
    unsigned* tickets;  // [CTAs][2]
    float scale, softcap;
    int box;            // rows of a TMA box
};

struct Barriers {
    uint64_t full[6], empty[6], q_full[2], s_full[2], p_full[2], joined[2], drain;
    uint32_t tmem;
    int abort;
    int last[2];
};

template <int D>
constexpr size_t smem_bytes() {
    return 1024 + 2 * tile_bytes<D>() + slots<D>() * tile_bytes<D>() + sizeof(Lengths) + sizeof(Barriers) + 64;
}

// ------------------------------------------------------------ tcgen05
// Descriptor of an operand in shared memory with the 128-byte swizzle: atoms
// of 8 rows x 128 bytes, `sbo` bytes between atoms along the rows, `lbo`
// between 64-value columns of an N-major operand (unused for K-major ones).
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return uint64_t((saddr >> 4) & 0x3fffu) | uint64_t((lbo >> 4) & 0x3fffu) << 16 |
           uint64_t((sbo >> 4) & 0x3fffu) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// kind::f16 with FP32 accumulation, M = 128.
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n, bool b_n_major) {
    const uint32_t t = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (uint32_t(b_n_major) << 16) | (uint32_t(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void ld32(uint32_t a, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void st32(uint32_t a, const float* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
        "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
        "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]),
        "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]),
        "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31])
        : "memory");
}
__device__ __forceinline__ void st16(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Waits for a barrier phase, for at most kWaitLimitNs or until the CTA aborts.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int* abort) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long start = globaltimer_ns();
    for (;;) {
        for (int i = 0; i < 32; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (*reinterpret_cast<volatile int*>(abort)) return false;
        if (globaltimer_ns() - start > kWaitLimitNs) {
            atomicExch(&g_device_error, kDevErrTimeout);
            atomicExch(abort, 1);
            return false;
        }
    }
}
// The same for a whole warp: every lane gets the same answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* abort) {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, abort));
}

// ------------------------------------------------------------ roles
// K and V tiles of the CTA's items into the ring, in the order the products
// take them.
template <int D>
__device__ __forceinline__ void load_role(const Params& p, const CUtensorMap* tmk, const CUtensorMap* tmv, Lengths& len,
                                          Barriers& bars, uint8_t* ring, paged::Share<kRows, kKeys> share) {
    constexpr int NS = slots<D>();
    const Desc& d = p.d;
    const int lane = threadIdx.x & 31;
    const int boxes = kKeys / p.box;                 // of a tile, at most 16
    const int i = lane & (boxes - 1), half = lane / boxes;
    const bool mine = half < D / 64;
    const uint32_t at = uint32_t(half) * kSub + uint32_t(i) * p.box * 128;
    unsigned used = 0;                               // slots filled so far
    bool ok = true;
    Item it;
    while (ok && share.next(d, len, it)) {
        const int q0 = len.q0[it.seq];
        const int end = paged::key_end<kRows, kKeys>(d, len.q0[it.seq + 1] - q0, len.kv[it.seq], it.tile);
        const int* table = d.block_table + (long long)it.seq * d.max_pages;
        auto find = [&](int t, int& page, int& off) {
            const int key = (it.key_tile + t) * kKeys + i * p.box;
            page = -1;
            off = 0;
            if (mine && t < it.count && key < end) {
                const int n = key / d.page_size;
                off = key - n * d.page_size;
                page = table[n];
                if (page < 0 || page >= d.n_pages) {
                    paged::flag_input();
                    page = -1;
                }
            }
        };
        int page, off;
        find(0, page, off);
        for (int t = 0; ok && t < it.count; ++t) {
            int next_page, next_off;
            find(t + 1, next_page, next_off);
            const uint32_t bytes = uint32_t(__popc(__ballot_sync(0xffffffffu, page >= 0))) * p.box * 128;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const int slot = used % NS;
                if (used >= NS) ok = warp_wait(&bars.empty[slot], (used / NS - 1) & 1, &bars.abort);
                if (!ok) break;
                if (lane == 0) {
                    if (bytes) mbar_arrive_expect_tx(&bars.full[slot], bytes);
                    else mbar_arrive(&bars.full[slot]);
                }
                __syncwarp();
                if (page >= 0)
                    asm volatile(
                        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(ring) + uint32_t(slot) * tile_bytes<D>() + at),
                        "l"(kv ? tmv : tmk), "r"(half * 64), "r"(off), "r"(it.head), "r"(page), "r"(smem_addr(&bars.full[slot]))
                        : "memory");
                ++used;
            }
            page = next_page;
            off = next_off;
        }
    }
    if (!ok)   // leave only when the copies in flight have landed
        for (unsigned u = used > NS ? used - NS : 0; u < used; ++u) mbar_wait(&bars.full[u % NS], (u / NS) & 1);
}

template <typename T, int D>
__device__ __forceinline__ bool mma_role(const Params& p, Lengths& len, Barriers& bars, uint32_t q_smem, uint32_t ring,
                                         uint32_t tmem, paged::Share<kRows, kKeys> share) {
    constexpr int NS = slots<D>();
    constexpr uint32_t kIdescS = idesc_f16<T>(kKeys, false), kIdescO = idesc_f16<T>(D, true);
    const int lane = threadIdx.x & 31;
    unsigned used = 0;                 // K and V tiles taken so far
    unsigned items[2] = {0, 0}, tiles[2] = {0, 0};
    Item it;
    auto qk = [&](int w, int slot) {   // S_w = Q_w K^T
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = uint32_t(k >> 2) * kSub + uint32_t(k & 3) * 32;
            mma_ss(tmem + w * 128, sw128_desc(q_smem + w * tile_bytes<D>() + off, 16, 1024),
                   sw128_desc(ring + slot * tile_bytes<D>() + off, 16, 1024), kIdescS, k > 0);
        }
    };
    auto pv = [&](int w, int slot, bool add) {   // O_w += P_w V
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
            mma_ts(tmem + 256 + w * D, tmem + w * 128 + k * 8,
                   sw128_desc(ring + slot * tile_bytes<D>() + uint32_t(k) * 2048, kSub, 1024), kIdescO, add || k > 0);
    };
    while (share.next(p.d, len, it)) {
        const int n = len.q0[it.seq + 1] - len.q0[it.seq];
        const int groups = n * p.d.group - it.tile * kRows > 128 ? 2 : 1;
        for (int w = 0; w < groups; ++w)
            if (!warp_wait(&bars.q_full[w], items[w]++ & 1, &bars.abort)) return false;
        if (!warp_wait(&bars.full[used % NS], (used / NS) & 1, &bars.abort)) return false;
        fence_after();
        if (lane == 0) {
            for (int w = 0; w < groups; ++w) {
                qk(w, used % NS);
                mma_commit(&bars.s_full[w]);
            }
            mma_commit(&bars.empty[used % NS]);
        }
        ++used;
        for (int t = 0; t < it.count; ++t) {
            const unsigned v = used, k = used + 1;
            const bool more = t + 1 < it.count;
            if (!warp_wait(&bars.full[v % NS], (v / NS) & 1, &bars.abort)) return false;
            for (int w = 0; w < groups; ++w) {
                if (!warp_wait(&bars.p_full[w], tiles[w]++ & 1, &bars.abort)) return false;
                if (more && w == 0 && !warp_wait(&bars.full[k % NS], (k / NS) & 1, &bars.abort)) return false;
                fence_after();
                if (lane == 0) {
                    pv(w, v % NS, t > 0);
                    if (w + 1 == groups) mma_commit(&bars.empty[v % NS]);
                    if (more) {
                        qk(w, k % NS);
                        if (w + 1 == groups) mma_commit(&bars.empty[k % NS]);
                    }
                    mma_commit(&bars.s_full[w]);
                }
            }
            used += more ? 2 : 1;
        }
    }
    return true;
}

template <typename T, int D, bool CAP>
__device__ __forceinline__ void softmax_role(const Params& p, Lengths& len, Barriers& bars, uint8_t* q_smem, uint8_t* ring,
                                             uint32_t tmem, int parts, paged::Share<kRows, kKeys> share) {
    constexpr int NS = slots<D>();
    constexpr float kLog2e = 1.4426950408889634f;
    const Desc& d = p.d;
    const int w = threadIdx.x >> 7, row = threadIdx.x & 127;
    const uint32_t lanes = uint32_t(row & ~31) << 16;
    const uint32_t t_s = tmem + w * 128 + lanes, t_o = tmem + 256 + w * D + lanes;
    // scores in units of log2 e; a negative scale turns the queries' sign
    const float c = CAP ? 1.0f : fabsf(p.scale) * kLog2e;
    const float cap_in = CAP ? 2.f * fabsf(p.scale) * kLog2e / p.softcap : 0.f, cap = p.softcap * kLog2e;
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    unsigned done = 0, used = 0;   // phases of s_full passed; key tiles of the CTA before this item
    Item it;
    while (share.next(d, len, it)) {
        const int q0 = len.q0[it.seq], n = len.q0[it.seq + 1] - q0, kv = len.kv[it.seq];
        const int first_row = it.tile * kRows + w * 128;
        const int rows = min(128, n * d.group - first_row);
        const unsigned tile0 = used;
        used += it.count;
        if (rows <= 0) continue;
        const int r = first_row + row;
        const int tok = r / d.group, g = r - tok * d.group;
        const bool live = row < rows;
        const int limit = !live ? 0 : d.causal ? max(0, min(kv, kv - n + tok + 1)) : kv;
        const int end = paged::key_end<kRows, kKeys>(d, n, kv, it.tile);
        {
            const T* src = static_cast<const T*>(p.q) + (long long)(q0 + tok) * d.q_stride + (long long)(it.head * d.group + g) * D;
            uint8_t* dst = q_smem + w * tile_bytes<D>() + row * 128;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                uint4 v = live ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
                v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
                *reinterpret_cast<uint4*>(dst + (i >> 3) * kSub + (((i & 7) ^ (row & 7)) << 4)) = v;
            }
            fence_async();
            fence_before();
            mbar_arrive(&bars.q_full[w]);
        }
        float m = -INFINITY, l = 0.f;
        for (int t = 0; t < it.count; ++t) {
            if (!warp_wait(&bars.s_full[w], done++ & 1, &bars.abort)) return;
            fence_after();
            float s[128];
#pragma unroll
            for (int i = 0; i < 4; ++i) ld32(t_s + i * 32, s + i * 32);
            wait_ld();
            const int key0 = (it.key_tile + t) * kKeys;
            if (CAP) {
#pragma unroll
                for (int i = 0; i < 128; ++i) s[i] = fap::cap_score(s[i], cap_in, cap);
            }
            if (__any_sync(0xffffffffu, limit < key0 + kKeys)) {
                const int lim = limit - key0;
#pragma unroll
                for (int i = 0; i < 128; ++i) s[i] = i < lim ? s[i] : -INFINITY;
            }
            float mx4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < 128; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], s[i]);
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            if (t == 0) {
                m = mx;
            } else {
                const bool rise = (mx - m) * c > kRise;
                if (__any_sync(0xffffffffu, rise)) {
                    const float a = rise ? paged::exp2_approx((m - mx) * c) : 1.f;
                    if (rise) m = mx;
                    l *= a;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        float o[32];
                        ld32(t_o + i * 32, o);
                        wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] *= a;
                        st32(t_o + i * 32, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.f : m * c;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t pk[16];
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float a = paged::exp2_approx(fmaf(s[i * 32 + j], c, -base));
                    const float b = paged::exp2_approx(fmaf(s[i * 32 + j + 1], c, -base));
                    sum[(j >> 1) & 1] += a;
                    sum[2 + ((j >> 1) & 1)] += b;
                    pk[j >> 1] = paged::pack2<T>(a, b);
                }
                st16(t_s + i * 16, pk);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (w == 0 && key0 + kKeys > end) {   // rows of V that no key of the tile's rows reaches
                const unsigned u = 2 * (tile0 + t) + 1;
                if (!warp_wait(&bars.full[u % NS], (u / NS) & 1, &bars.abort)) return;
                if (key0 + row >= end) {
                    uint8_t* v = ring + (u % NS) * tile_bytes<D>() + row * 128;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i)
                        *reinterpret_cast<uint4*>(v + (i >> 3) * kSub + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async();
            }
            wait_st();
            fence_before();
            mbar_arrive(&bars.p_full[w]);
        }
        if (!warp_wait(&bars.s_full[w], done++ & 1, &bars.abort)) return;   // the accumulator is complete
        fence_after();
        const float base = m == -INFINITY ? -INFINITY : m * c;
        const long long o_at = (long long)(q0 + tok) * d.o_stride + (long long)(it.head * d.group + g) * D;
        auto write = [&](int i, float (&o)[32], float inv) {   // columns 32 i .. 32 i + 31 of the row
            if (!live) return;
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] *= inv;
            if (p.o_f32) {
                float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.o) + o_at + i * 32);
#pragma unroll
                for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            } else {
                uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + o_at + i * 32);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    dst[j] = make_uint4(paged::pack2<T>(o[8 * j], o[8 * j + 1]), paged::pack2<T>(o[8 * j + 2], o[8 * j + 3]),
                                        paged::pack2<T>(o[8 * j + 4], o[8 * j + 5]), paged::pack2<T>(o[8 * j + 6], o[8 * j + 7]));
            }
        };
        auto write_lse = [&](float top, float total) {
            if (live && p.lse)
                p.lse[(long long)(q0 + tok) * d.n_head_q + it.head * d.group + g] =
                    total == 0.f ? -INFINITY : (top + log2f(total)) / kLog2e;
        };
        if (it.count == it.units) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                float o[32];
                ld32(t_o + i * 32, o);
                wait_ld();
                write(i, o, inv);
            }
            write_lse(base, l);
        } else {
            const long long slot = (long long)(blockIdx.x * 2 + (it.key_tile == 0)) * 2 + w;
            float4* dst = reinterpret_cast<float4*>(p.ws_o) + slot * (D / 4) * 128 + row;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                float o[32];
                ld32(t_o + i * 32, o);
                wait_ld();
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    __stcg(dst + (i * 8 + j) * 128, make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]));
            }
            __stcg(reinterpret_cast<float2*>(p.ws_ml) + slot * 128 + row, make_float2(base, l));
            const int c0 = paged::share_of(it.tile_first, len.total, parts);
            const int c1 = paged::share_of(it.tile_first + it.units - 1, len.total, parts);
            // one thread of the warpgroup takes the ticket when all have written
            __threadfence();
            mbar_arrive(&bars.joined[w]);
            if (!warp_wait(&bars.joined[w], 0, &bars.abort)) return;
            if (row == 0) bars.last[w] = atomicAdd(p.tickets + c0 * 2 + w, 1u) == unsigned(c1 - c0);
            mbar_arrive(&bars.joined[w]);
            if (!warp_wait(&bars.joined[w], 1, &bars.abort)) return;
            if (bars.last[w]) {   // join the parts in share order
                __threadfence();
                if (row == 0) p.tickets[c0 * 2 + w] = 0;   // ready for the next call
                const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + w * 128 + row;
                const float4* po = reinterpret_cast<const float4*>(p.ws_o) + (long long)w * (D / 4) * 128 + row;
                auto part = [&](int q) { return ((long long)q * 2 + (q == c0)) * 2; };
                float top = -INFINITY;
                for (int q = c0; q <= c1; ++q) top = fmaxf(top, __ldcg(ml + part(q) * 128).x);
                const float safe = top == -INFINITY ? 0.f : top;
                float total = 0.f;
                for (int q = c0; q <= c1; ++q) {
                    const float2 v = __ldcg(ml + part(q) * 128);
                    total = fmaf(paged::exp2_approx(v.x - safe), v.y, total);
                }
                const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll 1
                for (int i = 0; i < D / 32; ++i) {
                    float o[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0.f;
                    for (int q = c0; q <= c1; ++q) {
                        const float f = paged::exp2_approx(__ldcg(ml + part(q) * 128).x - safe);
                        float4 v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = __ldcg(po + (part(q) * (D / 4) + i * 8 + j) * 128);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            o[4 * j] = fmaf(f, v[j].x, o[4 * j]);
                            o[4 * j + 1] = fmaf(f, v[j].y, o[4 * j + 1]);
                            o[4 * j + 2] = fmaf(f, v[j].z, o[4 * j + 2]);
                            o[4 * j + 3] = fmaf(f, v[j].w, o[4 * j + 3]);
                        }
                    }
                    write(i, o, inv);
                }
                write_lse(top, total);
            }
        }
    }
}

template <typename T, int D, bool CAP>
__global__ void __launch_bounds__(kThreads, 1)
    fa_paged_tc_kernel(const Params p, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_smem = smem;
    uint8_t* ring = q_smem + 2 * tile_bytes<D>();
    Lengths& len = *reinterpret_cast<Lengths*>(ring + slots<D>() * tile_bytes<D>());
    Barriers& bars = *reinterpret_cast<Barriers*>(
        (reinterpret_cast<uintptr_t>(&len) + sizeof(Lengths) + 15) & ~uintptr_t(15));
    const int warp = threadIdx.x >> 5;

    if (threadIdx.x == kLoadWarp * 32) {
        prefetch_tensormap(&tmk);
        prefetch_tensormap(&tmv);
    }
    paged::read_lengths<kRows, kKeys, kThreads>(p.d, len);
    const int parts = len.ok ? int(min((long long)gridDim.x, len.total)) : 0;
    if (int(blockIdx.x) >= parts) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 6; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], 1);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(&bars.q_full[w], 128);
            mbar_init(&bars.s_full[w], 1);
            mbar_init(&bars.p_full[w], 128);
            mbar_init(&bars.joined[w], 128);
        }
        mbar_init(&bars.drain, 1);
        bars.abort = 0;
        fence_barrier_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&bars.tmem)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem);
    paged::Share<kRows, kKeys> share;
    share.begin(p.d, len, blockIdx.x, parts);

    if (warp == kLoadWarp)
        load_role<D>(p, &tmk, &tmv, len, bars, ring, share);
    else if (warp == kMmaWarp) {
        if (!mma_role<T, D>(p, len, bars, smem_addr(q_smem), smem_addr(ring), tmem, share)) {
            // leave only when the products in flight are done
            if ((threadIdx.x & 31) == 0) mma_commit(&bars.drain);
            __syncwarp();
            mbar_wait(&bars.drain, 0);
        }
    } else
        softmax_role<T, D, CAP>(p, len, bars, q_smem, ring, tmem, parts, share);

    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

}  // namespace fatc
}  // namespace p100b
