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
//                   once to the cache's 16-bit type (a second part, as in
//                   fa_paged.cuh, would be half as many products again, which
//                   bound this kernel) into tensor memory, in the scores'
//                   place; at the end the accumulator, normalised
//   warp 8          issues every tcgen05.mma: S = Q K^T (both from shared
//                   memory, K-major, 128-byte swizzle) and O += P V (P from
//                   tensor memory, V as it lies, N-major), M = 128 rows
//   warp 9          hands out the items and loads K and V tiles by TMA into a
//                   ring, one box per page or the largest power of two of rows
//                   that divides a page (so pages may end inside a tile)
//   warps 10, 11    load the tiles instead where a page is no multiple of 16
//                   tokens: rows gathered by 16-byte asynchronous copies
//
// The accumulator is rescaled only when a row's maximum has risen by more
// than 2^8 since the reference it uses (the probabilities then stay below 2^8,
// in FP16, whose reference is taken lower, below 2^15); the row's thread does it in place,
// between the product that the scores' arrival proves finished and the next.
// Rows of V behind the last visible key are zeroed in shared memory before
// their product, so what a page holds there reaches nothing.
//
// Tensor work bounds it: 4 x 128 x 128 x D MACs a unit (2048 cycles at D =
// 128).  One exponential per score on the special-function units takes as many
// cycles as the products.  Measured: 3800 cycles a unit; an 8192-token prompt
// of 32 / 8 heads of 128 in 521 us at full clock, 557 us (987 TFLOP/s) under
// the 1000 W cap; the same with two 64-key chains a row tile 581, two threads a
// row 593, two issuing warps 694, some of the exponentials by a polynomial 580
// and more.  Every wait is bounded; a role that gives up raises the device flag and the
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
using paged::add2;
using paged::fma2;
using paged::pair;
using paged::unpair;

constexpr int kRows = 256, kKeys = 128;
constexpr int kOver = 4;                  // what a row tile costs beyond its keys, in units
constexpr int kWholeFrom = 4;             // row tiles per CTA from which they are dealt out whole (1024 tiles: 557 us, cut 599)
constexpr int kThreads = 384;             // two softmax warpgroups; one of the issuing warp and the loading ones
constexpr int kMmaWarp = 8, kLoadWarp = 9, kGatherWarp = 10;
// Registers a thread after the split; 256 x 192 + 128 x 120 is what the block
// is launched with (384 x 168).
constexpr int kSoftmaxRegs = 192, kIssueRegs = 120;
static_assert(256 * kSoftmaxRegs + 128 * kIssueRegs <= kThreads * 168, "register split");
constexpr int kSub = 128 * 128;           // bytes of 128 rows x 64 values
constexpr float kRise = 8.0f;             // log2 of the rise that forces a rescale
// The reference lies that far below the maximum it was taken from, so that FP16
// probabilities stay below 2^15 and what it cannot hold of them, 2^-25, is below
// 2^-32 of the row's largest: many keys of a long context may lie there.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.f - kRise : 0.f;

template <int D>
__host__ __device__ constexpr int slots() { return D == 128 ? 4 : 8; }
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
    int box;            // rows of a TMA box, 0: gathered rows
    const void *k, *v;
};

// An item as the load warp hands it to the others, kJobs of them in a ring.
struct Job {
    int count;           // key tiles; 0: no more items
    int seq;
    int key_tile, row0;  // first key tile; first row of the row tile in its kv head
    int q0, n, kv, end, head;
    int whole;           // no other CTA has a part
    int units;           // else the key tiles of the whole row tile,
    long long first;     // and its first unit
};
constexpr int kJobs = 4;

struct Barriers {
    uint64_t full[8], empty[8], q_full[2], s_full[2], p_full[2][2], joined[2], job_full[kJobs], job_empty[kJobs], drain;
    uint32_t tmem;
    int abort;
    int last[2];
    Job jobs[kJobs];
};
using Units = paged::Share<kRows, kKeys, kOver>;

// Without the lengths.
template <int D>
constexpr size_t smem_bytes() {
    return 1024 + 2 * tile_bytes<D>() + slots<D>() * tile_bytes<D>() + sizeof(Barriers) + 64;
}

// ------------------------------------------------------------ tcgen05
// Descriptor of an operand in shared memory with the 128-byte swizzle: atoms
// of 8 rows x 128 bytes, `sbo` bytes between atoms along the rows, `lbo`
// between 64-value columns of an N-major operand (unused for K-major ones).
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return uint64_t((saddr >> 4) & 0x3fffu) | uint64_t((lbo >> 4) & 0x3fffu) << 16 |
           uint64_t((sbo >> 4) & 0x3fffu) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// kind::f16 with FP32 accumulation, M = 128; bit 13 negates A.
constexpr uint32_t kNegateA = 1u << 13;
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n, bool b_n_major) {
    const uint32_t t = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (uint32_t(b_n_major) << 16) | (uint32_t(n >> 3) << 17) | ((128u >> 4) << 24);
}
// The products and commits are called by a whole warp and issued by the lane
// that elect.sync picks (the same every time): with warp-uniform operands the
// descriptors stay in uniform registers.  Issued under a branch on the lane
// instead, every product waited for its operands' way there, 100 cycles each.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
        : "memory");
}
// A value that every lane of the warp has, as one the compiler knows to be uniform.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
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
// 16 columns.
__device__ __forceinline__ void ld16(uint32_t a, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(a)
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

__device__ __forceinline__ void st8(uint32_t a, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(a), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// Waits for a barrier phase, for at most kWaitLimitNs or until the CTA aborts;
// a whole warp calls it and every lane gets the same answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* abort) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const unsigned long long start = globaltimer_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 32; ++i)
            if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(abort) != 0)) return false;
        if (__any_sync(0xffffffffu, globaltimer_ns() - start > kWaitLimitNs)) {
            if ((threadIdx.x & 31) == 0) {
                atomicExch(&g_device_error, kDevErrTimeout);
                atomicExch(abort, 1);
            }
            return false;
        }
    }
}

// Capped scores, in units of log2: softcap log2 e tanh(y), y = scale / softcap
// times the score x.  For |y| <= 1/2 that is x p(x^2) with cap_score's polynomial.
// A tile with larger scores goes through cap_score first (its special-function
// operations would bound the kernel) and then through the polynomial 1, so that
// both take the same way to the probabilities.
struct Cap {
    float k[5];          // the coefficients of x^2
    float near, out;     // cap_score's arguments
    float most;          // the largest |x| for the polynomial
    __device__ __forceinline__ Cap(float scale, float softcap) {
        constexpr float kLog2e = 1.4426950408889634f;
        near = fap::cap_near(scale, softcap);
        out = softcap * kLog2e;
        float c = scale * kLog2e;
#pragma unroll
        for (int i = 0; i < 5; ++i, c = c * near * near) k[i] = fap::kTanh[i] * c;
        // elsewhere the powers would leave FP32's range, or hidden()'s value, about
        // -5e22 softcap, would not be far below every score
        most = near < 1e3f && softcap > 1e-15f && k[4] > 1e-37f && k[4] < 1e30f ? 0.5f / near : -1.f;
    }
    // A hidden score: x p(x^2) is far below every other's, and finite where p is 1.
    __device__ __forceinline__ float hidden(bool far) const { return far ? -1e18f : -1000.f * most; }
};

// ------------------------------------------------------------ roles
// Hands out the CTA's items and brings their K and V tiles into the ring, in
// the order the products take them.
template <int D>
__device__ __forceinline__ void load_role(const Params& p, const CUtensorMap* tmk, const CUtensorMap* tmv, const Lengths& len,
                                          Barriers& bars, uint8_t* ring, Units share) {
    constexpr int NS = slots<D>();
    const Desc& d = p.d;
    const int lane = threadIdx.x & 31;
    const int boxes = p.box ? kKeys / p.box : 1;     // of a tile, at most 16
    const int i = lane & (boxes - 1), half = lane / boxes;
    const bool mine = half < D / 64;
    const uint32_t at = uint32_t(half) * kSub + uint32_t(i) * p.box * 128;
    unsigned used = 0;                               // slots filled so far
    bool ok = true;
    for (unsigned j = 0; ok; ++j) {
        Item it;
        const bool more = share.next(d, len, it);
        if (j >= kJobs) ok = warp_wait(&bars.job_empty[j % kJobs], (j / kJobs - 1) & 1, &bars.abort);
        if (!ok) break;
        int end = 0;
        if (more) end = paged::key_end<kRows>(d, it.n, it.kv, it.tile);
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
        auto find = [&](int t, int& page, int& off) {
            page = -1;
            off = 0;
            if (!mine || t >= it.count) return;
            const int key = (it.key_tile + t) * kKeys + i * p.box;
            if (key < end) {
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

// The tiles of pages of any size: each of two warps gathers 64 keys' rows.  A
// slot is announced when the next one's copies are under way, its own have
// landed and are visible to the tensor cores.
template <typename T, int D>
__device__ __forceinline__ void gather_role(const Params& p, Barriers& bars, uint32_t ring) {
    constexpr int NS = slots<D>();
    constexpr int kChunks = D / 8, kStep = 32 / kChunks;   // 16-byte chunks of a row; rows of a copy of the warp
    const Desc& d = p.d;
    const int lane = threadIdx.x & 31, first = int((threadIdx.x >> 5) - kGatherWarp) * 64;
    const int chunk = lane % kChunks, sub = lane / kChunks;
    unsigned used = 0;
    auto announce = [&](unsigned u) {
        fence_async();
        mbar_arrive(&bars.full[u % NS]);
    };
    for (unsigned j = 0;; ++j) {
        if (!warp_wait(&bars.job_full[j % kJobs], (j / kJobs) & 1, &bars.abort)) return;
        const Job& job = bars.jobs[j % kJobs];
        const int count = job.count, end = job.end, key0 = job.key_tile * kKeys + first + lane;
        if (count == 0) return;
        const int* table = d.block_table + (long long)job.seq * d.max_pages;
        const long long head = job.head * d.head_stride + chunk * 8;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.job_empty[j % kJobs]);
        for (int t = 0; t < count; ++t) {
            long long at[2];   // where the rows of keys `lane` and `lane + 32` begin, -1: not read
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = key0 + t * kKeys + h * 32;
                at[h] = -1;
                if (key < end) {
                    const int n = key / d.page_size, page = table[n];
                    if (page < 0 || page >= d.n_pages) paged::flag_input();
                    else at[h] = page * d.page_stride + (long long)(key - n * d.page_size) * d.token_stride;
                }
            }
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv, ++used) {
                if (used >= NS && !warp_wait(&bars.empty[used % NS], (used / NS - 1) & 1, &bars.abort)) {
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    return;
                }
                const T* from = static_cast<const T*>(kv ? p.v : p.k) + head;
                const uint32_t slot = ring + (used % NS) * tile_bytes<D>() + (chunk >> 3) * kSub;
#pragma unroll 8
                for (int i = 0; i < 64; i += kStep) {
                    const long long o = __shfl_sync(0xffffffffu, i < 32 ? at[0] : at[1], (i & 31) + sub);
                    const int r = first + i + sub;
                    fap::cp_async16(slot + r * 128 + (((chunk & 7) ^ (r & 7)) << 4), from + (o < 0 ? 0 : o), o >= 0);
                }
                fap::cp_commit();
                if (t + kv > 0) {
                    fap::cp_wait<1>();
                    announce(used - 1);
                }
            }
        }
        fap::cp_wait<0>();
        announce(used - 1);
    }
}

// Issues the products; false when a wait was given up.
template <typename T, int D>
__device__ __forceinline__ bool mma_role(const Desc& d, float scale, Barriers& bars, uint32_t q_smem, uint32_t ring,
                                         uint32_t tmem) {
    constexpr int NS = slots<D>();
    // a negative scale turns the scores' sign here, so that the softmax has a positive one
    const uint32_t idesc_s = idesc_f16<T>(kKeys, false) | (scale < 0.f ? kNegateA : 0u);
    constexpr uint32_t kIdescO = idesc_f16<T>(D, true);
    const int lane = threadIdx.x & 31;
    unsigned used = 0;                 // K and V tiles taken so far
    unsigned items[2] = {0, 0}, tiles[2] = {0, 0};
    auto qk = [&](int w, int slot) {   // S_w = Q_w K^T
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = uint32_t(k >> 2) * kSub + uint32_t(k & 3) * 32;
            mma_ss(tmem + w * 128, sw128_desc(q_smem + w * tile_bytes<D>() + off, 16, 1024),
                   sw128_desc(ring + slot * tile_bytes<D>() + off, 16, 1024), idesc_s, k > 0);
        }
    };
    auto pv = [&](int w, int half, int slot, bool add) {   // O_w += P_w V over half of the keys
#pragma unroll
        for (int k = half * (kKeys / 32); k < (half + 1) * (kKeys / 32); ++k)
            mma_ts(tmem + 256 + w * D, tmem + w * 128 + k * 8,
                   sw128_desc(ring + slot * tile_bytes<D>() + uint32_t(k) * 2048, kSub, 1024), kIdescO, add || k > 0);
    };
    for (unsigned j = 0;; ++j) {
        if (!warp_wait(&bars.job_full[j % kJobs], (j / kJobs) & 1, &bars.abort)) return false;
        const Job& job = bars.jobs[j % kJobs];
        const int count = int(uniform(job.count));
        if (count == 0) return true;
        const int groups = int(uniform(job.n * d.group - job.row0 > 128 ? 2 : 1));
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.job_empty[j % kJobs]);
        if (!warp_wait(&bars.full[used % NS], (used / NS) & 1, &bars.abort)) return false;
        for (int w = 0; w < groups; ++w) {
            if (!warp_wait(&bars.q_full[w], items[w]++ & 1, &bars.abort)) return false;
            fence_after();
            qk(w, used % NS);
            mma_commit(&bars.s_full[w]);
            if (w + 1 == groups) mma_commit(&bars.empty[used % NS]);
        }
        ++used;
        for (int t = 0; t < count; ++t) {
            const unsigned v = used, k = used + 1;
            const bool more = t + 1 < count;
            if (!warp_wait(&bars.full[v % NS], (v / NS) & 1, &bars.abort)) return false;
            for (int w = 0; w < groups; ++w) {
                if (!warp_wait(&bars.p_full[w][0], tiles[w] & 1, &bars.abort)) return false;
                fence_after();
                pv(w, 0, v % NS, t > 0);
                if (more && w == 0 && !warp_wait(&bars.full[k % NS], (k / NS) & 1, &bars.abort)) return false;
                if (!warp_wait(&bars.p_full[w][1], tiles[w]++ & 1, &bars.abort)) return false;
                fence_after();
                pv(w, 1, v % NS, true);
                if (w + 1 == groups) mma_commit(&bars.empty[v % NS]);
                if (more) {
                    qk(w, k % NS);
                    if (w + 1 == groups) mma_commit(&bars.empty[k % NS]);
                }
                mma_commit(&bars.s_full[w]);
            }
            used += more ? 2 : 1;
        }
    }
}

// The row of a thread in an item.
struct Row {
    int tok, g, limit;   // token of the sequence, query head of the group, keys it sees
    bool live;
    __device__ __forceinline__ Row(const Desc& d, const Job& job, int w, int row) {
        const int rows = job.n * d.group - job.row0 - w * 128;
        const int r = job.row0 + w * 128 + row;
        tok = r / d.group;
        g = r - tok * d.group;
        live = row < rows;
        limit = !live ? 0 : d.causal ? max(0, min(job.kv, job.kv - job.n + tok + 1)) : job.kv;
    }
    __device__ __forceinline__ long long at(const Desc& d, const Job& job, long long stride, int D) const {
        return (long long)(job.q0 + tok) * stride + (long long)(job.head * d.group + g) * D;
    }
};

// The thread's query row on its way into shared memory (zeros for none).
template <typename T, int D>
__device__ __forceinline__ void load_query(const Params& p, const Job& job, int w, int row, uint32_t q_smem) {
    const Row r(p.d, job, w, row);
    const T* src = static_cast<const T*>(p.q) + (r.live ? r.at(p.d, job, p.d.q_stride, D) : 0);
    const uint32_t dst = q_smem + w * tile_bytes<D>() + row * 128;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) fap::cp_async16(dst + (i >> 3) * kSub + (((i & 7) ^ (row & 7)) << 4), src + i * 8, r.live);
}

template <typename T, int D, bool CAP>
__device__ __forceinline__ void softmax_role(const Params& p, Barriers& bars, uint32_t q_smem, uint8_t* ring, uint32_t tmem,
                                             long long total_units, int parts) {
    constexpr int NS = slots<D>();
    constexpr float kLog2e = 1.4426950408889634f;
    const Desc& d = p.d;
    const int w = threadIdx.x >> 7, row = threadIdx.x & 127;
    const uint32_t lanes = uint32_t(row & ~31) << 16;
    const uint32_t t_s = tmem + w * 128 + lanes, t_o = tmem + 256 + w * D + lanes;
    const float c = fabsf(p.scale) * kLog2e;   // of the scores to units of log2
    const Cap cap(fabsf(p.scale), CAP ? p.softcap : 1.f);
    unsigned done = 0, used = 0;   // phases of s_full passed; key tiles of the CTA before this item
    bool loaded = false;           // the item's query row is on its way
    for (unsigned j = 0;; ++j) {
        if (!warp_wait(&bars.job_full[j % kJobs], (j / kJobs) & 1, &bars.abort)) return;
        const Job& job = bars.jobs[j % kJobs];
        const int count = job.count;
        if (count == 0) return;
        if (job.n * d.group - job.row0 - w * 128 <= 0) {   // no rows for this warpgroup
            used += count;
            __syncwarp();
            if ((row & 31) == 0) mbar_arrive(&bars.job_empty[j % kJobs]);
            loaded = false;
            continue;
        }
        if (!loaded) load_query<T, D>(p, job, w, row, q_smem);
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_async();
        fence_before();
        mbar_arrive(&bars.q_full[w]);
        loaded = false;
        const int limit = Row(d, job, w, row).limit;
        float m = -INFINITY, l = 0.f;
        for (int t = 0; t < count; ++t) {
            const int key0 = (job.key_tile + t) * kKeys;   // key0 + kKeys may pass 2^31
            if (!warp_wait(&bars.s_full[w], done++ & 1, &bars.abort)) return;
            fence_after();
            float s[128];
#pragma unroll
            for (int i = 0; i < 4; ++i) ld32(t_s + i * 32, s + i * 32);
            wait_ld();
            if (t + 1 == count) {   // the last scores are there, so the queries' place is free for the next item's
                if (!warp_wait(&bars.job_full[(j + 1) % kJobs], ((j + 1) / kJobs) & 1, &bars.abort)) return;
                const Job& next = bars.jobs[(j + 1) % kJobs];
                if (next.count && next.n * d.group - next.row0 - w * 128 > 0) {
                    load_query<T, D>(p, next, w, row, q_smem);
                    loaded = true;
                }
            }
            const int lim = limit - key0;
            const bool masked = __any_sync(0xffffffffu, lim < kKeys);
            float hidden = -INFINITY, k[5];
            if (CAP) {
                if (masked) {   // whatever stands there must not look large
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i < lim ? s[i] : 0.f;
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
                for (int i = 0; i < 128; ++i) s[i] = i < lim ? s[i] : hidden;
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
            mx -= kLift<T>;
            if (t == 0) {
                m = mx;
            } else {
                const bool rise = mx - m > kRise;
                if (__any_sync(0xffffffffu, rise)) {
                    const float a = rise ? paged::exp2_approx(m - mx) : 1.f;
                    if (rise) m = mx;
                    l *= a;
#pragma unroll 1
                    for (int i = 0; i < D / 16; ++i) {   // few registers: the scores stay in theirs
                        float o[16];
                        ld16(t_o + i * 16, o);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] *= a;
                        st16(t_o + i * 16, reinterpret_cast<const uint32_t*>(o));
                    }
                }
            }
            if (w == 0 && job.end - key0 < kKeys) {   // rows of V that no key of the item's rows reaches
                const unsigned u = 2 * (used + t) + 1;
                if (!warp_wait(&bars.full[u % NS], (u / NS) & 1, &bars.abort)) return;
                if (row >= job.end - key0) {
                    uint8_t* v = ring + (u % NS) * tile_bytes<D>() + row * 128;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i)
                        *reinterpret_cast<uint4*>(v + (i >> 3) * kSub + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async();
            }
            const float base = m == -INFINITY ? 0.f : m;
            const uint64_t c2 = pair(c, c), b2 = pair(-base, -base);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int half = 0; half < 2; ++half) {   // the products with the first half start while the second is computed
#pragma unroll
                for (int i = 4 * half; i < 4 * half + 4; ++i) {
                    uint32_t pk[8];
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
                    }
                    st8(t_s + i * 8, pk);
                }
                wait_st();
                fence_before();
                mbar_arrive(&bars.p_full[w][half]);
            }
            {
                float a, b;
                unpair(add2(sum[0], sum[1]), a, b);
                l += a + b;
            }
        }
        used += count;
        if (!warp_wait(&bars.s_full[w], done++ & 1, &bars.abort)) return;   // the accumulator is complete
        fence_after();
        const Row r(d, job, w, row);
        const float base = m;
        const long long o_at = r.at(d, job, d.o_stride, D);
        auto write = [&](int i, float (&o)[32], float inv) {   // columns 32 i .. 32 i + 31 of the row
            if (!r.live) return;
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= inv;
            if (p.o_f32) {
                float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.o) + o_at + i * 32);
#pragma unroll
                for (int e = 0; e < 8; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            } else {
                uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.o) + o_at + i * 32);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    dst[e] = make_uint4(paged::pack2<T>(o[8 * e], o[8 * e + 1]), paged::pack2<T>(o[8 * e + 2], o[8 * e + 3]),
                                        paged::pack2<T>(o[8 * e + 4], o[8 * e + 5]), paged::pack2<T>(o[8 * e + 6], o[8 * e + 7]));
            }
        };
        auto write_lse = [&](float top, float total) {
            if (r.live && p.lse)
                p.lse[(long long)(job.q0 + r.tok) * d.n_head_q + job.head * d.group + r.g] =
                    total == 0.f ? -INFINITY : (top + log2f(total)) / kLog2e;
        };
        if (job.whole) {
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
            // the CTAs that have a part
            const int c0 = paged::share_of(job.first, total_units, parts), c1 = paged::share_of(job.first + job.units - 1, total_units, parts);
            const long long slot = (long long)(blockIdx.x * 2 + (job.key_tile == 0)) * 2 + w;
            float4* dst = reinterpret_cast<float4*>(p.ws_o) + slot * (D / 4) * 128 + row;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                float o[32];
                ld32(t_o + i * 32, o);
                wait_ld();
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    __stcg(dst + (i * 8 + e) * 128, make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]));
            }
            __stcg(reinterpret_cast<float2*>(p.ws_ml) + slot * 128 + row, make_float2(base, l));
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
                constexpr int kFew = 4;   // parts whose loads are all in flight together
                const int np = c1 - c0 + 1;
                float top = -INFINITY, total = 0.f, wt[kFew] = {0.f, 0.f, 0.f, 0.f};
                if (np <= kFew) {
                    float2 v[kFew];
#pragma unroll
                    for (int k = 0; k < kFew; ++k) v[k] = k < np ? __ldcg(ml + part(c0 + k) * 128) : make_float2(-INFINITY, 0.f);
#pragma unroll
                    for (int k = 0; k < kFew; ++k) top = fmaxf(top, v[k].x);
#pragma unroll
                    for (int k = 0; k < kFew; ++k) {
                        wt[k] = paged::exp2_approx(v[k].x - (top == -INFINITY ? 0.f : top));
                        total = fmaf(wt[k], v[k].y, total);
                    }
                } else {
#pragma unroll 4
                    for (int q = c0; q <= c1; ++q) top = fmaxf(top, __ldcg(ml + part(q) * 128).x);
#pragma unroll 4
                    for (int q = c0; q <= c1; ++q) {
                        const float2 v = __ldcg(ml + part(q) * 128);
                        total = fmaf(paged::exp2_approx(v.x - (top == -INFINITY ? 0.f : top)), v.y, total);
                    }
                }
                const float safe = top == -INFINITY ? 0.f : top;
                const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll 1
                for (int i = 0; i < D / 32; ++i) {
                    float o[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0.f;
                    auto add = [&](const float4 (&v)[8], float f) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            o[4 * e] = fmaf(f, v[e].x, o[4 * e]);
                            o[4 * e + 1] = fmaf(f, v[e].y, o[4 * e + 1]);
                            o[4 * e + 2] = fmaf(f, v[e].z, o[4 * e + 2]);
                            o[4 * e + 3] = fmaf(f, v[e].w, o[4 * e + 3]);
                        }
                    };
                    if (np <= kFew) {
                        float4 v[kFew][8];
#pragma unroll
                        for (int k = 0; k < kFew; ++k)
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                v[k][e] = k < np ? __ldcg(po + (part(c0 + k) * (D / 4) + i * 8 + e) * 128)
                                                 : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int k = 0; k < kFew; ++k) add(v[k], wt[k]);
                    } else {
#pragma unroll 2
                        for (int q = c0; q <= c1; ++q) {
                            const float f = paged::exp2_approx(__ldcg(ml + part(q) * 128).x - safe);
                            float4 v[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = __ldcg(po + (part(q) * (D / 4) + i * 8 + e) * 128);
                            add(v, f);
                        }
                    }
                    write(i, o, inv);
                }
                write_lse(top, total);
            }
        }
        __syncwarp();
        if ((row & 31) == 0) mbar_arrive(&bars.job_empty[j % kJobs]);
    }
}

template <typename T, int D, bool CAP>
__global__ void __launch_bounds__(kThreads, 1)
    fa_paged_tc_kernel(const Params p, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_smem = smem;
    uint8_t* ring = q_smem + 2 * tile_bytes<D>();
    Barriers& bars = *reinterpret_cast<Barriers*>(ring + slots<D>() * tile_bytes<D>());
    const Lengths len(reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(&bars + 1) + 15) & ~uintptr_t(15)), p.d.n_seq);
    const int warp = threadIdx.x >> 5;

    if (threadIdx.x == kLoadWarp * 32 && p.box) {
        prefetch_tensormap(&tmk);
        prefetch_tensormap(&tmv);
    }
    paged::read_lengths<kRows, kKeys, kOver, kThreads, true>(p.d, len, (long long)kWholeFrom * gridDim.x);
    const int parts = len.head->ok ? int(min((long long)gridDim.x, len.head->total)) : 0;
    if (int(blockIdx.x) >= parts) return;
    // what the first copies wait for, side by side: the barriers, tensor memory
    // and the load warp's place in the work
    if (threadIdx.x < 8) {
        mbar_init(&bars.full[threadIdx.x], p.box ? 1 : 64);
        mbar_init(&bars.empty[threadIdx.x], 1);
    } else if (threadIdx.x < 10) {
        const int w = threadIdx.x - 8;
        mbar_init(&bars.q_full[w], 128);
        mbar_init(&bars.s_full[w], 1);
        mbar_init(&bars.p_full[w][0], 128);
        mbar_init(&bars.p_full[w][1], 128);
        mbar_init(&bars.joined[w], 128);
    } else if (threadIdx.x < 10 + kJobs) {
        mbar_init(&bars.job_full[threadIdx.x - 10], 1);
        mbar_init(&bars.job_empty[threadIdx.x - 10], p.box ? 9 : 11);   // the softmax warps, the issuing one, the gathering ones
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
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem);
    if (warp < kMmaWarp) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        softmax_role<T, D, CAP>(p, bars, smem_addr(q_smem), ring, tmem, len.head->total, parts);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == kLoadWarp) {
            load_role<D>(p, &tmk, &tmv, len, bars, ring, share);
        } else if (warp == kMmaWarp) {
            if (!mma_role<T, D>(p.d, p.scale, bars, uniform(smem_addr(q_smem)), uniform(smem_addr(ring)),
                                uniform(tmem))) {
                // leave only when the products in flight are done
                mma_commit(&bars.drain);
                __syncwarp();
                mbar_wait(&bars.drain, 0);
            }
        } else if (p.box == 0) {
            gather_role<T, D>(p, bars, smem_addr(ring));
        }
    }

    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

}  // namespace fatc
}  // namespace p100b
