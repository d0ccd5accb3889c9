// paged.cuh — what the paged-cache kernels share: the 16-bit types, the
// descriptor as the kernels see it, the check of the device-resident lengths
// and the division of an attention call's work into equal shares.
//
// A paged cache holds pages of page_size token rows per kv head; sequence s
// finds token j in row j % page_size of page block_table[s][j / page_size].
// The n = q_start[s+1] - q_start[s] new tokens of a sequence are its last
// ones: new token i sits at position kv_len[s] - n + i.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace p100b {
namespace paged {

constexpr int kMaxSeq = 1024;   // sequences of one call: their lengths live in shared memory

struct Desc {
    int n_seq, n_tokens, max_q;
    int n_head_q, n_head_kv, group;
    int page_size, n_pages, max_pages;
    int causal;
    long long page_stride, head_stride, token_stride;   // of the pages, in elements
    long long q_stride, o_stride;                       // between tokens, in elements
    const int* block_table;   // [n_seq][max_pages]
    const int* q_start;       // [n_seq + 1]
    const int* kv_len;        // [n_seq]
};

// ------------------------------------------------------------ 16-bit types
template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Two floats rounded to nearest even, lo in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The floats of a pair.
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t v, float& lo, float& hi);
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t v, float& lo, float& hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    lo = f.x;
    hi = f.y;
}
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t v, float& lo, float& hi) {
    lo = __uint_as_float(v << 16);
    hi = __uint_as_float(v & 0xffff0000u);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------ pairs of floats
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ void flag_input() { atomicExch(&g_device_error, kDevErrInput); }

// ------------------------------------------------------------ shares
// An attention call is a list of row tiles, each with the key tiles that its
// rows see: unit = KEYS keys of ROWS query rows of one (sequence, kv head).
// The rows of a kv head are the (token, query head of the group) pairs in
// token order, so a tile serves every query head that reads its keys.  A row
// tile that sees no key still has one unit, which writes its zeros.
//
// Cut: units are ordered by sequence, kv head, row tile, key tile, each row
// tile with OVER more units behind it for what a row tile costs beyond its
// keys, and CTA c of P takes [c U / P, (c + 1) U / P): equal work whatever the
// lengths, a row tile cut only where a share ends.  Whole: with many row tiles
// per CTA they are dealt out uncut, the ones with the most keys of a sequence
// first and back and forth over the CTAs, so that neighbours in time read the
// same keys and nothing is joined.
struct Lengths {                     // in shared memory, the arrays sized by n_seq
    struct Head {
        long long total;             // units (cut) or row tiles (whole) of the call
        int ok;                      // the lengths are usable
        int whole;
    };
    Head* head;
    unsigned long long* first;       // [n_seq] units or row tiles before the sequence
    int* q0;                         // [n_seq + 1]
    int* kv;                         // [n_seq]
    unsigned* per_head;              // [n_seq] units or row tiles of one kv head

    __device__ Lengths(void* at, int n_seq) {   // 16-byte aligned
        head = static_cast<Head*>(at);
        first = reinterpret_cast<unsigned long long*>(head + 1);
        q0 = reinterpret_cast<int*>(first + n_seq);
        kv = q0 + n_seq + 1;
        per_head = reinterpret_cast<unsigned*>(kv + n_seq);
    }
    __host__ __device__ static size_t bytes(int n_seq) {
        return (sizeof(Head) + size_t(n_seq) * (8 + 3 * 4) + 4 + 127) / 128 * 128;
    }
};

template <int ROWS>
__host__ __device__ __forceinline__ int row_tiles(const Desc& d, int n) {
    return int(((long long)n * d.group + ROWS - 1) / ROWS);
}
// Keys [0, key_end) are seen by some row of the tile.
template <int ROWS>
__host__ __device__ __forceinline__ int key_end(const Desc& d, int n, int kv, int tile) {
    const int last = min((tile + 1) * ROWS, n * d.group) - 1;
    const int end = d.causal ? kv - n + last / d.group + 1 : kv;
    return max(0, min(end, kv));
}
template <int ROWS, int KEYS>
__host__ __device__ __forceinline__ int tile_units(const Desc& d, int n, int kv, int tile) {
    return max(0, key_end<ROWS>(d, n, kv, tile) - 1) / KEYS + 1;   // of up to 2^31 - 1 keys
}

// Units of one kv head of a lane's sequence, every lane of the warp its own:
// few row tiles alone, many by the whole warp.
template <int ROWS, int KEYS, int OVER>
__device__ __forceinline__ unsigned head_units(const Desc& d, int n, int kv, int tiles) {
    const int lane = threadIdx.x & 31;
    unsigned sum = 0;
    if (tiles <= 4)
        for (int t = 0; t < tiles; ++t) sum += tile_units<ROWS, KEYS>(d, n, kv, t) + OVER;
    unsigned left = __ballot_sync(0xffffffffu, tiles > 4);
    while (left) {
        const int l = __ffs(left) - 1;
        left &= left - 1;
        const int ln = __shfl_sync(0xffffffffu, n, l), lkv = __shfl_sync(0xffffffffu, kv, l),
                  lt = __shfl_sync(0xffffffffu, tiles, l);
        unsigned part = 0;
        for (int t = lane; t < lt; t += 32) part += tile_units<ROWS, KEYS>(d, ln, lkv, t) + OVER;
        part = __reduce_add_sync(0xffffffffu, part);
        if (lane == l) sum = part;
    }
    return sum;
}

// Reads and checks the lengths and counts the units; every thread of the CTA
// calls it.  Lengths that are out of order or out of range raise the device
// flag and make the call do nothing.  With MAY_BE_WHOLE, row tiles are dealt
// out whole from whole_from of them on.  A thread takes a sequence: one round
// of loads, and few meetings of the CTA, stand before the first copies.
template <int ROWS, int KEYS, int OVER, int THREADS, bool MAY_BE_WHOLE>
__device__ void read_lengths(const Desc& d, const Lengths& s, long long whole_from) {
    constexpr int W = (THREADS + 31) / 32;
    __shared__ unsigned long long s_part[W];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    bool good = true;
    long long mine = 0;   // row tiles of the thread's sequences, of all heads
    for (int i = tid; i < d.n_seq; i += THREADS) {
        const int q0 = d.q_start[i], q1 = d.q_start[i + 1], kv = d.kv_len[i];
        const int n = q1 - q0;
        good = good && q0 >= 0 && q1 >= q0 && n <= d.max_q && q1 <= d.n_tokens && kv >= 0 &&
               (long long)kv <= (long long)d.max_pages * d.page_size;
        s.q0[i] = q0;
        if (i + 1 == d.n_seq) s.q0[i + 1] = q1;
        s.kv[i] = kv;
        if (MAY_BE_WHOLE && good) mine += (long long)row_tiles<ROWS>(d, n) * d.n_head_kv;
    }
    if (MAY_BE_WHOLE) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
        if (lane == 0) s_part[warp] = (unsigned long long)mine;
    }
    if (!__syncthreads_and(good)) {
        if (tid == 0) s.head->ok = 0, flag_input();
        __syncthreads();
        return;
    }
    bool whole = false;
    if (MAY_BE_WHOLE) {
        long long tiles = 0;
        for (int w = 0; w < W; ++w) tiles += (long long)s_part[w];
        whole = tiles >= whole_from;
        __syncthreads();   // s_part is free
    }
    unsigned long long before = 0;   // units of the sequences of earlier rounds
    for (int i0 = 0; i0 < d.n_seq; i0 += THREADS) {
        const int i = i0 + tid;
        int n = 0, kv = 0, tiles = 0;
        if (i < d.n_seq) {
            n = s.q0[i + 1] - s.q0[i];
            kv = s.kv[i];
            tiles = row_tiles<ROWS>(d, n);
        }
        const unsigned own = whole ? unsigned(tiles) : head_units<ROWS, KEYS, OVER>(d, n, kv, tiles);
        const unsigned long long all = (unsigned long long)own * d.n_head_kv;
        unsigned long long v = all;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const unsigned long long u = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v += u;
        }
        if (lane == 31) s_part[warp] = v;
        __syncthreads();
        unsigned long long base = before;
        for (int w = 0; w < W; ++w) {
            if (w < warp) base += s_part[w];
            before += s_part[w];
        }
        if (i < d.n_seq) {
            s.per_head[i] = own;
            s.first[i] = base + v - all;
        }
        __syncthreads();
    }
    if (tid == 0) {
        s.head->total = (long long)before;
        s.head->whole = whole;
        s.head->ok = 1;
    }
    __syncthreads();
}

struct Item {
    int seq, head, tile;     // row tile of the sequence's head
    int n, kv;               // the sequence's new tokens and length
    int key_tile, count;     // key tiles [key_tile, key_tile + count) of the row tile are this CTA's
    int units;               // key tiles of the whole row tile
    long long tile_first;    // its first unit (cut)
};

// The first unit of share c of `parts`.
__host__ __device__ __forceinline__ long long share_begin(long long total, int c, int parts) {
    if (total < (1LL << 31) / parts) return unsigned(total) * unsigned(c) / unsigned(parts);   // a short division
    return total * c / parts;
}
// The CTA whose share of `parts` holds unit u: the largest c with
// share_begin(c) <= u.
__host__ __device__ __forceinline__ int share_of(long long u, long long total, int parts) {
    if (total < (1LL << 31) / parts) return int((unsigned(u + 1) * unsigned(parts) - 1) / unsigned(total));
    return int(((u + 1) * parts - 1) / total);
}

// One CTA's share as a list of items; the calls are warp-uniform.
template <int ROWS, int KEYS, int OVER>
struct Share {
    long long at, end;       // units left (cut); the next row tile (whole)
    int seq, head, tile, key_tile, tiles, n, kv, cta, parts, round;

    __device__ __forceinline__ void enter_seq(const Desc& d, const Lengths& s, int i) {
        seq = i;
        n = s.q0[i + 1] - s.q0[i];
        kv = s.kv[i];
        tiles = row_tiles<ROWS>(d, n);
    }
    // The last sequence whose first unit is at or before u.
    __device__ __forceinline__ int seq_of(const Desc& d, const Lengths& s, long long u) const {
        int lo = 0, hi = d.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if ((long long)s.first[mid] <= u) lo = mid; else hi = mid - 1;
        }
        return lo;
    }

    // cta's share of `parts`, at most one for each unit.
    __device__ __forceinline__ void begin(const Desc& d, const Lengths& s, int c, int p) {
        cta = c;
        parts = p;
        round = 0;
        if (s.head->whole) return;
        const long long total = s.head->total;
        at = share_begin(total, cta, parts);
        end = share_begin(total, cta + 1, parts);
        if (at >= end) return;
        enter_seq(d, s, seq_of(d, s, at));
        const unsigned long long in_seq = (unsigned long long)at - s.first[seq];
        head = in_seq >> 32 ? int(in_seq / s.per_head[seq]) : int(unsigned(in_seq) / s.per_head[seq]);
        unsigned rest = unsigned(in_seq - (unsigned long long)head * s.per_head[seq]);
        const int lane = threadIdx.x & 31;
        for (int t0 = 0;; t0 += 32) {   // the row tile that holds unit `rest` of the head
            const unsigned own = t0 + lane < tiles ? tile_units<ROWS, KEYS>(d, n, kv, t0 + lane) + OVER : 0;
            unsigned v = own;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const unsigned u = __shfl_up_sync(0xffffffffu, v, off);
                if (lane >= off) v += u;
            }
            const unsigned ahead = __ballot_sync(0xffffffffu, v <= rest);
            if (ahead != 0xffffffffu) {
                const int l = __popc(ahead);
                tile = t0 + l;
                key_tile = int(rest - __shfl_sync(0xffffffffu, v - own, l));
                break;
            }
            rest -= __shfl_sync(0xffffffffu, v, 31);
        }
    }

    __device__ __forceinline__ bool next(const Desc& d, const Lengths& s, Item& it) {
        if (s.head->whole) {
            const long long i = (long long)round * parts + (round & 1 ? parts - 1 - cta : cta);
            ++round;
            if (i >= s.head->total) return false;
            enter_seq(d, s, seq_of(d, s, i));
            const unsigned in_seq = unsigned((unsigned long long)i - s.first[seq]);
            it.tile = tiles - 1 - int(in_seq / d.n_head_kv);
            it.head = int(in_seq % d.n_head_kv);
            it.key_tile = 0;
            it.units = it.count = tile_units<ROWS, KEYS>(d, n, kv, it.tile);
            it.tile_first = 0;
        } else {
            for (;;) {
                if (at >= end) return false;
                while (tile == tiles) {
                    tile = 0;
                    if (tiles == 0 || ++head == d.n_head_kv) {
                        head = 0;
                        enter_seq(d, s, seq + 1);
                    }
                }
                it.tile = tile;
                it.head = head;
                it.units = tile_units<ROWS, KEYS>(d, n, kv, tile);
                it.key_tile = key_tile;
                it.tile_first = at - key_tile;
                it.count = int(min((long long)(it.units - key_tile), end - at));
                at += it.units - key_tile + OVER;
                key_tile = 0;
                ++tile;
                if (it.count > 0) break;   // else the share began behind the tile's last key tile
            }
        }
        it.seq = seq;
        it.n = n;
        it.kv = kv;
        return true;
    }
};

}  // namespace paged
}  // namespace p100b
