// rope.cuh — the append of new tokens to a paged cache (paged_append.cuh) with
// rotary positions computed from each pair's frequency: any positions, part of a
// head, both pairings, no table.
//
// Pair i of a head turns by position x f_i radians.  p100_rope holds f_i as
// the turns of one token, f_i / 2 pi, in units of 2^-64 turn: position x that,
// modulo 2^64, is the angle's part of a turn with an error of position x 2^-65
// turns, whatever the position (an FP32 product of 10^6 x f is off by 0.06
// rad).  As a signed number it is the angle in [-1/2, 1/2) turns; FP32 rounds it
// by 2^-24 of its size, and sincospi takes it from there.
//
// Value x_i of a head with partner x_j becomes r (x_i A_i + x_j B_i): r is the
// norm's factor, A_i = w_i m cos, B_i = -+ w_j m sin hold the norm's weights,
// the angle, its sign and the scale m, and are computed once a warp for all its
// heads of a kind (a lane the angles of two pairs, then shared by shuffles), while
// the first heads' loads are on their way.  All in FP32, two values an operation;
// the one rounding is the store to 16 bits.
//
// Bytes bound it, then the latency of a warp's chain: partners that lie in another
// lane come as the 16-bit values they were loaded as, values that do not turn and
// the v heads of the cache's own type go through, and the loops are written out by
// pairing and norm (with the branches inside 36 us below).  The cosines wait in
// shared memory for the k heads.  Blocks of four warps, five an SM: with eight the
// last ones leave SMs idle (30 us), with six of four the registers spill (27.5), with
// four too few warps are there (35).
// Measured: 2,777 tokens of 64 / 8 heads of 128 from bf16 with norms and halves
// 24.4 us, 0.71 of measured bandwidth; 8,192 of them from fp32 with norms 92 us,
// 0.83.
#pragma once
#include <type_traits>

#include "paged_append.cuh"

namespace p100b {
namespace paged {

constexpr int kRopeThreads = 128;

struct TurnParams {
    p100_rope rope;
    const int* position;   // [n_tokens] or null: the rows' own in their sequence
};

// (cos, sin) of `turns` a token at a position, times mscale.
__device__ __forceinline__ float2 turned(unsigned long long turns, int position, float mscale) {
    const long long part = (long long)(turns * (unsigned long long)position);
    float s, c;
    sincospif(__ll2float_rn(part) * 0x1p-63f, &s, &c);
    return make_float2(c * mscale, s * mscale);
}

// The values of 16 bytes, two by two.
template <typename S, int N>
__device__ __forceinline__ void pairs(const uint4& x, uint64_t (&y)[N]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    if constexpr (sizeof(S) == 4) {
        y[0] = pair(__uint_as_float(w[0]), __uint_as_float(w[1]));
        y[1] = pair(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a, b;
            unpack2<S>(w[i], a, b);
            y[i] = pair(a, b);
        }
    }
}

template <typename S, typename T, int D>
__global__ void __launch_bounds__(kRopeThreads, 5)
    append_rope_kernel(const AppendParams p, const __grid_constant__ TurnParams r) {
    constexpr int E = append_values<S>();
    constexpr int kLanes = D / E;              // of a head
    constexpr int kHeads = 32 / kLanes;        // of a step
    constexpr int U = append_steps<S>();
    __shared__ float s_cs[E][kRopeThreads], s_sn[E][kRopeThreads];
    __shared__ float s_heads[kRopeThreads * E];
    __shared__ unsigned long long s_turns[64];   // a lane's own index into the parameters is one access for each lane
    if (threadIdx.x < 64) s_turns[threadIdx.x] = r.rope.turns[threadIdx.x];
    __syncthreads();
    const int lane = threadIdx.x & 31, in_head = lane % kLanes, v0 = in_head * E;
    const Steps steps(p.d.n_head_q, p.d.n_head_kv, kHeads);
    const long long item = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const int t = int(item / p.warps);
    if (t >= p.d.n_tokens) return;
    const int share = int(item - (long long)t * p.warps);
    const int begin = int((long long)share * steps.all() / p.warps);
    const int end = int((long long)(share + 1) * steps.all() / p.warps);

    // the steps of kind 0 (q), 1 (k), 2 (v) are [first_of(kind), first_of(kind + 1))
    auto first_of = [&](int kind) { return kind == 0 ? 0 : steps.q + (kind - 1) * steps.kv; };
    const int own = lane / kLanes;             // this lane's head of a step
    const S* row = static_cast<const S*>(p.qkv) + t * p.qkv_stride + own * D + v0;
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

    const int given = r.position ? r.position[t] : 0;
    int q0, q1, kv;
    const int seq = find_seq(p.d, t, q0, q1, kv);
    if (seq < 0) return;   // a padding token
    const int pos = kv - (q1 - q0) + (t - q0), at_angle = r.position ? given : pos;
    const int page_at = pos / p.d.page_size;
    if (pos < 0 || page_at >= p.d.max_pages || at_angle < 0) {
        if (lane == 0) flag_input();
        return;
    }
    long long dst = 0;
    bool has_page = true;
    if (end > steps.q) {
        const int page = p.d.block_table[(long long)seq * p.d.max_pages + page_at];
        has_page = page >= 0 && page < p.d.n_pages;
        if (!has_page && lane == 0) flag_input();
        dst = page * p.d.page_stride + (pos - page_at * p.d.page_size) * p.d.token_stride;
    }

    const int dim = r.rope.rope_dim, half = dim / 2;
    const bool halves = r.rope.half, straight = half % E == 0;   // the partners of a lane's values lie in one lane
    const int partner = halves && straight && v0 < dim ? lane + (v0 < half ? half / E : -half / E) : lane;
    if (kind < 2) {   // of the lane's values: cosine and signed sine, 1 and 0 where they do not turn
        const float2 even = 2 * lane < half ? turned(s_turns[2 * lane], at_angle, r.rope.mscale) : make_float2(1.f, 0.f);
        const float2 odd = 2 * lane + 1 < half ? turned(s_turns[2 * lane + 1], at_angle, r.rope.mscale) : make_float2(1.f, 0.f);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int v = v0 + i, pair_of = halves ? (v < half ? v : v - half) : v / 2;
            const int from = (pair_of >> 1) & 31;
            const float c0 = __shfl_sync(0xffffffffu, even.x, from), c1 = __shfl_sync(0xffffffffu, odd.x, from);
            const float s0 = __shfl_sync(0xffffffffu, even.y, from), s1 = __shfl_sync(0xffffffffu, odd.y, from);
            const float s = pair_of & 1 ? s1 : s0;
            s_cs[i][threadIdx.x] = v < dim ? (pair_of & 1 ? c1 : c0) : 1.f;
            s_sn[i][threadIdx.x] = v >= dim ? 0.f : (halves ? v < half : i % 2 == 0) ? -s : s;
        }
    }
    for (int at = begin; at < end; ++kind) {
        const int base = first_of(kind), stop = min(end, first_of(kind + 1)) - base, from = at - base;
        const int heads = kind == 0 ? p.d.n_head_q : p.d.n_head_kv;
        const float* norm = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
        const S* src = source(kind);
        if (at != begin) load(src, from, stop, heads);
        T* to = kind == 0 ? static_cast<T*>(p.q) + t * p.d.q_stride : static_cast<T*>(kind == 2 ? p.v : p.k) + dst;
        const long long stride = kind == 0 ? D : p.d.head_stride;   // between heads
        to += own * stride + v0;
        uint64_t A[E / 2], B[E / 2];
        if (kind < 2) {
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                float a[2], b[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int v = v0 + i + e, other = v >= dim ? v : halves ? (v < half ? v + half : v - half) : v ^ 1;
                    a[e] = s_cs[i + e][threadIdx.x] * (norm ? norm[v] : 1.f);
                    b[e] = s_sn[i + e][threadIdx.x] * (norm ? norm[other] : 1.f);
                }
                A[i / 2] = pair(a[0], a[1]);
                B[i / 2] = pair(b[0], b[1]);
            }
        }
        // the steps of the kind, written out for its norm and its partners: in the
        // lane (0), in another lane (1), anywhere (2), none (3)
        auto steps_of = [&](auto normed, auto where) {
            constexpr bool kNorm = decltype(normed)::value;
            constexpr int kWhere = decltype(where)::value;
            for (int step = from; step < stop; step += U) {
                uint4 now[U];
#pragma unroll
                for (int u = 0; u < U; ++u) now[u] = x[u];
                load(src, step + U, stop, heads);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (step + u >= stop) break;
                    T* const place = to + (step + u) * kHeads * stride;
                    const bool live = (step + u) * kHeads + own < heads && (kind == 0 || has_page);
                    if (std::is_same<S, T>::value && kWhere == 3) {   // as they are
                        if (live) *reinterpret_cast<uint4*>(place) = now[u];
                        continue;
                    }
                    uint64_t y[E / 2];
                    pairs<S>(now[u], y);
                    if (kWhere < 3) {
                        uint64_t o[E / 2];   // the partners
                        if (kWhere == 0) {
#pragma unroll
                            for (int i = 0; i < E / 2; ++i) {
                                float a, b;
                                unpair(y[i], a, b);
                                o[i] = pair(b, a);
                            }
                        } else if (kWhere == 1) {
                            uint4 w;
                            w.x = __shfl_sync(0xffffffffu, now[u].x, partner);
                            w.y = __shfl_sync(0xffffffffu, now[u].y, partner);
                            w.z = __shfl_sync(0xffffffffu, now[u].z, partner);
                            w.w = __shfl_sync(0xffffffffu, now[u].w, partner);
                            pairs<S>(w, o);
                        } else {   // halves that end inside a lane: through shared memory
                            float* all = s_heads + (threadIdx.x >> 5) * 32 * E;
                            const float* head = all + own * D;
                            __syncwarp();
#pragma unroll
                            for (int i = 0; i < E / 2; ++i) unpair(y[i], all[lane * E + 2 * i], all[lane * E + 2 * i + 1]);
                            __syncwarp();
                            auto other = [&](int v) { return head[v >= dim ? v : v < half ? v + half : v - half]; };
#pragma unroll
                            for (int i = 0; i < E / 2; ++i) o[i] = pair(other(v0 + 2 * i), other(v0 + 2 * i + 1));
                        }
                        if (dim < D) {   // what does not turn takes nothing from a partner, which may be infinite
#pragma unroll
                            for (int i = 0; i < E / 2; ++i)
                                if (v0 + 2 * i >= dim) o[i] = 0;   // (dim is even)
                        }
                        uint64_t f = 0;
                        if (kNorm) {
                            uint64_t sq = mul2(y[0], y[0]);
#pragma unroll
                            for (int i = 1; i < E / 2; ++i) sq = fma2(y[i], y[i], sq);
                            float s0, s1;
                            unpair(sq, s0, s1);
                            float ss = s0 + s1;
#pragma unroll
                            for (int off = 1; off < kLanes; off <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
                            const float rr = rsqrtf(fmaf(ss, 1.0f / float(D), p.eps));
                            f = pair(rr, rr);
                        }
#pragma unroll
                        for (int i = 0; i < E / 2; ++i) {
                            y[i] = fma2(o[i], B[i], mul2(y[i], A[i]));
                            if (kNorm) y[i] = mul2(y[i], f);
                        }
                    }
                    if (live) {
                        float z[E];
#pragma unroll
                        for (int i = 0; i < E / 2; ++i) unpair(y[i], z[2 * i], z[2 * i + 1]);
                        store_values<T, E>(place, z);
                    }
                }
            }
        };
        auto by_norm = [&](auto where) {
            if (norm) steps_of(std::true_type(), where);
            else steps_of(std::false_type(), where);
        };
        if (kind == 2) steps_of(std::false_type(), std::integral_constant<int, 3>());
        else if (!halves) by_norm(std::integral_constant<int, 0>());
        else if (straight) by_norm(std::integral_constant<int, 1>());
        else by_norm(std::integral_constant<int, 2>());
        at = base + stop;
    }
}

}  // namespace paged
}  // namespace p100b
