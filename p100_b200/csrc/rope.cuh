// rope.cuh — rotary positions without a table: the rotation of the append
// kernel (paged_append.cuh) from each pair's frequency.
//
// Pair i of a head turns by position x f_i radians.  p100_rope holds f_i as
// the turns of one token, f_i / 2 pi, in units of 2^-64 turn: position x that,
// modulo 2^64, is the angle's part of a turn with an error of position x 2^-64
// turns, whatever the position (an FP32 product of 10^6 x f is off by 0.06
// rad).  As a signed number it is the angle in [-1/2, 1/2) turns; FP32 rounds it
// by 2^-24 of its size, and sincospi takes it from there.
//
// A lane computes the angles of its own values once for all heads that its
// warp handles, while the first heads' loads are on their way; a table would
// be 8 bytes read a pair and a limit on positions.
#pragma once
#include "paged_append.cuh"

namespace p100b {
namespace paged {

struct TurnParams {
    p100_rope rope;
    const int* position;   // [n_tokens] or null: the rows' own in their sequence
};

template <int E, int D>
struct ByTurns {
    using Params = TurnParams;
    static constexpr int kLanes = D / E;
    float2 cs[E];   // of the lane's pairs (adjacent ones: cs[0 .. E / 2)) or values
    int rotated;    // pairs (adjacent) or values of the lane that turn
    int partner;    // lane of the other halves, where they lie in one
    bool upper;     // the lane's values are second halves
    bool straight;  // the other halves of a lane lie in one lane, at the same places

    __device__ __forceinline__ static float2 angle(unsigned long long turns, int pos, float mscale) {
        const long long part = (long long)(turns * (unsigned long long)pos);
        float s, c;
        sincospif(__ll2float_rn(part) * 0x1p-63f, &s, &c);
        return make_float2(c * mscale, s * mscale);
    }
    __device__ __forceinline__ bool begin(const AppendParams&, const Params& r, int t, int pos, int in_head) {
        const int at = r.position ? r.position[t] : pos;
        if (at < 0) return false;
        const int dim = r.rope.rope_dim, v0 = in_head * E;
        if (r.rope.half) {
            const int half = dim / 2, lane = threadIdx.x & 31;
            straight = half % E == 0;
            rotated = max(0, min(E, dim - v0));
            upper = v0 >= half;
            partner = straight && rotated ? lane + (upper ? -half / E : half / E) : lane;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int v = v0 + i;
                cs[i] = i < rotated ? angle(r.rope.turns[v < half ? v : v - half], at, r.rope.mscale) : make_float2(1.f, 0.f);
            }
        } else {
            rotated = max(0, min(E / 2, (dim - v0) / 2));
#pragma unroll
            for (int i = 0; i < E / 2; ++i)
                cs[i] = i < rotated ? angle(r.rope.turns[v0 / 2 + i], at, r.rope.mscale) : make_float2(1.f, 0.f);
        }
        return true;
    }
    __device__ __forceinline__ bool turns(const AppendParams&, const Params&) const { return true; }
    // Values that do not turn are left alone, not multiplied by 1 and 0: they may be infinite.
    __device__ __forceinline__ void turn(const AppendParams&, const Params& r, float (&y)[E]) const {
        if (!r.rope.half) {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                const float a = y[2 * i], b = y[2 * i + 1];
                if (i < rotated) {
                    y[2 * i] = a * cs[i].x - b * cs[i].y;
                    y[2 * i + 1] = a * cs[i].y + b * cs[i].x;
                }
            }
        } else if (straight) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float o = __shfl_sync(0xffffffffu, y[i], partner);
                if (rotated) y[i] = upper ? o * cs[i].y + y[i] * cs[i].x : y[i] * cs[i].x - o * cs[i].y;
            }
        } else {   // halves that end inside a lane: through shared memory
            __shared__ float s_heads[kAppendThreads * E];
            const int lane = threadIdx.x & 31, half = r.rope.rope_dim / 2, v0 = lane % kLanes * E;
            float* all = s_heads + (threadIdx.x >> 5) * 32 * E;
            float* head = all + lane / kLanes * D;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < E; ++i) all[lane * E + i] = y[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (i < rotated) {
                    const bool second = v0 + i >= half;
                    const float o = head[v0 + i + (second ? -half : half)];
                    y[i] = second ? o * cs[i].y + y[i] * cs[i].x : y[i] * cs[i].x - o * cs[i].y;
                }
        }
    }
};

}  // namespace paged
}  // namespace p100b
