// Device helpers of 8-bit rows and row statistics, shared by the kernels that make such rows (rows8.hip, heads.hip).
#pragma once

#include "clk_common.h"

namespace clk {

namespace {

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

// Rows whose scale a / 127 would leave fp32's normal range count as zeros (then 127 / a is finite too).
constexpr float kTiny = 0x1p-119f;
constexpr uint32_t kInfBits = 0x7f800000u;

// |t| as an integer that orders like it, with infinities and NaN on top: a maximum that keeps them,
// where a float maximum drops NaN
__device__ __forceinline__ uint32_t abs_bits(float t) { return __builtin_bit_cast(uint32_t, t) & 0x7fffffffu; }

// A row of largest magnitude `bits`: that as a float, what its values are multiplied by before the rounding, and its
// scale times r. A row with an infinity or NaN is zeros with scale NaN, so everything computed from it is NaN.
__device__ __forceinline__ void row_scale(uint32_t bits, float r, float& a, float& inv, float& scale) {
    a = __builtin_bit_cast(float, bits);
    if (bits >= kInfBits) {
        inv = 0.f;
        scale = __builtin_nanf("");
    } else if (a < kTiny) {
        inv = 0.f;
        scale = 0.f;
    } else {
        inv = 127.f / a;
        scale = a * r / 127.f;
    }
}

// The integer nearest to 127 t / a, ties to even, where it lies within 2^-15 of a half: t inv carries inv's rounding, 127
// 2^-24 at most, which decides there. n = t inv to the nearest, f what t inv lies past it. Of 127 t - m a, m the
// half, the sign counts: 127 t is taken in two parts, m a has to be rounded nowhere (fma), and what is left of
// the two is a multiple of a's last bit too small to be rounded. Rows of huge values are taken times 2^-64 for it.
__device__ __forceinline__ int settle_half(float t, float a, float n, float f) {
    const float s = a > 0x1p100f ? 0x1p-64f : 1.f, ts = t * s;
    const float hi = 127.f * ts, lo = __builtin_fmaf(127.f, ts, -hi);
    const float e = __builtin_fmaf(-(n + __builtin_copysignf(0.5f, f)), a * s, hi) + lo;
    const int below = (int)n - (f < 0.f);
    return below + (e > 0.f || (e == 0.f && (below & 1)));
}
constexpr float kNearHalf = 0.5f - 0x1p-15f;

// The low bytes of four registers
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}

// 1 / sqrt(ss / C + eps) from a row's sum of squares
__device__ __forceinline__ float inv_rms(float ss, float inv_c, float eps) { return 1.f / sqrtf(ss * inv_c + eps); }

// A bf16 row with values past 2^40 has sums of squares, or products with w, past fp32's range; one of
// values below 2^-40 has them below it, which counts where eps is next to nothing. Such a row is taken
// with its values times a power of two (so every product stays what it was) and eps times its square.
__device__ __forceinline__ float row_shift(uint32_t bits, float eps) {
    if (bits >= kInfBits) return 1.f;
    const float a = __builtin_bit_cast(float, bits);
    return a >= 0x1p40f ? 0x1p-90f : a < 0x1p-40f && eps < 0x1p-100f ? 0x1p90f : 1.f;
}

// Whether a row taken times d is turned to 8 bits from its values as they are: huge ones whose products with w, of largest
// magnitude `bits` as they were taken, would lose low bits (or, under 2^-119, the row) by that. Those products
// are under 1 without d, and the scale is multiplied by d in the end.
__device__ __forceinline__ bool as_they_are(float d, uint32_t bits) {
    return d < 1.f && __builtin_bit_cast(float, bits) < 0x1p-90f;
}

// v of the lane that DPP control CTRL names
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
struct Sum {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }
};
struct Max {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
};

// op over each aligned group of W lanes (1 to 64), in every lane of it: by DPP within 16 lanes (pairs, quads,
// mirrored halves), then by swaps of 16- and 32-lane rows. Both lanes of a step take the same two
// values, so all lanes end with the same bits.
template <int W, typename Op>
__device__ __forceinline__ uint32_t lanes_all(uint32_t v, Op op) {
    if constexpr (W >= 2) v = op(v, dpp<0xB1>(v));   // quad_perm [1,0,3,2]
    if constexpr (W >= 4) v = op(v, dpp<0x4E>(v));   // quad_perm [2,3,0,1]
    if constexpr (W >= 8) v = op(v, dpp<0x141>(v));  // row_half_mirror
    if constexpr (W >= 16) v = op(v, dpp<0x140>(v));  // row_mirror
    if constexpr (W >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = op(s[0], s[1]);
    }
    if constexpr (W >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = op(s[0], s[1]);
    }
    return v;
}
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
    return __builtin_bit_cast(float, lanes_all<W>(__builtin_bit_cast(uint32_t, v), Sum()));
}
template <int W>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) { return lanes_all<W>(v, Max()); }

// 8 values of a row of largest magnitude a, inv = 127 / a, as the integers nearest to 127 t / a, ties to even. |t| <= a
// bounds them by 127, and the sum of one with 1.5 2^23 is rounded to integers and has them in its low byte.
// inv = 0 (a row of zeros) gives 0 also for a t that is not finite.
//
// Values and a of 16 bits (IN16): 127 t / a lies on a half or, t being 2^i times an integer T < 2^11, at least 1 / (254
// T) > 2^-19 of itself away from it, so the quotient rounded to fp32 (t inv, and t times what inv lacks, in one
// fma) is on the same side, or on the half.
// Other values: what may lie at a half is looked at again, one value in 16000 where they are spread. Half of a,
// which values made of 16-bit ones hit far more often, is 63.5, so 64. (The norm of [4099, 5120] bf16 with weights
// of 1 takes 28 us; 31 with that half settled like the others, 26.5 with halves as t inv has them.)
template <bool IN16>
__device__ __forceinline__ uint2v quant8(const float (&t)[8], float a, float inv) {
    constexpr float kUnits = 0x1.8p23f;
    uint32_t q[8];
    if constexpr (IN16) {
        const float lacks = __builtin_fmaf(-inv, a, 127.f) * inv * (1.f / 127.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            q[e] = __builtin_bit_cast(uint32_t, __builtin_fmaf(t[e], inv, t[e] * lacks) + kUnits);
        }
    } else {
        uint64_t near[8], any = 0;  // the lanes whose value e may lie at a half
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float r = __builtin_fmaf(t[e], inv, kUnits);
            q[e] = __builtin_bit_cast(uint32_t, r);
            near[e] = __ballot(fabsf(__builtin_fmaf(t[e], inv, kUnits - r)) > kNearHalf);
            any |= near[e];
        }
        if (any != 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (near[e] == 0) continue;
                const uint64_t half = __ballot(fabsf(t[e]) == 0.5f * a);
                if ((near[e] & ~half) != 0) {
                    const float n = __builtin_bit_cast(float, q[e]) - kUnits;
                    const float f = __builtin_fmaf(t[e], inv, -n);
                    const uint32_t settled = (uint32_t)settle_half(t[e], a, n, f);
                    q[e] = fabsf(f) > kNearHalf ? settled : q[e];
                }
                if (fabsf(t[e]) == 0.5f * a) q[e] = t[e] < 0.f ? (uint32_t)-64 : 64u;
            }
        }
    }
    const uint2v words{pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7])};
    return inv == 0.f ? uint2v{0, 0} : words;
}

}  // namespace

}  // namespace clk
