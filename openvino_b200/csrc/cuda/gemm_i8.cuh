// What the kernels of 8-bit whole-number products share: parameters and the epilogue's arithmetic.
//
//   out[t, n] = act((sum_k x[t, k] w[n, k] - zp[n] * sum_k x[t, k]) * x_scale[t] * w_scale[n] + bias[n]) + residual[t, n]
//
// x and w are signed bytes, zp is a byte's zero point in the same signed form. The sums are exact: with K <= kI8MaxK both terms together stay below 2^31
// (|x| <= 127, |w|, |zp| <= 128), so a sum that is split over CTAs has the same value in any order, and every kernel of this family gives the same integers for the same codes.
#pragma once
#include "gemm_common.cuh"

namespace ovb {

constexpr int kI8BlockK = 128;                      // bytes of a k-block: one 128-byte swizzle span
constexpr int kI8TileBytes = TILE_N * kI8BlockK;    // 128 weight rows of a k-block, one contiguous chunk of the packed weight
constexpr int kI8MaxK = 65536;                      // 127 * (128 + 128) * K < 2^31

struct I8Params {
    const uint8_t* w;             // packed chunks
    const float* x_scale;
    const int* x_sum;
    const float* w_scale;
    const int* w_zp;              // or NULL
    const void* bias;
    const void* residual;
    void* out;
    int* status;
    int T, N, K, KB;              // KB: k-blocks
    int ldo, ldr;
    int act, out_f32;
    float act_limit, act_slope, act_shift;
};

// Quantisation of a row y (x, or x * r * gamma with r = rsqrt(mean(x^2) + eps)):  a = max |y|;  q = round_half_even(y * (127 / a));  scale = a / 127;  sum = sum q.
// Quotients and products are rounded to 32 bits once each. With a norm z = x * gamma is quantised instead of y: r drops out of the codes and is a factor of the
// scale alone, so the sum of squares and the largest |z| come from one pass over the row (8192 rows of 4096: 28 us with two). |z| * (127 / max |z|) is at most 127 (1 + 2^-23), so no value has to
// be clamped. A row whose largest magnitude is below 2^-119, where 127 / a would not be finite, counts as zero (scale 0); one with a value that is not
// finite gets the scale NaN and codes of zero, so that every result of the row is NaN. The magnitudes are compared as integers, where NaN is the largest.
constexpr uint32_t kNotFinite = 0x7F800000u;
constexpr float kQuantFloor = 1.5046327690525280e-36f;      // 2^-119

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
// What a row is multiplied by to get its codes, 127 / max, or 0 where it has none; `r`: the norm's factor, or 1.
__device__ __forceinline__ float row_factor(uint32_t top, float r) {
    const float a = __uint_as_float(top);
    return top >= kNotFinite || a < kQuantFloor || __fmul_rn(a, r) < kQuantFloor ? 0.f : __fdiv_rn(127.f, a);
}
__device__ __forceinline__ float row_scale_of(uint32_t top, float r) {
    if (top >= kNotFinite || !(r < __int_as_float(0x7F800000))) return __int_as_float(0x7FFFFFFF);
    return row_factor(top, r) != 0.f ? __fdiv_rn(__fmul_rn(__uint_as_float(top), r), 127.f) : 0.f;
}

__host__ __device__ inline bool is_gated(int act) { return act == OVB_ACT_SWIGLU || act == OVB_ACT_GLU_LIMITED; }

// Forms of the epilogues. The code of one form is short: the uniform branches of an epilogue for all activations, which jump over long unrolled pieces, cost
// more than its arithmetic (512 x 4096 x 4096: 8100 of 31000 cycles with them).
constexpr int kI8Plain = 0;       // neither activation nor bias nor zero points
constexpr int kI8Gated = 1;       // gated, no zero points
constexpr int kI8GatedZp = 2;
constexpr int kI8Any = 3;         // not gated, all of them
constexpr bool i8_gated_form(int form) { return form == kI8Gated || form == kI8GatedZp; }
constexpr bool i8_zp_form(int form) { return form == kI8GatedZp || form == kI8Any; }
inline int i8_form(const ovb_gemm_i8_args* a) {
    if (is_gated(a->act)) return a->w_zp != nullptr ? kI8GatedZp : kI8Gated;
    return a->act == OVB_ACT_NONE && a->bias == nullptr && a->w_zp == nullptr ? kI8Plain : kI8Any;
}
// Codes of eight values, in order. 1.5 * 2^23 added to a value within +-2^22 rounds it to a whole number, halves to even, whose low byte is the sum's: the same
// as rint, without a conversion (of which an SM does 16 at a time).
__device__ __forceinline__ uint2 codes_of8(const float (&y)[8], float f) {
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(y[j], f), 12582912.f));      // (as pairs, mul.rn and add.rn come out fused)
    return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}
__device__ __forceinline__ int sum_of8(uint2 codes, int sum) { return __dp4a((int)codes.y, 0x01010101, __dp4a((int)codes.x, 0x01010101, sum)); }

// Eight values of a row: x, or x * gamma.
template <class E, bool NORM>
__device__ __forceinline__ void row_values(const uint4& x, const uint4& g, float (&v)[8]) {
    const E* e = reinterpret_cast<const E*>(&x);
    const E* w = reinterpret_cast<const E*>(&g);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        uint64_t y = pair_of(to_float(e[j]), to_float(e[j + 1]));
        if (NORM) y = mul2(y, pair_of(to_float(w[j]), to_float(w[j + 1])));
        unpair(y, v[j], v[j + 1]);
    }
}
// One pass over eight values: the largest magnitude (with a norm the bits of fp32, without one a pair of 16-bit magnitudes: see row_top) and, with a norm,
// the sum of squares of x.
template <class E, bool NORM>
__device__ __forceinline__ void row_pass(const uint4& x, const float (&v)[8], uint32_t& top, uint64_t& ss2) {
    if (NORM) {
        const E* e = reinterpret_cast<const E*>(&x);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint64_t y = pair_of(to_float(e[j]), to_float(e[j + 1]));
            ss2 = fma2(y, y, ss2);
            top = max(top, max(magnitude(v[j]), magnitude(v[j + 1])));
        }
    } else {
        constexpr uint32_t M = 0x7FFF7FFFu;
        top = __vmaxu2(top, __vmaxu2(__vmaxu2(x.x & M, x.y & M), __vmaxu2(x.z & M, x.w & M)));
    }
}
template <class E, bool NORM>
__device__ __forceinline__ uint32_t row_top(uint32_t top) {
    if (NORM) return top;
    const uint32_t half = max(top & 0xFFFFu, top >> 16);
    const uint16_t bits = (uint16_t)half;
    return magnitude(to_float(*reinterpret_cast<const E*>(&bits)));
}

// The roundings are written out, the residual's addition is __fadd_rn: left to the compiler, products and sums are fused in some kernels and paths and not in
// others, and a call's bits would go by its sizes and alignment.
template <int FORM>
__device__ __forceinline__ float i8_value(int acc, int zp, int sum, float scale, float bias) {
    const float v = float(i8_zp_form(FORM) ? acc - zp * sum : acc);
    return FORM == kI8Any ? fmaf(v, scale, bias) : __fmul_rn(v, scale);
}
// The activations of kI8Any, without branches, so that those of a thread's sixteen values overlap. 415 x 5520 x 896: SiLU with the division that IEEE wants,
// which branches at the ends of its range, 32 us, so 11.6 (9.4 without an activation); the tanh form of GELU one value after the other 39, so 12.0. The division is 2 ulp
// off, and 0 where an exponential leaves the range, as the limit is.
__device__ __forceinline__ float i8_sigmoid_of(float v, float x) { return __fdividef(v, 1.0f + __expf(-x)); }      // v / (1 + e^-x)
// tanh x = 2 / (1 + e^-2x) - 1; near 0, where that loses digits, its series (the next term is 3e-7 of the value at 1/4)
__device__ __forceinline__ float i8_tanh(float x) {
    const float x2 = x * x, near = x * fmaf(x2, fmaf(x2, fmaf(x2, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
    return x2 < 0.0625f ? near : i8_sigmoid_of(2.f, 2.f * x) - 1.f;
}
template <int N, class P>
__device__ __forceinline__ void i8_act_n(float (&v)[N], const P& p) {
    switch (p.act) {
        case OVB_ACT_NONE: break;
        case OVB_ACT_SILU:
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = i8_sigmoid_of(v[j], v[j]);
            break;
        case OVB_ACT_GELU_TANH:                         // v (1 + tanh u) / 2 = v / (1 + e^-2u), u = sqrt(2 / pi) (v + 0.044715 v^3)
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = i8_sigmoid_of(v[j], 1.5957691216f * fmaf(0.044715f * v[j] * v[j], v[j], v[j]));
            break;
        case OVB_ACT_SOFTCAP:
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = p.act_limit * i8_tanh(__fdividef(v[j], p.act_limit));
            break;
        case OVB_ACT_RELU:                              // (NaN stays in all of them: it marks a row that could not be quantised)
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];
            break;
        case OVB_ACT_RELU2:
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = v[j] < 0.f ? 0.f : v[j] * v[j];
            break;
        default: apply_act_n(v, p);                     // OVB_ACT_GELU_ERF
    }
}

template <class P>
__device__ __forceinline__ float i8_gate(const P& p, float g, float u) {
    if (p.act == OVB_ACT_SWIGLU) return i8_sigmoid_of(g, g) * u;
    g = g > p.act_limit ? p.act_limit : g;
    u = u > p.act_limit ? p.act_limit : u < -p.act_limit ? -p.act_limit : u;
    return i8_sigmoid_of(g, p.act_slope * g) * (u + p.act_shift);
}

// gemm_i8_pair.cu: many tokens, pairs of CTAs.
int gemm_i8_pair(const ovb_gemm_i8_args* a, const I8Params& p, cudaStream_t stream);

}  // namespace ovb
