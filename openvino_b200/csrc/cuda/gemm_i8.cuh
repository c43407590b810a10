// What the kernels of 8-bit whole-number products share: parameters and the epilogue's arithmetic.
//
//   out[t, n] = act((sum_k x[t, k] w[n, k] - zp[n] * sum_k x[t, k]) * x_scale[t] * w_scale[n] + bias[n]) + residual[t, n]
//
// x and w are signed bytes, zp is a byte's zero point in the same signed form. The sums are exact: with K <= kI8MaxK both terms together stay below 2^31
// (|x| <= 127, |w|, |zp| <= 128), so a sum that is split over CTAs has the same value in any order, and every kernel of this family gives the same integers.
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

__device__ __forceinline__ float i8_value(int acc, int zp, int sum, float scale) { return float(acc - zp * sum) * scale; }
__device__ __forceinline__ bool is_gated(int act) { return act == OVB_ACT_SWIGLU || act == OVB_ACT_GLU_LIMITED; }

// gemm_i8_pair.cu: many tokens, pairs of CTAs.
int gemm_i8_pair(const ovb_gemm_i8_args* a, const I8Params& p, cudaStream_t stream);

}  // namespace ovb
