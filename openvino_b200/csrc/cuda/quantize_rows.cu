// Rows of 16-bit values -> signed bytes with one scale per row, the RMS norm of the row on the way where there is one.
//
// The arithmetic is in gemm_i8.cuh; the norm's sums are held in 32 bits.
//
// What bounds it: memory, three bytes per value (two of them usually from L2). A row stays in registers between the passes: every thread holds HOLD
// pieces of eight columns.
#include "gemm_i8.cuh"

namespace ovb {

struct QuantParams {
    const void* x;
    const void* gamma;            // or NULL
    const int* row_idx;           // or NULL: rows 0 .. rows
    uint8_t* q;
    float* scale;
    int* sum;
    int rows, cols, x_rows;
    int64_t ldx;
    int ldq;
    float eps;
};

constexpr int kManyRows = 1024;

// The sum (largest) over the warps that share a row; every thread gets it.
template <int WPR, class T, class F>
__device__ __forceinline__ T over_row(T v, T* box, F&& f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (WPR == 1) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) box[warp] = v;
    __syncthreads();
    v = box[lane % WPR];
#pragma unroll
    for (int o = WPR / 2; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ void row_result(const QuantParams& p, int row, uint32_t top, int sum) {
    p.scale[row] = row_scale_of(top);
    p.sum[row] = sum;
}

__device__ __forceinline__ int source_row(const QuantParams& p, int row) {
    if (p.row_idx == nullptr) return row;
    const int r = p.row_idx[row];
    return r < 0 || r >= p.x_rows ? 0 : r;
}

// Rows of whole, aligned pieces of eight columns. WPR warps share a row; blocks of max(4, WPR) warps.
template <class E, bool NORM, int WPR, int HOLD>
__global__ void __launch_bounds__(WPR < 4 ? 128 : WPR * 32) quantize_rows_kernel(const QuantParams p) {
    constexpr int RPB = WPR < 4 ? 4 / WPR : 1, SPAN = WPR * 32;
    __shared__ float box_f[16];
    __shared__ uint32_t box_u[16];
    __shared__ int box_i[16];
    const int row = blockIdx.x * RPB + (RPB > 1 ? (int)threadIdx.x / SPAN : 0), at = threadIdx.x % SPAN;
    const int pieces = p.cols >> 3;
    pdl_enter();
    if (row >= p.rows) return;              // whole warps, and only where rows do not share a block's barriers
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const E*>(p.x) + (size_t)source_row(p, row) * p.ldx);
    const uint4* gamma = static_cast<const uint4*>(p.gamma);
    constexpr bool HELD = NORM && HOLD <= 4;            // with more pieces the weights do not fit the registers beside the row: they are read again
    uint4 x[HOLD], g[HELD ? HOLD : 1];
#pragma unroll
    for (int h = 0; h < HOLD; ++h) x[h] = at + h * SPAN < pieces ? __ldcg(src + at + h * SPAN) : make_uint4(0, 0, 0, 0);
    if (HELD) {
#pragma unroll
        for (int h = 0; h < HOLD; ++h)
            if (at + h * SPAN < pieces) g[h] = __ldg(gamma + at + h * SPAN);
    }
    float inv = 1.f;
    if (NORM) {
        uint64_t ss2 = pair_of(0.f);
#pragma unroll
        for (int h = 0; h < HOLD; ++h) {
            float v[8];
            row_values<E, false>(x[h], x[h], 1.f, v);
#pragma unroll
            for (int j = 0; j < 8; j += 2) ss2 = fma2(pair_of(v[j], v[j + 1]), pair_of(v[j], v[j + 1]), ss2);
        }
        float ss, ss1;
        unpair(ss2, ss, ss1);
        ss = over_row<WPR>(ss + ss1, box_f, [](float a, float b) { return a + b; });
        inv = rsqrtf(ss / (float)p.cols + p.eps);
    }
    auto weights = [&](int h) {
        if (NORM && !HELD) g[0] = __ldg(gamma + at + h * SPAN);
    };
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (at + h * SPAN < pieces) {
            weights(h);
            top = top_of8<E, NORM>(x[h], g[HELD ? h : 0], inv, top);
        }
    top = over_row<WPR>(row_top<E, NORM>(top), box_u, [](uint32_t a, uint32_t b) { return max(a, b); });
    const float f = row_factor(top);
    uint2* dst = reinterpret_cast<uint2*>(p.q + (size_t)row * p.ldq);
    int sum = 0;
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (at + h * SPAN < pieces) {
            float v[8];
            weights(h);
            row_values<E, NORM>(x[h], g[HELD ? h : 0], inv, v);
            const uint2 w = f != 0.f ? codes_of8(v, f) : make_uint2(0, 0);
            sum = sum_of8(w, sum);
            dst[at + h * SPAN] = w;
        }
    sum = over_row<WPR>(sum, box_i, [](int a, int b) { return a + b; });
    if (at == 0) row_result(p, row, top, sum);
}

// Any width, pitch and alignment: a block per row, which is read once for each pass.
template <class E>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const QuantParams p) {
    __shared__ float box_f[16];
    __shared__ uint32_t box_u[16];
    __shared__ int box_i[16];
    pdl_enter();
    const int row = blockIdx.x;
    const E* src = static_cast<const E*>(p.x) + (size_t)source_row(p, row) * p.ldx;
    const E* gamma = static_cast<const E*>(p.gamma);
    float inv = 1.f;
    if (gamma != nullptr) {
        float ss = 0.f;
        for (int k = threadIdx.x; k < p.cols; k += 256) ss = fmaf(to_float(src[k]), to_float(src[k]), ss);
        ss = over_row<8>(ss, box_f, [](float a, float b) { return a + b; });
        inv = rsqrtf(ss / (float)p.cols + p.eps);
    }
    auto value = [&](int k) { return gamma != nullptr ? to_float(src[k]) * inv * to_float(gamma[k]) : to_float(src[k]); };
    uint32_t top = 0;
    for (int k = threadIdx.x; k < p.cols; k += 256) top = max(top, magnitude(value(k)));
    top = over_row<8>(top, box_u, [](uint32_t a, uint32_t b) { return max(a, b); });
    const float f = row_factor(top);
    int sum = 0;
    for (int k = threadIdx.x; k < p.cols; k += 256) {
        const int c = f != 0.f ? __float2int_rn(__fmul_rn(value(k), f)) : 0;
        sum += c;
        p.q[(size_t)row * p.ldq + k] = (uint8_t)(c & 0xFF);
    }
    sum = over_row<8>(sum, box_i, [](int a, int b) { return a + b; });
    if (threadIdx.x == 0) row_result(p, row, top, sum);
}

template <class E, bool NORM>
static cudaError_t run_quantize(const QuantParams& p, cudaStream_t stream) {
    const bool whole = p.cols % 8 == 0 && p.ldx % 8 == 0 && p.ldq % 8 == 0 &&
                       ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.gamma)) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.q) & 7) == 0;
    if (!whole || p.cols > 32768) return launch_pdl(quantize_rows_any_kernel<E>, dim3(p.rows), dim3(256), 0, stream, p);
    auto go = [&](auto kern, int wpr) { return launch_pdl(kern, dim3(wpr < 4 ? (p.rows + 4 / wpr - 1) / (4 / wpr) : p.rows), dim3(wpr < 4 ? 128 : wpr * 32), 0, stream, p); };
    // Many rows: few warps to a row, with more of it each (from so many on that they fill the machine); few rows: many warps, for the time of one row.
    const bool many = p.rows >= kManyRows;
    if (p.cols <= 512) return go(quantize_rows_kernel<E, NORM, 1, 2>, 1);
    if (p.cols <= 1024) return go(quantize_rows_kernel<E, NORM, 1, 4>, 1);
    if (p.cols <= 2048) return many ? go(quantize_rows_kernel<E, NORM, 1, 8>, 1) : go(quantize_rows_kernel<E, NORM, 8, 1>, 8);
    if (p.cols <= 4096) return many ? go(quantize_rows_kernel<E, NORM, 4, 4>, 4) : go(quantize_rows_kernel<E, NORM, 8, 2>, 8);
    if (p.cols <= 8192) return many ? go(quantize_rows_kernel<E, NORM, 4, 8>, 4) : go(quantize_rows_kernel<E, NORM, 16, 2>, 16);
    if (p.cols <= 16384) return many ? go(quantize_rows_kernel<E, NORM, 8, 8>, 8) : go(quantize_rows_kernel<E, NORM, 16, 4>, 16);
    return go(quantize_rows_kernel<E, NORM, 16, 8>, 16);
}

}  // namespace ovb

extern "C" int ovb_quantize_rows(const ovb_quant_rows_args* a, ovb_stream_t stream_) {
    using namespace ovb;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    OVB_REQUIRE(a && a->x && a->q && a->scale && a->sum, "ovb_quantize_rows: null operand");
    OVB_REQUIRE(a->rows > 0 && a->cols > 0 && a->ldq >= a->cols && a->ldx >= 0, "ovb_quantize_rows: %d rows of %d columns, pitches %lld and %d", a->rows, a->cols,
                (long long)a->ldx, a->ldq);
    OVB_REQUIRE(a->row_idx == nullptr || a->x_rows > 0, "ovb_quantize_rows: row indices need the number of rows of x");
    QuantParams p;
    p.x = a->x;
    p.gamma = a->gamma;
    p.row_idx = a->row_idx;
    p.q = static_cast<uint8_t*>(a->q);
    p.scale = a->scale;
    p.sum = a->sum;
    p.rows = a->rows;
    p.cols = a->cols;
    p.x_rows = a->x_rows;
    p.ldx = a->ldx;
    p.ldq = a->ldq;
    p.eps = a->eps;
    const cudaError_t e = a->gamma != nullptr ? (a->f16 ? run_quantize<__half, true>(p, stream) : run_quantize<__nv_bfloat16, true>(p, stream))
                                              : (a->f16 ? run_quantize<__half, false>(p, stream) : run_quantize<__nv_bfloat16, false>(p, stream));
    OVB_CHECK_CUDA(e);
    return 0;
}
