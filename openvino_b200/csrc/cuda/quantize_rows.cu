// Rows of 16-bit values -> signed bytes with one scale per row, the RMS norm of the row on the way where there is one.
//
// The arithmetic is in gemm_i8.cuh; the norm's sums are held in 32 bits.
//
// What bounds it: memory, three bytes per value (two of them usually from L2). A row is read once and stays in registers until its largest magnitude is known:
// every thread holds HOLD pieces of eight columns, as they came or, with a norm, times the weights. Measured without and with a norm: 8192 x 4096 16.4 and
// 21.2 us, 8192 x 8192 29.7 and 43.7 us (6.8 and 4.6 TB/s; with a norm the instructions, 16 for a value, fill three quarters of the issue slots), 64 x 4096
// 1.8 and 2.0 us, of which most is the launch. Rows that do not lie in whole aligned pieces: 999 x 1333 3.5 and 3.9 us, 8192 x 500 5.5 and 7.5, 8192 x 4097
// 38 and 51 (value by value, in a block per row: 4.6 and 5.6, 17.9 and 21.3, 36 and 46).
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

// From so many rows on, a row gets few warps with more of it each, which are enough to fill the machine and spend less on meeting; below it many warps, for the
// time of one row. 600 rows, many warps and few: 2.9 and 2.3 us (2048 columns), 3.9 and 3.3 (4096), 5.2 and 4.5 (8192); 400 rows: 2.0 and 2.1, 2.5 and 2.5,
// 4.3 and 3.9; 8192 rows of 4096: 20.3 and 16.4.
constexpr int kManyRows = 512;

// f over the warps that share a row; every thread gets it.
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
// The sum of s and the largest t, one barrier for both.
template <int WPR>
__device__ __forceinline__ void over_row(float& s, uint32_t& t, float* box_s, uint32_t* box_t) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
    }
    if (WPR == 1) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
        box_s[warp] = s;
        box_t[warp] = t;
    }
    __syncthreads();
    s = box_s[lane % WPR];
    t = box_t[lane % WPR];
#pragma unroll
    for (int o = WPR / 2; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
    }
}

__device__ __forceinline__ void row_result(const QuantParams& p, int row, uint32_t top, float r, int sum) {
    p.scale[row] = row_scale_of(top, r);
    p.sum[row] = sum;
}

__device__ __forceinline__ int source_row(const QuantParams& p, int row) {
    if (p.row_idx == nullptr) return row;
    const int r = p.row_idx[row];
    return r < 0 || r >= p.x_rows ? 0 : r;
}

// The pieces at, at + SPAN, .. of a row at any place and of any width, zero behind its end. Loads are of the aligned 16-byte blocks that hold a byte of the row (an
// allocation that holds one byte of such a block holds it whole); a piece is shifted out of its block and the next, which the neighbouring lane holds.
template <class E, int HOLD, int SPAN>
__device__ __forceinline__ void load_pieces(const E* row, int cols, int at, uint4 (&x)[HOLD]) {
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15), lane = threadIdx.x & 31, blocks = (off + cols * 2 + 15) >> 4;
    const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(row) - off);
#pragma unroll
    for (int h = 0; h < HOLD; ++h) x[h] = at + h * SPAN < blocks ? __ldcg(from + at + h * SPAN) : make_uint4(0, 0, 0, 0);
    if (off != 0) {                         // the same for the warp
        uint4 behind[HOLD];
#pragma unroll
        for (int h = 0; h < HOLD; ++h) behind[h] = lane == 31 && at + h * SPAN + 1 < blocks ? __ldcg(from + at + h * SPAN + 1) : make_uint4(0, 0, 0, 0);
        const bool two = off & 8, one = off & 4;
        const int bits = (off & 2) * 8;
#pragma unroll
        for (int h = 0; h < HOLD; ++h) {
            uint32_t w[8] = {x[h].x, x[h].y, x[h].z, x[h].w, behind[h].x, behind[h].y, behind[h].z, behind[h].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t next = __shfl_down_sync(0xffffffffu, w[j], 1);
                if (lane != 31) w[4 + j] = next;
            }
#pragma unroll
            for (int j = 0; j < 6; ++j) w[j] = two ? w[j + 2] : w[j];
#pragma unroll
            for (int j = 0; j < 5; ++j) w[j] = one ? w[j + 1] : w[j];
            x[h] = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
        }
    }
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        const int left = cols - 8 * (at + h * SPAN);
        auto keep = [&](int j) { return left >= 2 * j + 2 ? 0xFFFFFFFFu : left == 2 * j + 1 ? 0xFFFFu : 0u; };
        x[h] = make_uint4(x[h].x & keep(0), x[h].y & keep(1), x[h].z & keep(2), x[h].w & keep(3));
    }
}

// Rows in pieces of eight columns, whole and aligned ones or (SHIFT) of any place and width. WPR warps share a row; blocks of max(4, WPR) warps.
template <class E, bool NORM, int WPR, int HOLD, bool SHIFT>
__global__ void __launch_bounds__(WPR < 4 ? 128 : WPR * 32) quantize_rows_kernel(const QuantParams p) {
    constexpr int RPB = WPR < 4 ? 4 / WPR : 1, SPAN = WPR * 32;
    __shared__ float box_f[16];
    __shared__ uint32_t box_u[16];
    __shared__ int box_i[16];
    const int row = blockIdx.x * RPB + (RPB > 1 ? (int)threadIdx.x / SPAN : 0), at = threadIdx.x % SPAN;
    const int pieces = SHIFT ? (p.cols + 7) >> 3 : p.cols >> 3;
    pdl_enter();
    if (row >= p.rows) return;              // whole warps, and only where rows do not share a block's barriers
    const E* line = static_cast<const E*>(p.x) + (size_t)source_row(p, row) * p.ldx;
    const uint4* src = reinterpret_cast<const uint4*>(line);
    const uint4* gamma = static_cast<const uint4*>(p.gamma);
    uint4 x[HOLD], g[NORM ? HOLD : 1];
    if (SHIFT) {
        load_pieces<E, HOLD, SPAN>(line, p.cols, at, x);
        if (NORM) load_pieces<E, NORM ? HOLD : 1, SPAN>(static_cast<const E*>(p.gamma), p.cols, at, g);
    } else {
#pragma unroll
        for (int h = 0; h < HOLD; ++h) {
            const bool in = at + h * SPAN < pieces;
            x[h] = in ? __ldcg(src + at + h * SPAN) : make_uint4(0, 0, 0, 0);
            if (NORM) g[h] = in ? __ldg(gamma + at + h * SPAN) : make_uint4(0, 0, 0, 0);
        }
    }
    uint32_t top = 0;
    uint64_t ss2 = pair_of(0.f);
    float v[NORM ? HOLD : 1][8];
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (NORM) row_values<E, NORM>(x[h], g[h % (NORM ? HOLD : 1)], v[h % (NORM ? HOLD : 1)]);
        row_pass<E, NORM>(x[h], v[h % (NORM ? HOLD : 1)], top, ss2);
    }
    float r = 1.f;
    top = row_top<E, NORM>(top);
    if (NORM) {
        float ss, ss1;
        unpair(ss2, ss, ss1);
        ss += ss1;
        over_row<WPR>(ss, top, box_f, box_u);
        r = rsqrtf(ss / (float)p.cols + p.eps);
    } else {
        top = over_row<WPR>(top, box_u, [](uint32_t a, uint32_t b) { return max(a, b); });
    }
    const float f = row_factor(top, r);
    uint2* dst = reinterpret_cast<uint2*>(p.q + (size_t)row * p.ldq);
    int sum = 0;
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (at + h * SPAN < pieces) {
            float (&y)[8] = v[h % (NORM ? HOLD : 1)];
            if (!NORM) row_values<E, NORM>(x[h], x[h], y);
            const uint2 w = f != 0.f ? codes_of8(y, f) : make_uint2(0, 0);
            sum = sum_of8(w, sum);
            if (!SHIFT || (at + h * SPAN) * 8 + 8 <= p.cols) {
                dst[at + h * SPAN] = w;
            } else {
                for (int j = 0; j < p.cols % 8; ++j) reinterpret_cast<uint8_t*>(dst + at + h * SPAN)[j] = (uint8_t)((j < 4 ? w.x >> (8 * j) : w.y >> (8 * (j - 4))) & 0xFF);
            }
        }
    sum = over_row<WPR>(sum, box_i, [](int a, int b) { return a + b; });
    if (at == 0) row_result(p, row, top, r, sum);
}

// More columns, or codes at any place: a block per row, which is read once for each pass.
template <class E>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const QuantParams p) {
    __shared__ float box_f[16];
    __shared__ uint32_t box_u[16];
    __shared__ int box_i[16];
    pdl_enter();
    const int row = blockIdx.x;
    const E* src = static_cast<const E*>(p.x) + (size_t)source_row(p, row) * p.ldx;
    const E* gamma = static_cast<const E*>(p.gamma);
    auto value = [&](int k) { return gamma != nullptr ? __fmul_rn(to_float(src[k]), to_float(gamma[k])) : to_float(src[k]); };
    float ss = 0.f, r = 1.f;
    uint32_t top = 0;
    for (int k = threadIdx.x; k < p.cols; k += 256) {
        ss = fmaf(to_float(src[k]), to_float(src[k]), ss);
        top = max(top, magnitude(value(k)));
    }
    over_row<8>(ss, top, box_f, box_u);
    if (gamma != nullptr) r = rsqrtf(ss / (float)p.cols + p.eps);
    const float f = row_factor(top, r);
    int sum = 0;
    for (int k = threadIdx.x; k < p.cols; k += 256) {
        const int c = f != 0.f ? __float2int_rn(__fmul_rn(value(k), f)) : 0;
        sum += c;
        p.q[(size_t)row * p.ldq + k] = (uint8_t)(c & 0xFF);
    }
    sum = over_row<8>(sum, box_i, [](int a, int b) { return a + b; });
    if (threadIdx.x == 0) row_result(p, row, top, r, sum);
}

template <class E, bool NORM, bool SHIFT>
static cudaError_t run_quantize(const QuantParams& p, cudaStream_t stream) {
    auto go = [&](auto kern, int wpr) { return launch_pdl(kern, dim3(wpr < 4 ? (p.rows + 4 / wpr - 1) / (4 / wpr) : p.rows), dim3(wpr < 4 ? 128 : wpr * 32), 0, stream, p); };
    const bool many = p.rows >= kManyRows;
    if (p.cols <= 512) return go(quantize_rows_kernel<E, NORM, 1, 2, SHIFT>, 1);
    if (p.cols <= 1024) return go(quantize_rows_kernel<E, NORM, 1, 4, SHIFT>, 1);
    if (p.cols <= 2048) return many ? go(quantize_rows_kernel<E, NORM, 1, 8, SHIFT>, 1) : go(quantize_rows_kernel<E, NORM, 8, 1, SHIFT>, 8);
    if (p.cols <= 4096) return many ? go(quantize_rows_kernel<E, NORM, 4, 4, SHIFT>, 4) : go(quantize_rows_kernel<E, NORM, 8, 2, SHIFT>, 8);
    if (p.cols <= 8192) return many ? go(quantize_rows_kernel<E, NORM, 4, 8, SHIFT>, 4) : go(quantize_rows_kernel<E, NORM, 16, 2, SHIFT>, 16);
    // with a norm eight pieces take too many registers here: 1024 rows of 14336 in 13.9 us, in 12.9 with four
    if (p.cols <= 16384) return many && !NORM ? go(quantize_rows_kernel<E, false, 8, 8, SHIFT>, 8) : go(quantize_rows_kernel<E, NORM, 16, 4, SHIFT>, 16);
    return go(quantize_rows_kernel<E, NORM, 16, 8, SHIFT>, 16);
}
template <class E, bool NORM>
static cudaError_t run_quantize(const QuantParams& p, cudaStream_t stream) {
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    if (p.cols > 32768 || p.ldq % 8 != 0 || (bits(p.q) & 7) != 0 || ((bits(p.x) | bits(p.gamma)) & 1) != 0)
        return launch_pdl(quantize_rows_any_kernel<E>, dim3(p.rows), dim3(256), 0, stream, p);
    const bool whole = p.cols % 8 == 0 && p.ldx % 8 == 0 && ((bits(p.x) | bits(p.gamma)) & 15) == 0;
    return whole ? run_quantize<E, NORM, false>(p, stream) : run_quantize<E, NORM, true>(p, stream);
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
