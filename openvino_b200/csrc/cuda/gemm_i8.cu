// Products of signed bytes on the tensor cores (tcgen05, kind::i8, 32-bit integer sums in tensor memory): the entry point, the weights' packing and
// the kernel of few tokens.
//
// The kernel: a CTA works on 128 weight rows (the M side) and up to 256 tokens (N); where that leaves SMs without work the k-blocks of a tile are
// shared by a cluster of up to eight CTAs. Nothing has to be expanded, so a stage is one bulk copy of a 16 KB weight chunk, packed in the swizzled
// order that the MMA reads, and one TMA box of tokens; rows behind the last token and columns behind K come as zeros. Weights are fetched before
// the kernel that wrote the tokens has finished. The partial sums are integers: they go to shared memory as [token][channel], every CTA of the cluster
// adds up its share of the tokens over all partials and finishes them, lanes along the channels.
//
// What bounds it: the weights' way from memory, 1 x 6144 x 4096 6.9 us (3.7 TB/s with its start-up of about 3), 1 x 4096 x 11008 10.8 us, 7 x 4096 x 14336 11.8 us (5.0), 64 x 28672 x 4096
// 21.5 us (5.5), 128256 x 4096 for one token 76.7 us (6.85); with some hundred tokens the rate at which MMAs are issued, 65 cycles each with 128 rows.
#include <atomic>
#include <type_traits>

#include "gemm_i8.cuh"

namespace ovb {

constexpr int kI8MaxStages = 12;
constexpr int kI8QuantWarps = 8;
constexpr int kI8Hold = 8;                          // pieces of eight columns of the row that a quantising thread holds
constexpr int i8_threads(bool fused) { return fused ? 64 + kI8QuantWarps * 32 : 256; }
constexpr int kI8FusedBlock = 16 * kI8BlockK;       // a k-block of the codes

struct I8TileParams : I8Params {
    int bt, stages, splits;
    int whole;                    // 16-bit results and residuals in groups of four aligned columns
    // quantisation in the kernel
    const void* raw;
    const void* gamma;
    const int* row_idx;
    int64_t ld_raw;
    int raw_rows;
    float eps;
};

// The row of a single token, quantised by eight warps into the swizzled operand of the MMA ([k-block][16 rows][128 bytes]; the other rows are not set,
// their sums are not read). Every CTA needs the largest magnitude of the whole row, so it reads it whole, and keeps the codes of its k-blocks. The loops stop
// behind the last piece in use: with all eight worked through whatever K is, the arithmetic of empty pieces took more than the row's own (1 x 6144 x 4096 with
// a norm 13.2 us, 7.0 without them).
template <class E>
__device__ __forceinline__ void i8_quantize_row(const I8TileParams& p, uint8_t* codes, int kb0, int kb1, float* row_scale, int* row_sum, float* box_f, uint32_t* box_u, int* box_i) {
    constexpr int SPAN = kI8QuantWarps * 32;
    const int tid = threadIdx.x - 64, warp = tid >> 5, lane = tid & 31, pieces = p.K >> 3;
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(SPAN) : "memory"); };
    uint4 x[kI8Hold], g[kI8Hold];
    int row = 0;
    if (p.row_idx != nullptr) {
        row = p.row_idx[0];
        if (row < 0 || row >= p.raw_rows) row = 0;
    }
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const E*>(p.raw) + row * p.ld_raw);
#pragma unroll
    for (int h = 0; h < kI8Hold; ++h) {
        if (h * SPAN >= pieces) break;
        const int at = tid + h * SPAN;
        x[h] = at < pieces ? __ldcg(src + at) : make_uint4(0, 0, 0, 0);
        g[h] = p.gamma != nullptr && at < pieces ? __ldg(static_cast<const uint4*>(p.gamma) + at) : make_uint4(0, 0, 0, 0);
    }
    // The sum of squares has the order of ovb_quantize_rows for few rows of 1025 to 4096 columns. Narrower and wider rows are shared by other numbers of warps there: the
    // codes are the same, the norm's factor and with it the row's scale may differ in their last bits.
    const bool norm = p.gamma != nullptr;
    uint32_t top = 0;
    uint64_t ss2 = pair_of(0.f);
#pragma unroll
    for (int h = 0; h < kI8Hold; ++h) {
        if (h * SPAN >= pieces) break;
        float v[8];
        if (norm) {
            row_values<E, true>(x[h], g[h], v);
            row_pass<E, true>(x[h], v, top, ss2);
        } else {
            row_pass<E, false>(x[h], v, top, ss2);
        }
    }
    float ss, ss1;
    unpair(ss2, ss, ss1);
    ss += ss1;
    top = norm ? top : row_top<E, false>(top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (lane == 0) {
        box_f[warp] = ss;
        box_u[warp] = top;
    }
    meet();
    ss = box_f[lane % kI8QuantWarps];
    top = box_u[lane % kI8QuantWarps];
#pragma unroll
    for (int o = kI8QuantWarps / 2; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const float r = norm ? rsqrtf(ss / (float)p.K + p.eps) : 1.f, f = row_factor(top, r);
    int sum = 0;
#pragma unroll
    for (int h = 0; h < kI8Hold; ++h) {
        if (h * SPAN >= pieces) break;
        const int at = tid + h * SPAN, kb = at >> 4;
        const bool mine = kb >= kb0 && kb < kb1;
        if (at >= pieces || (!mine && p.w_zp == nullptr)) continue;
        float v[8];
        if (norm) row_values<E, true>(x[h], g[h], v);
        else row_values<E, false>(x[h], x[h], v);
        const uint2 w = f != 0.f ? codes_of8(v, f) : make_uint2(0, 0);
        sum = sum_of8(w, sum);
        if (mine) *reinterpret_cast<uint2*>(codes + (kb - kb0) * kI8FusedBlock + ((at & 15) << 3)) = w;      // row 0 of the swizzle: in order
    }
    if (p.w_zp != nullptr) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) box_i[warp] = sum;
    }
    fence_proxy_async_smem();                           // the codes are read by the tensor cores
    meet();
    if (tid == 0) {
        *row_scale = row_scale_of(top, r);
        sum = 0;
        if (p.w_zp != nullptr)
            for (int w = 0; w < kI8QuantWarps; ++w) sum += box_i[w];
        *row_sum = sum;
    }
}

template <bool F16, bool FUSED, int FORM>
__global__ void __launch_bounds__(i8_threads(FUSED)) gemm_i8_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ I8TileParams p) {
    using E = typename Elem<F16>::type;
    constexpr int WARPS = i8_threads(FUSED) / 32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[kI8MaxStages], empty[kI8MaxStages], done, rows_ready;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ float row_scale[FUSED ? 1 : 256];
    __shared__ int row_sum[FUSED ? 1 : 256];
    volatile int* abort_flag = &abort_word;

    // the shuffle tells the compiler that a warp's index is the same in all lanes: the MMA loop below then runs on uniform registers
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;      // a cluster is the splits of one tile
    const int n0 = tile * TILE_N, t0 = blockIdx.y * p.bt;
    const int kb0 = (int)((int64_t)p.KB * split / p.splits), kb1 = (int)((int64_t)p.KB * (split + 1) / p.splits);
    const int stage_bytes = kI8TileBytes + (FUSED ? 0 : p.bt * kI8BlockK);
    // fused: the row's codes come first. The partial sums take the stages' place and are read by the other CTAs at this CTA's own offset, so room is left for the
    // largest share of the cluster, whichever this one is.
    uint8_t* stages = FUSED ? smem + (p.KB + p.splits - 1) / p.splits * kI8FusedBlock : smem;
    const uint32_t tmem_cols = p.bt <= 32 ? 32u : p.bt <= 64 ? 64u : p.bt <= 128 ? 128u : 256u;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        mbar_init(&rows_ready, 1);
        abort_word = 0;
        mbar_fence_init();
        if (!FUSED) tma_prefetch_desc(&tmX);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            const uint8_t* w = p.w + ((size_t)tile * p.KB + kb0) * kI8TileBytes;
            const int n = kb1 - kb0, ahead = n < p.stages ? n : p.stages;
            for (int i = 0; i < ahead; ++i) {           // weights are constants: they come before the tokens may be read
                mbar_arrive_expect_tx(&full[i], (uint32_t)stage_bytes);
                bulk_load_1d(stages + i * stage_bytes, w + (size_t)i * kI8TileBytes, kI8TileBytes, &full[i]);
            }
            if (!FUSED) {
                pdl_wait();
                for (int i = 0; i < ahead; ++i) tma_load_2d(stages + i * stage_bytes + kI8TileBytes, &tmX, &full[i], (kb0 + i) * kI8BlockK, t0);
            }
            int s = 0;
            uint32_t phase = 0;
            for (int i = ahead; i < n; ++i) {
                if (!mbar_wait(&empty[s], phase, abort_flag, p.status)) break;
                mbar_arrive_expect_tx(&full[s], (uint32_t)stage_bytes);
                bulk_load_1d(stages + s * stage_bytes, w + (size_t)i * kI8TileBytes, kI8TileBytes, &full[s]);
                if (!FUSED) tma_load_2d(stages + s * stage_bytes + kI8TileBytes, &tmX, &full[s], (kb0 + i) * kI8BlockK, t0);
                if (++s == p.stages) { s = 0; phase ^= 1; }
            }
            if (FUSED) pdl_wait();
            if (OVB_PDL_GEMM) pdl_trigger();
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc_i8(TILE_N, p.bt);
        int s = 0;
        uint32_t phase = 0;
        // no way out of the loop: once a wait has run out all later ones return at once, and what is computed then is not stored
        if (FUSED) mbar_wait(&rows_ready, 0, abort_flag, p.status);
        for (int kb = kb0; kb < kb1; ++kb) {
            mbar_wait(&full[s], phase, abort_flag, p.status);
            tc_fence_after_sync();
            const uint32_t a = smem_u32(stages) + s * stage_bytes;
            const uint64_t da = umma_desc_k_sw128(a, 1024), db = umma_desc_k_sw128(FUSED ? smem_u32(smem) + (kb - kb0) * kI8FusedBlock : a + kI8TileBytes, 1024);
            umma_i8_block_elect(tmem, da, db, idesc, kb > kb0 ? 1u : 0u, &empty[s]);
            if (++s == p.stages) { s = 0; phase ^= 1; }
        }
        umma_commit_elect(&done);
        __syncwarp();
    } else if (FUSED) {
        __shared__ float box_f[8];
        __shared__ uint32_t box_u[8];
        __shared__ int box_i[8];
        pdl_wait();
        i8_quantize_row<E>(p, smem, kb0, kb1, row_scale, row_sum, box_f, box_u, box_i);
        if (threadIdx.x == 64) mbar_arrive(&rows_ready);
    }
    // while the products run: the scales of this thread's four channels and of the tokens (which the kernel before this one may have written)
    const int n = n0 + lane * 4;
    float ws[4], b[4];
    int zp[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = n + i < p.N;
        ws[i] = in ? __ldg(p.w_scale + n + i) : 0.f;
        zp[i] = in && p.w_zp != nullptr ? __ldg(p.w_zp + n + i) : 0;
        b[i] = in && p.bias != nullptr ? to_float(static_cast<const E*>(p.bias)[n + i]) : 0.f;
    }
    pdl_wait();
    const int tokens = min(p.bt, p.T - t0);
    if (!FUSED)
        for (int t = threadIdx.x; t < tokens; t += WARPS * 32) {
            row_scale[t] = __ldcg(p.x_scale + t0 + t);
            row_sum[t] = __ldcg(p.x_sum + t0 + t);
        }
    mbar_wait(&done, 0, abort_flag, p.status);
    __syncthreads();
    const bool fine = *abort_flag == 0;
    // every copy has landed and every MMA has read its operands: the stages hold the partial sums now
    int* part = reinterpret_cast<int*>(stages);         // [bt][128]
    if (fine && warp < 8) {
        tc_fence_after_sync();
        const int q = warp & 3;
        for (int c = (warp >> 2) * 16; c < p.bt; c += 32) {
            uint32_t r[16];
            tmem_ld_x16(tmem + (uint32_t(q * 32) << 16) + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) part[(c + j) * TILE_N + q * 32 + lane] = (int)r[j];
        }
    }
    tc_fence_before_sync();
    if (p.splits > 1) {
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    if (fine) {
        const int share0 = tokens * split / p.splits, share1 = tokens * (split + 1) / p.splits;
        const uint32_t mine = smem_u32(part) + lane * 16;
        constexpr bool GATED = i8_gated_form(FORM);
        const int cols = GATED ? p.N >> 1 : p.N, col = GATED ? (n0 >> 1) + lane * 4 : n, left = GATED && lane >= 16 ? 0 : cols - col;
        // S partials of as many tokens as give sixteen loads in flight. WHOLE: 16-bit results, four columns of a row in one aligned access.
        auto finish = [&](auto count, auto kind) {
            constexpr int S = decltype(count)::value, AT_ONCE = FUSED ? 1 : S == 1 ? 4 : 16 / S;
            constexpr bool WHOLE = decltype(kind)::value;
            uint32_t from[S];
#pragma unroll
            for (int r = 0; r < S; ++r) from[r] = S == 1 ? mine : dsmem_addr(mine, (uint32_t)r);
#pragma unroll 1
            for (int first = share0 + warp; first < share1; first += WARPS * AT_ONCE) {
                float4 f[AT_ONCE][S];
                uint2 res[AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int t = min(first + i * WARPS, share1 - 1);          // the last one again, where there are no more
#pragma unroll
                    for (int r = 0; r < S; ++r) f[i][r] = S == 1 ? *reinterpret_cast<const float4*>(part + t * TILE_N + lane * 4) : ld_dsmem_f4(from[r] + t * (TILE_N * 4));
                    if (WHOLE && !GATED) {
                        res[i] = make_uint2(0, 0);
                        if (p.residual != nullptr && left > 0) res[i] = __ldcg(reinterpret_cast<const uint2*>(static_cast<const E*>(p.residual) + (size_t)(t0 + t) * p.ldr + col));
                    }
                }
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int t = min(first + i * WARPS, share1 - 1);
                    int a[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int r = 0; r < S; ++r) {
                        a[0] += __float_as_int(f[i][r].x);
                        a[1] += __float_as_int(f[i][r].y);
                        a[2] += __float_as_int(f[i][r].z);
                        a[3] += __float_as_int(f[i][r].w);
                    }
                    const float xs = row_scale[t];
                    const int sum = row_sum[t];
                    float v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = i8_value<FORM>(a[j], zp[j], sum, xs * ws[j], b[j]);
                    if (GATED) {
                        // rows 0 .. 63 of the tile are the gate, 64 .. 127 the up values of the same channels
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] = i8_gate(p, v[j], __shfl_down_sync(0xffffffffu, v[j], 16));
                    }
                    if (FORM == kI8Any) i8_act_n(v, p);
                    const size_t at = (size_t)(t0 + t) * p.ldo + col;
                    if (WHOLE) {
                        if (!GATED && p.residual != nullptr) {
                            const E* e = reinterpret_cast<const E*>(&res[i]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) v[j] = __fadd_rn(v[j], to_float(e[j]));
                        }
                        if (left > 0 && first + i * WARPS < share1) *reinterpret_cast<uint2*>(static_cast<E*>(p.out) + at) = make_uint2(pack_pair<E>(v[0], v[1]), pack_pair<E>(v[2], v[3]));
                    } else {
                        if (first + i * WARPS >= share1) continue;              // a residual in place is added once
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (j < left) {
                                if (p.residual != nullptr) v[j] = __fadd_rn(v[j], to_float(static_cast<const E*>(p.residual)[(size_t)(t0 + t) * p.ldr + col + j]));
                                if (p.out_f32) static_cast<float*>(p.out)[at + j] = v[j];
                                else static_cast<E*>(p.out)[at + j] = from_float<E>(v[j]);
                            }
                    }
                }
            }
        };
        auto finish_as = [&](auto kind) {
            switch (p.splits) {
                case 1: finish(std::integral_constant<int, 1>(), kind); break;
                case 2: finish(std::integral_constant<int, 2>(), kind); break;
                case 4: finish(std::integral_constant<int, 4>(), kind); break;
                default: finish(std::integral_constant<int, 8>(), kind); break;
            }
        };
        if (p.whole) finish_as(std::true_type());
        else finish_as(std::false_type());
    }
    if (p.splits > 1) {             // a CTA's partials stay until the others have read them
        cluster_arrive();
        cluster_wait();
    }
    __syncthreads();
    if (!fine) {
        // copies that are still in flight land before the shared memory is given back
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, tmem_cols);
    }
}

// [N, K] bytes, row pitch ldw -> chunks of 128 rows x 128 columns, 16-byte pieces in the order of the 128-byte swizzle, rows behind N and columns
// behind K zero. `flip` 0x80: unsigned bytes, which become signed ones (b - 128).
__global__ void __launch_bounds__(256) pack_i8_kernel(const uint8_t* __restrict__ w, uint4* __restrict__ out, int N, int K, int64_t ldw, int KB, int flip) {
    const int tile = blockIdx.x / KB, kb = blockIdx.x - tile * KB;
    for (int i = threadIdx.x; i < TILE_N * 8; i += blockDim.x) {
        const int row = i >> 3, piece = i & 7, n = tile * TILE_N + row, k = kb * kI8BlockK + piece * 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (n < N) {
            const uint8_t* src = w + (size_t)n * ldw + k;
            uint8_t* b = reinterpret_cast<uint8_t*>(&v);
            for (int j = 0; j < 16; ++j)
                if (k + j < K) b[j] = src[j] ^ (uint8_t)flip;
        }
        out[(size_t)blockIdx.x * (TILE_N * 8) + row * 8 + (piece ^ (row & 7))] = v;
    }
}

template <bool F16, bool FUSED, int FORM>
static int launch_i8_tile(const cudaLaunchConfig_t& cfg, const CUtensorMap& tm, const I8TileParams& p) {
    static std::atomic<bool> known[64];
    int dev = 0;
    OVB_CHECK_CUDA(cudaGetDevice(&dev));
    if (!known[dev & 63].load(std::memory_order_acquire)) {          // (twice at the same time does no harm)
        OVB_CHECK_CUDA(cudaFuncSetAttribute(gemm_i8_tile_kernel<F16, FUSED, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
        known[dev & 63].store(true, std::memory_order_release);
    }
    OVB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, gemm_i8_tile_kernel<F16, FUSED, FORM>, tm, p));
    return 0;
}
template <bool F16, bool FUSED>
static int launch_i8_tile(int form, const cudaLaunchConfig_t& cfg, const CUtensorMap& tm, const I8TileParams& p) {
    switch (form) {
        case kI8Plain: return launch_i8_tile<F16, FUSED, kI8Plain>(cfg, tm, p);
        case kI8Gated: return launch_i8_tile<F16, FUSED, kI8Gated>(cfg, tm, p);
        case kI8GatedZp: return launch_i8_tile<F16, FUSED, kI8GatedZp>(cfg, tm, p);
        default: return launch_i8_tile<F16, FUSED, kI8Any>(cfg, tm, p);
    }
}

// A single token's row is quantised by the product's kernel: whole aligned pieces of eight columns, as many as eight warps hold. us with a norm, one launch / two
// (whose second also costs the host 2.5): 1024 x 1024 3.9 / 5.3, 6144 x 4096 6.9 / 9.8, 14336 x 4096 11.3 / 13.5, 4096 x 14336 13.7 / 14.0; with larger
// weights the CTAs that follow on an SM each quantise the row again: 10240 x 8192 20.3 / 18.4, 28672 x 4096 23.7 / 22.6, 128256 x 4096 86.5 / 79.1. More rows
// take a microsecond each, one behind the other (4 x 4096 x 4096 10.5 / 8.5).
// Every CTA reads the whole row at a time of its own, so a result in the row's place has it quantised first, by a launch of its own.
constexpr int64_t kI8FusedWeights = 64 << 20;       // bytes
static bool i8_fused_size(int T, int N, int K) { return T == 1 && (int64_t)N * K <= kI8FusedWeights && K % 8 == 0 && K <= kI8QuantWarps * 32 * kI8Hold * 8; }
static bool i8_fuses(const ovb_gemm_i8_args* a) {
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    const uintptr_t rows = a->row_idx != nullptr ? ((uintptr_t)(a->raw_rows - 1) * (uintptr_t)a->ld_raw + (uintptr_t)a->K) * 2 : (uintptr_t)a->K * 2;
    const uintptr_t result = (uintptr_t)(is_gated(a->act) ? a->N / 2 : a->N) * (a->out_f32 ? 4 : 2);
    const bool apart = bits(a->out) >= bits(a->raw) + rows || bits(a->raw) >= bits(a->out) + result;
    return apart && a->raw != nullptr && i8_fused_size(a->T, a->N, a->K) && (a->row_idx == nullptr || a->ld_raw % 8 == 0) && ((bits(a->raw) | bits(a->gamma)) & 15) == 0;
}

// How a product is run: pairs of CTAs, or tiles of `bt` tokens whose K is shared by `splits` CTAs, with `room` KB of shared memory each (108: two to an SM).
struct I8Plan {
    bool pair;
    int bt, splits, room;
};

// The fastest of the candidates by an estimate in us, fitted to 607 products (1 to 4096 tokens, 256 to 28672 channels, K 256 to 14336, cold weights): the
// geometric mean of what the choice loses against the best candidate is 1.3 %, one in twenty loses more than 8 %, the worst 29 %.
//  * tiles: waves of CTAs, of clusters where K is shared (as many as the device holds), each with its start and epilogue, its k-blocks at the issue rate of the
//    products, the bytes that an SM takes (both shared by the CTAs of an SM) or the latency that its stages hide, whichever is longest; the exchange of
//    partial sums; never less than the weights take from memory
//  * pairs: waves of 256 x 256 tiles
// us, 1 x 6144 x 4096 6.9; 64 x 28672 x 4096 21.6 (pairs 26.7); 256 x 28672 x 4096 39.5, pairs 30.2; 512 x 4096 x 4096 13.3, pairs 15.0; 999 x 8192 x 8192
// 62.9, pairs 47.8.
static bool i8_plan(int T, int N, int KB, bool fused, I8Plan* plan) {
    const int tiles_n = ceil_div(N, TILE_N), t16 = T > 256 ? 256 : (T + 15) / 16 * 16;
    *plan = {true, 256, 1, 216};
    const double pair_waves = (double)(((int64_t)ceil_div(T, 256) * ceil_div(N, 256) + 73) / 74);
    double best_us = fused ? 1e30 : 7.044 + pair_waves * KB * 0.3226 + (pair_waves - 1) * 5.848;
    const double bytes_us = 1.314 + (double)N * KB * 128 / 6.4e6;
    static constexpr int heights[6] = {16, 32, 64, 128, 256, 0};
    int held[9] = {0, 148, 0, 0, 0, 0, 0, 0, 0};        // CTAs or clusters that the device holds, asked for where a candidate needs it
    for (int i = 0; i < 6; ++i) {
        const int bt = heights[i] ? heights[i] : t16;
        if (bt > t16 || (heights[i] == t16 && i < 5)) continue;          // (the last one is t16 itself)
        if (fused && bt != 16) continue;
        const int64_t tiles = (int64_t)tiles_n * ceil_div(T, bt);
        if (ceil_div(T, bt) > 65535) continue;
        for (int room = 108; room <= 216; room += 108) {
            const int per_sm = 216 / room, stages = room * 8 / (128 + bt) < kI8MaxStages ? room * 8 / (128 + bt) : kI8MaxStages;
            if (stages < 3) continue;
            for (int S = 1; S <= 8 && S <= KB; S *= 2) {
                if (S > 1 && tiles * S > 444) break;
                if (fused && ceil_div(KB, S) * kI8FusedBlock + 3 * kI8TileBytes > room * 1024) continue;      // the row's codes stay in shared memory
                if (held[S] == 0) held[S] = cluster_capacity(S);
                const int64_t slots = (int64_t)held[S] * per_sm;
                const double waves = (double)((tiles + slots - 1) / slots);
                const double share = tiles * S <= 148 ? 1 : per_sm;
                const double issue = 0.1886 * share, bytes = 0.005616 * (16 + bt / 8.0) * share, latency = 1.649 / stages;
                double block = issue > bytes ? issue : bytes;
                if (latency > block) block = latency;
                double us = waves * (5.365 + ceil_div(KB, S) * block + 0.007415 * bt / S * share);
                if (S > 1) us += 2.164 + 0.01968 * bt * (S - 1) / S;
                if (us < bytes_us) us = bytes_us;
                if (us < best_us) {
                    best_us = us;
                    *plan = {false, bt, S, room};
                }
            }
        }
    }
    return best_us < 1e30;
}

static int run_i8_tile(const ovb_gemm_i8_args* a, const I8Params& base, const I8Plan& plan, bool fused, cudaStream_t stream) {
    I8TileParams p;
    static_cast<I8Params&>(p) = base;
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    p.whole = !a->out_f32 && a->N % 4 == 0 && a->ldo % 4 == 0 && (bits(a->out) & 7) == 0 && (a->residual == nullptr || (a->ldr % 4 == 0 && (bits(a->residual) & 7) == 0));
    p.raw = a->raw;
    p.gamma = a->gamma;
    p.row_idx = a->row_idx;
    p.ld_raw = a->ld_raw;
    p.raw_rows = a->raw_rows;
    p.eps = a->eps;
    p.bt = plan.bt;
    p.splits = plan.splits;
    const int tiles = ceil_div(a->N, TILE_N), rows = ceil_div(a->T, p.bt);
    const int per_split = ceil_div(p.KB, p.splits);
    const int stage = kI8TileBytes + (fused ? 0 : p.bt * kI8BlockK), head = fused ? per_split * kI8FusedBlock : 0;
    p.stages = (plan.room * 1024 - head) / stage;
    if (p.stages > kI8MaxStages) p.stages = kI8MaxStages;
    if (p.stages > per_split) p.stages = per_split;
    int bytes = p.stages * stage;
    if (bytes < p.bt * TILE_N * 4) bytes = p.bt * TILE_N * 4;
    CUtensorMap tm;
    if (fused) memset(&tm, 0, sizeof(tm));
    else if (int rc = make_tmap_2d(&tm, a->x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->T, a->K, a->ldx, p.bt, kI8BlockK, true)) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(tiles * p.splits, rows);
    cfg.blockDim = dim3(i8_threads(fused));
    cfg.dynamicSmemBytes = head + bytes + 1024;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (p.splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = p.splits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const int form = i8_form(a);
    if (fused) return a->f16 ? launch_i8_tile<true, true>(form, cfg, tm, p) : launch_i8_tile<false, true>(form, cfg, tm, p);
    return a->f16 ? launch_i8_tile<true, false>(form, cfg, tm, p) : launch_i8_tile<false, false>(form, cfg, tm, p);
}

}  // namespace ovb

extern "C" {

int64_t ovb_pack_i8_bytes(int N, int K) {
    using namespace ovb;
    return (int64_t)ceil_div(N, TILE_N) * ceil_div(K, kI8BlockK) * kI8TileBytes;
}

int ovb_pack_i8(const void* w, int is_unsigned, void* w_out, int N, int K, int64_t ldw, ovb_stream_t stream_) {
    using namespace ovb;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    OVB_REQUIRE(w && w_out && N > 0 && K > 0 && ldw >= K, "ovb_pack_i8: null operand or empty weight N=%d K=%d", N, K);
    OVB_REQUIRE((reinterpret_cast<uintptr_t>(w_out) & 127) == 0, "ovb_pack_i8: the packed weight must be 128-byte aligned");
    const int KB = ceil_div(K, kI8BlockK);
    const int64_t chunks = (int64_t)ceil_div(N, TILE_N) * KB;
    OVB_REQUIRE(chunks <= INT32_MAX, "ovb_pack_i8: weight of %d x %d is too large", N, K);
    OVB_CHECK_CUDA(launch_serial(pack_i8_kernel, dim3((unsigned)chunks), dim3(256), 0, stream, (const uint8_t*)w, (uint4*)w_out, N, K, ldw, KB, is_unsigned ? 0x80 : 0));
    return 0;
}

int ovb_gemm_i8_launches(int T, int N, int K) { return ovb::i8_fused_size(T, N, K) ? 1 : 2; }

int ovb_gemm_i8(const ovb_gemm_i8_args* a, ovb_stream_t stream_) {
    using namespace ovb;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    OVB_REQUIRE(a && a->x && a->x_scale && a->x_sum && a->w && a->w_scale && a->out, "ovb_gemm_i8: null operand");
    OVB_REQUIRE(a->T > 0 && a->N > 0 && a->K > 0, "ovb_gemm_i8: empty problem T=%d N=%d K=%d", a->T, a->N, a->K);
    OVB_REQUIRE(a->K <= kI8MaxK, "ovb_gemm_i8: K = %d, 32-bit sums are exact up to %d", a->K, kI8MaxK);
    OVB_REQUIRE(a->ldx >= a->K && a->ldx % 16 == 0, "ovb_gemm_i8: the row pitch %d of x must be a multiple of 16 that holds K=%d", a->ldx, a->K);
    OVB_REQUIRE((reinterpret_cast<uintptr_t>(a->x) & 15) == 0 && (reinterpret_cast<uintptr_t>(a->w) & 127) == 0,
                "ovb_gemm_i8: x must be 16-byte and the packed weight 128-byte aligned");
    const bool gated = a->act == OVB_ACT_SWIGLU || a->act == OVB_ACT_GLU_LIMITED;
    OVB_REQUIRE(a->act >= OVB_ACT_NONE && a->act <= OVB_ACT_SOFTCAP, "ovb_gemm_i8: unknown activation %d", a->act);
    OVB_REQUIRE(!gated || (a->N % TILE_N == 0 && !a->out_f32 && a->residual == nullptr && a->bias == nullptr),
                "ovb_gemm_i8: a gated epilogue needs N %% 128 == 0, a 16-bit output and no bias / residual");
    OVB_REQUIRE(a->residual == nullptr || !a->out_f32, "ovb_gemm_i8: a residual belongs to a 16-bit output");
    const int cols = gated ? a->N / 2 : a->N;
    OVB_REQUIRE(a->ldo >= cols && (a->residual == nullptr || a->ldr >= cols), "ovb_gemm_i8: row pitch of the output %d or residual %d below %d columns", a->ldo, a->ldr, cols);
    OVB_REQUIRE(a->raw == nullptr || (a->ld_raw >= 0 && (a->row_idx == nullptr || a->raw_rows > 0)), "ovb_gemm_i8: row indices need the number of rows, rows their pitch");
    I8Plan plan;
    const int KB = ceil_div(a->K, kI8BlockK);
    const bool fused = i8_fuses(a) && i8_plan(a->T, a->N, KB, true, &plan);
    if (!fused) i8_plan(a->T, a->N, KB, false, &plan);
    if (a->raw != nullptr && !fused) {
        const ovb_quant_rows_args rows = {a->raw, a->gamma, a->row_idx, const_cast<void*>(a->x), const_cast<float*>(a->x_scale), const_cast<int*>(a->x_sum), a->ld_raw, a->T, a->K,
                                          a->raw_rows, a->ldx, a->f16, a->eps};
        if (int rc = ovb_quantize_rows(&rows, stream_)) return rc;
    }
    I8Params p;
    p.w = static_cast<const uint8_t*>(a->w);
    p.x_scale = a->x_scale;
    p.x_sum = a->x_sum;
    p.w_scale = a->w_scale;
    p.w_zp = a->w_zp;
    p.bias = a->bias;
    p.residual = a->residual;
    p.out = a->out;
    p.status = status_word();
    p.T = a->T; p.N = a->N; p.K = a->K;
    p.KB = KB;
    p.ldo = a->ldo; p.ldr = a->ldr;
    p.act = a->act; p.out_f32 = a->out_f32;
    p.act_limit = a->act_limit; p.act_slope = a->act_slope; p.act_shift = a->act_shift;
    return plan.pair ? gemm_i8_pair(a, p, stream) : run_i8_tile(a, p, plan, fused, stream);
}

}  // extern "C"
