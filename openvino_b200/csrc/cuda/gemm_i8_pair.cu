// Products of signed bytes, many tokens: pairs of CTAs (tcgen05, cta_group::2, kind::i8).
//
// What bounds it: the tensor pipe. A pair of SMs works on 256 tokens (the M side, 128 to each SM) x `bn` channels (256 or 128); every CTA loads its 128
// tokens and half of the weight rows, 32 KB for 256 x 256 x 128 products. The kernel is persistent and the accumulator exists twice in tensor memory
// (2 x 256 columns), so that the epilogue of a tile runs under the main loop of the next.
//  * warp 0: producer (TMA boxes of both operands; both CTAs' bytes are counted on the even CTA's barrier), warp 1 of the even CTA: MMAs of the pair
//  * warps 4 .. 11: epilogue. Tokens are the lanes, so a thread holds one row: adjacent channels lie in its registers, a gate and its up value too, and
//    results leave in whole 32-byte sectors. Scales, zero points and biases of the channels come from shared memory, the same for all lanes.
#include <mutex>

#include "gemm_i8.cuh"

namespace ovb {

constexpr int kI8PairStages = 6;
constexpr int kI8PairThreads = 384;
constexpr int kI8PairStageBytes = 2 * kI8TileBytes;                      // 128 tokens and up to 128 weight rows
constexpr int kI8PairChannels = 256;                                     // channels of a tile at most
constexpr int kI8PairSmem = kI8PairStages * kI8PairStageBytes + 2 * kI8PairChannels * 12 + 1024 + 1024;
constexpr int kI8PairBand = 8;                                           // token tiles per rasterisation band

struct I8PairParams : I8Params {
    int bn;                       // channels of a tile: 256 or 128
    int tiles_n, tiles_t;
};

// Tiles in bands of eight token tiles: a band's tokens stay in L2 while its weights pass once.
__device__ __forceinline__ bool i8_pair_tile(const I8PairParams& p, int idx, int& t0, int& n0) {
    if (idx >= p.tiles_n * p.tiles_t) return false;
    const int band_sz = kI8PairBand * p.tiles_n, band = idx / band_sz, r = idx - band * band_sz;
    const int in_band = min(kI8PairBand, p.tiles_t - band * kI8PairBand), n = r / in_band;
    t0 = (band * kI8PairBand + (r - n * in_band)) * 256;
    n0 = n * p.bn;
    return true;
}

__device__ __forceinline__ void pair_mma_i8_elect(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t* r) {
    tmem_ld_x16(taddr, r);
    tmem_ld_x16(taddr + 16, r + 16);
}

// 32 bytes at a time: one whole sector of the row that a lane owns
__device__ __forceinline__ void st_global_32(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void ld_global_32(const void* p, uint32_t* v) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p) : "memory");
}
template <class E>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    E e[2] = {from_float<E>(a), from_float<E>(b)};
    return *reinterpret_cast<uint32_t*>(e);
}

template <bool F16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kI8PairThreads, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const I8PairParams p) {
    using E = typename Elem<F16>::type;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* chan_scale = reinterpret_cast<float*>(smem + kI8PairStages * kI8PairStageBytes);      // [2][256] each
    float* chan_bias = chan_scale + 2 * kI8PairChannels;
    int* chan_zp = reinterpret_cast<int*>(chan_bias + 2 * kI8PairChannels);
    uint64_t* bars = reinterpret_cast<uint64_t*>(chan_zp + 2 * kI8PairChannels);
    uint64_t* full = bars;                              // [stages] even CTA: both CTAs' tiles have landed
    uint64_t* empty = bars + kI8PairStages;             // [stages] both CTAs: the stage has been read
    uint64_t* acc_full = bars + 2 * kI8PairStages;      // [2] both CTAs: accumulator complete
    uint64_t* acc_empty = acc_full + 2;                 // [2] even CTA: accumulator drained by the 16 epilogue warps of the pair
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* went_well = abort_flag + 1;           // [2]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kI8PairStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 16);
        }
        *abort_flag = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    const int pairs = (int)gridDim.x >> 1, first = (int)blockIdx.x >> 1;
    const int half_n = p.bn >> 1;                       // weight rows that a CTA loads
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int s = 0, t0, n0;
            uint32_t phase = 1;
            bool ok = true;
            const uint32_t tx = 2u * (kI8TileBytes + half_n * kI8BlockK);
            for (int idx = first; ok && i8_pair_tile(p, idx, t0, n0); idx += pairs) {
                // the weight's rows as they are packed: 128 of a chunk, chunk after chunk along K. Channels behind the last chunk are not there: the
                // box then reads the last chunk's again, and nothing of them is stored
                const int row = n0 + (int)rank * half_n;
                const int last = (p.N - 1) / TILE_N;
                int w_row = min(row / TILE_N, last) * p.KB * TILE_N + row % TILE_N;
                const int x_row = t0 + (int)rank * 128;
                for (int kb = 0; kb < p.KB; ++kb) {
                    ok = mbar_wait(&empty[s], phase, abort_flag, p.status);
                    if (!ok) break;
                    const uint32_t st = smem_u32(smem) + s * kI8PairStageBytes, bar = smem_u32(&full[s]);
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], tx);
                    pair_load_2d(st, &tmX, bar, kb * kI8BlockK, x_row);
                    pair_load_2d(st + kI8TileBytes, &tmW, bar, 0, w_row);
                    w_row += TILE_N;
                    if (++s == kI8PairStages) { s = 0; phase ^= 1; }
                }
            }
            if (OVB_PDL_GEMM) pdl_trigger();
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint64_t desc0 = umma_desc_k_sw128(smem_u32(smem), 1024);
            const uint32_t idesc = umma_idesc_i8(256, p.bn);
            int s = 0, buf = 0, t0, n0;
            uint32_t phase = 0, acc_phase = 1;
            bool ok = true;
            for (int idx = first; ok && i8_pair_tile(p, idx, t0, n0); idx += pairs) {
                ok = mbar_wait(&acc_empty[buf], acc_phase, abort_flag, p.status);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t d = tmem_base + uint32_t(buf * 256);
                for (int kb = 0; kb < p.KB; ++kb) {
                    ok = mbar_wait(&full[s], phase, abort_flag, p.status);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint64_t da = desc0 + (uint64_t)((s * kI8PairStageBytes) >> 4), db = da + (uint64_t)(kI8TileBytes >> 4);
#pragma unroll
                    for (int k = 0; k < kI8BlockK / 32; ++k) pair_mma_i8_elect(d, da + 2 * k, db + 2 * k, idesc, (kb | k) ? 1u : 0u);
                    pair_commit_elect(&empty[s]);
                    if (++s == kI8PairStages) { s = 0; phase ^= 1; }
                }
                if (!ok) break;
                pair_commit_elect(&acc_full[buf]);
                if (++buf == 2) { buf = 0; acc_phase ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2, tid = threadIdx.x - 128;
        const bool gated = is_gated(p.act);
        const uint32_t drained0 = dsmem_addr(smem_u32(&acc_empty[0]), 0);
        const int cols = half_n;                        // channels of this warp: [half * cols, + cols)
        const int out_cols = gated ? p.N >> 1 : p.N;
        int buf = 0, t0, n0;
        uint32_t acc_phase = 0;
        for (int idx = first; i8_pair_tile(p, idx, t0, n0); idx += pairs) {
            const int t = t0 + (int)rank * 128 + q * 32 + lane;
            const bool row = t < p.T;
            const float xs = row ? __ldcg(p.x_scale + t) : 0.f;
            const int sum = row && p.w_zp != nullptr ? __ldcg(p.x_sum + t) : 0;
            float* cs = chan_scale + buf * kI8PairChannels;
            float* cb = chan_bias + buf * kI8PairChannels;
            int* cz = chan_zp + buf * kI8PairChannels;
            if (tid < p.bn) {
                const int n = n0 + tid;
                cs[tid] = n < p.N ? __ldg(p.w_scale + n) : 0.f;
                if (p.bias != nullptr) cb[tid] = n < p.N ? to_float(static_cast<const E*>(p.bias)[n]) : 0.f;
                if (p.w_zp != nullptr) cz[tid] = n < p.N ? __ldg(p.w_zp + n) : 0;
            }
            // one thread polls and says how it ended; the others wait at the barrier, so that all eight warps go on or leave together
            if (tid == 0) went_well[buf] = mbar_wait(&acc_full[buf], acc_phase, abort_flag, p.status) ? 1 : 0;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (!went_well[buf]) break;
            tc_fence_after_sync();
            const uint32_t src = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(buf * 256 + half * cols);
            // 32 finished values of this row from column `first_col` on
            auto put = [&](float (&v)[32], int col) {
                const size_t at = (size_t)t * p.ldo + col;
                const bool whole = col + 32 <= out_cols;
                if (p.residual != nullptr) {
                    const E* r = static_cast<const E*>(p.residual) + (size_t)t * p.ldr + col;
                    if (row && whole && (reinterpret_cast<uintptr_t>(r) & 31) == 0) {
                        uint32_t w[16];
                        ld_global_32(r, w);
                        ld_global_32(r + 16, w + 8);
                        const E* e = reinterpret_cast<const E*>(w);
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] += to_float(e[i]);
                    } else if (row) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (col + i < out_cols) v[i] += to_float(r[i]);
                    }
                }
                if (!row) return;
                if (p.out_f32) {
                    float* o = static_cast<float*>(p.out) + at;
                    if (whole && (reinterpret_cast<uintptr_t>(o) & 31) == 0) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) st_global_32(o + i, reinterpret_cast<const uint32_t*>(v) + i);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (col + i < out_cols) o[i] = v[i];
                    }
                    return;
                }
                E* o = static_cast<E*>(p.out) + at;
                if (whole && (reinterpret_cast<uintptr_t>(o) & 31) == 0) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = pack_pair<E>(v[2 * i], v[2 * i + 1]);
                    st_global_32(o, w);
                    st_global_32(o + 16, w + 8);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (col + i < out_cols) o[i] = from_float<E>(v[i]);
                }
            };
            auto drained = [&]() {                      // the accumulator has been read by this warp
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_cluster(drained0 + buf * 8);
            };
            auto values = [&](const uint32_t (&r)[32], int c, float (&v)[32]) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 s4 = *reinterpret_cast<const float4*>(cs + c + i);
                    int a[4] = {(int)r[i], (int)r[i + 1], (int)r[i + 2], (int)r[i + 3]};
                    if (p.w_zp != nullptr) {
                        const int4 z = *reinterpret_cast<const int4*>(cz + c + i);
                        a[0] -= z.x * sum; a[1] -= z.y * sum; a[2] -= z.z * sum; a[3] -= z.w * sum;
                    }
                    v[i] = float(a[0]) * (xs * s4.x); v[i + 1] = float(a[1]) * (xs * s4.y);
                    v[i + 2] = float(a[2]) * (xs * s4.z); v[i + 3] = float(a[3]) * (xs * s4.w);
                    if (p.bias != nullptr) {
                        const float4 b = *reinterpret_cast<const float4*>(cb + c + i);
                        v[i] += b.x; v[i + 1] += b.y; v[i + 2] += b.z; v[i + 3] += b.w;
                    }
                }
            };
            if (gated) {
                // 128 channels of a weight tile: 64 of the gate, then the 64 up values. A warp finishes 32 output columns at a time, its half of them.
                for (int c = half * 32; c < (p.bn >> 1); c += 64) {
                    const int at = (c >> 6) * 128 + (c & 63);          // the gate's column in the tile
                    const uint32_t base = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(buf * 256);
                    uint32_t g[32], u[32];
                    tmem_ld_x32(base + at, g);
                    tmem_ld_x32(base + at + 64, u);
                    tmem_ld_wait();
                    if (c + 64 >= (p.bn >> 1)) drained();
                    float vg[32], vu[32];
                    values(g, at, vg);
                    values(u, at + 64, vu);
#pragma unroll
                    for (int i = 0; i < 32; ++i) vg[i] = p.act == OVB_ACT_SWIGLU ? __fdividef(vg[i], 1.0f + __expf(-vg[i])) * vu[i] : glu_limited(p, vg[i], vu[i]);
                    if (n0 + at < p.N) put(vg, (n0 >> 1) + c);
                }
            } else {
                for (int c = 0; c < cols; c += 32) {
                    uint32_t r[32];
                    tmem_ld_x32(src + c, r);
                    tmem_ld_wait();
                    if (c + 32 >= cols) drained();
                    float v[32];
                    values(r, half * cols + c, v);
                    apply_act_n(v, p);
                    const int col = n0 + half * cols + c;
                    if (col < p.N) put(v, col);
                }
            }
            if (++buf == 2) { buf = 0; acc_phase ^= 1; }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        // copies that are still in flight land before the shared memory is reused
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        __syncthreads();
    }
    cluster_arrive();
    cluster_wait();
    if (warp == 2) {
        tc_fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
    }
}

// Pairs of CTAs that are resident at a time.
template <bool F16>
static int resident_i8_pairs(int* pairs) {
    static std::mutex mu;
    static int known[64] = {0};
    int dev = 0;
    OVB_CHECK_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (known[dev & 63] == 0) {
        auto kern = gemm_i8_pair_kernel<F16>;
        OVB_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kI8PairSmem));
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3(148);
        cfg.blockDim = dim3(kI8PairThreads);
        cfg.dynamicSmemBytes = kI8PairSmem;
        int n = 0;
        OVB_CHECK_CUDA(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
        known[dev & 63] = n < 1 ? 1 : n;
    }
    *pairs = known[dev & 63];
    return 0;
}

template <bool F16>
static int run_i8_pair(const ovb_gemm_i8_args* a, const I8Params& base, cudaStream_t stream) {
    int pairs = 0;
    if (int rc = resident_i8_pairs<F16>(&pairs)) return rc;
    I8PairParams p;
    static_cast<I8Params&>(p) = base;
    p.tiles_t = ceil_div(a->T, 256);
    p.bn = 256;
    p.tiles_n = ceil_div(a->N, p.bn);
    CUtensorMap tmW, tmX;
    if (int rc = make_tmap_2d(&tmX, a->x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->T, a->K, a->ldx, 128, kI8BlockK, true)) return rc;
    // the chunks are already in the swizzled order of the MMA: plain boxes of rows of 128 bytes
    if (int rc = make_tmap_2d(&tmW, a->w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)ceil_div(a->N, TILE_N) * p.KB * TILE_N, kI8BlockK, kI8BlockK, p.bn / 2, kI8BlockK, false)) return rc;
    const int64_t tiles = (int64_t)p.tiles_n * p.tiles_t;
    OVB_CHECK_CUDA(launch_pdl(gemm_i8_pair_kernel<F16>, dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs)), dim3(kI8PairThreads), kI8PairSmem, stream, tmW, tmX, p));
    return 0;
}

int gemm_i8_pair(const ovb_gemm_i8_args* a, const I8Params& p, cudaStream_t stream) { return a->f16 ? run_i8_pair<true>(a, p, stream) : run_i8_pair<false>(a, p, stream); }

}  // namespace ovb
