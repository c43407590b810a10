// Products of signed bytes, many tokens: pairs of CTAs (tcgen05, cta_group::2, kind::i8).
//
// What bounds it: the tensor pipe, and in long runs the power cap. A pair of SMs works on 256 tokens (the M side, 128 to each SM) x 256 channels; every CTA
// loads its 128 tokens and half of the weight rows, 32 KB for 256 x 256 x 128 products. The kernel is persistent and the accumulator exists twice in tensor
// memory (2 x 256 columns), so that the epilogue of a tile runs under the main loop of the next. Measured: 8192 x 28672 x 4096 with the gate 590 us (3.26
// POP/s; twice the measured bf16 rate is 3.34), 999 x 8192 x 8192 47.5 us (2.8 POP/s: 128 tiles on 74 pairs), 333 x 4096 x 14336 28 us. Tiles of 128
// channels and pairs that share K gave nothing at sizes where they fill the machine better.
//  * warp 0: producer (TMA boxes of both operands; both CTAs' bytes are counted on the even CTA's barrier), warp 1 of the even CTA: MMAs of the pair
//  * warps 4 .. 11: epilogue. Tokens are the lanes, so a thread holds one row: adjacent channels lie in its registers, a gate and its up value too, and
//    results leave in whole 32-byte sectors. Scales, zero points and biases of the channels come from shared memory, the same for all lanes.
#include <mutex>
#include <type_traits>

#include "gemm_i8.cuh"

namespace ovb {

constexpr int kI8PairStages = 6;
constexpr int kI8PairThreads = 384;
constexpr int kI8PairStageBytes = 2 * kI8TileBytes;                      // 128 tokens and up to 128 weight rows
constexpr int kI8PairChannels = 256;                                     // channels of a tile, half of which each CTA loads
constexpr int kI8PairBox = 2048;                                         // 32 rows x 64 bytes of an epilogue warp, on their way from rows to lines
constexpr int kI8PairBand = 8;                                           // token tiles per rasterisation band
constexpr int kI8PairSmem = kI8PairStages * kI8PairStageBytes + 8 * kI8PairBox + 2 * kI8PairChannels * 12 + 1024 + 1024;

struct I8PairParams : I8Params {
    int tiles_n, tiles_t;
    int whole;                    // 16-bit results and residuals in aligned pieces of eight columns
};

// Tiles in bands of eight token tiles: a band's tokens stay in L2 while its weights pass once.
__device__ __forceinline__ bool i8_pair_tile(const I8PairParams& p, int idx, int& t0, int& n0) {
    if (idx >= p.tiles_n * p.tiles_t) return false;
    const int band_sz = kI8PairBand * p.tiles_n, band = idx / band_sz, r = idx - band * band_sz;
    const int in_band = min(kI8PairBand, p.tiles_t - band * kI8PairBand), n = r / in_band;
    t0 = (band * kI8PairBand + (r - n * in_band)) * 256;
    n0 = n * kI8PairChannels;
    return true;
}

// The four products of a k-block and the commit of its stage in both CTAs (see umma_i8_block_elect).
__device__ __forceinline__ void pair_i8_block_elect(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 t, 0, 0;\n\t"
        "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
        "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], a1, b1, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], a2, b2, %3, t;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], a3, b3, %3, t;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], %6;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(smem_u32(bar)), "h"((uint16_t)3)
        : "memory");
}
template <bool F16, int FORM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kI8PairThreads, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ I8PairParams p) {
    using E = typename Elem<F16>::type;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* boxes = smem + kI8PairStages * kI8PairStageBytes;
    float* chan_scale = reinterpret_cast<float*>(boxes + 8 * kI8PairBox);                          // [2][256] each
    float* chan_bias = chan_scale + 2 * kI8PairChannels;
    int* chan_zp = reinterpret_cast<int*>(chan_bias + 2 * kI8PairChannels);
    uint64_t* bars = reinterpret_cast<uint64_t*>(chan_zp + 2 * kI8PairChannels);
    uint64_t* full = bars;                              // [stages] even CTA: both CTAs' tiles have landed
    uint64_t* empty = bars + kI8PairStages;          // [stages] both CTAs: the stage has been read
    uint64_t* acc_full = bars + 2 * kI8PairStages;   // [2] both CTAs: accumulator complete
    uint64_t* acc_empty = acc_full + 2;                 // [2] even CTA: accumulator drained by the 16 epilogue warps of the pair
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* went_well = abort_flag + 1;           // [2]

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
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
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int s = 0, t0, n0;
            uint32_t phase = 1;
            bool ok = true;
            const uint32_t tx = 2u * kI8PairStageBytes;
            for (int idx = first; ok && i8_pair_tile(p, idx, t0, n0); idx += pairs) {
                // one packed chunk of 128 rows for every k-block. An odd last chunk is read by both CTAs; what the second one makes of it is not stored
                int w_row = min(n0 / TILE_N + (int)rank, (p.N - 1) / TILE_N) * p.KB * TILE_N;
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
            const uint32_t idesc = umma_idesc_i8(256, kI8PairChannels);
            int s = 0, buf = 0, t0, n0;
            uint32_t phase = 0, acc_phase = 1;
            // no way out of the loops: once a wait has run out all later ones return at once, and what is computed then is not stored
            for (int idx = first; i8_pair_tile(p, idx, t0, n0); idx += pairs) {
                mbar_wait(&acc_empty[buf], acc_phase, abort_flag, p.status);
                tc_fence_after_sync();
                const uint32_t d = tmem_base + uint32_t(buf * 256);
                for (int kb = 0; kb < p.KB; ++kb) {
                    mbar_wait(&full[s], phase, abort_flag, p.status);
                    tc_fence_after_sync();
                    const uint64_t da = desc0 + (uint64_t)((s * kI8PairStageBytes) >> 4), db = da + (uint64_t)(kI8TileBytes >> 4);
                    pair_i8_block_elect(d, da, db, idesc, kb > 0 ? 1u : 0u, &empty[s]);
                    if (++s == kI8PairStages) { s = 0; phase ^= 1; }
                }
                pair_commit_elect(&acc_full[buf]);
                if (++buf == 2) { buf = 0; acc_phase ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2, tid = threadIdx.x - 128;
        constexpr bool GATED = i8_gated_form(FORM);
        const uint32_t drained0 = dsmem_addr(smem_u32(&acc_empty[0]), 0);
        // A job is 32 columns of the result: 32 of the tile's, or the gate and the up values of the same channels (64 rows of a weight tile are the gate, then
        // 64 the up values), in two steps of 16. The two warps of a token quarter take jobs in turn.
        constexpr int RUNS = GATED ? 2 : 1;
        constexpr int JOBS = kI8PairChannels / (32 * RUNS);
        const int out_cols = GATED ? p.N >> 1 : p.N;
        auto column = [&](int job, int run, int step) { return (GATED ? (job >> 1) * 128 + (job & 1) * 32 + run * 64 : job * 32) + step * 16; };
        // this warp's box: 64 bytes of each of its 32 rows, pieces of 16 bytes placed so that rows and lines are both free of bank conflicts
        uint8_t* box = boxes + (warp - 4) * kI8PairBox;
        auto in_box = [&](int r, int piece) { return reinterpret_cast<uint4*>(box + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4)); };
        int buf = 0, t0, n0;
        uint32_t acc_phase = 0;
        for (int idx = first; i8_pair_tile(p, idx, t0, n0); idx += pairs) {
            const int t = t0 + (int)rank * 128 + q * 32 + lane;
            const bool row = t < p.T;
            const float xs = row ? __ldcg(p.x_scale + t) : 0.f;
            const int sum = row ? __ldcg(p.x_sum + t) : 0;
            float* cs = chan_scale + buf * kI8PairChannels;
            float* cb = chan_bias + buf * kI8PairChannels;
            int* cz = chan_zp + buf * kI8PairChannels;
            const int n = n0 + tid;                     // a channel for each of the 256 threads
            cs[tid] = n < p.N ? __ldg(p.w_scale + n) : 0.f;
            cb[tid] = n < p.N && p.bias != nullptr ? to_float(static_cast<const E*>(p.bias)[n]) : 0.f;
            cz[tid] = n < p.N && p.w_zp != nullptr ? __ldg(p.w_zp + n) : 0;
            const int first_row = t - lane, rows = min(32, p.T - first_row);           // of this warp; rows may be negative
            // The residual's 32 columns of a job, in aligned pieces of eight, are fetched a job ahead, the first ones before the products are complete.
            const bool res = !GATED && p.residual != nullptr, res_ahead = res && p.whole;
            uint4 ahead[GATED ? 1 : 4];
            auto fetch = [&](int job) {
                if (GATED) return;
                const E* from = static_cast<const E*>(p.residual) + (size_t)first_row * p.ldr + n0 + job * 32;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = i * 8 + (lane >> 2), c = (lane & 3) * 8;
                    if (r < rows && n0 + job * 32 + c < out_cols) ahead[GATED ? 0 : i] = __ldcg(reinterpret_cast<const uint4*>(from + (size_t)r * p.ldr + c));
                }
            };
            if (res_ahead) fetch(half);
            // one thread polls and says how it ended; the others wait at the barrier, so that all eight warps go on or leave together
            if (tid == 0) went_well[buf] = mbar_wait(&acc_full[buf], acc_phase, abort_flag, p.status) ? 1 : 0;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (!went_well[buf]) break;
            tc_fence_after_sync();
            const uint32_t src = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(buf * 256);
            auto values = [&](const uint32_t* r, int c, float* v) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 s4 = *reinterpret_cast<const float4*>(cs + c + i);
                    float4 b4 = make_float4(0.f, 0.f, 0.f, 0.f);
                    int4 z4 = make_int4(0, 0, 0, 0);
                    if (FORM == kI8Any) b4 = *reinterpret_cast<const float4*>(cb + c + i);
                    if (i8_zp_form(FORM)) z4 = *reinterpret_cast<const int4*>(cz + c + i);
                    v[i] = i8_value<FORM>((int)r[i], z4.x, sum, xs * s4.x, b4.x);
                    v[i + 1] = i8_value<FORM>((int)r[i + 1], z4.y, sum, xs * s4.y, b4.y);
                    v[i + 2] = i8_value<FORM>((int)r[i + 2], z4.z, sum, xs * s4.z, b4.z);
                    v[i + 3] = i8_value<FORM>((int)r[i + 3], z4.w, sum, xs * s4.w, b4.w);
                }
            };
            // 16 columns of a job as finished values, the residual not yet added
            auto compute = [&](int job, int step, float (&v)[16]) {
                uint32_t r[16 * RUNS];
#pragma unroll
                for (int run = 0; run < RUNS; ++run) tmem_ld_x16(src + column(job, run, step), r + 16 * run);
                tmem_ld_wait();
                values(r, column(job, 0, step), v);
                if (GATED) {
                    float u[16];
                    values(r + 16, column(job, RUNS - 1, step), u);
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = i8_gate(p, v[i], u[i]);
                } else if (FORM == kI8Any) {
                    i8_act_n(v, p);
                }
            };
            // 16-bit results: the box holds the 32 columns of the job, first of the residual, then of the result. WHOLE: aligned pieces of eight columns
            auto finish16 = [&](auto kind) {
                constexpr bool WHOLE = decltype(kind)::value;
#pragma unroll 1
                for (int job = half; job < JOBS; job += 2) {
                    const int col = (GATED ? n0 >> 1 : n0) + job * 32;
                    if (res) {
                        if (WHOLE) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) *in_box(i * 8 + (lane >> 2), lane & 3) = ahead[GATED ? 0 : i];
                            if (job + 2 < JOBS) fetch(job + 2);
                        } else {
                            const E* from = static_cast<const E*>(p.residual) + (size_t)first_row * p.ldr + col;
                            for (int r0 = 0; r0 < rows; r0 += 16) {
                                E e[16];
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                    if (r0 + i < rows && col + lane < out_cols) e[i] = from[(size_t)(r0 + i) * p.ldr + lane];
#pragma unroll
                                for (int i = 0; i < 16; ++i) reinterpret_cast<E*>(in_box(r0 + i, lane >> 3))[lane & 7] = e[i];
                            }
                        }
                        __syncwarp();
                    }
#pragma unroll
                    for (int step = 0; step < 2; ++step) {
                        float v[16];
                        compute(job, step, v);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint4* place = in_box(lane, step * 2 + h);
                            if (res) {
                                const uint4 raw = *place;
                                const E* e = reinterpret_cast<const E*>(&raw);
#pragma unroll
                                for (int i = 0; i < 8; ++i) v[h * 8 + i] = __fadd_rn(v[h * 8 + i], to_float(e[i]));
                            }
                            *place = make_uint4(pack_pair<E>(v[h * 8], v[h * 8 + 1]), pack_pair<E>(v[h * 8 + 2], v[h * 8 + 3]), pack_pair<E>(v[h * 8 + 4], v[h * 8 + 5]),
                                                pack_pair<E>(v[h * 8 + 6], v[h * 8 + 7]));
                        }
                    }
                    __syncwarp();
                    E* to = static_cast<E*>(p.out) + (size_t)first_row * p.ldo + col;
                    if (WHOLE) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = i * 8 + (lane >> 2), c = (lane & 3) * 8;
                            if (r < rows && col + c < out_cols) *reinterpret_cast<uint4*>(to + (size_t)r * p.ldo + c) = *in_box(r, lane & 3);
                        }
                    } else {
                        for (int r = 0; r < rows; ++r)
                            if (col + lane < out_cols) to[(size_t)r * p.ldo + lane] = reinterpret_cast<const E*>(in_box(r, lane >> 3))[lane & 7];
                    }
                    __syncwarp();
                }
            };
            // fp32 results: 16 columns at a time, two rows of them to a store
            auto finish32 = [&]() {
                for (int job = half; job < JOBS; job += 2)
                    for (int step = 0; step < 2; ++step) {
                        float v[16];
                        compute(job, step, v);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *in_box(lane, i) = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
                        __syncwarp();
                        const int c = lane & 15, col = n0 + job * 32 + step * 16 + c;
                        float* to = static_cast<float*>(p.out) + (size_t)first_row * p.ldo + col;
                        for (int r = lane >> 4; r < rows; r += 2)
                            if (col < out_cols) to[(size_t)r * p.ldo] = reinterpret_cast<const float*>(in_box(r, c >> 2))[c & 3];
                        __syncwarp();
                    }
            };
            if (!GATED && p.out_f32) finish32();
            else if (p.whole) finish16(std::true_type());
            else finish16(std::false_type());
            // the accumulator has been read by this warp
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_cluster(drained0 + buf * 8);
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

// Pairs of CTAs that are resident at a time, asked once per device.
template <bool F16, int FORM>
static int resident_i8_pairs(int* pairs) {
    static std::mutex mu;
    static int known[64] = {0};
    int dev = 0;
    OVB_CHECK_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (known[dev & 63] == 0) {
        OVB_CHECK_CUDA(cudaFuncSetAttribute(gemm_i8_pair_kernel<F16, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, kI8PairSmem));
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3(148);
        cfg.blockDim = dim3(kI8PairThreads);
        cfg.dynamicSmemBytes = kI8PairSmem;
        int n = 0;
        OVB_CHECK_CUDA(cudaOccupancyMaxActiveClusters(&n, gemm_i8_pair_kernel<F16, FORM>, &cfg));
        known[dev & 63] = n < 1 ? 1 : n;
    }
    *pairs = known[dev & 63];
    return 0;
}

template <bool F16, int FORM>
static int launch_i8_pair(const CUtensorMap& tmW, const CUtensorMap& tmX, const I8PairParams& p, cudaStream_t stream) {
    int pairs = 0;
    if (int rc = resident_i8_pairs<F16, FORM>(&pairs)) return rc;
    const int64_t tiles = (int64_t)p.tiles_n * p.tiles_t;
    OVB_CHECK_CUDA(launch_pdl(gemm_i8_pair_kernel<F16, FORM>, dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs)), dim3(kI8PairThreads), kI8PairSmem, stream, tmW, tmX, p));
    return 0;
}
template <bool F16>
static int launch_i8_pair(int form, const CUtensorMap& tmW, const CUtensorMap& tmX, const I8PairParams& p, cudaStream_t stream) {
    switch (form) {
        case kI8Plain: return launch_i8_pair<F16, kI8Plain>(tmW, tmX, p, stream);
        case kI8Gated: return launch_i8_pair<F16, kI8Gated>(tmW, tmX, p, stream);
        case kI8GatedZp: return launch_i8_pair<F16, kI8GatedZp>(tmW, tmX, p, stream);
        default: return launch_i8_pair<F16, kI8Any>(tmW, tmX, p, stream);
    }
}

int gemm_i8_pair(const ovb_gemm_i8_args* a, const I8Params& base, cudaStream_t stream) {
    I8PairParams p;
    static_cast<I8Params&>(p) = base;
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    const int out_cols = is_gated(a->act) ? a->N / 2 : a->N;
    p.whole = out_cols % 8 == 0 && a->ldo % 8 == 0 && (bits(a->out) & 15) == 0 && (a->residual == nullptr || (a->ldr % 8 == 0 && (bits(a->residual) & 15) == 0));
    p.tiles_t = ceil_div(a->T, 256);
    p.tiles_n = ceil_div(a->N, kI8PairChannels);
    CUtensorMap tmW, tmX;
    if (int rc = make_tmap_2d(&tmX, a->x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->T, a->K, a->ldx, 128, kI8BlockK, true)) return rc;
    // the chunks are already in the swizzled order of the MMA: plain boxes of rows of 128 bytes
    if (int rc = make_tmap_2d(&tmW, a->w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)ceil_div(a->N, TILE_N) * p.KB * TILE_N, kI8BlockK, kI8BlockK, TILE_N, kI8BlockK, false)) return rc;
    return a->f16 ? launch_i8_pair<true>(i8_form(a), tmW, tmX, p, stream) : launch_i8_pair<false>(i8_form(a), tmW, tmX, p, stream);
}

}  // namespace ovb
