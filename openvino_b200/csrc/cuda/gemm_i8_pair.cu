// Products of signed bytes, many tokens: pairs of CTAs (tcgen05, cta_group::2, kind::i8).
//
// What bounds it: the tensor pipe. A pair of SMs works on 256 tokens (the M side, 128 to each SM) x `bn` channels (256 or 128); every CTA loads its 128
// tokens and half of the weight rows, 32 KB for 256 x 256 x 128 products. The kernel is persistent and the accumulator exists twice in tensor memory
// (2 x 256 columns), so that the epilogue of a tile runs under the main loop of the next.
//  * warp 0: producer (TMA boxes of both operands; both CTAs' bytes are counted on the even CTA's barrier), warp 1 of the even CTA: MMAs of the pair
//  * warps 4 .. 11: epilogue. Tokens are the lanes, so a thread holds one row: adjacent channels lie in its registers, a gate and its up value too, and
//    results leave in whole 32-byte sectors. Scales, zero points and biases of the channels come from shared memory, the same for all lanes.
#include <mutex>
#include <stdlib.h>
#include <type_traits>

#include "gemm_i8.cuh"

namespace ovb {

constexpr int kI8PairMaxStages = 6;
constexpr int kI8PairThreads = 384;
constexpr int kI8PairStageBytes = 2 * kI8TileBytes;                      // 128 tokens and up to 128 weight rows
constexpr int kI8PairChannels = 256;                                     // channels of a tile at most
constexpr int kI8PairUnit = 64;                                          // channels that the epilogue takes at a time
constexpr int kI8PairBand = 8;                                           // token tiles per rasterisation band
constexpr int i8_pair_smem(int stages, int recv_bytes) { return stages * kI8PairStageBytes + recv_bytes + 2 * kI8PairChannels * 12 + 1024 + 1024; }

struct I8PairParams : I8Params {
    int bn;                       // channels of a tile: 256 or 128
    int tiles_n, tiles_t;
    int stages;
    int splits;                   // pairs that share the k-blocks of a tile (SPLIT)
    int recv_bytes;
    int whole;                    // 16-bit results and residuals in whole aligned sectors
    int prefetch;                 // k-blocks that weights are asked into L2 ahead
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

// The four products of a k-block and the commit of its stage in both CTAs (see umma_i8_block_elect).
__device__ __forceinline__ void pair_i8_block_elect(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint64_t* bar, uint16_t ctas) {
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
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(smem_u32(bar)), "h"(ctas)
        : "memory");
}
__device__ __forceinline__ void pair_commit_to_elect(uint64_t* bar, uint16_t ctas) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
        ::"r"(smem_u32(bar)), "h"(ctas)
        : "memory");
}

// 32 bytes at a time: one whole sector of the row that a lane owns
__device__ __forceinline__ void st_global_32(void* p, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void ld_global_32(const void* p, uint32_t* v) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p) : "memory");
}
// SPLIT: a cluster of `splits` pairs shares the k-blocks of one tile. The columns of the tile are shared out among the pairs: every CTA sends the partial
// sums of the others' columns from its registers into the shared memory of the CTA that finishes them for the same tokens.
template <bool F16, bool SPLIT, int FORM>
__global__ void __launch_bounds__(kI8PairThreads, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ I8PairParams p) {
    using E = typename Elem<F16>::type;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* recv = smem + p.stages * kI8PairStageBytes;
    float* chan_scale = reinterpret_cast<float*>(recv + p.recv_bytes);                          // [2][256] each
    float* chan_bias = chan_scale + 2 * kI8PairChannels;
    int* chan_zp = reinterpret_cast<int*>(chan_bias + 2 * kI8PairChannels);
    uint64_t* bars = reinterpret_cast<uint64_t*>(chan_zp + 2 * kI8PairChannels);
    uint64_t* full = bars;                              // [stages] even CTA: both CTAs' tiles have landed
    uint64_t* empty = bars + kI8PairMaxStages;          // [stages] both CTAs: the stage has been read
    uint64_t* acc_full = bars + 2 * kI8PairMaxStages;   // [2] both CTAs: accumulator complete
    uint64_t* acc_empty = acc_full + 2;                 // [2] even CTA: accumulator drained by the 16 epilogue warps of the pair
    uint64_t* received = acc_empty + 2;                 // the other pairs' sums of this CTA's columns have arrived
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(received + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* went_well = abort_flag + 1;           // [2]

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t cluster_rank = cluster_ctarank(), rank = cluster_rank & 1u, even = cluster_rank & ~1u;
    const int part = SPLIT ? (int)(cluster_rank >> 1) : 0;
    const uint16_t both = (uint16_t)(3u << even);
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 16);
        }
        mbar_init(received, 1);
        *abort_flag = 0;
        mbar_fence_init();
        if (SPLIT) mbar_arrive_expect_tx(received, (uint32_t)p.recv_bytes);
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
    const int ctas = SPLIT ? 2 * p.splits : 2;
    const int step = (int)gridDim.x / ctas, first = (int)blockIdx.x / ctas;
    const int kb0 = SPLIT ? (int)((int64_t)p.KB * part / p.splits) : 0, kb1 = SPLIT ? (int)((int64_t)p.KB * (part + 1) / p.splits) : p.KB;
    const int half_n = p.bn >> 1;                       // weight rows that a CTA loads
    // the rows of k-block kb of a tile's weights that this CTA loads, as they are packed: 128 of a chunk, chunk after chunk along K. Channels behind the last
    // chunk are not there: the box then reads the last chunk's again, and nothing of them is stored
    const int last_chunk = (p.N - 1) / TILE_N;
    auto weight_row = [&](int n0, int kb) {
        const int row = n0 + (int)rank * half_n;
        return (min(row / TILE_N, last_chunk) * p.KB + kb) * TILE_N + row % TILE_N;
    };
    auto prefetch = [&](int row) { bulk_prefetch_l2(p.w + (size_t)row * kI8BlockK, (uint32_t)(half_n * kI8BlockK)); };
    if (warp == 0 && lane == 0) {                       // weights are constants: they start for L2 before the tokens are there
        int t0, n0;
        if (i8_pair_tile(p, first, t0, n0))
            for (int kb = kb0; kb < min(kb1, kb0 + p.prefetch); ++kb) prefetch(weight_row(n0, kb));
    }
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int s = 0, t0, n0;
            uint32_t phase = 1;
            bool ok = true;
            const uint32_t tx = 2u * (kI8TileBytes + half_n * kI8BlockK);
            for (int idx = first; ok && i8_pair_tile(p, idx, t0, n0); idx += step) {
                int w_row = weight_row(n0, kb0);
                const int x_row = t0 + (int)rank * 128;
                for (int kb = kb0; kb < kb1; ++kb) {
                    ok = mbar_wait(&empty[s], phase, abort_flag, p.status);
                    if (!ok) break;
                    const uint32_t st = smem_u32(smem) + s * kI8PairStageBytes, bar = smem_u32(&full[s]);
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], tx);
                    if (kb + p.prefetch < kb1) prefetch(w_row + p.prefetch * TILE_N);
                    pair_load_2d(st, &tmX, bar, kb * kI8BlockK, x_row);
                    pair_load_2d(st + kI8TileBytes, &tmW, bar, 0, w_row);
                    w_row += TILE_N;
                    if (++s == p.stages) { s = 0; phase ^= 1; }
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
            // no way out of the loops: once a wait has run out all later ones return at once, and what is computed then is not stored
            for (int idx = first; i8_pair_tile(p, idx, t0, n0); idx += step) {
                mbar_wait(&acc_empty[buf], acc_phase, abort_flag, p.status);
                tc_fence_after_sync();
                const uint32_t d = tmem_base + uint32_t(buf * 256);
                for (int kb = kb0; kb < kb1; ++kb) {
                    mbar_wait(&full[s], phase, abort_flag, p.status);
                    tc_fence_after_sync();
                    const uint64_t da = desc0 + (uint64_t)((s * kI8PairStageBytes) >> 4), db = da + (uint64_t)(kI8TileBytes >> 4);
                    pair_i8_block_elect(d, da, db, idesc, kb > kb0 ? 1u : 0u, &empty[s], both);
                    if (++s == p.stages) { s = 0; phase ^= 1; }
                }
                pair_commit_to_elect(&acc_full[buf], both);
                if (++buf == 2) { buf = 0; acc_phase ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3, half = (warp - 4) >> 2, tid = threadIdx.x - 128;
        constexpr bool GATED = i8_gated_form(FORM);
        const uint32_t drained0 = dsmem_addr(smem_u32(&acc_empty[0]), even);
        const int units = p.bn / kI8PairUnit, own = SPLIT ? units / p.splits : units, unit0 = part * own;      // this CTA finishes `own` units from unit0 on
        const int out_cols = GATED ? p.N >> 1 : p.N;
        // A unit is 64 columns of the tile, two runs of 32: neighbours, or the gate and the up values of the same channels (rows 0 .. 63 of a weight tile are
        // the gate). A warp takes 16 columns of each run.
        auto run_at = [&](int u, int run) { return (GATED ? (u >> 1) * 128 + (u & 1) * 32 + run * 64 : u * 64 + run * 32) + half * 16; };
        // where the 16 bytes of four columns (from column 4 quad of run `run` of a CTA's unit u) of this thread's token arrive
        auto box = [&](int slot, int u, int run, int quad) { return ((((slot * own + u) * 2 + run) * 2 + half) * 4 + quad) * 2048 + (q * 32 + lane) * 16; };
        int buf = 0, t0, n0;
        uint32_t acc_phase = 0;
        for (int idx = first; i8_pair_tile(p, idx, t0, n0); idx += step) {
            const int t = t0 + (int)rank * 128 + q * 32 + lane;
            const bool row = t < p.T;
            const float xs = row ? __ldcg(p.x_scale + t) : 0.f;
            const int sum = row ? __ldcg(p.x_sum + t) : 0;
            float* cs = chan_scale + buf * kI8PairChannels;
            float* cb = chan_bias + buf * kI8PairChannels;
            int* cz = chan_zp + buf * kI8PairChannels;
            if (tid < p.bn) {
                const int n = n0 + tid;
                cs[tid] = n < p.N ? __ldg(p.w_scale + n) : 0.f;
                cb[tid] = n < p.N && p.bias != nullptr ? to_float(static_cast<const E*>(p.bias)[n]) : 0.f;
                cz[tid] = n < p.N && p.w_zp != nullptr ? __ldg(p.w_zp + n) : 0;
            }
            // one thread polls and says how it ended; the others wait at the barrier, so that all eight warps go on or leave together
            if (tid == 0) went_well[buf] = mbar_wait(&acc_full[buf], acc_phase, abort_flag, p.status) ? 1 : 0;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (!went_well[buf]) break;
            tc_fence_after_sync();
            const uint32_t src = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(buf * 256);
            auto drained = [&]() {                      // the accumulator has been read by this warp
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_cluster(drained0 + buf * 8);
            };
            if (SPLIT) {
                for (int o = 1; o < p.splits; ++o) {
                    const int to = (part + o) % p.splits, slot = part < to ? part : part - 1;      // the receiver's slots leave itself out
                    const uint32_t there = dsmem_addr(smem_u32(recv), (uint32_t)(2 * to) + rank), bar = dsmem_addr(smem_u32(received), (uint32_t)(2 * to) + rank);
                    for (int u = 0; u < own; ++u) {
                        uint32_t r[32];
                        tmem_ld_x16(src + run_at(to * own + u, 0), r);
                        tmem_ld_x16(src + run_at(to * own + u, 1), r + 16);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; ++i) st_async_v4(there + box(slot, u, i >> 2, i & 3), r + 4 * i, bar);
                    }
                }
                if (tid == 0) went_well[1] = mbar_wait(received, 0, abort_flag, p.status) ? 1 : 0;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (!went_well[1]) break;
            }
            uint8_t* out_row = static_cast<uint8_t*>(p.out) + (size_t)t * p.ldo * (p.out_f32 ? 4 : 2);
            const E* res_row = static_cast<const E*>(p.residual) + (size_t)t * p.ldr;
            // 16 finished values of this row from column `col` on; WHOLE: 16-bit results in whole aligned sectors
            auto put = [&](auto kind, const float* v, int col) {
                constexpr bool WHOLE = decltype(kind)::value;
                const bool there = row && col < out_cols;
                const E* r = res_row + col;
                if (WHOLE) {
                    uint32_t raw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                    if (!GATED && p.residual != nullptr) {
                        if (there) ld_global_32(r, raw);
                        const E* e = reinterpret_cast<const E*>(raw);
                        float w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = v[i] + to_float(e[i]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) raw[i] = pack_pair<E>(w[2 * i], w[2 * i + 1]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) raw[i] = pack_pair<E>(v[2 * i], v[2 * i + 1]);
                    }
                    if (there) st_global_32(reinterpret_cast<E*>(out_row) + col, raw);
                } else if (there) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (col + i < out_cols) {
                            const float w = p.residual != nullptr ? v[i] + to_float(r[i]) : v[i];
                            if (p.out_f32) reinterpret_cast<float*>(out_row)[col + i] = w;
                            else reinterpret_cast<E*>(out_row)[col + i] = from_float<E>(w);
                        }
                }
            };
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
            auto finish = [&](auto kind) {
#pragma unroll 1
                for (int u = unit0; u < unit0 + own; ++u) {
                    uint32_t r[32];
                    tmem_ld_x16(src + run_at(u, 0), r);
                    tmem_ld_x16(src + run_at(u, 1), r + 16);
                    tmem_ld_wait();
                    if (u + 1 == unit0 + own) drained();
                    if (SPLIT) {
                        for (int slot = 0; slot + 1 < p.splits; ++slot)
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const uint4 w = *reinterpret_cast<const uint4*>(recv + box(slot, u - unit0, i >> 2, i & 3));
                                r[4 * i] += w.x; r[4 * i + 1] += w.y; r[4 * i + 2] += w.z; r[4 * i + 3] += w.w;
                            }
                    }
                    float v[32];
                    values(r, run_at(u, 0), v);
                    values(r + 16, run_at(u, 1), v + 16);
                    if (GATED) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = i8_gate(p, v[i], v[16 + i]);
                        put(kind, v, (n0 >> 1) + u * 32 + half * 16);
                    } else {
                        if (FORM == kI8Any && p.act != OVB_ACT_NONE) apply_act_n(v, p);
                        put(kind, v, n0 + run_at(u, 0));
                        put(kind, v + 16, n0 + run_at(u, 1));
                    }
                }
            };
            if (p.whole) finish(std::true_type());
            else finish(std::false_type());
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

static cudaLaunchConfig_t i8_pair_config(unsigned grid, int ctas, int smem, cudaStream_t stream, cudaLaunchAttribute (&attr)[2]) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kI8PairThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cfg;
}

// Pairs of CTAs that are resident at a time, asked once per device.
template <bool F16, bool SPLIT, int FORM>
static int resident_i8_pairs(int* pairs) {
    static std::mutex mu;
    static int known[64] = {0};
    int dev = 0;
    OVB_CHECK_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (known[dev & 63] == 0) {
        const int smem = i8_pair_smem(kI8PairMaxStages, 0);
        OVB_CHECK_CUDA(cudaFuncSetAttribute(gemm_i8_pair_kernel<F16, SPLIT, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        cudaLaunchAttribute attr[2];
        cudaLaunchConfig_t cfg = i8_pair_config(148, 2, smem, nullptr, attr);
        cfg.numAttrs = 1;
        int n = 0;
        OVB_CHECK_CUDA(cudaOccupancyMaxActiveClusters(&n, gemm_i8_pair_kernel<F16, SPLIT, FORM>, &cfg));
        known[dev & 63] = n < 1 ? 1 : n;
    }
    *pairs = known[dev & 63];
    return 0;
}

template <bool F16, bool SPLIT, int FORM>
static int launch_i8_pair(const CUtensorMap& tmW, const CUtensorMap& tmX, const I8PairParams& p, cudaStream_t stream) {
    int pairs = 0;
    if (int rc = resident_i8_pairs<F16, SPLIT, FORM>(&pairs)) return rc;
    const int64_t tiles = (int64_t)p.tiles_n * p.tiles_t;
    const unsigned grid = SPLIT ? 2 * p.splits * (unsigned)tiles : 2 * (unsigned)(tiles < pairs ? tiles : pairs);
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = i8_pair_config(grid, 2 * p.splits, i8_pair_smem(p.stages, p.recv_bytes), stream, attr);
    OVB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, gemm_i8_pair_kernel<F16, SPLIT, FORM>, tmW, tmX, p));
    return 0;
}
template <bool F16, bool SPLIT>
static int launch_i8_pair(int form, const CUtensorMap& tmW, const CUtensorMap& tmX, const I8PairParams& p, cudaStream_t stream) {
    switch (form) {
        case kI8Plain: return launch_i8_pair<F16, SPLIT, kI8Plain>(tmW, tmX, p, stream);
        case kI8Gated: return launch_i8_pair<F16, SPLIT, kI8Gated>(tmW, tmX, p, stream);
        case kI8GatedZp: return launch_i8_pair<F16, SPLIT, kI8GatedZp>(tmW, tmX, p, stream);
        default: return launch_i8_pair<F16, SPLIT, kI8Any>(tmW, tmX, p, stream);
    }
}

int gemm_i8_pair(const ovb_gemm_i8_args* a, const I8Params& base, cudaStream_t stream) {
    I8PairParams p;
    static_cast<I8Params&>(p) = base;
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    const int out_cols = is_gated(a->act) ? a->N / 2 : a->N;
    p.whole = !a->out_f32 && out_cols % 16 == 0 && a->ldo % 16 == 0 && (bits(a->out) & 31) == 0 && (a->residual == nullptr || (a->ldr % 16 == 0 && (bits(a->residual) & 31) == 0));
    p.tiles_t = ceil_div(a->T, 256);
    p.bn = getenv("OVB_I8_BN") ? atoi(getenv("OVB_I8_BN")) : 256;
    p.splits = getenv("OVB_I8_PS") ? atoi(getenv("OVB_I8_PS")) : 1;
    p.prefetch = getenv("OVB_I8_PF") ? atoi(getenv("OVB_I8_PF")) : 0;
    p.tiles_n = ceil_div(a->N, p.bn);
    p.recv_bytes = (p.splits - 1) * (p.bn / p.splits) * 128 * 4;
    p.stages = kI8PairMaxStages - (p.recv_bytes + kI8PairStageBytes - 1) / kI8PairStageBytes;
    CUtensorMap tmW, tmX;
    if (int rc = make_tmap_2d(&tmX, a->x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->T, a->K, a->ldx, 128, kI8BlockK, true)) return rc;
    // the chunks are already in the swizzled order of the MMA: plain boxes of rows of 128 bytes
    if (int rc = make_tmap_2d(&tmW, a->w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)ceil_div(a->N, TILE_N) * p.KB * TILE_N, kI8BlockK, kI8BlockK, p.bn / 2, kI8BlockK, false)) return rc;
    const int form = i8_form(a);
    if (p.splits > 1) return a->f16 ? launch_i8_pair<true, true>(form, tmW, tmX, p, stream) : launch_i8_pair<false, true>(form, tmW, tmX, p, stream);
    return a->f16 ? launch_i8_pair<true, false>(form, tmW, tmX, p, stream) : launch_i8_pair<false, false>(form, tmW, tmX, p, stream);
}

}  // namespace ovb
