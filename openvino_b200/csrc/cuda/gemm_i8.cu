// Products of signed bytes on the tensor cores (tcgen05, kind::i8, 32-bit integer sums in tensor memory): the entry point, the weights' packing and
// the kernel of few tokens.
//
// The kernel: a CTA works on 128 weight rows (the M side) and up to 256 tokens (N); where that leaves SMs without work the k-blocks of a tile are
// shared by a cluster of up to eight CTAs. Nothing has to be expanded, so a stage is one bulk copy of a 16 KB weight chunk, packed in the swizzled
// order that the MMA reads, and one TMA box of tokens; rows behind the last token and columns behind K come as zeros. Weights are fetched before
// the kernel that wrote the tokens has finished. The partial sums are integers: they go to shared memory as [token][channel], every CTA of the cluster
// adds up its share of the tokens over all partials and finishes them, lanes along the channels.
#include <mutex>

#include "gemm_i8.cuh"

namespace ovb {

constexpr int kI8Threads = 128;
constexpr int kI8MaxStages = 12;

struct I8TileParams : I8Params {
    int bt, stages, splits;
};

template <class E>
__device__ __forceinline__ void i8_store4(const I8Params& p, int t, int col, int cols, float (&v)[4]) {
    // four adjacent columns of a token: one 8- or 16-byte access where all of them exist and the place is aligned
    if (p.residual != nullptr) {
        const E* r = static_cast<const E*>(p.residual) + (size_t)t * p.ldr + col;
        if (col + 4 <= cols && (reinterpret_cast<uintptr_t>(r) & 7) == 0) {
            const uint2 raw = __ldcg(reinterpret_cast<const uint2*>(r));
            const E* e = reinterpret_cast<const E*>(&raw);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += to_float(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < cols) v[i] += to_float(r[i]);
        }
    }
    if (p.out_f32) {
        float* o = static_cast<float*>(p.out) + (size_t)t * p.ldo + col;
        if (col + 4 <= cols && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
            *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < cols) o[i] = v[i];
        }
        return;
    }
    E* o = static_cast<E*>(p.out) + (size_t)t * p.ldo + col;
    E e[4] = {from_float<E>(v[0]), from_float<E>(v[1]), from_float<E>(v[2]), from_float<E>(v[3])};
    if (col + 4 <= cols && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
        *reinterpret_cast<uint2*>(o) = *reinterpret_cast<uint2*>(e);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < cols) o[i] = e[i];
    }
}

template <bool F16>
__global__ void __launch_bounds__(kI8Threads) gemm_i8_tile_kernel(const __grid_constant__ CUtensorMap tmX, const I8TileParams p) {
    using E = typename Elem<F16>::type;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int stage_bytes = kI8TileBytes + p.bt * kI8BlockK;
    __shared__ uint64_t full[kI8MaxStages], empty[kI8MaxStages], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;      // a cluster is the splits of one tile
    const int n0 = tile * TILE_N, t0 = blockIdx.y * p.bt;
    const int kb0 = (int)((int64_t)p.KB * split / p.splits), kb1 = (int)((int64_t)p.KB * (split + 1) / p.splits);
    const uint32_t tmem_cols = p.bt <= 32 ? 32u : p.bt <= 64 ? 64u : p.bt <= 128 ? 128u : 256u;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        abort_word = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tmX);
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
                bulk_load_1d(smem + i * stage_bytes, w + (size_t)i * kI8TileBytes, kI8TileBytes, &full[i]);
            }
            pdl_wait();
            for (int i = 0; i < ahead; ++i) tma_load_2d(smem + i * stage_bytes + kI8TileBytes, &tmX, &full[i], (kb0 + i) * kI8BlockK, t0);
            int s = 0;
            uint32_t phase = 0;
            for (int i = ahead; i < n; ++i) {
                if (!mbar_wait(&empty[s], phase, abort_flag, p.status)) break;
                mbar_arrive_expect_tx(&full[s], (uint32_t)stage_bytes);
                bulk_load_1d(smem + s * stage_bytes, w + (size_t)i * kI8TileBytes, kI8TileBytes, &full[s]);
                tma_load_2d(smem + s * stage_bytes + kI8TileBytes, &tmX, &full[s], (kb0 + i) * kI8BlockK, t0);
                if (++s == p.stages) { s = 0; phase ^= 1; }
            }
            if (OVB_PDL_GEMM) pdl_trigger();
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc_i8(TILE_N, p.bt);
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            ok = mbar_wait(&full[s], phase, abort_flag, p.status);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t a = smem_u32(smem) + s * stage_bytes;
            const uint64_t da = umma_desc_k_sw128(a, 1024), db = umma_desc_k_sw128(a + kI8TileBytes, 1024);
#pragma unroll
            for (int k = 0; k < kI8BlockK / 32; ++k) umma_i8_ss_elect(tmem, da + 2 * k, db + 2 * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
            umma_commit_elect(&empty[s]);
            if (++s == p.stages) { s = 0; phase ^= 1; }
        }
        if (ok) umma_commit_elect(&done);
        __syncwarp();
    }
    // every thread reads what the kernel before this one wrote (the tokens' scales), or writes over what it read
    pdl_wait();
    mbar_wait(&done, 0, abort_flag, p.status);
    __syncthreads();
    const bool fine = *abort_flag == 0;
    // every copy has landed and every MMA has read its operands: the stages hold the partial sums now
    int* part = reinterpret_cast<int*>(smem);           // [bt][128]
    if (fine) {
        tc_fence_after_sync();
        for (int c = 0; c < p.bt; c += 16) {
            uint32_t r[16];
            tmem_ld_x16(tmem + (uint32_t(warp * 32) << 16) + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) part[(c + j) * TILE_N + warp * 32 + lane] = (int)r[j];
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
        const int tokens = min(p.bt, p.T - t0), share0 = tokens * split / p.splits, share1 = tokens * (split + 1) / p.splits;
        const bool gated = is_gated(p.act);
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
        const uint32_t mine = smem_u32(part) + lane * 16;
        for (int t = share0 + warp; t < share1; t += kI8Threads / 32) {
            int4 a = make_int4(0, 0, 0, 0);
            if (p.splits > 1) {
                for (int r = 0; r < p.splits; ++r) {
                    const float4 f = ld_dsmem_f4(dsmem_addr(mine + t * (TILE_N * 4), (uint32_t)r));
                    a.x += __float_as_int(f.x); a.y += __float_as_int(f.y); a.z += __float_as_int(f.z); a.w += __float_as_int(f.w);
                }
            } else {
                a = *reinterpret_cast<const int4*>(part + t * TILE_N + lane * 4);
            }
            const float xs = __ldcg(p.x_scale + t0 + t);
            const int sum = p.w_zp != nullptr ? __ldcg(p.x_sum + t0 + t) : 0;
            float v[4] = {i8_value(a.x, zp[0], sum, xs * ws[0]) + b[0], i8_value(a.y, zp[1], sum, xs * ws[1]) + b[1],
                          i8_value(a.z, zp[2], sum, xs * ws[2]) + b[2], i8_value(a.w, zp[3], sum, xs * ws[3]) + b[3]};
            if (gated) {
                // rows 0 .. 63 of the tile are the gate, 64 .. 127 the up values of the same channels
                float u[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = __shfl_down_sync(0xffffffffu, v[i], 16);
                if (lane < 16) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = p.act == OVB_ACT_SWIGLU ? v[i] / (1.0f + __expf(-v[i])) * u[i] : glu_limited(p, v[i], u[i]);
                    i8_store4<E>(p, t0 + t, (n0 >> 1) + lane * 4, p.N >> 1, v);
                }
            } else {
                apply_act_n(v, p);
                i8_store4<E>(p, t0 + t, n, p.N, v);
            }
        }
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

template <bool F16>
static int set_up_i8_tile() {
    static std::mutex mu;
    static bool known[64] = {false};
    int dev = 0;
    OVB_CHECK_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (!known[dev & 63]) {
        OVB_CHECK_CUDA(cudaFuncSetAttribute(gemm_i8_tile_kernel<F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
        known[dev & 63] = true;
    }
    return 0;
}

static int run_i8_tile(const ovb_gemm_i8_args* a, const I8Params& base, cudaStream_t stream) {
    I8TileParams p;
    static_cast<I8Params&>(p) = base;
    p.bt = a->T <= 256 ? (a->T + 15) / 16 * 16 : 256;
    const int tiles = ceil_div(a->N, TILE_N), rows = ceil_div(a->T, p.bt);
    p.splits = 1;
    while (p.splits < 8 && (int64_t)tiles * rows * p.splits * 2 <= 160 && p.KB >= p.splits * 2) p.splits *= 2;
    const int stage = kI8TileBytes + p.bt * kI8BlockK;
    const int per_split = ceil_div(p.KB, p.splits);
    p.stages = (216 * 1024) / stage;
    if (p.stages > kI8MaxStages) p.stages = kI8MaxStages;
    if (p.stages > per_split) p.stages = per_split;
    int bytes = p.stages * stage;
    if (bytes < p.bt * TILE_N * 4) bytes = p.bt * TILE_N * 4;
    CUtensorMap tm;
    if (int rc = make_tmap_2d(&tm, a->x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->T, a->K, a->ldx, p.bt, kI8BlockK, true)) return rc;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(tiles * p.splits, rows);
    cfg.blockDim = dim3(kI8Threads);
    cfg.dynamicSmemBytes = bytes + 1024;
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
    if (a->f16) {
        if (int rc = set_up_i8_tile<true>()) return rc;
        OVB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, gemm_i8_tile_kernel<true>, tm, p));
    } else {
        if (int rc = set_up_i8_tile<false>()) return rc;
        OVB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, gemm_i8_tile_kernel<false>, tm, p));
    }
    return 0;
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
    if (a->raw != nullptr) {
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
    p.KB = ceil_div(a->K, kI8BlockK);
    p.ldo = a->ldo; p.ldr = a->ldr;
    p.act = a->act; p.out_f32 = a->out_f32;
    p.act_limit = a->act_limit; p.act_slope = a->act_slope; p.act_shift = a->act_shift;
    return a->T > 256 ? gemm_i8_pair(a, p, stream) : run_i8_tile(a, p, stream);
}

}  // extern "C"
