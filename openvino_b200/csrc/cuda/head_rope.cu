// Between the query / key / value projection and the attention: RMS norm of every query and key head, rotation by the position, and, for a serving
// step, the key and value rows of the new tokens into the paged cache. One pass over the projection.
//
//   y = x * rsqrt(mean_D(x^2) + eps) * w (where there are weights);  pairs (i, i + rot / 2), or (2 i, 2 i + 1) in the interleaved form, become
//   (a cos - b sin, b cos + a sin) * mult of the angle positions[t] * inv_freq[i];  dimensions from rot on stay.
//
// The angle is a product in 64 bits whose whole turns are taken off before anything is rounded to 32 bits: at position 100000 a 32-bit product is up to
// 4e-3 off, more than a bf16 rounding of the result. The angles of a token are the same for all heads: a block computes them once, in shared
// memory, while its first heads are on their way. Sums, norms and rotation are held in 32 bits, every result is rounded once.
//
// What bounds it: memory, each head read and written once. Eight elements of a head, two pieces of four, lie in one lane: the pair of a
// dimension is in the same lane, and the lanes of a head (8, 16 or 32) need shuffles for the sum of squares only.
#include "gemm_common.cuh"

namespace ovb {

struct HeadRopeParams : ovb_qk_rope_args {
    int* status;
    int heads, per_block;         // all heads of a token; heads of a block
};

constexpr int kRopeThreads = 256;
constexpr int kRopeBatch = 4;     // heads that a group of lanes has in flight

__device__ __forceinline__ float2 turn_of(int position, float inv_freq, float mult) {
    const double turns = (double)position * (double)inv_freq * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    return make_float2(c * mult, s * mult);
}

struct HeadAt {
    const void* src;              // + element
    void* dst;                    // NULL: not kept
    __half2* meta;
    int kind;                     // 0 query, 1 key, 2 value
};

template <class E, bool U8>
__device__ __forceinline__ HeadAt head_at(const HeadRopeParams& p, int b, int s, int h, int64_t slot) {
    HeadAt r;
    r.meta = nullptr;
    if (h < p.Hq) {
        r.kind = 0;
        r.src = static_cast<const E*>(p.q) + b * p.q_batch + s * p.q_token + h * p.q_head;
        r.dst = static_cast<E*>(p.q_out) + b * p.qo_batch + s * p.qo_token + h * p.qo_head;
        return r;
    }
    const bool value = h >= p.Hq + p.Hkv;
    const int g = value ? h - p.Hq - p.Hkv : h - p.Hq;
    r.kind = value ? 2 : 1;
    r.src = value ? static_cast<const E*>(p.v) + b * p.v_batch + s * p.v_token + g * p.v_head : static_cast<const E*>(p.k) + b * p.k_batch + s * p.k_token + g * p.k_head;
    if (p.k_cache == nullptr) {
        r.dst = static_cast<E*>(p.k_out) + b * p.ko_batch + s * p.ko_token + g * p.ko_head;
    } else if (slot < 0) {
        r.dst = nullptr;
    } else {
        const int64_t row = (slot / p.block_size * p.Hkv + g) * p.block_size + slot % p.block_size;
        void* cache = value ? p.v_cache : p.k_cache;
        r.dst = U8 ? static_cast<void*>(static_cast<uint8_t*>(cache) + row * p.D) : static_cast<void*>(static_cast<E*>(cache) + row * p.D);
        if (U8) r.meta = static_cast<__half2*>(value ? p.v_meta : p.k_meta) + row;
    }
    return r;
}

// The slot of a token, -1 where its rows are not kept.
__device__ __forceinline__ int64_t slot_of(const HeadRopeParams& p, int t) {
    if (p.k_cache == nullptr) return -1;
    const int slot = p.slot_map[t];
    if (slot >= p.slots) {
        if (threadIdx.x == 0) report_status(p.status, STATUS_BAD_INDEX);
        return -1;
    }
    return slot;
}

template <class E>
__device__ __forceinline__ void unpack4(uint2 raw, float (&v)[4]) {
    const E* e = reinterpret_cast<const E*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_float(e[i]);
}
template <class E>
__device__ __forceinline__ uint2 pack4(const float (&v)[4]) {
    E e[4] = {from_float<E>(v[0]), from_float<E>(v[1]), from_float<E>(v[2]), from_float<E>(v[3])};
    return *reinterpret_cast<uint2*>(e);
}

// Head sizes that are multiples of 8 up to 256, rotations that are multiples of 8, aligned heads. LANES lanes share a head.
template <class E, bool INTER, int LANES, bool U8>
__global__ void __launch_bounds__(kRopeThreads) head_rope_kernel(const __grid_constant__ HeadRopeParams p) {
    __shared__ float2 turn[128];
    constexpr int GROUPS = kRopeThreads / LANES;
    const int t = blockIdx.x, b = t / p.S, s = t - b * p.S;
    const int group = threadIdx.x / LANES, l = threadIdx.x % LANES;
    const int h_begin = blockIdx.y * p.per_block, h_end = min(p.heads, h_begin + p.per_block);
    const bool own = l * 8 < p.D;                       // this lane has elements
    const int pair0 = l * 4, half = p.rot >> 1;
    const bool turns = own && pair0 < half;
    // the two pieces of four elements; behind the rotated dimensions, and in the interleaved form, they are neighbours
    const int o0 = turns && !INTER ? pair0 : pair0 * 2, o1 = turns && !INTER ? half + pair0 : pair0 * 2 + 4;
    pdl_enter();
    float wq[8], wk[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) wq[j] = wk[j] = 1.f;
    if (own && p.q_norm != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) wq[j] = to_float(static_cast<const E*>(p.q_norm)[(j < 4 ? o0 : o1 - 4) + j]);
    }
    if (own && p.k_norm != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) wk[j] = to_float(static_cast<const E*>(p.k_norm)[(j < 4 ? o0 : o1 - 4) + j]);
    }
    const int64_t slot = slot_of(p, t);
    const int position = p.positions[b * p.pos_batch + s];
    bool have_turns = false;
    for (int base = h_begin; base < h_end; base += GROUPS * kRopeBatch) {
        uint2 r0[kRopeBatch], r1[kRopeBatch];
#pragma unroll
        for (int i = 0; i < kRopeBatch; ++i) {
            const int h = base + i * GROUPS + group;
            r0[i] = r1[i] = make_uint2(0, 0);
            if (h < h_end && own) {
                const E* src = static_cast<const E*>(head_at<E, U8>(p, b, s, h, slot).src);
                r0[i] = *reinterpret_cast<const uint2*>(src + o0);
                r1[i] = *reinterpret_cast<const uint2*>(src + o1);
            }
        }
        if (!have_turns) {
            if ((int)threadIdx.x < half) turn[threadIdx.x] = turn_of(position, p.inv_freq[threadIdx.x], p.mult);
            __syncthreads();
            have_turns = true;
        }
#pragma unroll
        for (int i = 0; i < kRopeBatch; ++i) {
            const int h = base + i * GROUPS + group;
            if (base + i * GROUPS >= h_end) break;      // the same for all threads of the block
            const bool live = h < h_end && own;
            const HeadAt at = head_at<E, U8>(p, b, s, h < h_end ? h : h_begin, slot);
            float a[4], c[4];
            unpack4<E>(r0[i], a);
            unpack4<E>(r1[i], c);
            const bool norm = at.kind == 0 ? p.q_norm != nullptr : at.kind == 1 && p.k_norm != nullptr;
            if (p.q_norm != nullptr || p.k_norm != nullptr) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) ss = fmaf(a[j], a[j], fmaf(c[j], c[j], ss));
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (norm) {
                    const float inv = rsqrtf(ss / (float)p.D + p.eps);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        a[j] = a[j] * inv * (at.kind == 0 ? wq[j] : wk[j]);
                        c[j] = c[j] * inv * (at.kind == 0 ? wq[4 + j] : wk[4 + j]);
                    }
                }
            }
            if (turns && at.kind != 2) {
                if (INTER) {
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        const float2 u = turn[pair0 + (j >> 1)], w = turn[pair0 + 2 + (j >> 1)];
                        const float a0 = a[j], c0 = c[j];
                        a[j] = a0 * u.x - a[j + 1] * u.y;
                        a[j + 1] = a[j + 1] * u.x + a0 * u.y;
                        c[j] = c0 * w.x - c[j + 1] * w.y;
                        c[j + 1] = c[j + 1] * w.x + c0 * w.y;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 u = turn[pair0 + j];
                        const float a0 = a[j];
                        a[j] = a0 * u.x - c[j] * u.y;
                        c[j] = c[j] * u.x + a0 * u.y;
                    }
                }
            }
            if (!U8 || at.kind == 0) {
                if (live && at.dst != nullptr) {
                    E* dst = static_cast<E*>(at.dst);
                    *reinterpret_cast<uint2*>(dst + o0) = pack4<E>(a);
                    *reinterpret_cast<uint2*>(dst + o1) = pack4<E>(c);
                }
            }
            if (U8) {
                // the arithmetic of ovb_rope_kv_write_u8: the pair is stored as fp16, so rows are quantised with the values that the reader will see
                float mn = INFINITY, mx = -INFINITY;
                if (own) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mn = fminf(mn, fminf(a[j], c[j]));
                        mx = fmaxf(mx, fmaxf(a[j], c[j]));
                    }
                }
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) {
                    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                }
                if (live && at.kind != 0 && at.dst != nullptr) {
                    float scale = __half2float(__float2half_rn((mx - mn) * (1.0f / 255.0f)));
                    if (!(scale > 0.f)) scale = 1.0f;
                    const float zp = __half2float(__float2half_rn(-mn / scale));
                    uint32_t w0 = 0, w1 = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        w0 |= (uint32_t)fminf(fmaxf(rintf(a[j] / scale + zp), 0.f), 255.f) << (8 * j);
                        w1 |= (uint32_t)fminf(fmaxf(rintf(c[j] / scale + zp), 0.f), 255.f) << (8 * j);
                    }
                    uint8_t* dst = static_cast<uint8_t*>(at.dst);
                    *reinterpret_cast<uint32_t*>(dst + o0) = w0;
                    *reinterpret_cast<uint32_t*>(dst + o1) = w1;
                    if (l == 0) *at.meta = __floats2half2_rn(scale, zp);
                }
            }
        }
    }
}

// Any even head size, rotation, pitch and alignment (16-bit rows): a warp per head, one element pair at a time.
template <class E>
__global__ void __launch_bounds__(kRopeThreads) head_rope_any_kernel(const __grid_constant__ HeadRopeParams p) {
    extern __shared__ float2 turn_any[];
    const int t = blockIdx.x, b = t / p.S, s = t - b * p.S;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h_begin = blockIdx.y * p.per_block, h_end = min(p.heads, h_begin + p.per_block);
    const int half = p.rot >> 1;
    pdl_enter();
    const int64_t slot = slot_of(p, t);
    const int position = p.positions[b * p.pos_batch + s];
    for (int i = threadIdx.x; i < half; i += kRopeThreads) turn_any[i] = turn_of(position, p.inv_freq[i], p.mult);
    __syncthreads();
    for (int h = h_begin + warp; h < h_end; h += kRopeThreads / 32) {
        const HeadAt at = head_at<E, false>(p, b, s, h, slot);
        if (at.dst == nullptr) continue;
        const E* src = static_cast<const E*>(at.src);
        E* dst = static_cast<E*>(at.dst);
        const E* w = static_cast<const E*>(at.kind == 0 ? p.q_norm : at.kind == 1 ? p.k_norm : nullptr);
        float inv = 1.f;
        if (w != nullptr) {
            float ss = 0.f;
            for (int d = lane; d < p.D; d += 32) ss = fmaf(to_float(src[d]), to_float(src[d]), ss);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv = rsqrtf(ss / (float)p.D + p.eps);
        }
        auto value = [&](int d) { return w != nullptr ? to_float(src[d]) * inv * to_float(w[d]) : to_float(src[d]); };
        const int turned = at.kind == 2 ? 0 : half;
        for (int i = lane; i < turned; i += 32) {
            const int d0 = p.interleaved ? 2 * i : i, d1 = p.interleaved ? 2 * i + 1 : half + i;
            const float a = value(d0), c = value(d1);
            const float2 u = turn_any[i];
            dst[d0] = from_float<E>(a * u.x - c * u.y);
            dst[d1] = from_float<E>(c * u.x + a * u.y);
        }
        for (int d = 2 * turned + lane; d < p.D; d += 32) dst[d] = from_float<E>(value(d));
    }
}

template <class E, bool INTER, bool U8>
static cudaError_t run_head_rope(const HeadRopeParams& p, dim3 grid, cudaStream_t stream) {
    if (p.D <= 64) return launch_pdl(head_rope_kernel<E, INTER, 8, U8>, grid, dim3(kRopeThreads), 0, stream, p);
    if (p.D <= 128) return launch_pdl(head_rope_kernel<E, INTER, 16, U8>, grid, dim3(kRopeThreads), 0, stream, p);
    return launch_pdl(head_rope_kernel<E, INTER, 32, U8>, grid, dim3(kRopeThreads), 0, stream, p);
}
template <class E>
static cudaError_t run_head_rope(const HeadRopeParams& p, dim3 grid, cudaStream_t stream) {
    if (p.kv_u8) return p.interleaved ? run_head_rope<E, true, true>(p, grid, stream) : run_head_rope<E, false, true>(p, grid, stream);
    return p.interleaved ? run_head_rope<E, true, false>(p, grid, stream) : run_head_rope<E, false, false>(p, grid, stream);
}

}  // namespace ovb

extern "C" int ovb_qk_norm_rope(const ovb_qk_rope_args* a, ovb_stream_t stream_) {
    using namespace ovb;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    OVB_REQUIRE(a && a->q && a->q_out && a->k && a->positions, "ovb_qk_norm_rope: null operand");
    OVB_REQUIRE(a->B > 0 && a->S > 0 && a->Hq > 0 && a->Hkv > 0 && (int64_t)a->B * a->S <= INT32_MAX, "ovb_qk_norm_rope: empty problem B=%d S=%d Hq=%d Hkv=%d", a->B, a->S, a->Hq, a->Hkv);
    OVB_REQUIRE(a->D > 0 && a->D % 2 == 0 && a->D <= 4096 && a->rot >= 0 && a->rot % 2 == 0 && a->rot <= a->D, "ovb_qk_norm_rope: head size %d, rotation %d", a->D, a->rot);
    OVB_REQUIRE(a->rot == 0 || a->inv_freq, "ovb_qk_norm_rope: a rotation needs frequencies");
    const bool cache = a->k_cache != nullptr;
    OVB_REQUIRE(cache ? a->v_cache && a->v && a->slot_map && a->block_size > 0 && a->slots > 0 : a->k_out && !a->v && !a->kv_u8,
                "ovb_qk_norm_rope: keys go to k_out, or with the values and their slots to the caches");
    HeadRopeParams p;
    static_cast<ovb_qk_rope_args&>(p) = *a;
    p.status = status_word();
    p.heads = a->Hq + a->Hkv * (cache ? 2 : 1);
    const int tokens = a->B * a->S;
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    uintptr_t at = bits(a->q) | bits(a->q_out) | bits(a->k) | bits(a->k_out) | bits(a->v) | (a->kv_u8 ? 0 : bits(a->k_cache) | bits(a->v_cache));
    int64_t pitch = a->q_batch | a->q_token | a->q_head | a->k_batch | a->k_token | a->k_head | a->qo_batch | a->qo_token | a->qo_head;
    pitch |= cache ? a->v_batch | a->v_token | a->v_head : a->ko_batch | a->ko_token | a->ko_head;
    const bool pieces = a->D % 8 == 0 && a->D <= 256 && a->rot % 8 == 0 && (at & 7) == 0 && (pitch & 3) == 0;
    if (a->kv_u8) {
        OVB_REQUIRE(a->k_meta && a->v_meta, "ovb_qk_norm_rope: a u8 cache needs its (scale, zero point) tables");
        OVB_REQUIRE(pieces && ((bits(a->k_cache) | bits(a->v_cache) | bits(a->k_meta) | bits(a->v_meta)) & 3) == 0,
                    "ovb_qk_norm_rope: the u8 cache is served for head sizes and rotations that are multiples of 8 up to 256, in heads that are 8-byte aligned");
    }
    // heads of a block: all from 512 tokens on (a block per token then fills every SM three times); with fewer, as many as its lanes take at a time
    const int lanes = a->D <= 64 ? 8 : a->D <= 128 ? 16 : 32, at_a_time = pieces ? kRopeThreads / lanes : kRopeThreads / 32;
    p.per_block = tokens >= 512 ? p.heads : at_a_time;
    const dim3 grid(tokens, ceil_div(p.heads, p.per_block));
    OVB_REQUIRE(grid.y <= 65535, "ovb_qk_norm_rope: %d heads", p.heads);
    if (pieces) OVB_CHECK_CUDA(a->f16 ? run_head_rope<__half>(p, grid, stream) : run_head_rope<__nv_bfloat16>(p, grid, stream));
    else OVB_CHECK_CUDA(launch_pdl(a->f16 ? head_rope_any_kernel<__half> : head_rope_any_kernel<__nv_bfloat16>, grid, dim3(kRopeThreads), (size_t)(a->rot >> 1) * sizeof(float2), stream, p));
    return 0;
}
