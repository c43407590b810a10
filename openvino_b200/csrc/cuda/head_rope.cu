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
// What bounds it: memory, each head read and written once; next to it the instructions, about 250 for a warp's round of four heads of 128. A lane holds two
// pieces of a head: the partner of a dimension is in the same lane, and the lanes of a head need shuffles for the sum of squares only. Measured: 8 x 1024 tokens
// of 64 + 8 + 8 heads of 128 into a 16-bit cache 60.7 us (5.5 TB/s), 4 x 2048 tokens of 32 + 8 heads, half of each turned 32.2 us (5.2 TB/s), 1 token 2.8 us.
#include "gemm_common.cuh"

namespace ovb {

struct HeadRopeParams : ovb_qk_rope_args {
    int* status;
    int src_step[3], dst_step[3]; // from head to head, queries, keys, values: elements, bytes
    int heads;                    // of a token, all kinds
    int rounds_q, rounds_k, rounds;                     // of a warp over the query heads, the key heads, all heads of a token
    int parts, per_warp;          // warps of a token and their rounds
    float inv_d;
};

constexpr int kRopeThreads = 128;
// Blocks resident on an SM, and rounds of heads that a warp has in flight besides the one at work: many warps with one round each where there are tokens for
// them, deeper warps where a token's heads are spread over warps and few rounds are left to each. us, many / few: 8 x 1024 tokens of 64 + 8 + 8 heads of 128
// 60.7 / 71.5, 1500 tokens of 32 + 8 + 8 11.7 / 13.4, 700 tokens 7.1 / 6.0, 200 tokens 4.8 / 4.1.
constexpr int rope_blocks(bool many) { return many ? 7 : 5; }
constexpr int rope_ahead(bool many) { return many ? 1 : 2; }
constexpr int kRopeManyTokens = 148 * 7;

__device__ __forceinline__ float2 turn_of(int position, float inv_freq, float mult) {
    const double turns = (double)position * (double)inv_freq * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    return make_float2(c * mult, s * mult);
}

// Where a token's heads are: a base for each kind.
template <class E>
struct TokenRows {
    const E* src[3];
    uint8_t* dst[3];              // NULL: not kept
    int64_t row;                  // of the first key (value) head in the cache
    bool outside;                 // the slot is behind the cache
};

template <class E, bool U8>
__device__ __forceinline__ TokenRows<E> token_rows(const HeadRopeParams& p, int t) {
    TokenRows<E> r;
    const int b = t / p.S, s = t - b * p.S;
    r.src[0] = static_cast<const E*>(p.q) + b * p.q_batch + s * p.q_token;
    r.src[1] = static_cast<const E*>(p.k) + b * p.k_batch + s * p.k_token;
    r.src[2] = static_cast<const E*>(p.v) + b * p.v_batch + s * p.v_token;
    r.dst[0] = reinterpret_cast<uint8_t*>(static_cast<E*>(p.q_out) + b * p.qo_batch + s * p.qo_token);
    r.row = 0;
    r.outside = false;
    if (p.k_cache == nullptr) {
        r.dst[1] = reinterpret_cast<uint8_t*>(static_cast<E*>(p.k_out) + b * p.ko_batch + s * p.ko_token);
        r.dst[2] = nullptr;
        return r;
    }
    const int slot = p.slot_map[t], size = U8 ? 1 : (int)sizeof(E);
    const bool inside = slot < p.slots;
    r.outside = !inside;
    const int blk = slot / p.block_size, off = slot - blk * p.block_size;
    r.row = (int64_t)blk * p.Hkv * p.block_size + off;
    r.dst[1] = slot >= 0 && inside ? static_cast<uint8_t*>(p.k_cache) + r.row * p.D * size : nullptr;
    r.dst[2] = slot >= 0 && inside ? static_cast<uint8_t*>(p.v_cache) + r.row * p.D * size : nullptr;
    return r;
}

// CH elements side by side, 8 or 16 bytes.
template <class E, int CH>
struct Piece {
    uint32_t w[CH / 2];
    __device__ __forceinline__ void load(const E* src) {
        if (CH == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            w[0] = v.x; w[1] = v.y; w[CH / 2 - 2] = v.z; w[CH / 2 - 1] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(src);
            w[0] = v.x; w[1] = v.y;
        }
    }
    __device__ __forceinline__ void store(void* dst) const {
        if (CH == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[CH / 2 - 2], w[CH / 2 - 1]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    }
    __device__ __forceinline__ void unpack(float (&v)[CH]) const {
        const E* e = reinterpret_cast<const E*>(w);
#pragma unroll
        for (int i = 0; i < CH; ++i) v[i] = to_float(e[i]);
    }
    __device__ __forceinline__ void pack(const float (&v)[CH]) {
#pragma unroll
        for (int i = 0; i < CH; i += 2) w[i / 2] = pack_pair<E>(v[i], v[i + 1]);
    }
};

// Heads and rotations of whole pieces, aligned heads. LANES lanes share a head, each with two pieces of CH elements: the partners of its CH pairs, or 2 CH
// neighbours. A warp works alone, on a token's heads or a part of them, with the heads of the next rounds on their way. The heads of a round are of one kind
// (queries, keys, values), so everything that depends on the kind is the same for the warp. The norm's weights are multiplied into the cosines and sines when
// the kind changes; values on their way to a 16-bit cache are copied as they are.
template <class E, bool INTER, int CH, int LANES, bool U8, bool MANY>
__global__ void __launch_bounds__(kRopeThreads, rope_blocks(MANY)) head_rope_kernel(const __grid_constant__ HeadRopeParams p) {
    __shared__ float2 turn_of_warp[kRopeThreads / 32][128];
    constexpr int GROUPS = 32 / LANES, AHEAD = rope_ahead(MANY);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int id = blockIdx.x * (kRopeThreads / 32) + warp, t = id / p.parts;
    const int group = lane / LANES, l = lane % LANES;
    const int begin = (id - t * p.parts) * p.per_warp, end = min(p.rounds, begin + p.per_warp);
    const bool own = l * 2 * CH < p.D;                  // this lane has elements
    const int pair0 = l * CH, half = p.rot >> 1;
    const bool turns = own && pair0 < half;
    // behind the rotated dimensions, and in the interleaved form, the two pieces are neighbours
    const int o0 = turns && !INTER ? pair0 : pair0 * 2, o1 = turns && !INTER ? half + pair0 : pair0 * 2 + CH;
    pdl_enter();
    if (t >= p.B * p.S) return;                         // whole warps, which share nothing
    const TokenRows<E> rows = token_rows<E, U8>(p, t);
    auto kind_of = [&](int round) { return round < p.rounds_q ? 0 : round < p.rounds_q + p.rounds_k ? 1 : 2; };
    // this lane's head of a round, among those of its kind; negative: none
    auto head_of = [&](int round, int kind) {
        const int h = (round - (kind == 0 ? 0 : kind == 1 ? p.rounds_q : p.rounds_q + p.rounds_k)) * GROUPS + group;
        return own && h < (kind == 0 ? p.Hq : p.Hkv) ? h : -1;
    };
    auto pick = [&](const auto& of, int kind) { return kind == 0 ? of[0] : kind == 1 ? of[1] : of[2]; };
    Piece<E, CH> r0[AHEAD], r1[AHEAD];
    auto fetch = [&](int round, Piece<E, CH>& a, Piece<E, CH>& c) {
        if (round >= end) return;
        const int kind = kind_of(round), h = head_of(round, kind);
        if (h >= 0) {
            const E* src = pick(rows.src, kind) + (int64_t)h * pick(p.src_step, kind);
            a.load(src + o0);
            c.load(src + o1);
        } else {
#pragma unroll
            for (int j = 0; j < CH / 2; ++j) a.w[j] = c.w[j] = 0;
        }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(begin + i, r0[i], r1[i]);
    float2* turn = turn_of_warp[warp];
    const int position = p.positions[(t / p.S) * p.pos_batch + t % p.S];
    for (int i = lane; i < half; i += 32) turn[i] = turn_of(position, p.inv_freq[i], p.mult);
    __syncwarp();
    if (rows.outside && lane == 0) report_status(p.status, STATUS_BAD_INDEX);
    // of an element and of its partner, in the first and in the second piece; the weights alone where nothing turns
    float fa[CH], ga[CH], fc[CH], gc[CH];
    const E* weight = nullptr;
    auto factors = [&](int kind) {
        weight = static_cast<const E*>(kind == 0 ? p.q_norm : p.k_norm);
#pragma unroll
        for (int j = 0; j < CH; ++j) fa[j] = fc[j] = 1.f;
        if (weight != nullptr && own) {
            Piece<E, CH> w0, w1;
            w0.load(weight + o0);
            w1.load(weight + o1);
            w0.unpack(fa);
            w1.unpack(fc);
        }
        if (!turns) return;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            if (INTER) {
                if (j % 2) continue;
                const float2 u = turn[pair0 + j / 2], v = turn[pair0 + (CH + j) / 2];
                const float a0 = fa[j], a1 = fa[j + 1], c0 = fc[j], c1 = fc[j + 1];
                fa[j] = a0 * u.x;
                ga[j] = -a1 * u.y;
                fa[j + 1] = a1 * u.x;
                ga[j + 1] = a0 * u.y;
                fc[j] = c0 * v.x;
                gc[j] = -c1 * v.y;
                fc[j + 1] = c1 * v.x;
                gc[j + 1] = c0 * v.y;
            } else {
                const float2 u = turn[pair0 + j];
                ga[j] = -fc[j] * u.y;
                gc[j] = fa[j] * u.y;
                fa[j] *= u.x;
                fc[j] *= u.x;
            }
        }
    };
    int current = -1;
    for (int base = begin; base < end; base += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int round = base + i;
            if (round >= end) break;
            const int kind = kind_of(round), h = head_of(round, kind);
            Piece<E, CH> x0 = r0[i], x1 = r1[i];
            fetch(round + AHEAD, r0[i], r1[i]);
            uint8_t* dst = h >= 0 ? pick(rows.dst, kind) : nullptr;
            if (dst != nullptr) dst += (int64_t)h * pick(p.dst_step, kind);
            float a[CH], c[CH];
            if (kind != 2) {
                if (kind != current) factors(current = kind);
                x0.unpack(a);
                x1.unpack(c);
                if (weight != nullptr) {
                    uint64_t ss2 = pair_of(0.f);
#pragma unroll
                    for (int j = 0; j < CH; j += 2) ss2 = fma2(pair_of(a[j], a[j + 1]), pair_of(a[j], a[j + 1]), fma2(pair_of(c[j], c[j + 1]), pair_of(c[j], c[j + 1]), ss2));
                    float ss, ss1;
                    unpair(ss2, ss, ss1);
                    ss += ss1;
#pragma unroll
                    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const uint64_t inv = pair_of(rsqrtf(fmaf(ss, p.inv_d, p.eps)));
#pragma unroll
                    for (int j = 0; j < CH; j += 2) {
                        unpair(mul2(pair_of(a[j], a[j + 1]), inv), a[j], a[j + 1]);
                        unpair(mul2(pair_of(c[j], c[j + 1]), inv), c[j], c[j + 1]);
                    }
                }
                if (turns) {
#pragma unroll
                    for (int j = 0; j < CH; j += 2) {
                        if (INTER) {
                            const float a0 = a[j], c0 = c[j];
                            a[j] = fmaf(a[j + 1], ga[j], a0 * fa[j]);
                            a[j + 1] = fmaf(a0, ga[j + 1], a[j + 1] * fa[j + 1]);
                            c[j] = fmaf(c[j + 1], gc[j], c0 * fc[j]);
                            c[j + 1] = fmaf(c0, gc[j + 1], c[j + 1] * fc[j + 1]);
                        } else {
                            const uint64_t a2 = pair_of(a[j], a[j + 1]), c2 = pair_of(c[j], c[j + 1]);
                            unpair(fma2(c2, pair_of(ga[j], ga[j + 1]), mul2(a2, pair_of(fa[j], fa[j + 1]))), a[j], a[j + 1]);
                            unpair(fma2(a2, pair_of(gc[j], gc[j + 1]), mul2(c2, pair_of(fc[j], fc[j + 1]))), c[j], c[j + 1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < CH; ++j) {
                        a[j] *= fa[j];
                        c[j] *= fc[j];
                    }
                }
                x0.pack(a);
                x1.pack(c);
            } else if (U8) {
                x0.unpack(a);
                x1.unpack(c);
            }
            if ((!U8 || kind == 0) && dst != nullptr) {
                x0.store(reinterpret_cast<E*>(dst) + o0);
                x1.store(reinterpret_cast<E*>(dst) + o1);
            }
            if (U8 && kind != 0) {
                // the arithmetic of ovb_rope_kv_write_u8: the pair is stored as fp16, so rows are quantised with the values that the reader will see
                float mn = INFINITY, mx = -INFINITY;
                if (own) {
#pragma unroll
                    for (int j = 0; j < CH; ++j) {
                        mn = fminf(mn, fminf(a[j], c[j]));
                        mx = fmaxf(mx, fmaxf(a[j], c[j]));
                    }
                }
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) {
                    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                }
                if (dst != nullptr) {
                    float scale = __half2float(__float2half_rn((mx - mn) * (1.0f / 255.0f)));
                    if (!(scale > 0.f)) scale = 1.0f;
                    const float zp = __half2float(__float2half_rn(-mn / scale));
                    uint32_t w0[CH / 4], w1[CH / 4];
#pragma unroll
                    for (int j = 0; j < CH; ++j) {
                        const uint32_t b0 = (uint32_t)fminf(fmaxf(rintf(a[j] / scale + zp), 0.f), 255.f), b1 = (uint32_t)fminf(fmaxf(rintf(c[j] / scale + zp), 0.f), 255.f);
                        w0[j / 4] = j % 4 == 0 ? b0 : w0[j / 4] | b0 << (8 * (j % 4));
                        w1[j / 4] = j % 4 == 0 ? b1 : w1[j / 4] | b1 << (8 * (j % 4));
                    }
#pragma unroll
                    for (int j = 0; j < CH / 4; ++j) {
                        reinterpret_cast<uint32_t*>(dst + o0)[j] = w0[j];
                        reinterpret_cast<uint32_t*>(dst + o1)[j] = w1[j];
                    }
                    if (l == 0) static_cast<__half2*>(kind == 2 ? p.v_meta : p.k_meta)[rows.row + (int64_t)h * p.block_size] = __floats2half2_rn(scale, zp);
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
    const int half = p.rot >> 1;
    pdl_enter();
    const TokenRows<E> rows = token_rows<E, false>(p, t);
    if (rows.outside && threadIdx.x == 0) report_status(p.status, STATUS_BAD_INDEX);
    const int position = p.positions[b * p.pos_batch + s];
    for (int i = threadIdx.x; i < half; i += kRopeThreads) turn_any[i] = turn_of(position, p.inv_freq[i], p.mult);
    __syncthreads();
    for (int h = warp; h < p.heads; h += kRopeThreads / 32) {
        const int kind = h < p.Hq ? 0 : h < p.Hq + p.Hkv ? 1 : 2, g = kind == 0 ? h : kind == 1 ? h - p.Hq : h - p.Hq - p.Hkv;
        if (rows.dst[kind] == nullptr) continue;
        const E* src = rows.src[kind] + (int64_t)g * p.src_step[kind];
        E* dst = reinterpret_cast<E*>(rows.dst[kind] + (int64_t)g * p.dst_step[kind]);
        const E* w = static_cast<const E*>(kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr);
        float inv = 1.f;
        if (w != nullptr) {
            float ss = 0.f;
            for (int d = lane; d < p.D; d += 32) ss = fmaf(to_float(src[d]), to_float(src[d]), ss);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv = rsqrtf(fmaf(ss, p.inv_d, p.eps));
        }
        auto value = [&](int d) { return w != nullptr ? to_float(src[d]) * inv * to_float(w[d]) : to_float(src[d]); };
        const int turned = kind == 2 ? 0 : half;
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

template <class E, bool INTER, int CH, bool U8, bool MANY>
static cudaError_t run_head_rope(const HeadRopeParams& p, dim3 grid, int lanes, cudaStream_t stream) {
    constexpr int FEW = 32 / CH;
    auto kern = lanes == FEW       ? head_rope_kernel<E, INTER, CH, FEW, U8, MANY>
                : lanes == 2 * FEW ? head_rope_kernel<E, INTER, CH, 2 * FEW, U8, MANY>
                                   : head_rope_kernel<E, INTER, CH, 4 * FEW, U8, MANY>;
    return launch_pdl(kern, grid, dim3(kRopeThreads), 0, stream, p);
}
template <class E, bool INTER, int CH, bool U8>
static cudaError_t run_head_rope(const HeadRopeParams& p, dim3 grid, int lanes, bool many, cudaStream_t stream) {
    return many ? run_head_rope<E, INTER, CH, U8, true>(p, grid, lanes, stream) : run_head_rope<E, INTER, CH, U8, false>(p, grid, lanes, stream);
}
template <class E, bool INTER>
static cudaError_t run_head_rope(const HeadRopeParams& p, dim3 grid, int ch, int lanes, bool many, cudaStream_t stream) {
    if (ch == 8) return p.kv_u8 ? run_head_rope<E, INTER, 8, true>(p, grid, lanes, many, stream) : run_head_rope<E, INTER, 8, false>(p, grid, lanes, many, stream);
    return p.kv_u8 ? run_head_rope<E, INTER, 4, true>(p, grid, lanes, many, stream) : run_head_rope<E, INTER, 4, false>(p, grid, lanes, many, stream);
}
template <class E>
static cudaError_t run_head_rope(const HeadRopeParams& p, dim3 grid, int ch, int lanes, bool many, cudaStream_t stream) {
    return p.interleaved ? run_head_rope<E, true>(p, grid, ch, lanes, many, stream) : run_head_rope<E, false>(p, grid, ch, lanes, many, stream);
}

}  // namespace ovb

extern "C" int ovb_qk_norm_rope(const ovb_qk_rope_args* a, ovb_stream_t stream_) {
    using namespace ovb;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    OVB_REQUIRE(a && a->q && a->q_out && a->k && a->positions, "ovb_qk_norm_rope: null operand");
    OVB_REQUIRE(a->B > 0 && a->S > 0 && a->Hq > 0 && a->Hkv > 0 && (int64_t)a->B * a->S <= INT32_MAX - kRopeThreads, "ovb_qk_norm_rope: empty or too large a problem B=%d S=%d Hq=%d Hkv=%d", a->B, a->S, a->Hq, a->Hkv);
    OVB_REQUIRE(a->D > 0 && a->D % 2 == 0 && a->D <= 4096 && a->rot >= 0 && a->rot % 2 == 0 && a->rot <= a->D, "ovb_qk_norm_rope: head size %d, rotation %d", a->D, a->rot);
    OVB_REQUIRE(a->rot == 0 || a->inv_freq, "ovb_qk_norm_rope: a rotation needs frequencies");
    const bool cache = a->k_cache != nullptr;
    OVB_REQUIRE(cache ? a->v_cache && a->v && a->slot_map && a->block_size > 0 && a->slots > 0 : a->k_out && !a->v && !a->kv_u8,
                "ovb_qk_norm_rope: keys go to k_out, or with the values and their slots to the caches");
    HeadRopeParams p;
    static_cast<ovb_qk_rope_args&>(p) = *a;
    p.status = status_word();
    p.heads = a->Hq + a->Hkv * (cache ? 2 : 1);
    p.inv_d = 1.f / (float)a->D;
    const int64_t to_cache = (int64_t)a->block_size * a->D * (a->kv_u8 ? 1 : 2), steps[6] = {a->q_head, a->k_head, cache ? a->v_head : 0, a->qo_head * 2, cache ? to_cache : a->ko_head * 2, to_cache};
    for (int i = 0; i < 6; ++i) {
        OVB_REQUIRE(steps[i] >= 0 && steps[i] <= INT32_MAX, "ovb_qk_norm_rope: heads %lld apart", (long long)steps[i]);
        (i < 3 ? p.src_step : p.dst_step)[i % 3] = (int)steps[i];
    }
    const int tokens = a->B * a->S;
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    uintptr_t at = bits(a->q_norm) | bits(a->k_norm) | bits(a->q) | bits(a->q_out) | bits(a->k) | bits(a->k_out) | bits(a->v) | (a->kv_u8 ? 0 : bits(a->k_cache) | bits(a->v_cache));
    int64_t pitch = a->q_batch | a->q_token | a->q_head | a->k_batch | a->k_token | a->k_head | a->qo_batch | a->qo_token | a->qo_head;
    pitch |= cache ? a->v_batch | a->v_token | a->v_head : a->ko_batch | a->ko_token | a->ko_head;
    // elements of a lane's two pieces: eight where heads, rotation and alignment allow it, else four
    const int ch = a->D % 16 == 0 && a->rot % 16 == 0 && (at & 15) == 0 && (pitch & 7) == 0 ? 8 : 4;
    const bool pieces = a->D % 8 == 0 && a->D <= 256 && a->rot % 8 == 0 && (at & 7) == 0 && (pitch & 3) == 0;
    if (a->kv_u8) {
        OVB_REQUIRE(a->k_meta && a->v_meta, "ovb_qk_norm_rope: a u8 cache needs its (scale, zero point) tables");
        OVB_REQUIRE(pieces && ((bits(a->k_cache) | bits(a->v_cache) | bits(a->k_meta) | bits(a->v_meta)) & 3) == 0,
                    "ovb_qk_norm_rope: the u8 cache is served for head sizes and rotations that are multiples of 8 up to 256, in heads that are 8-byte aligned");
    }
    if (!pieces) {
        OVB_CHECK_CUDA(launch_pdl(a->f16 ? head_rope_any_kernel<__half> : head_rope_any_kernel<__nv_bfloat16>, dim3(tokens), dim3(kRopeThreads), (size_t)(a->rot >> 1) * sizeof(float2),
                                  stream, p));
        return 0;
    }
    // parts of a token's heads: as many as rounds while all warps are resident at a time, fewer with more tokens
    const int lanes = (a->D <= 64 ? 32 : a->D <= 128 ? 64 : 128) / ch, groups = 32 / lanes;
    p.rounds_q = ceil_div(a->Hq, groups);
    p.rounds_k = ceil_div(a->Hkv, groups);
    p.rounds = p.rounds_q + p.rounds_k * (cache ? 2 : 1);
    const bool many = tokens >= kRopeManyTokens;
    const int64_t room = 148ll * rope_blocks(many) * (kRopeThreads / 32);
    int parts = (int)(room / tokens);
    parts = parts < 1 ? 1 : parts > p.rounds ? p.rounds : parts;
    p.per_warp = ceil_div(p.rounds, parts);
    p.parts = ceil_div(p.rounds, p.per_warp);
    const int64_t blocks = ((int64_t)tokens * p.parts + kRopeThreads / 32 - 1) / (kRopeThreads / 32);
    OVB_REQUIRE(blocks <= INT32_MAX, "ovb_qk_norm_rope: %d tokens", tokens);
    OVB_CHECK_CUDA(a->f16 ? run_head_rope<__half>(p, dim3((unsigned)blocks), ch, lanes, many, stream) : run_head_rope<__nv_bfloat16>(p, dim3((unsigned)blocks), ch, lanes, many, stream));
    return 0;
}
