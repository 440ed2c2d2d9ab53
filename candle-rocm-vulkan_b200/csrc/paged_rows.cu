// Rows into and out of a pool of cache pages, and rotary positions with several axes.
//
// A rotary position turns the pairs (u, v) of a head's first `rot` elements: u' = u cos a - v sin a, v' = v cos a + u sin a, with the
// angle a = position on the pair's axis x the pair's frequency. The turn by -a (inverse) is its transpose, and so its gradient.
// MXFP8: per 32 elements the power of two 2^(floor(log2 max) - 8) and the E4M3 codes of x over it, the codes and scales that
// quant_rows16_kernel writes.
//
// All three kernels are bound by memory: every element is read once and written once, in 16-byte pieces (8 elements a lane), a
// head's row by neighbouring lanes of one warp. The two elements of a pair that lie rot / 2 apart meet by a shuffle. A warp has
// one token: its lanes form the token's angles once (in f64: a position of a million times an f32 frequency has 48 bits), keep
// the eight pairs of theirs in registers and go over the token's heads, four rows' loads on their way at a time. Where tokens
// are few, a token's rows are shared among several warps, so that one decode step is one wave of short warps.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace b200 {

int pool_params(const B200PagedPool &pool, const char *what, PoolParams *p) {
    if (pool.dtype != B200_F16 && pool.dtype != B200_BF16 && pool.dtype != B200_FP8)
        return set_error(B200_ERR_BAD_ARG, "%s: a pool holds f16, bf16 or MXFP8 (B200_FP8), got dtype %d", what, pool.dtype);
    if (pool.n_blocks == 0 || pool.block_rows == 0 || pool.hkv == 0) return set_error(B200_ERR_BAD_ARG, "%s: an empty pool", what);
    if (pool.n_blocks >= (1u << 31) || pool.block_rows >= (1u << 24))
        return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: pages of %u rows, %u of them", what, pool.block_rows, pool.n_blocks);
    const bool mx = pool.dtype == B200_FP8;
    if (pool.d == 0 || pool.d > 256 || pool.d % (mx ? 32 : 8))
        return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: head dim %u (multiples of %d up to 256)", what, pool.d, mx ? 32 : 8);
    if (!pool.k || !pool.v || (mx && (!pool.k_scale || !pool.v_scale))) return set_error(B200_ERR_BAD_ARG, "%s: null pool pointer", what);
    const uint64_t es = mx ? 1 : 2;
    uint64_t low = reinterpret_cast<uintptr_t>(pool.k) | reinterpret_cast<uintptr_t>(pool.v);
    if (mx) low |= reinterpret_cast<uintptr_t>(pool.k_scale) | reinterpret_cast<uintptr_t>(pool.v_scale);
    for (int i = 0; i < 3; ++i) low |= (pool.k_strides[i] | pool.v_strides[i]) * es;
    if (low & 15) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: the pool's rows must start at multiples of 16 bytes", what);
    *p = PoolParams{static_cast<char *>(pool.k), static_cast<char *>(pool.v), mx ? pool.k_scale : nullptr, mx ? pool.v_scale : nullptr,
                    pool.k_strides[0] * es, pool.k_strides[1] * es, pool.k_strides[2] * es, pool.v_strides[0] * es, pool.v_strides[1] * es, pool.v_strides[2] * es,
                    pool.n_blocks, pool.block_rows, pool.hkv, pool.d, 0, 0};
    pool_div_init(pool.block_rows, &p->div_mul, &p->div_shr);
    return B200_OK;
}

constexpr int PR_WARPS = 4;  // per block

struct RotaryParams {
    const float *freq;
    const uint8_t *axis;
    const int64_t *pos;
    uint64_t pos_stride;
    uint32_t n_axes, rot;
    float sign;  // -1: turned back
};
// one operand of a call: heads rows per token
struct HeadsParams {
    const char *src;
    char *dst;
    uint64_t s_t, s_h, d_t, d_h;  // bytes
    uint32_t heads;
};
struct RowsParams {
    HeadsParams q, k, v;  // v.heads = 0: rotary_axes; k.dst and v.dst null: they go to the pool
    PoolParams pool;
    RotaryParams rot;
    const int64_t *slots;
    int32_t *status;
    uint32_t tokens, d, parts;  // warps per token
};

// eight elements as they are: four words of 16-bit elements, eight of f32
template <int DT>
struct Raw {
    static constexpr int N = DT == B200_F32 ? 8 : 4;
    uint32_t w[N];
};
template <int DT>
__device__ __forceinline__ void load8(const char *src, bool vec, Raw<DT> &r) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < Raw<DT>::N / 4; ++i) {
            const uint4 a = reinterpret_cast<const uint4 *>(src)[i];
            r.w[4 * i] = a.x, r.w[4 * i + 1] = a.y, r.w[4 * i + 2] = a.z, r.w[4 * i + 3] = a.w;
        }
    } else if (DT == B200_F32) {
#pragma unroll
        for (int i = 0; i < Raw<DT>::N; ++i) r.w[i] = reinterpret_cast<const uint32_t *>(src)[i];
    } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(src);
#pragma unroll
        for (int i = 0; i < Raw<DT>::N; ++i) r.w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
    }
}
// two elements as a pair of f32: the row kernels are bound by their instructions where rows are many, and multiply two at a time
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair2(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float lo2(f32x2 v) { return u2f((uint32_t)v); }
__device__ __forceinline__ float hi2(f32x2 v) { return u2f((uint32_t)(v >> 32)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
template <int DT>
__device__ __forceinline__ void values8(const Raw<DT> &r, f32x2 (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == B200_F32) x[i] = pair2(u2f(r.w[2 * i % Raw<DT>::N]), u2f(r.w[(2 * i + 1) % Raw<DT>::N]));
        else if (DT == B200_BF16) x[i] = pair2(u2f(r.w[i] << 16), u2f(r.w[i] & 0xffff0000u));
        else x[i] = pair2(f16_bits_to_f((uint16_t)r.w[i]), f16_bits_to_f((uint16_t)(r.w[i] >> 16)));
    }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const f32x2 (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == B200_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(hi2(x[i])), "f"(lo2(x[i])));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(hi2(x[i])), "f"(lo2(x[i])));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int DT>
__device__ __forceinline__ void store8(char *dst, bool vec, const f32x2 (&x)[4]) {
    if (DT == B200_F32) {
        if (vec) {
            *reinterpret_cast<float4 *>(dst) = make_float4(lo2(x[0]), hi2(x[0]), lo2(x[1]), hi2(x[1]));
            *reinterpret_cast<float4 *>(dst + 16) = make_float4(lo2(x[2]), hi2(x[2]), lo2(x[3]), hi2(x[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<float *>(dst)[2 * i] = lo2(x[i]), reinterpret_cast<float *>(dst)[2 * i + 1] = hi2(x[i]);
        }
    } else {
        const uint4 w = pack8<DT>(x);
        if (vec) {
            *reinterpret_cast<uint4 *>(dst) = w;
        } else {
            uint16_t *h = reinterpret_cast<uint16_t *>(dst);
            const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) h[2 * i] = (uint16_t)a[i], h[2 * i + 1] = (uint16_t)(a[i] >> 16);
        }
    }
}
// eight elements of a block of 32 (four lanes) -> codes and the block's scale; every lane of the row takes part
__device__ __forceinline__ uint2 mx8(const f32x2 (&x)[4], uint32_t &scale) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(lo2(x[i])), fabsf(hi2(x[i]))));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    scale = mx_scale_code(m, 8);
    if (scale == 0) return make_uint2(0u, 0u);  // a block of zeros (or with an infinity) has codes of zero
    const float r = e8m0_recip(scale);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x2 a = mul2(x[2 * i], pair2(r, r)), b = mul2(x[2 * i + 1], pair2(r, r));
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(hi2(a)), "f"(lo2(a)));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(hi2(b)), "f"(lo2(b)));
        w[i] = lo | (uint32_t)hi << 16;
    }
    // a magnitude of 0x7f is a NaN, which keeps its sign
    if ((((w[0] & 0x7f7f7f7fu) + 0x01010101u) | ((w[1] & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = f_to_e4m3(__fmul_rn(lo2(x[2 * i]), r)) | f_to_e4m3(__fmul_rn(hi2(x[2 * i]), r)) << 8 | f_to_e4m3(__fmul_rn(lo2(x[2 * i + 1]), r)) << 16 |
                   f_to_e4m3(__fmul_rn(hi2(x[2 * i + 1]), r)) << 24;
    }
    return make_uint2(w[0], w[1]);
}

// TURN: 0 nothing is turned, 1 pairs rot / 2 apart, 2 neighbouring pairs. POOL: 0 none (rotary_axes), 1 16-bit elements, 2 MXFP8;
// PDT: the 16-bit pool's type. LPR: lanes per row (8, 16 or 32).
// Bound by bytes and by latency alike, so the warps that fit count: 64 registers, eight blocks of four warps per SM (three of eight with 80: 46.2 us for
// 40.0, 8 191 tokens turned and written as MXFP8), and short blocks, since a token or half of one is all that a warp does. Chosen on bf16: f32 elements whose
// pairs lie half a head apart spill (5 003 tokens, 32 / 8 heads of 128: 52.2 us, neighbours 42.1, 31.7 at the copy's rate).
template <int DT, int TURN, int POOL, int PDT, int LPR>
__global__ void __launch_bounds__(PR_WARPS * 32, 8) paged_rows_kernel(const RowsParams p, const bool vec) {
    constexpr int RPW = 32 / LPR, PR_BATCH = 4;
    __shared__ float2 s_cs[PR_WARPS][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane % LPR, sub = lane / LPR;
    const uint64_t unit = (uint64_t)blockIdx.x * PR_WARPS + warp;
    const uint32_t token = (uint32_t)(unit / p.parts), part = (uint32_t)(unit % p.parts);
    if (token >= p.tokens) return;  // whole warps; nothing below waits for another warp
    const bool in = (uint32_t)c * 8 < p.d;
    const uint32_t half = p.rot.rot / 2;

    const uint32_t step = p.parts * RPW, mine = part * RPW;
    f32x2 co[4], si[4];
    int partner = lane;
    bool turned = false;
    if (TURN) {
        for (uint32_t f = lane; f < half; f += 32) {
            const uint32_t a = p.rot.axis ? min((uint32_t)p.rot.axis[f], p.rot.n_axes - 1) : 0u;
            // the angle in turns; its whole turns leave before it is rounded to f32, and what the rounding leaves (up to 2^-25 of a half turn, as much as
            // all other roundings of a turned element together) turns sine and cosine a little further
            const double t = (double)p.rot.pos[a * p.rot.pos_stride + token] * (double)p.rot.freq[f] * 0.15915494309189533577, h = 2.0 * (t - rint(t));
            const float hi = (float)h, lo = (float)(h - (double)hi) * 3.14159265358979f;
            float s0, k0;
            sincospif(hi, &s0, &k0);
            const float s = fmaf(lo, k0, s0), k = fmaf(-lo, s0, k0);
            s_cs[warp][f] = make_float2(k, s * p.rot.sign);
        }
        __syncwarp();
        turned = (uint32_t)c * 8 < p.rot.rot;
        if (turned) {
            if (TURN == 1) {
                const bool second = (uint32_t)c * 8 >= half;
                const uint32_t f0 = (uint32_t)c * 8 - (second ? half : 0u);
                partner = second ? lane - (int)(half / 8) : lane + (int)(half / 8);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 a = s_cs[warp][f0 + 2 * i], b = s_cs[warp][f0 + 2 * i + 1];
                    co[i] = pair2(a.x, b.x);
                    si[i] = second ? pair2(a.y, b.y) : pair2(-a.y, -b.y);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 cs = s_cs[warp][c * 4 + i];
                    co[i] = pair2(cs.x, cs.x);
                    si[i] = pair2(-cs.y, cs.y);
                }
            }
        }
    }
    int64_t slot = 0;
    uint32_t blk = 0, row = 0;
    bool kept = true;
    if (POOL) {
        slot = p.slots[token];
        const uint64_t cap = (uint64_t)p.pool.n_blocks * p.pool.block_rows;
        kept = slot >= 0 && (uint64_t)slot < cap;
        if (slot >= 0 && !kept && p.status && lane == 0 && part == 0) atomicExch(p.status, 3);
        if (kept) {
            blk = (uint32_t)((uint64_t)slot / p.pool.block_rows);
            row = (uint32_t)((uint64_t)slot - (uint64_t)blk * p.pool.block_rows);
        }
    }

    // The token's rows, q's heads, then k's, then v's, are dealt out to its warps RPW at a time. One operand's: a batch of loads, then the elements.
    auto operand = [&](uint32_t first, const HeadsParams &h, auto turn, auto store) {
        uint32_t r0 = mine;
        if (first >= r0 + RPW) r0 += (first - r0 - RPW + step) / step * step;  // the first of the warp's that reaches into the operand
        const char *src = h.src + token * h.s_t + (uint64_t)c * 8 * dtype_size(DT);
#pragma unroll 1
        for (; r0 < first + h.heads; r0 += PR_BATCH * step) {
            Raw<DT> raw[PR_BATCH];
#pragma unroll
            for (int j = 0; j < PR_BATCH; ++j) {
                const uint32_t hd = r0 + j * step + sub - first;  // (a row of the operand in front: out of range)
                if (hd < h.heads && in) load8<DT>(src + hd * h.s_h, vec, raw[j]);
                else
#pragma unroll
                    for (int i = 0; i < Raw<DT>::N; ++i) raw[j].w[i] = 0u;
            }
#pragma unroll
            for (int j = 0; j < PR_BATCH; ++j) {
                if (r0 + j * step >= first + h.heads) break;  // the whole warp
                const uint32_t hd = r0 + j * step + sub - first;
                f32x2 x[4];
                values8(raw[j], x);
                if (turn.value) {
                    f32x2 y[4];
                    if (TURN == 1) {
                        Raw<DT> other;
#pragma unroll
                        for (int i = 0; i < Raw<DT>::N; ++i) other.w[i] = __shfl_sync(0xffffffffu, raw[j].w[i], partner);
                        values8(other, y);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = pair2(hi2(x[i]), lo2(x[i]));
                    }
                    if (turned) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = fma2(x[i], co[i], mul2(y[i], si[i]));
                    }
                }
                store(hd, hd < h.heads && in, x);
            }
        }
    };
    using Turn = std::bool_constant<TURN != 0>;
    auto dense = [&](const HeadsParams &h) {
        char *dst = h.dst + token * h.d_t + (uint64_t)c * 8 * dtype_size(DT);
        const uint64_t d_h = h.d_h;
        return [dst, d_h, vec](uint32_t hd, bool there, const f32x2(&x)[4]) {
            if (there) store8<DT>(dst + hd * d_h, vec, x);
        };
    };
    if (p.q.heads) operand(0, p.q, Turn{}, dense(p.q));
    if constexpr (POOL == 0) {
        if (p.k.heads) operand(p.q.heads, p.k, Turn{}, dense(p.k));
    } else {
        auto pool = [&](char *plane, uint64_t sb, uint64_t sr, uint64_t sh, uint8_t *scales) {
            const uint32_t nb = p.pool.d / 32;
            char *dst = plane + blk * sb + row * sr + c * (POOL == 1 ? 16 : 8);
            uint8_t *sc = POOL == 2 ? scales + ((uint64_t)blk * p.pool.hkv * p.pool.block_rows + row) * nb + c / 4 : nullptr;
            const uint32_t sc_h = p.pool.block_rows * nb;
            const bool put = kept, first = (c & 3) == 0;
            return [=](uint32_t hd, bool there, const f32x2(&x)[4]) {
                if constexpr (POOL == 1) {
                    if (there && put) *reinterpret_cast<uint4 *>(dst + hd * sh) = pack8<PDT>(x);
                } else {
                    uint32_t scale;
                    const uint2 w = mx8(x, scale);
                    if (there && put) {
                        *reinterpret_cast<uint2 *>(dst + hd * sh) = w;
                        if (first) sc[(uint64_t)hd * sc_h] = (uint8_t)scale;
                    }
                }
            };
        };
        operand(p.q.heads, p.k, Turn{}, pool(p.pool.k, p.pool.k_sb, p.pool.k_sr, p.pool.k_sh, p.pool.ks));
        operand(p.q.heads + p.k.heads, p.v, std::false_type{}, pool(p.pool.v, p.pool.v_sb, p.pool.v_sr, p.pool.v_sh, p.pool.vs));
    }
}

template <int DT, int TURN, int POOL, int PDT>
static int rows_launch(const RowsParams &p, bool vec, cudaStream_t stream, const char *what) {
    const uint32_t chunks = p.d / 8, lpr = chunks <= 8 ? 8 : (chunks <= 16 ? 16 : 32), rows = p.q.heads + p.k.heads + p.v.heads;
    RowsParams r = p;
    // Two waves of warps and more (four where there is no pool): a warp goes over a whole token. Fewer tokens are shared among warps, down to one load a lane
    // (8 191 tokens into an MXFP8 pool: 40.0 us whole, 44.6 in halves; 5 003 turned alone, f32: 19.3 whole, 18.4 in thirds).
    const uint32_t most = std::max(1u, (rows * lpr + 31) / 32);
    r.parts = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(1, 148ull * 32 * (POOL ? 2 : 4) / std::max(p.tokens, 1u)));
    const uint64_t blocks = ((uint64_t)p.tokens * r.parts + PR_WARPS - 1) / PR_WARPS;
    if (blocks >= (1ull << 31)) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: %u tokens", what, p.tokens);
    if (lpr == 8) paged_rows_kernel<DT, TURN, POOL, PDT, 8><<<(unsigned)blocks, PR_WARPS * 32, 0, stream>>>(r, vec);
    else if (lpr == 16) paged_rows_kernel<DT, TURN, POOL, PDT, 16><<<(unsigned)blocks, PR_WARPS * 32, 0, stream>>>(r, vec);
    else paged_rows_kernel<DT, TURN, POOL, PDT, 32><<<(unsigned)blocks, PR_WARPS * 32, 0, stream>>>(r, vec);
    return check_launch(what);
}
template <int DT, int TURN>
static int rows_pool(const RowsParams &p, int pool, bool vec, cudaStream_t stream, const char *what) {
    switch (pool) {
    case B200_F16: return rows_launch<DT, TURN, 1, B200_F16>(p, vec, stream, what);
    case B200_BF16: return rows_launch<DT, TURN, 1, B200_BF16>(p, vec, stream, what);
    case B200_FP8: return rows_launch<DT, TURN, 2, B200_F16>(p, vec, stream, what);
    default: return TURN ? rows_launch<DT, TURN ? TURN : 1, 0, B200_F16>(p, vec, stream, what) : B200_OK;
    }
}
template <int DT>
static int rows_turn(const RowsParams &p, int turn, int pool, bool vec, cudaStream_t stream, const char *what) {
    if (turn == 1) return rows_pool<DT, 1>(p, pool, vec, stream, what);
    if (turn == 2) return rows_pool<DT, 2>(p, pool, vec, stream, what);
    return rows_pool<DT, 0>(p, pool, vec, stream, what);
}
static int rows_run(const RowsParams &p, int dtype, int turn, int pool, bool vec, cudaStream_t stream, const char *what) {
    if (dtype == B200_F32) return rows_turn<B200_F32>(p, turn, pool, vec, stream, what);
    if (dtype == B200_F16) return rows_turn<B200_F16>(p, turn, pool, vec, stream, what);
    return rows_turn<B200_BF16>(p, turn, pool, vec, stream, what);
}

static int rotary_params(const B200Rotary &a, uint32_t d, const char *what, RotaryParams *r) {
    if (a.n_axes == 0 || a.n_axes > 256) return set_error(B200_ERR_BAD_ARG, "%s: %u axes", what, a.n_axes);
    if (a.rot == 0 || a.rot > d || a.rot % 16) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: %u turned elements (multiples of 16 up to the head dim %u)", what, a.rot, d);
    *r = RotaryParams{a.freq, a.axis, a.pos, a.pos_stride, a.n_axes, a.rot, a.inverse ? -1.0f : 1.0f};
    return B200_OK;
}
static bool dtype_ok(int dt) { return dt == B200_F32 || dt == B200_F16 || dt == B200_BF16; }
static HeadsParams heads_params(const void *src, void *dst, const uint64_t (&ss)[2], const uint64_t (&ds)[2], uint32_t heads, uint64_t es) {
    return HeadsParams{static_cast<const char *>(src), static_cast<char *>(dst), ss[0] * es, ss[1] * es, ds[0] * es, ds[1] * es, heads};
}
// whether all of an operand's rows start on 16-byte boundaries
static bool aligned(const HeadsParams &h) {
    return h.heads == 0 || ((reinterpret_cast<uintptr_t>(h.src) | reinterpret_cast<uintptr_t>(h.dst) | h.s_t | h.s_h | h.d_t | h.d_h) & 15) == 0;
}

// ---- rows out of the pool ------------------------------------------------------------------------------------------------
struct UnpackParams {
    PoolParams pool;
    const int32_t *table;
    uint64_t table_stride;
    const uint32_t *cu;
    char *k, *v;
    uint64_t total;
    uint32_t b, table_cols, parts;
    int32_t *status;
};

// LPR lanes per row, eight elements each (sixteen codes a lane, and with them two stores of every other 16 bytes, took 48.9 us for 45).
template <int DT, int POOL, int PDT, int LPR>
__global__ void __launch_bounds__(PR_WARPS * 32) paged_unpack_kernel(const UnpackParams p) {
    constexpr int RPW = 32 / LPR, PR_BATCH = 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane % LPR, sub = lane / LPR;
    const uint64_t unit = (uint64_t)blockIdx.x * PR_WARPS + warp, t = unit / p.parts;
    const uint32_t part = (uint32_t)(unit % p.parts);
    const PoolParams &pl = p.pool;
    if (t >= p.total || t >= p.cu[p.b] || t < p.cu[0]) return;
    const uint32_t seq = pool_seq(p.cu, p.b, t, lane), j = (uint32_t)(t - p.cu[seq]);
    const uint32_t page = pool_div(j, pl.div_mul, pl.div_shr), row = j - page * pl.block_rows;
    const int id = page < p.table_cols ? p.table[seq * p.table_stride + page] : -1;
    const bool there = id >= 0 && (uint32_t)id < pl.n_blocks, in = (uint32_t)c * 8 < pl.d;
    if (!there && p.status && lane == 0 && part == 0) atomicExch(p.status, 3);
    const uint64_t blk = there ? (uint64_t)id : 0;
    // heads part x RPW + sub, and on by the step: k's and v's rows of each, addresses moved by sums alone
    constexpr int PIECE = POOL == 2 ? 8 : 16, ES = DT == B200_F32 ? 4 : 2;
    const uint32_t nb = pl.d / 32, step = p.parts * RPW, h0 = part * RPW + sub;
    const char *k_src = pl.k + blk * pl.k_sb + row * pl.k_sr + h0 * pl.k_sh + c * PIECE, *v_src = pl.v + blk * pl.v_sb + row * pl.v_sr + h0 * pl.v_sh + c * PIECE;
    const uint64_t k_step = step * pl.k_sh, v_step = step * pl.v_sh;
    uint64_t sc_at = POOL == 2 ? ((blk * pl.hkv + h0) * pl.block_rows + row) * nb + c / 4 : 0, to = ((t * pl.hkv + h0) * pl.d + c * 8) * ES;
    const uint64_t sc_step = (uint64_t)step * pl.block_rows * nb;
    const uint32_t to_step = step * pl.d * ES;
    auto out = [&](char *dst, const uint4 &w, uint32_t e) {
        if constexpr (POOL == 1 && DT == PDT) {
            *reinterpret_cast<uint4 *>(dst) = w;
        } else if constexpr (POOL == 1) {
            f32x2 x[4];
            Raw<PDT> raw;
            raw.w[0] = w.x, raw.w[1] = w.y, raw.w[2] = w.z, raw.w[3] = w.w;
            values8<PDT>(raw, x);
            store8<DT>(dst, true, x);
        } else if (DT == B200_BF16 || (DT == B200_F16 && e - 112u <= 30u)) {
            // a power of two that the type has: the product is exact, or rounded once
            constexpr bool B = DT == B200_BF16;
            uint32_t rest;
            const uint32_t f = pool_scale2<B>(e, e, rest);
            *reinterpret_cast<uint4 *>(dst) = make_uint4(pool_mul2<B>(pool_pair<B, 0>(w.x), f), pool_mul2<B>(pool_pair<B, 1>(w.x), f), pool_mul2<B>(pool_pair<B, 0>(w.y), f),
                                                         pool_mul2<B>(pool_pair<B, 1>(w.y), f));
        } else {
            const f32x2 s = pair2(e8m0_to_f(e), e8m0_to_f(e));
            const uint32_t a[2] = {w.x, w.y};
            f32x2 x[4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const uint32_t lo = cvt_e4m3x2_f16x2(a[y]), hi = cvt_e4m3x2_hi_f16x2(a[y]);  // exact
                x[2 * y] = mul2(pair2(f16_bits_to_f((uint16_t)lo), f16_bits_to_f((uint16_t)(lo >> 16))), s);
                x[2 * y + 1] = mul2(pair2(f16_bits_to_f((uint16_t)hi), f16_bits_to_f((uint16_t)(hi >> 16))), s);
            }
            store8<DT>(dst, true, x);
        }
    };
    const bool any_v = p.v != nullptr;
#pragma unroll 1
    for (uint32_t h = h0; h < pl.hkv + sub; h += PR_BATCH * step) {  // (the whole warp)
        uint4 w[PR_BATCH][2];
        uint32_t e[PR_BATCH][2];
#pragma unroll
        for (int i = 0; i < PR_BATCH; ++i) {
            const bool load = h + i * step < pl.hkv && in && there;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                w[i][x] = make_uint4(0u, 0u, 0u, 0u);
                e[i][x] = 127;
                if (!load || (x && !any_v)) continue;
                const char *src = x ? v_src : k_src;
                if (POOL == 1) {
                    w[i][x] = *reinterpret_cast<const uint4 *>(src);
                } else {
                    const uint2 a = *reinterpret_cast<const uint2 *>(src);
                    w[i][x].x = a.x, w[i][x].y = a.y;
                    e[i][x] = (x ? pl.vs : pl.ks)[sc_at];
                }
            }
            k_src += k_step, v_src += v_step, sc_at += sc_step;
        }
#pragma unroll
        for (int i = 0; i < PR_BATCH; ++i) {
            if (h + i * step < pl.hkv && in) {
                out(p.k + to, w[i][0], e[i][0]);
                if (any_v) out(p.v + to, w[i][1], e[i][1]);
            }
            to += to_step;
        }
    }
}

template <int DT, int POOL, int PDT>
static int unpack_launch(const UnpackParams &p, cudaStream_t stream) {
    const uint32_t chunks = p.pool.d / 8, lpr = chunks <= 8 ? 8 : (chunks <= 16 ? 16 : 32), rows = p.pool.hkv;
    UnpackParams r = p;
    const uint32_t most = std::max(1u, (rows * lpr + 31) / 32);
    r.parts = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(1, 148ull * 32 / p.total));
    const uint64_t blocks = (p.total * r.parts + PR_WARPS - 1) / PR_WARPS;
    if (blocks >= (1ull << 31)) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "paged_unpack: %llu rows", (unsigned long long)p.total);
    if (lpr == 8) paged_unpack_kernel<DT, POOL, PDT, 8><<<(unsigned)blocks, PR_WARPS * 32, 0, stream>>>(r);
    else if (lpr == 16) paged_unpack_kernel<DT, POOL, PDT, 16><<<(unsigned)blocks, PR_WARPS * 32, 0, stream>>>(r);
    else paged_unpack_kernel<DT, POOL, PDT, 32><<<(unsigned)blocks, PR_WARPS * 32, 0, stream>>>(r);
    return check_launch("paged_unpack");
}
template <int DT>
static int unpack_pool(const UnpackParams &p, int pool, cudaStream_t stream) {
    if (pool == B200_F16) return unpack_launch<DT, 1, B200_F16>(p, stream);
    if (pool == B200_BF16) return unpack_launch<DT, 1, B200_BF16>(p, stream);
    return unpack_launch<DT, 2, B200_F16>(p, stream);
}

}  // namespace b200

using namespace b200;

extern "C" int b200_rotary_axes(const B200RotaryArgs *a, b200_stream_t stream) {
    const char *what = "rotary_axes";
    if (!a) return set_error(B200_ERR_BAD_ARG, "%s: null args", what);
    if (!dtype_ok(a->dtype)) return set_error(B200_ERR_BAD_ARG, "%s: dtype %d (f32, f16, bf16)", what, a->dtype);
    if (a->d == 0 || a->d > 256 || a->d % 8) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: head dim %u (multiples of 8 up to 256)", what, a->d);
    RowsParams p = {};
    const int rc = rotary_params(a->rotary, a->d, what, &p.rot);
    if (rc) return rc;
    if (a->tokens == 0 || a->hq + a->hkv == 0) return B200_OK;
    if (!a->rotary.freq || !a->rotary.pos || (a->hq && (!a->q || !a->q_out)) || (a->hkv && (!a->k || !a->k_out))) return set_error(B200_ERR_BAD_ARG, "%s: null pointer", what);
    const uint64_t es = dtype_size(a->dtype);
    p.q = heads_params(a->q, a->q_out, a->q_strides, a->q_out_strides, a->hq, es);
    p.k = heads_params(a->k, a->k_out, a->k_strides, a->k_out_strides, a->hkv, es);
    p.tokens = a->tokens, p.d = a->d;
    return rows_run(p, a->dtype, a->rotary.interleaved ? 2 : 1, -1, aligned(p.q) && aligned(p.k), (cudaStream_t)stream, what);
}

extern "C" int b200_paged_append(const B200PagedAppendArgs *a, b200_stream_t stream) {
    const char *what = "paged_append";
    if (!a) return set_error(B200_ERR_BAD_ARG, "%s: null args", what);
    RowsParams p = {};
    int rc = pool_params(a->pool, what, &p.pool);
    if (rc) return rc;
    if (!dtype_ok(a->src_dtype)) return set_error(B200_ERR_BAD_ARG, "%s: dtype %d (f32, f16, bf16)", what, a->src_dtype);
    const bool turn = a->rotary.freq != nullptr;
    if (turn && (rc = rotary_params(a->rotary, a->pool.d, what, &p.rot))) return rc;
    const uint32_t hq = a->q ? a->hq : 0;
    if (hq && !turn) return set_error(B200_ERR_BAD_ARG, "%s: queries are given to be turned, but no frequencies", what);
    if (a->tokens == 0) return B200_OK;
    if (!a->k || !a->v || !a->slots || (hq && !a->q_out) || (turn && !a->rotary.pos)) return set_error(B200_ERR_BAD_ARG, "%s: null pointer", what);
    const uint64_t es = dtype_size(a->src_dtype), none[2] = {0, 0};
    p.q = heads_params(a->q, a->q_out, a->q_strides, a->q_out_strides, hq, es);
    p.k = heads_params(a->k, nullptr, a->k_strides, none, a->pool.hkv, es);
    p.v = heads_params(a->v, nullptr, a->v_strides, none, a->pool.hkv, es);
    p.slots = a->slots, p.status = a->status;
    p.tokens = a->tokens, p.d = a->pool.d;
    return rows_run(p, a->src_dtype, !turn ? 0 : (a->rotary.interleaved ? 2 : 1), a->pool.dtype, aligned(p.q) && aligned(p.k) && aligned(p.v), (cudaStream_t)stream, what);
}

extern "C" int b200_paged_unpack(const B200PagedUnpackArgs *a, b200_stream_t stream) {
    const char *what = "paged_unpack";
    if (!a) return set_error(B200_ERR_BAD_ARG, "%s: null args", what);
    UnpackParams p = {};
    const int rc = pool_params(a->pool, what, &p.pool);
    if (rc) return rc;
    if (!dtype_ok(a->dtype)) return set_error(B200_ERR_BAD_ARG, "%s: dtype %d (f32, f16, bf16)", what, a->dtype);
    if (a->total >= (1ull << 31)) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: %llu rows", what, (unsigned long long)a->total);
    if (a->b == 0 || a->total == 0) return B200_OK;
    if (!a->table || !a->cu_k || !a->k) return set_error(B200_ERR_BAD_ARG, "%s: null pointer", what);
    if ((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15) return set_error(B200_ERR_BAD_ARG, "%s: outputs must be 16-byte aligned", what);
    p.table = a->table, p.table_stride = a->table_stride, p.cu = a->cu_k;
    p.k = static_cast<char *>(a->k), p.v = static_cast<char *>(a->v);
    p.total = a->total, p.b = a->b, p.table_cols = a->table_cols, p.status = a->status;
    if (a->dtype == B200_F32) return unpack_pool<B200_F32>(p, a->pool.dtype, (cudaStream_t)stream);
    if (a->dtype == B200_F16) return unpack_pool<B200_F16>(p, a->pool.dtype, (cudaStream_t)stream);
    return unpack_pool<B200_BF16>(p, a->pool.dtype, (cudaStream_t)stream);
}
