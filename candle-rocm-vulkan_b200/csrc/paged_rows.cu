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
// the eight pairs of theirs in registers and go over the token's heads, the next four rows' loads on their way while four are worked on. Where tokens
// are few, a token's rows are shared among several warps, so that one decode step is one wave of short warps.
#include <algorithm>

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

constexpr int PR_WARPS = 8;  // per block

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
template <int DT>
__device__ __forceinline__ void values8(const Raw<DT> &r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (DT == B200_F32) x[i] = u2f(r.w[i % Raw<DT>::N]);
        else if (DT == B200_BF16) x[i] = i & 1 ? u2f(r.w[i / 2] & 0xffff0000u) : u2f(r.w[i / 2] << 16);
        else x[i] = f16_bits_to_f((uint16_t)(r.w[i / 2] >> (16 * (i & 1))));
    }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (DT == B200_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int DT>
__device__ __forceinline__ void store8(char *dst, bool vec, const float (&x)[8]) {
    if (DT == B200_F32) {
        if (vec) {
            *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(dst + 16) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<float *>(dst)[i] = x[i];
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
__device__ __forceinline__ uint2 mx8(const float (&x)[8], uint32_t &scale) {
    float m = fabsf(x[0]), z = x[0] * 0.0f;
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, fabsf(x[i])), z = fmaf(x[i], 0.0f, z);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    scale = mx_scale_code(m, 8);
    uint32_t w[2] = {0u, 0u};
    if (scale != 0) {  // a block of zeros (or with an infinity) has codes of zero
        const float r = e8m0_recip(scale);
        if (z != z) {  // a NaN keeps its sign
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i >> 2] |= f_to_e4m3(__fmul_rn(x[i], r)) << (8 * (i & 3));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint16_t h;
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(__fmul_rn(x[2 * i + 1], r)), "f"(__fmul_rn(x[2 * i], r)));
                w[i >> 1] |= (uint32_t)h << (16 * (i & 1));
            }
        }
    }
    return make_uint2(w[0], w[1]);
}

// TURN: 0 nothing is turned, 1 pairs rot / 2 apart, 2 neighbouring pairs. POOL: 0 none (rotary_axes), 1 16-bit elements, 2 MXFP8;
// PDT: the 16-bit pool's type. LPR: lanes per row (8, 16 or 32).
// Measured: see the launcher.
template <int DT, int TURN, int POOL, int PDT, int LPR>
__global__ void __launch_bounds__(PR_WARPS * 32) paged_rows_kernel(const RowsParams p, const bool vec) {
    constexpr int RPW = 32 / LPR, PR_BATCH = DT == B200_F32 ? 2 : 4;
    __shared__ float2 s_cs[PR_WARPS][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane % LPR, sub = lane / LPR;
    const uint64_t unit = (uint64_t)blockIdx.x * PR_WARPS + warp;
    const uint32_t token = (uint32_t)(unit / p.parts), part = (uint32_t)(unit % p.parts);
    if (token >= p.tokens) return;  // whole warps; nothing below waits for another warp
    const bool in = (uint32_t)c * 8 < p.d;
    const uint32_t half = p.rot.rot / 2;

    // the token's rows: q's heads, k's, v's; this warp's share of them, a batch's loads ahead of the one that is worked on
    const uint32_t nqk = p.q.heads + p.k.heads, rows = nqk + p.v.heads, step = p.parts * RPW;
    auto fetch = [&](uint32_t r0, Raw<DT> &w) {
        const uint32_t r = r0 + sub;
        if (r < rows && in) {
            const HeadsParams &h = r < p.q.heads ? p.q : (r < nqk ? p.k : p.v);
            const uint32_t hd = r < p.q.heads ? r : (r < nqk ? r - p.q.heads : r - nqk);
            load8<DT>(h.src + token * h.s_t + hd * h.s_h + (uint64_t)c * 8 * dtype_size(DT), vec, w);
        } else {
#pragma unroll
            for (int i = 0; i < Raw<DT>::N; ++i) w.w[i] = 0u;
        }
    };
    Raw<DT> next[PR_BATCH];
#pragma unroll
    for (int j = 0; j < PR_BATCH; ++j) fetch(part * RPW + j * step, next[j]);

    float co[8], si[8];
    int partner = lane;
    bool turned = false;
    if (TURN) {
        for (uint32_t f = lane; f < half; f += 32) {
            const uint32_t a = p.rot.axis ? min((uint32_t)p.rot.axis[f], p.rot.n_axes - 1) : 0u;
            // the angle in turns; its whole turns leave before it is rounded to f32
            const double t = (double)p.rot.pos[a * p.rot.pos_stride + token] * (double)p.rot.freq[f] * 0.15915494309189533577;
            float s, k;
            sincospif((float)(2.0 * (t - rint(t))), &s, &k);
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
                for (int i = 0; i < 8; ++i) {
                    const float2 cs = s_cs[warp][f0 + i];
                    co[i] = cs.x;
                    si[i] = second ? cs.y : -cs.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 cs = s_cs[warp][c * 4 + i];
                    co[2 * i] = co[2 * i + 1] = cs.x;
                    si[2 * i] = -cs.y, si[2 * i + 1] = cs.y;
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

#pragma unroll 1
    for (uint32_t base = part * RPW; base < rows; base += step * PR_BATCH) {
        Raw<DT> raw[PR_BATCH];
#pragma unroll
        for (int j = 0; j < PR_BATCH; ++j) raw[j] = next[j];
#pragma unroll
        for (int j = 0; j < PR_BATCH; ++j) fetch(base + (PR_BATCH + j) * step, next[j]);
#pragma unroll
        for (int j = 0; j < PR_BATCH; ++j) {
            const uint32_t r0 = base + j * step, r = r0 + sub;
            if (r0 >= rows) break;  // the whole warp
            const bool is_v = r >= nqk;
            float x[8];
            values8(raw[j], x);
            if (TURN && r0 < nqk) {
                float y[8];
                if (TURN == 1) {
                    Raw<DT> other;
#pragma unroll
                    for (int i = 0; i < Raw<DT>::N; ++i) other.w[i] = __shfl_sync(0xffffffffu, raw[j].w[i], partner);
                    values8(other, y);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
                }
                if (turned && !is_v) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], co[i], y[i] * si[i]);
                }
            }
            if (r < p.q.heads || (POOL == 0 && r < rows)) {
                const HeadsParams &h = r < p.q.heads ? p.q : p.k;
                const uint32_t hd = r < p.q.heads ? r : r - p.q.heads;
                if (in) store8<DT>(h.dst + token * h.d_t + hd * h.d_h + (uint64_t)c * 8 * dtype_size(DT), vec, x);
            }
            if (POOL && r0 + RPW > p.q.heads) {
                const bool mine = r >= p.q.heads && r < rows && kept && in;
                const uint32_t hd = is_v ? r - nqk : r - p.q.heads;
                const PoolParams &pl = p.pool;
                char *dst = is_v ? pl.v + blk * pl.v_sb + row * pl.v_sr + hd * pl.v_sh : pl.k + blk * pl.k_sb + row * pl.k_sr + hd * pl.k_sh;
                if (POOL == 1) {
                    if (mine) *reinterpret_cast<uint4 *>(dst + c * 16) = pack8<PDT>(x);
                } else {
                    uint32_t scale;
                    const uint2 w = mx8(x, scale);
                    if (mine) {
                        *reinterpret_cast<uint2 *>(dst + c * 8) = w;
                        if ((c & 3) == 0) (is_v ? pl.vs : pl.ks)[(((uint64_t)blk * pl.hkv + hd) * pl.block_rows + row) * (pl.d / 32) + c / 4] = (uint8_t)scale;
                    }
                }
            }
        }
    }
}

template <int DT, int TURN, int POOL, int PDT>
static int rows_launch(const RowsParams &p, bool vec, cudaStream_t stream, const char *what) {
    const uint32_t chunks = p.d / 8, lpr = chunks <= 8 ? 8 : (chunks <= 16 ? 16 : 32), rows = p.q.heads + p.k.heads + p.v.heads;
    RowsParams r = p;
    // a warp goes over a whole token where tokens fill the device; fewer tokens are shared among warps, down to one load a lane
    const uint32_t most = std::max(1u, (rows * lpr + 31) / 32);
    r.parts = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(1, 148ull * 32 / std::max(p.tokens, 1u)));
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

template <int DT, int POOL, int PDT, int LPR>
__global__ void __launch_bounds__(PR_WARPS * 32) paged_unpack_kernel(const UnpackParams p) {
    constexpr int RPW = 32 / LPR, PR_BATCH = 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane % LPR, sub = lane / LPR;
    const uint64_t unit = (uint64_t)blockIdx.x * PR_WARPS + warp, t = unit / p.parts;
    const uint32_t part = (uint32_t)(unit % p.parts);
    const PoolParams &pl = p.pool;
    if (t >= p.total || t >= p.cu[p.b]) return;
    const uint32_t seq = pool_seq(p.cu, p.b, t, lane), j = (uint32_t)(t - p.cu[seq]);
    const uint32_t page = pool_div(j, pl.div_mul, pl.div_shr), row = j - page * pl.block_rows;
    const int id = page < p.table_cols ? p.table[seq * p.table_stride + page] : -1;
    const bool there = id >= 0 && (uint32_t)id < pl.n_blocks, in = (uint32_t)c * 8 < pl.d;
    if (!there && p.status && lane == 0 && part == 0) atomicExch(p.status, 3);
    const uint64_t blk = there ? (uint64_t)id : 0;
    const uint32_t rows = pl.hkv * (p.v ? 2u : 1u);
    for (uint32_t base = part * RPW; base < rows; base += p.parts * RPW * PR_BATCH) {
        uint4 w[PR_BATCH];
        uint32_t e[PR_BATCH];
#pragma unroll
        for (int i = 0; i < PR_BATCH; ++i) {
            const uint32_t r = base + i * p.parts * RPW + sub;
            const bool is_v = r >= pl.hkv;
            const uint32_t hd = is_v ? r - pl.hkv : r;
            w[i] = make_uint4(0u, 0u, 0u, 0u);
            e[i] = 0;
            if (r < rows && in && there) {
                const char *src = is_v ? pl.v + blk * pl.v_sb + row * pl.v_sr + hd * pl.v_sh : pl.k + blk * pl.k_sb + row * pl.k_sr + hd * pl.k_sh;
                if (POOL == 1) {
                    w[i] = *reinterpret_cast<const uint4 *>(src + c * 16);
                } else {
                    const uint2 a = *reinterpret_cast<const uint2 *>(src + c * 8);
                    w[i].x = a.x, w[i].y = a.y;
                    e[i] = (is_v ? pl.vs : pl.ks)[((blk * pl.hkv + hd) * pl.block_rows + row) * (pl.d / 32) + c / 4];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < PR_BATCH; ++i) {
            const uint32_t r = base + i * p.parts * RPW + sub;
            if (r >= rows || !in) continue;
            const bool is_v = r >= pl.hkv;
            const uint32_t hd = is_v ? r - pl.hkv : r;
            char *dst = (is_v ? p.v : p.k) + ((t * pl.hkv + hd) * pl.d + c * 8) * dtype_size(DT);
            if (POOL == 1 && DT == PDT) {
                *reinterpret_cast<uint4 *>(dst) = w[i];
                continue;
            }
            float x[8];
            if (POOL == 1) {
                const uint32_t a[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[2 * k] = PDT == B200_BF16 ? bf16_bits_to_f((uint16_t)a[k]) : f16_bits_to_f((uint16_t)a[k]);
                    x[2 * k + 1] = PDT == B200_BF16 ? bf16_bits_to_f((uint16_t)(a[k] >> 16)) : f16_bits_to_f((uint16_t)(a[k] >> 16));
                }
            } else {
                const float s = e8m0_to_f(e[i]);
                const uint32_t a[2] = {w[i].x, w[i].y};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t lo = cvt_e4m3x2_f16x2(a[k]), hi = cvt_e4m3x2_hi_f16x2(a[k]);  // exact
                    x[4 * k] = f16_bits_to_f((uint16_t)lo) * s;
                    x[4 * k + 1] = f16_bits_to_f((uint16_t)(lo >> 16)) * s;
                    x[4 * k + 2] = f16_bits_to_f((uint16_t)hi) * s;
                    x[4 * k + 3] = f16_bits_to_f((uint16_t)(hi >> 16)) * s;
                }
            }
            store8<DT>(dst, true, x);
        }
    }
}

template <int DT, int POOL, int PDT>
static int unpack_launch(const UnpackParams &p, cudaStream_t stream) {
    const uint32_t chunks = p.pool.d / 8, lpr = chunks <= 8 ? 8 : (chunks <= 16 ? 16 : 32), rows = p.pool.hkv * (p.v ? 2u : 1u);
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
