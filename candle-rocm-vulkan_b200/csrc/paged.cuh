// What the kernels over a pool of cache pages share (paged_rows.cu: rows in and out, rotary positions; paged_attn.cu and
// fa_prefill_sm100.cu: attention): the pool as kernels see it, and the checks of its description.
#pragma once
#include "common.cuh"

namespace b200 {

struct PoolParams {
    char *k, *v;
    uint8_t *ks, *vs;                                    // MXFP8: E8M0 bytes (block, head, row, d / 32); else null
    uint64_t k_sb, k_sr, k_sh, v_sb, v_sr, v_sh;         // bytes
    uint32_t n_blocks, block_rows, hkv, d;
    uint32_t div_mul, div_shr;                           // n / block_rows for n < 2^31
};

// n / d for n < 2^31: q = (mulhi(n, mul) + n) >> shr
inline void pool_div_init(uint32_t d, uint32_t *mul, uint32_t *shr) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    *mul = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    *shr = s;
}
__device__ __forceinline__ uint32_t pool_div(uint32_t n, uint32_t mul, uint32_t shr) { return (uint32_t)(((uint64_t)__umulhi(n, mul) + n) >> shr); }

template <bool BF16>
__device__ __forceinline__ uint32_t pool_mul2(uint32_t a, uint32_t b) {
    uint32_t d;
    if (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// E4M3 codes as pairs of values: f16, or bf16 times 2^-120 (a code's exponent and mantissa in the places of a bf16's, its subnormals
// among that type's). A NaN is the code 0x7f, which the move makes 480: pool_codes4 puts a NaN there, pool_pair leaves the codes' magnitudes in
// `mag` for a look at all of a row at once (pool_nan). pool_codes4: the bytes of two words, pair by pair; pool_pair: bytes 2 I and 2 I + 1 of one.
// whether the magnitudes (or their maximum, lane by lane) are a NaN's; the pair x with NaNs where they are
__device__ __forceinline__ bool pool_nan(uint32_t mag) { return ((mag + 0x00100010u) & 0x08000800u) != 0; }
__device__ __forceinline__ uint32_t pool_nans(uint32_t x, uint32_t mag) {
    const uint32_t nan = (mag + 0x00100010u) & 0x08000800u;
    return x | ((nan << 4) - (nan >> 4));
}
template <bool BF16>
__device__ __forceinline__ void pool_codes4(uint32_t lo, uint32_t hi, uint32_t (&x)[4]) {
    if (BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = __byte_perm(lo, hi, (4u + i) << 12 | i << 4);
            const uint32_t mag = (t >> 4) & 0x07f007f0u;
            x[i] = pool_nans((t & 0x80008000u) | mag, mag);
        }
    } else {
        const uint32_t a = __byte_perm(lo, hi, 0x5140), b = __byte_perm(lo, hi, 0x7362);
        x[0] = cvt_e4m3x2_f16x2(a), x[1] = cvt_e4m3x2_hi_f16x2(a);
        x[2] = cvt_e4m3x2_f16x2(b), x[3] = cvt_e4m3x2_hi_f16x2(b);
    }
}
template <bool BF16, int I>
__device__ __forceinline__ uint32_t pool_pair(uint32_t w, uint32_t &mag) {
    if (BF16) {
        const uint32_t t = __byte_perm(w, w, (2u * I + 1u) << 12 | (2u * I) << 4);
        mag = (t >> 4) & 0x07f007f0u;
        return (t & 0x80008000u) | mag;
    }
    return I ? cvt_e4m3x2_hi_f16x2(w) : cvt_e4m3x2_f16x2(w);
}
// The multiplier that takes such a pair to its values, for the scales e0 and e1: f16 2^(e - 127), bf16 2^(e - 127 + 120). Scales outside the
// type's range (f16 e < 103, bf16 e > 134) go in two steps: `rest` is the second.
template <bool BF16>
__device__ __forceinline__ uint32_t pool_scale2(uint32_t e0, uint32_t e1, uint32_t &rest) {
    if (BF16) {
        const uint32_t m0 = min(e0, 134u), m1 = min(e1, 134u);
        rest = (e0 == 255u ? 255u : e0 - m0 + 127u) << 7 | (e1 == 255u ? 255u : e1 - m1 + 127u) << 23;  // (255 is an infinity, as for e8m0_to_f)
        return (m0 + 120u) << 7 | (m1 + 120u) << 23;
    }
    const uint32_t m0 = max(e0, 103u), m1 = max(e1, 103u);
    rest = pack_f16x2(e8m0_to_f(e0 + 127u - m0), e8m0_to_f(e1 + 127u - m1));
    return pack_f16x2(e8m0_to_f(m0), e8m0_to_f(m1));
}

// the sequence of packed row t: the last i with cu[i] <= t among 0 .. b - 1 (a warp at once, 32 probes a step)
__device__ __forceinline__ uint32_t pool_seq(const uint32_t *cu, uint32_t b, uint64_t t, int lane) {
    uint32_t lo = 0, n = b;  // the answer is in [lo, lo + n)
    while (n > 1) {
        const uint32_t step = (n + 31) / 32, at = lo + lane * step;
        const uint32_t hit = __ballot_sync(0xffffffffu, (uint32_t)lane * step < n && cu[at] <= t);
        const uint32_t last = hit ? 31 - __clz(hit) : 0;  // (cu ascends)
        lo += last * step;
        n = min(step, n - last * step);
    }
    return lo;
}

// checks the description and fills the kernels' view of it
int pool_params(const B200PagedPool &pool, const char *what, PoolParams *p);

}  // namespace b200
