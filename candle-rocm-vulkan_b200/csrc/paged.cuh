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
// E4M3 codes as pairs of values, exact, NaNs among them. pool_codes4: the bytes of two words, pair by pair; pool_pair: bytes 2 I and 2 I + 1 of one.
// To bf16 by way of f16 and f32, whose instructions are spread over the pipes (the code's bits moved to a bf16's places, with a look for NaNs: 638 for 740
// TFLOP/s of fa_paged_tma_kernel).
template <bool BF16>
__device__ __forceinline__ uint32_t pool_f16_as(uint32_t h) {
    if (!BF16) return h;
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(f16_bits_to_f((uint16_t)(h >> 16))), "f"(f16_bits_to_f((uint16_t)h)));
    return d;
}
template <bool BF16>
__device__ __forceinline__ void pool_codes4(uint32_t lo, uint32_t hi, uint32_t (&x)[4]) {
    const uint32_t a = __byte_perm(lo, hi, 0x5140), b = __byte_perm(lo, hi, 0x7362);
    x[0] = pool_f16_as<BF16>(cvt_e4m3x2_f16x2(a)), x[1] = pool_f16_as<BF16>(cvt_e4m3x2_hi_f16x2(a));
    x[2] = pool_f16_as<BF16>(cvt_e4m3x2_f16x2(b)), x[3] = pool_f16_as<BF16>(cvt_e4m3x2_hi_f16x2(b));
}
template <bool BF16, int I>
__device__ __forceinline__ uint32_t pool_pair(uint32_t w) {
    return pool_f16_as<BF16>(I ? cvt_e4m3x2_hi_f16x2(w) : cvt_e4m3x2_f16x2(w));
}
// The multiplier 2^(e - 127) of such a pair, for the scales e0 and e1. bf16 has all of them; f16's outside 103 .. 142 go in two steps, `rest` first: a small
// one is exact there (or the value less than half of f16's smallest number in any case), so that the second step rounds once, as a conversion would. A large
// one ends at 2^15, which with the second's 2^15 takes the smallest code, 2^-9, past f16's largest number; neither is infinite, so a code of zero stays zero.
template <bool BF16>
__device__ __forceinline__ uint32_t pool_scale2(uint32_t e0, uint32_t e1, uint32_t &rest) {
    if (BF16) {
        rest = 0x3f803f80u;
        return (e0 ? e0 << 7 : 0x40u) | (e1 ? e1 << 7 : 0x40u) << 16;
    }
    const uint32_t m0 = min(max(e0, 103u), 142u), m1 = min(max(e1, 103u), 142u);
    rest = pack_f16x2(e8m0_to_f(min(e0 + 127u - m0, 142u)), e8m0_to_f(min(e1 + 127u - m1, 142u)));
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
