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

// checks the description and fills the kernels' view of it
int pool_params(const B200PagedPool &pool, const char *what, PoolParams *p);

}  // namespace b200
