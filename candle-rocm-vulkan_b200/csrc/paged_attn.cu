// Attention of a ragged batch's new tokens over a pool of cache pages: b200_paged_attention, and its kernel for sequences with few
// new tokens. Per query head, o_t = sum_j w_tj v_j / sum_j w_tj with w_tj = exp(scale q_t . k_j (soft cap, ALiBi)) over the keys j that
// token t sees, in one pass with a running maximum and sum.
//
// Sequences with few packed query rows (token x head of the group) are bound by memory: every key and value is read once for at
// most 16 rows. The batch is ragged and only the device knows its lengths, so the work is divided there: a column is 16 rows of a
// sequence, a unit is what a block's four warps score at a time (64 or 128 keys), and the units of all columns, one behind the
// other, are cut into equal shares. Every kv head has the same shares, and blocks of neighbouring heads run side by side (two
// blocks per SM): in a page the heads' rows of a key lie next to one another, so they are read at about the same time. A block that holds all of
// a column writes its rows; parts of columns go to the workspace, two at most per block (where its share begins and
// where it ends), and a second grid joins them, its blocks told by the first's in which share a column begins that goes on behind it.
// In a block each warp has keys of its own, K and V in a ring of stages that it fills ahead of the column it is working on,
// across columns too; scores and sums run on mma.sync m16n8k16, and the warps' partial results meet in shared memory at a
// column's end.
//
// Measured (32 / 8 heads of 128; copy bandwidth 6 470 GB/s), L2 flushed: 64 sequences of 500 to 8192 keys, bf16, 195 us, 0.90 of the copy (179 to 192 back to
// back); 48 x 4 tokens over 4000 to 30000 keys, MXFP8, 419 us, 0.64 (384 to 407). There, at 387, the loads alone took 281 and the instructions alone 278, on two
// blocks of four warps per SM: what 251 registers leave, which 16 rows of accumulators need whatever the column has. A fifth warp per block for the copies (463: its registers come from the others), E4M3 operands for the scores with q in two parts
// (477) and the code without its rare forms (380) were tried.
//
// MXFP8 keys and values stay codes up to the registers. Scores: the codes are exact in f16; q is taken to f16 behind a power of
// two per row (a bf16 element keeps its eight bits unless it is 2^28 below the row's largest), and a block of 32 elements adds its
// sum times its scale in f32. Values and weights: see the products. Weights are rounded to 16 bits (f16 2^-11, bf16 2^-8 at most each, and these
// average out), as for 16-bit pools.
#include <algorithm>
#include <cuda.h>
#include <type_traits>

#include "fa_params.cuh"

namespace b200 {

constexpr int PA_WARPS = 4, PA_THREADS = PA_WARPS * 32, PA_ROWS = 16;
constexpr float PA_LOG2E = 1.4426950408889634f;

struct PaParams {
    const char *q;
    char *out;
    uint64_t q_st, q_sh, o_st, o_sh;  // bytes
    const uint32_t *cu_q;
    const int32_t *kv_len, *table;
    uint64_t table_stride;
    PoolParams pool;
    const float *alibi;
    int32_t *status;
    float *part_o;    // [blocks][2][16][d]
    float2 *part_ml;  // [blocks][2][16]: maximum (log 2), sum
    int4 *part_col;   // [blocks]: a column that begins in this share and goes on behind it (sequence, pack, parts, slot of the first); parts 0: none
    uint32_t b, hq, hkv, group, d, total_q, max_q, max_k, table_cols, alibi_bs;
    float scale, softcap;
    int32_t wl, wr;
    uint32_t shares;  // per kv head; blocks = shares x hkv
    uint32_t row_cap;  // sequences of more packed rows are on the tcgen05 tiles; 0: all are here
    uint32_t packs;    // the most groups of 16 rows that a sequence has here
};

// KIND: 0 f16, 1 bf16, 2 MXFP8 under f16 queries, 3 MXFP8 under bf16 queries
template <int HD, int KIND>
struct PA {
    static constexpr bool MX = KIND >= 2, BF16 = KIND & 1;
    static constexpr int ES = MX ? 1 : 2, RB = HD * ES;                   // bytes of a row
    static constexpr int KEYS = HD == 64 || (HD == 128 && MX) ? 32 : 16;  // of a warp's tile
    static constexpr int UNIT = KEYS * PA_WARPS, CPR = RB / 16, NB = HD / 32;
    static constexpr uint32_t TILE = KEYS * RB, STAGE = 2 * TILE;        // K, V
    static constexpr uint32_t SC = MX ? 2 * KEYS * NB : 0;               // scales of a stage
    static constexpr int NS = HD == 256 && !MX ? 2 : 3;
    static constexpr int COLS = RB < 128 ? 1 : RB / 128, COL_B = RB < 128 ? 64 : 128;  // columns of a tile and their bytes per row
    static constexpr int PARTS = HD == 128 && MX ? 4 : 2;                // pieces of a row that the warps' merge takes in turn (two blocks fit an SM)
    static constexpr int PIECE = HD / PARTS, MROW = PIECE + 2;           // floats per row: a piece, maximum, sum
    static constexpr uint32_t SM_SC = PA_WARPS * NS * STAGE, SM_MERGE = SM_SC + PA_WARPS * NS * SC, SM_BAR = SM_MERGE + PA_WARPS * PA_ROWS * MROW * 4, SMEM = SM_BAR + PA_WARPS * NS * 8;
    static constexpr uint32_t CL_ML = PA_ROWS * HD * 4;  // a cluster's partial rows lie at 0, their maxima and sums here
    static_assert(CL_ML + PA_ROWS * 8 <= SM_SC, "over the rings");
    // 16-byte chunk ch of row r of a tile, in 128-byte columns (64 where a row is no longer), swizzled
    __device__ static __forceinline__ uint32_t at(int r, int ch) {
        if (RB == 64) return r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
        return (ch >> 3) * (KEYS * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
    }
};

struct PaSeq {
    uint32_t q0, rows, packs;  // first token; packed rows; groups of 16 of them
    int lq, lk, ulo, uhi;      // units that some row sees
};
// keys [lo, hi) that packed row r sees
__device__ __forceinline__ void pa_range(const PaParams &p, const PaSeq &s, uint32_t r, int &lo, int &hi) {
    const int pos = (int)(r / p.group) + s.lk - s.lq;
    lo = p.wl >= 0 && pos > p.wl ? min(pos - p.wl, s.lk) : 0;
    hi = p.wr >= 0 && pos < s.lk - p.wr - 1 ? pos + p.wr + 1 : s.lk;
    hi = max(hi, lo);
}
// the sequence's units (of one head)
__device__ __forceinline__ uint64_t pa_seq(const PaParams &p, uint32_t b, int unit, PaSeq &s) {
    s.q0 = min(p.cu_q[b], p.total_q);
    const uint32_t end = min(p.cu_q[b + 1], p.total_q);
    s.lq = end > s.q0 ? (int)min(end - s.q0, p.max_q) : 0;
    s.lk = max(0, min(p.kv_len[b], (int)p.max_k));
    s.rows = (uint32_t)s.lq * p.group;
    s.packs = (s.rows + PA_ROWS - 1) / PA_ROWS;
    s.ulo = s.uhi = 0;
    if (s.rows == 0 || (p.row_cap && s.rows > p.row_cap)) return 0;
    int lo, hi, x;
    pa_range(p, s, 0, lo, x);
    pa_range(p, s, s.rows - 1, x, hi);
    s.ulo = lo / unit;
    s.uhi = hi > lo ? (hi + unit - 1) / unit : s.ulo + 1;  // rows that see nothing still have zeros to write
    return (uint64_t)(uint32_t)(s.uhi - s.ulo) * s.packs;
}

// Where the block (all of its threads; a multiple of 32, 256 at most) finds unit `target(total)` of all: the sequence and the unit
// within it. Every thread sums a run of sequences. `scratch`: ten words of shared memory.
struct PaPlace {
    uint64_t total, per, off;
    uint32_t seq;
};
template <typename F>
__device__ __forceinline__ PaPlace pa_place(const PaParams &p, int unit, uint64_t *scratch, F target) {
    uint64_t *const s_sum = scratch, *const s_at = scratch + 8;
    const uint32_t n = (p.b + blockDim.x - 1) / blockDim.x, first = min(threadIdx.x * n, p.b), last = min(first + n, p.b);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    uint64_t sum = 0;
    PaSeq s;
    for (uint32_t i = first; i < last; ++i) sum += pa_seq(p, i, unit, s);
    uint64_t upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    PaPlace at;
    at.total = 0;
    uint64_t before = upto - sum;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) before += s_sum[w];
        at.total += s_sum[w];
    }
    at.per = (at.total + p.shares - 1) / p.shares;
    const uint64_t want = target(at.per);
    if (want >= before && want < before + sum) {
        uint64_t rest = want - before;
        for (uint32_t i = first; i < last; ++i) {
            const uint64_t u = pa_seq(p, i, unit, s);
            if (rest < u) {
                s_at[0] = i;
                s_at[1] = rest;
                break;
            }
            rest -= u;
        }
    }
    __syncthreads();
    at.seq = (uint32_t)s_at[0];
    at.off = s_at[1];
    return at;
}

// a unit of a column of a sequence, and the way to the next one
struct PaCursor {
    PaSeq s;
    uint32_t seq, pack;
    int u, lo, hi;  // the unit; the keys that some row of the column sees
    __device__ __forceinline__ void enter(const PaParams &p) {
        int x;
        pa_range(p, s, pack * PA_ROWS, lo, x);
        pa_range(p, s, min(pack * PA_ROWS + PA_ROWS, s.rows) - 1, x, hi);
    }
    __device__ __forceinline__ void start(const PaParams &p, int unit, uint32_t seq_, uint64_t off) {
        seq = seq_;
        pa_seq(p, seq, unit, s);
        const uint32_t n = (uint32_t)(s.uhi - s.ulo);
        pack = (uint32_t)(off / n);
        u = s.ulo + (int)(off - (uint64_t)pack * n);
        enter(p);
    }
    __device__ __forceinline__ bool next(const PaParams &p, int unit) {  // true: another column
        if (++u < s.uhi) return false;
        if (++pack == s.packs) {
            pack = 0;
            while (++seq < p.b && pa_seq(p, seq, unit, s) == 0) {}
        }
        u = s.ulo;
        if (seq < p.b) enter(p);
        return true;
    }
};

__device__ __forceinline__ void pa_ldsm(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void pa_ldsm_trans(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ uint2 pa_lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t pa_lds8(uint32_t addr) {
    uint32_t v;
    asm volatile("{\n .reg .u16 t;\n ld.shared.u8 t, [%1];\n cvt.u32.u16 %0, t;\n}" : "=r"(v) : "r"(addr));
    return v;
}
template <bool BF16>
__device__ __forceinline__ void pa_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        mma_f16_16816(c, a[0], a[1], a[2], a[3], b0, b1);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pa_pack2(float lo, float hi) {
    uint32_t d;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ int g_paged_wait_failed = 0;  // a bounded wait for copies ran out

// MODE, how a block gets its units and keys:
//   PA_CHUNKS  a share; 16-byte chunks, each lane for itself (pages of odd sizes)
//   PA_COPIES  a share; tensor copies of `box` rows
//   PA_CLUSTER a column per cluster of blocks, each with every n-th unit, joined through distributed shared memory: no division of work to find out, no
//              second grid. Tensor copies.
enum { PA_CHUNKS = 0, PA_COPIES, PA_CLUSTER };
__device__ __forceinline__ uint32_t pa_cluster_size() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ uint32_t pa_cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void pa_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the pair of floats at shared address `addr` of the cluster's block `rank`
__device__ __forceinline__ float2 pa_peer(uint32_t addr, uint32_t rank) {
    float2 v;
    asm volatile("{\n .reg .u32 a;\n mapa.shared::cluster.u32 a, %2, %3;\n ld.shared::cluster.v2.f32 {%0, %1}, [a];\n}" : "=f"(v.x), "=f"(v.y) : "r"(addr), "r"(rank) : "memory");
    return v;
}
template <int HD, int KIND, int MODE>
__global__ void __launch_bounds__(PA_THREADS, HD == 256 ? 1 : 2) paged_decode_kernel(const PaParams p, const __grid_constant__ CUtensorMap tm_k,
                                                                                     const __grid_constant__ CUtensorMap tm_v, const uint32_t tm_order, const uint32_t box) {
    using C = PA<HD, KIND>;
    constexpr bool MX = C::MX, BF16 = C::BF16, TMA = MODE != PA_CHUNKS, CLUSTER = MODE == PA_CLUSTER;
    constexpr int KSTEPS = HD / 16, NT = HD / 8, KEYS = C::KEYS, KG = KEYS / 16, UNIT = C::UNIT;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * C::NS * C::STAGE, scales = smem_u32(smem) + C::SM_SC + warp * C::NS * C::SC;
    float *const mg = reinterpret_cast<float *>(smem + C::SM_MERGE);
    uint64_t *const bars = reinterpret_cast<uint64_t *>(smem + C::SM_BAR) + warp * C::NS;
    if (TMA && lane == 0) {
        for (int i = 0; i < C::NS; ++i) mbar_init(&bars[i], 1);
        mbar_fence_init();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (!CLUSTER && p.shares > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining grid may get ready
    const PoolParams &pl = p.pool;
    // Behind the tiles' kernel this grid may start before that one has ended (it needs nothing of it): the first block sees that it does not end before.
    auto in_order = [&]() { if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory"); };
    // which head, and which units: nu of them, every stride-th
    const uint32_t ranks = CLUSTER ? pa_cluster_size() : 1, rank = CLUSTER ? pa_cluster_rank() : 0, column = blockIdx.x / ranks;
    const uint32_t share = column / p.hkv, hk = column - share * p.hkv;
    PaCursor cur, lead;  // the unit being worked on, and the one to be asked for next
    int nu;
    uint32_t share_units = 0;
    if (CLUSTER) {
        cur.seq = share / p.packs;
        cur.pack = share - cur.seq * p.packs;
        const int n = pa_seq(p, cur.seq, UNIT, cur.s) ? cur.s.uhi - cur.s.ulo : 0;
        if (n == 0 || cur.pack >= cur.s.packs) return in_order();  // the whole cluster
        cur.u = cur.s.ulo + (int)rank;
        cur.enter(p);
        nu = (int)rank < n ? (n - (int)rank - 1) / (int)ranks + 1 : 0;
    } else {
        const PaPlace place = pa_place(p, UNIT, reinterpret_cast<uint64_t *>(mg), [&](uint64_t per) { return share * per; });
        const uint64_t u0 = share * place.per;
        if (tid == 0 && p.shares > 1) p.part_col[blockIdx.x] = make_int4(0, 0, 0, 0);
        if (u0 >= place.total) return in_order();
        nu = (int)min(place.per, place.total - u0);
        share_units = (uint32_t)place.per;
        cur.start(p, UNIT, place.seq, place.off);
    }
    lead = cur;
    auto advance = [&](PaCursor &at) {  // true: to another column
        if (!CLUSTER) return at.next(p, UNIT);
        at.u += (int)ranks;
        return false;
    };

    // A warp's keys of the lead's unit into stage st: lane i finds key i's row, then C::CPR lanes copy a row. What no row of the column
    // sees, and what a page outside the pool would hold, is zeros.
    auto request = [&](int st) {
        const int lo = lead.lo, hi = lead.hi, j = lead.u * UNIT + warp * KEYS + lane;
        const char *kr = nullptr, *vr = nullptr;
        uint64_t srow = 0;
        if (lane < KEYS && j >= lo && j < hi) {
            const uint32_t page = pool_div((uint32_t)j, pl.div_mul, pl.div_shr), row = (uint32_t)j - page * pl.block_rows;
            const int id = page < p.table_cols ? p.table[lead.seq * p.table_stride + page] : -1;
            if (id >= 0 && (uint32_t)id < pl.n_blocks) {
                kr = pl.k + (uint64_t)id * pl.k_sb + row * pl.k_sr + hk * pl.k_sh;
                vr = pl.v + (uint64_t)id * pl.v_sb + row * pl.v_sr + hk * pl.v_sh;
                srow = (((uint64_t)id * pl.hkv + hk) * pl.block_rows + row) * (p.d / 32);
            } else if (p.status) {
                atomicExch(p.status, 3);
            }
        }
        const uint32_t dst = ring + st * C::STAGE, ch = lane % C::CPR;
#pragma unroll
        for (int i = 0; i < KEYS * C::CPR / 32; ++i) {
            const int row = i * (32 / C::CPR) + lane / C::CPR;
            const char *ks = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(kr), row));
            const char *vs = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vr), row));
            const bool in = ks != nullptr && ch * 16 < p.d * C::ES;
            const uint32_t at = dst + C::at(row, ch);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(in ? ks + ch * 16 : pl.k), "r"(in ? 16 : 0) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + C::TILE), "l"(in ? vs + ch * 16 : pl.v), "r"(in ? 16 : 0) : "memory");
        }
        if (MX && lane < KEYS) {
            const uint32_t nb = p.d / 32, at = scales + st * C::SC + lane * C::NB;
#pragma unroll
            for (int i = 0; i < C::NB; ++i) {
                const bool in = kr != nullptr && (uint32_t)i < nb;
                const uint32_t ke = in ? pl.ks[srow + i] : 127u, ve = in ? pl.vs[srow + i] : 127u;
                asm volatile("st.shared.u8 [%0], %1;" ::"r"(at + i), "r"(ke) : "memory");
                asm volatile("st.shared.u8 [%0], %1;" ::"r"(at + KEYS * C::NB + i), "r"(ve) : "memory");
            }
        }
    };
    // TMA. The page of rows i x box .. of the warp's keys in the lead's unit, in lane i (-1: no row of the column sees any of them; -2: no page of
    // the pool, whose copy brings zeros); asked for one unit ahead, since the copies cannot leave without it.
    int ahead_row = 0;
    auto page_of = [&]() {
        const int j = lead.u * UNIT + warp * KEYS + lane * (int)box;
        ahead_row = 0;
        if (lane * (int)box >= KEYS || j >= lead.hi || j + (int)box <= lead.lo) return -1;
        const uint32_t page = pool_div((uint32_t)j, pl.div_mul, pl.div_shr);
        ahead_row = j - (int)(page * pl.block_rows);
        const int id = page < p.table_cols ? p.table[lead.seq * p.table_stride + page] : -1;
        return id >= 0 && (uint32_t)id < pl.n_blocks ? id : -2;
    };
    // copies of the lead's unit into stage st; false: nobody sees any of the warp's keys, nothing comes
    auto copy = [&](int st, int id, int row) {
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, id != -1));
        if (n == 0) return false;
        const uint32_t bar = smem_u32(&bars[st]), good = MX ? __popc(__ballot_sync(0xffffffffu, id >= 0)) : 0u;
        if (lane == 0) mbar_expect_tx(&bars[st], n * box * 2 * C::RB + good * box * 2 * C::NB);
        __syncwarp();
        if (id != -1) {
            const uint32_t dst = ring + st * C::STAGE + lane * box * C::COL_B;
            const int blk = id < 0 ? (int)pl.n_blocks : id;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const uint32_t ord = kv ? tm_order >> 8 : tm_order, ph = ord & 3u, pk = (ord >> 2) & 3u;
                const int c1 = ph == 0 ? (int)hk : (pk == 0 ? row : blk), c2 = ph == 1 ? (int)hk : (pk == 1 ? row : blk), c3 = ph == 2 ? (int)hk : (pk == 2 ? row : blk);
#pragma unroll
                for (int i = 0; i < C::COLS; ++i)
                    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                                     dst + kv * C::TILE + i * (KEYS * 128)),
                                 "l"(reinterpret_cast<uint64_t>(kv ? &tm_v : &tm_k)), "r"((MX ? 128 : 64) * i), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
                                 : "memory");
            }
            if (MX) {
                uint8_t *const at = smem + C::SM_SC + (warp * C::NS + st) * C::SC + lane * box * C::NB;
                if (id >= 0) {
                    const uint64_t from = (((uint64_t)id * pl.hkv + hk) * pl.block_rows + row) * C::NB;
                    bulk_g2s(at, pl.ks + from, box * C::NB, &bars[st]);
                    bulk_g2s(at + KEYS * C::NB, pl.vs + from, box * C::NB, &bars[st]);
                } else {
                    if (p.status) atomicExch(p.status, 3);
                    for (uint32_t i = 0; i < box * C::NB; ++i) at[i] = at[KEYS * C::NB + i] = 127;  // zeros times one
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // a later copy goes over them
                }
            } else if (id < 0 && p.status) {
                atomicExch(p.status, 3);
            }
        }
        return true;
    };
    uint32_t sent = 0, phase = 0;  // a bit per stage: copies are on their way; the parity that its barrier shows when they have landed
    int ahead = -1;
    if (TMA) {
        int ids[C::NS + 1], rows[C::NS + 1];  // all lookups before the first copy
#pragma unroll
        for (int t = 0; t <= C::NS; ++t) {
            ids[t] = t < nu ? page_of() : -1;
            rows[t] = ahead_row;
            if (t < nu - 1) advance(lead);
        }
        ahead = ids[C::NS];
        lead = cur;
#pragma unroll
        for (int t = 0; t < C::NS; ++t)
            if (t < nu) {
                if (copy(t, ids[t], rows[t])) sent |= 1u << t;
                advance(lead);
            }
    } else {
        for (int t = 0; t < C::NS; ++t) {
            if (t < nu) {
                request(t);
                advance(lead);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }
    bool ok = true;

    uint32_t qa[KSTEPS][4];
    float m[2], l[2], oacc[NT][4], sc[2], slope[2];
    int r_lo[2], r_hi[2], r_pos[2], lomax = 0, himin = 0;
    const bool special = p.softcap > 0.0f || p.alibi != nullptr, plain = !special && p.scale > 0.0f;
    if (CLUSTER) {  // a block may be without units
        m[0] = m[1] = -INFINITY, l[0] = l[1] = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) oacc[n][0] = oacc[n][1] = oacc[n][2] = oacc[n][3] = 0.0f;
    }
    // A column's end in this block: the four warps' partial results meet in shared memory, and go out as rows (whole), as a part to the workspace, or to
    // the block's shared memory for its cluster.
    auto finish = [&](const PaCursor &done, bool whole, uint64_t slot) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        }
        const int row = tid >> 3, ch = tid & 7;
        const uint32_t r = done.pack * PA_ROWS + row, tok = r / p.group;
        const bool there = r < done.s.rows;
        char *const orow = p.out + (done.s.q0 + tok) * p.o_st + (hk * p.group + r - tok * p.group) * p.o_sh;
        // a piece of the elements at a time: the warps' sums (and their maxima and weights), then eight threads per row
#pragma unroll
        for (int piece = 0; piece < C::PARTS; ++piece) {
            constexpr int NP = NT / C::PARTS;  // products' tiles of a piece
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float *dst = mg + (warp * PA_ROWS + g + 8 * e) * C::MROW;
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    const float x0 = oacc[piece * NP + n][2 * e], x1 = oacc[piece * NP + n][2 * e + 1];
                    if (MX) dst[2 * c * NP + n] = x0, dst[(2 * c + 1) * NP + n] = x1;
                    else *reinterpret_cast<float2 *>(dst + 8 * n + 2 * c) = make_float2(x0, x1);
                }
                if (c == 0) dst[C::PIECE] = m[e], dst[C::PIECE + 1] = l[e];
            }
            __syncthreads();
            if (!there) continue;
            float f[PA_WARPS], M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < PA_WARPS; ++w) M = fmaxf(M, mg[(w * PA_ROWS + row) * C::MROW + C::PIECE]);
            const float ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < PA_WARPS; ++w) {
                f[w] = fast_exp2(mg[(w * PA_ROWS + row) * C::MROW + C::PIECE] - ms);
                L += f[w] * mg[(w * PA_ROWS + row) * C::MROW + C::PIECE + 1];
            }
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
#pragma unroll 4
            for (int x = 2 * ch; x < C::PIECE; x += 16) {
                // the element that stands at x: MX has NP neighbours of every group of NT
                const uint32_t dd = MX ? x / NP * NT + piece * NP + x % NP : piece * C::PIECE + x;
                if (dd >= p.d) continue;
                float o0 = 0.0f, o1 = 0.0f;
#pragma unroll
                for (int w = 0; w < PA_WARPS; ++w) {
                    const float2 v = *reinterpret_cast<const float2 *>(mg + (w * PA_ROWS + row) * C::MROW + x);
                    o0 = fmaf(f[w], v.x, o0);
                    o1 = fmaf(f[w], v.y, o1);
                }
                if (CLUSTER) *reinterpret_cast<float2 *>(smem + (row * HD + dd) * 4) = make_float2(o0, o1);
                else if (whole) *reinterpret_cast<uint32_t *>(orow + dd * 2) = pa_pack2<BF16>(o0 * inv, o1 * inv);
                else *reinterpret_cast<float2 *>(p.part_o + (slot * PA_ROWS + row) * p.d + dd) = make_float2(o0, o1);
            }
            if (CLUSTER && piece == 0 && ch == 0) *reinterpret_cast<float2 *>(smem + C::CL_ML + row * 8) = make_float2(M, L);
            if (!CLUSTER && !whole && piece == 0 && ch == 0) p.part_ml[slot * PA_ROWS + row] = make_float2(M, L);
        }
    };
    bool begin = true;
    int seg_u = 0;
    uint32_t seg = 0;  // the block's segments so far
    for (int t = 0; t < nu; ++t) {
        if (begin) {
            // ---- a column: its rows of q as A fragments, their keys and scales
            begin = false;
            seg_u = cur.u;
#pragma unroll
            for (int n = 0; n < NT; ++n) oacc[n][0] = oacc[n][1] = oacc[n][2] = oacc[n][3] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t r = cur.pack * PA_ROWS + g + 8 * e;
                m[e] = -INFINITY, l[e] = 0.0f, slope[e] = 0.0f, sc[e] = p.scale;
                r_lo[e] = 0, r_hi[e] = cur.s.lk, r_pos[e] = 0;  // rows that do not exist see every key and are never stored
                const bool there = r < cur.s.rows;
                const uint32_t tok = there ? r / p.group : 0, h = hk * p.group + (there ? r - tok * p.group : 0);
                const char *src = p.q + (cur.s.q0 + tok) * p.q_st + h * p.q_sh;
                if (there) {
                    pa_range(p, cur.s, r, r_lo[e], r_hi[e]);
                    r_pos[e] = (int)tok + cur.s.lk - cur.s.lq;
                    if (p.alibi) slope[e] = p.alibi[(size_t)cur.seq * p.alibi_bs + h];
                }
                if (!MX) {
#pragma unroll
                    for (int ks = 0; ks < KSTEPS; ++ks) {
                        const uint32_t at = ks * 16 + 2 * c;
                        qa[ks][e] = there && at < p.d ? *reinterpret_cast<const uint32_t *>(src + at * 2) : 0u;
                        qa[ks][2 + e] = there && at + 8 < p.d ? *reinterpret_cast<const uint32_t *>(src + (at + 8) * 2) : 0u;
                    }
                } else {
                    // a block of 32 elements is two steps: lane c has its elements 8 c .. 8 c + 7, four a step
                    uint4 w[C::NB];
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < C::NB; ++i) {
                        const uint32_t at = i * 32 + 8 * c;
                        w[i] = there && at < p.d ? *reinterpret_cast<const uint4 *>(src + at * 2) : make_uint4(0u, 0u, 0u, 0u);
                        if (BF16) {
                            const uint32_t a[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(fabsf(u2f(a[k] << 16)), fabsf(u2f(a[k] & 0xffff0000u))));
                        }
                    }
                    float f = 1.0f;
                    if (BF16) {
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        const int ex = (int)((f2u(top) >> 23) & 0xffu);  // the row's largest lands in [2^14, 2^15)
                        const int fe = min(max(127 + 14 + 127 - ex, 27), 227);
                        f = u2f((uint32_t)fe << 23);
                        sc[e] = p.scale * u2f((uint32_t)(254 - fe) << 23);
                    }
#pragma unroll
                    for (int i = 0; i < C::NB; ++i) {
                        uint32_t a[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                        if (BF16)
#pragma unroll
                            for (int k = 0; k < 4; ++k) a[k] = pack_f16x2(u2f(a[k] << 16) * f, u2f(a[k] & 0xffff0000u) * f);
                        qa[2 * i][e] = a[0], qa[2 * i][2 + e] = a[1], qa[2 * i + 1][e] = a[2], qa[2 * i + 1][2 + e] = a[3];
                    }
                }
            }
            int x;
            pa_range(p, cur.s, min(cur.pack * PA_ROWS + PA_ROWS, cur.s.rows) - 1, lomax, x);
            pa_range(p, cur.s, cur.pack * PA_ROWS, x, himin);
        }
        const int j0 = cur.u * UNIT + warp * KEYS, st = t % C::NS;
        bool dirty = false;
        if (TMA) {
            if (sent >> st & 1u) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars[st], phase >> st & 1u));
                phase ^= 1u << st;
            }
            // values that no row of the column sees (rows of the page behind the last key, in front of a window; what was not copied)
            if (j0 < cur.lo || j0 + KEYS > cur.hi) {
                dirty = true;
                for (int i = lane; i < KEYS * C::CPR; i += 32) {
                    const int row = i / C::CPR;
                    if (j0 + row >= cur.lo && j0 + row < cur.hi) continue;
                    *reinterpret_cast<uint4 *>(smem + (warp * C::NS + st) * C::STAGE + C::TILE + C::at(row, i % C::CPR)) = make_uint4(0u, 0u, 0u, 0u);
                    if (MX && i % C::CPR == 0)
                        for (int k = 0; k < C::NB; ++k) smem[C::SM_SC + (warp * C::NS + st) * C::SC + (KEYS + row) * C::NB + k] = 127;
                }
            }
        } else {
            asm volatile("cp.async.wait_group %0;" ::"n"(C::NS - 1) : "memory");
        }
        __syncwarp();
        const uint32_t tk = ring + st * C::STAGE, tv = tk + C::TILE, tsc = scales + st * C::SC;

        // ---- scores
        float s[2 * KG][4];
#pragma unroll
        for (int n = 0; n < 2 * KG; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
        if (!MX) {
            const uint32_t kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
                for (int np = 0; np < KG; ++np) {
                    uint32_t b0, b1, b2, b3;
                    pa_ldsm(tk + C::at(np * 16 + kr, ks * 2 + kc), b0, b1, b2, b3);
                    pa_mma<BF16>(s[2 * np], qa[ks], b0, b1);
                    pa_mma<BF16>(s[2 * np + 1], qa[ks], b2, b3);
                }
        } else {
            const uint32_t nb = p.d / 32;
            uint2 sw[2 * KG];  // the scales of this lane's two keys of every eight
            if (C::NB == 4)
#pragma unroll
                for (int n = 0; n < 2 * KG; ++n) sw[n] = pa_lds64(tsc + (8 * n + 2 * c) * 4);
#pragma unroll
            for (int i = 0; i < C::NB; ++i) {
                if (!TMA && (uint32_t)i >= nb) break;
                const uint32_t(&q0)[4] = qa[2 * i], (&q1)[4] = qa[2 * i + 1];
#pragma unroll
                for (int n = 0; n < 2 * KG; ++n) {
                    const uint2 w = pa_lds64(tk + C::at(8 * n + g, 2 * i + (c >> 1)) + (c & 1) * 8);
                    float z[4];
                    mma_f16_16816_z(z, q0[0], q0[1], q0[2], q0[3], cvt_e4m3x2_f16x2(w.x), cvt_e4m3x2_hi_f16x2(w.x));
                    mma_f16_16816(z, q1[0], q1[1], q1[2], q1[3], cvt_e4m3x2_f16x2(w.y), cvt_e4m3x2_hi_f16x2(w.y));
                    // (the smallest scale, 2^-127, is half of the smallest normal number)
                    const float s0 = u2f(max(C::NB == 4 ? (i < 3 ? sw[n].x << (23 - 8 * (i & 3)) : sw[n].x >> 1) & 0x7f800000u : pa_lds8(tsc + (8 * n + 2 * c) * C::NB + i) << 23, 0x00400000u));
                    const float s1 = u2f(max(C::NB == 4 ? (i < 3 ? sw[n].y << (23 - 8 * (i & 3)) : sw[n].y >> 1) & 0x7f800000u : pa_lds8(tsc + (8 * n + 2 * c + 1) * C::NB + i) << 23, 0x00400000u));
                    s[n][0] = fmaf(z[0], s0, s[n][0]);
                    s[n][1] = fmaf(z[1], s1, s[n][1]);
                    s[n][2] = fmaf(z[2], s0, s[n][2]);
                    s[n][3] = fmaf(z[3], s1, s[n][3]);
                }
            }
        }
        // Tiles that every row sees as they are: the maximum of the sums, the scale in the exponent's multiply-add. The others (masks, soft cap, slopes,
        // a negative scale): scaled and masked one by one, apart from the first form's path.
        float mul[2] = {sc[0] * PA_LOG2E, sc[1] * PA_LOG2E}, mx[2];
        if (plain && j0 >= lomax && j0 + KEYS <= himin) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[e] = fmaxf(s[0][2 * e], s[0][2 * e + 1]);
#pragma unroll
                for (int n = 1; n < 2 * KG; ++n) mx[e] = fmaxf(mx[e], fmaxf(s[n][2 * e], s[n][2 * e + 1]));
                mx[e] *= mul[e];
            }
        } else {
            mx[0] = mx[1] = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2 * KG; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = i >> 1, j = j0 + 8 * n + 2 * c + (i & 1);
                    float x = s[n][i] * mul[e];
                    if (special) {
                        x = s[n][i] * sc[e];
                        if (p.softcap > 0.0f) x = p.softcap * tanhf(x / p.softcap);
                        x -= slope[e] * fabsf((float)(r_pos[e] - j));
                        x *= PA_LOG2E;
                    }
                    if (!(j >= r_lo[e] && j < r_hi[e])) x = -INFINITY;
                    s[n][i] = x;
                    mx[e] = fmaxf(mx[e], x);
                }
            mul[0] = mul[1] = 1.0f;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float mn = fmaxf(m[e], mx[e]), f = m[e] == -INFINITY ? 0.0f : fast_exp2(m[e] - mn);
                m[e] = mn;
                l[e] *= f;
#pragma unroll
                for (int n = 0; n < NT; ++n) oacc[n][2 * e] *= f, oacc[n][2 * e + 1] *= f;
            }
        }
        // weights up to 2^8, so that f16 holds those down to 2^-32 of the largest
        const float ms0 = m[0] == -INFINITY ? 0.0f : m[0] - 8.0f, ms1 = m[1] == -INFINITY ? 0.0f : m[1] - 8.0f;
#pragma unroll
        for (int n = 0; n < 2 * KG; ++n) {
            s[n][0] = fast_exp2(fmaf(s[n][0], mul[0], -ms0));
            s[n][1] = fast_exp2(fmaf(s[n][1], mul[0], -ms0));
            s[n][2] = fast_exp2(fmaf(s[n][2], mul[1], -ms1));
            s[n][3] = fast_exp2(fmaf(s[n][3], mul[1], -ms1));
            l[0] += s[n][0] + s[n][1];
            l[1] += s[n][2] + s[n][3];
        }
        // ---- O += P V
        auto weights = [&](auto bf, int kk, uint32_t(&pa)[4]) {
            pa[0] = pa_pack2<bf.value>(s[2 * kk][0], s[2 * kk][1]);
            pa[1] = pa_pack2<bf.value>(s[2 * kk][2], s[2 * kk][3]);
            pa[2] = pa_pack2<bf.value>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
            pa[3] = pa_pack2<bf.value>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
        };
        if (!MX) {
            const uint32_t vr = (lane & 7) + ((lane >> 3) & 1) * 8, vc = lane >> 4;
#pragma unroll
            for (int kk = 0; kk < KG; ++kk) {
                uint32_t pa[4];
                weights(std::bool_constant<BF16>{}, kk, pa);
#pragma unroll
                for (int np = 0; np < NT / 2; ++np) {
                    uint32_t b0, b1, b2, b3;
                    pa_ldsm_trans(tv + C::at(kk * 16 + vr, np * 2 + vc), b0, b1, b2, b3);
                    pa_mma<BF16>(oacc[2 * np], pa, b0, b1);
                    pa_mma<BF16>(oacc[2 * np + 1], pa, b2, b3);
                }
            }
        } else {
            // Column n = g of the products' tile i is element g HD / 8 + i: a lane reads the same bytes of its four keys. Values and weights in f16, also
            // under bf16 queries, where f16 holds every code times the scale exactly: 2^-9 2^-15 is its smallest number, 448 2^7 is below its largest, so scale
            // bytes from 112 to 134 (weights have three bits more there). f16 queries round values to f16 in any case and go down to byte 105, whose power
            // of two f16 still has. Tiles with scales outside that take the second form: two factors, or bf16 under bf16 queries.
            constexpr int W = HD / 32;  // words of a lane's elements
            constexpr uint32_t E_LO = BF16 ? 112 : 105, E_HI = 134;
            const uint32_t vsc = tsc + KEYS * C::NB + g * (HD / 8) / 32;
            uint32_t e[KG][4], off = 0;
#pragma unroll
            for (int kk = 0; kk < KG; ++kk)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    e[kk][k] = pa_lds8(vsc + (kk * 16 + 2 * c + (k & 1) + (k >> 1) * 8) * C::NB);
                    off = __viaddmax_u32(e[kk][k], 0u - E_LO, off);
                }
            auto products = [&](auto bf, auto far) {
                constexpr bool B = bf.value, FAR = far.value;
#pragma unroll
                for (int kk = 0; kk < KG; ++kk) {
                    uint32_t pa[4], f[2], rest[2];
                    weights(bf, kk, pa);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (FAR) f[k] = pool_scale2<B>(e[kk][2 * k], e[kk][2 * k + 1], rest[k]);
                        else f[k] = pack_f16x2(u2f(e[kk][2 * k] << 23), u2f(e[kk][2 * k + 1] << 23));
#pragma unroll
                    for (int i = 0; i < W; i += 2) {
                        uint32_t w[4][2];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint2 v = pa_lds64(tv + C::at(kk * 16 + 2 * c + (k & 1) + (k >> 1) * 8, (g * W + i) >> 2) + ((g * W + i) & 3) * 4);
                            w[k][0] = v.x, w[k][1] = v.y;
                        }
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t b[2][4];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                pool_codes4<B>(w[2 * k][x], w[2 * k + 1][x], b[k]);
#pragma unroll
                                for (int y = 0; y < 4; ++y) {
                                    if (FAR && !B) b[k][y] = pool_mul2<B>(b[k][y], rest[k]);
                                    b[k][y] = pool_mul2<B>(b[k][y], f[k]);
                                }
                            }
#pragma unroll
                            for (int y = 0; y < 4; ++y) pa_mma<B>(oacc[(i + x) * 4 + y], pa, b[0][y], b[1][y]);
                        }
                    }
                }
            };
            if (__any_sync(0xffffffffu, off > E_HI - E_LO)) products(std::bool_constant<BF16>{}, std::true_type{});
            else products(std::false_type{}, std::false_type{});
        }
        __syncwarp();  // the stage has been read
        if (TMA) {
            if (t + C::NS < nu) {
                if (dirty) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // it has been written, too
                sent = copy(st, ahead, ahead_row) ? sent | 1u << st : sent & ~(1u << st);
                advance(lead);
                if (t + C::NS + 1 < nu) ahead = page_of();
            } else {
                sent &= ~(1u << st);
            }
        } else {
            if (t + C::NS < nu) {
                request(st);
                advance(lead);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }

        // ---- the end of the column, or of the block's share
        if (!CLUSTER && (cur.u + 1 == cur.s.uhi || t + 1 == nu)) {
            finish(cur, seg_u == cur.s.ulo && cur.u + 1 == cur.s.uhi, 2ull * blockIdx.x + (seg ? 1 : 0));
            const uint32_t rest = (uint32_t)(cur.s.uhi - cur.u - 1);
            if (tid == 0 && rest && seg_u == cur.s.ulo)
                p.part_col[blockIdx.x] = make_int4((int)cur.seq, (int)cur.pack, (int)((rest - 1) / share_units) + 2, (int)(2 * blockIdx.x + (seg ? 1 : 0)));
            ++seg;
            begin = true;
        }
        advance(cur);
    }
    if (CLUSTER) {
        // the block's rows into its shared memory (the rings: every copy has been waited for), then the cluster's blocks share the outputs
        finish(cur, false, 0);
        pa_cluster_sync();
        const uint32_t at = smem_u32(smem), row0 = cur.pack * PA_ROWS, pairs = min((uint32_t)PA_ROWS, cur.s.rows - row0) * (p.d / 2);
        for (uint32_t i = rank * PA_THREADS + tid; i < pairs; i += ranks * PA_THREADS) {
            const uint32_t row = i / (p.d / 2), dd = 2 * (i - row * (p.d / 2));
            float2 ml[8], o[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                if (k >= ranks) break;
                ml[k] = pa_peer(at + C::CL_ML + row * 8, k);
                o[k] = pa_peer(at + (row * HD + dd) * 4, k);
            }
            float M = -INFINITY, L = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (k < ranks) M = fmaxf(M, ml[k].x);
            const float ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (k < ranks) {
                    const float f = fast_exp2(ml[k].x - ms);
                    L = fmaf(f, ml[k].y, L);
                    o0 = fmaf(f, o[k].x, o0);
                    o1 = fmaf(f, o[k].y, o1);
                }
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
            const uint32_t tok = (row0 + row) / p.group;
            *reinterpret_cast<uint32_t *>(p.out + (cur.s.q0 + tok) * p.o_st + (hk * p.group + row0 + row - tok * p.group) * p.o_sh + dd * 2) = pa_pack2<BF16>(o0 * inv, o1 * inv);
        }
        pa_cluster_sync();  // a block's shared memory is there until all have read it
    }
    if (!TMA) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (TMA && !ok && lane == 0) {
        for (int i = 0; i < C::NS; ++i) mbar_wait_bounded(&bars[i], 0, 1u << 12), mbar_wait_bounded(&bars[i], 1, 1u << 12);  // copies in flight land first
        atomicExch(&g_paged_wait_failed, 1);
    }
    in_order();
}

// Joins the parts of columns that lie in several shares: the block of the share in which a column begins (part_col). Its warps take rows and
// parts; a row's parts meet in shared memory.
template <bool BF16>
__global__ void __launch_bounds__(512) paged_join_kernel(const PaParams p) {
    __shared__ float s_o[16][256];
    __shared__ float s_l[16], s_m[16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 col = p.part_col[blockIdx.x];
    const uint32_t parts = (uint32_t)col.z, hk = blockIdx.x % p.hkv, row0 = (uint32_t)col.y * PA_ROWS;
    if (parts == 0) return;
    const uint32_t q0 = min(p.cu_q[col.x], p.total_q), all = min(min(p.cu_q[col.x + 1], p.total_q) - q0, p.max_q) * p.group, rows = min((uint32_t)PA_ROWS, all - row0);
    // warps per row, a power of two
    const uint32_t warps = blockDim.x >> 5;
    uint32_t per_row = warps;
    while (per_row > 1 && per_row * rows > warps) per_row /= 2;
    const uint32_t step = warps / per_row;
    for (uint32_t base = 0; base < rows; base += step) {
        const uint32_t row = base + warp / per_row, sub = warp % per_row;
        float M = -INFINITY, L = 0.0f, o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = 0.0f;
        if (row < rows)
            for (uint32_t k0 = sub; k0 < parts; k0 += 4 * per_row) {
                float2 ml[4];
                float4 v[4][2];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t part = k0 + k * per_row;
                    // a share's first segment is in its first slot; the column's first part has the slot that it says
                    const uint64_t slot = part == 0 ? (uint64_t)col.w : 2ull * (blockIdx.x + part * (uint64_t)p.hkv);
                    const bool in = part < parts;
                    ml[k] = in ? p.part_ml[slot * PA_ROWS + row] : make_float2(-INFINITY, 0.0f);
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const uint32_t d0 = hf * 128 + 4 * lane;
                        v[k][hf] = in && d0 < p.d ? *reinterpret_cast<const float4 *>(p.part_o + (slot * PA_ROWS + row) * p.d + d0) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                }
                const float mn = fmaxf(fmaxf(fmaxf(M, ml[0].x), fmaxf(ml[1].x, ml[2].x)), ml[3].x), ms = mn == -INFINITY ? 0.0f : mn;
                const float f = fast_exp2(M - ms);
                M = mn;
                L *= f;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] *= f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float w = fast_exp2(ml[k].x - ms);
                    L = fmaf(w, ml[k].y, L);
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        o[4 * hf] = fmaf(w, v[k][hf].x, o[4 * hf]);
                        o[4 * hf + 1] = fmaf(w, v[k][hf].y, o[4 * hf + 1]);
                        o[4 * hf + 2] = fmaf(w, v[k][hf].z, o[4 * hf + 2]);
                        o[4 * hf + 3] = fmaf(w, v[k][hf].w, o[4 * hf + 3]);
                    }
                }
            }
        if (per_row > 1) {
            if (lane == 0) s_m[warp] = M, s_l[warp] = L;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) *reinterpret_cast<float4 *>(&s_o[warp][hf * 128 + 4 * lane]) = make_float4(o[4 * hf], o[4 * hf + 1], o[4 * hf + 2], o[4 * hf + 3]);
            __syncthreads();
            if (sub == 0 && row < rows) {
                float mn = M;
                for (uint32_t w = 1; w < per_row; ++w) mn = fmaxf(mn, s_m[warp + w]);
                const float ms = mn == -INFINITY ? 0.0f : mn, f = fast_exp2(M - ms);
                L *= f;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] *= f;
                for (uint32_t w = 1; w < per_row; ++w) {
                    const float g = fast_exp2(s_m[warp + w] - ms);
                    L = fmaf(g, s_l[warp + w], L);
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[4 * hf + i] = fmaf(g, s_o[warp + w][hf * 128 + 4 * lane + i], o[4 * hf + i]);
                }
            }
            __syncthreads();
        }
        if (sub == 0 && row < rows) {
            const uint32_t r = row0 + row, tok = r / p.group;
            char *const orow = p.out + (q0 + tok) * p.o_st + (hk * p.group + r - tok * p.group) * p.o_sh;
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const uint32_t d0 = hf * 128 + 4 * lane;
                if (d0 < p.d)
                    *reinterpret_cast<uint2 *>(orow + d0 * 2) = make_uint2(pa_pack2<BF16>(o[4 * hf] * inv, o[4 * hf + 1] * inv), pa_pack2<BF16>(o[4 * hf + 2] * inv, o[4 * hf + 3] * inv));
            }
        }
    }
}

// Key splits of the tcgen05 tiles: one warp per token and head of the sequences that are theirs, as fa_combine_kernel. Rows whose item was not split
// say so in their first split's sum. (Four heads a warp, with fewer warps: 217 for 185 us, 700 tokens over 12000 keys.)
template <bool BF16>
__global__ void __launch_bounds__(128) paged_split_join(const PaParams p, const uint32_t row_cap, const float *__restrict__ part_o, const float *__restrict__ part_lse,
                                                        const uint32_t n_splits) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t rows = (uint64_t)p.total_q * p.hq;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint64_t row = (uint64_t)blockIdx.x * 4 + warp; row < rows; row += (uint64_t)gridDim.x * 4) {
        const uint32_t tok = (uint32_t)(row / p.hq), h = (uint32_t)(row - (uint64_t)tok * p.hq);
        if (tok >= p.cu_q[p.b]) return;
        const uint32_t seq = pool_seq(p.cu_q, p.b, tok, lane), q0 = p.cu_q[seq], lq = min(p.cu_q[seq + 1], p.total_q) - q0;  // (cut as in pa_seq)
        if (tok < q0 || tok - q0 >= min(lq, p.max_q) || min(lq, p.max_q) * p.group <= row_cap) continue;
        float e0 = (uint32_t)lane < n_splits ? part_lse[(uint64_t)lane * rows + row] : -INFINITY;
        if (__shfl_sync(0xffffffffu, e0, 0) == INFINITY) continue;  // not split
        float e1 = (uint32_t)lane + 32 < n_splits ? part_lse[(uint64_t)(lane + 32) * rows + row] : -INFINITY;
        float mx = fmaxf(e0, e1);
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        e0 = e0 == -INFINITY ? 0.0f : expf(e0 - mx);
        e1 = e1 == -INFINITY ? 0.0f : expf(e1 - mx);
        float wsum = e0 + e1;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) wsum += __shfl_xor_sync(0xffffffffu, wsum, k);
        const uint32_t d = 4 * lane;  // (head dims up to 128)
        float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t s0 = 0; s0 < n_splits; s0 += 4) {
            float4 v[4];
            float w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t s = s0 + k;
                w[k] = __shfl_sync(0xffffffffu, s < 32 ? e0 : e1, s & 31u);
                if (s >= n_splits || d >= p.d) w[k] = 0.0f;
                v[k] = w[k] != 0.0f ? *reinterpret_cast<const float4 *>(part_o + ((uint64_t)s * rows + row) * p.d + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) a[0] += w[k] * v[k].x, a[1] += w[k] * v[k].y, a[2] += w[k] * v[k].z, a[3] += w[k] * v[k].w;
        }
        if (d < p.d) {
            const float inv = wsum == 0.0f ? 0.0f : 1.0f / wsum;
            *reinterpret_cast<uint2 *>(p.out + (uint64_t)tok * p.o_st + h * p.o_sh + d * 2) = make_uint2(pa_pack2<BF16>(a[0] * inv, a[1] * inv), pa_pack2<BF16>(a[2] * inv, a[3] * inv));
        }
    }
}

struct PaPlan {
    PaParams p;
    int hd, kind, unit;
    uint32_t box;  // rows of a tensor copy, 0: 16-byte chunks
    uint32_t cluster;  // blocks of a cluster per column, 0: shares
    size_t ws_bytes, off_ml, off_col;
    // the tcgen05 tiles: sequences of more than 16 packed rows
    bool tiles, steps;  // they are launched; the kernel of this file is
    FaParams fa;
    FaPages pg;
    size_t off_split, off_lse;
};

static int pa_plan(const B200PagedAttnArgs *a, PaPlan &pl, bool may_map = true) {
    const char *what = "paged_attention";
    if (!a) return set_error(B200_ERR_BAD_ARG, "%s: null args", what);
    PaParams &p = pl.p;
    memset(&p, 0, sizeof(p));
    const int rc = pool_params(a->pool, what, &p.pool);
    if (rc) return rc;
    if (a->q_dtype != B200_F16 && a->q_dtype != B200_BF16) return set_error(B200_ERR_BAD_ARG, "%s: query dtype %d (f16, bf16)", what, a->q_dtype);
    if (a->pool.dtype != B200_FP8 && a->pool.dtype != a->q_dtype) return set_error(B200_ERR_BAD_ARG, "%s: a pool of dtype %d under queries of dtype %d", what, a->pool.dtype, a->q_dtype);
    if (a->hq == 0 || a->hq % a->pool.hkv) return set_error(B200_ERR_BAD_ARG, "%s: %u query heads are not a multiple of %u kv heads", what, a->hq, a->pool.hkv);
    if (a->max_k >= (1u << 30) || a->total_q >= (1u << 30)) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: %u tokens over %u keys", what, a->total_q, a->max_k);
    if ((uint64_t)a->max_q * (a->hq / a->pool.hkv) >= (1ull << 31)) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: %u tokens of a sequence", what, a->max_q);
    uint64_t low = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out);
    for (int i = 0; i < 2; ++i) low |= (a->q_strides[i] | a->out_strides[i]) * 2;
    if (low & 15) return set_error(B200_ERR_UNSUPPORTED_SHAPE, "%s: the rows of q and out must start at multiples of 16 bytes", what);
    p.q = static_cast<const char *>(a->q), p.out = static_cast<char *>(a->out);
    p.q_st = a->q_strides[0] * 2, p.q_sh = a->q_strides[1] * 2, p.o_st = a->out_strides[0] * 2, p.o_sh = a->out_strides[1] * 2;
    p.cu_q = a->cu_q, p.kv_len = a->kv_len, p.table = a->table, p.table_stride = a->table_stride;
    p.alibi = a->alibi, p.alibi_bs = a->alibi_bstride, p.status = a->status;
    p.b = a->b, p.hq = a->hq, p.hkv = a->pool.hkv, p.group = a->hq / a->pool.hkv, p.d = a->pool.d;
    p.total_q = a->total_q, p.max_q = a->max_q, p.max_k = (uint32_t)std::min<uint64_t>(a->max_k, (uint64_t)a->table_cols * a->pool.block_rows), p.table_cols = a->table_cols;
    p.scale = a->scale, p.softcap = a->softcap, p.wl = a->wl, p.wr = a->wr;
    pl.hd = p.d <= 64 ? 64 : (p.d <= 128 ? 128 : 256);
    const bool mx = a->pool.dtype == B200_FP8;
    pl.kind = (mx ? 2 : 0) + (a->q_dtype == B200_BF16 ? 1 : 0);
    pl.unit = PA_WARPS * (pl.hd == 64 || (pl.hd == 128 && mx) ? 32 : 16);
    // Tensor copies: pages of whole groups of at least eight rows; MXFP8 rows whose scales then move in 16-byte pieces. 16-byte chunks serve the others.
    const uint32_t keys = (uint32_t)pl.unit / PA_WARPS;
    pl.box = keys;
    while (a->pool.block_rows % pl.box) pl.box /= 2;
    if (pl.box < 8 || (mx && (p.d != (uint32_t)pl.hd || pl.box * (p.d / 32) % 16)) || !may_map || !fa_pool_maps(p.pool, a->pool.dtype, false, pl.box, nullptr, nullptr, nullptr)) pl.box = 0;
    int sms = 148, dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const uint64_t rows_max = (uint64_t)a->max_q * p.group, blocks = (uint64_t)sms * (pl.hd == 256 ? 1 : 2);
    // Columns over few keys: a cluster of up to eight blocks each, as many as are resident at once (clusters do not fill every place: 37 of eight
    // blocks took two waves, 32 one), up to 1152 keys a block, or 576 where the clusters leave half of the places empty. us, shares
    // and clusters, 32 / 8 heads of 128 over bf16 (lengths alike; spread evenly up to the longest): 1 x 300 keys 10.2, 7.1; 1 x 2000 14.7,
    // 10.8; 1 x 4000 16.3, 16.0; 1 x 8000 19.1, 25.9; 8 x 2000 24.2, 17.9 (18.0, 17.0); 8 x 4000 36.5, 30.7 (25.8, 27.3); 16 x 2000 36.7, 30.3
    // (29.5, 27.1); 16 x 4000 57.3, 52.2 (41.6, 50.9); 37 x 1000 35.7, 31.9 (39.5, 27.2). MXFP8: 8 x 4000 31.5, 26.3 (22.1, 24.3).
    auto cluster = [&](uint64_t packs, uint32_t keys_half) -> uint32_t {
        const uint64_t columns = (uint64_t)a->b * p.hkv * packs;
        if (!pl.box || columns == 0 || columns > blocks) return 0;
        uint32_t n = 8;
        while (n > 1 && columns * n > blocks / 8 * 7) n /= 2;
        return p.max_k <= (uint64_t)(columns * n * 2 > blocks ? keys_half : 576) * n ? n : 0;
    };
    // Short sequences stay here, long ones are on the tcgen05 tiles, where these take the call at all: one group of 16 packed rows (of
    // mma.sync) is bound by its keys' bytes, and two under MXFP8 are as fast as tiles whose codes are widened; small calls of up to four
    // in clusters (a tile is 23 us from end to end). us, here and there, 32 / 8 heads of 128 over 48 x 4000 keys: bf16 16 rows 139, 213;
    // 20 rows 251, 214; MXFP8 16 rows 122, 243; 32 rows 231, 244 (f16 221, 238); 48 rows 330, 244. Over 1 x 1000: bf16 16 rows 8.8, 24.0; 64 rows 11.1, 24.3. Where all
    // lengths are alike as far as the bounds tell, one kernel has all.
    const uint32_t few = rows_max <= 64 ? cluster((rows_max + PA_ROWS - 1) / PA_ROWS, 576) : 0;
    const uint32_t cap = few ? 64 : (mx ? 2 * PA_ROWS : PA_ROWS);
    pl.tiles = false, pl.steps = true;
    if (may_map && rows_max > cap) {
        FaParams &f = pl.fa;
        FaPages &g = pl.pg;
        memset(&f, 0, sizeof(f));
        memset(&g, 0, sizeof(g));
        f.q = a->q, f.o = a->out, f.cu_q = a->cu_q;
        f.b = a->b, f.lq = a->max_q, f.lk = p.max_k, f.hq = p.hq, f.hkv = p.hkv, f.d = p.d, f.group = p.group;
        f.q_ss = a->q_strides[0], f.q_sh = a->q_strides[1];
        f.scale = a->scale, f.softcap = a->softcap, f.alibi = a->alibi, f.kd = f.vd = 1.0f;
        f.wl = a->wl, f.wr = a->wr, f.varlen = 1, f.q_dtype = a->q_dtype;
        f.rows_total = (uint64_t)a->total_q * a->hq;
        g.pool = p.pool;
        g.table = a->table, g.kv_len = a->kv_len, g.status = a->status, g.table_stride = a->table_stride, g.table_cols = a->table_cols;
        g.o_ss = a->out_strides[0], g.o_sh = a->out_strides[1], g.total_q = a->total_q;
        const bool alike = (uint64_t)a->b * a->max_q == a->total_q;
        g.row_cap = alike ? 0 : cap;
        pl.tiles = fa_paged_tiles_take(f, g, a->pool.dtype);
        if (pl.tiles) {
            f.n_splits = fa_paged_tiles_splits(f, g, (uint32_t)sms);
            pl.steps = !alike;
            p.row_cap = cap;
        }
    }
    // as many shares as two blocks per SM (one at head dim 256), no more than there can be units
    const uint64_t packs = ((pl.tiles ? cap : rows_max) + PA_ROWS - 1) / PA_ROWS;
    const uint64_t most = std::max<uint64_t>((uint64_t)a->b * packs * ((p.max_k + pl.unit - 1) / pl.unit + 1), 1);
    p.shares = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(blocks / p.hkv, 1), most);
    p.packs = (uint32_t)packs;
    pl.cluster = packs == 1 ? cluster(1, 1152) : few;
    const size_t slots = (size_t)2 * p.shares * p.hkv;
    pl.off_split = pl.off_lse = 0;
    pl.off_ml = (slots * PA_ROWS * p.d * 4 + 255) / 256 * 256;
    pl.off_col = pl.off_ml + slots * PA_ROWS * 8;
    pl.ws_bytes = pl.steps && p.shares > 1 ? pl.off_col + slots * 8 : 0;
    if (pl.tiles && pl.fa.n_splits > 1) {
        pl.off_split = (pl.ws_bytes + 255) / 256 * 256;
        pl.off_lse = pl.off_split + (pl.fa.n_splits * pl.fa.rows_total * p.d * 4 + 255) / 256 * 256;
        pl.ws_bytes = pl.off_lse + pl.fa.n_splits * pl.fa.rows_total * 4;
    }
    return B200_OK;
}

template <int HD, int KIND, int MODE>
static int pa_launch_as(const PaPlan &pl, const CUtensorMap &tm_k, const CUtensorMap &tm_v, uint32_t order, cudaStream_t stream) {
    static thread_local bool done[16] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 16 || !done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(paged_decode_kernel<HD, KIND, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PA<HD, KIND>::SMEM);
        if (e != cudaSuccess) return set_error(B200_ERR_LAUNCH, "paged_attention: shared memory opt-in: %s", cudaGetErrorString(e));
        if (dev >= 0 && dev < 16) done[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(MODE == PA_CLUSTER ? pl.p.b * pl.p.packs * pl.p.hkv * pl.cluster : pl.p.shares * pl.p.hkv);
    cfg.blockDim = dim3(PA_THREADS);
    cfg.dynamicSmemBytes = PA<HD, KIND>::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    if (pl.tiles) {  // behind the tiles' kernel, which reads and writes nothing of this one's
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (MODE == PA_CLUSTER) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = pl.cluster, attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    cfg.attrs = attr;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_kernel<HD, KIND, MODE>, pl.p, tm_k, tm_v, order, pl.box);
    if (e != cudaSuccess) return set_error(B200_ERR_LAUNCH, "paged_attention: %s", cudaGetErrorString(e));
    return check_launch("paged_attention");
}
template <int HD, int KIND>
static int pa_launch(const PaPlan &pl, cudaStream_t stream) {
    CUtensorMap tm_k, tm_v;
    uint32_t order = 0;
    memset(&tm_k, 0, sizeof(tm_k)), memset(&tm_v, 0, sizeof(tm_v));
    const bool tma = pl.box && fa_pool_maps(pl.p.pool, KIND >= 2 ? B200_FP8 : (KIND & 1 ? B200_BF16 : B200_F16), KIND & 1, pl.box, &tm_k, &tm_v, &order);
    if (tma && pl.cluster) return pa_launch_as<HD, KIND, PA_CLUSTER>(pl, tm_k, tm_v, order, stream);
    const int rc = tma ? pa_launch_as<HD, KIND, PA_COPIES>(pl, tm_k, tm_v, order, stream) : pa_launch_as<HD, KIND, PA_CHUNKS>(pl, tm_k, tm_v, 0, stream);
    if (rc || pl.p.shares == 1) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((pl.p.shares - 1) * pl.p.hkv);
    cfg.blockDim = dim3(pl.p.b * 8 < pl.p.shares ? 512 : 256);  // columns over many shares: more warps for their parts
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_join_kernel<PA<HD, KIND>::BF16>, pl.p);
    if (e != cudaSuccess) return set_error(B200_ERR_LAUNCH, "paged_attention (join): %s", cudaGetErrorString(e));
    return check_launch("paged_attention (join)");
}
template <int HD>
static int pa_kind(const PaPlan &pl, cudaStream_t stream) {
    switch (pl.kind) {
    case 0: return pa_launch<HD, 0>(pl, stream);
    case 1: return pa_launch<HD, 1>(pl, stream);
    case 2: return pa_launch<HD, 2>(pl, stream);
    default: return pa_launch<HD, 3>(pl, stream);
    }
}

static int pa_steps(const PaPlan &pl, cudaStream_t stream) {
    if (pl.hd == 64) return pa_kind<64>(pl, stream);
    if (pl.hd == 128) return pa_kind<128>(pl, stream);
    return pa_kind<256>(pl, stream);
}
static int pa_tiles(const PaPlan &pl, int pool_dtype, cudaStream_t stream) {
    int rc = fa_paged_tiles_launch(pl.fa, pl.pg, pool_dtype, stream);
    if (rc || pl.fa.n_splits == 1) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<uint64_t>((pl.fa.rows_total + 3) / 4, 148ull * 16));
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, pl.kind & 1 ? paged_split_join<true> : paged_split_join<false>, pl.p, pl.pg.row_cap, (const float *)pl.fa.part_o,
                                             (const float *)pl.fa.part_lse, pl.fa.n_splits);
    if (e != cudaSuccess) return set_error(B200_ERR_LAUNCH, "paged_attention (split join): %s", cudaGetErrorString(e));
    return check_launch("paged_attention (split join)");
}

int paged_wait_status() {
    int v = 0;
    return cudaMemcpyFromSymbol(&v, g_paged_wait_failed, sizeof(int)) == cudaSuccess ? v : -1;
}
int paged_wait_clear() {
    const int zero = 0;
    return cudaMemcpyToSymbol(g_paged_wait_failed, &zero, sizeof(int)) == cudaSuccess ? 0 : -1;
}

}  // namespace b200

using namespace b200;

extern "C" size_t b200_paged_attention_workspace_bytes(const B200PagedAttnArgs *a) {
    PaPlan pl;
    if (pa_plan(a, pl)) return 0;
    const size_t need = pl.ws_bytes;
    if (!pl.tiles) return need;
    pa_plan(a, pl, false);  // should the driver refuse a tensor map
    return std::max(need, pl.ws_bytes);
}

extern "C" int b200_paged_attention(const B200PagedAttnArgs *a, b200_stream_t stream_) {
    PaPlan pl;
    int rc = pa_plan(a, pl);
    if (rc) return rc;
    if (a->b == 0 || a->total_q == 0 || a->max_q == 0) return B200_OK;
    if (!a->q || !a->out || !a->cu_q || !a->kv_len || !a->table) return set_error(B200_ERR_BAD_ARG, "paged_attention: null pointer");
    cudaStream_t stream = (cudaStream_t)stream_;
    for (int attempt = 0; attempt < 2; ++attempt) {
        if (pl.ws_bytes) {
            if (!a->workspace || a->workspace_bytes < pl.ws_bytes)
                return set_error(B200_ERR_WORKSPACE, "paged_attention: workspace of %zu bytes needed, %zu given", pl.ws_bytes, a->workspace ? a->workspace_bytes : (size_t)0);
            if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return set_error(B200_ERR_BAD_ARG, "paged_attention: workspace must be 16-byte aligned");
            char *ws = static_cast<char *>(a->workspace);
            pl.p.part_o = reinterpret_cast<float *>(ws);
            pl.p.part_ml = reinterpret_cast<float2 *>(ws + pl.off_ml);
            pl.p.part_col = reinterpret_cast<int4 *>(ws + pl.off_col);
            pl.fa.part_o = reinterpret_cast<float *>(ws + pl.off_split);
            pl.fa.part_lse = reinterpret_cast<float *>(ws + pl.off_lse);
        }
        rc = pl.tiles ? pa_tiles(pl, a->pool.dtype, stream) : B200_OK;
        if (rc != FA_NO_MAP) return rc || !pl.steps ? rc : pa_steps(pl, stream);
        // the driver refuses a tensor map of this call's tensors: nothing has been launched
        rc = pa_plan(a, pl, false);
        if (rc) return rc;
    }
    return rc;
}
