// Tensor-core kernel of products grouped by row, bf16: Y[r,:] = X[r,:] . W_g and dX[r,:] = dY[r,:] . W_g^T for the rows r of group g.
//
// The block is computed TRANSPOSED: the weight's columns (FWD; its rows for DX) are the MMA's M, the group's rows its N.  M comes in
// blocks of 128 a CTA and weights are that wide; N may be any multiple of 16 (32 for a pair), so a block has as many columns as
// the group has rows and no group pays for a row block it does not fill.  A group with more rows than a block takes is cut into
// equal pieces (the plan kernel's list).  For few rows a stage is nearly all weight: the kernel then streams weights at the rate the
// TMA unit fetches them, which is what bounds it.
//   RB = 1: 128 weight columns a CTA, accumulators double-buffered in TMEM.  RB = 2: 2 x 128, which share the rows' tile; with NMAX = 256
//   all of TMEM is then one block's.
//   CTAS = 2: a cluster of two CTAs drives M = 256 MMAs, each CTA staging its own weight columns and half of the rows.
//   NMAX: most rows of a block.  Few rows leave the shared memory to a deeper ring.
// What a stage costs, measured with all weights in L2: a row of a weight box starts at a multiple of
// 16 bytes and so covers two cache lines, about 4.5 clocks of the TMA unit; an aligned row of X costs 1.8.  A stage of 128 weight
// columns takes 650 clocks plus one for each row of X, a stage of 2 x 128 takes 1140 plus 2.4.
// The weights come from the shifted copies, which hold the fp32 array rounded to bf16 (at most 2^-8 of a weight; in a product it shows as
// 1.7e-3 of the result, root mean square, as much as rounding the result to bf16 does).  It is the linear layer's choice too: keeping
// the lost bits would take a second MMA and twice the weight loads, which are what bounds few rows.  Sums are fp32.
// Roles, ring, bounded waits and hash tables of the producers are those of rz_tc_kernel.cuh, except that four warps produce.  Accumulator
// rows are weight columns, so an epilogue thread owns one output column of 32 rows: bias is one value a thread, and 32 rows x 32 columns are transposed by
// 2-byte stores into a tile of 64-byte rows (a warp's lanes are neighbours in the row: no bank conflicts), which a bulk tensor
// store writes out; rows of a ragged end are stored one by one, since the rows behind belong to the next group.
#pragma once
#include "rz_common.h"
#include "rz_ptx.cuh"

using namespace rzptx;

namespace {

constexpr int ROWS_FWD = 0, ROWS_DX = 1;
constexpr int ROWS_A_BLOCK = 16384;      // 128 weight columns x 64 contraction elements
constexpr int ROWS_BATCH = 4;            // pipeline stages per hash batch of a producer warp
constexpr int ROWS_PRODUCERS = 4;        // warps that issue loads
constexpr int ROWS_MAX_BOXES = 8;        // weight boxes per stage at most
constexpr int ROWS_MAX_STAGES = 10;
constexpr int ROWS_SMEM_TABLE = ROWS_PRODUCERS * ROWS_BATCH * ROWS_MAX_BOXES * 8;
constexpr int ROWS_SMEM_BARS = (2 * ROWS_MAX_STAGES + 5) * 8;
constexpr int ROWS_SMEM_LIMIT = 232448;
constexpr int ROWS_TILE_BYTES = 2048;    // a warp's store tile: 32 rows x 32 columns

__host__ __device__ constexpr int rows_stage_bytes(int ctas, int rb, int nmax) { return rb * ROWS_A_BLOCK + nmax / ctas * 128; }
__host__ __device__ constexpr int rows_smem_fixed(int rb) { return 4 * rb * 2 * ROWS_TILE_BYTES + ROWS_SMEM_TABLE + ROWS_SMEM_BARS + 16 + 1024; }
__host__ __device__ constexpr int rows_stages(int ctas, int rb, int nmax)
{
    const int n = (ROWS_SMEM_LIMIT - rows_smem_fixed(rb)) / rows_stage_bytes(ctas, rb, nmax);
    return n > ROWS_MAX_STAGES ? ROWS_MAX_STAGES : n;
}
__host__ __device__ constexpr int rows_smem_total(int ctas, int rb, int nmax)
{
    return rows_stages(ctas, rb, nmax) * rows_stage_bytes(ctas, rb, nmax) + rows_smem_fixed(rb);
}

__host__ __device__ constexpr int rows_threads(int rb) { return 32 * (1 + 4 * rb + ROWS_PRODUCERS); }

struct TcRowsParams {
    RzHash hash;
    RzHash32 hash32;
    int bk_shift, bn_shift;     // log2 of the hash tile's sides, -1 for other sides
    const uint32_t *header;     // [0] = pieces
    const uint4 *entries;       // {group, first row, end, 0} of each piece, at most NMAX rows
    uint32_t group_tiles;       // hash-tile rows of one group's weight
    uint32_t cols, tiles_c;     // output columns (the weight's N or K), blocks of them
    uint32_t nchunks;           // pipeline stages of the contraction
    uint32_t br_log2;           // weight rows per box: 32, 64 or 128
    uint32_t group_pieces;      // pieces per rasterisation group
    float alpha;
    int relu;
    const float *bias;          // [groups][cols] or NULL
    __nv_bfloat16 *out;
    WaitCtx wait;
};

__device__ __forceinline__ void rows_wait_cycles(uint32_t bar, uint32_t parity, long long cycles)
{
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > cycles) break;
}

// mapW: shifted copies {element, slice row, copy}; mapR16, 64, All: the rows' matrix in boxes of 16 rows, 64 rows and all the rows
// that a CTA stages of a full block; mapC: the output in boxes of 32 x 32
template <int OP, int CTAS, int RB, int NMAX>
__global__ void __launch_bounds__(rows_threads(RB), 1)
rz_tc_rows_kernel(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapR16,
                  const __grid_constant__ CUtensorMap mapR64, const __grid_constant__ CUtensorMap mapRAll,
                  const __grid_constant__ CUtensorMap mapC, const TcRowsParams p)
{
    constexpr int KC = 64;                                    // contraction elements per stage: one 128-byte row
    constexpr int STAGES = rows_stages(CTAS, RB, NMAX);
    constexpr int STAGE_BYTES = rows_stage_bytes(CTAS, RB, NMAX);
    constexpr int A_BYTES = RB * ROWS_A_BLOCK;
    constexpr int PAIR_M = 128 * CTAS, ITEM_M = PAIR_M * RB;  // weight columns of an accumulator / of a block
    constexpr int NBUF = 2 * RB * NMAX <= 512 ? 2 : 1;
    constexpr int EPI_WARPS = 4 * RB;
    constexpr uint32_t N_STEP = 16 * CTAS;                    // MMA N granularity
    // A slot's fills come from different producers, and one bit of the phase tells the producer of stage c that stage c - STAGES has been
    // read.  The bit is right only if stage c - 2 STAGES has been read before it is looked at.  What the producer knows is that stage
    // c - ROWS_PRODUCERS - STAGES, which its own last stage waited for, has; stages are read in their order.
    static_assert(STAGES >= ROWS_PRODUCERS, "a producer must not be two phases ahead of a slot");
    static_assert(RB * NMAX <= 512 && NMAX % 32 == 0, "TMEM columns");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    constexpr int RING = STAGES * STAGE_BYTES, TILES = EPI_WARPS * 2 * ROWS_TILE_BYTES;
    const uint32_t bars = smem_base + RING + TILES + ROWS_SMEM_TABLE;
    const uint32_t bar_full = bars;                                // [STAGES] used in the leader CTA
    const uint32_t bar_empty = bars + 8 * ROWS_MAX_STAGES;         // [STAGES] one set per CTA
    const uint32_t bar_tfull = bars + 16 * ROWS_MAX_STAGES;        // [2]      one set per CTA
    const uint32_t bar_tempty = bars + 16 * ROWS_MAX_STAGES + 16;  // [2]      used in the leader CTA
    const uint32_t bar_drain = bars + 16 * ROWS_MAX_STAGES + 32;   // [1]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem_gen + RING + TILES + ROWS_SMEM_TABLE + ROWS_SMEM_BARS);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = (CTAS == 2) ? cluster_ctarank() : 0u;   // 0 = leader
    const uint32_t first_item = (CTAS == 2) ? cluster_id_x() : blockIdx.x;
    const uint32_t item_stride = gridDim.x / CTAS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_tfull + 8 * b, 1);
            mbar_init(bar_tempty + 8 * b, EPI_WARPS * CTAS);
        }
        mbar_init(bar_drain, 1);
        fence_barrier_init();
        fence_proxy_async();
        tma_prefetch_desc(&mapW);
        tma_prefetch_desc(&mapR16);
        tma_prefetch_desc(&mapR64);
        tma_prefetch_desc(&mapRAll);
        tma_prefetch_desc(&mapC);
    }
    if (warp == 1) {
        if (CTAS == 2) {
            tmem_alloc_pair(smem_u32(tmem_slot), 512);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_slot), 512);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync_all();   // the peer's barriers exist before anything signals them
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t *>(tmem_slot);

    grid_wait();   // (up to here: beside the kernel before this one)
    bool ok = true;
    const uint32_t pieces = ld_behind_wait(p.header);
    const uint32_t items = pieces * p.tiles_c;
    uint32_t group = 0, row = 0, row_end = 0, width = 0, tc = 0;   // the block decoded last; width = its rows, as the MMA's N
    // blocks are taken in groups of p.group_pieces pieces, column block after column block: the pieces of one group, which read the
    // same weights, run side by side.  The next block's piece is fetched while this one is worked on.
    uint4 ahead = make_uint4(0, 0, 0, 0);
    uint32_t ahead_tc = 0;
    auto fetch = [&](uint32_t item) {
        if (item >= items) return;
        const uint32_t per_group = p.group_pieces * p.tiles_c;
        const uint32_t g = item / per_group, within = item - g * per_group;
        const uint32_t first = g * p.group_pieces, n = min(pieces - first, p.group_pieces);
        ahead_tc = within / n;
        ahead = ld_behind_wait(p.entries + first + (within - ahead_tc * n));
    };
    auto decode = [&](uint32_t item) {   // the items of one role in their order
        tc = ahead_tc, group = ahead.x, row = ahead.y, row_end = ahead.z;
        width = (row_end - row + N_STEP - 1) / N_STEP * N_STEP;
        fetch(item + item_stride);
    };
    fetch(first_item);

    if (warp == 0 || warp >= 2 + EPI_WARPS) {
        // ===================== producers (both CTAs of a pair) =====================
        // A stage costs its producer some 300 clocks and 130 for each of its boxes (one thread, instruction after instruction), more
        // than the TMA unit or the tensor core needs for short stages: four warps take the stages in turn.
        const uint32_t which = warp == 0 ? 0u : warp - (1 + EPI_WARPS);   // 0 .. ROWS_PRODUCERS - 1
        uint2 *mine = reinterpret_cast<uint2 *>(smem_gen + RING + TILES) + which * (ROWS_BATCH * ROWS_MAX_BOXES);   // boxes: element in a copy, slice row << 3 | copy
        auto tile_of = [](uint32_t v, uint32_t side, int shift) { return shift >= 0 ? v >> shift : v / side; };
        const uint32_t br = 1u << p.br_log2, per_block_log2 = 7 - p.br_log2;
        const uint32_t boxes_log2 = (RB - 1) + per_block_log2, boxes = 1u << boxes_log2, box_bytes = br * 128u;   // (RB is 1 or 2)
        uint32_t full_base = bar_full;
        if (CTAS == 2) full_base = mapa_cluster(bar_full, 0);
        uint32_t slot = which % STAGES, phase = (which / STAGES & 1) ^ 1;   // this warp's next slot of the ring, and the parity that says it is free
        uint32_t skip = which;                                              // stages of other producers before this warp's next one
        for (uint32_t item = first_item; item < items && ok; item += item_stride) {
            decode(item);
            const uint32_t staged = width / CTAS, row0 = row + rank * staged;   // rows this CTA stages
            const uint32_t stage_tx = (uint32_t)CTAS * (A_BYTES + staged * 128u);
            const uint32_t tile0 = group * p.group_tiles;
            const uint32_t col0 = tc * ITEM_M + rank * 128;                     // weight columns of block r: col0 + r * PAIR_M
            uint32_t c = skip;
            while (c < p.nchunks && ok) {
                const uint32_t nb = min((uint32_t)ROWS_BATCH, (p.nchunks - c + ROWS_PRODUCERS - 1) / ROWS_PRODUCERS);
                __syncwarp();
                // the boxes' places, a batch of this warp's stages at once; in 32 bits where possible, and without divisions
                for (uint32_t e = lane; e < nb << boxes_log2; e += 32) {
                    const uint32_t stage = c + (e >> boxes_log2) * ROWS_PRODUCERS, j = e & (boxes - 1);
                    const uint32_t r = j >> per_block_log2, i = j & ((1u << per_block_log2) - 1);
                    uint32_t k, n;   // first weight row and column of the box
                    if (OP == ROWS_FWD) {
                        // boxes of a block: two halves of 64 columns, each in 64 / br parts along the contraction (br <= 64)
                        const uint32_t parts_log2 = 6 - p.br_log2;
                        n = col0 + r * PAIR_M + (i >> parts_log2) * 64;
                        k = stage * KC + (i & ((1u << parts_log2) - 1)) * br;
                    } else {
                        n = stage * KC;
                        k = col0 + r * PAIR_M + i * br;
                    }
                    const uint32_t pk = tile_of(k, (uint32_t)p.hash.BK, p.bk_shift), pn = tile_of(n, (uint32_t)p.hash.BN, p.bn_shift);
                    const uint32_t off = rz_tile_offset32(p.hash, p.hash32, tile0 + pk, pn), sh = off & 7u;
                    mine[e] = make_uint2(off - sh + (n - pn * (uint32_t)p.hash.BN), (k - pk * (uint32_t)p.hash.BK) << 3 | sh);
                }
                __syncwarp();
                if (lane == 0) {
                    for (uint32_t ci = 0; ci < nb; ++ci) {
                        if (!mbar_wait_bounded(bar_empty + 8 * slot, phase, RZ_WAIT_SMEM_EMPTY, p.wait, 2000)) {
                            ok = false;
                            break;
                        }
                        const uint32_t full = full_base + 8 * slot;
                        uint32_t dst = smem_base + slot * STAGE_BYTES;
                        if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * slot, stage_tx);
#pragma unroll 1
                        for (uint32_t j = 0; j < boxes; ++j, dst += box_bytes) {
                            const uint2 u = mine[(ci << boxes_log2) + j];
                            if (CTAS == 2) tma_load_3d_pair(dst, &mapW, full, (int32_t)u.x, (int32_t)(u.y >> 3), (int32_t)(u.y & 7u));
                            else tma_load_3d(dst, &mapW, full, (int32_t)u.x, (int32_t)(u.y >> 3), (int32_t)(u.y & 7u));
                        }
                        const int32_t d0 = (int32_t)((c + ci * ROWS_PRODUCERS) * KC);
                        if (staged == NMAX / CTAS) {
                            if (CTAS == 2) tma_load_2d_pair(dst, &mapRAll, full, d0, (int32_t)row0);
                            else tma_load_2d(dst, &mapRAll, full, d0, (int32_t)row0);
                        } else {
                            uint32_t r = 0;
#pragma unroll 1
                            for (; r + 64 <= staged; r += 64) {
                                if (CTAS == 2) tma_load_2d_pair(dst + r * 128, &mapR64, full, d0, (int32_t)(row0 + r));
                                else tma_load_2d(dst + r * 128, &mapR64, full, d0, (int32_t)(row0 + r));
                            }
#pragma unroll 1
                            for (; r < staged; r += 16) {
                                if (CTAS == 2) tma_load_2d_pair(dst + r * 128, &mapR16, full, d0, (int32_t)(row0 + r));
                                else tma_load_2d(dst + r * 128, &mapR16, full, d0, (int32_t)(row0 + r));
                            }
                        }
                        for (slot += ROWS_PRODUCERS; slot >= STAGES; slot -= STAGES) phase ^= 1u;
                    }
                }
                __syncwarp();
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                c += nb * ROWS_PRODUCERS;
            }
            skip = c - p.nchunks;
        }
        if (!ok && lane == 0 && rank == 0) {
            // give the loads already issued time to land before the CTA retires: a stage's barrier ends the phase it was armed in
            for (uint32_t s = 0; s < STAGES; ++s) {
                rows_wait_cycles(bar_full + 8 * s, 0, 2000000);
                rows_wait_cycles(bar_full + 8 * s, 1, 2000000);
            }
        }
    } else if (warp == 1) {
        // ===================== MMA issuer (leader CTA only) =====================
        constexpr uint32_t ATOM = KC * 128;   // bytes of a 64-column block of an M-major tile
        constexpr uint32_t a_lbo = OP == ROWS_FWD ? ATOM : 16, a_kstep = OP == ROWS_FWD ? 16 * 128 : 32;
        // descriptors differ in their low words only, by sixteenths of the address (which stays below 2^18)
        const uint64_t a0 = make_desc_sw128(smem_base, a_lbo, 1024, 2), b0 = make_desc_sw128(smem_base + A_BYTES, 16, 1024, 2);
        const uint32_t a_lo = (uint32_t)a0, a_hi = (uint32_t)(a0 >> 32), b_lo = (uint32_t)b0, b_hi = (uint32_t)(b0 >> 32);
        uint32_t n_items = 0, slot = 0, phase = 0;
        for (uint32_t item = first_item; item < items && ok && rank == 0; item += item_stride, ++n_items) {
            decode(item);
            const uint32_t buf = n_items % NBUF, tph = (n_items / NBUF) & 1;
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((OP == ROWS_FWD ? 1u : 0u) << 15) | ((width >> 3) << 17) |
                                   ((uint32_t)(PAIR_M >> 4) << 24);
            if (lane == 0) {
                if (!mbar_wait_bounded(bar_tempty + 8 * buf, tph ^ 1, RZ_WAIT_TMEM_EMPTY, p.wait, 2000)) ok = false;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + buf * RB * NMAX;
                uint32_t acc = 0;
#pragma unroll 1
                for (uint32_t c = 0; c < p.nchunks && ok; ++c) {
                    if (!mbar_wait_bounded(bar_full + 8 * slot, phase, RZ_WAIT_SMEM_FULL, p.wait)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t al = a_lo + slot * (STAGE_BYTES / 16), bl = b_lo + slot * (STAGE_BYTES / 16);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint64_t bd = (uint64_t)b_hi << 32 | (bl + kk * (32 / 16));
#pragma unroll
                        for (int r = 0; r < RB; ++r) {
                            const uint64_t ad = (uint64_t)a_hi << 32 | (al + (r * ROWS_A_BLOCK + kk * a_kstep) / 16);
                            if (CTAS == 2) tc_mma_pair<false>(d_tmem + r * NMAX, ad, bd, idesc, acc);
                            else tc_mma<false>(d_tmem + r * NMAX, ad, bd, idesc, acc);
                        }
                        acc = 1;
                    }
                    // frees this stage in both CTAs once the MMAs have read it
                    if (CTAS == 2) tc_commit_pair(bar_empty + 8 * slot, 3);
                    else tc_commit(bar_empty + 8 * slot);
                    if (++slot == STAGES) slot = 0, phase ^= 1u;
                }
                if (ok) {
                    if (CTAS == 2) tc_commit_pair(bar_tfull + 8 * buf, 3);
                    else tc_commit(bar_tfull + 8 * buf);
                }
            }
            __syncwarp();
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        }
        if (!ok && lane == 0 && rank == 0) {
            // MMAs may still be running: wait (bounded) until the tensor core has drained
            if (CTAS == 2) tc_commit_pair(bar_drain, 1);
            else tc_commit(bar_drain);
            rows_wait_cycles(bar_drain, 0, 20000000);
        }
    } else {
        // ===================== epilogue (both CTAs; each drains its own 128 weight columns) =====================
        const uint32_t q = warp & 3;                 // TMEM lane quarter this warp may read
        const uint32_t rblk = (warp - 2) >> 2;       // which accumulator of the block
        uint8_t *tiles = smem_gen + RING + (warp - 2) * 2 * ROWS_TILE_BYTES;
        uint32_t tempty_base = bar_tempty, flip = 0;
        if (CTAS == 2) tempty_base = mapa_cluster(bar_tempty, 0);
        uint32_t n_items = 0;
        for (uint32_t item = first_item; item < items && ok; item += item_stride, ++n_items) {
            decode(item);
            const uint32_t buf = n_items % NBUF, tph = (n_items / NBUF) & 1;
            const uint32_t cbase = tc * ITEM_M + rblk * PAIR_M + rank * 128 + q * 32, col = cbase + lane;   // this thread's output column
            const bool col_ok = col < p.cols;
            const float bias = p.bias && col_ok ? __ldg(p.bias + (size_t)group * p.cols + col) : 0.f;
            bool mine = true;
            if (lane == 0) mine = mbar_wait_bounded(bar_tfull + 8 * buf, tph, RZ_WAIT_TMEM_FULL, p.wait, 20000);
            ok = __shfl_sync(0xffffffffu, (int)mine, 0) != 0;
            if (!ok) break;
            tc_fence_after();
            const uint32_t acc = tmem_base + ((q * 32u) << 16) + (buf * RB + rblk) * NMAX;
            // A warp whose columns all lie past the matrix stores nothing, and must not turn its tiles over either: the wait below lets the
            // newest store go on reading its tile, which is right only while every turn goes with a store.
            const uint32_t chunks = cbase < p.cols ? (row_end - row + 31) / 32 : 0u;
            uint32_t next[32];
            if (chunks) tmem_ld_32x32(acc, next);
#pragma unroll 1
            for (uint32_t c = 0; c < chunks; ++c) {
                uint32_t v[32];
                tmem_ld_wait_regs(next);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = next[j];
                if (c + 1 < chunks) tmem_ld_32x32(acc + (c + 1) * 32, next);   // streams while this chunk is converted and stored
                const uint32_t r0 = row + c * 32, rows = min(32u, row_end - r0);
                uint16_t h[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    float f = __uint_as_float(v[j]) * p.alpha + bias;
                    if (p.relu && f < 0.f) f = 0.f;   // (a NaN stays one)
                    h[j] = __bfloat16_as_ushort(__float2bfloat16_rn(f));
                }
                if (rows == 32) {
                    // the tile about to be rewritten: the store before the last must have read it
                    if (lane == 0) bulk_wait_group_read1();
                    __syncwarp();
                    uint16_t *tile = reinterpret_cast<uint16_t *>(tiles + flip * ROWS_TILE_BYTES);
#pragma unroll
                    for (int j = 0; j < 32; ++j) tile[j * 32 + lane] = h[j];
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&mapC, smem_u32(tile), (int32_t)cbase, (int32_t)r0);   // (columns past the matrix are clipped)
                        bulk_commit_group();
                    }
                    flip ^= 1;
                } else if (col_ok) {
                    __nv_bfloat16 *o = p.out + (size_t)r0 * p.cols + col;
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if ((uint32_t)j < rows) o[(size_t)j * p.cols] = __ushort_as_bfloat16(h[j]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CTAS == 2) mbar_arrive_cluster(tempty_base + 8 * buf);
                else mbar_arrive(bar_tempty + 8 * buf);
            }
        }
        if (lane == 0) bulk_wait_group0();   // bulk stores still in flight read this CTA's shared memory
    }

    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync_all();   // neither CTA retires while the peer may still signal or read it
    if (warp == 1) {
        tc_fence_after();
        __syncwarp();
        if (CTAS == 2) tmem_dealloc_pair(tmem_base, 512);
        else tmem_dealloc(tmem_base, 512);
    }
}

}  // namespace
