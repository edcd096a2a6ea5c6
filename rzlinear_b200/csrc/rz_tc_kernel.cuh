// Tensor-core (tcgen05 + TMEM + TMA) kernels of the RzLinear path for sm_100a.
//
// One persistent, warp-specialised kernel template covers the three contractions:
//   OP_FWD  Y [M,N] = X  [M,K] . W[K,N]      A = X tile  (K-major),  B = W slice (N-major)
//   OP_DX   dX[M,K] = dY [M,N] . W[K,N]^T    A = dY tile (K-major),  B = W slice (K-major)
//   OP_DW   dH     += dY^T[N,M] . X[M,K]     A = dY tile (M-major),  B = X tile  (N-major): the TRANSPOSE of the
//                                             weight-gradient block, so that a warp's 32 accumulator rows are 32
//                                             consecutive words of a slice row and reductions need no transpose
// CTAS = 1, RB = 1: a CTA owns a 128 x 256 output block (tcgen05.mma cta_group::1, M = 128).
// CTAS = 2, RB = 1: two CTAs of a cluster own a 256 x 256 block (cta_group::2, M = 256): each CTA
//           stages its 128 rows of A and its 128 columns of B.  The leader CTA (rank 0) issues the
//           MMAs for both; the barriers that gate them live in the leader.
// CTAS = 2, RB = 2: the pair owns a 512 x 256 block as two M = 256 MMAs per K-step that share B: each CTA
//           stages 2 x 128 rows of A and 128 columns of B, i.e. 48 KB per 1024 tensor-clocks instead of
//           32 KB per 512.  The main loop is bound by operand bytes per flop moved through an SM (L2 -> SM
//           reads of about 50 B/clk, and the shared-memory port that TMA writes and the MMAs' operand reads
//           share), so this is the fast configuration; it is used whenever the output has at least 512 rows.
// SPLIT = 1 (fp32 precision on the tensor cores, RB = 1 only): operands are fp32; four extra warps split every
//           staged tile in shared memory into hi = the tf32-representable part and lo = x - hi, and each K-step
//           issues hi*hi + hi*lo + lo*hi (three tf32 MMAs, fp32 accumulate): fp32-grade results (the dropped
//           lo*lo term and the rounding of lo are of relative order 2^-22) at a third of the tf32 rate.
// Accumulators live in TMEM (512 columns): with RB = 1 two 256-column buffers alternate so the epilogue of
// one block overlaps the main loop of the next; with RB = 2 both halves are accumulators of one block.
// Warp 0 produces (TMA loads into a ring of 128-byte-swizzled shared-memory tiles), warp 1 issues
// tcgen05.mma, 4*RB epilogue warps drain TMEM: they scale/bias/convert and store (FWD, DX) or scatter-add
// into the hashed gradient with warp-wide coalesced reductions (DW).  EW = 4 (DW, RB = 1): sixteen epilogue
// warps for weight gradients of short contractions, whose scatter outlasts the main loop.
//
// The virtual weight is never materialised.  For every pipeline stage the producer warp computes
// the hash-tile offsets in registers and TMA-loads the matching rows of the slice.  TMA needs a
// 16-byte aligned start, and a slice starts at any element, so FWD and DX read a "shadow" of the
// hashed array: NS element-shifted copies in the compute type (NS = 8 bf16 / 4 tf32); the copy
// whose shift equals offset mod NS holds the slice at an aligned position.  (Twice as many copies would
// align rows to 32-byte sectors - four L2 sectors per 128-byte row instead of five, worth 8 % when emulated -
// but the larger footprint costs more L2 misses than that; measured, not adopted.)  The shadow tensor map
// is 3-D {element, slice row (stride BN), copy}.
//
// GROUPED = 1: the rows of X, Y, dY and dX come in consecutive groups (the experts of a layer), each with a weight of its own.
//           The groups' weights are one virtual matrix, one below the other: group g's tile rows begin at g * group_tiles.  A plan
//           built on the device from the row offsets lists pieces {group, first row, end}: FWD and DX take a piece as the rows of
//           an output block (stores stop at its end), DW as the contraction of a whole weight's blocks.  The rows behind a
//           group belong to the next one, so DW reads X and dY through maps of the group's own that end with the group: the
//           TMA unit fills the last stage up with zeros.  Split precision in a grouped launch spreads a contraction over
//           chains that accumulate in TMEM columns of their own, where the ungrouped launch splits blocks: the tensor core
//           truncates when it adds, about 2.2e-8 of the sum a step (measured), so the error goes with the chain's length.
//
// Every TMA load is a plain per-CTA copy of this GPU's memory; no kernel touches peer-GPU memory.
// Every mbarrier wait is bounded: a wait that runs out records a code in the device status word and
// all roles leave their loops, the producer waits for its loads in flight, the MMA thread for its
// MMAs, TMEM is freed and the kernel returns.
#pragma once
#include <type_traits>

#include "rz_common.h"
#include "rz_ptx.cuh"

using namespace rzptx;

namespace {

constexpr int OP_FWD = 0, OP_DX = 1, OP_DW = 2;

constexpr int TILE_R = 128;  // rows per CTA and accumulator (MMA M = 128 * CTAS)
constexpr int A_BLOCK_BYTES = 16384;  // one 128-row block of A per stage
constexpr int BATCH = 8;     // pipeline stages per hash batch of the producer warp
constexpr int MAX_TPS = 8;   // B boxes per stage at most
constexpr int GROUP_ROWS = 8;   // row tiles per rasterisation group (4 when a tile has two row blocks)

// Shared-memory budget (227 KB per CTA): the operand ring takes what the other parts leave.
// The weight-gradient epilogue reduces straight from registers and needs no staging, so its ring gets the space.
constexpr int SMEM_TABLE = 3 * BATCH * MAX_TPS * 4;
constexpr int MAX_STAGES = 7;
constexpr int SMEM_BARS = (3 * MAX_STAGES + 5) * 8;
constexpr int SMEM_LIMIT = 232448;
// per epilogue warp: a 32-row x 128-byte store staging tile (FWD, DX); nothing for the weight gradient
// `ew`: epilogue warps per TMEM lane quarter and row block (weight gradient of short contractions: 4)
__host__ __device__ constexpr int smem_epi(int op, int rb, int ew = 1) { return op == OP_DW ? 0 : 4 * rb * ew * 4096; }
__host__ __device__ constexpr int load_bytes(int ctas, int rb, int nc) { return rb * A_BLOCK_BYTES + (nc / ctas) * 128; }
__host__ __device__ constexpr int stage_bytes(int ctas, int rb, int split, int nc) { return load_bytes(ctas, rb, nc) * (split ? 2 : 1); }
__host__ __device__ constexpr int num_stages(int op, int ctas, int rb, int split, int nc, int ew = 1)
{
    int n = (SMEM_LIMIT - 1024 - 16 - SMEM_BARS - SMEM_TABLE - smem_epi(op, rb, ew)) / stage_bytes(ctas, rb, split, nc);
    return n > MAX_STAGES ? MAX_STAGES : n;
}
__host__ __device__ constexpr int smem_total(int op, int ctas, int rb, int split, int nc, int ew = 1)
{
    return num_stages(op, ctas, rb, split, nc, ew) * stage_bytes(ctas, rb, split, nc) + smem_epi(op, rb, ew) + SMEM_TABLE + SMEM_BARS +
           16 + 1024;
}
__host__ __device__ constexpr int num_threads(int rb, int split, int ew = 1) { return 64 + 128 * rb * ew + (split ? 128 : 0); }

struct TcParams {
    RzHash hash;
    uint32_t M, K, N;
    uint32_t rows, cols;        // output extents (elements)
    uint32_t tiles_r, tiles_c;
    uint32_t nchunks;           // pipeline stages along the whole contraction
    uint32_t nsplit, chunks_per_split;   // blocks from index n_main on are split into nsplit parts of the contraction
    uint32_t n_main;                      // blocks [0, n_main) run their whole contraction in one work item
    uint32_t total_items;
    uint32_t units;             // > 0: the launch's (block, stage) units are dealt out in equal ranges (tiles * nchunks)
    uint32_t br;                // slice rows per B box (FWD: min(BK, stage depth); DX: min(BK, B columns of this CTA))
    uint32_t kparts;            // FWD: B boxes along the contraction per 128-byte column block (stage depth / br)
    uint32_t group_rows;        // row tiles per rasterisation group
    uint32_t a_lbo, a_sbo, b_lbo, b_sbo;                     // descriptor strides, bytes
    uint32_t a_layout, b_layout;                            // descriptor swizzle layout type
    uint32_t idesc;
    float alpha;
    int relu;
    const float *bias;
    void *out;
    float *dH;
    float *ws;                  // FWD / DX with a split contraction: fp32 partial sums [rows][cols]
    WaitCtx wait;               // where bounded waits report
    uint32_t tma_store;         // FWD / DX: write the output with bulk tensor stores (0 = plain 16-byte stores)
};

// What a grouped launch needs besides; `header` and `entries` are written by the plan kernel before it.
struct TcGroupParams : TcParams {
    RzHash32 hash32;
    const uint32_t *header;     // [0] = pieces
    const uint4 *entries;       // {group, first row, end, 0} of each piece
    const CUtensorMap *maps;    // DW: {dY, X} of each group
    uint32_t group_tiles;       // hash-tile rows of one group's weight
};

__device__ __forceinline__ void wait_cycles(uint32_t bar, uint32_t parity, long long cycles)
{
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > cycles) break;
}

template <int OP, bool TF32, int CTAS, int RB, int SPLIT, int NC, int EW, int GROUPED = 0>
__global__ void __launch_bounds__(num_threads(RB, SPLIT, EW), 1)
rz_tc_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
             const __grid_constant__ CUtensorMap mapC,
             const std::conditional_t<GROUPED != 0, TcGroupParams, TcParams> p)
{
    constexpr int ES = TF32 ? 4 : 2;        // operand element size
    constexpr int EPR = 128 / ES;           // elements per 128-byte swizzle row
    constexpr int KC = EPR;                 // contraction elements per stage
    constexpr int NS = 16 / ES;             // shifted shadow copies
    constexpr int MMAS = 4;                 // tcgen05.mma per stage (K = 16 bf16 / 8 tf32 each)
    constexpr int ATOM = KC * 128;          // bytes of one 128-byte-wide column block of an MN-major tile
    constexpr int TILE_C = NC;              // columns of the block (MMA N)
    constexpr int B_COLS = TILE_C / CTAS;   // columns of B this CTA stages
    constexpr int B_BYTES = B_COLS * 128;
    constexpr int A_BYTES = RB * A_BLOCK_BYTES;
    constexpr int LOAD_BYTES = A_BYTES + B_BYTES;                 // what TMA brings per stage and CTA
    constexpr int STAGE_BYTES = LOAD_BYTES * (SPLIT ? 2 : 1);     // SPLIT: the lo parts sit LOAD_BYTES above the hi parts
    constexpr int STAGES = num_stages(OP, CTAS, RB, SPLIT, NC, EW);
    constexpr bool PAIR_LOADS = (CTAS == 2) && !SPLIT;            // loads of both CTAs counted on the leader's barrier
    constexpr int EPI_WARPS = 4 * RB * EW;
    static_assert(EW == 1 || (OP == OP_DW && !SPLIT && ((RB == 1 && EW == 4) || (RB == 2 && EW == 2))),
                  "extra epilogue warps: weight gradient only (sixteen warps either way)");
    static_assert(!SPLIT || (TF32 && RB == 1), "split precision: fp32 operands, one row block");
    constexpr int SMEM_RING = STAGES * STAGE_BYTES;
    constexpr int SMEM_EPI_OP = smem_epi(OP, RB, EW);
    // accumulator sets in TMEM: 2 = double-buffered; 1 when both halves are in use by one block (two row blocks, or
    // the main + correction accumulators of split precision)
    constexpr int NBUF = (RB == 2 || SPLIT) ? 1 : 2;
    static_assert(STAGE_BYTES == stage_bytes(CTAS, RB, SPLIT, NC), "stage size");
    static_assert(NC == 256 || (CTAS == 1 && RB == 1), "narrow blocks: single CTA only");
    static_assert(2 * RB * NC <= 512 || RB == 2, "TMEM columns");
    // Split precision keeps the hi*hi sums and the (2^-11 smaller) hi*lo + lo*hi corrections in separate accumulators:
    // the tensor core truncates when it adds into an fp32 accumulator (about 2e-8 of the accumulator per MMA), so
    // the corrections must not cost the main chain two more truncating adds per K-step.  Chains are further bounded
    // by splitting long contractions on the host side.
    constexpr int CHAINS = (GROUPED && SPLIT) ? 512 / NC - 1 : 1;   // main accumulators a contraction may be spread over
    constexpr int CORR_COL = CHAINS * NC;   // TMEM column offset of the correction accumulator (SPLIT only)
    static_assert(RB == 1 || CTAS == 2, "two row blocks only with CTA pairs");
    constexpr int A_ATOMS = TILE_R / EPR;
    constexpr int B_ATOMS = B_COLS / EPR;
    constexpr int PAIR_R = TILE_R * CTAS;   // rows of one accumulator across the pair
    constexpr int ITEM_R = PAIR_R * RB;     // rows of a work item
    static_assert(STAGES <= MAX_STAGES, "barrier storage");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    float *epi_scratch = reinterpret_cast<float *>(smem_gen + SMEM_RING);
    uint32_t *tab_x = reinterpret_cast<uint32_t *>(smem_gen + SMEM_RING + SMEM_EPI_OP);
    uint32_t *tab_y = tab_x + BATCH * MAX_TPS;
    uint32_t *tab_z = tab_y + BATCH * MAX_TPS;
    const uint32_t bars = smem_base + SMEM_RING + SMEM_EPI_OP + SMEM_TABLE;
    const uint32_t bar_full = bars;                           // [STAGES]  used in the leader CTA
    const uint32_t bar_empty = bars + 8 * MAX_STAGES;         // [STAGES]  one set per CTA
    const uint32_t bar_tfull = bars + 16 * MAX_STAGES;        // [2]       one set per CTA
    const uint32_t bar_tempty = bars + 16 * MAX_STAGES + 16;  // [2]       used in the leader CTA
    const uint32_t bar_drain = bars + 16 * MAX_STAGES + 32;   // [1]
    const uint32_t bar_split = bars + 16 * MAX_STAGES + 40;   // [STAGES]  SPLIT only, used in the leader CTA
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem_gen + SMEM_RING + SMEM_EPI_OP + SMEM_TABLE + SMEM_BARS);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = (CTAS == 2) ? cluster_ctarank() : 0u;   // 0 = leader
    const uint32_t first_item = (CTAS == 2) ? cluster_id_x() : blockIdx.x;
    const uint32_t item_stride = gridDim.x / CTAS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
            mbar_init(bar_split + 8 * s, 4 * CTAS);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_tfull + 8 * b, 1);
            mbar_init(bar_tempty + 8 * b, EPI_WARPS * CTAS);
        }
        mbar_init(bar_drain, 1);
        fence_barrier_init();
        fence_proxy_async();
        if (!(GROUPED && OP == OP_DW)) {   // (those maps are the groups', in global memory)
            tma_prefetch_desc(&mapA);
            tma_prefetch_desc(&mapB);
        }
        if (OP != OP_DW) tma_prefetch_desc(&mapC);
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

    bool ok = true;

    // Work of this CTA (pair).  Two schedules:
    //  * items: work item i = one block with its whole contraction, or one of the nsplit parts of a split block; the
    //    CTA takes items first_item, first_item + item_stride, ...
    //  * units (p.units > 0, small grids whose every block is split): the (block, stage) pairs of the whole launch,
    //    block-major, are dealt out in equal contiguous ranges, one per CTA, so every SM gets the same number of
    //    stages whatever the number of blocks; a range that crosses a block boundary is worked off as two segments.
    // `item` below is the cursor of either schedule; decode() turns it into a block and a stage range and sets the
    // next cursor.  `tile` is the block index in rasterisation order, `partial` says that the segment is only a part
    // of its block's contraction (its result goes to the workspace as fp32 partial sums).
    uint32_t cur_begin = first_item, cur_end = p.total_items;
    uint32_t tiles_r = p.tiles_r;
    if constexpr (GROUPED) {
        grid_wait();   // (up to here: beside the kernel before this one)
        const uint32_t pieces = ld_behind_wait(p.header);
        if (OP != OP_DW) tiles_r = pieces;
        cur_end = OP == OP_DW ? pieces * p.tiles_r * p.tiles_c : pieces * p.tiles_c;
    }
    if (p.units) {
        cur_begin = (uint32_t)(((uint64_t)first_item * p.units) / item_stride);
        cur_end = (uint32_t)(((uint64_t)(first_item + 1) * p.units) / item_stride);
    }
    uint32_t tile = 0, next_item = 0;
    bool partial = false;
    uint32_t piece_row = 0, piece_end = 0, piece_group = 0;   // GROUPED: the piece of the block decoded last
    auto decode = [&](uint32_t item, uint32_t &tr, uint32_t &tc, uint32_t &c_begin, uint32_t &c_end) {
        if constexpr (GROUPED && OP == OP_DW) {
            const uint32_t per_piece = p.tiles_r * p.tiles_c, piece = item / per_piece;
            const uint4 e = ld_behind_wait(p.entries + piece);
            piece_group = e.x, piece_row = e.y, piece_end = e.z;
            tile = item - piece * per_piece;
            c_begin = 0;
            c_end = (piece_end - piece_row + KC - 1) / KC;
            next_item = item + item_stride;
        } else if (p.units) {
            tile = item / p.nchunks;
            c_begin = item - tile * p.nchunks;
            c_end = min(p.nchunks, c_begin + (cur_end - item));
            partial = true;
            next_item = item + (c_end - c_begin);
        } else {
            uint32_t split = 0;
            if (item < p.n_main) {
                tile = item;
                partial = false;
            } else {
                const uint32_t idx = item - p.n_main, q = idx / p.nsplit;
                tile = p.n_main + q;
                split = idx - q * p.nsplit;
                partial = p.nsplit > 1;
            }
            c_begin = partial ? split * p.chunks_per_split : 0u;
            c_end = partial ? min(p.nchunks, c_begin + p.chunks_per_split) : p.nchunks;
            next_item = item + item_stride;
        }
        uint32_t per_group = p.group_rows * p.tiles_c;
        uint32_t group = tile / per_group, within = tile - group * per_group;
        uint32_t first_r = group * p.group_rows;
        uint32_t gsz = min(tiles_r - first_r, p.group_rows);
        tr = first_r + within % gsz;
        tc = within / gsz;
        if constexpr (GROUPED && OP != OP_DW) {
            const uint4 e = ld_behind_wait(p.entries + tr);
            piece_group = e.x, piece_row = e.y, piece_end = e.z;
        }
    };
    // first row of a block in its matrix (DW: in the transposed weight)
    auto block_row = [&](uint32_t tr) { return GROUPED && OP != OP_DW ? piece_row : tr * ITEM_R; };
    // first hash-tile row of the block's weight
    auto first_tile = [&]() -> uint32_t {
        if constexpr (GROUPED) return piece_group * p.group_tiles;
        return 0u;
    };

    if (warp == 0) {
        // ===================== producer (both CTAs of a pair) =====================
        uint32_t it = 0;  // stages armed so far
        uint32_t slot = 0, phase = 1;   // (weight gradient) the ring's next slot, and the parity that says it is free
        uint32_t fenced_group = 0xffffffffu;   // (GROUPED DW) group whose maps this thread has acquired
        // transaction bytes of a stage are counted on the leader's barrier
        uint32_t full_base = bar_full;
        if (PAIR_LOADS) full_base = mapa_cluster(bar_full, 0);
        for (uint32_t item = cur_begin; item < cur_end && ok; item = next_item) {
            uint32_t tr, tc, c_begin, c_end;
            decode(item, tr, tc, c_begin, c_end);
            const uint32_t row0 = block_row(tr) + rank * TILE_R;   // first output row staged by this CTA (A); row block r adds r * PAIR_R
            const uint32_t col0 = tc * TILE_C + rank * B_COLS;     // first output column staged by this CTA (B)
            const CUtensorMap *ma = &mapA, *mb = &mapB;
            if constexpr (GROUPED && OP == OP_DW) {
                ma = p.maps + 2 * piece_group, mb = ma + 1;
                if (lane == 0 && piece_group != fenced_group) {   // the maps were written by a kernel, not by the host
                    tma_acquire_desc(ma);
                    tma_acquire_desc(mb);
                    fenced_group = piece_group;
                }
            }
            if constexpr (OP == OP_DW) {
                // nothing to hash: one thread, with the ring's position and the addresses counted up (a stage's four loads and what is
                // around them took it 800 clocks with both divided and multiplied out, longer than the stage's MMAs)
                if (lane == 0) {
                    int32_t d0 = (int32_t)(c_begin * KC + (GROUPED ? piece_row : 0u));
#pragma unroll 1
                    for (uint32_t left = c_end - c_begin; left; --left, d0 += KC) {
                        if (!mbar_wait_bounded(bar_empty + 8 * slot, phase, RZ_WAIT_SMEM_EMPTY, p.wait, 2000)) {
                            ok = false;
                            break;
                        }
                        const uint32_t full = full_base + 8 * slot, sa = smem_base + slot * STAGE_BYTES;
                        if (!PAIR_LOADS) mbar_arrive_expect_tx(bar_full + 8 * slot, LOAD_BYTES);
                        else if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * slot, LOAD_BYTES * CTAS);
#pragma unroll
                        for (int r = 0; r < RB; ++r) {
#pragma unroll
                            for (int a = 0; a < A_ATOMS; ++a) {
                                if (PAIR_LOADS) tma_load_2d_pair(sa + r * A_BLOCK_BYTES + a * ATOM, ma, full, (int32_t)(row0 + r * PAIR_R + a * EPR), d0);
                                else tma_load_2d(sa + r * A_BLOCK_BYTES + a * ATOM, ma, full, (int32_t)(row0 + r * PAIR_R + a * EPR), d0);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < B_ATOMS; ++j) {
                            if (PAIR_LOADS) tma_load_2d_pair(sa + A_BYTES + j * ATOM, mb, full, (int32_t)(col0 + j * EPR), d0);
                            else tma_load_2d(sa + A_BYTES + j * ATOM, mb, full, (int32_t)(col0 + j * EPR), d0);
                        }
                        ++it;
                        if (++slot == STAGES) slot = 0, phase ^= 1u;
                    }
                }
                __syncwarp();
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                continue;
            }
            for (uint32_t cb = c_begin; cb < c_end && ok; cb += BATCH) {
                const uint32_t nb = min((uint32_t)BATCH, c_end - cb);
                {
                    const uint32_t tps = (OP == OP_FWD) ? (uint32_t)B_ATOMS * p.kparts : (uint32_t)B_COLS / p.br;
                    for (uint32_t e = lane; e < nb * tps; e += 32) {
                        const uint32_t ci = e / tps, j = e - ci * tps;
                        uint32_t pk, pn, x_in, y_in;
                        if (OP == OP_FWD) {
                            // box j = (128-byte column block ja, part hh of the stage's contraction rows)
                            const uint32_t ja = j / p.kparts, hh = j - ja * p.kparts;
                            const uint32_t k0 = (cb + ci) * KC + hh * p.br, n = col0 + ja * EPR;
                            pk = k0 / (uint32_t)p.hash.BK;
                            y_in = k0 - pk * (uint32_t)p.hash.BK;
                            pk += first_tile();
                            pn = n / (uint32_t)p.hash.BN;
                            x_in = n - pn * (uint32_t)p.hash.BN;
                        } else {
                            const uint32_t n0 = (cb + ci) * KC, ko = col0 + j * p.br;
                            pn = n0 / (uint32_t)p.hash.BN;
                            x_in = n0 - pn * (uint32_t)p.hash.BN;
                            pk = ko / (uint32_t)p.hash.BK;
                            y_in = ko - pk * (uint32_t)p.hash.BK;
                            pk += first_tile();
                        }
                        const uint32_t off = (uint32_t)rz_tile_offset(p.hash, pk, pn);
                        const uint32_t sh = off & (NS - 1);
                        tab_x[ci * MAX_TPS + j] = off - sh + x_in;
                        tab_y[ci * MAX_TPS + j] = y_in;
                        tab_z[ci * MAX_TPS + j] = sh;
                    }
                    __syncwarp();
                }
                if (lane == 0) {
                    for (uint32_t ci = 0; ci < nb; ++ci) {
                        const uint32_t g = it + ci, s = g % STAGES, ph = (g / STAGES) & 1;
                        if (!mbar_wait_bounded(bar_empty + 8 * s, ph ^ 1, RZ_WAIT_SMEM_EMPTY, p.wait, 2000)) {
                            ok = false;
                            it += ci;
                            break;
                        }
                        const uint32_t full = full_base + 8 * s;
                        const uint32_t sa = smem_base + s * STAGE_BYTES, sb = sa + A_BYTES;
                        if (PAIR_LOADS) {
                            if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, LOAD_BYTES * CTAS);
                        } else {
                            mbar_arrive_expect_tx(bar_full + 8 * s, LOAD_BYTES);
                        }
                        const uint32_t d0 = (cb + ci) * KC;  // contraction start of this stage
#pragma unroll
                        for (int r = 0; r < RB; ++r) {
                            if (PAIR_LOADS)
                                tma_load_2d_pair(sa + r * A_BLOCK_BYTES, &mapA, full, (int32_t)d0, (int32_t)(row0 + r * PAIR_R));
                            else
                                tma_load_2d(sa, &mapA, full, (int32_t)d0, (int32_t)row0);
                        }
                        const uint32_t tps = (OP == OP_FWD) ? (uint32_t)B_ATOMS * p.kparts : (uint32_t)B_COLS / p.br;
                        const uint32_t box_bytes = p.br * 128u;   // (FWD: boxes of one column block are consecutive)
                        for (uint32_t j = 0; j < tps; ++j) {
                            const int32_t x = (int32_t)tab_x[ci * MAX_TPS + j], y = (int32_t)tab_y[ci * MAX_TPS + j],
                                          z = (int32_t)tab_z[ci * MAX_TPS + j];
                            if (PAIR_LOADS) tma_load_3d_pair(sb + j * box_bytes, &mapB, full, x, y, z);
                            else tma_load_3d(sb + j * box_bytes, &mapB, full, x, y, z);
                        }
                    }
                    if (ok) it += nb;
                }
                __syncwarp();
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                it = __shfl_sync(0xffffffffu, it, 0);
            }
        }
        if (!ok && lane == 0 && (rank == 0 || !PAIR_LOADS)) {
            // give the loads already issued time to land before the CTA retires
            const uint32_t lo = it > STAGES ? it - STAGES : 0;
            for (uint32_t g = lo; g < it; ++g) wait_cycles(bar_full + 8 * (g % STAGES), (g / STAGES) & 1, 4000000);
        }
    } else if (warp == 1) {
        // ===================== MMA issuer (leader CTA only) =====================
        // One thread issues everything, instruction after instruction: what does not change from stage to stage is kept out of the
        // loop (with descriptors built and ring positions divided per MMA, issuing a stage of four MMAs took 800 clocks, more than
        // the tensor core takes to run them).  A descriptor's low word holds the address in sixteenths, below 2^14: adding to it
        // cannot carry.
        constexpr uint32_t MN_KSTEP = (TF32 ? 8 : 16) * 128;   // contraction rows per MMA x 128-byte rows
        constexpr uint32_t A_KSTEP = OP == OP_DW ? MN_KSTEP : 32, B_KSTEP = OP == OP_DX ? 32 : MN_KSTEP;
        const uint64_t a0 = make_desc_sw128(smem_base, p.a_lbo, p.a_sbo, p.a_layout);
        const uint64_t b0 = make_desc_sw128(smem_base + A_BYTES, p.b_lbo, p.b_sbo, p.b_layout);
        const uint32_t a_lo = (uint32_t)a0, b_lo = (uint32_t)b0;
        const uint64_t a_hi = a0 >> 32 << 32, b_hi = b0 >> 32 << 32;
        const uint32_t bar_ready = SPLIT ? bar_split : bar_full;
        uint32_t n_items = 0, slot = 0, phase = 0;
        for (uint32_t item = cur_begin; item < cur_end && ok && rank == 0; item = next_item, ++n_items) {
            uint32_t tr, tc, c_begin, c_end;
            decode(item, tr, tc, c_begin, c_end);
            const uint32_t buf = n_items % NBUF, tph = (n_items / NBUF) & 1;
            if (lane == 0) {
                if (!mbar_wait_bounded(bar_tempty + 8 * buf, tph ^ 1, RZ_WAIT_TMEM_EMPTY, p.wait, 2000)) ok = false;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + buf * RB * TILE_C;
                // (CHAINS > 1) stages per main accumulator, and the one in use
                const uint32_t chain_len = (c_end - c_begin + CHAINS - 1) / CHAINS;
                uint32_t chain_left = chain_len, chain_col = 0, acc = 0, corr_acc = 0;
#pragma unroll 1
                for (uint32_t left = c_end - c_begin; left && ok; --left) {
                    if (!mbar_wait_bounded(bar_ready + 8 * slot, phase, RZ_WAIT_SMEM_FULL, p.wait)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t al = a_lo + slot * (STAGE_BYTES / 16), bl = b_lo + slot * (STAGE_BYTES / 16);
                    if (CHAINS > 1) {
                        if (chain_left == 0) chain_left = chain_len, chain_col += NC, acc = 0;
                        --chain_left;
                    }
#pragma unroll
                    for (int kk = 0; kk < MMAS; ++kk) {
                        const uint64_t bd = b_hi | (bl + kk * (B_KSTEP / 16));
#pragma unroll
                        for (int r = 0; r < RB; ++r) {
                            const uint64_t ad = a_hi | (al + (r * A_BLOCK_BYTES + kk * A_KSTEP) / 16);
                            if (CTAS == 2) tc_mma_pair<TF32>(d_tmem + chain_col + r * TILE_C, ad, bd, p.idesc, acc);
                            else tc_mma<TF32>(d_tmem + chain_col, ad, bd, p.idesc, acc);
                            if (SPLIT) {
                                // + hi(A) * lo(B) + lo(A) * hi(B)
                                const uint64_t ad_lo = a_hi | (al + (LOAD_BYTES + kk * A_KSTEP) / 16);
                                const uint64_t bd_lo = b_hi | (bl + (LOAD_BYTES + kk * B_KSTEP) / 16);
                                if (CTAS == 2) {
                                    tc_mma_pair<TF32>(d_tmem + CORR_COL, ad, bd_lo, p.idesc, corr_acc);
                                    tc_mma_pair<TF32>(d_tmem + CORR_COL, ad_lo, bd, p.idesc, 1u);
                                } else {
                                    tc_mma<TF32>(d_tmem + CORR_COL, ad, bd_lo, p.idesc, corr_acc);
                                    tc_mma<TF32>(d_tmem + CORR_COL, ad_lo, bd, p.idesc, 1u);
                                }
                            }
                        }
                        acc = corr_acc = 1;
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
            wait_cycles(bar_drain, 0, 20000000);
        }
    } else if (warp < 2 + EPI_WARPS) {
        // ===================== epilogue (both CTAs; each drains its own 128 rows) =====================
        const uint32_t q = warp & 3;          // TMEM lane quarter this warp may read
        const uint32_t rblk = ((warp - 2) >> 2) % RB;   // which accumulator (row block) of the item this warp drains
        const uint32_t cgrp = ((warp - 2) >> 2) / RB;   // EW > 1: this warp takes the 32-column chunks cgrp, cgrp + EW, ...
        uint32_t own = 0;                                     // mask of those chunks
#pragma unroll
        for (int c2 = 0; c2 < TILE_C / 32; ++c2)
            if (c2 % EW == (int)cgrp) own |= 1u << c2;
        float *scratch = epi_scratch + (warp - 2) * 1024;   // (FWD / DX staging tile; unused by the weight gradient)
        uint32_t tempty_base = bar_tempty;
        if (CTAS == 2) tempty_base = mapa_cluster(bar_tempty, 0);
        uint32_t n_items = 0;
        for (uint32_t item = cur_begin; item < cur_end && ok; item = next_item, ++n_items) {
            uint32_t tr, tc, c_begin, c_end;
            decode(item, tr, tc, c_begin, c_end);
            const uint32_t buf = n_items % NBUF, tph = (n_items / NBUF) & 1;
            const uint32_t rbase = block_row(tr) + rblk * PAIR_R + rank * TILE_R + q * 32;   // first row of this warp
            const uint32_t row_end = GROUPED && OP != OP_DW ? piece_end : p.rows;            // rows behind it are not stored
            // main accumulators in use besides the first
            const uint32_t more_chains = CHAINS > 1 ? (c_end - c_begin - 1) / ((c_end - c_begin + CHAINS - 1) / CHAINS) : 0u;
            // Weight gradient.  The block is computed TRANSPOSED (A = dY, B = X): an accumulator row (TMEM lane) is an
            // output column n of the virtual weight and an accumulator column is a weight row k.  A thread thus holds,
            // for its n, 32 consecutive k of a chunk, and the 32 lanes of a warp hold 32 consecutive n - which are 32
            // consecutive words of one slice row.  Every reduction instruction is therefore one coalesced 128-byte
            // segment straight out of the registers that tcgen05.ld filled: no transpose through shared memory.
            // A chunk (32 k) lies inside one hash tile (tiles are multiples of 32 both ways).  Chunks of different
            // tiles of one tile column that land on exactly the same addresses (colliding offsets, same rows inside the
            // tile) are summed in registers first, so such a collision costs one set of reductions instead of one
            // per tile.  Lane c (< chunks per block) holds the destination of chunk c.
            uint32_t key_off = 0, key_rel = 0, eqmask = 0, n_rel = 0;
            if (OP == OP_DW) {
                const uint32_t pn = rbase / (uint32_t)p.hash.BN;
                n_rel = rbase - pn * (uint32_t)p.hash.BN;
                if (lane < TILE_C / 32) {
                    const uint32_t kcol = tc * TILE_C + lane * 32, pk = kcol / (uint32_t)p.hash.BK;
                    key_rel = kcol - pk * (uint32_t)p.hash.BK;
                    if constexpr (GROUPED) key_off = rz_tile_offset32(p.hash, p.hash32, first_tile() + pk, pn);
                    else key_off = (uint32_t)rz_tile_offset(p.hash, pk, pn);
                }
#pragma unroll
                for (int c2 = 0; c2 < TILE_C / 32; ++c2) {
                    const uint32_t o2 = __shfl_sync(0xffffffffu, key_off, c2), r2 = __shfl_sync(0xffffffffu, key_rel, c2);
                    if (o2 == key_off && r2 == key_rel) eqmask |= 1u << c2;
                }
            }
            // (destinations first, then the wait: the hash and the comparisons overlap the block's MMAs)
            // one lane per warp polls (sleeping in the barrier unit between polls); the others wait for it
            bool mine = true;
            if (lane == 0) mine = mbar_wait_bounded(bar_tfull + 8 * buf, tph, RZ_WAIT_TMEM_FULL, p.wait, 20000);
            ok = __shfl_sync(0xffffffffu, (int)mine, 0) != 0;
            if (!ok) break;
            tc_fence_after();
            if (OP == OP_DW && EW > 1 && RB == 1) {
                // Scatter-bound weight gradient.  The warp pulls all its chunks out of TMEM at once and hands the
                // accumulator back before it starts on the reductions, so the next blocks' MMAs never wait for the
                // scatter; loads from TMEM then come in one short burst per block instead of trickling in between
                // the MMAs for the whole epilogue.
                constexpr int NCH = (TILE_C / 32 + EW - 1) / EW;   // chunks per warp
                uint32_t vv[NCH][32];
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    const int c = (int)cgrp + j * EW;
                    if (c < TILE_C / 32) tmem_ld_32x32(tmem_base + ((q * 32u) << 16) + buf * TILE_C + c * 32, vv[j]);
                }
#pragma unroll
                for (int j = 0; j < NCH; ++j) tmem_ld_wait_regs(vv[j]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {   // relaxed: a release would wait for the previous block's reductions still in flight
                    if (CTAS == 2) mbar_arrive_cluster_relaxed(tempty_base + 8 * buf);
                    else mbar_arrive_relaxed(bar_tempty + 8 * buf);
                }
                if (rbase >= p.N) continue;
                const bool lane_ok = rbase + lane < p.N;
                const uint32_t bn = (uint32_t)p.hash.BN;
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    const int c = (int)cgrp + j * EW;
                    if (c >= TILE_C / 32) break;
                    const uint32_t same = __shfl_sync(0xffffffffu, eqmask, c) & own;
                    if (same & ((1u << c) - 1u)) continue;   // summed into an earlier chunk of this warp
                    const uint32_t kcol = tc * TILE_C + c * 32;
                    uint32_t nk = kcol < p.K ? min(32u, p.K - kcol) : 0u;   // weight rows of this chunk that exist
                    float acc[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) acc[e] = __uint_as_float(vv[j][e]);
#pragma unroll
                    for (int j2 = j + 1; j2 < NCH; ++j2) {
                        const int c2 = (int)cgrp + j2 * EW;
                        if (c2 < TILE_C / 32 && ((same >> c2) & 1u)) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) acc[e] += __uint_as_float(vv[j2][e]);
                            const uint32_t kcol2 = tc * TILE_C + c2 * 32;
                            nk = max(nk, kcol2 < p.K ? min(32u, p.K - kcol2) : 0u);
                        }
                    }
                    const uint32_t off = __shfl_sync(0xffffffffu, key_off, c), rel = __shfl_sync(0xffffffffu, key_rel, c);
                    float *dst = p.dH + off + (uint64_t)rel * bn + n_rel + lane;
                    if (lane_ok) {
                        if (nk == 32) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) atomicAdd(dst + (size_t)e * bn, acc[e] * p.alpha);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if ((uint32_t)e < nk) atomicAdd(dst + (size_t)e * bn, acc[e] * p.alpha);
                        }
                    }
                }
                continue;
            }
#pragma nv_diag_suppress 128   // (the one-row-block EW > 1 instantiations never reach the generic chunk loop)
            // FWD / DX: the next chunk streams out of TMEM while this one is converted and stored
            constexpr bool PREFETCH = (OP != OP_DW) && !SPLIT;
            const uint32_t acc_addr = tmem_base + ((q * 32u) << 16) + (buf * RB + rblk) * TILE_C;
            uint32_t vnext[32];
            if (PREFETCH) tmem_ld_32x32(acc_addr + cgrp * 32, vnext);
#pragma unroll 1
            for (int c = (int)cgrp; c < TILE_C / 32; c += EW) {
                uint32_t v[32];
                uint32_t same = 0;
                if (OP == OP_DW) {
                    same = __shfl_sync(0xffffffffu, eqmask, c) & own;   // merge only among this warp's chunks
                    if (same & ((1u << c) - 1u)) continue;   // already merged into an earlier chunk
                }
                if (PREFETCH) {
                    tmem_ld_wait_regs(vnext);
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = vnext[j];
                    if (c + EW < TILE_C / 32) tmem_ld_32x32(acc_addr + (c + EW) * 32, vnext);
                } else {
                    tmem_ld_32x32(acc_addr + c * 32, v);
                    tmem_ld_wait();
                }
                if (SPLIT) {   // main + correction accumulators, added with round-to-nearest
                    uint32_t w[32];
                    tmem_ld_32x32(tmem_base + ((q * 32u) << 16) + CORR_COL + c * 32, w);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(w[j]));
                    if (CHAINS > 1) {
#pragma unroll 1
                        for (uint32_t k = 1; k <= more_chains; ++k) {
                            tmem_ld_32x32(tmem_base + ((q * 32u) << 16) + k * NC + c * 32, w);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(w[j]));
                        }
                    }
                }
                const uint32_t col = tc * TILE_C + c * 32;
                // a bulk store clips at the matrix edge only: rows of a group's ragged end are stored one by one
                const bool bulk = p.tma_store && (!GROUPED || rbase + 32 <= row_end);
                if (OP != OP_DW && p.tma_store && (partial || TF32 || !(c & 1))) {
                    // the staging tile is about to be rewritten: the bulk store issued from it must have read it
                    if (lane == 0) bulk_wait_group_read0();
                    __syncwarp();
                }
                if (OP == OP_DW) {
                    float acc[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[j] = __uint_as_float(v[j]);
                    uint32_t nk = col < p.K ? min(32u, p.K - col) : 0u;   // weight rows of this chunk that exist
                    uint32_t rest = same & ~((2u << c) - 1u);   // later chunks with the same destination
                    while (rest) {
                        const int c2 = __ffs(rest) - 1;
                        rest &= rest - 1;
                        tmem_ld_32x32(tmem_base + ((q * 32u) << 16) + (buf * RB + rblk) * TILE_C + c2 * 32, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) acc[j] += __uint_as_float(v[j]);
                        if (SPLIT) {
                            tmem_ld_32x32(tmem_base + ((q * 32u) << 16) + CORR_COL + c2 * 32, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) acc[j] += __uint_as_float(v[j]);
                            if (CHAINS > 1) {
#pragma unroll 1
                                for (uint32_t k = 1; k <= more_chains; ++k) {
                                    tmem_ld_32x32(tmem_base + ((q * 32u) << 16) + k * NC + c2 * 32, v);
                                    tmem_ld_wait();
#pragma unroll
                                    for (int j = 0; j < 32; ++j) acc[j] += __uint_as_float(v[j]);
                                }
                            }
                        }
                        const uint32_t col2 = tc * TILE_C + c2 * 32;
                        nk = max(nk, col2 < p.K ? min(32u, p.K - col2) : 0u);
                    }
                    const uint32_t off = __shfl_sync(0xffffffffu, key_off, c), rel = __shfl_sync(0xffffffffu, key_rel, c);
                    if (rbase + lane < p.N) {
                        // lane = weight column n, register e = weight row k: one coalesced 128-byte reduction per k
                        float *dst = p.dH + off + (uint64_t)rel * (uint32_t)p.hash.BN + n_rel + lane;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if ((uint32_t)e < nk) atomicAdd(dst + (size_t)e * (uint32_t)p.hash.BN, acc[e] * p.alpha);
                    }
                } else if (partial) {
                    // split contraction: add the raw fp32 partial sums into this block's ITEM_R x NC workspace tile (a
                    // finalize kernel scales, adds the bias and converts); staged like the store path so every
                    // reduction is a full row segment
                    uint8_t *stage = reinterpret_cast<uint8_t *>(scratch);
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        uint4 u;
                        u.x = v[4 * g + 0];
                        u.y = v[4 * g + 1];
                        u.z = v[4 * g + 2];
                        u.w = v[4 * g + 3];
                        *reinterpret_cast<uint4 *>(stage + lane * 128 + ((g ^ (lane & 7)) * 16)) = u;
                    }
                    __syncwarp();
                    const uint32_t cc = lane & 7, ccol = col + cc * 4;
                    float *wtile = p.ws + (size_t)(tile - p.n_main) * (ITEM_R * NC) +
                                   (size_t)(rbase - tr * ITEM_R) * NC + (c * 32 + cc * 4);
#pragma unroll
                    for (int it4 = 0; it4 < 8; ++it4) {
                        const uint32_t rr = it4 * 4 + (lane >> 3);
                        const uint4 u = *reinterpret_cast<const uint4 *>(stage + rr * 128 + ((cc ^ (rr & 7)) * 16));
                        const uint32_t grow = rbase + rr;
                        if (grow < p.rows && ccol < p.cols)
                            asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(wtile + (size_t)rr * NC),
                                         "f"(__uint_as_float(u.x)), "f"(__uint_as_float(u.y)), "f"(__uint_as_float(u.z)),
                                         "f"(__uint_as_float(u.w))
                                         : "memory");
                    }
                    __syncwarp();
                } else {
                    // scale (+ bias, ReLU), convert, and stage this lane's row segment in shared memory in
                    // 16-byte chunks (chunk index XOR row keeps both phases bank-conflict free); once a
                    // 128-byte row segment is complete the warp writes it out 4 full rows per instruction.
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]) * p.alpha;
                    if (OP == OP_FWD) {
                        if (p.bias) {
                            const float *bias = p.bias + (GROUPED ? (size_t)piece_group * p.cols : 0);
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (col + j < p.cols) f[j] += __ldg(bias + col + j);
                        }
                        if (p.relu) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) f[j] = GROUPED ? (f[j] < 0.f ? 0.f : f[j]) : fmaxf(f[j], 0.f);   // (grouped: a NaN stays one)
                        }
                    }
                    uint8_t *stage = reinterpret_cast<uint8_t *>(scratch);
                    constexpr int CHUNKS_PER_LD = TF32 ? 8 : 4;          // 16-byte chunks produced per 32 columns
                    const int cbase = TF32 ? 0 : (c & 1) * 4;             // bf16: two loads fill one 128-byte row
#pragma unroll
                    for (int g = 0; g < CHUNKS_PER_LD; ++g) {
                        uint4 u;
                        if (TF32) {
                            u.x = __float_as_uint(f[4 * g + 0]);
                            u.y = __float_as_uint(f[4 * g + 1]);
                            u.z = __float_as_uint(f[4 * g + 2]);
                            u.w = __float_as_uint(f[4 * g + 3]);
                        } else {
                            __nv_bfloat162 h0 = __floats2bfloat162_rn(f[8 * g + 0], f[8 * g + 1]);
                            __nv_bfloat162 h1 = __floats2bfloat162_rn(f[8 * g + 2], f[8 * g + 3]);
                            __nv_bfloat162 h2 = __floats2bfloat162_rn(f[8 * g + 4], f[8 * g + 5]);
                            __nv_bfloat162 h3 = __floats2bfloat162_rn(f[8 * g + 6], f[8 * g + 7]);
                            u.x = *reinterpret_cast<uint32_t *>(&h0);
                            u.y = *reinterpret_cast<uint32_t *>(&h1);
                            u.z = *reinterpret_cast<uint32_t *>(&h2);
                            u.w = *reinterpret_cast<uint32_t *>(&h3);
                        }
                        *reinterpret_cast<uint4 *>(stage + lane * 128 + (((cbase + g) ^ (lane & 7)) * 16)) = u;
                    }
                    if ((TF32 || (c & 1)) && bulk) {
                        // one bulk tensor store per staged 32-row x 128-byte tile (the tile is in the 128-byte-swizzle
                        // layout the store expects; rows and columns past the matrix edge are clipped by the unit)
                        const uint32_t col_seg = TF32 ? col : col - 32;
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0 && rbase < row_end && col_seg < p.cols) {
                            tma_store_2d(&mapC, smem_u32(stage), (int32_t)col_seg, (int32_t)rbase);
                            bulk_commit_group();
                        }
                    } else if (TF32 || (c & 1)) {
                        __syncwarp();
                        constexpr int EPC = TF32 ? 4 : 8;                 // elements per 16-byte chunk
                        const uint32_t col_seg = TF32 ? col : col - 32;   // first column of the staged 128-byte segment
                        const uint32_t cc = lane & 7, ccol = col_seg + cc * EPC;
#pragma unroll
                        for (int it4 = 0; it4 < 8; ++it4) {
                            const uint32_t rr = it4 * 4 + (lane >> 3);
                            const uint4 u = *reinterpret_cast<const uint4 *>(stage + rr * 128 + ((cc ^ (rr & 7)) * 16));
                            const uint32_t grow = rbase + rr;
                            if (grow < row_end && ccol < p.cols)
                                *reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(p.out) +
                                                           ((size_t)grow * p.cols + ccol) * (TF32 ? 4 : 2)) = u;
                        }
                        __syncwarp();
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CTAS == 2) mbar_arrive_cluster(tempty_base + 8 * buf);
                else mbar_arrive(bar_tempty + 8 * buf);
            }
        }
        if (OP != OP_DW && lane == 0) bulk_wait_group0();   // bulk stores still in flight read this CTA's shared memory
    }

    else if (SPLIT) {
        // ===================== splitter (SPLIT only): hi/lo parts of every staged tile =====================
        const uint32_t tid = threadIdx.x - (2 + EPI_WARPS) * 32;   // 0..127
        uint32_t split_base = bar_split;
        if (CTAS == 2) split_base = mapa_cluster(bar_split, 0);
        uint32_t it = 0;
        for (uint32_t item = cur_begin; item < cur_end && ok; item = next_item) {
            uint32_t tr, tc, c_begin, c_end;
            decode(item, tr, tc, c_begin, c_end);
            for (uint32_t c = c_begin; c < c_end && ok; ++c, ++it) {
                const uint32_t s = it % STAGES, ph = (it / STAGES) & 1;
                bool mine = mbar_wait_bounded(bar_full + 8 * s, ph, RZ_WAIT_SMEM_FULL, p.wait, 1000);
                ok = __all_sync(0xffffffffu, mine);
                if (!ok) break;
                uint4 *hi = reinterpret_cast<uint4 *>(smem_gen + s * STAGE_BYTES);
                uint4 *lo = reinterpret_cast<uint4 *>(smem_gen + s * STAGE_BYTES + LOAD_BYTES);
#pragma unroll 4
                for (uint32_t v = tid; v < LOAD_BYTES / 16; v += 128) {
                    uint4 x = hi[v], h, l;
                    h.x = x.x & 0xFFFFE000u;
                    h.y = x.y & 0xFFFFE000u;
                    h.z = x.z & 0xFFFFE000u;
                    h.w = x.w & 0xFFFFE000u;
                    l.x = __float_as_uint(__uint_as_float(x.x) - __uint_as_float(h.x));
                    l.y = __float_as_uint(__uint_as_float(x.y) - __uint_as_float(h.y));
                    l.z = __float_as_uint(__uint_as_float(x.z) - __uint_as_float(h.z));
                    l.w = __float_as_uint(__uint_as_float(x.w) - __uint_as_float(h.w));
                    hi[v] = h;
                    lo[v] = l;
                }
                fence_proxy_async();   // the tensor core reads these tiles through the async proxy
                __syncwarp();
                if (lane == 0) {
                    if (CTAS == 2) mbar_arrive_cluster(split_base + 8 * s);
                    else mbar_arrive(bar_split + 8 * s);
                }
            }
        }
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
