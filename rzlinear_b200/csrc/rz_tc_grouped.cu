// Tensor-core launches of products grouped by row: bf16 products run rz_tc_rows.cuh, their weight gradient and all fp32 operations
// the GROUPED instantiations of rz_tc_kernel.cuh.  The number of blocks is known on the device only, so every launch fills the machine (one CTA or CTA pair per
// SM or pair of SMs) and the kernel deals the planned pieces' blocks out round robin.
#include <atomic>
#include <cstring>

#include "rz_tc_host.h"
#include "rz_tc_kernel.cuh"
#include "rz_tc_rows.cuh"

using namespace rztc;

namespace {

int usable_sms(const rz_problem *pb)
{
    const int n = num_sms() - (pb->sm_reserve > 0 ? pb->sm_reserve : 0);
    return n < 2 ? 2 : n;
}

// Per kernel variant and device, once: the shared-memory opt-in, and how many blocks (pairs) can be resident.
template <auto Kernel, int CTAS>
int resident(const rz_problem *pb, int threads, int smem, int *slots)
{
    static std::atomic<int> ready[64];   // 0 = not set up, else resident blocks / pairs + 1
    int dev = 0;
    int st = rz_record_cuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (st) return st;
    const bool cacheable = dev >= 0 && dev < 64;
    const int known = cacheable ? ready[dev].load(std::memory_order_acquire) : 0;
    *slots = num_sms() / CTAS;
    if (known) {
        *slots = known - 1;
    } else {
        st = rz_record_cuda(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "set max dynamic shared memory");
        if (st) return st;
        if (CTAS == 2) {
            cudaLaunchConfig_t cfg;
            cudaLaunchAttribute attr[1];
            memset(&cfg, 0, sizeof(cfg));
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
            cfg.blockDim = dim3(threads, 1, 1);
            cfg.dynamicSmemBytes = smem;
            cfg.gridDim = dim3(2 * (unsigned)*slots, 1, 1);
            cfg.attrs = attr, cfg.numAttrs = 1;
            int clusters = 0;
            if (cudaOccupancyMaxActiveClusters(&clusters, Kernel, &cfg) == cudaSuccess && clusters > 0 && clusters < *slots) *slots = clusters;
            (void)cudaGetLastError();
        }
        if (cacheable) ready[dev].store(*slots + 1, std::memory_order_release);
    }
    if (pb->sm_reserve > 0) {   // leave SMs idle for whatever the caller runs beside this kernel
        *slots -= (pb->sm_reserve + CTAS - 1) / CTAS;
        if (*slots < 1) *slots = 1;
    }
    return RZ_OK;
}

// One CTA (pair) per slot, or per block where `most` says that there are fewer.
template <int CTAS, typename Kernel, typename... Args>
int launch_persistent(Kernel kernel, int threads, int smem, int slots, uint64_t most, cudaStream_t stream, const Args &...args)
{
    if (most >= 0x80000000ull) return RZ_ERR_SHAPE;   // block numbers are 32-bit words
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    memset(&cfg, 0, sizeof(cfg));
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CTAS, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    // The kernel sets itself up (barriers, TMEM) beside the one before it, the plan's, and waits for that before it reads anything.
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.gridDim = dim3((unsigned)(most < (uint64_t)slots ? most : (uint64_t)slots) * CTAS, 1, 1);
    cfg.attrs = attr, cfg.numAttrs = CTAS == 2 ? 2 : 1;
    const int st = rz_record_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), "grouped tcgen05 kernel launch");
    rz_count_launch(1);
    if (st) return st;
    return rz_record_cuda(cudaGetLastError(), "grouped tcgen05 kernel launch");
}

// ---- bf16 products (rz_tc_rows.cuh) -----------------------------------------------------------------------------------------

// weight rows per box: whole boxes per hash tile
uint32_t rows_box_log2(const rz_problem *pb, int op)
{
    if (pb->BK < 64) return 5;   // (BK is 32, 64 or a multiple of 64)
    return op == RZ_OP_BACKWARD_INPUT && pb->BK % 128 == 0 ? 7 : 6;
}

int log2_or_none(int32_t v)
{
    int l = 0;
    while (v >> l > 1) ++l;
    return (1 << l) == v ? l : -1;
}

template <int OP, int CTAS, int RB, int NMAX>
int launch_rows(const RzLaunchCtx &c, const RzGroupPieces &pieces, const void *rows, const void *copies, const float *bias, void *out)
{
    const rz_problem *pb = c.pb;
    constexpr int op = OP == ROWS_FWD ? RZ_OP_FORWARD : RZ_OP_BACKWARD_INPUT;
    const int64_t depth = OP == ROWS_FWD ? pb->K : pb->N, cols = OP == ROWS_FWD ? pb->N : pb->K;
    TcRowsParams p;
    memset(&p, 0, sizeof(p));
    p.hash = c.hash;
    p.header = pieces.header, p.entries = pieces.entries, p.group_tiles = pieces.group_tiles;
    p.cols = (uint32_t)cols;
    p.tiles_c = (uint32_t)((cols + 128 * CTAS * RB - 1) / (128 * CTAS * RB));
    p.nchunks = (uint32_t)((depth + 63) / 64);
    // (blocks and stages at the edges hash tiles a little beyond the last group's weight)
    p.hash32 = rz_hash32(c.hash, (uint64_t)pieces.groups * pieces.group_tiles + 512 / 32, (uint64_t)(pb->N + pb->BN - 1) / pb->BN + 512 / 64);
    p.bk_shift = log2_or_none(pb->BK), p.bn_shift = log2_or_none(pb->BN);
    p.br_log2 = rows_box_log2(pb, op);
    p.group_pieces = 8;
    p.alpha = pb->alpha;
    p.relu = OP == ROWS_FWD && (pb->flags & RZ_FLAG_RELU) ? 1 : 0;
    p.bias = bias;
    p.out = static_cast<__nv_bfloat16 *>(out);
    int st = rz_wait_context(&p.wait, 2000000000ll);   // also refuses to launch behind a kernel whose wait gave up
    if (st) return st;
    CUtensorMap mapW, mapR16, mapR64, mapRAll, mapC;
    st = map_shadow(&mapW, pb, OP == ROWS_FWD, copies, 1u << p.br_log2, false);
    if (st) return st;
    st = map_matrix(&mapR16, false, 0, rows, pb->M, depth, 64, 16, false);
    if (st) return st;
    st = map_matrix(&mapR64, false, 0, rows, pb->M, depth, 64, 64, false);
    if (st) return st;
    st = map_matrix(&mapRAll, false, 0, rows, pb->M, depth, 64, NMAX / CTAS, false);
    if (st) return st;
    st = map_matrix(&mapC, false, PLAIN_LAYOUT, out, pb->M, cols, 32, 32, false);
    if (st) return st;
    constexpr int SMEM = rows_smem_total(CTAS, RB, NMAX), THREADS = rows_threads(RB);
    static_assert(SMEM <= ROWS_SMEM_LIMIT, "shared memory budget");
    int slots = 0;
    st = resident<rz_tc_rows_kernel<OP, CTAS, RB, NMAX>, CTAS>(pb, THREADS, SMEM, &slots);
    if (st) return st;
    return launch_persistent<CTAS>(rz_tc_rows_kernel<OP, CTAS, RB, NMAX>, THREADS, SMEM, slots, (uint64_t)pieces.most * p.tiles_c, c.stream, mapW,
                                   mapR16, mapR64, mapRAll, mapC, p);
}

template <int OP>
int launch_rows_any(const RzLaunchCtx &c, const RzTcGroupPlan &plan, const RzGroupPieces &pieces, const void *rows, const void *copies,
                    const float *bias, void *out)
{
    if (plan.rb == 2 && plan.nc == 256) return launch_rows<OP, 2, 2, 256>(c, pieces, rows, copies, bias, out);
    if (plan.rb == 2) return launch_rows<OP, 2, 2, 128>(c, pieces, rows, copies, bias, out);
    if (plan.ctas == 2) return launch_rows<OP, 2, 1, 256>(c, pieces, rows, copies, bias, out);
    if (plan.nc == 256) return launch_rows<OP, 1, 1, 256>(c, pieces, rows, copies, bias, out);
    return launch_rows<OP, 1, 1, 64>(c, pieces, rows, copies, bias, out);
}

// Block shape of a bf16 product by an estimate of its time: waves of blocks over the SMs, times a block's stages at what a stage of
// the shape takes (clocks, `fixed` + `per_row` * rows of the block: fits to the cases measured in rz_tc_rows.cuh), plus what a block
// costs besides.  The host knows the rows and the groups but not how the rows are spread: it reckons with groups of the mean size
// that end half a piece late.
RzTcGroupPlan rows_plan(const rz_problem *pb, int groups, int op)
{
    static const struct {
        int ctas, rb, nmax;
        double fixed, per_row;
    } shapes[] = {{2, 2, 256, 1140.0, 2.4}, {2, 1, 256, 650.0, 1.0}, {1, 1, 256, 700.0, 1.2}, {2, 2, 128, 1140.0, 2.4}, {1, 1, 64, 700.0, 1.2}};
    const double used = (double)(pb->M < groups ? pb->M : groups), mean = (double)pb->M / used;
    const int64_t cols = op == RZ_OP_FORWARD ? pb->N : pb->K;
    const double stages = (double)(((op == RZ_OP_FORWARD ? pb->K : pb->N) + 63) / 64);
    const int sms = usable_sms(pb), forced = forced_shape();
    RzTcGroupPlan best = {};
    double best_time = -1.0;
    for (int i = 0; i < 5; ++i) {
        const auto &s = shapes[i];
        double pieces = mean / s.nmax + 0.5;
        if (pieces < 1.0) pieces = 1.0;
        const double items = used * pieces * (double)((cols + 128 * s.ctas * s.rb - 1) / (128 * s.ctas * s.rb));
        double waves = items * s.ctas / sms;
        waves = waves < 1.0 ? 1.0 : waves + 0.5;               // half a wave is lost at the end
        // (accumulators that fill TMEM: the epilogue does not overlap the next block)
        const double besides = s.rb * s.nmax > 256 ? 10000.0 : 4000.0;
        const double time = waves * (stages * (s.fixed + s.per_row * mean / pieces) + besides);
        if (best_time < 0.0 || time < best_time || i == forced) {
            best_time = i == forced ? 0.0 : time;
            best.ctas = s.ctas, best.rb = s.rb, best.nc = s.nmax, best.step = (uint32_t)s.nmax, best.even = true;
        }
    }
    return best;
}

// ---- GROUPED instantiations of rz_tc_kernel.cuh -------------------------------------------------------------------------------

template <int OP, bool TF32, int CTAS, int RB, int SPLIT, int NC, int EW = 1>
int launch(const RzLaunchCtx &c, const CUtensorMap &mapA, const CUtensorMap &mapB, const CUtensorMap &mapC, TcGroupParams &p,
           const RzGroupPieces &pieces)
{
    const rz_problem *pb = c.pb;
    constexpr int ES = TF32 ? 4 : 2, KC = 128 / ES, PAIR_R = TILE_R * CTAS, ITEM_R = PAIR_R * RB;
    constexpr int SMEM_TOTAL = smem_total(OP, CTAS, RB, SPLIT, NC, EW);
    static_assert(SMEM_TOTAL <= SMEM_LIMIT, "shared memory budget");
    p.hash = c.hash;
    p.M = (uint32_t)pb->M, p.K = (uint32_t)pb->K, p.N = (uint32_t)pb->N;
    p.rows = OP == OP_DW ? p.N : p.M;   // (the weight gradient is computed transposed: N x K)
    p.cols = OP == OP_FWD ? p.N : p.K;
    p.tiles_r = OP == OP_DW ? (p.rows + ITEM_R - 1) / ITEM_R : 0;   // FWD, DX: the planned pieces
    p.tiles_c = (p.cols + NC - 1) / NC;
    p.nchunks = ((OP == OP_FWD ? p.K : p.N) + KC - 1) / KC;         // DW: a piece's rows
    const uint32_t stage = (uint32_t)KC, bk = (uint32_t)pb->BK, bcols = (uint32_t)(NC / CTAS);
    p.br = OP == OP_FWD ? (bk < stage ? bk : stage) : (bk < bcols ? bk : bcols);
    p.kparts = stage / (bk < stage ? bk : stage);
    p.group_rows = GROUP_ROWS / RB;
    p.nsplit = 1, p.chunks_per_split = p.nchunks;
    p.n_main = 0xffffffffu;   // every block runs its whole contraction
    p.total_items = 0, p.units = 0;
    p.alpha = pb->alpha;
    p.relu = (pb->flags & RZ_FLAG_RELU) ? 1 : 0;
    p.tma_store = 1;
    p.header = pieces.header, p.entries = pieces.entries, p.group_tiles = pieces.group_tiles;
    // (blocks at the edges hash tiles a little beyond the last group's weight)
    p.hash32 = rz_hash32(c.hash, (uint64_t)pieces.groups * pieces.group_tiles + 512 / 32, (uint64_t)(pb->N + pb->BN - 1) / pb->BN + 512 / 32);
    int st = rz_wait_context(&p.wait, 2000000000ll);   // also refuses to launch behind a kernel whose wait gave up
    if (st) return st;

    // shared-memory descriptors (bytes), as in the ungrouped launches
    const uint32_t atom = KC * 128, mn_sbo = TF32 ? 512 : 1024, mn_layout = TF32 ? 1 : 2;
    p.a_layout = p.b_layout = 2;
    p.a_lbo = p.b_lbo = 16, p.a_sbo = p.b_sbo = 1024;   // K-major
    if (OP != OP_DX) p.b_lbo = atom, p.b_sbo = mn_sbo, p.b_layout = mn_layout;
    if (OP == OP_DW) p.a_lbo = atom, p.a_sbo = mn_sbo, p.a_layout = mn_layout;
    const uint32_t a_major = OP == OP_DW ? 1u : 0u, b_major = OP == OP_DX ? 0u : 1u, fmt = TF32 ? 2u : 1u;
    p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (a_major << 15) | (b_major << 16) | ((uint32_t)(NC >> 3) << 17) |
              ((uint32_t)(PAIR_R >> 4) << 24);

    constexpr int THREADS = num_threads(RB, SPLIT, EW);
    int slots = 0;
    st = resident<rz_tc_kernel<OP, TF32, CTAS, RB, SPLIT, NC, EW, 1>, CTAS>(pb, THREADS, SMEM_TOTAL, &slots);
    if (st) return st;
    const uint64_t most = (uint64_t)pieces.most * p.tiles_c * (OP == OP_DW ? p.tiles_r : 1);
    return launch_persistent<CTAS>(rz_tc_kernel<OP, TF32, CTAS, RB, SPLIT, NC, EW, 1>, THREADS, SMEM_TOTAL, slots, most, c.stream, mapA, mapB, mapC,
                                   p);
}

template <int OP>
int launch_any(const RzLaunchCtx &c, const RzTcGroupPlan &plan, const CUtensorMap &mapA, const CUtensorMap &mapB, const CUtensorMap &mapC,
               TcGroupParams &p, const RzGroupPieces &pieces)
{
    if (c.pb->precision == RZ_PREC_FP32) {
        if (plan.nc == 128) return launch<OP, true, 1, 1, 1, 128>(c, mapA, mapB, mapC, p, pieces);
        return launch<OP, true, 1, 1, 1, 64>(c, mapA, mapB, mapC, p, pieces);
    }
    constexpr int W1 = OP == OP_DW ? 4 : 1, W2 = OP == OP_DW ? 2 : 1;   // epilogue warps per TMEM lane quarter and row block
    if constexpr (OP == OP_DW) {
        if (c.pb->precision == RZ_PREC_BF16) {
            if (plan.rb == 2) return launch<OP, false, 2, 2, 0, 256, W2>(c, mapA, mapB, mapC, p, pieces);
            if (plan.ctas == 2) return launch<OP, false, 2, 1, 0, 256, W1>(c, mapA, mapB, mapC, p, pieces);
            if (plan.nc == 256) return launch<OP, false, 1, 1, 0, 256, W1>(c, mapA, mapB, mapC, p, pieces);
            if (plan.nc == 128) return launch<OP, false, 1, 1, 0, 128, W1>(c, mapA, mapB, mapC, p, pieces);
            return launch<OP, false, 1, 1, 0, 64, W1>(c, mapA, mapB, mapC, p, pieces);
        }
    }
    if (plan.rb == 2) return launch<OP, true, 2, 2, 0, 256, W2>(c, mapA, mapB, mapC, p, pieces);
    if (plan.ctas == 2) return launch<OP, true, 2, 1, 0, 256, W1>(c, mapA, mapB, mapC, p, pieces);
    if (plan.nc == 256) return launch<OP, true, 1, 1, 0, 256, W1>(c, mapA, mapB, mapC, p, pieces);
    if (plan.nc == 128) return launch<OP, true, 1, 1, 0, 128, W1>(c, mapA, mapB, mapC, p, pieces);
    return launch<OP, true, 1, 1, 0, 64, W1>(c, mapA, mapB, mapC, p, pieces);
}

}  // namespace

// Block shape by an estimate of the time: waves of blocks over the SMs, times a block's stages (or, weight gradient, its
// scatter where that is longer), at the relative tensor throughput each shape sustains.  The host knows the rows and the groups
// but not how the rows are spread: it reckons with even groups, each with half a ragged block at its end.
RzTcGroupPlan rz_tc_grouped_plan(const rz_problem *pb, int groups, int op)
{
    if (pb->precision == RZ_PREC_BF16 && op != RZ_OP_BACKWARD_WEIGHT) return rows_plan(pb, groups, op);
    static const struct {
        int ctas, rb, nc;
        double speed;
    } shapes[] = {{2, 2, 256, 1.00}, {2, 1, 256, 0.80}, {1, 1, 256, 0.58}, {1, 1, 128, 0.40}, {1, 1, 64, 0.25}};
    const bool bf16 = pb->precision == RZ_PREC_BF16, split = pb->precision == RZ_PREC_FP32, dw = op == RZ_OP_BACKWARD_WEIGHT;
    const double kc = bf16 ? 64.0 : 32.0;
    const double used = (double)(pb->M < groups ? pb->M : groups), mean = (double)pb->M / used;
    const int64_t cols = op == RZ_OP_FORWARD ? pb->N : pb->K;
    const int sms = usable_sms(pb);
    RzTcGroupPlan best = {1, 1, 64, 128, false};
    double best_time = -1.0;
    const int forced = forced_shape();
    for (int i = 0; i < 5; ++i) {
        const auto &s = shapes[i];
        // split precision: no pairs, and at least three chains; seven where three would be longer than 1440 elements (4e-6)
        const int64_t depth = dw ? 2048 : op == RZ_OP_FORWARD ? pb->K : pb->N;
        if (split && (s.ctas == 2 || s.nc == 256 || (s.nc == 128 && depth > 3 * 1440))) continue;
        const int64_t bcols = s.nc / s.ctas;                   // whole B boxes per hash tile (input gradient)
        if (op == RZ_OP_BACKWARD_INPUT && (pb->BK <= bcols ? bcols % pb->BK != 0 : pb->BK % bcols != 0)) continue;
        const double slots = (double)(sms / s.ctas), tiles_c = (double)((cols + s.nc - 1) / s.nc);
        const int item_r = TILE_R * s.ctas * s.rb;
        double items, stages;
        uint32_t step = (uint32_t)item_r;
        if (dw) {
            // at most 2048 rows in one accumulation chain: the tensor core truncates when it adds
            step = 2048;
            const double blocks = (double)((pb->N + item_r - 1) / item_r) * tiles_c;
            const double pieces = used * (double)((int64_t)((mean + step - 1) / step));
            items = pieces * blocks;
            stages = mean * used / pieces / kc + 1.0;
            if (s.rb == 2) stages += 19.0;                     // its scatter does not overlap the next block
            else if (stages < 8.0) stages = 8.0;               // shorter contractions are bound by the scatter
        } else {
            const double per_group = mean / item_r + 0.5;
            items = used * (per_group < 1.0 ? 1.0 : per_group) * tiles_c;
            stages = (double)((op == RZ_OP_FORWARD ? pb->K : pb->N)) / kc + (s.rb == 2 ? 10.0 : 3.0);
        }
        double waves = items / slots;
        waves = waves < 1.0 ? 1.0 : waves + 0.5;               // half a wave is lost at the end
        const double time = waves * stages * (double)(s.rb * s.nc) / s.speed;
        if (best_time < 0.0 || time < best_time || i == forced) {
            best_time = i == forced ? 0.0 : time;
            best.ctas = s.ctas, best.rb = s.rb, best.nc = s.nc, best.step = step;
        }
    }
    return best;
}

int rz_tc_grouped_forward(const RzLaunchCtx &c, const RzTcGroupPlan &plan, const RzGroupPieces &pieces, const void *X, const void *copies,
                          const float *bias, void *Y)
{
    const rz_problem *pb = c.pb;
    if (pb->precision == RZ_PREC_BF16) return launch_rows_any<ROWS_FWD>(c, plan, pieces, X, copies, bias, Y);
    const Geometry g = geometry(pb);
    TcGroupParams p;
    memset(&p, 0, sizeof(p));
    p.bias = bias;
    p.out = Y;
    CUtensorMap mapA, mapB, mapC;
    int st = map_matrix(&mapA, true, 0, X, pb->M, pb->K, g.epr, TILE_R, false);
    if (st) return st;
    st = map_shadow(&mapB, pb, true, copies, pb->BK < g.epr ? pb->BK : g.epr, false);
    if (st) return st;
    st = map_matrix(&mapC, true, 0, Y, pb->M, pb->N, g.epr, 32, false);
    if (st) return st;
    return launch_any<OP_FWD>(c, plan, mapA, mapB, mapC, p, pieces);
}

int rz_tc_grouped_backward_input(const RzLaunchCtx &c, const RzTcGroupPlan &plan, const RzGroupPieces &pieces, const void *dY,
                                 const void *copies, void *dX)
{
    const rz_problem *pb = c.pb;
    if (pb->precision == RZ_PREC_BF16) return launch_rows_any<ROWS_DX>(c, plan, pieces, dY, copies, nullptr, dX);
    const Geometry g = geometry(pb);
    TcGroupParams p;
    memset(&p, 0, sizeof(p));
    p.out = dX;
    CUtensorMap mapA, mapB, mapC;
    int st = map_matrix(&mapA, true, 0, dY, pb->M, pb->N, g.epr, TILE_R, false);
    if (st) return st;
    const uint32_t bcols = (uint32_t)(plan.nc / plan.ctas);
    st = map_shadow(&mapB, pb, false, copies, (uint32_t)pb->BK < bcols ? (uint32_t)pb->BK : bcols, false);
    if (st) return st;
    st = map_matrix(&mapC, true, 0, dX, pb->M, pb->K, g.epr, 32, false);
    if (st) return st;
    return launch_any<OP_DX>(c, plan, mapA, mapB, mapC, p, pieces);
}

int rz_tc_grouped_backward_weight(const RzLaunchCtx &c, const RzTcGroupPlan &plan, const RzGroupPieces &pieces, const void *maps, float *dH)
{
    TcGroupParams p;
    memset(&p, 0, sizeof(p));
    p.dH = dH;
    p.maps = static_cast<const CUtensorMap *>(maps);
    CUtensorMap unused;   // the groups' own maps are on the device
    memset(&unused, 0, sizeof(unused));
    return launch_any<OP_DW>(c, plan, unused, unused, unused, p, pieces);
}
