// Products grouped by row: the plan that a launch reads on the device, the bias / ReLU pass of the backward, and the choice
// between the tensor-core kernels (rz_tc_grouped.cu) and the FMA kernels (rz_simt.cu).
//
// The row offsets live on the device (a router wrote them a moment ago), so the host does not know how many blocks there are.
// A small kernel turns the offsets into a list of pieces - at most `step` consecutive rows of one group - and the product kernels
// take their work from that list.  It also clears the output rows that belong to no group and, for the weight gradient, makes each
// group's tensor maps, which end where the group ends.
#include "rz_common.h"
#include "rz_ptx.cuh"
#include "rz_tc_host.h"

namespace {

constexpr int PLAN_THREADS = 1024;

struct PlanList {
    uint32_t *header;       // [0] = pieces
    uint4 *entries;
    uint32_t step;          // most rows of a piece
    uint32_t even;          // != 0: a group's pieces are equal, in multiples of 16 rows; else all but the last have `step` rows
};

constexpr int MAX_LISTS = 3;

struct PlanArgs {
    const int32_t *offsets;
    uint32_t groups, M, lists;
    PlanList list[MAX_LISTS];
    CUtensorMap *maps;      // NULL: none wanted
    uint8_t *out;           // NULL: no rows to clear
    uint64_t row_bytes;
    float *zero[2];         // arrays to clear as a whole (NULL: none)
    uint64_t zero_words[2];
};

// inclusive scan over the block with `op`; every thread's value and the total over the block
template <typename Op>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *warp_sums, Op op, uint32_t *total)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= (uint32_t)d) v = op(v, y);
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = warp_sums[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= (uint32_t)d) s = op(s, y);
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    if (warp) v = op(v, warp_sums[warp - 1]);
    *total = warp_sums[31];
    __syncthreads();
    return v;
}

// Block b < lists writes list b; the blocks behind make the maps and clear rows (block 0 where there are none).
__global__ void __launch_bounds__(PLAN_THREADS)
rz_group_plan_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const PlanArgs p)
{
    __shared__ uint32_t bound[RZ_GROUPS_MAX + 1];   // offsets within [0, M], never falling
    __shared__ uint32_t first[RZ_GROUPS_MAX + 1];   // pieces before each group
    __shared__ uint32_t warp_sums[32];
    __shared__ __align__(128) CUtensorMap staged[PLAN_THREADS / 32];
    rzptx::grid_launch_dependents();
    const uint32_t G = p.groups, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    uint32_t carry = 0;
    for (uint32_t b0 = 0; b0 <= G; b0 += PLAN_THREADS) {
        const uint32_t i = b0 + tid;
        uint32_t v = 0, total;
        if (i <= G) {
            const int32_t o = p.offsets[i];
            v = o < 0 ? 0u : min((uint32_t)o, p.M);
        }
        v = block_scan(v, warp_sums, [](uint32_t a, uint32_t b) { return max(a, b); }, &total);
        if (i <= G) bound[i] = max(v, carry);
        carry = max(carry, total);
    }
    __syncthreads();

    const bool alone = gridDim.x == p.lists;
    if (blockIdx.x < p.lists) {
        const PlanList list = p.list[blockIdx.x];
        carry = 0;
        for (uint32_t b0 = 0; b0 < G; b0 += PLAN_THREADS) {
            const uint32_t g = b0 + tid;
            uint32_t total;
            const uint32_t n = g < G ? (bound[g + 1] - bound[g] + list.step - 1) / list.step : 0u;
            const uint32_t before = block_scan(n, warp_sums, [](uint32_t a, uint32_t b) { return a + b; }, &total) - n;
            if (g < G) first[g] = carry + before;
            carry += total;
        }
        if (tid == 0) list.header[0] = carry;
        __syncthreads();
        for (uint32_t i = tid; i < carry; i += PLAN_THREADS) {
            uint32_t lo = 0, hi = G;   // the last group whose first piece is not behind i (and which has pieces)
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (first[mid] <= i) lo = mid;
                else hi = mid;
            }
            uint32_t rows = list.step;
            if (list.even) {
                const uint32_t n = bound[lo + 1] - bound[lo], count = (n + list.step - 1) / list.step;
                rows = ((n + count - 1) / count + 15) / 16 * 16;   // (<= step, a multiple of 16; the last piece is not empty)
            }
            const uint32_t row = bound[lo] + (i - first[lo]) * rows;
            list.entries[i] = make_uint4(lo, row, min(row + rows, bound[lo + 1]), 0u);
        }
        if (!alone || blockIdx.x) return;
    }
    const uint32_t helper = alone ? 0 : blockIdx.x - p.lists, helpers = alone ? 1 : gridDim.x - p.lists;

    if (p.maps) {
        const uint32_t dst = rzptx::smem_u32(&staged[warp]);
        for (uint32_t m = helper * (PLAN_THREADS / 32) + warp; m < 2 * G; m += helpers * (PLAN_THREADS / 32)) {
            const uint32_t *src = reinterpret_cast<const uint32_t *>((m & 1) ? &mapB : &mapA);
            reinterpret_cast<uint32_t *>(&staged[warp])[lane] = src[lane];
            __syncwarp();
            if (lane == 0) rzptx::tma_replace_rows(dst, max(1u, bound[(m >> 1) + 1]));
            __syncwarp();
            rzptx::tma_publish_desc(p.maps + m, dst);
            __syncwarp();
        }
    }
    const uint64_t step = (uint64_t)helpers * PLAN_THREADS, at = (uint64_t)helper * PLAN_THREADS + tid;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        float *o = p.zero[z];
        if (!o) continue;
        const uint64_t n = p.zero_words[z];
        const uint64_t head = min(n, (uint64_t)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(o) & 15u)) & 15u) / 4), quads = (n - head) / 4;
        if (at < head) o[at] = 0.f;
        for (uint64_t i = at; i < quads; i += step) reinterpret_cast<float4 *>(o + head)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        const uint64_t done = head + 4 * quads;
        if (at < n - done) o[done + at] = 0.f;
    }
    if (p.out) {
        const uint64_t head = (uint64_t)bound[0] * p.row_bytes, tail = (uint64_t)bound[G] * p.row_bytes, end = (uint64_t)p.M * p.row_bytes;
        if (((p.row_bytes | reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0) {
            uint4 *o = reinterpret_cast<uint4 *>(p.out);
            const uint4 zero = make_uint4(0, 0, 0, 0);
            for (uint64_t i = at; i < head / 16; i += step) o[i] = zero;
            for (uint64_t i = tail / 16 + at; i < end / 16; i += step) o[i] = zero;
        } else {
            uint16_t *o = reinterpret_cast<uint16_t *>(p.out);   // elements have two or four bytes
            for (uint64_t i = at; i < head / 2; i += step) o[i] = 0;
            for (uint64_t i = tail / 2 + at; i < end / 2; i += step) o[i] = 0;
        }
    }
}

// ---- workspace: lists (header, pieces), tensor maps -----------------------------------------------------------------------------
constexpr uint32_t SIMT_ROWS = 64, SIMT_CHUNK = 2048;   // rows of an FMA block; rows one block of the FMA weight gradient sums
constexpr uint32_t PREPARE_ROWS = 32;                   // rows a block of the bias pass sums

uint32_t most_pieces(const rz_problem *pb, int groups, uint32_t step) { return (uint32_t)(pb->M / step) + (uint32_t)groups; }

size_t pieces_bytes(const rz_problem *pb, int groups, uint32_t step)
{
    return (256 + sizeof(uint4) * (size_t)most_pieces(pb, groups, step) + 255) / 256 * 256;
}

struct Step {
    uint32_t rows;
    bool even;
};

Step step_of(const rz_problem *pb, int groups, int op, bool tc)
{
    if (tc) {
        const RzTcGroupPlan plan = rz_tc_grouped_plan(pb, groups, op);
        return Step{plan.step, plan.even};
    }
    return Step{op == RZ_OP_BACKWARD_WEIGHT ? SIMT_CHUNK : SIMT_ROWS, false};
}

// A plan under construction: lists are added one behind the other in the workspace, then one launch writes them all.
struct Plan {
    const RzLaunchCtx &c;
    int groups;
    uint8_t *ws;
    size_t used = 0;
    PlanArgs args = {};
    CUtensorMap mapA = {}, mapB = {};

    Plan(const RzLaunchCtx &c_, int groups_, const int32_t *offsets, void *ws_) : c(c_), groups(groups_), ws(static_cast<uint8_t *>(ws_))
    {
        args.offsets = offsets;
        args.groups = (uint32_t)groups_, args.M = (uint32_t)c_.pb->M;
    }
    RzGroupPieces add(const Step &s)
    {
        const uint32_t step = s.rows;
        RzGroupPieces pieces;
        PlanList &l = args.list[args.lists++];
        l.step = step;
        l.even = s.even;
        l.header = reinterpret_cast<uint32_t *>(ws + used);
        l.entries = reinterpret_cast<uint4 *>(ws + used + 256);
        used += pieces_bytes(c.pb, groups, step);
        pieces.header = l.header, pieces.entries = l.entries;
        pieces.most = most_pieces(c.pb, groups, step);
        pieces.groups = (uint32_t)groups;
        pieces.group_tiles = (uint32_t)((c.pb->K + c.pb->BK - 1) / c.pb->BK);
        return pieces;
    }
    // each group's maps of dY (mapA) and X (mapB)
    CUtensorMap *add_maps()
    {
        args.maps = reinterpret_cast<CUtensorMap *>(ws + used);
        used += 2 * sizeof(CUtensorMap) * (size_t)groups;
        return args.maps;
    }
    void zero(int z, float *words, uint64_t n) { args.zero[z] = words, args.zero_words[z] = n; }
    // rows of `out` that belong to no group are cleared
    void clear(void *out, uint64_t row_bytes) { args.out = static_cast<uint8_t *>(out), args.row_bytes = row_bytes; }
    int launch()
    {
        // helper blocks: one for each 256 KB of rows that may have to be cleared, each 64 KB of an array, each 32 maps
        uint64_t helpers = args.out ? (uint64_t)args.M * args.row_bytes >> 18 : 0;
        const uint64_t arrays = (args.zero_words[0] + args.zero_words[1]) >> 14;
        if (helpers < arrays) helpers = arrays;
        if (args.maps && helpers < (uint64_t)groups / 16) helpers = (uint64_t)groups / 16;
        if (helpers > 147) helpers = 147;
        rz_group_plan_kernel<<<(unsigned)(args.lists + helpers), PLAN_THREADS, 0, c.stream>>>(mapA, mapB, args);
        rz_count_launch(1);
        return rz_record_cuda(cudaGetLastError(), "group plan launch");
    }
};

// ---- bias gradient and ReLU mask -----------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Block = one piece and 256 * V columns, V of them a thread (V > 1: rows aligned for V-element accesses).  MASK: dYm = dY where the saved
// output does not say 0.  Bound by reading dY: 16384 x 4096 bf16 takes 33 us (4.1 TB/s), with one-word reductions and the mask's test
// between a row's load and the next's 46.
template <typename T, int V, bool MASK>
__global__ void __launch_bounds__(256)
rz_grouped_prepare_kernel(const T *__restrict__ dY, const T *__restrict__ Y, T *__restrict__ dYm, float *__restrict__ bias_grad,
                          uint32_t N, RzGroupPieces pieces)
{
    struct alignas(V * sizeof(T)) Pack {
        T e[V];
    };
    constexpr int U = 4;
    if (blockIdx.x >= __ldg(pieces.header)) return;
    const uint4 piece = __ldg(pieces.entries + blockIdx.x);
    const uint32_t col = (blockIdx.y * blockDim.x + threadIdx.x) * V;
    if (col >= N) return;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
#pragma unroll 1
    for (uint32_t r = piece.y; r < piece.z; r += U) {
        Pack g[U], y[MASK ? U : 1];
        const size_t at = (size_t)r * N + col;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r + u < piece.z) {
                g[u] = *reinterpret_cast<const Pack *>(dY + at + (size_t)u * N);
                if (MASK) y[MASK ? u : 0] = *reinterpret_cast<const Pack *>(Y + at + (size_t)u * N);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (r + u < piece.z) {
                if (MASK) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (to_f32<T>(y[MASK ? u : 0].e[i]) <= 0.f) g[u].e[i] = T(0.f);   // (not for a NaN: its gradient goes on)
                    *reinterpret_cast<Pack *>(dYm + at + (size_t)u * N) = g[u];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += to_f32<T>(g[u].e[i]);
            }
        }
    }
    if (bias_grad) {
        float *dst = bias_grad + (size_t)piece.x * N + col;
        if (V >= 4 && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
#pragma unroll
            for (int i = 0; i + 4 <= V; i += 4)
                asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(dst + i), "f"(sum[i]), "f"(sum[i + 1]), "f"(sum[i + 2]),
                             "f"(sum[i + 3])
                             : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) atomicAdd(dst + i, sum[i]);
        }
    }
}

template <typename T>
int launch_prepare(const RzLaunchCtx &c, const RzGroupPieces &pieces, const void *dY, const void *Y, void *dYm, float *bias_grad)
{
    const uint32_t N = (uint32_t)c.pb->N;
    constexpr int V = 16 / sizeof(T);
    const uintptr_t bits = reinterpret_cast<uintptr_t>(dY) | reinterpret_cast<uintptr_t>(Y) | reinterpret_cast<uintptr_t>(dYm);
    const bool vec = N % V == 0 && (bits & 15u) == 0;
    const uint32_t per_block = vec ? 256 * V : 256;
    const dim3 grid(pieces.most, (N + per_block - 1) / per_block, 1);
    if (grid.y > 65535u) return RZ_ERR_SHAPE;
    auto run = [&](auto kernel) {
        kernel<<<grid, 256, 0, c.stream>>>((const T *)dY, (const T *)Y, (T *)dYm, bias_grad, N, pieces);
    };
    if (Y) vec ? run(rz_grouped_prepare_kernel<T, V, true>) : run(rz_grouped_prepare_kernel<T, 1, true>);
    else vec ? run(rz_grouped_prepare_kernel<T, V, false>) : run(rz_grouped_prepare_kernel<T, 1, false>);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "grouped gradient preparation launch");
}

uint64_t element_bytes(const rz_problem *pb) { return pb->io_dtype == RZ_BF16 ? 2 : 4; }

}  // namespace

size_t rz_grouped_workspace(const rz_problem *pb, int groups, bool tc)
{
    // the backward's three lists and the weight gradient's maps, or the forward's list
    const size_t forward = pieces_bytes(pb, groups, step_of(pb, groups, RZ_OP_FORWARD, tc).rows);
    const size_t backward = pieces_bytes(pb, groups, PREPARE_ROWS) + pieces_bytes(pb, groups, step_of(pb, groups, RZ_OP_BACKWARD_INPUT, tc).rows) +
                            pieces_bytes(pb, groups, step_of(pb, groups, RZ_OP_BACKWARD_WEIGHT, tc).rows) +
                            (tc ? 2 * sizeof(CUtensorMap) * (size_t)groups : 0);
    return forward > backward ? forward : backward;
}

int rz_grouped_run_forward(const RzLaunchCtx &c, int groups, const int32_t *offsets, const void *X, const float *hashed, const void *copies,
                           const float *bias, void *Y, void *ws, bool tc)
{
    Plan plan(c, groups, offsets, ws);
    const RzGroupPieces pieces = plan.add(step_of(c.pb, groups, RZ_OP_FORWARD, tc));
    plan.clear(Y, element_bytes(c.pb) * (uint64_t)c.pb->N);
    const int st = plan.launch();
    if (st) return st;
    if (tc) return rz_tc_grouped_forward(c, rz_tc_grouped_plan(c.pb, groups, RZ_OP_FORWARD), pieces, X, copies, bias, Y);
    return rz_simt_grouped_forward(c, pieces, X, hashed, bias, Y);
}

int rz_grouped_run_backward(const RzLaunchCtx &c, int groups, const int32_t *offsets, const void *X, const void *dY, const void *Y,
                            const float *hashed, const void *copies, void *dYm, float *bias_grad, void *dX, float *dH, void *ws, bool tc)
{
    const rz_problem *pb = c.pb;
    static_assert(sizeof(CUtensorMap) == 128, "tensor maps are 128 bytes");
    const bool prepare = Y || bias_grad;
    const void *grad = Y ? dYm : dY;   // what the products see
    Plan plan(c, groups, offsets, ws);
    RzGroupPieces rows, blocks, chunks;
    int st;
    if (prepare) rows = plan.add(Step{PREPARE_ROWS, false});
    if (dX) {
        blocks = plan.add(step_of(pb, groups, RZ_OP_BACKWARD_INPUT, tc));
        plan.clear(dX, element_bytes(pb) * (uint64_t)pb->K);
    }
    const CUtensorMap *maps = nullptr;
    if (dH) {
        chunks = plan.add(step_of(pb, groups, RZ_OP_BACKWARD_WEIGHT, tc));
        if (tc) {   // A = dY, B = X, boxes of one 128-byte row by a stage's contraction rows
            const rztc::Geometry g = rztc::geometry(pb);
            const bool tf32 = pb->precision != RZ_PREC_BF16;
            st = rztc::map_matrix(&plan.mapA, tf32, true, grad, pb->M, pb->N, g.epr, g.epr, false);
            if (st) return st;
            st = rztc::map_matrix(&plan.mapB, tf32, true, X, pb->M, pb->K, g.epr, g.epr, false);
            if (st) return st;
            maps = plan.add_maps();
        }
    }
    if (bias_grad) plan.zero(0, bias_grad, (uint64_t)groups * (uint64_t)pb->N);
    if (dH && !(pb->flags & RZ_FLAG_ACCUMULATE_DH)) plan.zero(1, dH, (uint64_t)pb->H);
    st = plan.launch();
    if (st) return st;
    if (prepare) {
        st = pb->io_dtype == RZ_BF16 ? launch_prepare<__nv_bfloat16>(c, rows, dY, Y, dYm, bias_grad)
                                     : launch_prepare<float>(c, rows, dY, Y, dYm, bias_grad);
        if (st) return st;
    }
    if (dX) {
        st = tc ? rz_tc_grouped_backward_input(c, rz_tc_grouped_plan(pb, groups, RZ_OP_BACKWARD_INPUT), blocks, grad, copies, dX)
                : rz_simt_grouped_backward_input(c, blocks, grad, hashed, dX);
        if (st) return st;
    }
    if (!dH) return RZ_OK;
    if (tc) return rz_tc_grouped_backward_weight(c, rz_tc_grouped_plan(pb, groups, RZ_OP_BACKWARD_WEIGHT), chunks, maps, dH);
    return rz_simt_grouped_backward_weight(c, chunks, X, grad, dH);
}
