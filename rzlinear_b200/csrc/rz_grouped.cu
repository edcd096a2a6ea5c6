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

struct PlanArgs {
    const int32_t *offsets;
    uint32_t groups, M, step;
    uint32_t *header;
    uint4 *entries;
    CUtensorMap *maps;      // NULL: none wanted
    uint8_t *out;           // NULL: no rows to clear
    uint64_t row_bytes;
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

// Block 0 lists the pieces; the other blocks (block 0 too when it is alone) make the maps and clear rows.
__global__ void __launch_bounds__(PLAN_THREADS)
rz_group_plan_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const PlanArgs p)
{
    __shared__ uint32_t bound[RZ_GROUPS_MAX + 1];   // offsets within [0, M], never falling
    __shared__ uint32_t first[RZ_GROUPS_MAX + 1];   // pieces before each group
    __shared__ uint32_t warp_sums[32];
    __shared__ __align__(128) CUtensorMap staged[PLAN_THREADS / 32];
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

    if (blockIdx.x == 0) {
        carry = 0;
        for (uint32_t b0 = 0; b0 < G; b0 += PLAN_THREADS) {
            const uint32_t g = b0 + tid;
            uint32_t total;
            const uint32_t n = g < G ? (bound[g + 1] - bound[g] + p.step - 1) / p.step : 0u;
            const uint32_t before = block_scan(n, warp_sums, [](uint32_t a, uint32_t b) { return a + b; }, &total) - n;
            if (g < G) first[g] = carry + before;
            carry += total;
        }
        if (tid == 0) p.header[0] = carry;
        __syncthreads();
        for (uint32_t i = tid; i < carry; i += PLAN_THREADS) {
            uint32_t lo = 0, hi = G;   // the last group whose first piece is not behind i (and which has pieces)
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (first[mid] <= i) lo = mid;
                else hi = mid;
            }
            const uint32_t row = bound[lo] + (i - first[lo]) * p.step;
            p.entries[i] = make_uint4(lo, row, min(row + p.step, bound[lo + 1]), 0u);
        }
        if (gridDim.x > 1) return;
    }
    const uint32_t helper = gridDim.x > 1 ? blockIdx.x - 1 : 0, helpers = gridDim.x > 1 ? gridDim.x - 1 : 1;

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
    if (p.out) {
        const uint64_t head = (uint64_t)bound[0] * p.row_bytes, tail = (uint64_t)bound[G] * p.row_bytes, end = (uint64_t)p.M * p.row_bytes;
        const uint64_t step = (uint64_t)helpers * PLAN_THREADS, at = (uint64_t)helper * PLAN_THREADS + tid;
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

// ---- workspace: header, pieces, tensor maps ------------------------------------------------------------------------------
constexpr uint32_t SIMT_ROWS = 64, SIMT_CHUNK = 2048;   // rows of an FMA block; rows one block of the FMA weight gradient sums
constexpr uint32_t PREPARE_ROWS = 64;                   // rows a block of the bias pass sums

uint32_t most_pieces(const rz_problem *pb, int groups, uint32_t step) { return (uint32_t)(pb->M / step) + (uint32_t)groups; }

size_t pieces_bytes(const rz_problem *pb, int groups, uint32_t step)
{
    return (256 + sizeof(uint4) * (size_t)most_pieces(pb, groups, step) + 255) / 256 * 256;
}

uint32_t step_of(const rz_problem *pb, int groups, int op, bool tc)
{
    if (tc) return rz_tc_grouped_plan(pb, groups, op).step;
    return op == RZ_OP_BACKWARD_WEIGHT ? SIMT_CHUNK : SIMT_ROWS;
}

// Lists the pieces in `ws`.  `out`: rows of no group are cleared there.  `maps`: where each group's maps go, from mapA and mapB.
int plan_pieces(const RzLaunchCtx &c, int groups, const int32_t *offsets, uint32_t step, void *ws, void *out, uint64_t row_bytes,
                CUtensorMap *maps, const CUtensorMap *mapA, const CUtensorMap *mapB, RzGroupPieces *pieces)
{
    const rz_problem *pb = c.pb;
    PlanArgs p;
    p.offsets = offsets;
    p.groups = (uint32_t)groups, p.M = (uint32_t)pb->M, p.step = step;
    p.header = static_cast<uint32_t *>(ws);
    p.entries = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(ws) + 256);
    p.maps = maps;
    p.out = static_cast<uint8_t *>(out), p.row_bytes = row_bytes;
    static const CUtensorMap none = {};
    // helper blocks: one for each 256 KB that may have to be cleared, or for each 32 maps
    uint64_t helpers = out ? (uint64_t)pb->M * row_bytes >> 18 : 0;
    if (maps && helpers < (uint64_t)groups / 16) helpers = (uint64_t)groups / 16;
    if (helpers > 147) helpers = 147;
    rz_group_plan_kernel<<<(unsigned)(1 + helpers), PLAN_THREADS, 0, c.stream>>>(mapA ? *mapA : none, mapB ? *mapB : none, p);
    rz_count_launch(1);
    pieces->header = p.header;
    pieces->entries = p.entries;
    pieces->most = most_pieces(pb, groups, step);
    pieces->group_tiles = (uint32_t)((pb->K + pb->BK - 1) / pb->BK);
    return rz_record_cuda(cudaGetLastError(), "group plan launch");
}

// ---- bias gradient and ReLU mask -----------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Block = one piece and 256 * V columns, V of them a thread (V > 1: rows aligned for V-element accesses).
template <typename T, int V>
__global__ void __launch_bounds__(256)
rz_grouped_prepare_kernel(const T *__restrict__ dY, const T *__restrict__ Y, T *__restrict__ dYm, float *__restrict__ bias_grad,
                          uint32_t N, RzGroupPieces pieces)
{
    struct alignas(V * sizeof(T)) Pack {
        T e[V];
    };
    if (blockIdx.x >= __ldg(pieces.header)) return;
    const uint4 piece = __ldg(pieces.entries + blockIdx.x);
    const uint32_t col = (blockIdx.y * blockDim.x + threadIdx.x) * V;
    if (col >= N) return;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
#pragma unroll 4
    for (uint32_t r = piece.y; r < piece.z; ++r) {
        const size_t at = (size_t)r * N + col;
        Pack g = *reinterpret_cast<const Pack *>(dY + at);
        if (Y) {
            const Pack y = *reinterpret_cast<const Pack *>(Y + at);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (!(to_f32<T>(y.e[i]) > 0.f)) g.e[i] = T(0.f);
        }
        if (dYm) *reinterpret_cast<Pack *>(dYm + at) = g;
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += to_f32<T>(g.e[i]);
    }
    if (bias_grad) {
#pragma unroll
        for (int i = 0; i < V; ++i) atomicAdd(bias_grad + (size_t)piece.x * N + col + i, sum[i]);
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
    if (vec)
        rz_grouped_prepare_kernel<T, V><<<grid, 256, 0, c.stream>>>((const T *)dY, (const T *)Y, (T *)dYm, bias_grad, N, pieces);
    else
        rz_grouped_prepare_kernel<T, 1><<<grid, 256, 0, c.stream>>>((const T *)dY, (const T *)Y, (T *)dYm, bias_grad, N, pieces);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "grouped gradient preparation launch");
}

uint64_t element_bytes(const rz_problem *pb) { return pb->io_dtype == RZ_BF16 ? 2 : 4; }

}  // namespace

size_t rz_grouped_workspace(const rz_problem *pb, int groups, bool tc)
{
    // one size for all operations of a layer: the longest list (the bias pass has one too), then the weight gradient's maps
    size_t most = pieces_bytes(pb, groups, PREPARE_ROWS);
    for (int op = RZ_OP_FORWARD; op <= RZ_OP_BACKWARD_WEIGHT; ++op) {
        const size_t b = pieces_bytes(pb, groups, step_of(pb, groups, op, tc));
        if (b > most) most = b;
    }
    return most + (tc ? 2 * sizeof(CUtensorMap) * (size_t)groups : 0);
}

int rz_grouped_run_forward(const RzLaunchCtx &c, int groups, const int32_t *offsets, const void *X, const float *hashed, const void *copies,
                           const float *bias, void *Y, void *ws, bool tc)
{
    RzGroupPieces pieces;
    int st = plan_pieces(c, groups, offsets, step_of(c.pb, groups, RZ_OP_FORWARD, tc), ws, Y, element_bytes(c.pb) * (uint64_t)c.pb->N, nullptr,
                         nullptr, nullptr, &pieces);
    if (st) return st;
    if (tc) return rz_tc_grouped_forward(c, rz_tc_grouped_plan(c.pb, groups, RZ_OP_FORWARD), pieces, X, copies, bias, Y);
    return rz_simt_grouped_forward(c, pieces, X, hashed, bias, Y);
}

int rz_grouped_run_backward_input(const RzLaunchCtx &c, int groups, const int32_t *offsets, const void *dY, const float *hashed,
                                  const void *copies, void *dX, void *ws, bool tc)
{
    RzGroupPieces pieces;
    int st = plan_pieces(c, groups, offsets, step_of(c.pb, groups, RZ_OP_BACKWARD_INPUT, tc), ws, dX, element_bytes(c.pb) * (uint64_t)c.pb->K,
                         nullptr, nullptr, nullptr, &pieces);
    if (st) return st;
    if (tc) return rz_tc_grouped_backward_input(c, rz_tc_grouped_plan(c.pb, groups, RZ_OP_BACKWARD_INPUT), pieces, dY, copies, dX);
    return rz_simt_grouped_backward_input(c, pieces, dY, hashed, dX);
}

int rz_grouped_run_backward_weight(const RzLaunchCtx &c, int groups, const int32_t *offsets, const void *X, const void *dY, float *dH,
                                   void *ws, bool tc)
{
    const rz_problem *pb = c.pb;
    RzGroupPieces pieces;
    if (!tc) {
        int st = plan_pieces(c, groups, offsets, SIMT_CHUNK, ws, nullptr, 0, nullptr, nullptr, nullptr, &pieces);
        if (st) return st;
        return rz_simt_grouped_backward_weight(c, pieces, X, dY, dH);
    }
    const rztc::Geometry g = rztc::geometry(pb);
    const bool tf32 = pb->precision != RZ_PREC_BF16;
    CUtensorMap mapA, mapB;   // A = dY, B = X, boxes of one 128-byte row by a stage's contraction rows
    int st = rztc::map_matrix(&mapA, tf32, true, dY, pb->M, pb->N, g.epr, g.epr);
    if (st) return st;
    st = rztc::map_matrix(&mapB, tf32, true, X, pb->M, pb->K, g.epr, g.epr);
    if (st) return st;
    const RzTcGroupPlan plan = rz_tc_grouped_plan(pb, groups, RZ_OP_BACKWARD_WEIGHT);
    static_assert(sizeof(CUtensorMap) == 128, "tensor maps are 128 bytes");   // (they stand behind the list)
    CUtensorMap *maps = reinterpret_cast<CUtensorMap *>(static_cast<uint8_t *>(ws) + (rz_grouped_workspace(pb, groups, true) - 2 * sizeof(CUtensorMap) * (size_t)groups));
    st = plan_pieces(c, groups, offsets, plan.step, ws, nullptr, 0, maps, &mapA, &mapB, &pieces);
    if (st) return st;
    return rz_tc_grouped_backward_weight(c, plan, pieces, maps, dH);
}

int rz_grouped_run_grad_prepare(const RzLaunchCtx &c, int groups, const int32_t *offsets, const void *dY, const void *Y, void *dYm,
                                float *bias_grad, void *ws)
{
    RzGroupPieces pieces;
    int st;
    if (bias_grad) {
        st = rz_record_cuda(cudaMemsetAsync(bias_grad, 0, sizeof(float) * (size_t)groups * (size_t)c.pb->N, c.stream), "zero bias gradient");
        if (st) return st;
    }
    st = plan_pieces(c, groups, offsets, PREPARE_ROWS, ws, nullptr, 0, nullptr, nullptr, nullptr, &pieces);
    if (st) return st;
    if (c.pb->io_dtype == RZ_BF16) return launch_prepare<__nv_bfloat16>(c, pieces, dY, Y, dYm, bias_grad);
    return launch_prepare<float>(c, pieces, dY, Y, dYm, bias_grad);
}
