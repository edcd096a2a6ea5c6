// Host side of the tensor-core kernels (rz_tc_kernel.cuh): block shapes, tensor maps, launches of the linear layer's three
// operations; the shadow copies, the optimiser step and the finalize pass of split contractions.
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "rz_tc_host.h"
#include "rz_tc_kernel.cuh"

using namespace rztc;

namespace {

// ---- self-test of the bounded-wait machinery ---------------------------------------------------
// One thread waits on an mbarrier that nothing will ever complete.  The wait must give up after
// `limit` cycles, leave its code in the status word and let the kernel return normally.
__global__ void rz_wait_selftest_kernel(WaitCtx w)
{
    __shared__ __align__(8) uint64_t bar;
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&bar), 1);
        fence_barrier_init();
        (void)mbar_wait_bounded(smem_u32(&bar), 0, RZ_WAIT_SELFTEST, w);
    }
}

// ---- shadow copies and SGD -----------------------------------------------------------------

__device__ __forceinline__ uint32_t to_tf32(float v)
{
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}

// copy s, element j  =  convert(hashed[j + s])   (0 past the end); one thread writes NS elements of every copy
// `raw` (fp32 elements only): keep every mantissa bit, for the split-precision kernels that form hi/lo themselves
template <bool TF32>
__global__ void rz_shadow_kernel(const float *__restrict__ hashed, uint8_t *__restrict__ shadow, uint32_t H, uint32_t Hc,
                                 size_t copy_stride, int raw)
{
    constexpr int NS = TF32 ? 4 : 8;
    const uint32_t groups = Hc / NS;
    for (uint32_t g = blockIdx.x * blockDim.x + threadIdx.x; g < groups; g += gridDim.x * blockDim.x) {
        const uint32_t j0 = g * NS;
        float v[2 * NS];
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) v[i] = (j0 + i < H) ? hashed[j0 + i] : 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            uint4 u;
            if (TF32) {
                u.x = raw ? __float_as_uint(v[s + 0]) : to_tf32(v[s + 0]);
                u.y = raw ? __float_as_uint(v[s + 1]) : to_tf32(v[s + 1]);
                u.z = raw ? __float_as_uint(v[s + 2]) : to_tf32(v[s + 2]);
                u.w = raw ? __float_as_uint(v[s + 3]) : to_tf32(v[s + 3]);
            } else {
                __nv_bfloat162 h0 = __floats2bfloat162_rn(v[s + 0], v[s + 1]);
                __nv_bfloat162 h1 = __floats2bfloat162_rn(v[s + 2], v[s + 3]);
                __nv_bfloat162 h2 = __floats2bfloat162_rn(v[s + 4], v[s + 5]);
                __nv_bfloat162 h3 = __floats2bfloat162_rn(v[s + 6], v[s + 7]);
                u.x = *reinterpret_cast<uint32_t *>(&h0);
                u.y = *reinterpret_cast<uint32_t *>(&h1);
                u.z = *reinterpret_cast<uint32_t *>(&h2);
                u.w = *reinterpret_cast<uint32_t *>(&h3);
            }
            *reinterpret_cast<uint4 *>(shadow + s * copy_stride + (size_t)g * 16) = u;
        }
    }
}

__global__ void rz_sgd_kernel(float *__restrict__ hashed, const float *__restrict__ dH, float lr, uint32_t H)
{
    const uint32_t n4 = H / 4;
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < n4; i += gridDim.x * blockDim.x) {
        float4 h = reinterpret_cast<float4 *>(hashed)[i];
        const float4 g = reinterpret_cast<const float4 *>(dH)[i];
        h.x -= lr * g.x;
        h.y -= lr * g.y;
        h.z -= lr * g.z;
        h.w -= lr * g.w;
        reinterpret_cast<float4 *>(hashed)[i] = h;
    }
    if (blockIdx.x == 0 && threadIdx.x < (H & 3u)) {
        const uint32_t i = n4 * 4 + threadIdx.x;
        hashed[i] -= lr * dH[i];
    }
}

// v = momentum * v + dH;  hashed -= lr * v   (heavy-ball SGD on the hashed array)
__global__ void rz_sgd_momentum_kernel(float *__restrict__ hashed, const float *__restrict__ dH, float *__restrict__ vel,
                                       float lr, float momentum, uint32_t H)
{
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < H; i += gridDim.x * blockDim.x) {
        const float v = momentum * vel[i] + dH[i];
        vel[i] = v;
        hashed[i] -= lr * v;
    }
}

// The optimiser step and the shadow refresh in ONE pass over the hashed array:
//   (velocity = momentum * velocity + dH;)   hashed -= lr * (velocity | dH);   copy s, element j = convert(hashed[j + s]).
// A thread owns one aligned group of NS elements: it updates them in place and writes the NS 16-byte pieces of the
// shifted copies that start in its group.  Those pieces reach NS - 1 elements into the NEXT group, whose new values
// come from the neighbouring lane (shuffle) or warp (shared memory) of the same chunk of SGD_CHUNK groups.  The last group of
// a chunk has its neighbour in another block, which may or may not have updated it yet: its pieces for copies
// 1 .. NS-1 are left to the block that finishes last (a ticket counter tells which), which by then reads final values.
constexpr int SGD_CHUNK = 1024;    // groups per block iteration (= threads per block): few chunk boundaries for the last block
constexpr int SGD_TICKETS = 64;    // launches that may be in flight at once, one ticket word each
__device__ unsigned g_sgd_ticket[SGD_TICKETS];

template <bool TF32>
__device__ __forceinline__ uint4 shadow_piece(const float *v, int raw)
{
    uint4 u;
    if (TF32) {
        u.x = raw ? __float_as_uint(v[0]) : to_tf32(v[0]);
        u.y = raw ? __float_as_uint(v[1]) : to_tf32(v[1]);
        u.z = raw ? __float_as_uint(v[2]) : to_tf32(v[2]);
        u.w = raw ? __float_as_uint(v[3]) : to_tf32(v[3]);
    } else {
        __nv_bfloat162 h0 = __floats2bfloat162_rn(v[0], v[1]);
        __nv_bfloat162 h1 = __floats2bfloat162_rn(v[2], v[3]);
        __nv_bfloat162 h2 = __floats2bfloat162_rn(v[4], v[5]);
        __nv_bfloat162 h3 = __floats2bfloat162_rn(v[6], v[7]);
        u.x = *reinterpret_cast<uint32_t *>(&h0);
        u.y = *reinterpret_cast<uint32_t *>(&h1);
        u.z = *reinterpret_cast<uint32_t *>(&h2);
        u.w = *reinterpret_cast<uint32_t *>(&h3);
    }
    return u;
}

template <bool TF32, bool MOMENTUM>
__global__ void __launch_bounds__(SGD_CHUNK)
rz_sgd_shadow_kernel(float *__restrict__ hashed, const float *__restrict__ dH, float *__restrict__ vel, float lr, float momentum,
                     uint8_t *__restrict__ shadow, uint32_t H, uint32_t Hc, size_t copy_stride, int raw, unsigned *ticket)
{
    constexpr int NS = TF32 ? 4 : 8;
    __shared__ float first_of_warp[SGD_CHUNK / 32][NS];
    __shared__ bool is_last;
    const uint32_t groups = Hc / NS, nchunks = (groups + SGD_CHUNK - 1) / SGD_CHUNK;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint32_t chunk = blockIdx.x; chunk < nchunks; chunk += gridDim.x) {
        const uint32_t g = chunk * SGD_CHUNK + threadIdx.x, j0 = g * NS;
        float nv[2 * NS];   // new values of this group, then of the next one
#pragma unroll
        for (int i = 0; i < NS; ++i) nv[i] = 0.f;
        if (g < groups && j0 < H) {
            if (j0 + NS <= H) {
#pragma unroll
                for (int q = 0; q < NS / 4; ++q) {
                    float4 h = reinterpret_cast<float4 *>(hashed + j0)[q];
                    float4 d = reinterpret_cast<const float4 *>(dH + j0)[q];
                    if (MOMENTUM) {
                        const float4 v = reinterpret_cast<float4 *>(vel + j0)[q];
                        d.x = momentum * v.x + d.x, d.y = momentum * v.y + d.y, d.z = momentum * v.z + d.z, d.w = momentum * v.w + d.w;
                        reinterpret_cast<float4 *>(vel + j0)[q] = d;
                    }
                    h.x -= lr * d.x, h.y -= lr * d.y, h.z -= lr * d.z, h.w -= lr * d.w;
                    reinterpret_cast<float4 *>(hashed + j0)[q] = h;
                    nv[4 * q + 0] = h.x, nv[4 * q + 1] = h.y, nv[4 * q + 2] = h.z, nv[4 * q + 3] = h.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    if (j0 + i < H) {
                        float d = dH[j0 + i];
                        if (MOMENTUM) {
                            d = momentum * vel[j0 + i] + d;
                            vel[j0 + i] = d;
                        }
                        nv[i] = hashed[j0 + i] - lr * d;
                        hashed[j0 + i] = nv[i];
                    }
                }
            }
        }
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < NS; ++i) first_of_warp[warp][i] = nv[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NS; ++i) nv[NS + i] = __shfl_down_sync(0xffffffffu, nv[i], 1);
        const bool chunk_end = threadIdx.x == SGD_CHUNK - 1;
        if (lane == 31 && !chunk_end) {
#pragma unroll
            for (int i = 0; i < NS; ++i) nv[NS + i] = first_of_warp[warp + 1][i];
        }
        const bool deferred = chunk_end && g + 1 < groups;   // the neighbour group belongs to another block
        if (chunk_end) {
#pragma unroll
            for (int i = 0; i < NS; ++i) nv[NS + i] = 0.f;   // (past the end of the array when not deferred)
        }
        if (g < groups) {
#pragma unroll
            for (int s2 = 0; s2 < NS; ++s2)
                if (s2 == 0 || !deferred)
                    *reinterpret_cast<uint4 *>(shadow + s2 * copy_stride + (size_t)g * 16) = shadow_piece<TF32>(nv + s2, raw);
        }
        __syncthreads();   // first_of_warp is rewritten by the next chunk
    }
    // the block that finishes last fills in the pieces that straddle chunk boundaries
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) is_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    for (uint32_t b = threadIdx.x; b + 1 < nchunks; b += SGD_CHUNK) {
        const uint32_t g = b * SGD_CHUNK + SGD_CHUNK - 1, j0 = g * NS;
        float nv[2 * NS];
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) nv[i] = (j0 + i < H) ? __ldcg(hashed + j0 + i) : 0.f;
#pragma unroll
        for (int s2 = 1; s2 < NS; ++s2)
            *reinterpret_cast<uint4 *>(shadow + s2 * copy_stride + (size_t)g * 16) = shadow_piece<TF32>(nv + s2, raw);
    }
    if (threadIdx.x == 0) *ticket = 0;   // ready for the next launch that draws this ticket word
}

// out = convert(alpha * partial_sums (+ bias) (ReLU)) for the blocks of a FWD / DX launch whose contraction was
// split: block n_main + i owns workspace tile i (item_r x nc floats, row-major); gridDim.y CTAs share a block.
struct FinalizeGeom {
    uint32_t rows, cols, item_r, nc, tiles_r, tiles_c, group_rows, n_main, n_tiles;
};

template <typename T>
__global__ void rz_finalize_kernel(const float *__restrict__ ws, T *__restrict__ out, const float *__restrict__ bias,
                                   FinalizeGeom g, float alpha, int relu)
{
    const uint32_t quads_per_row = g.nc / 4;
    for (uint32_t i = blockIdx.x; i + g.n_main < g.n_tiles; i += gridDim.x) {
        const uint32_t tile = g.n_main + i;
        const uint32_t per_group = g.group_rows * g.tiles_c;
        const uint32_t group = tile / per_group, within = tile - group * per_group;
        const uint32_t first_r = group * g.group_rows;
        const uint32_t gsz = min(g.tiles_r - first_r, g.group_rows);
        const uint32_t tr = first_r + within % gsz, tc = within / gsz;
        const float *wt = ws + (size_t)i * g.item_r * g.nc;
        const uint32_t valid_rows = min(g.item_r, g.rows - tr * g.item_r);   // rows of the block that exist
        const uint32_t nq = valid_rows * quads_per_row;
        for (uint32_t e = blockIdx.y * blockDim.x + threadIdx.x; e < nq; e += blockDim.x * gridDim.y) {
            const uint32_t lr = e / quads_per_row, lc = (e - lr * quads_per_row) * 4;
            const uint32_t row = tr * g.item_r + lr, col = tc * g.nc + lc;
            if (row >= g.rows || col >= g.cols) continue;   // cols is a multiple of 4
            float4 v = *reinterpret_cast<const float4 *>(wt + (size_t)lr * g.nc + lc);
            v.x *= alpha, v.y *= alpha, v.z *= alpha, v.w *= alpha;
            if (bias) v.x += bias[col], v.y += bias[col + 1], v.z += bias[col + 2], v.w += bias[col + 3];
            if (relu) v.x = fmaxf(v.x, 0.f), v.y = fmaxf(v.y, 0.f), v.z = fmaxf(v.z, 0.f), v.w = fmaxf(v.w, 0.f);
            const size_t o = (size_t)row * g.cols + col;
            if (sizeof(T) == 4) {
                *reinterpret_cast<float4 *>(reinterpret_cast<float *>(out) + o) = v;
            } else {
                __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
                uint2 u;
                u.x = *reinterpret_cast<uint32_t *>(&lo);
                u.y = *reinterpret_cast<uint32_t *>(&hi);
                *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(out) + o) = u;
            }
        }
    }
}

// ---- host side -----------------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode()
{
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(ptr);
    }
    return fn;
}

// `mn_major`: the tile feeds an M/N-major operand; for 32-bit elements that needs the 32-byte-chunk flavour
// of the 128-byte swizzle, every other case uses the 16-byte-chunk one.
// Encoded maps are pure functions of (base, type, swizzle flavour, extents, strides, box): each host thread keeps
// the last few it made, so steady-state launches (the same tensors step after step) encode nothing.
struct MapKey {
    const void *base;
    uint64_t dims[3], strides[2];
    uint32_t box[3];
    int rank, tf32, mn_major;
    bool operator==(const MapKey &o) const { return memcmp(this, &o, sizeof(MapKey)) == 0; }
};
struct MapCache {
    static constexpr int N = 16;
    MapKey key[N];
    alignas(64) CUtensorMap map[N];
    int used = 0, next = 0;
};

}  // namespace

namespace rztc {

int encode(CUtensorMap *map, bool tf32, int mn_major, void *base, int rank, const uint64_t *dims,
           const uint64_t *strides_bytes, const uint32_t *box, bool keep)
{
    static thread_local MapCache cache;
    MapKey k;
    memset(&k, 0, sizeof(k));   // (padding too: keys are compared bytewise)
    k.base = base, k.rank = rank, k.tf32 = tf32, k.mn_major = mn_major;
    for (int i = 0; i < rank; ++i) k.dims[i] = dims[i], k.box[i] = box[i];
    for (int i = 0; i + 1 < rank; ++i) k.strides[i] = strides_bytes[i];
    for (int i = 0; keep && i < cache.used; ++i)
        if (cache.key[i] == k) {
            *map = cache.map[i];
            return RZ_OK;
        }
    EncodeTiledFn fn = get_encode();
    if (!fn) return rz_record_cuda(cudaErrorUnknown, "cuTensorMapEncodeTiled not available");
    // The encoder is a driver call and wants a context current on this thread.  A thread that has made no
    // runtime call yet (an autograd worker, say) has none: a null free binds the device's primary context.
    static thread_local bool bound = false;
    if (!bound) {
        int st = rz_record_cuda(cudaFree(nullptr), "bind the primary context");
        if (st) return st;
        bound = true;
    }
    cuuint64_t gdim[3];
    cuuint64_t gstr[2];
    cuuint32_t bx[3], estr[3];
    for (int i = 0; i < rank; ++i) {
        gdim[i] = dims[i];
        bx[i] = box[i];
        estr[i] = 1;
    }
    for (int i = 0; i + 1 < rank; ++i) gstr[i] = strides_bytes[i];
    CUresult r = fn(map, tf32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, base,
                    gdim, gstr, bx, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    mn_major == PLAIN_LAYOUT ? CU_TENSOR_MAP_SWIZZLE_NONE
                    : (tf32 && mn_major)     ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B
                                             : CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        char msg[96];
        snprintf(msg, sizeof(msg), "cuTensorMapEncodeTiled failed (CUresult %d, rank %d)", (int)r, rank);
        return rz_record_cuda(cudaErrorInvalidValue, msg);
    }
    if (!keep) return RZ_OK;
    const int slot = cache.used < MapCache::N ? cache.used++ : (cache.next = (cache.next + 1) % MapCache::N);
    cache.key[slot] = k;
    cache.map[slot] = *map;
    return RZ_OK;
}

int num_sms()
{
    static int cached[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!cached[dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        cached[dev] = n;
    }
    return cached[dev];
}

}  // namespace rztc

namespace {

// SMs a launch may occupy: all of them, less the ones the problem asks to leave idle (a collective that should
// run beside a persistent kernel needs SMs of its own); never fewer than two.
int usable_sms(const rz_problem *pb)
{
    int n = num_sms() - (pb->sm_reserve > 0 ? pb->sm_reserve : 0);
    return n < 2 ? 2 : n;
}

uint32_t env_u32(const char *name, uint32_t dflt)
{
    const char *s = getenv(name);
    return s ? (uint32_t)strtoul(s, nullptr, 0) : dflt;
}

// Bring-up / A-B knobs, read from the environment once (rz_reload_env() reads them again):
//   RZ_TC_CONFIG 1..5 forces a block shape, RZ_TC_NOSPLIT=1 turns contraction splitting off, RZ_TC_EW_STAGES is the
//   longest contraction (stages) that gets the sixteen-warp weight-gradient epilogue, RZ_TC_GROUP the rasterisation
//   group (row tiles), RZ_TC_TMA_STORE=0 plain stores instead of bulk tensor stores, RZ_TC_VERBOSE=1 one line per launch,
//   RZ_TC_UNIT_RANGES=0 keeps fully split launches on nsplit equal parts per block instead of equal stage ranges,
//   RZ_TC_DW_EW2=0 gives the two-row-block weight gradient eight epilogue warps instead of sixteen.
struct Knobs {
    std::atomic<uint32_t> config{0}, no_split{0}, ew_stages{64}, group{0}, tma_store{1}, verbose{0}, unit_ranges{1}, dw_ew2{1};
    std::atomic<bool> ready{false};
};
Knobs g_knobs;

void load_knobs()
{
    g_knobs.config.store(env_u32("RZ_TC_CONFIG", 0));
    g_knobs.no_split.store(env_u32("RZ_TC_NOSPLIT", 0));
    g_knobs.ew_stages.store(env_u32("RZ_TC_EW_STAGES", 64));
    g_knobs.group.store(env_u32("RZ_TC_GROUP", 0));
    g_knobs.tma_store.store(env_u32("RZ_TC_TMA_STORE", 1));
    g_knobs.verbose.store(env_u32("RZ_TC_VERBOSE", 0));
    g_knobs.unit_ranges.store(env_u32("RZ_TC_UNIT_RANGES", 1));
    g_knobs.dw_ew2.store(env_u32("RZ_TC_DW_EW2", 1));
    g_knobs.ready.store(true, std::memory_order_release);
}

const Knobs &knobs()
{
    if (!g_knobs.ready.load(std::memory_order_acquire)) load_knobs();
    return g_knobs;
}

// Block shape of a launch.  (ctas, rb, nc): CTAs per block (2 = cluster pair driving cta_group::2 MMAs), row
// blocks per pair, block columns.  Blocks are rows = 128*ctas*rb by nc.
struct TcConfig {
    int ctas, rb, nc;
    int nsplit;   // parts the contraction of the blocks from n_main on is split into (1 = no block is split)
    int n_main;   // blocks [0, n_main) keep their whole contraction; 0 with nsplit > 1 = every block is split
    int ew;       // epilogue warps per TMEM lane quarter (0 or 1 = one; 4 = weight gradient of a short contraction)
};

// Candidates from the largest block down, with the relative tensor throughput each sustains when the grid
// fills the machine (the wide pair blocks move the fewest L2 bytes per flop; narrow single-CTA blocks are
// L2-bound but keep every SM busy on small grids).
const struct {
    TcConfig cfg;
    double speed;
} kCandidates[] = {
    {{2, 2, 256, 1, 0}, 1.00}, {{2, 1, 256, 1, 0}, 0.80}, {{1, 1, 256, 1, 0}, 0.58}, {{1, 1, 128, 1, 0}, 0.40}, {{1, 1, 64, 1, 0}, 0.25},
};

// Pick the block shape with the best (occupancy of the last wave) x (shape throughput), among the shapes the
// problem allows.  RZ_TC_CONFIG = 1..5 forces one shape (1 = 128x256 single CTA,
// 2 = pair 256x256, 3 = pair 512x256, 4 = single 128x128, 5 = single 128x64).
TcConfig choose_config(const rz_problem *pb, int op)
{
    const bool bf16 = pb->precision == RZ_PREC_BF16;
    const bool split = pb->precision == RZ_PREC_FP32;
    const int64_t rows = (op == RZ_OP_BACKWARD_WEIGHT) ? pb->N : pb->M;   // (weight gradient: transposed block, N x K)
    const int64_t cols = (op == RZ_OP_FORWARD) ? pb->N : pb->K;
    const int64_t depth = (op == RZ_OP_FORWARD) ? pb->K : (op == RZ_OP_BACKWARD_INPUT ? pb->N : pb->M);
    const int64_t stages = (depth + (bf16 ? 63 : 31)) / (bf16 ? 64 : 32);
    const int sms = usable_sms(pb);
    auto allowed = [&](const TcConfig &c) {
        if (split && c.rb == 2) return false;                       // split precision has no two-row-block variant
        // with two row blocks the epilogue cannot overlap the next main loop: the contraction must amortise it
        // (the weight gradient's scatter epilogue is several times as long as a store epilogue; measured: at 32 stages
        // the one-row-block pair with sixteen epilogue warps is 4 % ahead, at 64 stages two row blocks are 6 % ahead)
        if (c.rb == 2 && stages < (op == RZ_OP_BACKWARD_WEIGHT ? 48 : 12)) return false;
        const int64_t bcols = c.nc / c.ctas;                        // whole B boxes per hash tile (input gradient)
        if (op == RZ_OP_BACKWARD_INPUT && (pb->BK <= bcols ? bcols % pb->BK != 0 : pb->BK % bcols != 0)) return false;
        return true;
    };
    // Small grids: split the contraction over several blocks so that every SM has work.  The weight gradient adds
    // its partial blocks straight into the hashed gradient; FWD / DX add fp32 partials into a workspace that a
    // finalize kernel scales and converts (two more small launches, so only contractions of 64 stages or more are
    // split).  At least 16 pipeline stages per part.
    auto split_for = [&](int64_t items, int64_t slots) {
        if (items * 2 > slots) return (int64_t)1;
        if (op != RZ_OP_BACKWARD_WEIGHT && stages < 64) return (int64_t)1;
        int64_t want = slots / items, most = stages / (op == RZ_OP_BACKWARD_WEIGHT ? 8 : 16);
        if (most < 1) most = 1;
        return want < most ? want : most;
    };
    const uint32_t forced = knobs().config.load(std::memory_order_relaxed);
    const bool no_split = knobs().no_split.load(std::memory_order_relaxed) != 0;
    TcConfig best = kCandidates[4].cfg;
    double best_score = -1.0;
    for (int i = 0; i < 5; ++i) {
        const auto &cand = kCandidates[i];
        TcConfig c = cand.cfg;
        if (!allowed(c)) continue;
        const int64_t block_rows = (int64_t)TILE_R * c.ctas * c.rb;
        const int64_t items = ((rows + block_rows - 1) / block_rows) * ((cols + c.nc - 1) / c.nc);
        const int64_t slots = sms / c.ctas;
        if (!no_split) c.nsplit = (int)split_for(items, slots);
        if (split) {   // bound the accumulation chains of split precision: at most 2048 contraction elements per part
            const int64_t need = (depth + 2047) / 2048;
            if (c.nsplit < need) c.nsplit = (int)need;
        }
        // Ragged last wave: the blocks left over after the full waves are split along the contraction, so the tail costs
        // ceil(tail * parts / slots) / parts of a wave instead of a whole one.  Every part pays the block's epilogue
        // again (FWD / DX: fp32 reductions into the workspace, which only those blocks go through, plus the finalize
        // launch; DW: its scatter, which it pays anyway), counted here in pipeline stages.
        const int64_t tail = items % slots;
        double tail_waves = 1.0;   // time of the last wave, in whole-contraction blocks
        if (!no_split && c.nsplit == 1 && items > slots && tail > 0 && stages >= 32) {
            const bool dw = op == RZ_OP_BACKWARD_WEIGHT;
            const double per_part = dw ? (c.rb == 2 ? 19.0 : 4.0) : (c.rb == 2 ? 10.0 : 5.0);
            const double whole = (double)stages + (dw ? per_part : 0.0);
            int64_t best_parts = 1;
            const int64_t most = stages / 8 < 16 ? stages / 8 : 16;
            for (int64_t parts = 2; parts <= most; ++parts) {
                const double t = (double)((tail * parts + slots - 1) / slots) * ((double)stages / (double)parts + per_part) / whole +
                                 (dw ? 0.0 : 0.05);
                if (t < tail_waves - 0.04) {
                    tail_waves = t;
                    best_parts = parts;
                }
            }
            if (best_parts > 1) {
                c.nsplit = (int)best_parts;
                c.n_main = (int)(items - tail);
            }
        }
        // Weight gradient of a short contraction: the scatter epilogue (one reduction per 32 elements, issued by
        // one warp per scheduler) outlasts the main loop; sixteen epilogue warps hide its instruction latency.
        if (op == RZ_OP_BACKWARD_WEIGHT && !split && c.rb == 1 && stages / c.nsplit <= (int64_t)knobs().ew_stages.load(std::memory_order_relaxed))
            c.ew = 4;
        // Two row blocks: the scatter cannot overlap the next block's MMAs, so it should at least be short - sixteen
        // epilogue warps (two per TMEM lane quarter and row block) keep twice as many reductions in flight as eight.
        if (op == RZ_OP_BACKWARD_WEIGHT && !split && c.rb == 2 && knobs().dw_ew2.load(std::memory_order_relaxed)) c.ew = 2;
        if (forced >= 1 && forced <= 5) {
            static const int order[5] = {2, 1, 0, 3, 4};
            if (order[forced - 1] == i) return c;
            continue;
        }
        if (rows < block_rows / 2 && c.ctas * c.rb > 1) continue;   // do not pair CTAs over rows that do not exist
        // time in waves of whole-contraction blocks, against the ideal items / slots
        double waves;
        if (c.nsplit == 1) {
            waves = (double)((items + slots - 1) / slots);
        } else if (c.n_main == 0) {
            waves = (double)((items * c.nsplit + slots - 1) / slots) / c.nsplit + 0.1;
        } else {
            waves = (double)(c.n_main / slots) + tail_waves;
        }
        const double occupancy = ((double)items / (double)slots) / waves;
        // useful fraction of the block (ragged last row block)
        const double fill = (double)rows / (double)(((rows + block_rows - 1) / block_rows) * block_rows);
        const double score = (occupancy > 1.0 ? 1.0 : occupancy) * fill * cand.speed;
        if (score > best_score * 1.02) {   // prefer the larger block on near ties
            best_score = score;
            best = c;
        }
    }
    return best;
}

// fp32 partial-sum workspace a FWD / DX launch with split blocks needs: one block-sized tile per split block
// (0 for whole-contraction launches and for DW, which adds its parts straight into the hashed gradient)
size_t workspace_bytes(const rz_problem *pb, int op)
{
    if (op == RZ_OP_BACKWARD_WEIGHT) return 0;
    const TcConfig c = choose_config(pb, op);
    if (c.nsplit <= 1) return 0;
    const int64_t cols = (op == RZ_OP_BACKWARD_INPUT) ? pb->K : pb->N;
    const int64_t block_rows = (int64_t)TILE_R * c.ctas * c.rb;
    const int64_t items = ((pb->M + block_rows - 1) / block_rows) * ((cols + c.nc - 1) / c.nc);
    return (size_t)(items - c.n_main) * (size_t)block_rows * (size_t)c.nc * sizeof(float);
}

uint32_t dx_box_rows(const rz_problem *pb, const TcConfig &c)
{
    const uint32_t bcols = (uint32_t)(c.nc / c.ctas);
    return (uint32_t)pb->BK < bcols ? (uint32_t)pb->BK : bcols;
}

// FWD: slice rows per B box - a stage's contraction rows, or one hash tile of them when tiles are shorter
uint32_t fwd_box_rows(const rz_problem *pb)
{
    const uint32_t kc = pb->precision == RZ_PREC_BF16 ? 64u : 32u;
    return (uint32_t)pb->BK < kc ? (uint32_t)pb->BK : kc;
}

template <int OP, bool TF32, int CTAS, int RB, int SPLIT, int NC, int EW = 1>
int launch_tc(const RzLaunchCtx &c, const CUtensorMap &mapA, const CUtensorMap &mapB, const CUtensorMap &mapC, TcParams &p,
              const TcConfig &plan)
{
    const rz_problem *pb = c.pb;
    constexpr int ES = TF32 ? 4 : 2;
    constexpr int EPR = 128 / ES;
    constexpr int KC = EPR;
    constexpr int PAIR_R = TILE_R * CTAS;
    constexpr int ITEM_R = PAIR_R * RB;
    constexpr int NTHREADS = num_threads(RB, SPLIT, EW);
    constexpr int STAGES_HOST = num_stages(OP, CTAS, RB, SPLIT, NC, EW);
    p.hash = c.hash;
    p.M = (uint32_t)pb->M;
    p.K = (uint32_t)pb->K;
    p.N = (uint32_t)pb->N;
    p.rows = (OP == OP_DW) ? p.N : p.M;                  // (the weight gradient is computed transposed: N x K)
    p.cols = (OP == OP_FWD) ? p.N : p.K;
    const uint32_t depth = (OP == OP_FWD) ? p.K : (OP == OP_DX ? p.N : p.M);
    p.tiles_r = (p.rows + ITEM_R - 1) / ITEM_R;
    p.tiles_c = (p.cols + NC - 1) / NC;
    p.nchunks = (depth + KC - 1) / KC;
    p.br = OP == OP_FWD ? fwd_box_rows(pb) : dx_box_rows(pb, TcConfig{CTAS, RB, NC});
    p.kparts = KC / fwd_box_rows(pb);
    p.group_rows = knobs().group.load(std::memory_order_relaxed);
    if (p.group_rows < 1) p.group_rows = GROUP_ROWS / RB;

    auto kern = rz_tc_kernel<OP, TF32, CTAS, RB, SPLIT, NC, EW>;
    constexpr int SMEM_TOTAL = smem_total(OP, CTAS, RB, SPLIT, NC, EW);
    static_assert(SMEM_TOTAL <= SMEM_LIMIT, "shared memory budget");
    // Per kernel variant and device, once: the shared-memory opt-in and (pairs) how many clusters fit the device.
    // Both are properties of the variant, and asking the runtime again on every call costs several microseconds
    // of host time, which is what small problems are bound by.
    static std::atomic<int> ready[64];   // 0 = not set up, else resident blocks / pairs + 1
    int dev = 0;
    int st = rz_record_cuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (st) return st;
    const bool cacheable = dev >= 0 && dev < 64;
    int known = cacheable ? ready[dev].load(std::memory_order_acquire) : 0;
    if (!known) {
        st = rz_record_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_TOTAL),
                            "set max dynamic shared memory");
        if (st) return st;
    }

    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr[1];
    cfg.blockDim = dim3(NTHREADS, 1, 1);
    cfg.dynamicSmemBytes = SMEM_TOTAL;
    cfg.stream = c.stream;
    cfg.numAttrs = 0;
    // number of blocks (CTAS = 1) or CTA pairs (CTAS = 2) that can be resident at once
    int slots = num_sms() / CTAS;
    if (CTAS == 2) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(2 * (unsigned)slots, 1, 1);
        if (known) {
            slots = known - 1;
        } else {
            int clusters = 0;
            if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) == cudaSuccess && clusters > 0 && clusters < slots)
                slots = clusters;
            (void)cudaGetLastError();
        }
    }
    if (!known && cacheable) ready[dev].store(slots + 1, std::memory_order_release);
    if (pb->sm_reserve > 0) {   // leave SMs idle for whatever the caller runs beside this kernel
        slots -= (pb->sm_reserve + CTAS - 1) / CTAS;
        if (slots < 1) slots = 1;
    }

    const uint32_t tiles = p.tiles_r * p.tiles_c;
    p.nsplit = plan.nsplit > 1 ? (uint32_t)plan.nsplit : 1u;
    p.n_main = plan.nsplit > 1 ? (uint32_t)plan.n_main : tiles;
    if (OP != OP_DW && !p.ws) p.nsplit = 1, p.n_main = tiles;   // no workspace given: whole contraction per block
    if (p.n_main > tiles) p.n_main = tiles;
    if (p.nsplit > p.nchunks) p.nsplit = p.nchunks;
    p.chunks_per_split = (p.nchunks + p.nsplit - 1) / p.nsplit;
    p.nsplit = (p.nchunks + p.chunks_per_split - 1) / p.chunks_per_split;
    if (p.nsplit <= 1) p.nsplit = 1, p.n_main = tiles;
    p.total_items = p.n_main + (tiles - p.n_main) * p.nsplit;
    p.alpha = pb->alpha;
    p.relu = (pb->flags & RZ_FLAG_RELU) ? 1 : 0;
    st = rz_wait_context(&p.wait, 2000000000ll);   // also refuses to launch behind a kernel whose wait gave up
    if (st) return st;
    p.tma_store = knobs().tma_store.load(std::memory_order_relaxed);

    // shared-memory descriptors (bytes)
    const uint32_t atom = KC * 128;
    const uint32_t mn_sbo = TF32 ? 512 : 1024;        // tf32 M/N-major: rows group by 4 (32-byte-chunk swizzle)
    const uint32_t mn_layout = TF32 ? 1 : 2;
    p.a_layout = p.b_layout = 2;
    if (OP == OP_FWD) {
        p.a_lbo = 16, p.a_sbo = 1024;             // K-major
        p.b_lbo = atom, p.b_sbo = mn_sbo;   // N-major
        p.b_layout = mn_layout;
    } else if (OP == OP_DX) {
        p.a_lbo = 16, p.a_sbo = 1024;
        p.b_lbo = 16, p.b_sbo = 1024;
    } else {
        p.a_lbo = atom, p.a_sbo = mn_sbo;
        p.b_lbo = atom, p.b_sbo = mn_sbo;
        p.a_layout = p.b_layout = mn_layout;
    }
    const uint32_t a_major = (OP == OP_DW) ? 1u : 0u, b_major = (OP == OP_DX) ? 0u : 1u;
    const uint32_t fmt = TF32 ? 2u : 1u;
    p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (a_major << 15) | (b_major << 16) | ((uint32_t)(NC >> 3) << 17) |
              ((uint32_t)(PAIR_R >> 4) << 24);

    uint32_t blocks = p.total_items < (uint32_t)slots ? p.total_items : (uint32_t)slots;
    // Small grids whose every block is split anyway (FWD / DX): deal the (block, stage) units out in equal ranges
    // instead of nsplit equal parts per block, so that every SM works whatever the number of blocks (40 blocks in
    // 3 parts keep 120 of 148 SMs busy; 148 ranges keep them all).  Not for split precision, whose parts also
    // bound the accumulation chains.
    p.units = 0;
    if (OP != OP_DW && !SPLIT && p.nsplit > 1 && p.n_main == 0 && knobs().unit_ranges.load(std::memory_order_relaxed)) {
        const uint32_t units = tiles * p.nchunks;
        uint32_t ranges = units / 8 < (uint32_t)slots ? units / 8 : (uint32_t)slots;   // at least 8 stages per range
        if (ranges > blocks) {
            p.units = units;
            blocks = ranges;
        }
    }
    if (knobs().verbose.load(std::memory_order_relaxed))   // bring-up aid: one line per launch on stderr
        fprintf(stderr, "rz_tc op %d tf32 %d block (%d,%d,%d) ew %d stages %d: %u blocks, %u whole + %u x %u parts, %d slots, %u units in %u ranges\n", OP,
                (int)TF32, CTAS, RB, NC, EW, STAGES_HOST, tiles, p.n_main, tiles - p.n_main, p.nsplit, slots, p.units, p.units ? blocks : 0u);
    cfg.gridDim = dim3(blocks * CTAS, 1, 1);
    const bool partial = OP != OP_DW && p.nsplit > 1;
    const uint32_t split_tiles = tiles - p.n_main;
    if (partial) {
        st = rz_record_cuda(cudaMemsetAsync(p.ws, 0, sizeof(float) * (size_t)split_tiles * ITEM_R * NC, c.stream),
                            "zero workspace");
        if (st) return st;
    }
    st = rz_record_cuda(cudaLaunchKernelEx(&cfg, kern, mapA, mapB, mapC, p), "tcgen05 kernel launch");
    rz_count_launch(1);
    if (st) return st;
    st = rz_record_cuda(cudaGetLastError(), "tcgen05 kernel launch");
    if (st || !partial) return st;
    FinalizeGeom fg;
    fg.rows = p.rows, fg.cols = p.cols, fg.item_r = ITEM_R, fg.nc = NC, fg.tiles_r = p.tiles_r, fg.tiles_c = p.tiles_c;
    fg.group_rows = p.group_rows, fg.n_main = p.n_main, fg.n_tiles = tiles;
    // about four CTAs per SM in total, several per block when few blocks were split
    unsigned per_tile = (148u * 4u + split_tiles - 1) / split_tiles;
    if (per_tile > 32u) per_tile = 32u;
    const dim3 fblocks(split_tiles < 148u * 4u ? split_tiles : 148u * 4u, per_tile, 1);
    const float *fbias = OP == OP_FWD ? p.bias : nullptr;   // bias and ReLU belong to the forward pass only
    const int frelu = OP == OP_FWD ? p.relu : 0;
    if (TF32)
        rz_finalize_kernel<float><<<fblocks, 256, 0, c.stream>>>(p.ws, (float *)p.out, fbias, fg, p.alpha, frelu);
    else
        rz_finalize_kernel<__nv_bfloat16><<<fblocks, 256, 0, c.stream>>>(p.ws, (__nv_bfloat16 *)p.out, fbias, fg, p.alpha, frelu);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "finalize launch");
}

template <int OP>
int launch_tc_any(const RzLaunchCtx &c, const CUtensorMap &mapA, const CUtensorMap &mapB, const CUtensorMap &mapC, TcParams &p,
                  const TcConfig &cfg)
{
    const int prec = c.pb->precision;
    if (prec == RZ_PREC_FP32) {   // split precision: fp32 operands, three tf32 MMAs per product
        if (cfg.ctas == 2) return launch_tc<OP, true, 2, 1, 1, 256>(c, mapA, mapB, mapC, p, cfg);
        if (cfg.nc == 256) return launch_tc<OP, true, 1, 1, 1, 256>(c, mapA, mapB, mapC, p, cfg);
        if (cfg.nc == 128) return launch_tc<OP, true, 1, 1, 1, 128>(c, mapA, mapB, mapC, p, cfg);
        return launch_tc<OP, true, 1, 1, 1, 64>(c, mapA, mapB, mapC, p, cfg);
    }
    const bool tf32 = prec == RZ_PREC_TF32;
    if (OP == OP_DW && cfg.ew == 4 && cfg.rb == 1) {   // scatter-bound weight gradient: sixteen epilogue warps
        constexpr int W = (OP == OP_DW) ? 4 : 1;       // (keeps the other operations from instantiating the variant)
        if (cfg.ctas == 2)
            return tf32 ? launch_tc<OP, true, 2, 1, 0, 256, W>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 2, 1, 0, 256, W>(c, mapA, mapB, mapC, p, cfg);
        if (cfg.nc == 256)
            return tf32 ? launch_tc<OP, true, 1, 1, 0, 256, W>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 1, 1, 0, 256, W>(c, mapA, mapB, mapC, p, cfg);
        if (cfg.nc == 128)
            return tf32 ? launch_tc<OP, true, 1, 1, 0, 128, W>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 1, 1, 0, 128, W>(c, mapA, mapB, mapC, p, cfg);
        return tf32 ? launch_tc<OP, true, 1, 1, 0, 64, W>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 1, 1, 0, 64, W>(c, mapA, mapB, mapC, p, cfg);
    }
    if (OP == OP_DW && cfg.ctas == 2 && cfg.rb == 2 && cfg.ew == 2) {
        constexpr int W = (OP == OP_DW) ? 2 : 1;
        return tf32 ? launch_tc<OP, true, 2, 2, 0, 256, W>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 2, 2, 0, 256, W>(c, mapA, mapB, mapC, p, cfg);
    }
    if (cfg.ctas == 2 && cfg.rb == 2)
        return tf32 ? launch_tc<OP, true, 2, 2, 0, 256>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 2, 2, 0, 256>(c, mapA, mapB, mapC, p, cfg);
    if (cfg.ctas == 2)
        return tf32 ? launch_tc<OP, true, 2, 1, 0, 256>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 2, 1, 0, 256>(c, mapA, mapB, mapC, p, cfg);
    if (cfg.nc == 256)
        return tf32 ? launch_tc<OP, true, 1, 1, 0, 256>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 1, 1, 0, 256>(c, mapA, mapB, mapC, p, cfg);
    if (cfg.nc == 128)
        return tf32 ? launch_tc<OP, true, 1, 1, 0, 128>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 1, 1, 0, 128>(c, mapA, mapB, mapC, p, cfg);
    return tf32 ? launch_tc<OP, true, 1, 1, 0, 64>(c, mapA, mapB, mapC, p, cfg) : launch_tc<OP, false, 1, 1, 0, 64>(c, mapA, mapB, mapC, p, cfg);
}

}  // namespace

namespace rztc {

int forced_shape()
{
    static const int order[5] = {2, 1, 0, 3, 4};   // RZ_TC_CONFIG 1..5 -> index of kCandidates
    const uint32_t forced = knobs().config.load(std::memory_order_relaxed);
    return forced >= 1 && forced <= 5 ? order[forced - 1] : -1;
}

// 2-D map over a row-major matrix [rows][cols] of the operand type
int map_matrix(CUtensorMap *map, bool tf32, int mn_major, const void *base, uint64_t rows, uint64_t cols,
               uint32_t box_cols, uint32_t box_rows, bool keep)
{
    const int es = tf32 ? 4 : 2;
    uint64_t dims[2] = {cols, rows};
    uint64_t strides[1] = {cols * (uint64_t)es};
    uint32_t box[2] = {box_cols, box_rows};
    return encode(map, tf32, mn_major, const_cast<void *>(base), 2, dims, strides, box, keep);
}

// 3-D map over the shadow: {element of a copy, slice row (stride BN elements), copy}
int map_shadow(CUtensorMap *map, const rz_problem *pb, bool mn_major, const void *shadow, uint32_t box_rows, bool keep)
{
    const Geometry g = geometry(pb);
    const bool tf32 = pb->precision != RZ_PREC_BF16;
    uint64_t dims[3] = {g.Hc, (uint64_t)pb->BK, (uint64_t)g.ns};
    uint64_t strides[2] = {(uint64_t)pb->BN * g.es, (uint64_t)g.copy_stride};
    uint32_t box[3] = {(uint32_t)g.epr, box_rows, 1};
    return encode(map, tf32, mn_major, const_cast<void *>(shadow), 3, dims, strides, box, keep);
}

}  // namespace rztc

int rz_tc_wait_selftest(long long limit_cycles, cudaStream_t stream)
{
    RzWaitCtx w;
    int st = rz_wait_context(&w, limit_cycles);
    if (st) return st;
    rz_wait_selftest_kernel<<<1, 32, 0, stream>>>(w);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "wait self-test launch");
}

bool rz_tc_supported(const rz_problem *pb, int op)
{
    (void)op;
    const Geometry g = geometry(pb);
    // a 128-byte operand row must lie inside one hash tile along n; along k a pipeline stage (one such row of
    // contraction elements) is made of whole hash tiles or lies inside one, and tiles are multiples of the 32 rows
    // an epilogue warp scatters
    if (pb->BN % g.epr || pb->BK % 32) return false;
    if (pb->BK < g.epr ? (g.epr % pb->BK != 0) : (pb->BK % g.epr != 0)) return false;
    if (pb->BK <= 64 ? (64 % pb->BK != 0) : (pb->BK % 64 != 0)) return false;   // whole B boxes per hash tile (narrowest block)
    if ((pb->K * g.es) % 16 || (pb->N * g.es) % 16) return false;
    if (pb->K < g.epr || pb->N < g.epr) return false;   // at least one full 128-byte row of every operand
    return true;
}

size_t rz_tc_copies_bytes(const rz_problem *pb)
{
    const Geometry g = geometry(pb);
    return g.copy_stride * (size_t)g.ns;
}

size_t rz_tc_shadow_bytes(const rz_problem *pb)
{
    // the shifted copies, then the fp32 workspace of split-contraction launches (forward and input gradient share it)
    const size_t wf = workspace_bytes(pb, RZ_OP_FORWARD), wi = workspace_bytes(pb, RZ_OP_BACKWARD_INPUT);
    return rz_tc_copies_bytes(pb) + (wf > wi ? wf : wi);
}

bool rz_tc_needs_workspace(const rz_problem *pb, int op)
{
    // split precision bounds its accumulation chains by splitting long contractions: that launch cannot do without
    if (pb->precision != RZ_PREC_FP32 || op == RZ_OP_BACKWARD_WEIGHT) return false;
    return (op == RZ_OP_FORWARD ? pb->K : pb->N) > 2048;
}

void rz_tc_reload_env() { load_knobs(); }

// Workspace of a launch inside the caller's scratch: behind the copies, if the scratch is large enough to hold it
// (a scratch that only holds the copies makes the launch run every block's whole contraction instead).
static int workspace_of(const rz_problem *pb, void *shadow, size_t shadow_bytes, int op, float **ws)
{
    *ws = nullptr;
    const size_t need = workspace_bytes(pb, op), copies = rz_tc_copies_bytes(pb);
    if (shadow_bytes < copies) return RZ_ERR_SCRATCH;
    if (need == 0) return RZ_OK;
    if (shadow_bytes >= copies + need)
        *ws = reinterpret_cast<float *>(static_cast<uint8_t *>(shadow) + copies);
    else if (rz_tc_needs_workspace(pb, op))
        return RZ_ERR_SCRATCH;
    return RZ_OK;
}

int rz_tc_shadow_refresh(const RzLaunchCtx &c, const float *hashed, void *shadow)
{
    const Geometry g = geometry(c.pb);
    const uint32_t groups = g.Hc / g.ns;
    uint32_t blocks = (groups + 255) / 256;
    if (blocks > 148 * 8) blocks = 148 * 8;
    if (c.pb->precision != RZ_PREC_BF16)
        rz_shadow_kernel<true><<<blocks, 256, 0, c.stream>>>(hashed, (uint8_t *)shadow, (uint32_t)c.pb->H, g.Hc, g.copy_stride,
                                                            c.pb->precision == RZ_PREC_FP32 ? 1 : 0);
    else
        rz_shadow_kernel<false><<<blocks, 256, 0, c.stream>>>(hashed, (uint8_t *)shadow, (uint32_t)c.pb->H, g.Hc, g.copy_stride, 0);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "shadow refresh launch");
}

int rz_tc_sgd_step(const RzLaunchCtx &c, float *hashed, const float *dH, float *velocity, float lr, float momentum, void *shadow)
{
    const uint32_t H = (uint32_t)c.pb->H;
    if (!shadow) {   // no tensor-core scratch to keep in step: the update alone
        uint32_t blocks = velocity ? (H + 255) / 256 : (H / 4 + 255) / 256;
        if (blocks < 1) blocks = 1;
        if (blocks > 148 * 8) blocks = 148 * 8;
        if (velocity) rz_sgd_momentum_kernel<<<blocks, 256, 0, c.stream>>>(hashed, dH, velocity, lr, momentum, H);
        else rz_sgd_kernel<<<blocks, 256, 0, c.stream>>>(hashed, dH, lr, H);
        rz_count_launch(1);
        return rz_record_cuda(cudaGetLastError(), "sgd launch");
    }
    // update + shadow refresh in one pass; each launch in flight draws its own ticket word
    static std::atomic<unsigned> next_ticket{0};
    const unsigned slot = next_ticket.fetch_add(1, std::memory_order_relaxed) % SGD_TICKETS;
    unsigned *ticket = nullptr;
    int st = rz_record_cuda(cudaGetSymbolAddress(reinterpret_cast<void **>(&ticket), g_sgd_ticket), "ticket address");
    if (st) return st;
    ticket += slot;
    const Geometry g = geometry(c.pb);
    const uint32_t groups = g.Hc / g.ns;
    uint32_t blocks = (groups + SGD_CHUNK - 1) / SGD_CHUNK;
    if (blocks > 148 * 2) blocks = 148 * 2;
    const bool tf32 = c.pb->precision != RZ_PREC_BF16;
    const int raw = c.pb->precision == RZ_PREC_FP32 ? 1 : 0;
    uint8_t *sh = static_cast<uint8_t *>(shadow);
    if (tf32 && velocity)
        rz_sgd_shadow_kernel<true, true><<<blocks, SGD_CHUNK, 0, c.stream>>>(hashed, dH, velocity, lr, momentum, sh, H, g.Hc, g.copy_stride, raw, ticket);
    else if (tf32)
        rz_sgd_shadow_kernel<true, false><<<blocks, SGD_CHUNK, 0, c.stream>>>(hashed, dH, nullptr, lr, 0.f, sh, H, g.Hc, g.copy_stride, raw, ticket);
    else if (velocity)
        rz_sgd_shadow_kernel<false, true><<<blocks, SGD_CHUNK, 0, c.stream>>>(hashed, dH, velocity, lr, momentum, sh, H, g.Hc, g.copy_stride, 0, ticket);
    else
        rz_sgd_shadow_kernel<false, false><<<blocks, SGD_CHUNK, 0, c.stream>>>(hashed, dH, nullptr, lr, 0.f, sh, H, g.Hc, g.copy_stride, 0, ticket);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "sgd + shadow launch");
}

int rz_tc_forward(const RzLaunchCtx &c, const void *X, void *shadow, size_t shadow_bytes, const float *bias, void *Y)
{
    const rz_problem *pb = c.pb;
    const bool tf32 = pb->precision != RZ_PREC_BF16;
    const Geometry g = geometry(pb);
    TcParams p;
    memset(&p, 0, sizeof(p));
    p.bias = bias;
    p.out = Y;
    int st = workspace_of(pb, shadow, shadow_bytes, RZ_OP_FORWARD, &p.ws);
    if (st) return st;
    CUtensorMap mapA, mapB;
    st = map_matrix(&mapA, tf32, false, X, pb->M, pb->K, g.epr, TILE_R);
    if (st) return st;
    st = map_shadow(&mapB, pb, true, shadow, fwd_box_rows(pb));
    if (st) return st;
    // output map for the epilogue's bulk stores: 32-row x 128-byte boxes
    CUtensorMap mapC;
    st = map_matrix(&mapC, tf32, false, Y, pb->M, pb->N, g.epr, 32);
    if (st) return st;
    return launch_tc_any<OP_FWD>(c, mapA, mapB, mapC, p, choose_config(pb, RZ_OP_FORWARD));
}

int rz_tc_backward_input(const RzLaunchCtx &c, const void *dY, void *shadow, size_t shadow_bytes, void *dX)
{
    const rz_problem *pb = c.pb;
    const bool tf32 = pb->precision != RZ_PREC_BF16;
    const Geometry g = geometry(pb);
    TcParams p;
    memset(&p, 0, sizeof(p));
    p.out = dX;
    int st = workspace_of(pb, shadow, shadow_bytes, RZ_OP_BACKWARD_INPUT, &p.ws);
    if (st) return st;
    CUtensorMap mapA, mapB;
    st = map_matrix(&mapA, tf32, false, dY, pb->M, pb->N, g.epr, TILE_R);
    if (st) return st;
    const TcConfig config = choose_config(pb, RZ_OP_BACKWARD_INPUT);
    st = map_shadow(&mapB, pb, false, shadow, dx_box_rows(pb, config));
    if (st) return st;
    CUtensorMap mapC;
    st = map_matrix(&mapC, tf32, false, dX, pb->M, pb->K, g.epr, 32);
    if (st) return st;
    return launch_tc_any<OP_DX>(c, mapA, mapB, mapC, p, config);
}

int rz_tc_backward_weight(const RzLaunchCtx &c, const void *X, const void *dY, float *dH)
{
    const rz_problem *pb = c.pb;
    const bool tf32 = pb->precision != RZ_PREC_BF16;
    const Geometry g = geometry(pb);
    CUtensorMap mapA, mapB;   // A = dY (accumulator rows = n), B = X (accumulator columns = k)
    int st = map_matrix(&mapA, tf32, true, dY, pb->M, pb->N, g.epr, g.epr);
    if (st) return st;
    st = map_matrix(&mapB, tf32, true, X, pb->M, pb->K, g.epr, g.epr);
    if (st) return st;
    TcParams p;
    memset(&p, 0, sizeof(p));
    p.dH = dH;
    return launch_tc_any<OP_DW>(c, mapA, mapB, mapA, p, choose_config(pb, RZ_OP_BACKWARD_WEIGHT));   // (no output map)
}
