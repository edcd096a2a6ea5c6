// Rows picked by an index: stable counting sort of row keys, embedding lookup in a virtual table, and the lookup's
// gradient by sorted tokens.
//
// The table is a virtual weight W[V, D] like any other of this library: row k is cut into segments of BN columns, and
// segment pn of row k is the contiguous run of words  hashed[ off(k / BK, pn) + (k % BK) * BN ... + BN ).
//
// Every kernel here is bound by memory or by the reductions into the hashed gradient, so they are plain SIMT kernels: what
// matters is that every request is a full 128-byte line of consecutive words, that a hash (about 60 integer instructions) is
// computed by 32 lanes for 32 segments at once, and that few launches are made.
#include "rz_common.h"

namespace {

constexpr uint32_t FULL = 0xffffffffu;

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void store_pair(float *p, float a, float b) { *reinterpret_cast<float2 *>(p) = make_float2(a, b); }
__device__ __forceinline__ void store_pair(__nv_bfloat16 *p, float a, float b) { *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(a, b); }

// A token that selects a row of the table: inside [0, V) and not the padding row.
__device__ __forceinline__ bool live_id(int64_t id, uint32_t V, int64_t padding) { return id >= 0 && id < (int64_t)V && id != padding; }

// ---- stable counting sort ---------------------------------------------------------------------------------------------
// order = row numbers by ascending key, equal keys by ascending row; offsets[b] = rows whose key is below b.  Keys outside
// [0, bins) form one more bin behind the last.  A block owns a contiguous range of tiles of SORT_TILE rows, so the sort is
// two launches whatever the length: block histograms, then every block sums the histograms before its own (148 blocks at
// most: 148 x 1025 words out of L2) and places its rows; up to one tile a single launch does both.  Within a tile the
// warps own consecutive pieces and count their keys in a table of their own: a row's place is the count of equal keys in
// earlier blocks, earlier tiles, earlier warps, earlier steps of its warp and lower lanes of its step - an exact, and so
// reproducible, rank without any atomic on a shared counter.
constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32, SORT_ITEMS = 4;
constexpr int SORT_TILE = SORT_THREADS * SORT_ITEMS;
constexpr int SORT_MAX_BINS = 1024, SORT_MAX_BLOCKS = 148;

__device__ __forceinline__ uint32_t sort_bin(const int64_t *__restrict__ keys, uint32_t row, uint32_t bins)
{
    const int64_t k = keys[row];
    return (k >= 0 && k < (int64_t)bins) ? (uint32_t)k : bins;
}

__global__ void __launch_bounds__(SORT_THREADS)
rz_sort_count_kernel(const int64_t *__restrict__ keys, uint32_t rows, uint32_t bins, uint32_t rows_per_block,
                     uint32_t *__restrict__ hist)
{
    __shared__ uint32_t count[SORT_MAX_BINS + 1];
    for (uint32_t b = threadIdx.x; b <= bins; b += SORT_THREADS) count[b] = 0;
    __syncthreads();
    const uint32_t lo = blockIdx.x * rows_per_block, hi = min(rows, lo + rows_per_block);
    for (uint32_t r = lo + threadIdx.x; r < hi; r += SORT_THREADS) atomicAdd(&count[sort_bin(keys, r, bins)], 1u);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b <= bins; b += SORT_THREADS) hist[(size_t)blockIdx.x * (bins + 1) + b] = count[b];
}

// exclusive prefix sum over the block of one value per thread, plus the total
__device__ __forceinline__ uint32_t block_exclusive_scan(uint32_t v, uint32_t *warp_sums, uint32_t nwarps, uint32_t *total)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(FULL, x, d);
        if (lane >= (uint32_t)d) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = lane < nwarps ? warp_sums[lane] : 0u;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t y = __shfl_up_sync(FULL, s, d);
            if (lane >= (uint32_t)d) s += y;
        }
        if (lane < nwarps) warp_sums[lane] = s;
    }
    __syncthreads();
    const uint32_t before = warp ? warp_sums[warp - 1] : 0u;
    *total = warp_sums[nwarps - 1];
    __syncthreads();
    return before + x - v;
}

// `hist` NULL: one block, one tile.
__global__ void __launch_bounds__(SORT_THREADS)
rz_sort_place_kernel(const int64_t *__restrict__ keys, uint32_t rows, uint32_t bins, uint32_t rows_per_block,
                     const uint32_t *__restrict__ hist, int32_t *__restrict__ order, int32_t *__restrict__ offsets)
{
    extern __shared__ uint32_t sort_smem[];
    __shared__ uint32_t warp_sums[SORT_WARPS];
    const uint32_t nb = bins + 1;
    uint32_t *base = sort_smem;            // [nb] where the block's next row of a bin goes
    uint32_t *count = sort_smem + nb;      // [SORT_WARPS][nb]
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t lo = blockIdx.x * rows_per_block, hi = min(rows, lo + rows_per_block);

    if (hist) {
        uint32_t carry = 0;
        for (uint32_t b0 = 0; b0 < nb; b0 += SORT_THREADS) {
            const uint32_t b = b0 + threadIdx.x;
            uint32_t mine = 0, all = 0;
            if (b < nb) {
#pragma unroll 8
                for (uint32_t k = 0; k < gridDim.x; ++k) {
                    const uint32_t v = hist[(size_t)k * nb + b];
                    all += v;
                    if (k < blockIdx.x) mine += v;
                }
            }
            uint32_t total;
            const uint32_t before = block_exclusive_scan(all, warp_sums, SORT_WARPS, &total) + carry;
            carry += total;
            if (b < nb) {
                base[b] = before + mine;
                if (blockIdx.x == 0) offsets[b] = (int32_t)before;
            }
        }
    }

    for (uint32_t t0 = lo; t0 < hi; t0 += SORT_TILE) {
        for (uint32_t i = threadIdx.x; i < SORT_WARPS * nb; i += SORT_THREADS) count[i] = 0;
        uint32_t bin[SORT_ITEMS], rank[SORT_ITEMS];
        const uint32_t first = t0 + warp * (32 * SORT_ITEMS) + lane;
#pragma unroll
        for (int j = 0; j < SORT_ITEMS; ++j) bin[j] = first + j * 32 < hi ? sort_bin(keys, first + j * 32, bins) : FULL;
        __syncthreads();
        uint32_t *mine = count + warp * nb;
#pragma unroll
        for (int j = 0; j < SORT_ITEMS; ++j) {
            const uint32_t same = __match_any_sync(FULL, bin[j]);
            const uint32_t leader = __ffs(same) - 1;
            uint32_t old = 0;
            if (lane == leader && bin[j] != FULL) {
                old = mine[bin[j]];
                mine[bin[j]] = old + __popc(same);
            }
            rank[j] = __shfl_sync(FULL, old, leader) + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
        }
        __syncthreads();
        // counts of the warps -> where each warp's first row of a bin goes
        uint32_t carry = 0;
        for (uint32_t b0 = 0; b0 < nb; b0 += SORT_THREADS) {
            const uint32_t b = b0 + threadIdx.x;
            uint32_t sum = 0;
            if (b < nb) {
#pragma unroll
                for (int w = 0; w < SORT_WARPS; ++w) {
                    const uint32_t v = count[w * nb + b];
                    count[w * nb + b] = sum;
                    sum += v;
                }
            }
            if (hist) {
                if (b < nb) {
                    const uint32_t at = base[b];
                    base[b] = at + sum;
#pragma unroll
                    for (int w = 0; w < SORT_WARPS; ++w) count[w * nb + b] += at;
                }
            } else {
                uint32_t total;
                const uint32_t at = block_exclusive_scan(sum, warp_sums, SORT_WARPS, &total) + carry;
                carry += total;
                if (b < nb) {
                    offsets[b] = (int32_t)at;
#pragma unroll
                    for (int w = 0; w < SORT_WARPS; ++w) count[w * nb + b] += at;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SORT_ITEMS; ++j)
            if (bin[j] != FULL) order[mine[bin[j]] + rank[j]] = (int32_t)(first + j * 32);
        __syncthreads();
    }
    if (!hist && rows == 0)   // nothing to sort: all bins are empty
        for (uint32_t b = threadIdx.x; b < nb; b += SORT_THREADS) offsets[b] = 0;
}

// ---- embedding lookup -------------------------------------------------------------------------------------------------
// out[t, :] = alpha * W[ids[t], :], zeros for a token that selects no row.  The (token, segment) pairs are numbered token by
// token; a warp takes `per_warp` consecutive ones, its lanes hash one each, then the warp copies the segments one after
// the other, two words a lane (PAIRS: rows and segments of an even number of words, the output aligned for pairs).
// A slice starts at any word, so the reads are 4-byte loads that L1 joins; the stores are whole lines.
template <typename T, bool PAIRS>
__global__ void __launch_bounds__(256)
rz_embedding_kernel(const int64_t *__restrict__ ids, int64_t padding, const float *__restrict__ hashed, T *__restrict__ out,
                    RzHash hash, uint64_t total, uint32_t V, uint32_t D, uint32_t nn, uint32_t per_warp, float alpha)
{
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t stride = (uint64_t)gridDim.x * (blockDim.x / 32) * per_warp;
    const uint32_t BN = (uint32_t)hash.BN, BK = (uint32_t)hash.BK;
    for (uint64_t u0 = ((uint64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5)) * per_warp; u0 < total; u0 += stride) {
        const uint32_t n = (uint32_t)min((uint64_t)per_warp, total - u0);
        uint64_t src = 0, dst = 0;
        uint32_t len = 0;
        bool live = false;
        if (lane < n) {
            const uint64_t u = u0 + lane, t = u / nn;
            const uint32_t pn = (uint32_t)(u - t * nn);
            const int64_t id = ids[t];
            live = live_id(id, V, padding);
            dst = t * D + (uint64_t)pn * BN;
            len = min(BN, D - pn * BN);
            if (live) {
                const uint32_t k = (uint32_t)id, pk = k / BK;
                src = rz_tile_offset(hash, pk, pn) + (uint64_t)(k - pk * BK) * BN;
            }
        }
#pragma unroll 4
        for (uint32_t j = 0; j < n; ++j) {
            const uint64_t s = __shfl_sync(FULL, src, j), d = __shfl_sync(FULL, dst, j);
            const uint32_t m = __shfl_sync(FULL, len, j);
            const bool l = __shfl_sync(FULL, (int)live, j) != 0;
            if (PAIRS) {
                for (uint32_t c = 2 * lane; c < m; c += 64) {
                    const float a = l ? __ldg(hashed + s + c) * alpha : 0.f, b = l ? __ldg(hashed + s + c + 1) * alpha : 0.f;
                    store_pair(out + d + c, a, b);
                }
            } else {
                for (uint32_t c = lane; c < m; c += 32) out[d + c] = from_f32<T>(l ? __ldg(hashed + s + c) * alpha : 0.f);
            }
        }
    }
}

// ---- embedding gradient -----------------------------------------------------------------------------------------------
// dH[word of (k, n)] += alpha * sum over the tokens t with ids[t] = k of dOut[t, n].
//
// A token that occurs often would add the same words over and over, and reductions (1.3e12 a second at best, whatever their
// width) cost more than reading: 2 bytes at 6.5 TB/s are 3.3e12 elements a second.  So chunks of the batch are sorted by
// token first, runs of one token are summed in registers in 32 bits, and one reduction per word and run is made.  Sorting
// within chunks is one launch, needs no exchange between blocks and finds nearly all repetitions (a token that returns in
// another chunk costs one more reduction per word).
constexpr int CHUNK_THREADS = 1024, CHUNK_WARPS = 32;

template <int ITEMS>
__global__ void __launch_bounds__(CHUNK_THREADS)
rz_token_sort_kernel(const int64_t *__restrict__ ids, int64_t padding, uint32_t T, uint32_t V, int passes,
                     uint32_t *__restrict__ sorted_id, uint32_t *__restrict__ sorted_row)
{
    constexpr uint32_t CHUNK = CHUNK_THREADS * ITEMS;
    extern __shared__ __align__(16) uint8_t chunk_smem[];
    uint32_t *skey = reinterpret_cast<uint32_t *>(chunk_smem);                    // [CHUNK]
    uint32_t *count = skey + CHUNK;                                               // [CHUNK_WARPS][256]
    uint16_t *spos = reinterpret_cast<uint16_t *>(count + CHUNK_WARPS * 256);     // [CHUNK]
    __shared__ uint32_t warp_sums[32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t begin = blockIdx.x * CHUNK, valid = min(CHUNK, T - begin);
    const uint32_t first = warp * (32 * ITEMS) + lane;
    uint32_t key[ITEMS], pos[ITEMS], rank[ITEMS];
    // tokens without a row get key V: they go behind all others; slots behind the batch go behind those
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const uint32_t i = first + j * 32;
        pos[j] = i;
        key[j] = FULL;
        if (i < valid) {
            const int64_t id = ids[begin + i];
            key[j] = live_id(id, V, padding) ? (uint32_t)id : V;
        }
    }
    uint32_t *mine = count + warp * 256;
    for (int p = 0; p < passes; ++p) {
        for (uint32_t i = threadIdx.x; i < CHUNK_WARPS * 256; i += CHUNK_THREADS) count[i] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const uint32_t d = (key[j] >> (8 * p)) & 255u;
            const uint32_t same = __match_any_sync(FULL, d);
            const uint32_t leader = __ffs(same) - 1;
            uint32_t old = 0;
            if (lane == leader) {
                old = mine[d];
                mine[d] = old + __popc(same);
            }
            rank[j] = __shfl_sync(FULL, old, leader) + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
        }
        __syncthreads();
        uint32_t sum = 0;
        if (threadIdx.x < 256) {
#pragma unroll 8
            for (int w = 0; w < CHUNK_WARPS; ++w) {
                const uint32_t v = count[w * 256 + threadIdx.x];
                count[w * 256 + threadIdx.x] = sum;
                sum += v;
            }
        }
        uint32_t total;
        const uint32_t at = block_exclusive_scan(sum, warp_sums, CHUNK_WARPS, &total);
        if (threadIdx.x < 256) {
#pragma unroll 8
            for (int w = 0; w < CHUNK_WARPS; ++w) count[w * 256 + threadIdx.x] += at;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const uint32_t dst = mine[(key[j] >> (8 * p)) & 255u] + rank[j];
            skey[dst] = key[j];
            spos[dst] = (uint16_t)pos[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            key[j] = skey[first + j * 32];
            pos[j] = spos[first + j * 32];
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const uint32_t i = first + j * 32;
        if (i < valid) {
            sorted_id[begin + i] = key[j];
            sorted_row[begin + i] = begin + pos[j];
        }
    }
}

// A warp takes 32 consecutive places of the sorted batch and 64 columns: lane l sums columns c0 + l and c0 + 32 + l, so that a
// reduction instruction covers 32 consecutive words.  ALIGNED (BN a multiple of 32): each half lies in one segment, and
// lane i hashes place i's segments for the whole warp; otherwise every lane hashes its own columns at the end of a run.
// PACKED (bf16, even rows): one 4-byte load brings columns c0 + 2l and c0 + 2l + 1, exchanged between the lanes at the end of a
// run.  `sorted_id` NULL: places are the tokens themselves (batches too short to be worth sorting).
template <typename T, bool ALIGNED, bool PACKED>
__global__ void __launch_bounds__(256)
rz_embedding_grad_kernel(const int64_t *__restrict__ ids, int64_t padding, const uint32_t *__restrict__ sorted_id,
                         const uint32_t *__restrict__ sorted_row, const T *__restrict__ dout, float *__restrict__ dH, RzHash hash,
                         uint32_t T_, uint32_t V, uint32_t D, uint32_t colblocks, uint64_t units, float alpha)
{
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t unit = (uint64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    if (unit >= units) return;
    const uint32_t pb = (uint32_t)(unit / colblocks), cb = (uint32_t)(unit - (uint64_t)pb * colblocks);
    const uint32_t BN = (uint32_t)hash.BN, BK = (uint32_t)hash.BK;
    const uint32_t c0 = cb * 64, colA = c0 + lane, colB = colA + 32;
    const uint32_t place = pb * 32 + lane;

    uint32_t id = V, row = 0;
    if (place < T_) {
        if (sorted_id) {
            id = sorted_id[place];
            row = sorted_row[place];
        } else {
            const int64_t v = ids[place];
            id = live_id(v, V, padding) ? (uint32_t)v : V;
            row = place;
        }
    }
    const uint32_t live = __ballot_sync(FULL, id < V);
    if (!live) return;
    const uint32_t pk = id / BK, k_in = id - pk * BK;
    // where the words of this lane's place begin: of columns [c0, c0 + 32) and [c0 + 32, c0 + 64)
    uint32_t dstA = 0, dstB = 0;
    if (ALIGNED) {
        const uint32_t pnA = c0 / BN, pnB = (c0 + 32) / BN;
        if (id < V) {
            const uint32_t offA = (uint32_t)rz_tile_offset(hash, pk, pnA);
            const uint32_t offB = pnB == pnA || c0 + 32 >= D ? offA : (uint32_t)rz_tile_offset(hash, pk, pnB);
            dstA = offA + k_in * BN + (c0 - pnA * BN);
            dstB = offB + k_in * BN + (c0 + 32 - pnB * BN);
        }
    }
    const uint32_t next = __shfl_down_sync(FULL, id, 1);
    const uint32_t ends = __ballot_sync(FULL, lane == 31 || next != id);   // last place of each run

    float a = 0.f, b = 0.f;
    constexpr int U = 8;
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += U) {
        if (((live >> i0) & ((1u << U) - 1u)) == 0) continue;
        float va[U], vb[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t r = __shfl_sync(FULL, row, i0 + i);
            const T *src = dout + (size_t)r * D;
            va[i] = vb[i] = 0.f;
            if (!((live >> (i0 + i)) & 1u)) continue;
            if (PACKED) {
                if (c0 + 2 * lane < D) {
                    const uint32_t w = __ldg(reinterpret_cast<const uint32_t *>(src + c0) + lane);
                    va[i] = __uint_as_float(w << 16), vb[i] = __uint_as_float(w & 0xffff0000u);
                }
            } else {
                if (colA < D) va[i] = to_f32<T>(src[colA]);
                if (colB < D) vb[i] = to_f32<T>(src[colB]);
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            a += va[i], b += vb[i];
            if (!((ends >> (i0 + i)) & 1u)) continue;
            if ((live >> (i0 + i)) & 1u) {
                float x = a, y = b;
                if (PACKED) {   // columns 2l, 2l + 1 -> l, 32 + l
                    const uint32_t h = lane >> 1;
                    const float xa = __shfl_sync(FULL, a, h), xb = __shfl_sync(FULL, b, h);
                    const float ya = __shfl_sync(FULL, a, 16 + h), yb = __shfl_sync(FULL, b, 16 + h);
                    x = (lane & 1) ? xb : xa, y = (lane & 1) ? yb : ya;
                }
                if (ALIGNED) {
                    const uint32_t dA = __shfl_sync(FULL, dstA, i0 + i), dB = __shfl_sync(FULL, dstB, i0 + i);
                    if (colA < D) atomicAdd(dH + dA + lane, x * alpha);
                    if (colB < D) atomicAdd(dH + dB + lane, y * alpha);
                } else {
                    const uint32_t k = __shfl_sync(FULL, id, i0 + i), tk = k / BK, kin = k - tk * BK;
                    if (colA < D) {
                        const uint32_t pn = colA / BN;
                        atomicAdd(dH + rz_tile_offset(hash, tk, pn) + (uint64_t)kin * BN + (colA - pn * BN), x * alpha);
                    }
                    if (colB < D) {
                        const uint32_t pn = colB / BN;
                        atomicAdd(dH + rz_tile_offset(hash, tk, pn) + (uint64_t)kin * BN + (colB - pn * BN), y * alpha);
                    }
                }
            }
            a = b = 0.f;
        }
    }
}

// Batches up to this length are not sorted: one launch less, and few repetitions to find.
constexpr int64_t UNSORTED_TOKENS = 256;

template <int ITEMS>
int launch_token_sort(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, int passes, uint32_t *sid, uint32_t *srow)
{
    constexpr uint32_t CHUNK = CHUNK_THREADS * ITEMS;
    constexpr int SMEM = CHUNK * 4 + CHUNK_WARPS * 256 * 4 + CHUNK * 2;
    const uint32_t T = (uint32_t)c.pb->M;
    int st = rz_record_cuda(cudaFuncSetAttribute(rz_token_sort_kernel<ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM),
                            "set max dynamic shared memory");
    if (st) return st;
    rz_token_sort_kernel<ITEMS><<<(T + CHUNK - 1) / CHUNK, CHUNK_THREADS, SMEM, c.stream>>>(ids, padding, T, (uint32_t)c.pb->K, passes,
                                                                                         sid, srow);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "token sort launch");
}

template <typename T>
int launch_embedding(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const float *hashed, void *out)
{
    const rz_problem *pb = c.pb;
    const uint32_t D = (uint32_t)pb->N, nn = (D + pb->BN - 1) / (uint32_t)pb->BN;
    const uint64_t total = (uint64_t)pb->M * nn;
    // segments per warp: 32 (one hash evaluation for 32 of them) once that leaves enough warps, fewer for short batches
    uint32_t per_warp = 32;
    while (per_warp > 1 && total / per_warp < 148 * 32) per_warp >>= 1;
    const uint64_t warps = (total + per_warp - 1) / per_warp;
    uint64_t blocks = (warps + 7) / 8;
    if (blocks > 148 * 64) blocks = 148 * 64;
    const bool pairs = D % 2 == 0 && pb->BN % 2 == 0 && (reinterpret_cast<uintptr_t>(out) & (2 * sizeof(T) - 1)) == 0;
    if (pairs)
        rz_embedding_kernel<T, true><<<(unsigned)blocks, 256, 0, c.stream>>>(ids, padding, hashed, (T *)out, c.hash, total,
                                                                            (uint32_t)pb->K, D, nn, per_warp, pb->alpha);
    else
        rz_embedding_kernel<T, false><<<(unsigned)blocks, 256, 0, c.stream>>>(ids, padding, hashed, (T *)out, c.hash, total,
                                                                             (uint32_t)pb->K, D, nn, per_warp, pb->alpha);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "embedding launch");
}

template <typename T>
int launch_embedding_grad(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const uint32_t *sid, const uint32_t *srow,
                          const void *dout, float *dH)
{
    const rz_problem *pb = c.pb;
    const uint32_t D = (uint32_t)pb->N, M = (uint32_t)pb->M;
    const uint32_t colblocks = (D + 63) / 64;
    const uint64_t units = (uint64_t)((M + 31) / 32) * colblocks, blocks = (units + 7) / 8;
    if (blocks > 0x7fffffffull) return RZ_ERR_SHAPE;
    const bool aligned = pb->BN % 32 == 0;
    const bool packed = sizeof(T) == 2 && D % 2 == 0 && (reinterpret_cast<uintptr_t>(dout) & 3u) == 0;
    auto run = [&](auto kernel) {
        kernel<<<(unsigned)blocks, 256, 0, c.stream>>>(ids, padding, sid, srow, (const T *)dout, dH, c.hash, M, (uint32_t)pb->K, D,
                                                       colblocks, units, pb->alpha);
    };
    constexpr bool P = sizeof(T) == 2;   // (the packed load exists for 2-byte elements only)
    if (aligned && packed) run(rz_embedding_grad_kernel<T, true, P>);
    else if (aligned) run(rz_embedding_grad_kernel<T, true, false>);
    else if (packed) run(rz_embedding_grad_kernel<T, false, P>);
    else run(rz_embedding_grad_kernel<T, false, false>);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "embedding gradient launch");
}

uint32_t sort_blocks(int64_t rows, uint32_t *rows_per_block)
{
    const uint64_t tiles = ((uint64_t)rows + SORT_TILE - 1) / SORT_TILE;
    uint64_t blocks = tiles < SORT_MAX_BLOCKS ? tiles : SORT_MAX_BLOCKS;
    if (blocks < 1) blocks = 1;
    const uint64_t per = (tiles + blocks - 1) / blocks;
    *rows_per_block = (uint32_t)(per * SORT_TILE);
    return (uint32_t)((tiles + per - 1) / (per ? per : 1));
}

}  // namespace

size_t rz_rows_sort_scratch(int64_t rows, int64_t bins)
{
    uint32_t per = 0;
    const uint32_t blocks = rows > 0 ? sort_blocks(rows, &per) : 1;
    return blocks <= 1 ? 0 : sizeof(uint32_t) * (size_t)blocks * (size_t)(bins + 1);
}

int rz_rows_sort_max_bins() { return SORT_MAX_BINS; }

int rz_rows_sort(const int64_t *keys, int64_t rows, int64_t bins, int32_t *order, int32_t *offsets, void *scratch, cudaStream_t stream)
{
    uint32_t per = SORT_TILE;
    const uint32_t blocks = rows > 0 ? sort_blocks(rows, &per) : 1;
    uint32_t *hist = blocks > 1 ? static_cast<uint32_t *>(scratch) : nullptr;
    const int smem = (int)(sizeof(uint32_t) * (SORT_WARPS + 1) * (size_t)(bins + 1));
    int st = rz_record_cuda(cudaFuncSetAttribute(rz_sort_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)(sizeof(uint32_t) * (SORT_WARPS + 1) * (SORT_MAX_BINS + 1))),
                            "set max dynamic shared memory");
    if (st) return st;
    if (hist) {
        rz_sort_count_kernel<<<blocks, SORT_THREADS, 0, stream>>>(keys, (uint32_t)rows, (uint32_t)bins, per, hist);
        rz_count_launch(1);
    }
    rz_sort_place_kernel<<<blocks, SORT_THREADS, smem, stream>>>(keys, (uint32_t)rows, (uint32_t)bins, per, hist, order, offsets);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "row sort launch");
}

int rz_rows_embedding(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const float *hashed, void *out)
{
    if (c.pb->io_dtype == RZ_BF16) return launch_embedding<__nv_bfloat16>(c, ids, padding, hashed, out);
    return launch_embedding<float>(c, ids, padding, hashed, out);
}

size_t rz_rows_embedding_scratch(const rz_problem *pb) { return pb->M <= UNSORTED_TOKENS ? 0 : sizeof(uint32_t) * 2 * (size_t)pb->M; }

int rz_rows_embedding_grad(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const void *dout, float *dH, void *scratch)
{
    const rz_problem *pb = c.pb;
    uint32_t *sid = nullptr, *srow = nullptr;
    if (pb->M > UNSORTED_TOKENS) {
        sid = static_cast<uint32_t *>(scratch);
        srow = sid + pb->M;
        int bits = 1;   // of the largest key, V
        while (bits < 32 && (pb->K >> bits)) ++bits;
        const int passes = (bits + 7) / 8;
        const int st = pb->M <= CHUNK_THREADS * 2   ? launch_token_sort<2>(c, ids, padding, passes, sid, srow)
                       : pb->M <= CHUNK_THREADS * 4 ? launch_token_sort<4>(c, ids, padding, passes, sid, srow)
                                                    : launch_token_sort<8>(c, ids, padding, passes, sid, srow);
        if (st) return st;
    }
    if (pb->io_dtype == RZ_BF16) return launch_embedding_grad<__nv_bfloat16>(c, ids, padding, sid, srow, dout, dH);
    return launch_embedding_grad<float>(c, ids, padding, sid, srow, dout, dH);
}
