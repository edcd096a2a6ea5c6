// Rows picked by an index: stable counting sort of row keys, embedding lookup in a virtual table, and the lookup's gradient,
// token by token.
//
// The table is a virtual weight W[V, D] like any other of this library: row k is cut into segments of BN columns, and
// segment pn of row k is the contiguous run of words  hashed[ off(k / BK, pn) + (k % BK) * BN ... + BN ).
//
// Every kernel here is bound by memory or by the reductions into the hashed gradient, so they are plain SIMT kernels: what
// matters is that every request is a full 128-byte line of consecutive words, that a hash (about 60 integer instructions) is
// computed by 32 lanes for 32 segments at once, and that few launches are made.
#include <atomic>
#include <cstring>
#include <type_traits>

#include "rz_common.h"
#include "rz_ptx.cuh"

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

__device__ __forceinline__ void red_pair(float *p, float a, float b)
{
    asm volatile("red.global.add.v2.f32 [%0], {%1, %2};" ::"l"(p), "f"(a), "f"(b) : "memory");
}

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
constexpr int SORT_MAX_BINS = RZ_SORT_MAX_BINS, SORT_MAX_BLOCKS = 148;

// Lanes whose `bits` low key bits equal this lane's, one vote per bit.
__device__ __forceinline__ uint32_t same_key(uint32_t key, int bits)
{
    uint32_t same = FULL;
    for (int b = 0; b < bits; ++b) {
        const uint32_t set = __ballot_sync(FULL, (key >> b) & 1u);
        same &= (key >> b) & 1u ? set : ~set;
    }
    return same;
}

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
                     int bits, const uint32_t *__restrict__ hist, int32_t *__restrict__ order, int32_t *__restrict__ offsets)
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
            const uint32_t same = same_key(bin[j], bits);   // (`bits` hold every bin, and a value for the slots behind the rows)
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
                    RzHash hash, RzHash32 hash32, uint64_t total, uint32_t V, uint32_t D, uint32_t nn, uint32_t per_warp, float alpha)
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
                src = rz_tile_offset32(hash, hash32, pk, pn) + (uint64_t)(k - pk * BK) * BN;
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
    // a token sort may run beside this kernel: the grid ends after it does.  (One block waits; if all did, the ones not yet
    // started would wait for those that had finished.)
    if (blockIdx.x == 0) rzptx::grid_wait();
}

// The same for hash tiles and rows of whole 64-word pieces: a unit is 64 words, so every unit is full, its place in the output
// is its number, and what the copy loop fetches from the hashing lane is one 32-bit word.  What bounds it is issue: the two 4-byte
// loads of a pair that may begin at an odd word, a shuffle and a store for every 64 words.  8192 x 4096 bf16 (31 MB read from
// DRAM, 67 MB written): 22.7 us, 28.8 without the loop of its own for 32 live units; 16384 x 4096: 41 us.
template <typename T>
__global__ void __launch_bounds__(256)
rz_embedding_pieces_kernel(const int64_t *__restrict__ ids, int64_t padding, const float *__restrict__ hashed, T *__restrict__ out,
                           RzHash hash, RzHash32 hash32, uint64_t total, uint32_t V, uint32_t per_row, uint32_t per_warp, float alpha)
{
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t stride = (uint64_t)gridDim.x * (blockDim.x / 32) * per_warp;
    const uint32_t BN = (uint32_t)hash.BN, BK = (uint32_t)hash.BK;
    for (uint64_t u0 = ((uint64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5)) * per_warp; u0 < total; u0 += stride) {
        const uint32_t n = (uint32_t)min((uint64_t)per_warp, total - u0);
        uint32_t src = FULL;   // (no word has this number)
        if (lane < n) {
            const uint64_t u = u0 + lane;
            // (a 64-bit division takes as long as copying four pieces)
            const uint64_t t = total <= FULL ? (uint32_t)u / per_row : u / per_row;
            const uint32_t col = (uint32_t)(u - t * per_row) * 64, pn = col / BN;
            const int64_t id = ids[t];
            if (live_id(id, V, padding)) {
                const uint32_t k = (uint32_t)id, pk = k / BK;
                src = rz_tile_offset32(hash, hash32, pk, pn) + (k - pk * BK) * BN + (col - pn * BN);
            }
        }
        T *dst = out + u0 * 64 + 2 * lane;
        const float *const words = hashed + 2 * lane;
        constexpr int U = 8;
        if (n == 32 && __all_sync(FULL, src != FULL)) {
#pragma unroll 1
            for (uint32_t j0 = 0; j0 < 32; j0 += U, dst += U * 64) {
                float a[U], b[U];
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    const float *w = words + __shfl_sync(FULL, src, j0 + j);
                    a[j] = __ldg(w), b[j] = __ldg(w + 1);
                }
#pragma unroll
                for (int j = 0; j < U; ++j) store_pair(dst + j * 64, a[j] * alpha, b[j] * alpha);
            }
            continue;
        }
        for (uint32_t j0 = 0; j0 < n; j0 += U) {
            float a[U], b[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const uint32_t s = __shfl_sync(FULL, src, j0 + j);   // (lanes from n on hold FULL)
                a[j] = b[j] = 0.f;
                if (s != FULL) a[j] = __ldg(words + s), b[j] = __ldg(words + s + 1);
            }
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (j0 + j < n) store_pair(dst + (size_t)(j0 + j) * 64, a[j] * alpha, b[j] * alpha);
        }
    }
    // a token sort may run beside this kernel: the grid ends after it does.  (One block waits; if all did, the ones not yet
    // started would wait for those that had finished.)
    if (blockIdx.x == 0) rzptx::grid_wait();
}

// ---- embedding gradient -----------------------------------------------------------------------------------------------
// dH[word of (k, n)] += alpha * sum over the tokens t with ids[t] = k of dOut[t, n].
//
// A token that occurs often would add the same words over and over, and reductions (0.9 to 1.08e12 words a second at rows of 64 words in
// random places, whatever the instruction's width) cost more than reading: 2 bytes at 6.5 TB/s are 3.3e12 elements a second.  So the tokens are brought together first: runs
// of one token are then summed in registers in 32 bits, and one reduction per word and run is made.
//
// One CTA sorts a chunk of up to 16384 tokens (least significant digits first, digits of up to 8 bits, ranks from votes; a warp-wide
// match instruction takes some 180 cycles of the SM), which finds nearly all repetitions: a token that returns in another chunk
// costs one more reduction per word.  The sort is slow - 17 us for 8192 tokens, all latency - but needs nothing of the gradient, so the
// forward call makes it, on a few SMs beside the lookup, which takes the others.
// (Instead, one launch in the backward: a cluster of eight CTAs counting chunks of 32768 tokens in a hash table in its shared memory
// took 31 us for 16384 tokens, a table in L2 19 us and, for 131072 tokens, 112 us.)
constexpr int CHUNK_THREADS = 1024, CHUNK_WARPS = 32;

template <int ITEMS>
__global__ void __launch_bounds__(CHUNK_THREADS)
rz_token_sort_kernel(const int64_t *__restrict__ ids, int64_t padding, uint32_t T, uint32_t V, int passes, int width,
                     uint32_t *__restrict__ sorted_id, uint32_t *__restrict__ sorted_row)
{
    constexpr uint32_t CHUNK = CHUNK_THREADS * ITEMS;
    extern __shared__ __align__(16) uint8_t chunk_smem[];
    uint32_t *skey = reinterpret_cast<uint32_t *>(chunk_smem);                    // [CHUNK]
    uint32_t *count = skey + CHUNK;                                               // [CHUNK_WARPS][256]
    uint16_t *spos = reinterpret_cast<uint16_t *>(count + CHUNK_WARPS * 256);     // [CHUNK]
    __shared__ uint32_t warp_sums[32];
    rzptx::grid_launch_dependents();   // the lookup runs beside this kernel, and waits for it at its end
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1u << width;
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
            const uint32_t d = (key[j] >> (width * p)) & (digits - 1u);
            const uint32_t same = same_key(d, width);
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
        if (threadIdx.x < digits) {
#pragma unroll 8
            for (int w = 0; w < CHUNK_WARPS; ++w) {
                const uint32_t v = count[w * 256 + threadIdx.x];
                count[w * 256 + threadIdx.x] = sum;
                sum += v;
            }
        }
        uint32_t total;
        const uint32_t at = block_exclusive_scan(sum, warp_sums, CHUNK_WARPS, &total);
        if (threadIdx.x < digits) {
#pragma unroll 8
            for (int w = 0; w < CHUNK_WARPS; ++w) count[w * 256 + threadIdx.x] += at;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const uint32_t dst = mine[(key[j] >> (width * p)) & (digits - 1u)] + rank[j];
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

// The 32 places of the sorted batch that a warp works on: lane i holds place i's table row and row of dOut.
struct Places {
    uint32_t id, row, live, ends;   // (live, ends: masks over the places; ends = last place of a run of one token)
};

// `sorted_id` NULL: places are the tokens themselves (batches too short to be worth sorting).
__device__ __forceinline__ Places load_places(const int64_t *__restrict__ ids, int64_t padding, const uint32_t *__restrict__ sorted_id,
                                              const uint32_t *__restrict__ sorted_row, uint32_t block, uint32_t T, uint32_t V)
{
    const uint32_t lane = threadIdx.x & 31, place = block * 32 + lane;
    Places p;
    p.id = V, p.row = 0;
    if (place < T) {
        if (sorted_id) {
            p.id = sorted_id[place];
            p.row = sorted_row[place];
        } else {
            const int64_t v = ids[place];
            p.id = live_id(v, V, padding) ? (uint32_t)v : V;
            p.row = place;
        }
    }
    p.live = __ballot_sync(FULL, p.id < V);
    const uint32_t next = __shfl_down_sync(FULL, p.id, 1);
    p.ends = __ballot_sync(FULL, lane == 31 || next != p.id);
    return p;
}

// Two neighbouring elements as they are loaded, and their values.
template <typename T> struct Pair;
template <> struct Pair<float> {
    float2 v = make_float2(0.f, 0.f);
    __device__ __forceinline__ void load(const float *p) { v = __ldg(reinterpret_cast<const float2 *>(p)); }
    __device__ __forceinline__ float first() const { return v.x; }
    __device__ __forceinline__ float second() const { return v.y; }
};
template <> struct Pair<__nv_bfloat16> {
    uint32_t v = 0;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { v = __ldg(reinterpret_cast<const uint32_t *>(p)); }
    __device__ __forceinline__ float first() const { return __uint_as_float(v << 16); }
    __device__ __forceinline__ float second() const { return __uint_as_float(v & 0xffff0000u); }
};

// Whole hash-tile columns of 32 and rows of pairs: a warp takes 32 places and S pieces of 64 columns, lane l columns 2l and 2l + 1 of
// each piece (one load).  The words of a piece are consecutive (WHOLE: hash tiles of 64 columns and their multiples), or those of
// either half of it are, and begin anywhere: where they begin at an even word the pairs are reduced as they are, elsewhere each
// lane takes its left neighbour's second value and the first and the last word go alone.  Lane i hashes place i's tiles for the
// whole warp.  What a place costs by itself - its row, its tests - is shared by S pieces.
// 16384 x 4096 bf16, 9 in 10 tokens live, text: 43 us with S = 2 in blocks of 128 threads; 50 with S = 1 and 53 with S = 4 (blocks
// of 256: 54).  With neither reductions nor reads from DRAM it takes 40 with S = 4: latency bounds it, since the loads of the next U places
// are issued behind the reductions of these.  The 22 M words it adds (5400 runs) would take 21 us at 1.06e12 a second, the 121 MB it
// reads 20 us, and 47 % of the issue slots are used.
constexpr int GRAD_THREADS = 128;

template <typename T, int S, bool WHOLE>
__global__ void __launch_bounds__(GRAD_THREADS)
rz_embedding_grad_pairs_kernel(const int64_t *__restrict__ ids, int64_t padding, const uint32_t *__restrict__ sorted_id,
                               const uint32_t *__restrict__ sorted_row, const T *__restrict__ dout, float *__restrict__ dH, RzHash hash, RzHash32 hash32,
                               uint32_t T_, uint32_t V, uint32_t D, uint32_t colblocks, uint64_t units, float alpha)
{
    constexpr int RUNS = WHOLE ? 1 : 2, LANES = 32 / RUNS;   // runs of consecutive words in a piece, lanes of one
    const uint32_t lane = threadIdx.x & 31, run = lane / LANES, in_run = lane % LANES;
    const uint64_t unit = (uint64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    if (unit >= units) return;
    const uint32_t block = (uint32_t)(unit / colblocks), c0 = (uint32_t)(unit - (uint64_t)block * colblocks) * (64 * S);
    const uint32_t BN = (uint32_t)hash.BN, BK = (uint32_t)hash.BK;
    const Places p = load_places(ids, padding, sorted_id, sorted_row, block, T_, V);
    if (!p.live) return;
    uint32_t dst[S][RUNS];   // first word of this lane's place in each run
    {
        const uint32_t pk = p.id / BK, k_in = p.id - pk * BK;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int r = 0; r < RUNS; ++r) {
                const uint32_t col = c0 + s * 64 + r * 32, pn = col / BN;
                dst[s][r] = p.id < V && col < D ? rz_tile_offset32(hash, hash32, pk, pn) + k_in * BN + (col - pn * BN) : 0u;
            }
    }
    const T *src = dout + c0 + 2 * lane;
    float *const base = dH + 2 * in_run;
    float a[S], b[S];
#pragma unroll
    for (int s = 0; s < S; ++s) a[s] = b[s] = 0.f;
    constexpr int U = S * sizeof(T) >= 16 ? 4 : 8;   // places whose loads are in flight together

    // ALL: all 64 S columns exist, and all 32 places have a token
    auto add_places = [&](auto all) {
        constexpr bool ALL = decltype(all)::value;
#pragma unroll 1
        for (int i0 = 0; i0 < 32; i0 += U) {
            const uint32_t live = p.live >> i0, ends = p.ends >> i0;
            if (!ALL && (live & ((1u << U) - 1u)) == 0) continue;
            Pair<T> v[U][S];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const T *at = src + (size_t)__shfl_sync(FULL, p.row, i0 + i) * D;
                if (ALL || ((live >> i) & 1u)) {
#pragma unroll
                    for (int s = 0; s < S; ++s)
                        if (ALL || c0 + s * 64 + 2 * lane < D) v[i][s].load(at + s * 64);   // (rows are pairs)
                }
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
#pragma unroll
                for (int s = 0; s < S; ++s) a[s] += v[i][s].first(), b[s] += v[i][s].second();
                if (!((ends >> i) & 1u)) continue;
                if (ALL || ((live >> i) & 1u)) {
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        if (!ALL && c0 + s * 64 >= D) break;
                        uint32_t d = __shfl_sync(FULL, dst[s][0], i0 + i);
                        if (!WHOLE) {
                            const uint32_t d1 = __shfl_sync(FULL, dst[s][RUNS - 1], i0 + i);
                            if (run) d = d1;
                        }
                        // columns of this run that exist
                        const uint32_t col = c0 + s * 64 + run * 32;
                        const uint32_t width = ALL ? 2 * LANES : min(D - min(col, D), 2u * LANES);
                        float *word = base + d;
                        const float x = a[s] * alpha, y = b[s] * alpha;
                        if (WHOLE ? (d & 1u) : __any_sync(0xffffffffu, d & 1u)) {
                            const float left = __shfl_up_sync(FULL, y, 1);
                            const bool odd = d & 1u, first = in_run == 0, last = 2 * in_run + 2 == width;
                            if (2 * in_run < width && !(odd && first)) red_pair(word - odd, odd ? left : x, odd ? x : y);
                            if (odd && width && (first || last)) atomicAdd(word + !first, first ? x : y);
                            if (odd && first && last) atomicAdd(word + 1, y);   // (a run of two columns)
                        } else if (ALL || 2 * in_run < width) {
                            red_pair(word, x, y);
                        }
                    }
                }
#pragma unroll
                for (int s = 0; s < S; ++s) a[s] = b[s] = 0.f;
            }
        }
    };
    if (c0 + 64 * S <= D && p.live == FULL) add_places(std::true_type());
    else add_places(std::false_type());
}

// Any hash tile, row length and alignment: a warp takes 32 places and up to 64 columns of one segment, lane l columns l and 32 + l of
// them, so that a reduction instruction covers 32 consecutive words.
template <typename T>
__global__ void __launch_bounds__(GRAD_THREADS)
rz_embedding_grad_kernel(const int64_t *__restrict__ ids, int64_t padding, const uint32_t *__restrict__ sorted_id,
                         const uint32_t *__restrict__ sorted_row, const T *__restrict__ dout, float *__restrict__ dH, RzHash hash, RzHash32 hash32,
                         uint32_t T_, uint32_t V, uint32_t D, uint32_t colblocks, uint64_t units, float alpha)
{
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t unit = (uint64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    if (unit >= units) return;
    const uint32_t block = (uint32_t)(unit / colblocks), cb = (uint32_t)(unit - (uint64_t)block * colblocks);
    const uint32_t BN = (uint32_t)hash.BN, BK = (uint32_t)hash.BK;
    const uint32_t per_segment = (BN + 63) / 64, pn = cb / per_segment, in_segment = (cb - pn * per_segment) * 64;
    const uint32_t end = min(BN, D - pn * BN);   // columns of the segment that exist
    if (in_segment >= end) return;
    const Places p = load_places(ids, padding, sorted_id, sorted_row, block, T_, V);
    if (!p.live) return;
    uint32_t dst = 0;
    if (p.id < V) {
        const uint32_t pk = p.id / BK, k_in = p.id - pk * BK;
        dst = rz_tile_offset32(hash, hash32, pk, pn) + k_in * BN + in_segment;
    }
    const bool has_a = in_segment + lane < end, has_b = in_segment + lane + 32 < end;
    const T *src = dout + (size_t)pn * BN + in_segment + lane;
    float a = 0.f, b = 0.f;
    constexpr int U = 8;
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += U) {
        const uint32_t live = p.live >> i0, ends = p.ends >> i0;
        if ((live & ((1u << U) - 1u)) == 0) continue;
        float va[U], vb[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t r = __shfl_sync(FULL, p.row, i0 + i);
            const T *at = src + (size_t)r * D;
            va[i] = vb[i] = 0.f;
            if ((live >> i) & 1u) {
                if (has_a) va[i] = to_f32<T>(at[0]);
                if (has_b) vb[i] = to_f32<T>(at[32]);
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            a += va[i], b += vb[i];
            if (!((ends >> i) & 1u)) continue;
            if ((live >> i) & 1u) {
                float *word = dH + __shfl_sync(FULL, dst, i0 + i) + lane;
                if (has_a) atomicAdd(word, a * alpha);
                if (has_b) atomicAdd(word + 32, b * alpha);
            }
            a = b = 0.f;
        }
    }
}

// The shared-memory opt-in of a kernel, once per device.
template <auto Kernel>
int allow_smem(int bytes)
{
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    int st = rz_record_cuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (st) return st;
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return RZ_OK;
    st = rz_record_cuda(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "set max dynamic shared memory");
    if (st) return st;
    done.fetch_or(bit, std::memory_order_release);
    return RZ_OK;
}

// Which batches are sorted: those with more than 2^22 words to add, where the sort saves more than the 4 us of reductions that it
// costs the host to launch it (1777 x 1000 fp32, lookup and gradient: 117 us of host time with it, 105 without; on the device the
// gradient takes 7 us either way).  Unsorted, 2^22 words bf16 take 13 to 17 us, clearing dH included, with one token alone (a warp joins
// the 32 places it sees), text or all tokens distinct (28 us for text in rows of 64 words), and at worst, two tokens in alternation,
// 20 us in rows of 4096 words, 29 in rows of 1024, 153 in rows of 64.
bool sorts_tokens(const rz_problem *pb) { return pb->M > 256 && pb->M * pb->N > (int64_t)1 << 22; }

// Where a plan (the caller's buffer) has the sorted tokens; NULL for batches that are not sorted.
struct SortedTokens {
    uint32_t *id = nullptr, *row = nullptr;
    SortedTokens(const rz_problem *pb, void *plan)
    {
        if (!plan || !sorts_tokens(pb)) return;
        id = static_cast<uint32_t *>(plan);
        row = id + pb->M;
    }
};

template <int ITEMS>
int launch_token_sort(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const SortedTokens &sorted)
{
    constexpr uint32_t CHUNK = CHUNK_THREADS * ITEMS;
    constexpr int SMEM = CHUNK * 4 + CHUNK_WARPS * 256 * 4 + CHUNK * 2;
    const uint32_t T = (uint32_t)c.pb->M;
    int bits = 1;   // of the largest key, K
    while (bits < 32 && (c.pb->K >> bits)) ++bits;
    const int passes = (bits + 7) / 8, width = (bits + passes - 1) / passes;
    const int st = allow_smem<rz_token_sort_kernel<ITEMS>>(SMEM);
    if (st) return st;
    rz_token_sort_kernel<ITEMS><<<(T + CHUNK - 1) / CHUNK, CHUNK_THREADS, SMEM, c.stream>>>(ids, padding, T, (uint32_t)c.pb->K, passes, width,
                                                                                         sorted.id, sorted.row);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "token sort launch");
}

int sort_tokens(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const SortedTokens &sorted)
{
    // the longest chunks whose sort (about 2.2 us for each 1024 tokens) the lookup hides, going by its bytes
    const rz_problem *pb = c.pb;
    const double lookup_us = (double)pb->M * (double)pb->N * (pb->io_dtype == RZ_BF16 ? 6.0 : 8.0) / 6e6;
    if (pb->M > CHUNK_THREADS * 8 && lookup_us > 40.0) return launch_token_sort<16>(c, ids, padding, sorted);
    if (pb->M > CHUNK_THREADS * 4 && lookup_us > 20.0) return launch_token_sort<8>(c, ids, padding, sorted);
    if (pb->M > CHUNK_THREADS * 2) return launch_token_sort<4>(c, ids, padding, sorted);
    return launch_token_sort<2>(c, ids, padding, sorted);
}

RzHash32 table_hash(const RzLaunchCtx &c)
{
    const rz_problem *pb = c.pb;
    return rz_hash32(c.hash, (uint64_t)(pb->K + pb->BK - 1) / pb->BK, (uint64_t)(pb->N + pb->BN - 1) / pb->BN);
}

template <typename T>
int launch_embedding(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const float *hashed, void *out_, bool beside)
{
    const rz_problem *pb = c.pb;
    T *out = static_cast<T *>(out_);
    const uint32_t V = (uint32_t)pb->K, D = (uint32_t)pb->N, nn = (D + pb->BN - 1) / (uint32_t)pb->BN;
    const RzHash32 hash32 = table_hash(c);
    const bool aligned = (reinterpret_cast<uintptr_t>(out) & (2 * sizeof(T) - 1)) == 0;
    const bool pieces = aligned && D % 64 == 0 && pb->BN % 64 == 0;
    const uint64_t total = (uint64_t)pb->M * (pieces ? D / 64 : nn);
    // segments per warp: 32 (one hash evaluation for 32 of them) once that leaves enough warps, fewer for short batches
    uint32_t per_warp = 32;
    while (per_warp > 1 && total / per_warp < 148 * 32) per_warp >>= 1;
    const uint64_t warps = (total + per_warp - 1) / per_warp;
    uint64_t blocks = (warps + 7) / 8;
    if (blocks > 148 * 64) blocks = 148 * 64;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = c.stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = beside ? 1 : 0;   // start while the token sort launched before runs
    cudaError_t e;
    if (pieces)
        e = cudaLaunchKernelEx(&cfg, rz_embedding_pieces_kernel<T>, ids, padding, hashed, out, c.hash, hash32, total, V, D / 64, per_warp, pb->alpha);
    else if (aligned && D % 2 == 0 && pb->BN % 2 == 0)
        e = cudaLaunchKernelEx(&cfg, rz_embedding_kernel<T, true>, ids, padding, hashed, out, c.hash, hash32, total, V, D, nn, per_warp, pb->alpha);
    else
        e = cudaLaunchKernelEx(&cfg, rz_embedding_kernel<T, false>, ids, padding, hashed, out, c.hash, hash32, total, V, D, nn, per_warp, pb->alpha);
    rz_count_launch(1);
    return rz_record_cuda(e, "embedding launch");
}

template <typename T>
int launch_embedding_grad(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const SortedTokens &sorted, const void *dout,
                          float *dH)
{
    const rz_problem *pb = c.pb;
    const uint32_t D = (uint32_t)pb->N, M = (uint32_t)pb->M, BN = (uint32_t)pb->BN;
    const bool pairs = BN % 32 == 0 && D % 2 == 0 && (reinterpret_cast<uintptr_t>(dout) & (2 * sizeof(T) - 1)) == 0 &&
                       (reinterpret_cast<uintptr_t>(dH) & 7u) == 0;
    const RzHash32 hash32 = table_hash(c);
    // two pieces of 64 columns a warp where that leaves eight warps per SM, one for short batches
    const bool whole = BN % 64 == 0;
    const uint32_t most = (M + 31) / 32;
    const int pieces = pairs && D >= 128 && (uint64_t)most * ((D + 127) / 128) >= 148 * 8 ? 2 : 1;
    const uint32_t colblocks = pairs ? (D + 64 * pieces - 1) / (64 * pieces) : (D + BN - 1) / BN * ((BN + 63) / 64);
    const uint64_t units = (uint64_t)most * colblocks, blocks = (units + GRAD_THREADS / 32 - 1) / (GRAD_THREADS / 32);
    if (blocks > 0x7fffffffull) return RZ_ERR_SHAPE;
    auto run = [&](auto kernel) {
        kernel<<<(unsigned)blocks, GRAD_THREADS, 0, c.stream>>>(ids, padding, sorted.id, sorted.row, (const T *)dout, dH, c.hash, hash32, M, (uint32_t)pb->K, D,
                                                       colblocks, units, pb->alpha);
    };
    if (pairs && pieces == 2) whole ? run(rz_embedding_grad_pairs_kernel<T, 2, true>) : run(rz_embedding_grad_pairs_kernel<T, 2, false>);
    else if (pairs) whole ? run(rz_embedding_grad_pairs_kernel<T, 1, true>) : run(rz_embedding_grad_pairs_kernel<T, 1, false>);
    else run(rz_embedding_grad_kernel<T>);
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

int rz_rows_sort(const int64_t *keys, int64_t rows, int64_t bins, int32_t *order, int32_t *offsets, void *scratch, cudaStream_t stream)
{
    uint32_t per = SORT_TILE;
    const uint32_t blocks = rows > 0 ? sort_blocks(rows, &per) : 1;
    uint32_t *hist = blocks > 1 ? static_cast<uint32_t *>(scratch) : nullptr;
    int bits = 1;   // of the largest bin number, `bins`, plus one value more
    while (((bins + 1) >> bits) != 0) ++bits;
    const int smem = (int)(sizeof(uint32_t) * (SORT_WARPS + 1) * (size_t)(bins + 1));
    int st = allow_smem<rz_sort_place_kernel>((int)(sizeof(uint32_t) * (SORT_WARPS + 1) * (SORT_MAX_BINS + 1)));
    if (st) return st;
    if (hist) {
        rz_sort_count_kernel<<<blocks, SORT_THREADS, 0, stream>>>(keys, (uint32_t)rows, (uint32_t)bins, per, hist);
        rz_count_launch(1);
    }
    rz_sort_place_kernel<<<blocks, SORT_THREADS, smem, stream>>>(keys, (uint32_t)rows, (uint32_t)bins, per, bits, hist, order, offsets);
    rz_count_launch(1);
    return rz_record_cuda(cudaGetLastError(), "row sort launch");
}

int rz_rows_embedding(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const float *hashed, void *out, void *plan)
{
    const SortedTokens sorted(c.pb, plan);
    if (sorted.id) {
        const int st = sort_tokens(c, ids, padding, sorted);
        if (st) return st;
    }
    if (c.pb->io_dtype == RZ_BF16) return launch_embedding<__nv_bfloat16>(c, ids, padding, hashed, out, sorted.id != nullptr);
    return launch_embedding<float>(c, ids, padding, hashed, out, sorted.id != nullptr);
}

size_t rz_rows_embedding_plan(const rz_problem *pb) { return sorts_tokens(pb) ? sizeof(uint32_t) * 2 * (size_t)pb->M : 0; }

int rz_rows_embedding_grad(const RzLaunchCtx &c, const int64_t *ids, int64_t padding, const void *dout, float *dH, const void *plan)
{
    const SortedTokens sorted(c.pb, const_cast<void *>(plan));
    if (c.pb->io_dtype == RZ_BF16) return launch_embedding_grad<__nv_bfloat16>(c, ids, padding, sorted, dout, dH);
    return launch_embedding_grad<float>(c, ids, padding, sorted, dout, dH);
}
