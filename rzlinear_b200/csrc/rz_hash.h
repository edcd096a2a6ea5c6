// ROBE-Z tile hash shared by the host entry points and every kernel.
//
// offset(pk, pn) is the start of tile (pk, pn)'s contiguous BK*BN slice in the hashed array.
// Single level  : ((pk*R3 + pn*R2 + R1) mod R0) mod (H - BK*BN)
//                 (reference: python/rz_linear/impl/RzLinearIdx.py:70-71)
// Two level     : ((((pk*R3+pn*R2+R1) mod R0)*R0 + ((pk*R7+pn*R5+R4) mod R0)) mod (H - BK*BN))
//                 (reference: python/rz_linear/impl/RzLinearForward.py:316,349)
// All operands are non-negative; with every R < 2^31 and tile coordinates < 2^31 every
// intermediate fits in 64 unsigned bits (two level: a*R0 + b < 2^62).
//
// The two moduli are fixed per call, so `v mod d` is computed exactly without a division:
// with m = floor((2^64 - 1) / d), q = floor(v * m / 2^64) is floor(v / d) or one less, hence
// r = v - q*d lies in [0, 2d) and one conditional subtraction finishes it.
#pragma once
#include <stdint.h>

#if defined(__CUDACC__)
#define RZ_HD __host__ __device__ __forceinline__
#else
#define RZ_HD inline
#endif

struct RzHash {
    uint64_t R0, R1, R2, R3, R4, R5, R7;
    uint64_t range;    // H - BK*BN
    uint64_t m_R0;     // floor((2^64-1) / R0)
    uint64_t m_range;  // floor((2^64-1) / range)
    int32_t BK, BN;
    int32_t two_level;
    int32_t pad;
};

RZ_HD uint64_t rz_mulhi64(uint64_t a, uint64_t b)
{
#if defined(__CUDA_ARCH__)
    return __umul64hi(a, b);
#else
    return (uint64_t)(((unsigned __int128)a * (unsigned __int128)b) >> 64);
#endif
}

RZ_HD uint64_t rz_fastmod(uint64_t v, uint64_t d, uint64_t m)
{
    uint64_t r = v - rz_mulhi64(v, m) * d;
    return r >= d ? r - d : r;
}

inline void rz_hash_finish(RzHash &h)
{
    h.m_R0 = ~(uint64_t)0 / h.R0;
    h.m_range = ~(uint64_t)0 / h.range;
}

RZ_HD uint64_t rz_tile_offset(const RzHash &h, uint32_t pk, uint32_t pn)
{
    uint64_t a = rz_fastmod((uint64_t)pk * h.R3 + (uint64_t)pn * h.R2 + h.R1, h.R0, h.m_R0);
    if (h.two_level) {
        uint64_t b = rz_fastmod((uint64_t)pk * h.R7 + (uint64_t)pn * h.R5 + h.R4, h.R0, h.m_R0);
        a = a * h.R0 + b;
    }
    return rz_fastmod(a, h.range, h.m_range);
}

// The same offsets in 32-bit arithmetic where the sizes allow it, for kernels that hash about as often as they load: a 64-bit
// modulus costs some 40 instructions, a 32-bit one 4.  `linear32`: the residues of R make both linear forms fit 32 bits for every tile
// of the matrix (the default prime 45007, up to about 95000 tile rows).  `square32`: R0^2 <= 2^32, so the combined two-level value
// fits; a single-level value always does.  v mod d as in rz_fastmod, with m = floor((2^32 - 1) / d).
struct RzHash32 {
    uint32_t R0, R1, R2, R3, R4, R5, R7;   // residues mod R0
    uint32_t m_R0, range, m_range;
    uint32_t linear32, square32;
};

RZ_HD uint32_t rz_mulhi32(uint32_t a, uint32_t b)
{
#if defined(__CUDA_ARCH__)
    return __umulhi(a, b);
#else
    return (uint32_t)(((uint64_t)a * b) >> 32);
#endif
}

RZ_HD uint32_t rz_fastmod32(uint32_t v, uint32_t d, uint32_t m)
{
    const uint32_t r = v - rz_mulhi32(v, m) * d;
    return r >= d ? r - d : r;
}

// tiles (pk, pn) with pk < tile_rows and pn < tile_cols
inline RzHash32 rz_hash32(const RzHash &h, uint64_t tile_rows, uint64_t tile_cols)
{
    RzHash32 s;
    s.R0 = (uint32_t)h.R0;
    s.R1 = (uint32_t)(h.R1 % h.R0), s.R2 = (uint32_t)(h.R2 % h.R0), s.R3 = (uint32_t)(h.R3 % h.R0);
    s.R4 = (uint32_t)(h.R4 % h.R0), s.R5 = (uint32_t)(h.R5 % h.R0), s.R7 = (uint32_t)(h.R7 % h.R0);
    s.m_R0 = 0xffffffffu / s.R0;
    s.range = (uint32_t)h.range;
    s.m_range = 0xffffffffu / s.range;
    const uint64_t lim = (uint64_t)1 << 32, pk = tile_rows - 1, pn = tile_cols - 1;   // (all factors are below 2^31)
    s.linear32 = pk * s.R3 + pn * s.R2 + s.R1 < lim && (!h.two_level || pk * s.R7 + pn * s.R5 + s.R4 < lim);
    s.square32 = !h.two_level || h.R0 * h.R0 <= lim;
    return s;
}

RZ_HD uint32_t rz_tile_offset32(const RzHash &h, const RzHash32 &s, uint32_t pk, uint32_t pn)
{
    uint32_t a, b = 0;
    if (s.linear32) {
        a = rz_fastmod32(pk * s.R3 + pn * s.R2 + s.R1, s.R0, s.m_R0);
        if (h.two_level) b = rz_fastmod32(pk * s.R7 + pn * s.R5 + s.R4, s.R0, s.m_R0);
    } else {
        a = (uint32_t)rz_fastmod((uint64_t)pk * s.R3 + (uint64_t)pn * s.R2 + s.R1, h.R0, h.m_R0);
        if (h.two_level) b = (uint32_t)rz_fastmod((uint64_t)pk * s.R7 + (uint64_t)pn * s.R5 + s.R4, h.R0, h.m_R0);
    }
    if (s.square32) return rz_fastmod32(h.two_level ? a * s.R0 + b : a, s.range, s.m_range);
    return (uint32_t)rz_fastmod((uint64_t)a * s.R0 + b, h.range, h.m_range);
}
