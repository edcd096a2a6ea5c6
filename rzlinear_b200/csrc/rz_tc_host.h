// Host helpers shared by the launchers of the tensor-core kernels (defined in rz_tc.cu).
#pragma once
#include <cuda.h>

#include "rz_common.h"

namespace rztc {

// Element size, elements per 128-byte operand row and layout of the shifted copies for a problem's precision.
struct Geometry {
    int es, epr, ns;
    uint32_t Hc;
    size_t copy_stride;
};

inline Geometry geometry(const rz_problem *pb)
{
    Geometry g;
    const bool tf32 = pb->precision != RZ_PREC_BF16;   // fp32 elements (tf32 and split-precision fp32)
    g.es = tf32 ? 4 : 2;
    g.epr = 128 / g.es;
    g.ns = 16 / g.es;
    g.Hc = (uint32_t)((pb->H + 63) / 64 * 64);
    g.copy_stride = ((size_t)g.Hc * g.es + 255) / 256 * 256;
    return g;
}

// Tensor maps.  `keep`: the host thread remembers the last few it made, for calls that repeat with the same buffers.
// `mn_major`: 0 = K-major operand, 1 = M/N-major, PLAIN_LAYOUT = rows one behind the other without a swizzle
constexpr int PLAIN_LAYOUT = 2;
int encode(CUtensorMap *map, bool tf32, int mn_major, void *base, int rank, const uint64_t *dims, const uint64_t *strides_bytes,
           const uint32_t *box, bool keep);
// 2-D map over a row-major matrix [rows][cols] of the operand type
int map_matrix(CUtensorMap *map, bool tf32, int mn_major, const void *base, uint64_t rows, uint64_t cols, uint32_t box_cols,
               uint32_t box_rows, bool keep = true);
// 3-D map over the shadow: {element of a copy, slice row (stride BN elements), copy}
int map_shadow(CUtensorMap *map, const rz_problem *pb, bool mn_major, const void *shadow, uint32_t box_rows, bool keep = true);
int num_sms();
// Block shape that RZ_TC_CONFIG forces, counted from the largest (0 = pair 512 x 256 .. 4 = 128 x 64), or -1
int forced_shape();

}  // namespace rztc
