// fg_rows.h -- rows of any alignment read and written 16 bytes a lane, shared by
// the layer norm, embedding and checkpoint kernels.
//
// Chunk j of a row holds its columns [j * E, j * E + E) wherever the row starts, so
// that per-column operands (gamma, beta, the weights' partial sums) lie the same
// way for every row; the memory system splits the accesses of rows between 16-byte
// boundaries.  The last chunk of a row whose length is no multiple of E goes one
// element at a time.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "fg_half.h"
#include "fg_softmax_any.h"  // Io: a chunk's elements
#include "fg_softmax_row.h"  // sums over 16 lanes

namespace fg {
namespace rows {

using smany::Io;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // at any element
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Columns [col, col + E) of `row`, of which `left` = C - col are inside it (zeros
// past them; nothing is read where left <= 0).
template <int DT>
__device__ __forceinline__ u32x4 load(const typename Io<DT>::T *row, int col, int left) {
    constexpr int E = Io<DT>::E;
    u32x4 w = {0u, 0u, 0u, 0u};
    if (left >= E) {
        w = *reinterpret_cast<const u32x4_any *>(row + col);
    } else if (left > 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e >= left) continue;
            if constexpr (DT == kF32) w[e] = __float_as_uint(row[col + e]);
            else w[e >> 1] |= (uint32_t)row[col + e] << (16 * (e & 1));
        }
    }
    return w;
}
template <int DT>
__device__ __forceinline__ void store(typename Io<DT>::T *row, int col, int left, u32x4 w) {
    constexpr int E = Io<DT>::E;
    if (left >= E) {
        *reinterpret_cast<u32x4_any *>(row + col) = w;
    } else if (left > 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (e >= left) continue;
            if constexpr (DT == kF32) row[col + e] = __uint_as_float(w[e]);
            else row[col + e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
    }
}

// Sum over a wave's 64 lanes (all active), the same in every lane: the 16-lane
// rows by DPP, then the four rows' sums.
__device__ __forceinline__ float wave_sum(float s) {
    s = smrow::row16_sum(s);
    auto of = [&](int lane) {
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s), lane));
    };
    return (of(0) + of(16)) + (of(32) + of(48));
}

}  // namespace rows
}  // namespace fg
