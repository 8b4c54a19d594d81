// fg_bits8.h -- the 8-bit form of a row's values (k_ckpt8.hip has its definition):
// int8 elements and an exponent byte per 32 columns, made a 16-byte chunk of the row a
// lane by the checkpoint and RMS norm kernels.
#pragma once

#include <hip/hip_runtime.h>

#include "fg_rows.h"

namespace fg {
namespace bits8 {

constexpr int kBlock = 32;  // columns per exponent byte
typedef rows::u32x2 u32x2_byte __attribute__((aligned(1)));
typedef uint32_t u32_byte __attribute__((aligned(1)));

// E signed bytes in one access; the bytes of the row's last, partial chunk in turn.
template <int E>
struct Bytes {
    uint32_t w[E / 4];
    __device__ __forceinline__ void load(const int8_t *row, int j, int nb, int C) {
        const int8_t *p = row + (size_t)j * E;
        if (j < nb) {
            if constexpr (E == 8) {
                const rows::u32x2 v = *reinterpret_cast<const u32x2_byte *>(p);
                w[0] = v[0];
                w[1] = v[1];
            } else {
                w[0] = *reinterpret_cast<const u32_byte *>(p);
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < E / 4; ++k) w[k] = 0;
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (j * E + k < C) w[k / 4] |= (uint32_t)(uint8_t)p[k] << (8 * (k & 3));
    }
    __device__ __forceinline__ void store(int8_t *row, int j, int nb, int C) const {
        int8_t *p = row + (size_t)j * E;
        if (j < nb) {
            if constexpr (E == 8) *reinterpret_cast<u32x2_byte *>(p) = rows::u32x2{w[0], w[1]};
            else *reinterpret_cast<u32_byte *>(p) = w[0];
            return;
        }
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (j * E + k < C) p[k] = (int8_t)(w[k / 4] >> (8 * (k & 3)));
    }
    __device__ __forceinline__ int get(int k) const {
        return (int)(int8_t)(w[k / 4] >> (8 * (k & 3)));
    }
};

// A chunk of a block: its bytes, from its values and the largest magnitude of the
// block's (as fp32 bits, NaN above infinity above numbers); returns the exponent byte.
// Every lane of the block is active (4 lanes, 8 of four elements).
template <int E>
__device__ __forceinline__ int quantise(const float (&v)[E], Bytes<E> &o) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    m = max(m, (uint32_t)smrow::dpp_i<smrow::kDppSwap1>((int)m));
    m = max(m, (uint32_t)smrow::dpp_i<smrow::kDppSwap2>((int)m));
    if constexpr (E == 4) m = max(m, (uint32_t)smrow::dpp_i<smrow::kDppHalfMirror>((int)m));
    const int b = max(1, (int)(m >> 23));
#pragma unroll
    for (int k = 0; k < E; k += 4) {
        uint32_t p = 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const float s = __builtin_rintf(__builtin_amdgcn_ldexpf(v[k + n], 133 - b));
            const int c = (int)__builtin_amdgcn_fmed3f(s, -127.0f, 127.0f);
            p |= ((uint32_t)c & 255u) << (8 * n);
        }
        o.w[k / 4] = b == 255 ? 0u : p;
    }
    return b;
}

}  // namespace bits8
}  // namespace fg
