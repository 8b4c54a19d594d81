// fg_rows.h -- rows of any alignment read and written 16 bytes a lane, shared by
// the layer norm, embedding and checkpoint kernels.
//
// Chunk j of a row holds its columns [j * E, j * E + E) wherever the row starts, so
// that per-column operands (gamma, beta, the weights' partial sums) lie the same
// way for every row; the memory system splits the accesses of rows between 16-byte
// boundaries.  The fewer than E columns past the last whole chunk go one to a lane
// (a lane that loaded a partial chunk element by element would wait for each
// element, and its branches cost the whole wave).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "fg_half.h"
#include "fg_softmax_any.h"  // Io: a chunk's elements
#include "fg_softmax_row.h"  // sums over 16 lanes

namespace fg {
namespace rows {

// Longest row, in columns: counts of columns are then exact in fp32, byte offsets
// within a row fit 32 bits, and a grid's y dimension holds a row's workgroups.
constexpr int kMaxCols = 1 << 23;
// Whether a grid's x dimension holds `blocks` workgroups: fewer than 2^32 threads.
inline bool grid_holds(int64_t blocks, int threads) {
    return blocks * threads < int64_t(1) << 32;
}

// Whether an output that a call may go without (NULL) is none of its other buffers.
inline bool apart(const void *out, std::initializer_list<const void *> others) {
    for (const void *o : others)
        if (out && out == o) return false;
    return true;
}

using smany::Io;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // at any element
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Chunk j of `row` (32-bit offsets: rows of fewer than 2^32 bytes).
template <int DT>
__device__ __forceinline__ u32x4 load(const typename Io<DT>::T *row, int j) {
    return *reinterpret_cast<const u32x4_any *>(reinterpret_cast<const char *>(row) +
                                                (uint32_t)j * 16u);
}
// (Stores are non-temporal: layer norm forward bf16 8192 x 4096 28.4 -> 23.0 us, fp32
// 16384 x 1024 26.4 -> 21.7, backward 2048 x 4096 bf16 16.2 -> 15.3.  Loads are not:
// the shapes that fit the caches lost up to 40 %.)
template <int DT>
__device__ __forceinline__ void store(typename Io<DT>::T *row, int j, u32x4 w) {
    __builtin_nontemporal_store(
        w, reinterpret_cast<u32x4_any *>(reinterpret_cast<char *>(row) + (uint32_t)j * 16u));
}

// A row's chunk j where j is below its whole chunks nb, else what the row has of it,
// one element after the other (zeros past the row's end).
template <int DT>
struct Chunk {
    using IO = Io<DT>;
    static constexpr int E = IO::E;
    static __device__ __forceinline__ u32x4 load(const typename IO::T *row, int j, int nb, int C) {
        if (j < nb) return rows::load<DT>(row, j);
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = j * E + e < C ? IO::load1(row, j * E + e) : 0.0f;
        return IO::pack(v);
    }
    static __device__ __forceinline__ void store(typename IO::T *row, int j, int nb, int C,
                                                 const float (&v)[E]) {
        if (j < nb) {
            rows::store<DT>(row, j, IO::pack(v));
            return;
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (j * E + e < C) IO::store1(row, j * E + e, v[e]);
    }
};

// The same where a partial chunk may take columns of the one before it too: it is then
// the row's last E columns, in one access, and both lanes that have a column must make
// the same of it.  Rows of fewer than E columns go element by element.
template <int DT>
struct Tail {
    using IO = Io<DT>;
    static constexpr int E = IO::E;
    int C, first;  // the lane's first column
    bool whole;
    __device__ __forceinline__ Tail(int j, int cols)
        : C(cols), first(cols < E ? j * E : min(j * E, cols - E)), whole(cols >= E) {}
    __device__ __forceinline__ uint32_t bytes() const {
        return (uint32_t)first * (uint32_t)sizeof(typename IO::T);
    }
    __device__ __forceinline__ u32x4 load(const typename IO::T *row) const {
        if (whole)
            return *reinterpret_cast<const u32x4_any *>(reinterpret_cast<const char *>(row) +
                                                        bytes());
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e < C ? IO::load1(row, e) : 0.0f;
        return IO::pack(v);
    }
    __device__ __forceinline__ void store(typename IO::T *row, const float (&v)[E]) const {
        if (whole) {
            __builtin_nontemporal_store(
                IO::pack(v),
                reinterpret_cast<u32x4_any *>(reinterpret_cast<char *>(row) + bytes()));
            return;
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < C) IO::store1(row, e, v[e]);
    }
    // Adds v to the row: columns of the chunk before j's are its lane's.
    __device__ __forceinline__ void add(typename IO::T *row, int j, const float (&v)[E]) const {
        if (first == j * E && whole) {
            const u32x4 was = load(row);
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = v[e] + IO::get(was, e);
            store(row, o);
            return;
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (first + e >= j * E && first + e < C)
                IO::store1(row, first + e, v[e] + IO::load1(row, first + e));
    }
};

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
