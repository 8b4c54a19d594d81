// fg_attention.h -- what the attention kernels (fg_attention_kernel.h) and their entry
// points (k_attention.hip) share: arguments, and the launches of each element type
// (k_attention_{bf16,f16,f32}.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace fg {
namespace attn {

// x / d for 0 <= x < 2^31, d >= 1, by a product: with m = ceil(2^(31 + s) / d),
// 2^s >= d, x m / 2^(31 + s) is off by less than x / 2^31 of 1 / d.
struct Div {
    uint32_t mul = 0, shift = 0, by = 1;
    Div() = default;
    explicit Div(uint32_t d) : by(d) {
        while ((1u << shift) < d) ++shift;
        mul = (uint32_t)(((uint64_t(1) << (31 + shift)) + d - 1) / d);
    }
    __device__ __forceinline__ int of(int x) const {
        return by == 1 ? x : (int)(__umulhi((uint32_t)x << 1, mul) >> shift);
    }
};

// Matrices have a row per token and a leading dimension in elements; head h is the
// columns [h D, h D + D).  A row of a key head's work is a pair (token i, head g of its
// group), row i G + g of the sequence: the heads of a group read the same keys, and a
// sequence's rows are contiguous.
struct Args {
    const void *q, *k, *v;
    const uint32_t *qs, *ks, *klens;  // klens: the keys used of each sequence's (or NULL)
    int64_t ldq, ldk, ldv;
    int n, Tq, Tk, KV, G, D, causal;
    float scale;
    Div group;
    // Forward.
    void *out;
    int64_t ldo;
    float *lse;    // [heads][Tq], or NULL
    float *part;   // splits > 1: [splits][KV Tq G][D] sums, then as many (m, l) pairs
    int splits, slots;
    // Backward: out, lse as above.
    const void *dout;
    int64_t lddo, lddq, lddk, lddv;
    void *dq, *dk, *dv;
    float *rows;   // [3][KV Tq G]: log2 of the sum, delta; of a row of large scores, the
                   // maximum's and beside it the sum's (otherwise 0)
    float *tiles;  // [KV][slots][4][4]: of a wave's 32 rows the largest |dout| and |delta|
                   // (fp16), and whether one has large scores
    float *kpart;  // ksplits > 1: dK's and dV's sums, [2][ksplits][KV Tk][D] (dQ's: part)
    int kslots, ksplits, accumulate;
    int fill;  // workgroups that the splits are to come to
};

// Rows of a workgroup (of the few rows' one), and keys of one in the backward's pass over
// the keys.
constexpr int kRows = 128, kFewRows = 32, kKeys = 128;

// Launches on `st`; 0 or the HIP error.  dma: rows of K and V (and of the other
// operands) are whole 16-byte chunks at 16-byte boundaries, and D is the tile's width.
template <int DT>
int forward(hipStream_t st, const Args &a, bool few, bool dma);
template <int DT>
int backward(hipStream_t st, const Args &a, bool dma);
template <int DT>
int combine(hipStream_t st, const Args &a);

}  // namespace attn
}  // namespace fg
