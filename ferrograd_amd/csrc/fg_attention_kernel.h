// fg_attention_kernel.h -- attention over packed sequences, forward and backward, on
// CDNA4 matrix cores.  Included by k_attention_{bf16,f16,f32}.hip.  The reference has
// no attention; its nearest operators are the matmul and softmax nodes
// (crates/ferrograd-nn/src/op/matmul/mod.rs:17-188, op/softmax.rs:14-759).
//
//   S = scale Q K^T, -inf where a key is not visible;  P = softmax of S's rows
//   O = P V,  lse = log sum exp of S's rows
//   delta = rows' sums of dO O,  dS = P (dO V^T - delta)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
// Key j of lk is visible to query i of lq if j < lk and, causal, j <= i + lk - lq.
//
// One layout serves every product.  An MFMA's result has its column in the lane and
// its rows in the lane's registers, rows 8 (r / 4) + 4 h + r % 4 for register r of lane
// half h; an operand has its row (or column) in the lane and 8 of the summed index in
// its registers.  So S^T = K Q^T (keys in registers, a query a lane) is, rounded, the
// second operand of O^T = V^T P^T and dQ^T = K^T dS^T as it stands, and S = Q K^T
// (queries in registers, a key a lane) that of dV^T = dO^T P and dK^T = Q^T dS -- if the
// first operand takes its 8 of the summed index in the same order, 4 h + 0..3 and
// 8 + 4 h + 0..3 of each 16.  Softmax statistics are a lane's own, but for the half of
// the keys that lane ^ 32 holds.
//
// In 16 bits P and dS are rounded to the type between their two products, since a matrix
// instruction takes both operands in one type: bf16 outputs are then off by 0.0018 to
// 0.0022 of their norm, gradients by 0.0024, where their own rounding alone is 0.0015 to
// 0.0017.  What the rounding leaves, as an operand of its own, would take half as many
// matrix instructions again.
//
// Tiles sit in LDS as rows of DP elements, a few chunks apart, with 16-byte chunk c of
// row r at c ^ swz(r): read by rows (16 lanes a cycle, the same chunk of 16 rows) and,
// through the transposing reads, by columns (4 rows of 4 chunks a cycle), both reach
// every bank once.  (With three bits of the row and no gaps, two lanes a bank, half of
// LDS's time: SQ_LDS_BANK_CONFLICT 5.5e7 of 1.1e8 in dQ's kernel.)
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "fg_attention.h"
#include "fg_half.h"
#include "fg_sched.h"

namespace fg {
namespace attn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
// A score, or a row's log-sum, in units of log 2, whose rounding is 2^-4 and more.
constexpr float kFar = 0x1p20f;
__device__ __forceinline__ bool is_far(float x, float from = kFar) {
    return fabsf(x) > from && fabsf(x) < INFINITY;
}

// Bits of a chunk's place that its row sets, and the chunks left free before a row: one
// every 4 rows, of 8 chunks (128 bytes) two every 8, so that what a wave's direct load
// writes, 1 KiB, is of one piece.  Rows of 96 elements, which no direct load brings: one a
// row.
template <int CH>
__device__ __forceinline__ int swz(int row) {
    if (CH == 12 || CH == 24) return 0;
    return CH == 8 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 1) : (row & 3) << 2;
}
template <int CH>
__device__ __forceinline__ constexpr int gap(int row) {
    return CH == 12 || CH == 24 ? row : CH == 8 ? (row >> 3) * 2 : row >> 2;
}

template <int DT>
struct Type {
    static constexpr bool kWide = DT == kF32;
    using T = typename std::conditional<kWide, float, uint16_t>::type;
    using Frag = typename std::conditional<kWide, f32x8, u32x4>::type;
    static constexpr int E = kWide ? 4 : 8;  // elements of a 16-byte chunk

    // A 32x32 block's product over 16 of the summed index.  fp32: eight instructions of
    // two (one of a lane half each), element j of both operands in the j-th.
    static __device__ __forceinline__ f32x16 mfma(const Frag &a, const Frag &b, f32x16 c) {
        if constexpr (kWide) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
            return c;
        } else if constexpr (DT == kBF16) {
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                           __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                           0);
        } else {
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                          __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        }
    }
    // Registers 8 u .. 8 u + 7 of a block of fp32 values, rounded, as an operand.
    static __device__ __forceinline__ Frag pack(const f32x16 &s, int u) {
        Frag f;
        if constexpr (kWide) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = s[8 * u + j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = s[8 * u + 2 * j], y = s[8 * u + 2 * j + 1];
                if constexpr (DT == kBF16)
                    f[j] = __builtin_bit_cast(uint32_t,
                                              __builtin_convertvector((f32x2{x, y}), bf16x2));
                else f[j] = (uint32_t)f_to_f16(x) | ((uint32_t)f_to_f16(y) << 16);
            }
        }
        return f;
    }
    static __device__ __forceinline__ float get(const Frag &f, int j) {
        if constexpr (kWide) return f[j];
        else return h16_to_f(DT, (uint16_t)(f[j >> 1] >> (16 * (j & 1))));
    }
    static __device__ __forceinline__ float load1(const T *p) {
        if constexpr (kWide) return *p;
        else return h16_to_f(DT, *p);
    }
    static __device__ __forceinline__ void store1(T *p, float v) {
        if constexpr (kWide) *p = v;
        else *p = f_to_h16(DT, v);
    }
    static __device__ __forceinline__ Frag load8(const T *p) {
        Frag f;
        if constexpr (kWide) {
            const f32x4 x = *reinterpret_cast<const f32x4_any *>(p);
            const f32x4 y = *reinterpret_cast<const f32x4_any *>(p + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = j < 4 ? x[j & 3] : y[j & 3];
        } else {
            f = *reinterpret_cast<const u32x4_any *>(p);
        }
        return f;
    }
    // Elements d .. d + 7 of a row of D (zeros past it; row NULL: zeros).
    static __device__ __forceinline__ Frag load8(const T *row, int d, int D) {
        if (row && d + 8 <= D) return load8(row + d);
        Frag f;
        T e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = row && d + j < D ? row[d + j] : T(0);
        if constexpr (kWide) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = e[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = (uint32_t)e[2 * j] | ((uint32_t)e[2 * j + 1] << 16);
        }
        return f;
    }
    // Four values from column d on of a row of D; (=|+=), each rounded once.
    static __device__ __forceinline__ void store4(T *row, int d, int D, f32x4 v, bool add) {
        if (d + 4 <= D) {
            if constexpr (kWide) {
                f32x4_any *p = reinterpret_cast<f32x4_any *>(row + d);
                *p = add ? *p + v : v;
            } else {
                u32x2_any *p = reinterpret_cast<u32x2_any *>(row + d);
                if (add) {
                    const u32x2 w = *p;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] += h16_to_f(DT, (uint16_t)(w[e >> 1] >> (16 * (e & 1))));
                }
                u32x2 w;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (DT == kBF16)
                        w[j] = __builtin_bit_cast(
                            uint32_t,
                            __builtin_convertvector((f32x2{v[2 * j], v[2 * j + 1]}), bf16x2));
                    else
                        w[j] = (uint32_t)f_to_f16(v[2 * j]) |
                               ((uint32_t)f_to_f16(v[2 * j + 1]) << 16);
                }
                *p = w;
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < D) store1(row + d + e, add ? v[e] + load1(row + d + e) : v[e]);
    }
};

// ------------------------------------------------------------------ LDS tiles
// A lane's places in tiles of rows of DP elements, computed once: what the swizzle makes
// of a chunk's bits; everything else of an address is a constant.
template <int DT, int DP>
struct Lanes {
    static constexpr bool kWide = DT == kF32;
    static constexpr int E = kWide ? 4 : 8, CH = DP / E;
    int row[4], col[kWide ? 8 : 4], lane;
    static __device__ __forceinline__ int place(int r, int c) {
        return r * DP + (gap<CH>(r) + (c ^ swz<CH>(r))) * E;
    }
    __device__ __forceinline__ explicit Lanes(int lane_) : lane(lane_) {
        const int h = lane >> 5, l32 = lane & 31;
        const int e = (lane >> 2) & 3, q = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kWide) {
                row[i] = place(l32, (4 * i + 2 * h) % CH);
                col[i] = place(4 * h + i, l32 >> 2) + (l32 & 3);
                col[4 + i] = place(4 * h + i, 8 + (l32 >> 2)) + (l32 & 3);
            } else {
                row[i] = place(l32, (4 * i + h) % CH);
                col[i] = place(4 * h + e, (4 * i + 2 * ((lane >> 4) & 1) + (q >> 1)) % CH) +
                         4 * (q & 1);
            }
        }
    }
};

// ROWS rows of DP elements.
template <int DT, int DP, int ROWS>
struct Tile {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    using Frag = typename Ty::Frag;
    static constexpr int E = Ty::E, CH = DP / E;  // chunks of a row
    static constexpr int kElems = ROWS * DP + gap<CH>(ROWS) * E;
    static constexpr int kChunks = ROWS * CH;

    // Rows 32 b + lane % 32, elements 16 ks + 8 h .. + 7: an operand with the tile's rows in
    // lanes.
    static __device__ __forceinline__ Frag by_row(const T *t, int b, int ks,
                                                  const Lanes<DT, DP> &L) {
        t += b * (32 * DP + gap<CH>(32) * E);
        if constexpr (Ty::kWide) {
            Frag f;
            const T *p = t + L.row[ks & 3] + 64 * (ks >> 2);
            const f32x4 x = *reinterpret_cast<const f32x4 *>(p);
            const f32x4 y = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = j < 4 ? x[j & 3] : y[j & 3];
            return f;
        } else {
            return *reinterpret_cast<const u32x4 *>(t + L.row[ks >> 1] + 16 * (ks & 1));
        }
    }
    // Columns 32 d + lane % 32, rows r0 + 4 h + 0..3 and r0 + 8 + 4 h + 0..3 (r0 a multiple
    // of 16): an operand with the tile's columns in lanes.  16 bits: two transposing reads,
    // in which source lane 4 e + q of each 16 reads 4 elements of row e, and lane l gets
    // column l's rows.
    static __device__ __forceinline__ Frag by_column(const T *t, int r0, int d,
                                                     const Lanes<DT, DP> &L) {
        t += r0 / 16 * (16 * DP + gap<CH>(16) * E);
        constexpr int kHalf = 8 * DP + gap<CH>(8) * E;
        Frag f;
        if constexpr (Ty::kWide) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                f[j] = t[L.col[4 * (d & 1) + (j & 3)] + (j >> 2) * kHalf + 64 * (d >> 1)];
        } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const v4i16 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) v4i16 *)(t + L.col[d] + half * kHalf));
                const u32x2 w = __builtin_bit_cast(u32x2, v);
                f[2 * half] = w[0];
                f[2 * half + 1] = w[1];
            }
        }
        return f;
    }
    // Whether the whole tile is finite (by one wave).
    static __device__ __forceinline__ bool finite(const T *t, int lane) {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        uint32_t top = 0;
#pragma unroll 4
        for (int c = lane; c < kChunks; c += 64) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(t + (c + gap<CH>(c / CH)) * E);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (Ty::kWide) {
                    top = max(top, w[e] & 0x7fffffffu);
                } else {
                    top = __builtin_bit_cast(
                        uint32_t,
                        __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                  __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu)));
                }
            }
        }
        constexpr uint32_t kInf = DT == kF16 ? 0x7c00u : 0x7f80u;
        bool bad;
        if constexpr (Ty::kWide) bad = top >= 0x7f800000u;
        else bad = (top & 0xffffu) >= kInf || (top >> 16) >= kInf;
        return !__any(bad);
    }
};

// Moves a tile's rows from memory, NT threads together.  DMA: straight into LDS, lane l
// of a wave load at its 16 l bytes, the source chosen so that the chunks land swizzled;
// rows past the last are the last again.  Otherwise through registers, zeros past the last
// row and column.
template <int DT, int DP, int ROWS, int NT, bool DMA>
struct Mover {
    using Tl = Tile<DT, DP, ROWS>;
    using T = typename Tl::T;
    static constexpr int E = Tl::E, CH = Tl::CH;
    static constexpr int kPer = (Tl::kChunks + NT - 1) / NT;
    static constexpr int kLoadRows = 64 / CH;  // rows of a wave load: of one swizzle
    static_assert(!DMA || Tl::kChunks % NT == 0, "whole chunks a thread");
    u32x4 v[DMA ? 1 : kPer];

    // DMA: row r at offset_of(r) bytes from the (uniform) base.
    template <class F>
    static __device__ __forceinline__ void direct(T *lds, int tid, const T *base, F offset_of) {
        const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint32_t c = ((lane % CH) ^ swz<CH>(lane / CH)) * 16;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int row = (wave * kPer + i) * kLoadRows;
            lds_dma16(base, offset_of(row + lane / CH) + c, lds + row * DP + gap<CH>(row) * E);
        }
    }
    // Otherwise: row r from row_at(r); with rows and D, zeros past them.
    template <class F>
    __device__ __forceinline__ void fetch(int tid, F row_at) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int pos = i * NT + tid;
            v[i] = *reinterpret_cast<const u32x4_any *>(row_at(pos / CH) + pos % CH * E);
        }
    }
    template <class F>
    __device__ __forceinline__ void fetch(int tid, int rows, int D, F row_at) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int pos = i * NT + tid, row = pos / CH, d = (pos % CH) * E;
            if (Tl::kChunks % NT && row >= ROWS) break;
            const T *p = row_at(row) + d;
            v[i] = u32x4{0u, 0u, 0u, 0u};
            if (row < rows && d + E <= D) {
                v[i] = *reinterpret_cast<const u32x4_any *>(p);
            } else if (row < rows && d < D) {
                T e[E];
#pragma unroll
                for (int k = 0; k < E; ++k) e[k] = d + k < D ? p[k] : T(0);
                v[i] = __builtin_bit_cast(u32x4, e);
            }
        }
    }
    // `rows` rows (the tile's, or as many as are left) ld elements apart, from base on.
    __device__ __forceinline__ void load(T *lds, int tid, const T *base, int64_t ld, int rows,
                                         int D) {
        if constexpr (!DMA) {
            fetch(tid, rows, D, [&](int r) { return base + min(r, rows - 1) * ld; });
        } else if (rows >= ROWS) {
            // One offset for all of a lane's loads.
            const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
            const uint32_t bytes = (uint32_t)ld * sizeof(T);
            const uint32_t at =
                lane / CH * bytes + ((lane % CH) ^ swz<CH>(lane / CH)) * 16;
            const char *from =
                reinterpret_cast<const char *>(base) + wave * kPer * kLoadRows * bytes;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int row = (wave * kPer + i) * kLoadRows;
                lds_dma16(from + i * kLoadRows * bytes, at, lds + row * DP + gap<CH>(row) * E);
            }
        } else {
            const uint32_t bytes = (uint32_t)ld * sizeof(T);
            direct(lds, tid, base, [&](int r) { return (uint32_t)min(r, rows - 1) * bytes; });
        }
    }
    __device__ __forceinline__ void store(T *lds, int tid) const {
        if constexpr (!DMA) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int pos = i * NT + tid, row = pos / CH, c = pos % CH;
                if (Tl::kChunks % NT && row >= ROWS) break;
                *reinterpret_cast<u32x4 *>(lds + Lanes<DT, DP>::place(row, c)) = v[i];
            }
        }
    }
};

// What the scheduler is to send in turn: N LDS reads, or N matrix instructions with R
// reads after each.  (Left to itself the compiler waits for each pair of reads where
// registers are few.)
template <int N>
__device__ __forceinline__ void reads() {
    __builtin_amdgcn_sched_group_barrier(0x100, N, 0);
}
template <int N, int R>
__device__ __forceinline__ void products() {
    each_of<N>([](auto) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (R) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    });
}

// The wave's direct loads have landed and its LDS reads are done, and every other
// wave's.  (The builtin tells the compiler, which otherwise waits for operands loaded
// before the loop where they are used: for the next tile's loads, just sent, with them.)
__device__ __forceinline__ void landed() {
    wait_vmcnt<0>();
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A tile is in LDS.  Through registers the wave's loads had landed before it was stored;
// the builtin says so to the compiler here too.
template <bool DMA>
__device__ __forceinline__ void staged() {
    if constexpr (DMA) {
        landed();
    } else {
        wait_vmcnt<0>();
        __syncthreads();
    }
}

// ------------------------------------------------------------------ sequences
// Sequence of work slot `slot` and its tile there: sequence s has the slots from
// start(s) = first(s) / per + s on (first: its first row, or key), at least as many as
// tiles, so that neither a list of tiles nor the lengths on the host are needed.  A wave
// tries 64 sequences at a time.
struct Place {
    int seq, tile;
};
template <class F>
__device__ __forceinline__ Place place_of(int slot, int n, F start) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = n;  // the sequence is in [lo, lo + len)
    while (len > 1) {
        const int step = (len + 63) >> 6;
        const int s = lo + lane * step;
        const bool past = lane * step < len && start(s) <= slot;
        const int k = max(1, (int)__popcll(__ballot(past))) - 1;
        lo += k * step;
        len = min(step, len - k * step);
        if (step == 1) break;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    return {lo, slot - start(lo)};
}

// A sequence's rows and keys, whatever its offsets say within the matrices.
struct Seq {
    int q0, lq, k0, lk;
    __device__ __forceinline__ Seq(const Args &a, int s) {
        q0 = (int)min(a.qs[s], (uint32_t)a.Tq);
        lq = max(0, (int)min(a.qs[s + 1], (uint32_t)a.Tq) - q0);
        k0 = (int)min(a.ks[s], (uint32_t)a.Tk);
        lk = max(0, (int)min(a.ks[s + 1], (uint32_t)a.Tk) - k0);
        if (a.klens) lk = (int)min((uint32_t)lk, a.klens[s]);
    }
};

// Tiles of a split in the backward: the same for all sequences, so that a long one has
// more splits and no workgroup many times the work of the others.  With w workgroups of t
// tiles each in a sequence's pass, those of p tiles are at most sum(w t) / p + sum(w):
// `fill` with this p (128 rows or keys at least).  A wave computes it from the starts.
// (Five sequences of up to 777 tokens, 6 heads of 72 over 3, fp32: equal splits of every
// sequence took 200 us in the two passes.)
template <int KT, bool KEYS>
__device__ __forceinline__ int split_tiles(const Args &a) {
    constexpr int kLeast = 128 / KT, kWg = KEYS ? kKeys : kRows;
    float work = 0.0f, wgs = 0.0f;
    for (int s = threadIdx.x & 63; s < a.n; s += 64) {
        const Seq sq(a, s);
        const int rows = sq.lq * a.G, of = KEYS ? sq.lk : rows, over = KEYS ? rows : sq.lk;
        const float w = (float)((of + kWg - 1) / kWg);
        wgs += w;
        // (Explicitly fused: every kernel that asks gets the same number.)
        work = __builtin_fmaf(w, (float)((over + KT - 1) / KT), work);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        work += __shfl_xor(work, o);
        wgs += __shfl_xor(wgs, o);
    }
    const float p = (a.causal ? 0.5f : 1.0f) * work * a.KV / fmaxf(1.0f, a.fill - wgs * a.KV);
    return __builtin_amdgcn_readfirstlane(max(kLeast, (int)fminf(p, 1e6f) + 1));
}

// Tiles of split y, from the first on; used: splits that have any, or 1.
struct Share {
    int t0, t1, used;
    __device__ __forceinline__ Share(int tiles, int splits, int each, int y) {
        const int per = max(each, (tiles - 1) / splits + 1);
        t0 = min(y * per, max(tiles, 0));
        t1 = min(t0 + per, max(tiles, 0));
        used = tiles > 0 ? (tiles - 1) / per + 1 : 1;
    }
};

// Key head and slot of a workgroup.  Consecutive workgroups go to the 8 XCDs in turn:
// the key heads vary fastest, eight at a time where they come in eights, so that an
// XCD's L2 keeps few heads' keys.
struct Work {
    int kv, slot;
    __device__ __forceinline__ Work(int bid, int KV, int slots) {
        const int by = KV % 8 == 0 ? 8 : KV;
        const int g = bid / (by * slots), in = bid - g * by * slots;
        slot = in / by;
        kv = g * by + in - slot * by;
    }
};

// Where a tile in which not every key is visible to every row holds an infinity or NaN,
// the matrix instructions would bring it, times 0, to rows that do not see it.  A
// workgroup that meets such a tile (or scores or log-sums past kFar) does its work over, a
// wave an output row, lanes over 64 of the summed index and then over the row's columns,
// what is not visible left out.
// Sum over a row's D columns of x y, x the wave's row, y the lane's (lanes that are on).
template <int DT>
__device__ __forceinline__ float dot(const typename Type<DT>::T *x, const typename Type<DT>::T *y,
                                     int D, bool on) {
    float s = 0.0f;
    if (on)
        for (int d = 0; d < D; ++d) s += Type<DT>::load1(x + d) * Type<DT>::load1(y + d);
    return s;
}
// acc[i] (column lane + 64 i) += w times the row's.
template <int DT>
__device__ __forceinline__ void add_row(float (&acc)[2], float w, const typename Type<DT>::T *row,
                                        int D, int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < D) acc[i] += w * Type<DT>::load1(row + lane + 64 * i);
}
template <int DT>
__device__ __forceinline__ void put_row(typename Type<DT>::T *row, const float (&acc)[2], float f,
                                        int D, int lane, bool add) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = lane + 64 * i;
        if (d < D)
            Type<DT>::store1(row + d, acc[i] * f + (add ? Type<DT>::load1(row + d) : 0.0f));
    }
}

template <int NB>
__device__ __forceinline__ void clear(f32x16 (&acc)[NB]) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][r] = 0.0f;
}
__device__ __forceinline__ f32x16 all16(float x) {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = x;
    return z;
}
// Keeps a value from being spread over 16 registers once and for all.
__device__ __forceinline__ float fresh(float x) {
    asm volatile("" : "+v"(x));
    return x;
}
// A block's rows' numbers, from those of rows 4 h on.
__device__ __forceinline__ f32x16 rows16(const float *p) {
    f32x16 z;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(p + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[4 * q + e] = v[e];
    }
    return z;
}

// ------------------------------------------------------------------- forward
// A wave's 32 rows (one a lane, both halves): queries as operands, running statistics
// and O^T.  m is a score that the exponentials are taken from, raised only by scores far
// above it (the sums stay far from overflow; the quotient is the same), so that O is
// seldom rescaled.  fp16 probabilities carry a factor of 2^8: the smallest that count
// stay above the type's subnormals.
template <int DT, int DP, int KT>
struct Rows {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    using Tl = Tile<DT, DP, KT>;
    static constexpr int NB = DP / 32, NK = DP / 16, KB = KT / 32;
    static constexpr float kUp = DT == kF16 ? 8.0f : 0.0f, kRaise = DT == kF16 ? 4.0f : 8.0f;
    typename Ty::Frag q[NK];
    f32x16 o[NB];
    float m = -INFINITY, l = 0.0f;
    bool bad = false;  // a tile of keys not all visible held an infinity or NaN, or m is far

    // Scores of keys key0 .. key0 + KT - 1 (s), the visible of which, up to `last` for the
    // lane's row, become probabilities; whole: every one is visible to every row of the
    // wave.
    __device__ __forceinline__ void weigh(f32x16 (&s)[KB], int key0, int last, bool whole, float c,
                                          int h) {
        if (!whole) {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = key0 + 32 * b + 8 * (r >> 2) + 4 * h + (r & 3);
                    s[b][r] = key <= last ? s[b][r] : -INFINITY;
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any((top - m) * c > kRaise)) {
            const float to = fmaxf(m, top);
            const float f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - to) * c);
            m = to;
            // (Exponentials from a rounded m c: past kFar the rounding would be in them.)
            bad |= fabsf(to) * c > kFar && fabsf(to) < INFINITY;
            l *= f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[b][r] *= f;
        }
        const float from = (m == -INFINITY ? 0.0f : m * c) - kUp;
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], c, -from));
                part[r & 3] += s[b][r];
            }
        l += (part[0] + part[1]) + (part[2] + part[3]);
    }
    // Their values, from tile v.
    __device__ __forceinline__ void values(const T *v, const f32x16 (&s)[KB], bool whole,
                                           const Lanes<DT, DP> &L) {
        if (!whole) bad |= !Tl::finite(v, L.lane);
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename Ty::Frag p = Ty::pack(s[b], u);
#pragma unroll
                for (int d = 0; d < NB; ++d)
                    o[d] = Ty::mfma(Tl::by_column(v, 32 * b + 16 * u, d, L), p, o[d]);
            }
    }
};

// Where a row's outputs go.  at: its place among the key head's rows.
template <int DT, int DP>
__device__ __forceinline__ void write_row(const Args &a, int kv, int split, int row, int token,
                                          int g, int h, const f32x16 (&o)[DP / 32], float m,
                                          float l, float c) {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    constexpr float kUp = Rows<DT, DP, 32>::kUp;
    if (a.splits > 1) {
        const int64_t rows = (int64_t)a.KV * a.Tq * a.G;
        const int64_t at = (int64_t)split * rows + (int64_t)kv * a.Tq * a.G + row;
        if (h == 0) {
            float *ml = a.part + a.splits * rows * a.D + 2 * at;
            ml[0] = m;
            ml[1] = l;
        }
        if (l == 0.0f) return;
        float *p = a.part + at * a.D;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                Type<kF32>::store4(p, 32 * b + 8 * q + 4 * h, a.D,
                                   f32x4{o[b][4 * q], o[b][4 * q + 1], o[b][4 * q + 2],
                                         o[b][4 * q + 3]},
                                   false);
        return;
    }
    const int head = kv * a.G + g;
    const float f = 1.0f / l;
    T *p = static_cast<T *>(a.out) + token * a.ldo + (int64_t)head * a.D;
    // (Without a sum 0, also where a value that counts nothing was infinite.)
    auto of = [&](float x) { return l == 0.0f ? 0.0f : x * f; };
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            Ty::store4(p, 32 * b + 8 * q + 4 * h, a.D,
                       f32x4{of(o[b][4 * q]), of(o[b][4 * q + 1]), of(o[b][4 * q + 2]),
                             of(o[b][4 * q + 3])},
                       false);
    if (a.lse && h == 0)
        a.lse[(int64_t)head * a.Tq + token] =
            l == 0.0f ? -INFINITY : (m * c + (__log2f(l) - kUp)) * kLn2;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Rows row0 .. row1 - 1 of a sequence over its keys key0 .. key1 - 1, carefully.
template <int DT>
__device__ void careful_fwd(const Args &a, const Seq &sq, int kv, int split, int row0, int row1,
                            int key0, int key1, int wave, int lane) {
    using T = typename Type<DT>::T;
    constexpr float kUp = Rows<DT, 32, 32>::kUp;
    const float c = a.scale * kLog2e;
    const T *k = static_cast<const T *>(a.k) + sq.k0 * a.ldk + (int64_t)kv * a.D;
    const T *v = static_cast<const T *>(a.v) + sq.k0 * a.ldv + (int64_t)kv * a.D;
    for (int row = row0 + wave; row < row1; row += 4) {
        const int i = a.group.of(row), head = kv * a.G + row - i * a.G, token = sq.q0 + i;
        const int end = min(min(key1, sq.lk), a.causal ? i + sq.lk - sq.lq + 1 : sq.lk);
        const T *q = static_cast<const T *>(a.q) + token * a.ldq + (int64_t)head * a.D;
        float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
        for (int j0 = key0; j0 < end; j0 += 64) {
            const int j = j0 + lane;
            const float x = dot<DT>(q, k + j * a.ldk, a.D, j < end);
            const float to = fmaxf(m, wave_max(j < end ? x : -INFINITY));
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - to) * c);
            m = to;
            const float from = m == -INFINITY ? 0.0f : m;
            const float p = j < end ? __builtin_amdgcn_exp2f((x - from) * c + kUp) : 0.0f;
            l = (l == 0.0f ? 0.0f : l * f) + wave_add(p);
#pragma unroll
            for (int e = 0; e < 2; ++e) acc[e] = acc[e] == 0.0f ? 0.0f : acc[e] * f;
            for (int n = 0; n < min(64, end - j0); ++n)
                add_row<DT>(acc, __shfl(p, n), v + (j0 + n) * a.ldv, a.D, lane);
        }
        if (l == 0.0f) acc[0] = acc[1] = 0.0f;
        if (a.splits > 1) {
            const int64_t rows = (int64_t)a.KV * a.Tq * a.G;
            const int64_t at =
                (int64_t)split * rows + (int64_t)kv * a.Tq * a.G + sq.q0 * a.G + row;
            if (lane == 0) {
                float *ml = a.part + a.splits * rows * a.D + 2 * at;
                ml[0] = m;
                ml[1] = l;
            }
            put_row<kF32>(a.part + at * a.D, acc, 1.0f, a.D, lane, false);
            continue;
        }
        put_row<DT>(static_cast<T *>(a.out) + token * a.ldo + (int64_t)head * a.D, acc,
                    l == 0.0f ? 0.0f : 1.0f / l, a.D, lane, false);
        if (a.lse && lane == 0)
            a.lse[(int64_t)head * a.Tq + token] =
                l == 0.0f ? -INFINITY : (m * c + (__log2f(l) - kUp)) * kLn2;
    }
}

// Four waves of 32 rows, the same keys for all: K and V tiles of KT keys, two stages.  (A
// wave's 32 queries and their sums take half of its registers at D 128 with two waves a
// SIMD, which 16 bits need to hide the exponentials behind the other wave's products.)
// bf16, 8 sequences of up to 4096, 32 heads of 128 over 8, causal: 680 us, 860 TFLOP/s,
// where a square library product reaches 1213 (fp16 705 us): the matrix units are busy 40 %
// of the cycles and the vector unit about 47 %, LDS 21 %, at 2.2 GHz, where that product
// keeps the matrix units busy 70 %, at 2.0.  Two waves a SIMD take turns at the two units;
// reads sent further ahead, wave priorities and fewer maxima all left 687 to 694.  Tiles
// that come through registers (heads of other widths, rows off 16-byte boundaries): 4
// sequences of 2048, 175 us and 187.  fp32, one wave a SIMD: 8 sequences of up to 4096, 8
// heads of 128 over 2, 1.67 ms, 88 TFLOP/s of 144.
template <int DT>
constexpr int keys_of() {
    return DT == kF32 ? 32 : 64;
}

template <int DT, int DP, bool DMA>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DT == kF32 ? 1 : 2))) void
att_fwd(const Args a) {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    constexpr int KT = keys_of<DT>();
    using Tl = Tile<DT, DP, KT>;
    __shared__ __attribute__((aligned(16))) T lds[4 * Tl::kElems];
    const Work w(blockIdx.x, a.KV, a.slots);
    const Place pl = place_of(a.slots - 1 - w.slot, a.n, [&](int s) {
        return (int)min(a.qs[s], (uint32_t)a.Tq) * a.G / kRows + s;
    });
    const Seq sq(a, pl.seq);
    const int rows = sq.lq * a.G, m0 = pl.tile * kRows;
    if (pl.tile < 0 || m0 >= rows) return;  // (a slot of no tile)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, l32 = lane & 31, off = sq.lk - sq.lq;
    const float c = a.scale * kLog2e;
    const T *k = static_cast<const T *>(a.k) + sq.k0 * a.ldk + (int64_t)w.kv * a.D;
    const T *v = static_cast<const T *>(a.v) + sq.k0 * a.ldv + (int64_t)w.kv * a.D;
    // The last key that a row sees.
    auto last_of = [&](int row) {
        return a.causal ? min(sq.lk - 1, a.group.of(row) + off) : sq.lk - 1;
    };
    const int w0 = m0 + 32 * wave, row = w0 + l32;
    const int token = sq.q0 + a.group.of(row), g = row - (token - sq.q0) * a.G;
    const int last = row < rows ? last_of(row) : -1;
    const int wave_first = w0 < rows ? last_of(w0) : -1;
    const int wave_last = w0 < rows ? last_of(min(w0 + 31, rows - 1)) : -1;
    const int keys = last_of(min(m0 + kRows, rows) - 1) + 1;
    const int tiles = keys > 0 ? (keys - 1) / KT + 1 : 0;
    const int t0 = (int)((int64_t)tiles * blockIdx.y / a.splits);
    const int t1 = (int)((int64_t)tiles * (blockIdx.y + 1) / a.splits);

    const Lanes<DT, DP> L(lane);
    Rows<DT, DP, KT> st;
    const T *qrow = row < rows ? static_cast<const T *>(a.q) + token * a.ldq +
                                     (int64_t)(w.kv * a.G + g) * a.D
                               : nullptr;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) st.q[ks] = Ty::load8(qrow, 16 * ks + 8 * h, a.D);
    clear(st.o);

    Mover<DT, DP, KT, 256, DMA> mk, mv;
    auto load = [&](int t) {
        T *to = lds + (t & 1) * 2 * Tl::kElems;
        const int key0 = t * KT, left = sq.lk - key0;
        mk.load(to, tid, k + key0 * a.ldk, a.ldk, left, a.D);
        mv.load(to + Tl::kElems, tid, v + key0 * a.ldv, a.ldv, left, a.D);
    };
    auto store = [&](int t) {
        T *to = lds + (t & 1) * 2 * Tl::kElems;
        mk.store(to, tid);
        mv.store(to + Tl::kElems, tid);
    };
    if (t0 < t1) {
        load(t0);
        store(t0);
    }
    for (int t = t0; t < t1; ++t) {
        // The tile has landed, and every wave is done with the one before it.
        staged<DMA>();
        if (t + 1 < t1) load(t + 1);
        const int key0 = t * KT;
        const T *at = lds + (t & 1) * 2 * Tl::kElems;
        if (key0 <= wave_last) {
            const bool whole = key0 + KT - 1 <= wave_first;
            f32x16 s[KT / 32];
#pragma unroll
            for (int b = 0; b < KT / 32; ++b) {
                s[b] = all16(0.0f);
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks)
                    s[b] = Ty::mfma(Tl::by_row(at, b, ks, L), st.q[ks], s[b]);
            }
            st.weigh(s, key0, last, whole, c, h);
            st.values(at + Tl::kElems, s, whole, L);
        }
        if (t + 1 < t1) store(t + 1);
    }
    if (__syncthreads_or(st.bad)) {
        careful_fwd<DT>(a, sq, w.kv, blockIdx.y, m0, min(m0 + kRows, rows), t0 * KT, t1 * KT, wave,
                        lane);
        return;
    }
    st.l += __shfl_xor(st.l, 32);
    if (row < rows)
        write_row<DT, DP>(a, w.kv, blockIdx.y, sq.q0 * a.G + row, token, g, h, st.o, st.m, st.l, c);
}

// Few rows (single tokens: a group's heads): 32 rows a workgroup, whose four waves take
// key tiles in turn without barriers; their statistics and sums are joined at the end.
// Bound by the keys' and values' bytes: a wave's next keys load into the registers that
// hold this tile's as soon as its scores are taken, the next values as soon as these have
// gone to the wave's LDS (for the transposing reads), so that about 16 KiB a wave, 128 a
// CU, are in flight.  FULL: heads of DP columns.  8 tokens over caches of up to 8192, bf16,
// 32 heads of 128 over 8: 32 us.
constexpr int kFewKeys = 32;
template <int DT, int DP, bool FULL>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DT == kF32 ? 1 : 2))) void
att_fwd_few(const Args a) {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    constexpr int KT = kFewKeys, NB = DP / 32, NK = DP / 16;
    using Tl = Tile<DT, DP, KT>;
    // A wave's values; at the end its O^T, 32 x DP floats, of waves 1 to 3.
    constexpr int kWave = Tl::kElems * (int)sizeof(T) > 32 * DP * 4 ? Tl::kElems
                                                                   : 32 * DP * 4 / (int)sizeof(T);
    __shared__ __attribute__((aligned(16))) T lds[4 * kWave];
    __shared__ float ml[4][32][2];
    const Work w(blockIdx.x, a.KV, a.slots);
    const Place pl = place_of(w.slot, a.n, [&](int s) {
        return (int)min(a.qs[s], (uint32_t)a.Tq) * a.G / kFewRows + s;
    });
    const Seq sq(a, pl.seq);
    const int rows = sq.lq * a.G, m0 = pl.tile * kFewRows;
    if (pl.tile < 0 || m0 >= rows) return;  // (a slot of no tile)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, l32 = lane & 31, off = sq.lk - sq.lq;
    const float c = a.scale * kLog2e;
    const T *k = static_cast<const T *>(a.k) + sq.k0 * a.ldk + (int64_t)w.kv * a.D;
    const T *v = static_cast<const T *>(a.v) + sq.k0 * a.ldv + (int64_t)w.kv * a.D;
    auto last_of = [&](int row) {
        return a.causal ? min(sq.lk - 1, a.group.of(row) + off) : sq.lk - 1;
    };
    const int row = m0 + l32;
    const int token = sq.q0 + a.group.of(row), g = row - (token - sq.q0) * a.G;
    const int last = row < rows ? last_of(row) : -1;
    const int first = last_of(m0);
    const int keys = last_of(min(m0 + kFewRows, rows) - 1) + 1;
    const int tiles = keys > 0 ? (keys - 1) / KT + 1 : 0;
    const int t0 = (int)((int64_t)tiles * blockIdx.y / a.splits) + wave;
    const int t1 = (int)((int64_t)tiles * (blockIdx.y + 1) / a.splits);

    const Lanes<DT, DP> L(lane);
    Rows<DT, DP, KT> st;
    typename Ty::Frag kf[NK];
    Mover<DT, DP, KT, 64, false> mv;
    // (Rows past the sequence's keys: its last again.)
    auto load_k = [&](int t) {
        const T *p = k + min(t * KT + l32, sq.lk - 1) * a.ldk;
#pragma unroll
        for (int ks = 0; ks < NK; ++ks)
            kf[ks] = FULL ? Ty::load8(p + 16 * ks + 8 * h) : Ty::load8(p, 16 * ks + 8 * h, a.D);
    };
    auto load_v = [&](int t) {
        const int key0 = t * KT, left = sq.lk - key0;
        const T *p = v + key0 * a.ldv;
        auto at = [&](int r) { return p + min(r, left - 1) * a.ldv; };
        if constexpr (FULL) mv.fetch(lane, at);
        else mv.fetch(lane, left, a.D, at);
    };
    if (t0 < t1) {
        load_k(t0);
        load_v(t0);
    }
    const T *qrow = row < rows ? static_cast<const T *>(a.q) + token * a.ldq +
                                     (int64_t)(w.kv * a.G + g) * a.D
                               : nullptr;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) st.q[ks] = Ty::load8(qrow, 16 * ks + 8 * h, a.D);
    clear(st.o);
    T *mine = lds + wave * kWave;
    for (int t = t0; t < t1; t += 4) {
        const int key0 = t * KT;
        const bool whole = key0 + KT - 1 <= first, more = t + 4 < t1;
        f32x16 s[1] = {all16(0.0f)};
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) s[0] = Ty::mfma(kf[ks], st.q[ks], s[0]);
        if (more) load_k(t + 4);
        st.weigh(s, key0, last, whole, c, h);
        __builtin_amdgcn_wave_barrier();  // (after the reads of the values before)
        mv.store(mine, lane);
        __builtin_amdgcn_wave_barrier();
        if (more) load_v(t + 4);
        st.values(mine, s, whole, L);
    }
    if (__syncthreads_or(st.bad)) {
        careful_fwd<DT>(a, sq, w.kv, blockIdx.y, m0, min(m0 + kFewRows, rows), (t0 - wave) * KT,
                        t1 * KT, wave, lane);
        return;
    }
    st.l += __shfl_xor(st.l, 32);
    // Join the waves: from their largest m, O scaled by each wave into its own LDS, added
    // by the first.
    if (h == 0) {
        ml[wave][l32][0] = st.m;
        ml[wave][l32][1] = st.l;
    }
    __syncthreads();
    float m = ml[0][l32][0];
#pragma unroll
    for (int k = 1; k < 4; ++k) m = fmaxf(m, ml[k][l32][0]);
    const float f = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((st.m - m) * c);
    float l = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float mk_ = ml[k][l32][0];
        l += mk_ == -INFINITY ? ml[k][l32][1]  // (0, or NaN)
                              : ml[k][l32][1] * __builtin_amdgcn_exp2f((mk_ - m) * c);
    }
    float *os = reinterpret_cast<float *>(mine);
    const bool any = st.l != 0.0f;  // (a wave without keys adds nothing)
    if (wave > 0) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                os[(16 * b + r) * 64 + lane] = any ? st.o[b][r] * f : 0.0f;
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float s = any ? st.o[b][r] * f : 0.0f;
#pragma unroll
            for (int k = 1; k < 4; ++k)
                s += reinterpret_cast<const float *>(lds + k * kWave)[(16 * b + r) * 64 + lane];
            st.o[b][r] = s;
        }
    if (row < rows)
        write_row<DT, DP>(a, w.kv, blockIdx.y, sq.q0 * a.G + row, token, g, h, st.o, m, l, c);
}

// Joins a row's splits, a wave a row, 4 rows a workgroup; rows of no sequence are left.
template <int DT>
__global__ __launch_bounds__(256) void att_combine(const Args a) {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    constexpr float kUp = Rows<DT, 32, 32>::kUp;
    const int lane = threadIdx.x & 63;
    const int64_t rows = (int64_t)a.KV * a.Tq * a.G;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= rows) return;
    const int kv = (int)(at / ((int64_t)a.Tq * a.G));
    const int row = (int)(at - (int64_t)kv * a.Tq * a.G);
    const int token = a.group.of(row), g = row - token * a.G;
    const Place pl = place_of(token, a.n, [&](int s) { return (int)min(a.qs[s], (uint32_t)a.Tq); });
    const Seq sq(a, pl.seq);
    if (token < sq.q0 || token >= sq.q0 + sq.lq) return;
    const float c = a.scale * kLog2e;
    const float *ml = a.part + a.splits * rows * a.D;
    // Lane s takes split s's weight.
    float m = -INFINITY, l = 0.0f;
    if (lane < a.splits) {
        m = ml[2 * (lane * rows + at)];
        l = ml[2 * (lane * rows + at) + 1];
    }
    float top = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float f = m == -INFINITY ? (l == l ? 0.0f : l) : __builtin_amdgcn_exp2f((m - top) * c);
    float sum = l == 0.0f ? 0.0f : l * f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    const int head = kv * a.G + g;
    T *p = static_cast<T *>(a.out) + token * a.ldo + (int64_t)head * a.D;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    for (int d = lane; d < ((a.D + 63) & ~63); d += 64) {
        float s = 0.0f;
        for (int k = 0; k < a.splits; ++k) {
            const float fk = __shfl(f, k), lk = __shfl(l, k);
            if (lk != 0.0f && d < a.D) s += fk * a.part[(k * rows + at) * a.D + d];
        }
        if (d < a.D) Ty::store1(p + d, s * inv);
    }
    if (a.lse && lane == 0)
        a.lse[(int64_t)head * a.Tq + token] =
            sum == 0.0f ? -INFINITY : (top * c + (__log2f(sum) - kUp)) * kLn2;
}

// ------------------------------------------------------------------ backward
// dS of fp16 tensors carries a power of two that brings it near 1, whatever dout's size:
// probabilities of long rows times small gradients would be subnormal.  It is taken from
// the largest |dout| (as if V were of order 1) and lowered, the sums with it, where what is
// carried would pass 2^15: |dS| reaches |dout| |V| D, past the type's range from |V| = 64
// on.  The pass over rows looks at what it carries, a power a row; the pass over keys, which
// knows its keys' V, at what that can be, |dout| sum |V| + |delta|, a power a key.  (4
// sequences of 2048, 16 heads of 64 over 8: 266 us for both; 297 where the second looked at
// what it carries too.)
__device__ __forceinline__ int exponent_above(float x) {
    return max((int)((__float_as_uint(x) & 0x7fffffffu) >> 23) - 126, -100);
}
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }
// 16 bits: a score's accumulator starts at -lse / c, dP's at -delta, in the units of the
// products, so that neither is subtracted after them (their roundings, 8 u |lse|, are far
// below the types').  fp32 would take 64 such roundings of lse.
template <int DT>
constexpr bool kFold = DT != kF32;
constexpr float kUpDs = 4.0f;  // its power above 1 / the largest |dout|
constexpr int kTopDs = 15;     // and the power of two that nothing carried passes
constexpr float kUpP = 8.0f;   // fp16: the probabilities' that dV is summed from

// Lowers the power of dS where a lane's number (of its row; both halves) would pass
// 2^kTopDs: of the block ds and of the sums acc, by `down`, which is returned (0: as they
// were).  What is not finite stays what it is.
template <int NB>
__device__ __forceinline__ int lower(f32x16 &ds, f32x16 (&acc)[NB]) {
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
    if (!__any(top > pow2(kTopDs))) return 0;
    top = fmaxf(top, __shfl_xor(top, 32));
    const int down = top < INFINITY ? max(0, exponent_above(top) - kTopDs) : 0;
    const float f = pow2(-down);
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][r] *= f;
    return down;
}

// A gradient's row: where it goes, or, in splits, to split blockIdx.y's fp32 rows of
// `part`, `rows` of them, at place `at`.
template <int DT, int DP>
__device__ __forceinline__ void put_grad(const Args &a, float *part, int64_t rows, int64_t at,
                                         int splits, typename Type<DT>::T *to,
                                         const f32x16 (&x)[DP / 32], float f, int h) {
    auto each = [&](auto put) {
#pragma unroll
        for (int b = 0; b < DP / 32; ++b)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                put(32 * b + 8 * q + 4 * h, f32x4{x[b][4 * q] * f, x[b][4 * q + 1] * f,
                                                  x[b][4 * q + 2] * f, x[b][4 * q + 3] * f});
    };
    if (splits > 1) {
        float *p = part + (blockIdx.y * rows + at) * a.D;
        each([&](int d, f32x4 v) { Type<kF32>::store4(p, d, a.D, v, false); });
    } else {
        each([&](int d, f32x4 v) { Type<DT>::store4(to, d, a.D, v, a.accumulate); });
    }
}

// dQ of rows row0 .. row1 - 1, and dK and dV of keys key0 .. key1 - 1, carefully.
template <int DT>
__device__ void careful_bwd_q(const Args &a, const Seq &sq, int kv, int row0, int row1, int key0,
                              int key1, int wave, int lane) {
    using T = typename Type<DT>::T;
    const float c = a.scale * kLog2e;
    const T *k = static_cast<const T *>(a.k) + sq.k0 * a.ldk + (int64_t)kv * a.D;
    const T *v = static_cast<const T *>(a.v) + sq.k0 * a.ldv + (int64_t)kv * a.D;
    for (int row = row0 + wave; row < row1; row += 4) {
        const int i = a.group.of(row), head = kv * a.G + row - i * a.G, token = sq.q0 + i;
        const int end = min(min(key1, sq.lk), a.causal ? i + sq.lk - sq.lq + 1 : sq.lk);
        const int64_t col = (int64_t)head * a.D;
        const T *q = static_cast<const T *>(a.q) + token * a.ldq + col;
        const T *dout = static_cast<const T *>(a.dout) + token * a.lddo + col;
        // (Not from a.rows, which another split's workgroup may be writing.)
        const float lse = a.lse[(int64_t)head * a.Tq + token];
        // (As in att_bwd_q: a row of no key, or of none but scores of -inf.)
        const bool none = lse == -INFINITY;
        const int64_t rows = (int64_t)a.KV * a.Tq * a.G;
        const int64_t at = (int64_t)kv * a.Tq * a.G + sq.q0 * a.G + row;
        // A far row's lse is its maximum rounded, and little of its sum: both again, the sum
        // beside the maximum (and what the product with c rounds off).
        float lse2 = none ? INFINITY : lse * kLog2e, rest = 0.0f;
        if (is_far(lse2)) {
            const int all = a.causal ? min(sq.lk, i + sq.lk - sq.lq + 1) : sq.lk;
            float m = -INFINITY, l = 0.0f;
            for (int j0 = 0; j0 < all; j0 += 64) {
                const bool on = j0 + lane < all;
                const float x = dot<DT>(q, k + (j0 + lane) * a.ldk, a.D, on);
                const float to = fmaxf(m, wave_max(on ? x : -INFINITY));
                const float from = to == -INFINITY ? 0.0f : to;
                l = (l == 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f((m - to) * c)) +
                    wave_add(on ? __builtin_amdgcn_exp2f((x - from) * c) : 0.0f);
                m = to;
            }
            lse2 = m == -INFINITY ? INFINITY : m * c;
            rest = m == -INFINITY ? 0.0f : __builtin_fmaf(m, c, -lse2) + __log2f(l);
            if (blockIdx.y == 0 && lane == 0) {
                a.rows[at] = lse2;
                a.rows[2 * rows + at] = rest;
            }
        }
        const T *out = static_cast<const T *>(a.out) + token * a.ldo + col;
        float delta = 0.0f;
        for (int d = lane; d < a.D; d += 64)
            delta += Type<DT>::load1(dout + d) * Type<DT>::load1(out + d);
        delta = none ? 0.0f : wave_add(delta);
        float acc[2] = {0.0f, 0.0f};
        for (int j0 = key0; j0 < end; j0 += 64) {
            const int j = j0 + lane;
            const float x = dot<DT>(q, k + j * a.ldk, a.D, j < end);
            const float dp = dot<DT>(dout, v + j * a.ldv, a.D, j < end);
            const float ds =
                __builtin_amdgcn_exp2f(__builtin_fmaf(x, c, -lse2) - rest) * (dp - delta);
            for (int e = 0; e < min(64, end - j0); ++e)
                add_row<DT>(acc, __shfl(ds, e), k + (j0 + e) * a.ldk, a.D, lane);
        }
        if (a.splits > 1)
            put_row<kF32>(a.part + (blockIdx.y * rows + at) * a.D, acc, a.scale, a.D, lane, false);
        else
            put_row<DT>(static_cast<T *>(a.dq) + token * a.lddq + col, acc, a.scale, a.D, lane,
                        a.accumulate);
    }
}
template <int DT>
__device__ void careful_bwd_kv(const Args &a, const Seq &sq, int kv, int key0, int key1, int row0,
                               int row1, int wave, int lane) {
    using T = typename Type<DT>::T;
    const float c = a.scale * kLog2e;
    const int rows = min(row1, sq.lq * a.G), off = sq.lk - sq.lq;
    const T *q = static_cast<const T *>(a.q) + sq.q0 * a.ldq + (int64_t)kv * a.G * a.D;
    const T *dout = static_cast<const T *>(a.dout) + sq.q0 * a.lddo + (int64_t)kv * a.G * a.D;
    const int64_t n = (int64_t)a.KV * a.Tq * a.G, col = (int64_t)kv * a.D;
    const float *stats = a.rows + (int64_t)kv * a.Tq * a.G + sq.q0 * a.G;
    auto at = [&](const T *base, int64_t ld, int row) {
        const int i = a.group.of(row);
        return base + i * ld + (int64_t)(row - i * a.G) * a.D;
    };
    for (int key = key0 + wave; key < key1; key += 4) {
        const T *k = static_cast<const T *>(a.k) + (sq.k0 + key) * a.ldk + col;
        const T *v = static_cast<const T *>(a.v) + (sq.k0 + key) * a.ldv + col;
        float dk[2] = {0.0f, 0.0f}, dv[2] = {0.0f, 0.0f};
        for (int r0 = max(row0, a.causal ? max(0, key - off) * a.G : 0); r0 < rows; r0 += 64) {
            const int row = min(r0 + lane, rows - 1);
            const bool on = r0 + lane < rows;
            const float x = dot<DT>(k, at(q, a.ldq, row), a.D, on);
            const float dp = dot<DT>(v, at(dout, a.lddo, row), a.D, on);
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c, -stats[row]) -
                                                   stats[2 * n + row]);
            const float ds = p * (dp - stats[n + row]);
            for (int e = 0; e < min(64, rows - r0); ++e) {
                add_row<DT>(dk, __shfl(ds, e), at(q, a.ldq, r0 + e), a.D, lane);
                add_row<DT>(dv, __shfl(p, e), at(dout, a.lddo, r0 + e), a.D, lane);
            }
        }
        if (a.ksplits > 1) {
            const int64_t keys = (int64_t)a.KV * a.Tk;
            const int64_t at = blockIdx.y * keys + (int64_t)kv * a.Tk + sq.k0 + key;
            put_row<kF32>(a.kpart + at * a.D, dk, a.scale, a.D, lane, false);
            put_row<kF32>(a.kpart + (a.ksplits * keys + at) * a.D, dv, 1.0f, a.D, lane, false);
            continue;
        }
        put_row<DT>(static_cast<T *>(a.dk) + (sq.k0 + key) * a.lddk + col, dk, a.scale, a.D, lane,
                    a.accumulate);
        put_row<DT>(static_cast<T *>(a.dv) + (sq.k0 + key) * a.lddv + col, dv, 1.0f, a.D, lane,
                    a.accumulate);
    }
}

// Of a sequence's rows, 32 at a time, the record that its pass over rows leaves.
enum { kBig, kDelta, kIsFar, kRecord = 4 };
__device__ __forceinline__ float *records(const Args &a, int seq, int kv, int q0) {
    static_assert(kRows == 4 * 32, "a record a wave");
    return a.tiles + ((int64_t)kv * a.slots + q0 * a.G / kRows + seq) * (4 * kRecord);
}

// Waves that a SIMD is to hold: three of tiles of 64 columns fit, left to itself the
// compiler takes a few registers more than that for the careful way.
template <int DT, int DP>
constexpr int bwd_waves() {
    return DT == kF32 ? 1 : DP == 64 ? 3 : 2;
}

// dQ, 32 rows a wave, in the forward's layout; and for the pass over the keys, in the
// order of the key head's rows, log2 of their sums, delta and (fp16) their largest |dout|.
// bf16, 8 sequences of up to 4096, 32 heads of 128 over 8: 0.95 ms, 930 TFLOP/s of its
// three products.
template <int DT, int DP, bool DMA>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(bwd_waves<DT, DP>()))) void
att_bwd_q(const Args a) {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    constexpr int KT = keys_of<DT>(), NB = DP / 32, NK = DP / 16;
    using Tl = Tile<DT, DP, KT>;
    __shared__ __attribute__((aligned(16))) T lds[4 * Tl::kElems];
    const Work w(blockIdx.x, a.KV, a.slots);
    const Place pl = place_of(a.slots - 1 - w.slot, a.n, [&](int s) {
        return (int)min(a.qs[s], (uint32_t)a.Tq) * a.G / kRows + s;
    });
    const Seq sq(a, pl.seq);
    const int rows = sq.lq * a.G, m0 = pl.tile * kRows;
    if (pl.tile < 0 || m0 >= rows) return;  // (a slot of no tile)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, l32 = lane & 31, off = sq.lk - sq.lq;
    const float c = a.scale * kLog2e;
    const T *k = static_cast<const T *>(a.k) + sq.k0 * a.ldk + (int64_t)w.kv * a.D;
    const T *v = static_cast<const T *>(a.v) + sq.k0 * a.ldv + (int64_t)w.kv * a.D;
    auto last_of = [&](int row) {
        return a.causal ? min(sq.lk - 1, a.group.of(row) + off) : sq.lk - 1;
    };
    const int w0 = m0 + 32 * wave;
    const int wave_first = w0 < rows ? last_of(w0) : -1;
    const int wave_last = w0 < rows ? last_of(min(w0 + 32, rows) - 1) : -1;
    const int keys = last_of(min(m0 + kRows, rows) - 1) + 1;
    const int tiles = keys > 0 ? (keys - 1) / KT + 1 : 0;
    const Share share(tiles, a.splits, a.splits > 1 ? split_tiles<KT, false>(a) : 1, blockIdx.y);
    if ((int)blockIdx.y >= share.used) return;
    const int t0 = share.t0, t1 = share.t1;

    typename Ty::Frag q[NK], dout[NK];
    const int row = w0 + l32;
    const int token = sq.q0 + a.group.of(row), head = w.kv * a.G + row - (token - sq.q0) * a.G;
    const T *qrow = nullptr, *drow = nullptr, *orow = nullptr;
    if (row < rows) {
        const int64_t col = (int64_t)head * a.D;
        qrow = static_cast<const T *>(a.q) + token * a.ldq + col;
        drow = static_cast<const T *>(a.dout) + token * a.lddo + col;
        orow = static_cast<const T *>(a.out) + token * a.ldo + col;
    }
    float delta = 0.0f, big = 0.0f;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
        q[ks] = Ty::load8(qrow, 16 * ks + 8 * h, a.D);
        dout[ks] = Ty::load8(drow, 16 * ks + 8 * h, a.D);
        const typename Ty::Frag o = Ty::load8(orow, 16 * ks + 8 * h, a.D);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = Ty::get(dout[ks], j);
            delta += d * Ty::get(o, j);
            if constexpr (DT == kF16) big = fmaxf(big, fabsf(d));
        }
    }
    delta += __shfl_xor(delta, 32);
    if constexpr (DT == kF16) big = fmaxf(big, __shfl_xor(big, 32));
    // A row of no key (its lse -inf): every probability 0.
    float lse2 = INFINITY;
    bool far = false;
    if (row < rows) {
        const float x = a.lse[(int64_t)head * a.Tq + token];
        lse2 = x == -INFINITY ? INFINITY : x * kLog2e;
        far = is_far(lse2);
        if (x == -INFINITY) delta = 0.0f;
        if (h == 0 && blockIdx.y == 0) {
            const int64_t n = (int64_t)a.KV * a.Tq * a.G;
            const int64_t at = (int64_t)w.kv * a.Tq * a.G + sq.q0 * a.G + row;
            if (!far) {  // (else the careful way's)
                a.rows[at] = lse2;
                a.rows[2 * n + at] = 0.0f;
            }
            a.rows[n + at] = delta;
        }
    }
    float tile_big = 0.0f, tile_delta = 0.0f;
    if constexpr (DT == kF16) {
        tile_big = wave_max(big);
        tile_delta = wave_max(fabsf(delta));
    }
    const int last = row < rows ? last_of(row) : -1;
    int up = DT == kF16 ? (int)kUpDs - exponent_above(big) : 0;
    auto power = [&] { return (lse2 - (float)up) * (kFold<DT> ? 1.0f / c : 1.0f); };
    float from = power();

    Mover<DT, DP, KT, 256, DMA> mk, mv;
    auto load = [&](int t) {
        T *to = lds + (t & 1) * 2 * Tl::kElems;
        const int key0 = t * KT, left = sq.lk - key0;
        mk.load(to, tid, k + key0 * a.ldk, a.ldk, left, a.D);
        mv.load(to + Tl::kElems, tid, v + key0 * a.ldv, a.ldv, left, a.D);
    };
    auto store = [&](int t) {
        T *to = lds + (t & 1) * 2 * Tl::kElems;
        mk.store(to, tid);
        mv.store(to + Tl::kElems, tid);
    };
    const Lanes<DT, DP> L(lane);
    bool bad = far;  // or a tile of keys not all visible held an infinity or NaN
    f32x16 dq[NB];
    clear(dq);
    if (t0 < t1) {
        load(t0);
        store(t0);
    }
    const bool any_far = __any(far);
    if (lane == 0 && blockIdx.y == 0) {
        float *p = records(a, pl.seq, w.kv, sq.q0) + (4 * pl.tile + wave) * kRecord;
        p[kBig] = tile_big;
        p[kDelta] = tile_delta;
        p[kIsFar] = any_far;
    }
    for (int t = t0; t < t1; ++t) {
        staged<DMA>();
        if (t + 1 < t1) load(t + 1);
        const int key0 = t * KT;
        const T *kt = lds + (t & 1) * 2 * Tl::kElems, *vt = kt + Tl::kElems;
        if (key0 <= wave_last) {
            const bool whole = key0 + KT - 1 <= wave_first;
            if (!whole) bad |= !Tl::finite(kt, lane);
#pragma unroll
            for (int b = 0; b < KT / 32; ++b) {
                f32x16 s = all16(kFold<DT> ? fresh(-from) : 0.0f);
                f32x16 dp = all16(kFold<DT> ? fresh(-delta) : 0.0f);
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) {
                    s = Ty::mfma(Tl::by_row(kt, b, ks, L), q[ks], s);
                    if (Ty::kWide) dp = Ty::mfma(Tl::by_row(vt, b, ks, L), dout[ks], dp);
                }
                if (!Ty::kWide)
#pragma unroll
                    for (int ks = 0; ks < NK; ++ks)
                        dp = Ty::mfma(Tl::by_row(vt, b, ks, L), dout[ks], dp);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if constexpr (kFold<DT>)
                        s[r] = __builtin_amdgcn_exp2f(s[r] * c) * dp[r];
                    else
                        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -from)) *
                               (dp[r] - delta);
                }
                if (!whole) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int key = key0 + 32 * b + 8 * (r >> 2) + 4 * h + (r & 3);
                        s[r] = key <= last ? s[r] : 0.0f;
                    }
                }
                if constexpr (DT == kF16) {
                    if (const int down = lower(s, dq)) {
                        up -= down;
                        from = power();
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const typename Ty::Frag ds = Ty::pack(s, u);
#pragma unroll
                    for (int d = 0; d < NB; ++d)
                        dq[d] = Ty::mfma(Tl::by_column(kt, 32 * b + 16 * u, d, L), ds, dq[d]);
                }
            }
        }
        if (t + 1 < t1) store(t + 1);
    }
    if (__syncthreads_or(bad)) {
        careful_bwd_q<DT>(a, sq, w.kv, m0, min(m0 + kRows, rows), t0 * KT, t1 * KT, wave, lane);
        return;
    }
    if (row >= rows) return;
    put_grad<DT, DP>(a, a.part, (int64_t)a.KV * a.Tq * a.G,
                     (int64_t)w.kv * a.Tq * a.G + sq.q0 * a.G + row, a.splits,
                     static_cast<T *>(a.dq) + token * a.lddq + (int64_t)head * a.D, dq,
                     a.scale * pow2(-up), h);
}

// dK and dV, 32 keys a wave (a key a lane, both halves), over the rows that see them: of
// all the group's heads, so the sum over a key head's queries is one accumulator's.  K
// stays in registers and V in LDS: with both in registers there were none left to read
// ahead into (D 128: each matrix instruction waited for its LDS read, and spilled operands
// for the next tile's loads in flight; 8 sequences of up to 4096, 32 heads over 8: 2.05 ms
// and 1.6), and 64 keys a wave, for half the LDS reads, leave one wave a SIMD (2.3 ms).
// Its four products are 740 TFLOP/s, less than dQ's three by what its LDS reads (five
// operands of each tile) add beside them.  Through registers at D 128 the tiles' addresses
// spill (bf16, 4 sequences of 2048: backward 0.66 ms in all, off 16-byte boundaries 1.8).
template <int DT, int DP, bool DMA>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(bwd_waves<DT, DP>()))) void
att_bwd_kv(const Args a) {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    constexpr int RT = 32, NB = DP / 32, NK = DP / 16;
    constexpr float kUpV = DT == kF16 ? kUpP : 0.0f;
    using Tl = Tile<DT, DP, RT>;
    using Vt = Tile<DT, DP, kKeys>;
    __shared__ __attribute__((aligned(16))) T lds[4 * Tl::kElems + Vt::kElems];
    T *vlds = lds + 4 * Tl::kElems;
    __shared__ __attribute__((aligned(16))) float stats[2][3][RT];
    const Work w(blockIdx.x, a.KV, a.kslots);
    const Place pl = place_of(w.slot, a.n, [&](int s) {
        return (int)min(a.ks[s], (uint32_t)a.Tk) / kKeys + s;
    });
    const Seq sq(a, pl.seq);
    const int n0 = pl.tile * kKeys;
    if (pl.tile < 0 || n0 >= sq.lk) return;  // (a slot of no tile)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, l32 = lane & 31, off = sq.lk - sq.lq;
    const float c = a.scale * kLog2e;
    const int rows = sq.lq * a.G;
    // The first row that sees a key.
    auto first_of = [&](int key) {
        return key >= sq.lk ? rows : a.causal ? max(0, key - off) * a.G : 0;
    };
    const int begin = first_of(n0) / RT, tiles = rows > 0 ? (rows - 1) / RT + 1 - begin : 0;
    const Share share(tiles, a.ksplits, a.ksplits > 1 ? split_tiles<RT, true>(a) : 1, blockIdx.y);
    if ((int)blockIdx.y >= share.used) return;
    const int kw = n0 + 32 * wave;
    const int wave_first = first_of(kw), wave_last = first_of(kw + 31);

    typename Ty::Frag kf[NK];
    const int key = kw + l32, first = first_of(key);
    const T *krow = nullptr;
    if (key < sq.lk)
        krow = static_cast<const T *>(a.k) + (sq.k0 + key) * a.ldk + (int64_t)w.kv * a.D;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) kf[ks] = Ty::load8(krow, 16 * ks + 8 * h, a.D);
    Mover<DT, DP, RT, 256, DMA> mq, md;
    const T *qb = static_cast<const T *>(a.q) + sq.q0 * a.ldq + (int64_t)w.kv * a.G * a.D;
    const T *db = static_cast<const T *>(a.dout) + sq.q0 * a.lddo + (int64_t)w.kv * a.G * a.D;
    const int64_t n = (int64_t)a.KV * a.Tq * a.G;
    const float *rs = a.rows + (int64_t)w.kv * a.Tq * a.G + sq.q0 * a.G;
    const float *tile_at = records(a, pl.seq, w.kv, sq.q0);
    constexpr int kStats = DT == kF16 ? 3 : 2;  // fp16: a record's first two numbers too
    float sv = 0.0f;
    auto load = [&](int t) {
        T *to = lds + (t & 1) * 2 * Tl::kElems;
        const int r0 = t * RT, left = rows - r0;
        const int what = tid / RT, r = tid % RT;
        if (what < 2)  // (rows past the last: probability 0)
            sv = r < left ? rs[what * n + r0 + r] : what == 0 ? INFINITY : 0.0f;
        else if (what < kStats && r < 2)
            sv = tile_at[t * kRecord + r];
        // (From the tile's first token on.)
        const int i0 = a.group.of(r0);
        const T *qt = qb + i0 * a.ldq, *dt = db + i0 * a.lddo;
        if constexpr (DMA) {
            auto at = [&](int64_t ld, int r) {
                const int x = min(r0 + r, rows - 1), i = a.group.of(x);
                return ((uint32_t)(i - i0) * (uint32_t)ld + (uint32_t)(x - i * a.G) * a.D) *
                       (uint32_t)sizeof(T);
            };
            mq.direct(to, tid, qt, [&](int r) { return at(a.ldq, r); });
            md.direct(to + Tl::kElems, tid, dt, [&](int r) { return at(a.lddo, r); });
        } else {
            auto at = [&](const T *base, int64_t ld, int r) {
                const int x = min(r0 + r, rows - 1), i = a.group.of(x);
                return base + (i - i0) * ld + (int64_t)(x - i * a.G) * a.D;
            };
            mq.fetch(tid, left, a.D, [&](int r) { return at(qt, a.ldq, r); });
            md.fetch(tid, left, a.D, [&](int r) { return at(dt, a.lddo, r); });
        }
    };
    auto store = [&](int t) {
        T *to = lds + (t & 1) * 2 * Tl::kElems;
        mq.store(to, tid);
        md.store(to + Tl::kElems, tid);
        const int what = tid / RT;
        if (what < kStats)
            stats[t & 1][what][tid % RT] = what == 0 ? (kUpV - sv) * (kFold<DT> ? 1.0f / c : 1.0f)
                                           : what == 1 ? -sv
                                                       : sv;
    };
    const Lanes<DT, DP> L(lane);
    bool bad = false;  // a tile of rows that do not all see every key held an infinity or NaN
    f32x16 dk[NB], dv[NB];
    clear(dk);
    clear(dv);
    int up = DT == kF16 ? 100 : 0;  // fp16: the power of two that the lane's key's dK carries
    float values = 0.0f;            // and the sum of its |V|
    const int t0 = begin + share.t0, t1 = begin + share.t1;
    float far = 0.0f;  // (not looked at before the loop's end: nothing waits for it)
    if (t0 < t1) {
        if (t0 + tid < t1) far = tile_at[(t0 + tid) * kRecord + kIsFar];
        for (int t = t0 + tid + 256; t < t1; t += 256) far += tile_at[t * kRecord + kIsFar];
        Mover<DT, DP, kKeys, 256, DMA> mv;
        mv.load(vlds, tid,
                static_cast<const T *>(a.v) + (sq.k0 + n0) * a.ldv + (int64_t)w.kv * a.D, a.ldv,
                sq.lk - n0, a.D);
        mv.store(vlds, tid);
        load(t0);
        store(t0);
        if constexpr (DT == kF16) {
            staged<DMA>();
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) {
                const typename Ty::Frag f = Vt::by_row(vlds, wave, ks, L);
#pragma unroll
                for (int j = 0; j < 8; ++j) values += fabsf(Ty::get(f, j));
            }
            values += __shfl_xor(values, 32);
        }
    }
    for (int t = t0; t < t1; ++t) {
        staged<DMA>();
        if (t + 1 < t1) load(t + 1);
        const int r0 = t * RT;
        const T *qt = lds + (t & 1) * 2 * Tl::kElems, *dt = qt + Tl::kElems;
        const float *st = stats[t & 1][0];
        if (r0 + RT > wave_first) {
            const bool whole = r0 >= wave_last && r0 + RT <= rows;
            if (!whole) bad |= !(Tl::finite(qt, lane) && Tl::finite(dt, lane));
            float fs = 1.0f;
            if constexpr (DT == kF16) {
                const float big = st[2 * RT + kBig];
                const int e = min((int)kUpDs - exponent_above(big),
                                  kTopDs - exponent_above(big * values + st[2 * RT + kDelta]));
                if (__any(e < up)) {
                    const float f = pow2(min(e - up, 0));
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) dk[b][r] *= f;
                    up = min(e, up);
                }
                fs = pow2(up - (int)kUpP);
            }
            f32x16 p = kFold<DT> ? rows16(st + 4 * h) : all16(0.0f);
            f32x16 dp = kFold<DT> ? rows16(st + RT + 4 * h) : all16(0.0f);
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) {
                p = Ty::mfma(Tl::by_row(qt, 0, ks, L), kf[ks], p);
                if (Ty::kWide)
                    dp = Ty::mfma(Tl::by_row(dt, 0, ks, L), Vt::by_row(vlds, wave, ks, L), dp);
            }
            if (!Ty::kWide)
#pragma unroll
                for (int ks = 0; ks < NK; ++ks)
                    dp = Ty::mfma(Tl::by_row(dt, 0, ks, L), Vt::by_row(vlds, wave, ks, L), dp);
            if constexpr (!Ty::kWide) {
                // Three ahead, after the rows' eight: dP's products take two reads each.
                // (1.65 -> 1.59 ms; dQ's and the forward's scores gained nothing.)
                reads<8 + 3>();
                products<NK - 3, 1>();
                products<NK, 2>();
                products<3, 0>();
            }
            if constexpr (kFold<DT>) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[r] = __builtin_amdgcn_exp2f(p[r] * c);
                    dp[r] = p[r] * (DT == kF16 ? dp[r] * fs : dp[r]);
                }
            } else {
                const f32x16 lse = rows16(st + 4 * h), delta = rows16(st + RT + 4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], c, lse[r]));
                    dp[r] = p[r] * (dp[r] + delta[r]);
                }
            }
            if (!whole) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int x = r0 + 8 * (r >> 2) + 4 * h + (r & 3);
                    const bool on = x >= first && x < rows;
                    p[r] = on ? p[r] : 0.0f;
                    dp[r] = on ? dp[r] : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename Ty::Frag f = Ty::pack(p, u);
#pragma unroll
                for (int d = 0; d < NB; ++d)
                    dv[d] = Ty::mfma(Tl::by_column(dt, 16 * u, d, L), f, dv[d]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const typename Ty::Frag f = Ty::pack(dp, u);
#pragma unroll
                for (int d = 0; d < NB; ++d)
                    dk[d] = Ty::mfma(Tl::by_column(qt, 16 * u, d, L), f, dk[d]);
            }
        }
        if (t + 1 < t1) store(t + 1);
    }
    if (__syncthreads_or(bad || far != 0.0f)) {
        careful_bwd_kv<DT>(a, sq, w.kv, n0, min(n0 + kKeys, sq.lk), t0 * RT, t1 * RT, wave, lane);
        return;
    }
    if (key >= sq.lk) return;
    const int64_t keys = (int64_t)a.KV * a.Tk, at = (int64_t)w.kv * a.Tk + sq.k0 + key;
    const int64_t col = (int64_t)w.kv * a.D;
    put_grad<DT, DP>(a, a.kpart, keys, at, a.ksplits,
                     static_cast<T *>(a.dk) + (sq.k0 + key) * a.lddk + col, dk,
                     a.scale * pow2(-up), h);
    put_grad<DT, DP>(a, a.kpart + a.ksplits * keys * a.D, keys, at, a.ksplits,
                     static_cast<T *>(a.dv) + (sq.k0 + key) * a.lddv + col, dv, pow2(-(int)kUpV),
                     h);
}

// The splits' gradients added in order, a wave a row: of dQ, then dK, then dV, those that
// are in splits.  Rows of no sequence are left.
template <int DT>
__global__ __launch_bounds__(256) void att_bwd_combine(const Args a) {
    using Ty = Type<DT>;
    using T = typename Ty::T;
    const int lane = threadIdx.x & 63;
    const int64_t rows = a.splits > 1 ? (int64_t)a.KV * a.Tq * a.G : 0;
    const int64_t keys = a.ksplits > 1 ? (int64_t)a.KV * a.Tk : 0;
    int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= rows + 2 * keys) return;
    const float *p;
    T *to;
    int64_t step;
    int splits;
    if (at < rows) {
        const int kv = (int)(at / ((int64_t)a.Tq * a.G));
        const int row = (int)(at - (int64_t)kv * a.Tq * a.G), token = a.group.of(row);
        const Place pl =
            place_of(token, a.n, [&](int s) { return (int)min(a.qs[s], (uint32_t)a.Tq); });
        const Seq sq(a, pl.seq);
        if (token < sq.q0 || token >= sq.q0 + sq.lq) return;
        to = static_cast<T *>(a.dq) + token * a.lddq +
             (int64_t)(kv * a.G + row - token * a.G) * a.D;
        p = a.part + at * a.D;
        step = rows * a.D;
        // (The tiles of its workgroup in the pass over the rows.)
        constexpr int KT = keys_of<DT>();
        const int all = sq.lq * a.G;
        const int end = min(((token - sq.q0) * a.G + row - token * a.G) / kRows * kRows + kRows, all);
        const int keys =
            a.causal ? min(sq.lk, a.group.of(end - 1) + sq.lk - sq.lq + 1) : sq.lk;
        splits = Share(keys > 0 ? (keys - 1) / KT + 1 : 0, a.splits, split_tiles<KT, false>(a), 0).used;
    } else {
        at -= rows;
        const bool value = at >= keys;
        if (value) at -= keys;
        const int kv = (int)(at / a.Tk), key = (int)(at - (int64_t)kv * a.Tk);
        const Place pl =
            place_of(key, a.n, [&](int s) { return (int)min(a.ks[s], (uint32_t)a.Tk); });
        const Seq sq(a, pl.seq);
        if (key < sq.k0 || key >= sq.k0 + sq.lk) return;
        to = (value ? static_cast<T *>(a.dv) + key * a.lddv : static_cast<T *>(a.dk) + key * a.lddk) +
             (int64_t)kv * a.D;
        p = a.kpart + ((value ? a.ksplits * keys : 0) + at) * a.D;
        step = keys * a.D;
        const int all = sq.lq * a.G, n0 = (key - sq.k0) / kKeys * kKeys;
        const int begin = (a.causal ? max(0, n0 - (sq.lk - sq.lq)) * a.G : 0) / 32;
        splits = Share(all > 0 ? (all - 1) / 32 + 1 - begin : 0, a.ksplits,
                       split_tiles<32, true>(a), 0)
                     .used;
    }
    float acc[2] = {0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 64 * i < a.D) acc[i] += p[s * step + lane + 64 * i];
    put_row<DT>(to, acc, 1.0f, a.D, lane, a.accumulate);
}

// ------------------------------------------------------------------ launches
template <int DT, class F>
void with_width(int D, bool dma, F f) {
    using std::integral_constant;
    constexpr bool kDma = DT != kF32;
    auto with = [&](auto dp) {
        if (kDma && dma) f(dp, std::integral_constant<bool, kDma>{});
        else f(dp, std::false_type{});
    };
    if (D <= 64) with(integral_constant<int, 64>{});
    else if (D <= 96) f(integral_constant<int, 96>{}, std::false_type{});
    else with(integral_constant<int, 128>{});
}

template <int DT, class F>
void with_few(int D, F f) {
    using std::integral_constant;
    auto with = [&](auto dp) {
        if (D == dp()) f(dp, std::true_type{});
        else f(dp, std::false_type{});
    };
    if (D <= 64) with(integral_constant<int, 64>{});
    else if (D <= 96) with(integral_constant<int, 96>{});
    else with(integral_constant<int, 128>{});
}

template <int DT>
int forward(hipStream_t st, const Args &a, bool few, bool dma) {
    const dim3 grid(a.KV * a.slots, a.splits);
    with_width<DT>(a.D, dma, [&](auto dp, auto d) {
        if (!few) att_fwd<DT, dp(), d()><<<grid, 256, 0, st>>>(a);
    });
    if (few) with_few<DT>(a.D, [&](auto dp, auto full) {
        att_fwd_few<DT, dp(), full()><<<grid, 256, 0, st>>>(a);
    });
    return (int)hipGetLastError();
}
template <int DT>
int combine(hipStream_t st, const Args &a) {
    att_combine<DT><<<((int64_t)a.KV * a.Tq * a.G - 1) / 4 + 1, 256, 0, st>>>(a);
    return (int)hipGetLastError();
}
template <int DT>
int backward(hipStream_t st, const Args &a, bool dma) {
    with_width<DT>(a.D, dma, [&](auto dp, auto d) {
        att_bwd_q<DT, dp(), d()><<<dim3(a.KV * a.slots, a.splits), 256, 0, st>>>(a);
        att_bwd_kv<DT, dp(), d()><<<dim3(a.KV * a.kslots, a.ksplits), 256, 0, st>>>(a);
    });
    const int64_t rows = (a.splits > 1 ? (int64_t)a.KV * a.Tq * a.G : 0) +
                         (a.ksplits > 1 ? 2 * (int64_t)a.KV * a.Tk : 0);
    if (rows) att_bwd_combine<DT><<<(rows - 1) / 4 + 1, 256, 0, st>>>(a);
    return (int)hipGetLastError();
}

}  // namespace attn
}  // namespace fg
