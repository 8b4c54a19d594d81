// k_rms_norm.hip -- RMS norm over the last dimension with the residual's addition,
// y in 8 bits beside it where asked, and the backward pass, for gfx950.  The
// reference has no normalisation; its row operator is the softmax node
// (crates/ferrograd-nn/src/op/softmax.rs:14-759).
//
// Forward, for a row of C elements:
//   s = x + r, rounded to the tensors' type (without r: s = x)
//   rstd = 1 / sqrt(sum(s^2) / C + eps),  y = s * rstd * gamma
//   8 bits: k_ckpt8.hip's form of y, from its fp32 values (y itself is rounded)
// Backward, with xh = s * rstd and g = dy * gamma:
//   dx = rstd * (g - xh * mean(g * xh)) + ds,  dgamma = sum over rows of dy * xh
// (dx is x's gradient and r's: s passes it to both.)  Sums are fp32, each output is
// rounded once.
//
// Both directions are bound by HBM: a row is read once, held in registers between its
// sum and its output, and written once.  bf16, 16384 x 4096 with a residual: forward 77 us,
// with the 8 bits 95 (606 MB), backward 96 (537 MB, 5.6 TB/s; a large copy reaches 4.9);
// fp32 rows of 2051 at odd strides, 4099 of them, backward 31 us.  32 x 4096: 5 us, of
// which the kernel is 3.6.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "fg_bits8.h"
#include "fg_half.h"
#include "fg_internal.h"
#include "fg_rows.h"

namespace {

using fg::bits8::Bytes;
using fg::rows::apart;
using fg::rows::Io;
using fg::rows::Tail;
using fg::rows::u32x4;

template <class T>
struct Fwd {
    const T *x, *r, *gamma;
    T *s, *y;
    int8_t *q;
    uint8_t *e;
    float *rstd, eps;
    int ldx, ldr, lds, ldy, ldq, lde, R, C;
};
template <class T>
struct Bwd {
    const T *s, *dy, *gamma, *ds;
    const float *rstd;
    T *dx;
    float *partial;
    int lds, lddy, ldds, lddx, R, C;
    int rows;  // of a split of rms_bwd_cols
};

// The sum over a row's L lanes (whole waves), the same in every lane.  Waves wait at
// one barrier; sm: a float per wave, which nothing of the sum before the last uses.
template <int L>
__device__ __forceinline__ float row_sum(float v, float *sm, int t) {
    if constexpr (L == 16) return fg::smrow::row16_sum(v);
    v = fg::rows::wave_sum(v);
    if constexpr (L > 64) {
        if ((t & 63) == 0) sm[t >> 6] = v;
        __syncthreads();
        v = sm[0];
#pragma unroll
        for (int k = 1; k < L / 64; ++k) v += sm[k];
    }
    return v;
}

// Chunk j of a row of C columns: its values, zeros past the row's end.  own: the first
// of them that is the chunk's own (the row's last chunk may begin with columns of the
// one before it, fg::rows::Tail).
template <int DT>
struct Piece {
    static constexpr int E = Io<DT>::E;
    Tail<DT> tail;
    int own;
    bool in;
    __device__ __forceinline__ Piece(int j, int C)
        : tail(j, C), own(j * E - tail.first), in(j * E < C) {}
    template <class T>
    __device__ __forceinline__ u32x4 load(const T *row) const {
        return in ? tail.load(row) : u32x4{0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ bool mine(int e) const { return e >= own; }
    // The chunk's own columns and no others: for a row that other lanes still read.
    template <class T>
    __device__ __forceinline__ void store_own(T *row, const float (&v)[E]) const {
        if (own == 0) {
            tail.store(row, v);
            return;
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (mine(e)) Io<DT>::store1(row, tail.first + e, v[e]);
    }
};

// ------------------------------------------------------------------ forward
// What a row's chunk writes: s, y and the 8 bits, from the row's rstd.  Every lane
// calls it (a block's lanes exchange its largest value).  OWN: no column that another
// chunk's lane may still have to read.
template <int DT, bool OWN = false>
__device__ __forceinline__ void write_chunk(const Fwd<typename Io<DT>::T> &a, size_t row, int j,
                                            bool in, const Piece<DT> &p, u32x4 w, float rs) {
    using IO = Io<DT>;
    constexpr int E = IO::E;
    float v[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = IO::get(w, e);
    const u32x4 g = a.gamma ? p.load(a.gamma) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = v[e] * rs * (a.gamma ? IO::get(g, e) : 1.0f);
    if (in && p.in) {
        if (a.s) {
            if constexpr (OWN) p.store_own(a.s + row * a.lds, v);
            else p.tail.store(a.s + row * a.lds, v);
        }
        if (a.y) {
            if constexpr (OWN) p.store_own(a.y + row * a.ldy, o);
            else p.tail.store(a.y + row * a.ldy, o);
        }
    }
    if (!a.q) return;
    // The chunk's own columns from its first element on.
    float own[E];
#pragma unroll
    for (int e = 0; e < E; ++e) own[e] = p.in ? o[e] : 0.0f;
    if (p.own > 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float c = 0.0f;
#pragma unroll
            for (int k = 0; k < E; ++k) c = k == e + p.own ? o[k] : c;
            own[e] = p.in ? c : 0.0f;
        }
    }
    Bytes<E> bytes;
    const int b = fg::bits8::quantise<E>(own, bytes);
    if (!in || !p.in) return;
    bytes.store(a.q + row * a.ldq, j, a.C / E, a.C);
    constexpr int kLanes = fg::bits8::kBlock / E;
    if (j % kLanes == 0) a.e[row * a.lde + j / kLanes] = (uint8_t)b;
}

// The chunk of s, as stored, and its squares' sum.
template <int DT>
__device__ __forceinline__ u32x4 read_chunk(const Fwd<typename Io<DT>::T> &a, size_t row,
                                            bool in, const Piece<DT> &p, float &sum) {
    using IO = Io<DT>;
    constexpr int E = IO::E;
    u32x4 w = {0u, 0u, 0u, 0u};
    if (in) w = p.load(a.x + row * a.ldx);
    if (a.r && in) {
        const u32x4 r = p.load(a.r + row * a.ldr);
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = IO::get(w, e) + IO::get(r, e);
        w = IO::pack(v);
    }
    float q = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float v = IO::get(w, e);
        q += p.mine(e) ? v * v : 0.0f;
    }
    sum += q;
    return w;
}

// A row in registers of L lanes, NV chunks a lane, NG rows a workgroup.  Outputs go out
// after the row's sum, so that they may be x or r: a row's last chunk reads columns that
// another lane writes.
template <int DT, int NV, int L, int NG>
__global__ __launch_bounds__(L *NG) void rms_fwd(const Fwd<typename Io<DT>::T> a) {
    __shared__ float sm[NG][(L + 63) / 64];
    const int grp = threadIdx.x / L, t = threadIdx.x % L;
    const size_t row = (size_t)blockIdx.x * NG + grp;
    const bool in = row < (size_t)a.R;
    u32x4 w[NV];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        w[i] = read_chunk<DT>(a, row, in, Piece<DT>(t + i * L, a.C), sum);
    const float rs = 1.0f / sqrtf(row_sum<L>(sum, sm[grp], t) / (float)a.C + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
        write_chunk<DT>(a, row, t + i * L, in, Piece<DT>(t + i * L, a.C), w[i], rs);
    if (a.rstd && in && t == 0) a.rstd[row] = rs;
}

// Rows longer than registers hold: the second pass reads x and r again, the row's last
// chunk before anything is written over the one before it.
constexpr int kLongL = 1024;
template <int DT>
__global__ __launch_bounds__(kLongL) void rms_fwd_long(const Fwd<typename Io<DT>::T> a) {
    __shared__ float sm[kLongL / 64];
    const int t = threadIdx.x;
    const size_t row = blockIdx.x;
    constexpr int E = Io<DT>::E;
    const int chunks = (a.C - 1) / E + 1;
    float sum = 0.0f;
    for (int j = t; j < chunks; j += kLongL) read_chunk<DT>(a, row, true, Piece<DT>(j, a.C), sum);
    const float rs = 1.0f / sqrtf(row_sum<kLongL>(sum, sm, t) / (float)a.C + a.eps);
    const Piece<DT> last(chunks - 1, a.C);
    float unused = 0.0f;
    const u32x4 wl = read_chunk<DT>(a, row, true, last, unused);
    __syncthreads();
    for (int j0 = 0; j0 < chunks; j0 += kLongL) {  // (all lanes of a block, to the last)
        const int j = j0 + t;
        const Piece<DT> p(j, a.C);
        const u32x4 w = j == chunks - 1 ? wl : read_chunk<DT>(a, row, true, p, unused);
        write_chunk<DT, true>(a, row, j, true, p, w, rs);
    }
    if (a.rstd && t == 0) a.rstd[row] = rs;
}

// ----------------------------------------------------------------- backward
// The row in registers; dgamma's sums of a lane's columns stay in its registers over
// the workgroup's rows and go out once, as partial[workgroup][C]: a CU's worth of threads
// (512), so that the partial sums are few (4 MB beside 537 at 16384 x 4096 of bf16).
template <int DT, int NV, int L, int NG>
__global__ __launch_bounds__(L *NG) void rms_bwd(const Bwd<typename Io<DT>::T> a) {
    using IO = Io<DT>;
    constexpr int E = IO::E;
    __shared__ float sm[2][NG][(L + 63) / 64];
    extern __shared__ float cols[];  // [C], NG > 1
    const int grp = threadIdx.x / L, t = threadIdx.x % L;
    float ag[NV][E];
    u32x4 g[NV], ws[NV], wd[NV], wr[NV];
    float rs = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (a.gamma) g[i] = Piece<DT>(t + i * L, a.C).load(a.gamma);
#pragma unroll
        for (int e = 0; e < E; ++e) ag[i][e] = 0.0f;
    }
    const size_t rows = a.R, step = (size_t)gridDim.x * NG;
    size_t row = (size_t)blockIdx.x * NG + grp;
    auto fetch = [&](size_t r) {
        const bool in = r < rows;
        rs = in ? a.rstd[r] : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Piece<DT> p(t + i * L, a.C);
            const u32x4 zero = {0u, 0u, 0u, 0u};
            ws[i] = in ? p.load(a.s + r * a.lds) : zero;
            wd[i] = in ? p.load(a.dy + r * a.lddy) : zero;
            wr[i] = in && a.ds ? p.load(a.ds + r * a.ldds) : zero;
        }
    };
    fetch(row);
    int it = 0;
    for (size_t r0 = (size_t)blockIdx.x * NG; r0 < rows; r0 += step, ++it) {
        u32x4 vs[NV], vd[NV], vr[NV];
        const float k = rs;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            vs[i] = ws[i];
            vd[i] = wd[i];
            vr[i] = wr[i];
            const Piece<DT> p(t + i * L, a.C);
            float q = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = IO::get(vd[i], e), s = IO::get(vs[i], e);
                const float gd = a.gamma ? d * IO::get(g[i], e) : d;
                q += p.mine(e) ? gd * s : 0.0f;
                ag[i][e] += d * (s * k);
            }
            sum += q;
        }
        const size_t at = row;
        row += step;
        if (r0 + step < rows) fetch(row);
        const float mean = row_sum<L>(sum, sm[it & 1][grp], t) * k / (float)a.C;
        if (a.dx && at < rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const Piece<DT> p(t + i * L, a.C);
                if (!p.in) continue;
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = IO::get(vd[i], e);
                    const float gd = a.gamma ? d * IO::get(g[i], e) : d;
                    o[e] = k * (gd - IO::get(vs[i], e) * k * mean);
                    if (a.ds) o[e] += IO::get(vr[i], e);
                }
                p.tail.store(a.dx + at * a.lddx, o);
            }
        }
    }
    if (!a.partial) return;
    float *out = a.partial + (size_t)blockIdx.x * a.C;
    if constexpr (NG > 1) {
        // The groups' sums, in order.
        for (int n = 0; n < NG; ++n) {
            if (grp == n) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const Piece<DT> p(t + i * L, a.C);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int c = p.tail.first + e;
                        if (p.in && p.mine(e) && c < a.C)
                            cols[c] = n == 0 ? ag[i][e] : cols[c] + ag[i][e];
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.C; c += L * NG) out[c] = cols[c];
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Piece<DT> p(t + i * L, a.C);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (p.in && p.mine(e) && p.tail.first + e < a.C) out[p.tail.first + e] = ag[i][e];
        }
    }
}

// Longer rows: dgamma's sums by columns first (dx may replace what they read), then a
// workgroup a row, whose second pass reads the row again.
constexpr int kColsNT = 256;
template <int DT>
__global__ __launch_bounds__(kColsNT) void rms_bwd_cols(const Bwd<typename Io<DT>::T> a) {
    using IO = Io<DT>;
    constexpr int E = IO::E;
    const Piece<DT> p(blockIdx.x * kColsNT + threadIdx.x, a.C);
    if (!p.in) return;
    float ag[E] = {};
    const int r0 = blockIdx.y * a.rows, r1 = min(a.R, r0 + a.rows);
#pragma unroll 4
    for (int r = r0; r < r1; ++r) {
        const u32x4 s = p.load(a.s + (size_t)r * a.lds), d = p.load(a.dy + (size_t)r * a.lddy);
        const float k = a.rstd[r];
#pragma unroll
        for (int e = 0; e < E; ++e) ag[e] += IO::get(d, e) * (IO::get(s, e) * k);
    }
    float *out = a.partial + (size_t)blockIdx.y * a.C;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (p.mine(e) && p.tail.first + e < a.C) out[p.tail.first + e] = ag[e];
}
template <int DT>
__global__ __launch_bounds__(kLongL) void rms_bwd_long(const Bwd<typename Io<DT>::T> a) {
    using IO = Io<DT>;
    constexpr int E = IO::E;
    __shared__ float sm[kLongL / 64];
    const int t = threadIdx.x;
    const size_t row = blockIdx.x;
    const auto *sr = a.s + row * a.lds, *dr = a.dy + row * a.lddy;
    const auto *er = a.ds ? a.ds + row * a.ldds : nullptr;
    const int chunks = (a.C - 1) / E + 1;
    const float k = a.rstd[row];
    float sum = 0.0f;
    for (int j = t; j < chunks; j += kLongL) {
        const Piece<DT> p(j, a.C);
        const u32x4 s = p.load(sr), d = p.load(dr);
        const u32x4 g = a.gamma ? p.load(a.gamma) : s;
        float q = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float gd = a.gamma ? IO::get(d, e) * IO::get(g, e) : IO::get(d, e);
            q += p.mine(e) ? gd * IO::get(s, e) : 0.0f;
        }
        sum += q;
    }
    const float mean = row_sum<kLongL>(sum, sm, t) * k / (float)a.C;
    // The row's last chunk before anything is written over the one before it.
    const Piece<DT> last(chunks - 1, a.C);
    const u32x4 zero = {0u, 0u, 0u, 0u};
    const u32x4 ls = last.load(sr), ld = last.load(dr), lr = er ? last.load(er) : zero;
    __syncthreads();
    for (int j = t; j < chunks; j += kLongL) {
        const Piece<DT> p(j, a.C);
        const bool end = j == chunks - 1;
        const u32x4 s = end ? ls : p.load(sr), d = end ? ld : p.load(dr);
        const u32x4 r = end ? lr : er ? p.load(er) : zero;
        const u32x4 g = a.gamma ? p.load(a.gamma) : s;
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float gd = a.gamma ? IO::get(d, e) * IO::get(g, e) : IO::get(d, e);
            o[e] = k * (gd - IO::get(s, e) * k * mean);
            if (er) o[e] += IO::get(r, e);
        }
        p.store_own(a.dx + row * a.lddx, o);
    }
}

// dgamma[c] (=|+=) the splits' sums in a fixed order: 32 columns by 32 groups of
// splits, then the groups.
__global__ __launch_bounds__(1024) void rms_bwd_final(const float *__restrict__ partial,
                                                      void *dgamma, int dtype, int splits, int C,
                                                      int accumulate) {
    __shared__ float sm[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float s = 0.0f;
    if (c < C)
        for (int k = y; k < splits; k += 32) s += partial[(size_t)k * C + c];
    sm[y][x] = s;
    __syncthreads();
    if (y || c >= C) return;
#pragma unroll
    for (int k = 1; k < 32; ++k) s += sm[k][x];
    if (accumulate) s += fg::load_as_f(dgamma, dtype, c);
    fg::store_from_f(dgamma, dtype, c, s);
}

// ------------------------------------------------------------------ launches
// f(chunks a lane, lanes of a row, rows of a workgroup) for rows of `chunks` chunks;
// false: none holds them.  The first that does: idle lanes cost more than idle chunks
// (16384 x 4096 bf16 forward, 512 chunks: 256 lanes of two 77 us, of four 78, 512 lanes of
// four 88); rows longer than all are read twice (1024 x 65536: held 83 us, read twice 113).
template <class F>
bool fwd_kind(int chunks, F f) {
    auto with = [&](auto nv, auto l, auto ng) {
        if (chunks > nv() * l()) return false;
        f(nv, l, ng);
        return true;
    };
    using std::integral_constant;
#define FG_RMS(NV, L, NG)                                                           \
    with(integral_constant<int, NV>{}, integral_constant<int, L>{}, \
         integral_constant<int, NG>{})
    return FG_RMS(1, 16, 16) || FG_RMS(1, 64, 4) || FG_RMS(2, 64, 4) || FG_RMS(2, 256, 1) ||
           FG_RMS(4, 256, 1) || FG_RMS(4, 512, 1) || FG_RMS(4, 1024, 1) || FG_RMS(8, 1024, 1);
}
// LONGER: rows of up to 2048 chunks too, for fp32 (4096 x 8192: 103 us, the longer rows'
// kernels 142); 16-bit rows of as many chunks have twice the columns' sums (4096 x 16384:
// 192 us and 151).
template <bool LONGER, class F>
bool bwd_kind(int chunks, F f) {
    auto with = [&](auto nv, auto l, auto ng) {
        if (chunks > nv() * l()) return false;
        f(nv, l, ng);
        return true;
    };
    using std::integral_constant;
    if (FG_RMS(1, 16, 32) || FG_RMS(1, 64, 8) || FG_RMS(1, 128, 4) || FG_RMS(1, 256, 2) ||
        FG_RMS(1, 512, 1) || FG_RMS(2, 512, 1))
        return true;
    if constexpr (LONGER) return FG_RMS(2, 1024, 1);
    return false;
}
#undef FG_RMS

int chunks_of(int dtype, int C) { return (C - 1) / (dtype == FG_DTYPE_F32 ? 4 : 8) + 1; }

// How a backward's rows are shared out: workgroups of the held rows, or splits of the
// long rows' columns.
struct Split {
    int splits = 0, rows = 0, strips = 0;
    bool held = false;
};
Split split_of(int cus, int dtype, int R, int C) {
    Split s;
    const int chunks = chunks_of(dtype, C);
    auto share = [&](auto, auto l, auto ng) {
        const int per_cu = std::max(1, 512 / (l() * ng()));
        s.splits = std::min(R > 0 ? (R - 1) / ng() + 1 : 0, cus * per_cu);
    };
    s.held = dtype == FG_DTYPE_F32 ? bwd_kind<true>(chunks, share) : bwd_kind<false>(chunks, share);
    if (s.held) return s;
    s.strips = (chunks - 1) / kColsNT + 1;
    const int want = std::max(1, std::min((4 * cus - 1) / s.strips + 1, (R + 15) / 16));
    s.rows = R > 0 ? (R - 1) / want + 1 : 1;
    s.splits = R > 0 ? (R - 1) / s.rows + 1 : 0;
    return s;
}

template <int DT>
void launch_fwd(fg_ctx *ctx, Fwd<void> v) {
    using T = typename Io<DT>::T;
    const Fwd<T> a{static_cast<const T *>(v.x), static_cast<const T *>(v.r),
                   static_cast<const T *>(v.gamma), static_cast<T *>(v.s), static_cast<T *>(v.y),
                   v.q, v.e, v.rstd, v.eps, v.ldx, v.ldr, v.lds, v.ldy, v.ldq, v.lde, v.R, v.C};
    if (!fwd_kind((a.C - 1) / Io<DT>::E + 1, [&](auto nv, auto l, auto ng) {
            rms_fwd<DT, nv(), l(), ng()>
                <<<(a.R - 1) / ng() + 1, l() * ng(), 0, ctx->stream>>>(a);
        }))
        rms_fwd_long<DT><<<a.R, kLongL, 0, ctx->stream>>>(a);
}

template <int DT>
int launch_bwd(fg_ctx *ctx, const Split &s, Bwd<void> v) {
    using T = typename Io<DT>::T;
    const Bwd<T> a{static_cast<const T *>(v.s), static_cast<const T *>(v.dy),
                   static_cast<const T *>(v.gamma), static_cast<const T *>(v.ds), v.rstd,
                   static_cast<T *>(v.dx), v.partial, v.lds, v.lddy, v.ldds, v.lddx, v.R, v.C,
                   s.rows};
    hipStream_t st = ctx->stream;
    if (s.held) {
        bwd_kind<DT == fg::kF32>((a.C - 1) / Io<DT>::E + 1, [&](auto nv, auto l, auto ng) {
            const size_t lds = ng() > 1 && a.partial ? (size_t)a.C * sizeof(float) : 0;
            rms_bwd<DT, nv(), l(), ng()><<<s.splits, l() * ng(), lds, st>>>(a);
        });
        FG_LAUNCH_CHECK("rms_bwd");
        return FG_OK;
    }
    if (a.partial) {
        rms_bwd_cols<DT><<<dim3(s.strips, s.splits), kColsNT, 0, st>>>(a);
        FG_LAUNCH_CHECK("rms_bwd_cols");
    }
    if (a.dx) {
        rms_bwd_long<DT><<<a.R, kLongL, 0, st>>>(a);
        FG_LAUNCH_CHECK("rms_bwd_long");
    }
    return FG_OK;
}

}  // namespace

namespace fg {
uint64_t rms_norm_bwd_ws_bytes(int cus, int dtype, int R, int C) {
    return (uint64_t)std::max(split_of(cus > 0 ? cus : 256, dtype, R, C).splits, 1) * (uint64_t)C *
           sizeof(float);
}
int rms_norm_bwd_dispatches(int cus, int dtype, int R, int C, bool dx, bool weights) {
    const Split s = split_of(cus > 0 ? cus : 256, dtype, R, C);
    return (s.held ? (int)(dx || weights) : (int)dx + (int)weights) + (int)weights;
}
}  // namespace fg

FG_API int fg_rms_norm(fg_ctx *ctx, int dtype, const void *d_x, int ldx, const void *d_r, int ldr,
                       const void *d_gamma, float eps, int R, int C, void *d_s, int lds, void *d_y,
                       int ldy, int8_t *d_q, int ldq, uint8_t *d_e, int lde, float *d_rstd) {
    const char *who = "fg_rms_norm";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape R=%d C=%d", who, R, C);
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(d_x && (d_y || d_q), FG_ERR_INVALID_ARGUMENT,
               "%s: x and y (or its 8 bits) are required", who);
    FG_REQUIRE((d_q == nullptr) == (d_e == nullptr), FG_ERR_INVALID_ARGUMENT,
               "%s: the 8 bits need their elements and their exponents", who);
    FG_REQUIRE((d_r == nullptr) == (d_s == nullptr), FG_ERR_INVALID_ARGUMENT,
               "%s: r needs s, where the sum is kept, and s needs r", who);
    FG_REQUIRE(ldx >= C && (!d_r || (ldr >= C && lds >= C)) && (!d_y || ldy >= C), FG_ERR_SHAPE,
               "%s: ldx=%d, ldr=%d, lds=%d or ldy=%d < C=%d", who, ldx, ldr, lds, ldy, C);
    FG_REQUIRE(!d_q || (ldq >= C && lde >= (C - 1) / fg::bits8::kBlock + 1), FG_ERR_SHAPE,
               "%s: ldq=%d or lde=%d too small for C=%d", who, ldq, lde, C);
    FG_REQUIRE(eps > 0.0f && eps < INFINITY, FG_ERR_INVALID_ARGUMENT,
               "%s: eps must be positive and finite", who);
    FG_REQUIRE((d_y != d_x || ldy == ldx) && (!d_r || d_y != d_r || ldy == ldr) &&
                   (!d_s || d_s != d_x || lds == ldx) && (!d_s || d_s != d_r || lds == ldr),
               FG_ERR_INVALID_ARGUMENT,
               "%s: y or s is x or r, but of another leading dimension", who);
    FG_REQUIRE(fg::rows::grid_holds(R, kLongL), FG_ERR_OUT_OF_BOUNDS, "%s: %d rows of %d columns",
               who, R, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_y, {d_gamma, d_s, d_q, d_e, d_rstd}) &&
                   apart(d_s, {d_gamma, d_q, d_e, d_rstd}) &&
                   apart(d_q, {d_x, d_r, d_gamma, d_e, d_rstd}) &&
                   apart(d_e, {d_x, d_r, d_gamma, d_rstd}) && apart(d_rstd, {d_x, d_r, d_gamma}),
               FG_ERR_INVALID_ARGUMENT,
               "%s: an output is another output or an input but x or r", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const Fwd<void> a{d_x, d_r, d_gamma, d_s, d_y, d_q, d_e, d_rstd, eps,
                      ldx, ldr, lds, ldy, ldq, lde, R, C};
    if (dtype == FG_DTYPE_F32) launch_fwd<fg::kF32>(ctx, a);
    else if (dtype == FG_DTYPE_BF16) launch_fwd<fg::kBF16>(ctx, a);
    else launch_fwd<fg::kF16>(ctx, a);
    FG_LAUNCH_CHECK("rms_fwd");
    return FG_OK;
}

FG_API int fg_rms_norm_bwd(fg_ctx *ctx, int dtype, const void *d_s, int lds, const void *d_dy,
                           int lddy, const void *d_gamma, const float *d_rstd, int R, int C,
                           const void *d_ds, int ldds, void *d_dx, int lddx, void *d_dgamma,
                           int dgamma_accumulate) {
    const char *who = "fg_rms_norm_bwd";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape R=%d C=%d", who, R, C);
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(lds >= C && lddy >= C && (!d_ds || ldds >= C) && (!d_dx || lddx >= C), FG_ERR_SHAPE,
               "%s: lds=%d, lddy=%d, ldds=%d or lddx=%d < C=%d", who, lds, lddy, ldds, lddx, C);
    FG_REQUIRE(d_s && d_dy && d_rstd, FG_ERR_INVALID_ARGUMENT, "%s: s, dy and rstd are required",
               who);
    FG_REQUIRE(!d_ds || d_dx, FG_ERR_INVALID_ARGUMENT, "%s: ds is added to dx, which is NULL", who);
    FG_REQUIRE((d_dx != d_s || lddx == lds) && (d_dx != d_dy || lddx == lddy) &&
                   (!d_ds || d_dx != d_ds || lddx == ldds),
               FG_ERR_INVALID_ARGUMENT,
               "%s: dx is s, dy or ds, but of another leading dimension", who);
    FG_REQUIRE(fg::rows::grid_holds(R, kLongL), FG_ERR_OUT_OF_BOUNDS, "%s: %d rows of %d columns",
               who, R, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_dx, {d_gamma, d_rstd}) &&
                   apart(d_dgamma, {d_s, d_dy, d_gamma, d_ds, d_rstd, d_dx}),
               FG_ERR_INVALID_ARGUMENT,
               "%s: an output is another output or an input (but dx, which may be s, dy or ds)",
               who);
    FG_HIP(hipSetDevice(ctx->device));
    const Split s = split_of(ctx->cu_count, dtype, R, C);
    float *partial = nullptr;
    if (d_dgamma) {
        partial = (float *)fg::workspace(ctx, fg::rms_norm_bwd_ws_bytes(ctx->cu_count, dtype, R, C));
        if (!partial) return FG_ERR_OUT_OF_MEMORY;
    }
    if (R > 0 && (d_dx || d_dgamma)) {
        const Bwd<void> a{d_s, d_dy, d_gamma, d_ds, d_rstd, d_dx, partial,
                          lds, lddy, ldds, lddx, R, C, 0};
        const int rc = dtype == FG_DTYPE_F32    ? launch_bwd<fg::kF32>(ctx, s, a)
                       : dtype == FG_DTYPE_BF16 ? launch_bwd<fg::kBF16>(ctx, s, a)
                                                : launch_bwd<fg::kF16>(ctx, s, a);
        if (rc) return rc;
    }
    if (partial) {
        rms_bwd_final<<<(C - 1) / 32 + 1, 1024, 0, ctx->stream>>>(partial, d_dgamma, dtype,
                                                                 s.splits, C, dgamma_accumulate);
        FG_LAUNCH_CHECK("rms_bwd_final");
    }
    return FG_OK;
}
