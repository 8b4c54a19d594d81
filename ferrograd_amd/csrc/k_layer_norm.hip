// k_layer_norm.hip -- layer norm over the last dimension, forward and
// backward with the reduction of the weights' gradients, for gfx950.  The
// reference has no normalisation; its row operator is the softmax node
// (crates/ferrograd-nn/src/op/softmax.rs:14-759).
//
// Forward, for a row x of C elements:
//   mean = sum(x) / C, var = sum((x - mean)^2) / C, rstd = 1 / sqrt(var + eps)
//   y = (x - mean) * rstd * gamma + beta
// Backward, with xh = (x - mean) * rstd and g = dy * gamma:
//   dx = rstd * (g - mean(g) - xh * mean(g * xh))
//   dgamma = sum over rows of dy * xh, dbeta = sum over rows of dy
// All sums are fp32; each output is rounded to its type once.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "fg_half.h"
#include "fg_internal.h"
#include "fg_rows.h"

namespace {

using fg::rows::Io;
using fg::rows::u32x4;
using fg::rows::wave_sum;

// The sum over a row's NW waves of v (its own waves' sums in turn), the same in
// every lane.  One barrier; sm: NW floats that nothing of the last two sums uses.
template <int NW>
__device__ __forceinline__ float row_sum(float v, float *sm, int wave) {
    v = wave_sum(v);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 0) sm[wave] = v;
        __syncthreads();
        v = sm[0];
#pragma unroll
        for (int k = 1; k < NW; ++k) v += sm[k];
    }
    return v;
}

// ------------------------------------------------------------------ forward
// A row is held in registers by NW waves, NV chunks a lane, NG rows at once in a
// workgroup; the workgroup walks the rows with gamma and beta held, and the next
// rows' loads go out before this one's sums.
template <int DT, int NV, int NW, int NG>
__global__ __launch_bounds__(64 * NW * NG) void ln_fwd(
    const typename Io<DT>::T *x, int ldx, const typename Io<DT>::T *gamma,
    const typename Io<DT>::T *beta, float eps, int R, int C, typename Io<DT>::T *y, int ldy,
    float *mean, float *rstd) {
    using IO = Io<DT>;
    constexpr int E = IO::E, NT = 64 * NW;
    __shared__ float sm[2][2][NG][NW];
    const int grp = threadIdx.x / NT, t = threadIdx.x % NT, wave = t >> 6;
    u32x4 g[NV], b[NV], w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (t + i * NT) * E;
        if (gamma) g[i] = fg::rows::load<DT>(gamma, col, C - col);
        if (beta) b[i] = fg::rows::load<DT>(beta, col, C - col);
    }
    const float n = (float)C;  // (sums are divided: a constant row's mean is then exact)
    uint32_t r = blockIdx.x * NG + grp;  // (unsigned: past R by less than a step)
    const uint32_t rows = R, step = gridDim.x * NG;
    auto fetch = [&](uint32_t row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (t + i * NT) * E;
            w[i] = fg::rows::load<DT>(x + (size_t)row * ldx, col, row < rows ? C - col : 0);
        }
    };
    fetch(r);
    for (uint32_t r0 = blockIdx.x * NG, it = 0; r0 < rows; r0 += step, ++it) {
        u32x4 v[NV];
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = w[i];
#pragma unroll
            for (int e = 0; e < E; ++e) s += IO::get(v[i], e);
        }
        const uint32_t row = r;
        r += step;
        if (r0 + step < rows) fetch(r);
        const float mu = row_sum<NW>(s, sm[it & 1][0][grp], wave) / n;
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int left = C - (t + i * NT) * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = IO::get(v[i], e) - mu;
                q += e < left ? d * d : 0.0f;
            }
        }
        const float rs = 1.0f / sqrtf(row_sum<NW>(q, sm[it & 1][1][grp], wave) / n + eps);
        if (row < rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = (t + i * NT) * E;
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    o[e] = (IO::get(v[i], e) - mu) * rs;
                    if (gamma) o[e] *= IO::get(g[i], e);
                    if (beta) o[e] += IO::get(b[i], e);
                }
                fg::rows::store<DT>(y + (size_t)row * ldy, col, C - col, IO::pack(o));
            }
            if (t == 0) {
                if (mean) mean[row] = mu;
                if (rstd) rstd[row] = rs;
            }
        }
    }
}

// Rows longer than registers hold: three passes over the row, the second and third
// from the caches where they hold it.
constexpr int kLongNW = 16;
template <int DT>
__global__ __launch_bounds__(64 * kLongNW) void ln_fwd_long(
    const typename Io<DT>::T *x, int ldx, const typename Io<DT>::T *gamma,
    const typename Io<DT>::T *beta, float eps, int C, typename Io<DT>::T *y, int ldy, float *mean,
    float *rstd) {
    using IO = Io<DT>;
    constexpr int E = IO::E, NT = 64 * kLongNW;
    __shared__ float sm[2][kLongNW];
    const auto *xr = x + (size_t)blockIdx.x * ldx;
    auto *yr = y + (size_t)blockIdx.x * ldy;
    const int wave = threadIdx.x >> 6;
    const float n = (float)C;  // (sums are divided: a constant row's mean is then exact)
    float s = 0.0f;
    for (int64_t col = threadIdx.x * E; col < C; col += NT * E) {
        const u32x4 w = fg::rows::load<DT>(xr, (int)col, C - (int)col);
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) p += IO::get(w, e);
        s += p;
    }
    const float mu = row_sum<kLongNW>(s, sm[0], wave) / n;
    float q = 0.0f;
    for (int64_t col = threadIdx.x * E; col < C; col += NT * E) {
        const int left = C - (int)col;
        const u32x4 w = fg::rows::load<DT>(xr, (int)col, left);
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = IO::get(w, e) - mu;
            p += e < left ? d * d : 0.0f;
        }
        q += p;
    }
    const float rs = 1.0f / sqrtf(row_sum<kLongNW>(q, sm[1], wave) / n + eps);
    for (int64_t c64 = threadIdx.x * E; c64 < C; c64 += NT * E) {
        const int col = (int)c64, left = C - col;
        const u32x4 w = fg::rows::load<DT>(xr, col, left);
        u32x4 g, b;
        if (gamma) g = fg::rows::load<DT>(gamma, col, left);
        if (beta) b = fg::rows::load<DT>(beta, col, left);
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            o[e] = (IO::get(w, e) - mu) * rs;
            if (gamma) o[e] *= IO::get(g, e);
            if (beta) o[e] += IO::get(b, e);
        }
        fg::rows::store<DT>(yr, col, left, IO::pack(o));
    }
    if (threadIdx.x == 0) {
        if (mean) mean[blockIdx.x] = mu;
        if (rstd) rstd[blockIdx.x] = rs;
    }
}

// ----------------------------------------------------------------- backward
// The row in registers as above (one sum phase a row: mean and rstd are given),
// with the weights' gradients of a lane's columns summed in its registers over the
// workgroup's rows, over its NG rows at once in LDS, and written once per workgroup
// as partial[workgroup][2][C].
template <int DT, int NV, int NW, int NG, bool WEIGHTS>
__global__ __launch_bounds__(64 * NW * NG) void ln_bwd(
    const typename Io<DT>::T *x, int ldx, const typename Io<DT>::T *dy, int lddy,
    const typename Io<DT>::T *gamma, const float *mean, const float *rstd, int R, int C,
    typename Io<DT>::T *dx, int lddx, int accumulate, float *partial) {
    using IO = Io<DT>;
    constexpr int E = IO::E, NT = 64 * NW;
    __shared__ float sm[2][2][NG][NW];
    extern __shared__ float cols[];  // [2][C]
    const int grp = threadIdx.x / NT, t = threadIdx.x % NT, wave = t >> 6;
    u32x4 g[NV], wx[NV], wd[NV];
    float ag[WEIGHTS ? NV : 1][E], ab[WEIGHTS ? NV : 1][E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int col = (t + i * NT) * E;
        if (gamma) g[i] = fg::rows::load<DT>(gamma, col, C - col);
        if constexpr (WEIGHTS) {
#pragma unroll
            for (int e = 0; e < E; ++e) ag[i][e] = ab[i][e] = 0.0f;
        }
    }
    const float n = (float)C;  // (sums are divided: a constant row's mean is then exact)
    uint32_t r = blockIdx.x * NG + grp;  // (unsigned: past R by less than a step)
    const uint32_t rows = R, step = gridDim.x * NG;
    float mu = 0.0f, rs = 0.0f;
    auto fetch = [&](uint32_t row) {
        const bool in = row < rows;
        mu = in ? mean[row] : 0.0f;
        rs = in ? rstd[row] : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (t + i * NT) * E;
            wx[i] = fg::rows::load<DT>(x + (size_t)row * ldx, col, in ? C - col : 0);
            wd[i] = fg::rows::load<DT>(dy + (size_t)row * lddy, col, in ? C - col : 0);
        }
    };
    fetch(r);
    for (uint32_t r0 = blockIdx.x * NG, it = 0; r0 < rows; r0 += step, ++it) {
        u32x4 vx[NV], vd[NV];
        const float m = mu, k = rs;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            vx[i] = wx[i];
            vd[i] = wd[i];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = IO::get(vd[i], e), xh = (IO::get(vx[i], e) - m) * k;
                const float gd = gamma ? d * IO::get(g[i], e) : d;
                s1 += gd;
                s2 += gd * xh;
                if constexpr (WEIGHTS) {
                    ag[i][e] += d * xh;
                    ab[i][e] += d;
                }
            }
        }
        const uint32_t row = r;
        r += step;
        if (r0 + step < rows) fetch(r);
        if (dx) {
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
            if constexpr (NW > 1) {
                float(*p)[NW] = sm[it & 1][0] + grp, (*q)[NW] = sm[it & 1][1] + grp;
                if ((threadIdx.x & 63) == 0) {
                    (*p)[wave] = s1;
                    (*q)[wave] = s2;
                }
                __syncthreads();
                s1 = (*p)[0];
                s2 = (*q)[0];
#pragma unroll
                for (int h = 1; h < NW; ++h) {
                    s1 += (*p)[h];
                    s2 += (*q)[h];
                }
            }
            const float m1 = s1 / n, m2 = s2 / n;
            if (row < rows) {
                auto *out = dx + (size_t)row * lddx;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int col = (t + i * NT) * E;
                    float o[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float d = IO::get(vd[i], e), xh = (IO::get(vx[i], e) - m) * k;
                        o[e] = k * ((gamma ? d * IO::get(g[i], e) : d) - m1 - xh * m2);
                    }
                    if (accumulate) {
                        const u32x4 was = fg::rows::load<DT>(out, col, C - col);
#pragma unroll
                        for (int e = 0; e < E; ++e) o[e] += IO::get(was, e);
                    }
                    fg::rows::store<DT>(out, col, C - col, IO::pack(o));
                }
            }
        }
    }
    if constexpr (WEIGHTS) {
        for (int h = 0; h < NG; ++h) {  // the row groups in turn
            if (grp == h) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int col = (t + i * NT) * E + e;
                        if (col >= C) continue;
                        float a = ag[i][e], c = ab[i][e];
                        if (h > 0) {
                            a += cols[col];
                            c += cols[C + col];
                        }
                        if (h + 1 < NG) {
                            cols[col] = a;
                            cols[C + col] = c;
                        } else {
                            partial[(size_t)blockIdx.x * 2 * C + col] = a;
                            partial[(size_t)blockIdx.x * 2 * C + C + col] = c;
                        }
                    }
            }
            if (h + 1 < NG) __syncthreads();
        }
    }
}

// Rows longer than that: the row twice for dx ...
template <int DT>
__global__ __launch_bounds__(64 * kLongNW) void ln_bwd_long(
    const typename Io<DT>::T *x, int ldx, const typename Io<DT>::T *dy, int lddy,
    const typename Io<DT>::T *gamma, const float *mean, const float *rstd, int C,
    typename Io<DT>::T *dx, int lddx, int accumulate) {
    using IO = Io<DT>;
    constexpr int E = IO::E, NT = 64 * kLongNW;
    __shared__ float sm[2][kLongNW];
    const size_t r = blockIdx.x;
    const auto *xr = x + r * ldx, *dr = dy + r * lddy;
    auto *out = dx + r * lddx;
    const int wave = threadIdx.x >> 6;
    const float n = (float)C, m = mean[r], k = rstd[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c64 = threadIdx.x * E; c64 < C; c64 += NT * E) {
        const int col = (int)c64, left = C - col;
        const u32x4 wx = fg::rows::load<DT>(xr, col, left), wd = fg::rows::load<DT>(dr, col, left);
        u32x4 g;
        if (gamma) g = fg::rows::load<DT>(gamma, col, left);
        float p1 = 0.0f, p2 = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = IO::get(wd, e), gd = gamma ? d * IO::get(g, e) : d;
            p1 += gd;
            p2 += gd * ((IO::get(wx, e) - m) * k);
        }
        s1 += p1;
        s2 += p2;
    }
    const float m1 = row_sum<kLongNW>(s1, sm[0], wave) / n;
    const float m2 = row_sum<kLongNW>(s2, sm[1], wave) / n;
    for (int64_t c64 = threadIdx.x * E; c64 < C; c64 += NT * E) {
        const int col = (int)c64, left = C - col;
        const u32x4 wx = fg::rows::load<DT>(xr, col, left), wd = fg::rows::load<DT>(dr, col, left);
        u32x4 g;
        if (gamma) g = fg::rows::load<DT>(gamma, col, left);
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = IO::get(wd, e), xh = (IO::get(wx, e) - m) * k;
            o[e] = k * ((gamma ? d * IO::get(g, e) : d) - m1 - xh * m2);
        }
        if (accumulate) {
            const u32x4 was = fg::rows::load<DT>(out, col, left);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += IO::get(was, e);
        }
        fg::rows::store<DT>(out, col, left, IO::pack(o));
    }
}

// ... and the columns of a strip over a split of the rows, a chunk a lane.
constexpr int kColsNT = 256;
template <int DT>
__global__ __launch_bounds__(kColsNT) void ln_bwd_cols(const typename Io<DT>::T *x, int ldx,
                                                       const typename Io<DT>::T *dy, int lddy,
                                                       const float *mean, const float *rstd, int R,
                                                       int C, int rows, float *partial) {
    using IO = Io<DT>;
    constexpr int E = IO::E;
    const int64_t c64 = ((int64_t)blockIdx.x * kColsNT + threadIdx.x) * E;
    if (c64 >= C) return;
    const int col = (int)c64, left = C - col;
    const int r0 = blockIdx.y * rows, r1 = min(R, r0 + rows);
    float ag[E], ab[E];
#pragma unroll
    for (int e = 0; e < E; ++e) ag[e] = ab[e] = 0.0f;
#pragma unroll 4
    for (int r = r0; r < r1; ++r) {
        const u32x4 wx = fg::rows::load<DT>(x + (size_t)r * ldx, col, left);
        const u32x4 wd = fg::rows::load<DT>(dy + (size_t)r * lddy, col, left);
        const float m = mean[r], k = rstd[r];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = IO::get(wd, e);
            ag[e] += d * ((IO::get(wx, e) - m) * k);
            ab[e] += d;
        }
    }
    float *p = partial + (size_t)blockIdx.y * 2 * C;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e < left) {
            p[col + e] = ag[e];
            p[(size_t)C + col + e] = ab[e];
        }
}

// Adds the partial sums of each column: 16 threads a column, each a run of them in
// order, then the 16 in order.
constexpr int kFinalCols = 64, kFinalGroups = 16;
__global__ __launch_bounds__(kFinalCols *kFinalGroups) void ln_bwd_final(
    int dt, const float *__restrict__ partial, int splits, int C, void *dgamma, int acc_g,
    void *dbeta, int acc_b) {
    __shared__ float sh[kFinalGroups][kFinalCols];
    const int c = threadIdx.x % kFinalCols, q = threadIdx.x / kFinalCols;
    const int64_t at = (int64_t)blockIdx.x * kFinalCols + c;  // of the 2 C columns
    const int per = (splits + kFinalGroups - 1) / kFinalGroups;
    int k = q * per;
    const int end = min(splits, k + per);
    const int64_t N = 2 * (int64_t)C;
    float s = 0.0f;
    if (at < N) {
        for (; k + 8 <= end; k += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = partial[(k + u) * N + at];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; k < end; ++k) s += partial[k * N + at];
    }
    sh[q][c] = s;
    __syncthreads();
    if (q != 0 || at >= N) return;
#pragma unroll
    for (int n = 1; n < kFinalGroups; ++n) s += sh[n][c];
    void *out = at < C ? dgamma : dbeta;
    if (!out) return;
    const int64_t i = at < C ? at : at - C;
    fg::store_from_f(out, dt, i, (at < C ? acc_g : acc_b) ? fg::load_as_f(out, dt, i) + s : s);
}

// ------------------------------------------------------------------ choices
// Runs f<NV, NW, NG>() for a row of `chunks` 16-byte chunks; false: longer than
// any holds.
template <class F>
bool fwd_kind(int chunks, bool few, F f) {
    using std::integral_constant;
#define FG_LN_KIND(NV, NW, NG)                                              \
    if (chunks <= NV * NW * 64) {                                           \
        f(integral_constant<int, NV>{}, integral_constant<int, NW>{},       \
          integral_constant<int, NG>{});                                    \
        return true;                                                        \
    }
    if (few) {
        FG_LN_KIND(1, 1, 1)
        FG_LN_KIND(1, 4, 1)
        FG_LN_KIND(1, 16, 1)
    }
    FG_LN_KIND(1, 1, 4)
    FG_LN_KIND(2, 1, 4)
    FG_LN_KIND(4, 1, 4)
    FG_LN_KIND(2, 4, 1)
    FG_LN_KIND(4, 4, 1)
    FG_LN_KIND(4, 8, 1)
    FG_LN_KIND(4, 16, 1)
    return false;
}

template <int DT, class F>
bool bwd_kind(int chunks, F f) {
    using std::integral_constant;
    FG_LN_KIND(1, 1, 8)
    FG_LN_KIND(2, 1, 8)
    FG_LN_KIND(2, 2, 4)
    FG_LN_KIND(2, 4, 2)
    FG_LN_KIND(2, 8, 1)
    FG_LN_KIND(2, 16, 1)
    if constexpr (DT == fg::kF32) {
        FG_LN_KIND(4, 16, 1)
    }
#undef FG_LN_KIND
    return false;
}

template <int DT>
void launch_fwd(fg_ctx *ctx, const void *x, int ldx, const void *gamma, const void *beta,
                float eps, int R, int C, void *y, int ldy, float *mean, float *rstd) {
    using T = typename Io<DT>::T;
    const T *xt = static_cast<const T *>(x), *gt = static_cast<const T *>(gamma),
            *bt = static_cast<const T *>(beta);
    T *yt = static_cast<T *>(y);
    const int chunks = (C - 1) / Io<DT>::E + 1;
    const bool few = R < 2 * ctx->cu_count;
    const bool held = fwd_kind(chunks, few, [&](auto nv, auto nw, auto ng) {
        const int per_cu = 32 / (nw() * ng());
        const int grid = std::min((R - 1) / ng() + 1, ctx->cu_count * std::max(1, per_cu));
        ln_fwd<DT, nv(), nw(), ng()><<<grid, 64 * nw() * ng(), 0, ctx->stream>>>(
            xt, ldx, gt, bt, eps, R, C, yt, ldy, mean, rstd);
    });
    if (!held)
        ln_fwd_long<DT><<<R, 64 * kLongNW, 0, ctx->stream>>>(xt, ldx, gt, bt, eps, C, yt, ldy, mean,
                                                             rstd);
}

// How a backward call's rows are shared out: workgroups of the held rows, or the
// row splits of the long ones.
struct Split {
    int splits = 0, rows = 0, strips = 0;
    bool held = false;
};
Split split_of(int cus, int dtype, int R, int C) {
    Split s;
    const int E = dtype == FG_DTYPE_F32 ? 4 : 8, chunks = (C - 1) / E + 1;
    auto held = [&](auto, auto, auto ng) {
        s.splits = std::min(R > 0 ? (R - 1) / ng() + 1 : 0, 2 * cus);
    };
    s.held = E == 4 ? bwd_kind<fg::kF32>(chunks, held) : bwd_kind<fg::kBF16>(chunks, held);
    if (s.held) return s;
    s.strips = (chunks - 1) / kColsNT + 1;
    const int want = std::max(1, std::min((4 * cus - 1) / s.strips + 1, (R + 15) / 16));
    s.rows = R > 0 ? (R - 1) / want + 1 : 1;
    s.splits = R > 0 ? (R - 1) / s.rows + 1 : 0;
    return s;
}

template <int DT>
int launch_bwd(fg_ctx *ctx, const Split &s, const void *x, int ldx, const void *dy, int lddy,
               const void *gamma, const float *mean, const float *rstd, int R, int C, void *dx,
               int lddx, int accumulate, float *partial) {
    using T = typename Io<DT>::T;
    const T *xt = static_cast<const T *>(x), *dt = static_cast<const T *>(dy),
            *gt = static_cast<const T *>(gamma);
    T *ot = static_cast<T *>(dx);
    hipStream_t st = ctx->stream;
    if (s.held) {
        bwd_kind<DT>((C - 1) / Io<DT>::E + 1, [&](auto nv, auto nw, auto ng) {
            const size_t lds = ng() > 1 ? 2 * (size_t)C * sizeof(float) : 0;
            if (partial)
                ln_bwd<DT, nv(), nw(), ng(), true><<<s.splits, 64 * nw() * ng(), lds, st>>>(
                    xt, ldx, dt, lddy, gt, mean, rstd, R, C, ot, lddx, accumulate, partial);
            else
                ln_bwd<DT, nv(), nw(), ng(), false><<<s.splits, 64 * nw() * ng(), 0, st>>>(
                    xt, ldx, dt, lddy, gt, mean, rstd, R, C, ot, lddx, accumulate, partial);
        });
        FG_LAUNCH_CHECK("ln_bwd");
        return FG_OK;
    }
    // The weights' gradients first: dx may be written over x or dy.
    if (partial) {
        ln_bwd_cols<DT><<<dim3(s.strips, s.splits), kColsNT, 0, st>>>(xt, ldx, dt, lddy, mean, rstd,
                                                                     R, C, s.rows, partial);
        FG_LAUNCH_CHECK("ln_bwd_cols");
    }
    if (dx) {
        ln_bwd_long<DT><<<R, 64 * kLongNW, 0, st>>>(xt, ldx, dt, lddy, gt, mean, rstd, C, ot, lddx,
                                                    accumulate);
        FG_LAUNCH_CHECK("ln_bwd_long");
    }
    return FG_OK;
}

}  // namespace

namespace fg {
uint64_t layer_norm_bwd_ws_bytes(int cus, int dtype, int R, int C) {
    const Split s = split_of(cus > 0 ? cus : 256, dtype, R, C);
    return (uint64_t)std::max(s.splits, 1) * 2 * (uint64_t)C * sizeof(float);
}
}  // namespace fg

FG_API int fg_layer_norm(fg_ctx *ctx, int dtype, const void *d_x, int ldx, const void *d_gamma,
                         const void *d_beta, float eps, int R, int C, void *d_y, int ldy,
                         float *d_mean, float *d_rstd) {
    const char *who = "fg_layer_norm";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape R=%d C=%d", who, R, C);
    FG_REQUIRE(ldx >= C && ldy >= C, FG_ERR_SHAPE, "%s: ldx=%d or ldy=%d < C=%d", who, ldx, ldy,
               C);
    FG_REQUIRE(eps > 0.0f && eps < INFINITY, FG_ERR_INVALID_ARGUMENT,
               "%s: eps must be positive and finite", who);
    FG_REQUIRE(d_x && d_y, FG_ERR_INVALID_ARGUMENT, "%s: x and y are required", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    if (dtype == FG_DTYPE_F32)
        launch_fwd<fg::kF32>(ctx, d_x, ldx, d_gamma, d_beta, eps, R, C, d_y, ldy, d_mean, d_rstd);
    else if (dtype == FG_DTYPE_BF16)
        launch_fwd<fg::kBF16>(ctx, d_x, ldx, d_gamma, d_beta, eps, R, C, d_y, ldy, d_mean, d_rstd);
    else
        launch_fwd<fg::kF16>(ctx, d_x, ldx, d_gamma, d_beta, eps, R, C, d_y, ldy, d_mean, d_rstd);
    FG_LAUNCH_CHECK("ln_fwd");
    return FG_OK;
}

FG_API int fg_layer_norm_bwd(fg_ctx *ctx, int dtype, const void *d_x, int ldx, const void *d_dy,
                             int lddy, const void *d_gamma, const float *d_mean,
                             const float *d_rstd, int R, int C, void *d_dx, int lddx,
                             int accumulate, void *d_dgamma, int dgamma_accumulate, void *d_dbeta,
                             int dbeta_accumulate) {
    const char *who = "fg_layer_norm_bwd";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape R=%d C=%d", who, R, C);
    FG_REQUIRE(ldx >= C && lddy >= C && (!d_dx || lddx >= C), FG_ERR_SHAPE,
               "%s: ldx=%d, lddy=%d or lddx=%d < C=%d", who, ldx, lddy, lddx, C);
    FG_REQUIRE(d_x && d_dy && d_mean && d_rstd, FG_ERR_INVALID_ARGUMENT,
               "%s: x, dy, mean and rstd are required", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_HIP(hipSetDevice(ctx->device));
    const Split s = split_of(ctx->cu_count, dtype, R, C);
    float *partial = nullptr;
    if (d_dgamma || d_dbeta) {
        partial =
            (float *)fg::workspace(ctx, fg::layer_norm_bwd_ws_bytes(ctx->cu_count, dtype, R, C));
        if (!partial) return FG_ERR_OUT_OF_MEMORY;
    }
    if (R > 0 && (d_dx || partial)) {
        auto launch = dtype == FG_DTYPE_F32    ? launch_bwd<fg::kF32>
                      : dtype == FG_DTYPE_BF16 ? launch_bwd<fg::kBF16>
                                               : launch_bwd<fg::kF16>;
        if (int rc = launch(ctx, s, d_x, ldx, d_dy, lddy, d_gamma, d_mean, d_rstd, R, C, d_dx, lddx,
                            accumulate, partial))
            return rc;
    }
    if (partial) {
        ln_bwd_final<<<(unsigned)((2 * (int64_t)C - 1) / kFinalCols + 1), kFinalCols * kFinalGroups,
                       0, ctx->stream>>>(dtype, partial, s.splits, C, d_dgamma, dgamma_accumulate,
                                         d_dbeta, dbeta_accumulate);
        FG_LAUNCH_CHECK("ln_bwd_final");
    }
    return FG_OK;
}
