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
//
// Both directions are bound by HBM: a row is read once and held on the CU between its
// sums and its output, and the weights' gradients ride along as per-workgroup sums.
// bf16 16384 x 8192 forward 97.9 us (5.5 TB/s), fp32 16384 x 4096 backward 144 us
// (5.6 TB/s).  Small batches are bound by what a launch costs (32 rows of 2048: 3.2 us
// of GPU time); backward batches of a few rows a CU also by the partial sums, which a
// second launch adds (2048 x 4096 bf16: 11 us and 3.6).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "fg_half.h"
#include "fg_internal.h"
#include "fg_rows.h"

namespace {

using fg::rows::apart;
using fg::rows::Io;
using fg::rows::u32x4;

// How a row lies on its L lanes (fg_rows.h): lane t holds whole chunks t, t + L, ...
// below nb, and column `single` where it is below C.
template <int DT>
struct Lanes {
    int nb, single;
    __device__ __forceinline__ Lanes(int C, int t) {
        constexpr int E = Io<DT>::E;
        nb = C / E;
        single = t < C - nb * E ? nb * E + t : C;
    }
};

// The sum over a row's L lanes, the same in every lane: 16 lanes of a wave, or its
// L / 64 waves' sums in turn.  Waves wait at one barrier; sm: a float per wave of
// the row, which nothing of the sum before the last uses.
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

// A kernel's arguments are one or two structs: with a dozen arguments the runtime takes
// up to 0.9 us more for a launch (layer norm backward of 64 rows, a call 5.4 us and 4.9).
template <class T>
struct Fwd {
    const T *x, *gamma, *beta;
    T *y;
    float *mean, *rstd, eps;
    int ldx, ldy, R, C;
};
template <class T>
struct Bwd {
    const T *x, *dy, *gamma;
    const float *mean, *rstd;
    T *dx;
    float *partial;
    int ldx, lddy, lddx, R, C, accumulate;
    int rows;           // ln_bwd_cols: of a split; ln_bwd_few: of a workgroup
    int row_blocks;     // ln_bwd_few
    void *dgamma, *dbeta;
    int acc_g, acc_b;
};

// ------------------------------------------------------------------ forward
// A row is held in registers by L lanes, NV chunks a lane, NG rows at once in a
// workgroup; the workgroup walks the rows with gamma and beta held, and the next
// rows' loads go out before this one's sums.  The variance is summed from x - mean
// (a difference of squares would lose a row far from zero), and sums are divided by
// C, so that the mean of a constant row is exact where its sums are (of 16-bit values up
// to 2^13 columns; fp32 values of many digits round).
template <int DT, int NV, int L, int NG>
__global__ __launch_bounds__(L *NG) void ln_fwd(const Fwd<typename Io<DT>::T> a) {
    const auto *x = a.x;
    const auto *gamma = a.gamma, *beta = a.beta;
    auto *y = a.y;
    float *mean = a.mean, *rstd = a.rstd;
    const float eps = a.eps;
    const int ldx = a.ldx, ldy = a.ldy, R = a.R, C = a.C;
    using IO = Io<DT>;
    constexpr int E = IO::E, NS = (L + 63) / 64;
    __shared__ float sm[2][2][NG][NS];
    const int grp = threadIdx.x / L, t = threadIdx.x % L;
    const Lanes<DT> ln(C, t);
    const bool one = ln.single < C;
    const float n = (float)C;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    u32x4 g[NV], b[NV], w[NV];
    float g1 = 1.0f, b1 = 0.0f, w1 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = t + i * L;
        g[i] = gamma && j < ln.nb ? fg::rows::load<DT>(gamma, j) : zero;
        b[i] = beta && j < ln.nb ? fg::rows::load<DT>(beta, j) : zero;
    }
    if (gamma && one) g1 = IO::load1(gamma, ln.single);
    if (beta && one) b1 = IO::load1(beta, ln.single);
    uint32_t r = blockIdx.x * NG + grp;  // (unsigned: past R by less than a step)
    const uint32_t rows = R, step = gridDim.x * NG;
    auto fetch = [&](uint32_t row) {
        const auto *xr = x + (size_t)row * ldx;
        const bool in = row < rows;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = t + i * L;
            w[i] = in && j < ln.nb ? fg::rows::load<DT>(xr, j) : zero;
        }
        w1 = in && one ? IO::load1(xr, ln.single) : 0.0f;
    };
    fetch(r);
    for (uint32_t r0 = blockIdx.x * NG, it = 0; r0 < rows; r0 += step, ++it) {
        u32x4 v[NV];
        const float v1 = w1;
        float s = v1;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = w[i];
#pragma unroll
            for (int e = 0; e < E; ++e) s += IO::get(v[i], e);
        }
        const uint32_t row = r;
        r += step;
        if (r0 + step < rows) fetch(r);
        const float mu = row_sum<L>(s, sm[it & 1][0][grp], t) / n;
        float q = one ? (v1 - mu) * (v1 - mu) : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float p = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = IO::get(v[i], e) - mu;
                p += d * d;
            }
            q += t + i * L < ln.nb ? p : 0.0f;
        }
        const float rs = 1.0f / sqrtf(row_sum<L>(q, sm[it & 1][1][grp], t) / n + eps);
        if (row < rows) {
            auto *yr = y + (size_t)row * ldy;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = t + i * L;
                if (j >= ln.nb) continue;
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    o[e] = (IO::get(v[i], e) - mu) * rs;
                    if (gamma) o[e] *= IO::get(g[i], e);
                    if (beta) o[e] += IO::get(b[i], e);
                }
                fg::rows::store<DT>(yr, j, IO::pack(o));
            }
            if (one) IO::store1(yr, ln.single, (v1 - mu) * rs * g1 + b1);
            if (t == 0) {
                if (mean) mean[row] = mu;
                if (rstd) rstd[row] = rs;
            }
        }
    }
}

// A row per workgroup and nothing else held (gamma and beta come from the caches
// where the output needs them), so that two or more rows share a CU and their loads
// overlap one another's sums: bf16 4096 x 12000 40.1 us in workgroups of 512, 46.0 in
// ones of 1024; 2048 x 16384 24.3 us, 5.5 TB/s.  The longest rows a CU holds two of take 16
// chunks a lane (fp32 1024 x 32768 51.5 us, 66.7 with 8 chunks in registers for two
// workgroups of 1024, which do not suffice), one a CU where there are no more rows than
// CUs (bf16 64 x 65536 10.9 us, 15.3).  Of twice that length (fp32 65536) a CU holds one
// row, whose loads, sums and stores take turns: 8192 rows 4.7 TB/s, of 32768 columns 5.1.
template <int DT, int NV, int L>
__global__ __launch_bounds__(L) __attribute__((amdgpu_waves_per_eu(NV > 4 ? 4 : 8))) void ln_fwd_wide(
    const Fwd<typename Io<DT>::T> a) {
    const auto *x = a.x;
    const auto *__restrict__ gamma = a.gamma, *__restrict__ beta = a.beta;
    auto *y = a.y;
    float *mean = a.mean, *rstd = a.rstd;
    const float eps = a.eps;
    const int ldx = a.ldx, ldy = a.ldy, C = a.C;
    using IO = Io<DT>;
    constexpr int E = IO::E;
    __shared__ float sm[2][L / 64];
    const auto *xr = x + (size_t)blockIdx.x * ldx;
    auto *yr = y + (size_t)blockIdx.x * ldy;
    const int t = threadIdx.x;
    const Lanes<DT> ln(C, t);
    const bool one = ln.single < C;
    const float n = (float)C;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    u32x4 w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = t + i * L < ln.nb ? fg::rows::load<DT>(xr, t + i * L) : zero;
    float v1 = one ? IO::load1(xr, ln.single) : 0.0f;
    float s = v1;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) p += IO::get(w[i], e);
        s += p;
    }
    const float mu = row_sum<L>(s, sm[0], t) / n;
    fg::smany::repack(w);
    float q = one ? (v1 - mu) * (v1 - mu) : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = IO::get(w[i], e) - mu;
            p += d * d;
        }
        q += t + i * L < ln.nb ? p : 0.0f;
    }
    const float rs = 1.0f / sqrtf(row_sum<L>(q, sm[1], t) / n + eps);
    fg::smany::repack(w);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = t + i * L;
        if (j >= ln.nb) continue;
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = (IO::get(w[i], e) - mu) * rs;
        if (gamma) {
            const u32x4 g = fg::rows::load<DT>(gamma, j);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= IO::get(g, e);
        }
        if (beta) {
            const u32x4 b = fg::rows::load<DT>(beta, j);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += IO::get(b, e);
        }
        fg::rows::store<DT>(yr, j, IO::pack(o));
    }
    if (one) {
        v1 = (v1 - mu) * rs;
        if (gamma) v1 *= IO::load1(gamma, ln.single);
        if (beta) v1 += IO::load1(beta, ln.single);
        IO::store1(yr, ln.single, v1);
    }
    if (t == 0) {
        if (mean) mean[blockIdx.x] = mu;
        if (rstd) rstd[blockIdx.x] = rs;
    }
}

// Rows longer than registers hold: three passes over the row, the second and third
// from the caches where they hold it.
constexpr int kLongL = 1024;
template <int DT>
__global__ __launch_bounds__(kLongL) void ln_fwd_long(const Fwd<typename Io<DT>::T> a) {
    const auto *x = a.x;
    const auto *gamma = a.gamma, *beta = a.beta;
    auto *y = a.y;
    float *mean = a.mean, *rstd = a.rstd;
    const float eps = a.eps;
    const int ldx = a.ldx, ldy = a.ldy, C = a.C;
    using IO = Io<DT>;
    constexpr int E = IO::E;
    __shared__ float sm[2][kLongL / 64];
    const auto *xr = x + (size_t)blockIdx.x * ldx;
    auto *yr = y + (size_t)blockIdx.x * ldy;
    const int t = threadIdx.x;
    const Lanes<DT> ln(C, t);
    const bool one = ln.single < C;
    const float n = (float)C;
    float v1 = one ? IO::load1(xr, ln.single) : 0.0f;
    float s = v1;
#pragma unroll 4
    for (int j = t; j < ln.nb; j += kLongL) {
        const u32x4 w = fg::rows::load<DT>(xr, j);
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) p += IO::get(w, e);
        s += p;
    }
    const float mu = row_sum<kLongL>(s, sm[0], t) / n;
    float q = one ? (v1 - mu) * (v1 - mu) : 0.0f;
#pragma unroll 4
    for (int j = t; j < ln.nb; j += kLongL) {
        const u32x4 w = fg::rows::load<DT>(xr, j);
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = IO::get(w, e) - mu;
            p += d * d;
        }
        q += p;
    }
    const float rs = 1.0f / sqrtf(row_sum<kLongL>(q, sm[1], t) / n + eps);
#pragma unroll 2
    for (int j = t; j < ln.nb; j += kLongL) {
        const u32x4 w = fg::rows::load<DT>(xr, j);
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = (IO::get(w, e) - mu) * rs;
        if (gamma) {
            const u32x4 g = fg::rows::load<DT>(gamma, j);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= IO::get(g, e);
        }
        if (beta) {
            const u32x4 b = fg::rows::load<DT>(beta, j);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += IO::get(b, e);
        }
        fg::rows::store<DT>(yr, j, IO::pack(o));
    }
    if (one) {
        v1 = (v1 - mu) * rs;
        if (gamma) v1 *= IO::load1(gamma, ln.single);
        if (beta) v1 += IO::load1(beta, ln.single);
        IO::store1(yr, ln.single, v1);
    }
    if (t == 0) {
        if (mean) mean[blockIdx.x] = mu;
        if (rstd) rstd[blockIdx.x] = rs;
    }
}

// ----------------------------------------------------------------- backward
// With c = x - mean and gd = dy * gamma, a row needs the sums of gd and gd * c:
//   dx = rstd * (gd - sum(gd) / C - c * rstd * (rstd * sum(gd * c) / C))
// The row in registers as above (one sum phase: mean and rstd are given), with the
// weights' gradients of a lane's columns summed in its registers over the
// workgroup's rows, over its NG rows at once in LDS, and written once per workgroup
// as partial[workgroup][2][Cp] (Cp: C rounded up to 4).  A workgroup a CU: with two,
// the sums cost more than the rows gain (bf16 2048 x 4096 15.3 and 19.2 us, 16384 x 1024
// 22.7 and 26.0); 1024 threads instead of 512 take 17.4 and 25.8.
__host__ __device__ constexpr int64_t padded(int64_t C) { return (C + 3) & ~int64_t(3); }
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int DT, int NV, int L, int NG, bool WEIGHTS>
__global__ __launch_bounds__(L *NG) void ln_bwd(const Bwd<typename Io<DT>::T> a) {
    const auto *x = a.x, *dy = a.dy;
    const auto *gamma = a.gamma;
    const float *mean = a.mean, *rstd = a.rstd;
    auto *dx = a.dx;
    const int ldx = a.ldx, lddy = a.lddy, lddx = a.lddx, C = a.C, accumulate = a.accumulate;
    const int R = a.R;
    float *partial = a.partial;
    using IO = Io<DT>;
    constexpr int E = IO::E, NS = (L + 63) / 64;
    __shared__ float sm[2][2][NG][NS];
    extern __shared__ f32x4 cols[];  // [2][Cp]
    const int grp = threadIdx.x / L, t = threadIdx.x % L;
    const Lanes<DT> ln(C, t);
    const bool one = ln.single < C;
    const float n = (float)C;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    u32x4 wx[NV], wd[NV];
    float g[NV][E], ag[NV][E], ab[NV][E];
    float g1 = 1.0f, ag1 = 0.0f, ab1 = 0.0f, wx1 = 0.0f, wd1 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = t + i * L;
        const u32x4 v = gamma && j < ln.nb ? fg::rows::load<DT>(gamma, j) : zero;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            g[i][e] = gamma ? IO::get(v, e) : 1.0f;
            ag[i][e] = ab[i][e] = 0.0f;
        }
    }
    if (gamma && one) g1 = IO::load1(gamma, ln.single);
    uint32_t r = blockIdx.x * NG + grp;  // (unsigned: past R by less than a step)
    const uint32_t rows = R, step = gridDim.x * NG;
    float mu = 0.0f, rs = 0.0f;
    auto fetch = [&](uint32_t row) {
        const bool in = row < rows;
        const auto *xr = x + (size_t)row * ldx, *dr = dy + (size_t)row * lddy;
        mu = in ? mean[row] : 0.0f;
        rs = in ? rstd[row] : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = t + i * L;
            const bool mine = in && j < ln.nb;
            wx[i] = mine ? fg::rows::load<DT>(xr, j) : zero;
            wd[i] = mine ? fg::rows::load<DT>(dr, j) : zero;
        }
        wx1 = in && one ? IO::load1(xr, ln.single) : 0.0f;
        wd1 = in && one ? IO::load1(dr, ln.single) : 0.0f;
    };
    fetch(r);
    for (uint32_t r0 = blockIdx.x * NG, it = 0; r0 < rows; r0 += step, ++it) {
        float c[NV][E], gd[NV][E];
        const float m = mu, k = rs;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = IO::get(wd[i], e);
                c[i][e] = IO::get(wx[i], e) - m;
                gd[i][e] = d * g[i][e];
                s1 += gd[i][e];
                s2 += gd[i][e] * c[i][e];
                if constexpr (WEIGHTS) {
                    ag[i][e] += d * k * c[i][e];
                    ab[i][e] += d;
                }
            }
        const float c1 = wx1 - m, gd1 = wd1 * g1;
        s1 += gd1;
        s2 += gd1 * c1;
        if constexpr (WEIGHTS) {
            ag1 += wd1 * k * c1;
            ab1 += wd1;
        }
        const uint32_t row = r;
        r += step;
        if (r0 + step < rows) fetch(r);
        if (!dx) continue;
        if constexpr (L == 16) {
            s1 = fg::smrow::row16_sum(s1);
            s2 = fg::smrow::row16_sum(s2);
        } else {
            s1 = fg::rows::wave_sum(s1);
            s2 = fg::rows::wave_sum(s2);
        }
        if constexpr (L > 64) {
            float *p = sm[it & 1][0][grp], *q = sm[it & 1][1][grp];
            if ((t & 63) == 0) {
                p[t >> 6] = s1;
                q[t >> 6] = s2;
            }
            __syncthreads();
            s1 = p[0];
            s2 = q[0];
#pragma unroll
            for (int h = 1; h < NS; ++h) {
                s1 += p[h];
                s2 += q[h];
            }
        }
        const float m1 = s1 / n, m2 = k * (k * s2 / n);
        if (row >= rows) continue;  // (the last rows of a group; no barrier follows but the next row's)
        auto *out = dx + (size_t)row * lddx;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = t + i * L;
            if (j >= ln.nb) continue;
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = k * (gd[i][e] - m1 - c[i][e] * m2);
            if (accumulate) {
                const u32x4 was = fg::rows::load<DT>(out, j);
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += IO::get(was, e);
            }
            fg::rows::store<DT>(out, j, IO::pack(o));
        }
        if (one) {
            float o = k * (gd1 - m1 - c1 * m2);
            if (accumulate) o += IO::load1(out, ln.single);
            IO::store1(out, ln.single, o);
        }
    }
    if constexpr (WEIGHTS) {
        const int64_t Cp = padded(C);
        if constexpr (L == 16) {  // the wave's four rows
            auto over4 = [](float v) {
                v += __shfl_xor(v, 16);
                return v + __shfl_xor(v, 32);
            };
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    ag[i][e] = over4(ag[i][e]);
                    ab[i][e] = over4(ab[i][e]);
                }
            ag1 = over4(ag1);
            ab1 = over4(ab1);
        }
        // Then the workgroup's row groups (waves of rows) in turn.
        constexpr int kTurns = L == 16 ? NG / 4 : NG;
        const int turn = L == 16 ? threadIdx.x >> 6 : grp;
        float *lds = reinterpret_cast<float *>(cols);
        float *part = partial + (size_t)blockIdx.x * 2 * Cp;
        for (int h = 0; h < kTurns; ++h) {
            if (turn == h && (L != 16 || (threadIdx.x & 63) < 16)) {
                const bool last = h + 1 == kTurns;
                auto pass = [&](float (&a)[NV][E], float a1, int64_t at) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const int j = t + i * L;
                        if (j >= ln.nb) continue;
#pragma unroll
                        for (int q = 0; q < E / 4; ++q) {
                            const int64_t to = at + (int64_t)j * E + 4 * q;
                            f32x4 v = {a[i][4 * q], a[i][4 * q + 1], a[i][4 * q + 2],
                                       a[i][4 * q + 3]};
                            if (h > 0) v += *reinterpret_cast<f32x4 *>(lds + to);
                            *reinterpret_cast<f32x4 *>((last ? part : lds) + to) = v;
                        }
                    }
                    if (one) {
                        if (h > 0) a1 += lds[at + ln.single];
                        (last ? part : lds)[at + ln.single] = a1;
                    }
                };
                pass(ag, ag1, 0);
                pass(ab, ab1, Cp);
            }
            if (h + 1 < kTurns) __syncthreads();
        }
    }
}

// The same for rows whose weight gradients leave no registers for a second row's loads:
// their sums are in LDS, 16 bytes a lane in each access, x and dy stay packed, gamma
// comes from the caches.  fp32 512 x 16384 38.4 us (sums in registers and one row's
// loads at a time 44.2), a quarter of it the partial sums, as large as two rows a
// workgroup are.
template <int DT, int NV>
__global__ __launch_bounds__(1024) void ln_bwd_wide(const Bwd<typename Io<DT>::T> a) {
    const auto *x = a.x, *dy = a.dy;
    const auto *__restrict__ gamma = a.gamma;
    const float *mean = a.mean, *rstd = a.rstd;
    auto *dx = a.dx;
    const int ldx = a.ldx, lddy = a.lddy, lddx = a.lddx, C = a.C, accumulate = a.accumulate;
    const int R = a.R;
    float *partial = a.partial;
    using IO = Io<DT>;
    constexpr int E = IO::E, L = 1024, Q = E / 4;
    __shared__ float sm[2][2][L / 64];
    __shared__ f32x4 acc[NV][2][Q][L];  // a lane's own
    const int t = threadIdx.x;
    const Lanes<DT> ln(C, t);
    const bool one = ln.single < C;
    const float n = (float)C;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    float ag1 = 0.0f, ab1 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int q = 0; q < Q; ++q) acc[i][0][q][t] = acc[i][1][q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float g1 = gamma && one ? IO::load1(gamma, ln.single) : 1.0f;
    const uint32_t rows = R;
    u32x4 nx[NV], nd[NV];
    float nx1, nd1, nm, nk;
    auto fetch = [&](uint32_t row) {
        const auto *xr = x + (size_t)row * ldx, *dr = dy + (size_t)row * lddy;
        nm = mean[row];
        nk = rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool mine = t + i * L < ln.nb;
            nx[i] = mine ? fg::rows::load<DT>(xr, t + i * L) : zero;
            nd[i] = mine ? fg::rows::load<DT>(dr, t + i * L) : zero;
        }
        nx1 = one ? IO::load1(xr, ln.single) : 0.0f;
        nd1 = one ? IO::load1(dr, ln.single) : 0.0f;
    };
    uint32_t row = blockIdx.x;
    fetch(row);  // (no workgroup without a row)
    for (uint32_t it = 0; row < rows; row += gridDim.x, ++it) {
        u32x4 wx[NV], wd[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            wx[i] = nx[i];
            wd[i] = nd[i];
        }
        const float m = nm, k = nk, c1 = nx1 - m, d1 = nd1, gd1 = d1 * g1;
        if (row + gridDim.x < rows) fetch(row + gridDim.x);
        float s1 = gd1, s2 = gd1 * c1;
        ag1 += d1 * k * c1;
        ab1 += d1;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            u32x4 g = zero;
            if (gamma && t + i * L < ln.nb) g = fg::rows::load<DT>(gamma, t + i * L);
            float p1 = 0.0f, p2 = 0.0f;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                f32x4 ag = acc[i][0][q][t], ab = acc[i][1][q][t];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int e = 4 * q + h;
                    const float d = IO::get(wd[i], e), c = IO::get(wx[i], e) - m;
                    const float gd = gamma ? d * IO::get(g, e) : d;
                    p1 += gd;
                    p2 += gd * c;
                    ag[h] += d * k * c;
                    ab[h] += d;
                }
                acc[i][0][q][t] = ag;
                acc[i][1][q][t] = ab;
            }
            s1 += p1;
            s2 += p2;
        }
        if (!dx) continue;
        fg::smany::repack(wx);
        fg::smany::repack(wd);
        s1 = fg::rows::wave_sum(s1);
        s2 = fg::rows::wave_sum(s2);
        float *p = sm[it & 1][0], *q = sm[it & 1][1];
        if ((t & 63) == 0) {
            p[t >> 6] = s1;
            q[t >> 6] = s2;
        }
        __syncthreads();
        s1 = p[0];
        s2 = q[0];
#pragma unroll
        for (int h = 1; h < L / 64; ++h) {
            s1 += p[h];
            s2 += q[h];
        }
        const float m1 = s1 / n, m2 = k * (k * s2 / n);
        auto *out = dx + (size_t)row * lddx;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = t + i * L;
            if (j >= ln.nb) continue;
            u32x4 g = zero;
            if (gamma) g = fg::rows::load<DT>(gamma, j);
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = IO::get(wd[i], e), c = IO::get(wx[i], e) - m;
                o[e] = k * ((gamma ? d * IO::get(g, e) : d) - m1 - c * m2);
            }
            if (accumulate) {
                const u32x4 was = fg::rows::load<DT>(out, j);
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += IO::get(was, e);
            }
            fg::rows::store<DT>(out, j, IO::pack(o));
        }
        if (one) {
            float o = k * (gd1 - m1 - c1 * m2);
            if (accumulate) o += IO::load1(out, ln.single);
            IO::store1(out, ln.single, o);
        }
    }
    const int64_t Cp = padded(C);
    float *part = partial + (size_t)blockIdx.x * 2 * Cp;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = t + i * L;
        if (j >= ln.nb) continue;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            float *to = part + (size_t)j * E + 4 * q;
            *reinterpret_cast<f32x4 *>(to) = acc[i][0][q][t];
            *reinterpret_cast<f32x4 *>(to + Cp) = acc[i][1][q][t];
        }
    }
    if (one) {
        part[ln.single] = ag1;
        part[Cp + ln.single] = ab1;
    }
}

// Rows longer than that: dx from a row held packed, a workgroup a row, as ln_fwd_wide
// (longer still: the row twice) ...
template <int DT, int NV>
__global__ __launch_bounds__(1024) void ln_bwd_dx(const Bwd<typename Io<DT>::T> a) {
    const auto *x = a.x, *dy = a.dy;
    const auto *__restrict__ gamma = a.gamma;
    const float *mean = a.mean, *rstd = a.rstd;
    auto *dx = a.dx;
    const int ldx = a.ldx, lddy = a.lddy, lddx = a.lddx, C = a.C, accumulate = a.accumulate;
    using IO = Io<DT>;
    constexpr int E = IO::E, L = 1024;
    __shared__ float sm[2][L / 64];
    const size_t row = blockIdx.x;
    const auto *xr = x + row * ldx, *dr = dy + row * lddy;
    auto *out = dx + row * lddx;
    const int t = threadIdx.x;
    const Lanes<DT> ln(C, t);
    const bool one = ln.single < C;
    const float n = (float)C, m = mean[row], k = rstd[row];
    const u32x4 zero = {0u, 0u, 0u, 0u};
    u32x4 wx[NV], wd[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const bool mine = t + i * L < ln.nb;
        wx[i] = mine ? fg::rows::load<DT>(xr, t + i * L) : zero;
        wd[i] = mine ? fg::rows::load<DT>(dr, t + i * L) : zero;
    }
    float c1 = 0.0f, gd1 = 0.0f;
    if (one) {
        c1 = IO::load1(xr, ln.single) - m;
        gd1 = IO::load1(dr, ln.single);
        if (gamma) gd1 *= IO::load1(gamma, ln.single);
    }
    float s1 = gd1, s2 = gd1 * c1;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (t + i * L >= ln.nb) continue;
        u32x4 g = zero;
        if (gamma) g = fg::rows::load<DT>(gamma, t + i * L);
        float p1 = 0.0f, p2 = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = IO::get(wd[i], e), gd = gamma ? d * IO::get(g, e) : d;
            p1 += gd;
            p2 += gd * (IO::get(wx[i], e) - m);
        }
        s1 += p1;
        s2 += p2;
    }
    const float m1 = row_sum<L>(s1, sm[0], t) / n;
    const float m2 = k * (k * row_sum<L>(s2, sm[1], t) / n);
    fg::smany::repack(wx);
    fg::smany::repack(wd);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = t + i * L;
        if (j >= ln.nb) continue;
        u32x4 g = zero;
        if (gamma) g = fg::rows::load<DT>(gamma, j);
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = IO::get(wd[i], e), c = IO::get(wx[i], e) - m;
            o[e] = k * ((gamma ? d * IO::get(g, e) : d) - m1 - c * m2);
        }
        if (accumulate) {
            const u32x4 was = fg::rows::load<DT>(out, j);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += IO::get(was, e);
        }
        fg::rows::store<DT>(out, j, IO::pack(o));
    }
    if (one) {
        float o = k * (gd1 - m1 - c1 * m2);
        if (accumulate) o += IO::load1(out, ln.single);
        IO::store1(out, ln.single, o);
    }
}

// A row by L lanes, twice from memory.
template <int DT, int L>
__device__ __forceinline__ void bwd_long_row(size_t r, const Bwd<typename Io<DT>::T> &a,
                                             float (*sm)[kLongL / 64]) {
    const auto *x = a.x, *dy = a.dy;
    const auto *gamma = a.gamma;
    const float *mean = a.mean, *rstd = a.rstd;
    auto *dx = a.dx;
    const int ldx = a.ldx, lddy = a.lddy, lddx = a.lddx, C = a.C, accumulate = a.accumulate;
    using IO = Io<DT>;
    constexpr int E = IO::E;
    const auto *xr = x + r * ldx, *dr = dy + r * lddy;
    auto *out = dx + r * lddx;
    const int t = threadIdx.x % L;
    const Lanes<DT> ln(C, t);
    const bool one = ln.single < C;
    const float n = (float)C, m = mean[r], k = rstd[r];
    float c1 = 0.0f, gd1 = 0.0f;
    if (one) {
        c1 = IO::load1(xr, ln.single) - m;
        gd1 = IO::load1(dr, ln.single);
        if (gamma) gd1 *= IO::load1(gamma, ln.single);
    }
    float s1 = gd1, s2 = gd1 * c1;
    auto chunk = [&](int j, float (&c)[E], float (&gd)[E]) {
        const u32x4 wx = fg::rows::load<DT>(xr, j), wd = fg::rows::load<DT>(dr, j);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            c[e] = IO::get(wx, e) - m;
            gd[e] = IO::get(wd, e);
        }
        if (gamma) {
            const u32x4 g = fg::rows::load<DT>(gamma, j);
#pragma unroll
            for (int e = 0; e < E; ++e) gd[e] *= IO::get(g, e);
        }
    };
#pragma unroll 4
    for (int j = t; j < ln.nb; j += L) {
        float c[E], gd[E], p1 = 0.0f, p2 = 0.0f;
        chunk(j, c, gd);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            p1 += gd[e];
            p2 += gd[e] * c[e];
        }
        s1 += p1;
        s2 += p2;
    }
    const float m1 = row_sum<L>(s1, sm[0], t) / n;
    const float m2 = k * (k * row_sum<L>(s2, sm[1], t) / n);
#pragma unroll 2
    for (int j = t; j < ln.nb; j += L) {
        float c[E], o[E];
        chunk(j, c, o);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = k * (o[e] - m1 - c[e] * m2);
        if (accumulate) {
            const u32x4 was = fg::rows::load<DT>(out, j);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += IO::get(was, e);
        }
        fg::rows::store<DT>(out, j, IO::pack(o));
    }
    if (one) {
        float o = k * (gd1 - m1 - c1 * m2);
        if (accumulate) o += IO::load1(out, ln.single);
        IO::store1(out, ln.single, o);
    }
}

template <int DT>
__global__ __launch_bounds__(kLongL) void ln_bwd_long(const Bwd<typename Io<DT>::T> a) {
    __shared__ float sm[2][kLongL / 64];
    bwd_long_row<DT, kLongL>(blockIdx.x, a, sm);
}

// Few rows (kFewRows, or kFewShort short ones), where launches count: one for everything,
// workgroups of one row, or of 16 short ones, for dx, and behind them workgroups of 16
// chunks of columns for the weights, whose 64 groups of lanes take every 64th row and are
// added in order.  bf16, in two
// launches as below and in this one: 64 x 4096 9.1 us and 6.2, 256 x 16384 22.5 and
// 12.2; 512 x 512 10.0 and 6.5, 640 x 2048 10.2 and 8.5, but 1024 x 2048 10.5 and 11.4,
// fp32 512 x 4096 12.1 and 14.9.
constexpr int kFewWave = 256;  // whole chunks of a row that a wave takes
constexpr int kFewRows = 256, kFewShort = 640, kFewLanes = 16, kFewGroups = kLongL / kFewLanes;
template <int DT>
__global__ __launch_bounds__(kLongL) void ln_bwd_few(const Bwd<typename Io<DT>::T> a) {
    const auto *x = a.x, *dy = a.dy;
    const float *mean = a.mean, *rstd = a.rstd;
    const int ldx = a.ldx, lddy = a.lddy, R = a.R, C = a.C, row_blocks = a.row_blocks;
    using IO = Io<DT>;
    constexpr int E = IO::E, kCols = kFewLanes * E;
    __shared__ float sm[2][kLongL / 64];
    __shared__ float sh[kFewGroups][kCols];
    if ((int)blockIdx.x < row_blocks) {
        const int r = (int)blockIdx.x * a.rows + (int)(threadIdx.x >> 6);
        if (a.rows == 1) bwd_long_row<DT, kLongL>(blockIdx.x, a, sm);
        else if (r < a.R) bwd_long_row<DT, 64>(r, a, sm);
        return;
    }
    const int lane = threadIdx.x % kFewLanes, group = threadIdx.x / kFewLanes;
    const int strip = (int)blockIdx.x - row_blocks, j = strip * kFewLanes + lane;
    const int nb = C / E;  // (the columns past the last whole chunk, one to a lane after it)
    float ag[E], ab[E];
#pragma unroll
    for (int e = 0; e < E; ++e) ag[e] = ab[e] = 0.0f;
    if (j < nb) {
#pragma unroll 4
        for (int r = group; r < R; r += kFewGroups) {
            const u32x4 wx = fg::rows::load<DT>(x + (size_t)r * ldx, j);
            const u32x4 wd = fg::rows::load<DT>(dy + (size_t)r * lddy, j);
            const float m = mean[r], k = rstd[r];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = IO::get(wd, e);
                ag[e] += d * k * (IO::get(wx, e) - m);
                ab[e] += d;
            }
        }
    } else if (nb * E + (j - nb) < C) {
        const int col = nb * E + (j - nb);
#pragma unroll 4
        for (int r = group; r < R; r += kFewGroups) {
            const float d = IO::load1(dy + (size_t)r * lddy, col);
            ag[0] += d * rstd[r] * (IO::load1(x + (size_t)r * ldx, col) - mean[r]);
            ab[0] += d;
        }
    }
    // The groups' sums in order, a column a thread.
    auto add = [&](const float (&v)[E], void *out, int acc) {
#pragma unroll
        for (int e = 0; e < E; ++e) sh[group][lane * E + e] = v[e];
        __syncthreads();
        const int at = strip * kFewLanes + (int)threadIdx.x / E, e = threadIdx.x % E;
        const int col = at < nb ? at * E + e : e == 0 ? nb * E + (at - nb) : C;
        if ((int)threadIdx.x < kCols && col < C && out) {
            float s = sh[0][threadIdx.x];
            const int used = min(kFewGroups, R);
#pragma unroll 8
            for (int g = 1; g < used; ++g) s += sh[g][threadIdx.x];
            fg::store_from_f(out, DT, col, acc ? fg::load_as_f(out, DT, col) + s : s);
        }
        __syncthreads();
    };
    add(ag, a.dgamma, a.acc_g);
    add(ab, a.dbeta, a.acc_b);
}

// ... and the columns of a strip over a split of the rows, a chunk a lane (the
// columns past the last whole chunk, one to a lane, in the strip after it).  x and dy
// are read twice: bf16 512 x 65536 72 us, 4.6 TB/s of what both read and write.
constexpr int kColsNT = 256;
template <int DT>
__global__ __launch_bounds__(kColsNT) void ln_bwd_cols(const Bwd<typename Io<DT>::T> a) {
    const auto *x = a.x, *dy = a.dy;
    const float *mean = a.mean, *rstd = a.rstd;
    const int ldx = a.ldx, lddy = a.lddy, R = a.R, C = a.C, rows = a.rows;
    float *partial = a.partial;
    using IO = Io<DT>;
    constexpr int E = IO::E;
    const int nb = C / E, j = blockIdx.x * kColsNT + threadIdx.x;
    const int r0 = blockIdx.y * rows, r1 = min(R, r0 + rows);
    const int64_t Cp = padded(C);
    float *p = partial + (size_t)blockIdx.y * 2 * Cp;
    if (j < nb) {
        float ag[E], ab[E];
#pragma unroll
        for (int e = 0; e < E; ++e) ag[e] = ab[e] = 0.0f;
#pragma unroll 4
        for (int r = r0; r < r1; ++r) {
            const u32x4 wx = fg::rows::load<DT>(x + (size_t)r * ldx, j);
            const u32x4 wd = fg::rows::load<DT>(dy + (size_t)r * lddy, j);
            const float m = mean[r], k = rstd[r];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = IO::get(wd, e);
                ag[e] += d * k * (IO::get(wx, e) - m);
                ab[e] += d;
            }
        }
#pragma unroll
        for (int q = 0; q < E; q += 4) {
            float *to = p + (size_t)j * E + q;
            *reinterpret_cast<f32x4 *>(to) = f32x4{ag[q], ag[q + 1], ag[q + 2], ag[q + 3]};
            *reinterpret_cast<f32x4 *>(to + Cp) = f32x4{ab[q], ab[q + 1], ab[q + 2], ab[q + 3]};
        }
    } else if (nb * E + (j - nb) < C) {
        const int col = nb * E + (j - nb);
        float ag = 0.0f, ab = 0.0f;
#pragma unroll 4
        for (int r = r0; r < r1; ++r) {
            const float d = IO::load1(dy + (size_t)r * lddy, col);
            ag += d * rstd[r] * (IO::load1(x + (size_t)r * ldx, col) - mean[r]);
            ab += d;
        }
        p[col] = ag;
        p[Cp + col] = ab;
    }
}

// Adds the partial sums of each column: GROUPS threads a column, each a run of them in
// order, then the groups' sums in order.
struct Final {
    const float *partial;
    void *dgamma, *dbeta;
    int dt, splits, C, acc_g, acc_b;
};
template <int COLS, int GROUPS>
__global__ __launch_bounds__(COLS *GROUPS) void ln_bwd_final(const Final a) {
    const float *__restrict__ partial = a.partial;
    const int splits = a.splits, C = a.C, dt = a.dt;
    __shared__ float sh[GROUPS][COLS];
    const int c = threadIdx.x % COLS, q = threadIdx.x / COLS;
    const int64_t Cp = padded(C), N = 2 * Cp;
    const int64_t at = (int64_t)blockIdx.x * COLS + c;
    const int64_t i = at < Cp ? at : at - Cp;
    const int per = (splits + GROUPS - 1) / GROUPS;
    int k = q * per;
    const int end = min(splits, k + per);
    const bool mine = at < N && i < C;
    float s = 0.0f;
    if (mine) {
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
    if (q != 0 || !mine) return;
#pragma unroll
    for (int h = 1; h < GROUPS; ++h) s += sh[h][c];
    void *out = at < Cp ? a.dgamma : a.dbeta;
    if (!out) return;
    const int acc = at < Cp ? a.acc_g : a.acc_b;
    fg::store_from_f(out, dt, i, acc ? fg::load_as_f(out, dt, i) + s : s);
}

constexpr int kFewSums = 64;  // (bf16 512 x 65536: 32 sums a column 12 us, by 4 threads 5)

// ------------------------------------------------------------------ choices
// Runs f<NV, L, NG>() for a row of `chunks` whole 16-byte chunks; false: longer
// than any holds.  Forward batches that do not fill the GPU (fewer than two rows a CU)
// take one chunk a lane, as many lanes as the row has (bf16 of 2048, 32 rows 3.3 us
// and 4.0, 511 rows 3.6 and 4.3; 2048 rows of 1024 and more are slower so: 8192 x 4096
// 37.7 us and 23.5).
#define FG_LN_KIND(NV, L, NG)                                         \
    if (chunks <= NV * L) {                                           \
        f(integral_constant<int, NV>{}, integral_constant<int, L>{},  \
          integral_constant<int, NG>{});                              \
        return true;                                                  \
    }
template <class F>
bool fwd_kind(int chunks, bool few, F f) {
    using std::integral_constant;
    if (few) {
        FG_LN_KIND(1, 64, 1)
        FG_LN_KIND(1, 256, 1)
        FG_LN_KIND(1, 1024, 1)
    }
    FG_LN_KIND(1, 16, 16)
    FG_LN_KIND(2, 16, 16)
    FG_LN_KIND(1, 64, 4)
    FG_LN_KIND(2, 64, 4)
    FG_LN_KIND(4, 64, 4)
    FG_LN_KIND(2, 256, 1)
    FG_LN_KIND(4, 256, 1)
    return false;
}
template <int DT, class F>
bool bwd_kind(int chunks, F f) {
    using std::integral_constant;
    FG_LN_KIND(1, 16, 32)
    FG_LN_KIND(2, 16, 32)
    FG_LN_KIND(1, 64, 8)
    FG_LN_KIND(2, 64, 8)
    FG_LN_KIND(2, 128, 4)
    FG_LN_KIND(2, 256, 2)
    FG_LN_KIND(2, 512, 1)
    return false;
}
#undef FG_LN_KIND

template <int DT>
void launch_fwd(fg_ctx *ctx, const void *x, int ldx, const void *gamma, const void *beta,
                float eps, int R, int C, void *y, int ldy, float *mean, float *rstd) {
    using T = typename Io<DT>::T;
    const Fwd<T> a{static_cast<const T *>(x), static_cast<const T *>(gamma),
                   static_cast<const T *>(beta), static_cast<T *>(y), mean, rstd, eps, ldx, ldy, R,
                   C};
    const bool few = R < 2 * ctx->cu_count;
    const bool held = fwd_kind(C / Io<DT>::E, few, [&](auto nv, auto l, auto ng) {
        // Waves a CU walking the rows: all it holds, or 12 where a lane holds more than a
        // chunk (bf16 16384 x 512 7.6 us, with 12 8.8; 8192 x 1024 7.5, with 32 8.3).
        const int per_cu = (nv() == 1 ? 32 : 12) * 64 / (l() * ng());
        const int grid = std::min((R - 1) / ng() + 1, ctx->cu_count * std::max(1, per_cu));
        ln_fwd<DT, nv(), l(), ng()><<<grid, l() * ng(), 0, ctx->stream>>>(a);
    });
    const int chunks = C / Io<DT>::E;
    if (held) return;
#define FG_LN_WIDE(NV, L)                                 \
    if (chunks <= NV * L) {                               \
        ln_fwd_wide<DT, NV, L><<<R, L, 0, ctx->stream>>>(a); \
        return;                                           \
    }
    FG_LN_WIDE(4, 256)
    FG_LN_WIDE(4, 512)
    FG_LN_WIDE(4, 1024)
    if (R <= ctx->cu_count) FG_LN_WIDE(8, 1024)
    FG_LN_WIDE(16, 512)
    FG_LN_WIDE(16, 1024)
#undef FG_LN_WIDE
    ln_fwd_long<DT><<<R, kLongL, 0, ctx->stream>>>(a);
}

// How a backward call's rows are shared out: workgroups of the held rows, or the
// row splits of the long ones.
struct Split {
    int splits = 0, rows = 0, strips = 0;
    bool held = false, wide = false;
};
Split split_of(int cus, int dtype, int R, int C) {
    Split s;
    const int E = dtype == FG_DTYPE_F32 ? 4 : 8, chunks = C / E;
    auto held = [&](auto, auto, auto ng) {
        s.splits = std::min(R > 0 ? (R - 1) / ng() + 1 : 0, cus);
    };
    s.held = E == 4 ? bwd_kind<fg::kF32>(chunks, held) : bwd_kind<fg::kBF16>(chunks, held);
    if (s.held) return s;
    s.wide = chunks <= (E == 4 ? 4 : 2) * 1024;
    if (s.wide) {
        s.splits = std::min(R, cus);
        return s;
    }
    s.strips = (chunks + C % E - 1) / kColsNT + 1;
    const int want = std::max(1, std::min((4 * cus - 1) / s.strips + 1, (R + 15) / 16));
    s.rows = R > 0 ? (R - 1) / want + 1 : 1;
    s.splits = R > 0 ? (R - 1) / s.rows + 1 : 0;
    return s;
}

template <int DT>
int launch_bwd(fg_ctx *ctx, const Split &s, const Bwd<typename Io<DT>::T> &a) {
    hipStream_t st = ctx->stream;
    const int chunks = a.C / Io<DT>::E;
    if (s.held) {
        bwd_kind<DT>(chunks, [&](auto nv, auto l, auto ng) {
            const size_t lds = ng() > 1 ? 2 * (size_t)padded(a.C) * sizeof(float) : 0;
            if (a.partial)
                ln_bwd<DT, nv(), l(), ng(), true><<<s.splits, l() * ng(), lds, st>>>(a);
            else
                ln_bwd<DT, nv(), l(), ng(), false><<<s.splits, l() * ng(), 0, st>>>(a);
        });
        FG_LAUNCH_CHECK("ln_bwd");
        return FG_OK;
    }
    if (s.wide && a.partial) {
        auto kernel = ln_bwd_wide<DT, 2>;
        if constexpr (DT == fg::kF32)
            if (chunks > 2 * 1024) kernel = ln_bwd_wide<DT, 4>;
        kernel<<<s.splits, 1024, 0, st>>>(a);
        FG_LAUNCH_CHECK("ln_bwd_wide");
        return FG_OK;
    }
    // The weights' gradients first: dx may be written over x or dy.
    if (a.partial) {
        ln_bwd_cols<DT><<<dim3(s.strips, s.splits), kColsNT, 0, st>>>(a);
        FG_LAUNCH_CHECK("ln_bwd_cols");
    }
    if (a.dx && chunks <= 8 * 1024) {
        auto kernel = chunks <= 2 * 1024   ? ln_bwd_dx<DT, 2>
                      : chunks <= 4 * 1024 ? ln_bwd_dx<DT, 4>
                                           : ln_bwd_dx<DT, 8>;
        kernel<<<a.R, 1024, 0, st>>>(a);
        FG_LAUNCH_CHECK("ln_bwd_dx");
    } else if (a.dx) {
        ln_bwd_long<DT><<<a.R, kLongL, 0, st>>>(a);
        FG_LAUNCH_CHECK("ln_bwd_long");
    }
    return FG_OK;
}

template <int DT>
int launch_bwd_few(fg_ctx *ctx, Bwd<typename Io<DT>::T> a) {
    constexpr int E = Io<DT>::E;
    const int chunks = a.C / E;
    const int strips = a.dgamma || a.dbeta ? (a.C / E + a.C % E - 1) / kFewLanes + 1 : 0;
    auto launch = [&](int rows, int cols) {
        if (rows + cols == 0) return;
        a.rows = chunks <= kFewWave ? kLongL / 64 : 1;
        a.row_blocks = rows ? (rows - 1) / a.rows + 1 : 0;
        ln_bwd_few<DT><<<a.row_blocks + cols, kLongL, 0, ctx->stream>>>(a);
    };
    // The columns first where dx replaces what they read.
    const bool in_place = a.dx && (a.dx == a.x || a.dx == a.dy);
    if (in_place) launch(0, strips);
    launch(a.dx ? a.R : 0, in_place ? 0 : strips);
    FG_LAUNCH_CHECK("ln_bwd_few");
    return FG_OK;
}

// Whether a backward takes ln_bwd_few.
bool few_rows(int dtype, int R, int C) {
    return R <= kFewRows || (R <= kFewShort && C / (dtype == FG_DTYPE_F32 ? 4 : 8) <= kFewWave);
}

// The rows' launches: all of a few rows' backward, else dx and the partial sums.
template <int DT>
int launch_rows(fg_ctx *ctx, const Split &s, const void *x, int ldx, const void *dy, int lddy,
                const void *gamma, const float *mean, const float *rstd, int R, int C, void *dx,
                int lddx, int accumulate, void *dgamma, int acc_g, void *dbeta, int acc_b,
                float *partial) {
    using T = typename Io<DT>::T;
    Bwd<T> a{};
    a.x = static_cast<const T *>(x);
    a.dy = static_cast<const T *>(dy);
    a.gamma = static_cast<const T *>(gamma);
    a.mean = mean;
    a.rstd = rstd;
    a.dx = static_cast<T *>(dx);
    a.partial = partial;
    a.ldx = ldx;
    a.lddy = lddy;
    a.lddx = lddx;
    a.R = R;
    a.C = C;
    a.accumulate = accumulate;
    a.rows = s.rows;
    a.dgamma = dgamma;
    a.acc_g = acc_g;
    a.dbeta = dbeta;
    a.acc_b = acc_b;
    return few_rows(DT, R, C) ? launch_bwd_few<DT>(ctx, a) : launch_bwd<DT>(ctx, s, a);
}

// Rows that registers do not hold two of take a workgroup each, of 1024 threads at most.
bool rows_fit(int dtype, int R, int C) {
    return C / (dtype == FG_DTYPE_F32 ? 4 : 8) <= 1024 || fg::rows::grid_holds(R, 1024);
}

}  // namespace

namespace fg {
uint64_t layer_norm_bwd_ws_bytes(int cus, int dtype, int R, int C) {
    const Split s = split_of(cus > 0 ? cus : 256, dtype, R, C);
    return (uint64_t)std::max(s.splits, 1) * 2 * (uint64_t)padded(C) * sizeof(float);
}
int layer_norm_bwd_dispatches(int cus, int dtype, int R, int C, bool dx, bool weights) {
    if (few_rows(dtype, R, C)) return 1;  // (a plan's dx is a buffer of its own)
    const Split s = split_of(cus > 0 ? cus : 256, dtype, R, C);
    const bool one = s.held || (s.wide && weights);
    return (one ? (dx || weights) : (int)dx + (int)weights) + (int)weights;
}
}  // namespace fg

FG_API int fg_layer_norm(fg_ctx *ctx, int dtype, const void *d_x, int ldx, const void *d_gamma,
                         const void *d_beta, float eps, int R, int C, void *d_y, int ldy,
                         float *d_mean, float *d_rstd) {
    const char *who = "fg_layer_norm";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape R=%d C=%d", who, R, C);
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(ldx >= C && ldy >= C, FG_ERR_SHAPE, "%s: ldx=%d or ldy=%d < C=%d", who, ldx, ldy,
               C);
    FG_REQUIRE(eps > 0.0f && eps < INFINITY, FG_ERR_INVALID_ARGUMENT,
               "%s: eps must be positive and finite", who);
    FG_REQUIRE(d_x && d_y, FG_ERR_INVALID_ARGUMENT, "%s: x and y are required", who);
    FG_REQUIRE(d_y != d_x || ldy == ldx, FG_ERR_INVALID_ARGUMENT, "%s: y is x, but ldy=%d, ldx=%d",
               who, ldy, ldx);
    FG_REQUIRE(rows_fit(dtype, R, C), FG_ERR_OUT_OF_BOUNDS, "%s: %d rows of %d columns", who, R, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_y, {d_gamma, d_beta, d_mean, d_rstd}) &&
                   apart(d_mean, {d_x, d_gamma, d_beta, d_rstd}) &&
                   apart(d_rstd, {d_x, d_gamma, d_beta}),
               FG_ERR_INVALID_ARGUMENT, "%s: an output is another output or an input but x", who);
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
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(ldx >= C && lddy >= C && (!d_dx || lddx >= C), FG_ERR_SHAPE,
               "%s: ldx=%d, lddy=%d or lddx=%d < C=%d", who, ldx, lddy, lddx, C);
    FG_REQUIRE(d_x && d_dy && d_mean && d_rstd, FG_ERR_INVALID_ARGUMENT,
               "%s: x, dy, mean and rstd are required", who);
    FG_REQUIRE((d_dx != d_x || lddx == ldx) && (d_dx != d_dy || lddx == lddy),
               FG_ERR_INVALID_ARGUMENT, "%s: dx is x or dy, but of another leading dimension", who);
    FG_REQUIRE(!d_dgamma || d_dgamma != d_dbeta, FG_ERR_INVALID_ARGUMENT,
               "%s: dgamma is dbeta", who);
    FG_REQUIRE(!accumulate || (d_dx != d_x && d_dx != d_dy), FG_ERR_INVALID_ARGUMENT,
               "%s: dx is x or dy and adds to itself", who);
    FG_REQUIRE(rows_fit(dtype, R, C), FG_ERR_OUT_OF_BOUNDS, "%s: %d rows of %d columns", who, R, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_dx, {d_gamma, d_mean, d_rstd}) &&
                   apart(d_dgamma, {d_x, d_dy, d_gamma, d_mean, d_rstd, d_dx}) &&
                   apart(d_dbeta, {d_x, d_dy, d_gamma, d_mean, d_rstd, d_dx}),
               FG_ERR_INVALID_ARGUMENT,
               "%s: an output is another output or an input (but dx, which may be x or dy)", who);
    FG_HIP(hipSetDevice(ctx->device));
    const Split s = split_of(ctx->cu_count, dtype, R, C);
    const bool few = R > 0 && few_rows(dtype, R, C);
    float *partial = nullptr;
    if ((d_dgamma || d_dbeta) && !few) {
        partial =
            (float *)fg::workspace(ctx, fg::layer_norm_bwd_ws_bytes(ctx->cu_count, dtype, R, C));
        if (!partial) return FG_ERR_OUT_OF_MEMORY;
    }
    if (R > 0 && (d_dx || d_dgamma || d_dbeta)) {
        auto launch = dtype == FG_DTYPE_F32    ? launch_rows<fg::kF32>
                      : dtype == FG_DTYPE_BF16 ? launch_rows<fg::kBF16>
                                               : launch_rows<fg::kF16>;
        if (int rc = launch(ctx, s, d_x, ldx, d_dy, lddy, d_gamma, d_mean, d_rstd, R, C, d_dx, lddx,
                            accumulate, d_dgamma, dgamma_accumulate, d_dbeta, dbeta_accumulate,
                            partial))
            return rc;
    }
    if (partial) {
        // 32 threads a column (half of them: 0.2 to 0.5 us longer), or 4 for few sums.
        const Final f{partial, d_dgamma, d_dbeta, dtype, s.splits, C, dgamma_accumulate,
                      dbeta_accumulate};
        auto final = [&](auto cols, auto groups) {
            ln_bwd_final<cols(), groups()>
                <<<(unsigned)((2 * padded(C) - 1) / cols() + 1), cols() * groups(), 0,
                   ctx->stream>>>(f);
        };
        using std::integral_constant;
        if (s.splits > kFewSums) final(integral_constant<int, 32>{}, integral_constant<int, 32>{});
        else final(integral_constant<int, 64>{}, integral_constant<int, 4>{});
        FG_LAUNCH_CHECK("ln_bwd_final");
    }
    return FG_OK;
}
