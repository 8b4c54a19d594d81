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

#include "fg_half.h"
#include "fg_internal.h"

namespace {

constexpr int kNT = 256;
constexpr int kCols = 256;  // columns per workgroup of the weights' gradients

__device__ __forceinline__ float block_sum(float s, float *sm) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < kNT / 64; ++k) t += sm[k];
    __syncthreads();
    return t;
}

__global__ __launch_bounds__(kNT) void ln_fwd_row(int dt, const void *x, int ldx,
                                                  const void *gamma, const void *beta, float eps,
                                                  int C, void *y, int ldy, float *mean,
                                                  float *rstd) {
    __shared__ float sm[kNT / 64];
    const uint64_t r = blockIdx.x, xr = r * ldx, yr = r * ldy;
    float s = 0.0f;
    for (int c = threadIdx.x; c < C; c += kNT) s += fg::load_as_f(x, dt, xr + c);
    const float mu = block_sum(s, sm) / (float)C;
    float q = 0.0f;
    for (int c = threadIdx.x; c < C; c += kNT) {
        const float d = fg::load_as_f(x, dt, xr + c) - mu;
        q += d * d;
    }
    const float rs = 1.0f / sqrtf(block_sum(q, sm) / (float)C + eps);
    for (int c = threadIdx.x; c < C; c += kNT) {
        float v = (fg::load_as_f(x, dt, xr + c) - mu) * rs;
        if (gamma) v *= fg::load_as_f(gamma, dt, c);
        if (beta) v += fg::load_as_f(beta, dt, c);
        fg::store_from_f(y, dt, yr + c, v);
    }
    if (threadIdx.x == 0) {
        if (mean) mean[r] = mu;
        if (rstd) rstd[r] = rs;
    }
}

__global__ __launch_bounds__(kNT) void ln_bwd_row(int dt, const void *x, int ldx, const void *dy,
                                                  int lddy, const void *gamma, const float *mean,
                                                  const float *rstd, int C, void *dx, int lddx,
                                                  int accumulate) {
    __shared__ float sm[kNT / 64];
    const uint64_t r = blockIdx.x, xr = r * ldx, yr = r * lddy, dr = r * lddx;
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < C; c += kNT) {
        float g = fg::load_as_f(dy, dt, yr + c);
        if (gamma) g *= fg::load_as_f(gamma, dt, c);
        s1 += g;
        s2 += g * ((fg::load_as_f(x, dt, xr + c) - mu) * rs);
    }
    const float m1 = block_sum(s1, sm) / (float)C, m2 = block_sum(s2, sm) / (float)C;
    for (int c = threadIdx.x; c < C; c += kNT) {
        float g = fg::load_as_f(dy, dt, yr + c);
        if (gamma) g *= fg::load_as_f(gamma, dt, c);
        const float xh = (fg::load_as_f(x, dt, xr + c) - mu) * rs;
        const float d = rs * (g - m1 - xh * m2);
        fg::store_from_f(dx, dt, dr + c, accumulate ? fg::load_as_f(dx, dt, dr + c) + d : d);
    }
}

// Row splits of the weights' gradients: partial[split][0][c] sums dy * xh over
// the split's rows, partial[split][1][c] sums dy.
struct Split {
    int strips, splits, rows;
};
Split split_of(int cus, int R, int C) {
    Split s;
    s.strips = (C + kCols - 1) / kCols;
    const int want = std::max(1, std::min((4 * cus + s.strips - 1) / s.strips, (R + 15) / 16));
    s.rows = R > 0 ? (R + want - 1) / want : 1;
    s.splits = R > 0 ? (R + s.rows - 1) / s.rows : 0;
    return s;
}

__global__ __launch_bounds__(kCols) void ln_bwd_cols(int dt, const void *x, int ldx, const void *dy,
                                                     int lddy, const float *mean,
                                                     const float *rstd, int R, int C, int rows,
                                                     float *partial) {
    const int c = blockIdx.x * kCols + threadIdx.x;
    if (c >= C) return;
    const int r0 = blockIdx.y * rows, r1 = min(R, r0 + rows);
    float g = 0.0f, b = 0.0f;
    for (int r = r0; r < r1; ++r) {
        const float d = fg::load_as_f(dy, dt, (uint64_t)r * lddy + c);
        g += d * ((fg::load_as_f(x, dt, (uint64_t)r * ldx + c) - mean[r]) * rstd[r]);
        b += d;
    }
    partial[(2 * (uint64_t)blockIdx.y) * C + c] = g;
    partial[(2 * (uint64_t)blockIdx.y + 1) * C + c] = b;
}

__global__ __launch_bounds__(kCols) void ln_bwd_final(int dt, const float *partial, int splits,
                                                      int C, void *dgamma, int acc_g, void *dbeta,
                                                      int acc_b) {
    const int c = blockIdx.x * kCols + threadIdx.x;
    if (c >= C) return;
    float g = 0.0f, b = 0.0f;
    for (int k = 0; k < splits; ++k) {
        g += partial[(2 * (uint64_t)k) * C + c];
        b += partial[(2 * (uint64_t)k + 1) * C + c];
    }
    if (dgamma) fg::store_from_f(dgamma, dt, c, acc_g ? fg::load_as_f(dgamma, dt, c) + g : g);
    if (dbeta) fg::store_from_f(dbeta, dt, c, acc_b ? fg::load_as_f(dbeta, dt, c) + b : b);
}

}  // namespace

namespace fg {
uint64_t layer_norm_bwd_ws_bytes(int cus, int R, int C) {
    const Split s = split_of(cus > 0 ? cus : 256, R, C);
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
    ln_fwd_row<<<R, kNT, 0, ctx->stream>>>(dtype, d_x, ldx, d_gamma, d_beta, eps, C, d_y, ldy,
                                           d_mean, d_rstd);
    FG_LAUNCH_CHECK("ln_fwd_row");
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
    // The weights' gradients first: dx may be written over x or dy.
    if (d_dgamma || d_dbeta) {
        const Split s = split_of(ctx->cu_count, R, C);
        float *partial =
            (float *)fg::workspace(ctx, fg::layer_norm_bwd_ws_bytes(ctx->cu_count, R, C));
        if (!partial) return FG_ERR_OUT_OF_MEMORY;
        if (R > 0) {
            ln_bwd_cols<<<dim3(s.strips, s.splits), kCols, 0, ctx->stream>>>(
                dtype, d_x, ldx, d_dy, lddy, d_mean, d_rstd, R, C, s.rows, partial);
            FG_LAUNCH_CHECK("ln_bwd_cols");
        }
        ln_bwd_final<<<s.strips, kCols, 0, ctx->stream>>>(dtype, partial, s.splits, C, d_dgamma,
                                                          dgamma_accumulate, d_dbeta,
                                                          dbeta_accumulate);
        FG_LAUNCH_CHECK("ln_bwd_final");
    }
    if (d_dx && R > 0) {
        ln_bwd_row<<<R, kNT, 0, ctx->stream>>>(dtype, d_x, ldx, d_dy, lddy, d_gamma, d_mean, d_rstd,
                                               C, d_dx, lddx, accumulate);
        FG_LAUNCH_CHECK("ln_bwd_row");
    }
    return FG_OK;
}
