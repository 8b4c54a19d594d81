// k_ckpt8.hip -- activations kept in 8 bits between forward and backward, and
// the backward passes that read them, for gfx950.  The reference keeps every
// saved value in its own type (forward_saved, crates/fused_gpu/src/dispatch/
// mod.rs:509-575).
//
// Format (the OCP MX layout with 8-bit integer elements): 32 consecutive
// columns of a row share one exponent byte b, the last block of a row may be
// short.  With b = max(1, exponent field of the block's largest |x| as fp32):
//   q = clamp(rint(x * 2^(133 - b)), -127, 127)    restored: q * 2^(b - 133)
// so |x| < 2^(b - 126) uses all seven bits, and the error is at most half a
// step, 2^(b - 134) (a whole step where q is clamped, |x| > 127.5 steps).
// Scaling by a power of two is exact, so the only rounding is rint, and a
// restored value has at most 7 significant bits and no bit below what its type
// can hold: it is exact in fp32, fp16 and bf16.  A block that holds an infinity
// or NaN gets b = 255 and is restored as NaN.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fg_act.h"
#include "fg_half.h"
#include "fg_internal.h"

namespace {

constexpr int kNT = 256;
constexpr int kBlock = 32;  // columns per exponent byte

__device__ __forceinline__ float restore(int q, int b) {
    return b == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf((float)q, b - 133);
}

// 32 lanes per block of columns; blockIdx.x walks (row, block) pairs.
__global__ __launch_bounds__(kNT) void ckpt8_save_k(int dt, const void *x, int ldx, uint64_t pairs,
                                                    int nb, int C, int8_t *q, int ldq, uint8_t *e,
                                                    int lde) {
    const int lane = threadIdx.x & 31;
    for (uint64_t p = (uint64_t)blockIdx.x * (kNT / 32) + (threadIdx.x >> 5); p < pairs;
         p += (uint64_t)gridDim.x * (kNT / 32)) {
        const uint64_t r = p / nb;
        const int blk = (int)(p % nb), c = blk * kBlock + lane;
        const float v = c < C ? fg::load_as_f(x, dt, r * ldx + c) : 0.0f;
        uint32_t m = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
        const int b = max(1, (int)(m >> 23));
        const float s = __builtin_rintf(__builtin_amdgcn_ldexpf(v, 133 - b));
        if (c < C)
            q[r * ldq + c] = b == 255 ? (int8_t)0 : (int8_t)fminf(fmaxf(s, -127.0f), 127.0f);
        if (lane == 0) e[r * lde + blk] = (uint8_t)b;
    }
}

// What: 0 restores z and / or h = act(z), 1 writes dz = dh * act'(z) to z.
template <int WHAT>
__global__ __launch_bounds__(kNT) void ckpt8_load_k(int dt, int act, const int8_t *q, int ldq,
                                                    const uint8_t *e, int lde, uint64_t n, int C,
                                                    void *z, int ldz, void *h, int ldh) {
    for (uint64_t i = (uint64_t)blockIdx.x * kNT + threadIdx.x; i < n;
         i += (uint64_t)gridDim.x * kNT) {
        const uint64_t r = i / C;
        const int c = (int)(i % C);
        const float v = restore(q[r * ldq + c], e[r * lde + c / kBlock]);
        if constexpr (WHAT == 0) {
            if (z) fg::store_from_f(z, dt, r * ldz + c, v);
            if (h) fg::store_from_f(h, dt, r * ldh + c, fg::act_fwd(act, v));
        } else {
            const float d = fg::load_as_f(h, dt, r * ldh + c);
            fg::store_from_f(z, dt, r * ldz + c, d * fg::act_grad(act, v));
        }
    }
}

unsigned grid_of(uint64_t work) {
    return (unsigned)std::min<uint64_t>((work + kNT - 1) / kNT, 1u << 20);
}

int check_q(const char *who, int dtype, int R, int C, const void *q, int ldq, const void *e,
            int lde) {
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape %d x %d", who, R, C);
    FG_REQUIRE(ldq >= C, FG_ERR_SHAPE, "%s: ldq=%d < %d columns", who, ldq, C);
    FG_REQUIRE(lde >= (C - 1) / kBlock + 1, FG_ERR_SHAPE,
               "%s: lde=%d < %d exponents (one per 32 columns)", who, lde, (C - 1) / kBlock + 1);
    FG_REQUIRE(q && e, FG_ERR_INVALID_ARGUMENT, "%s: q and e are required", who);
    return FG_OK;
}

}  // namespace

FG_API int fg_ckpt8_save(fg_ctx *ctx, int dtype, const void *d_x, int ldx, int R, int C,
                         int8_t *d_q, int ldq, uint8_t *d_e, int lde) {
    const char *who = "fg_ckpt8_save";
    if (int rc = check_q(who, dtype, R, C, d_q, ldq, d_e, lde)) return rc;
    FG_REQUIRE(ldx >= C, FG_ERR_SHAPE, "%s: ldx=%d < C=%d", who, ldx, C);
    FG_REQUIRE(d_x, FG_ERR_INVALID_ARGUMENT, "%s: x is required", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const int nb = (C - 1) / kBlock + 1;
    const uint64_t pairs = (uint64_t)R * nb;
    ckpt8_save_k<<<grid_of(pairs * 32), kNT, 0, ctx->stream>>>(dtype, d_x, ldx, pairs, nb, C, d_q,
                                                               ldq, d_e, lde);
    FG_LAUNCH_CHECK("ckpt8_save");
    return FG_OK;
}

FG_API int fg_ckpt8_load(fg_ctx *ctx, int dtype, int act, const int8_t *d_q, int ldq,
                         const uint8_t *d_e, int lde, int R, int C, void *d_z, int ldz, void *d_h,
                         int ldh) {
    const char *who = "fg_ckpt8_load";
    if (int rc = check_q(who, dtype, R, C, d_q, ldq, d_e, lde)) return rc;
    FG_REQUIRE(act >= FG_ACT_NONE && act <= FG_ACT_GELU, FG_ERR_INVALID_ARGUMENT,
               "%s: bad act %d", who, act);
    FG_REQUIRE(d_z || d_h, FG_ERR_INVALID_ARGUMENT, "%s: z or h is required", who);
    FG_REQUIRE((!d_z || ldz >= C) && (!d_h || ldh >= C), FG_ERR_SHAPE,
               "%s: ldz=%d or ldh=%d < C=%d", who, ldz, ldh, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const uint64_t n = (uint64_t)R * C;
    ckpt8_load_k<0><<<grid_of(n), kNT, 0, ctx->stream>>>(dtype, act, d_q, ldq, d_e, lde, n, C, d_z,
                                                         ldz, d_h, ldh);
    FG_LAUNCH_CHECK("ckpt8_load");
    return FG_OK;
}

FG_API int fg_act_bwd_ckpt8(fg_ctx *ctx, int dtype, int act, const void *d_dH, int lddh,
                            const int8_t *d_q, int ldq, const uint8_t *d_e, int lde, int R, int C,
                            void *d_dZ, int lddz) {
    const char *who = "fg_act_bwd_ckpt8";
    if (int rc = check_q(who, dtype, R, C, d_q, ldq, d_e, lde)) return rc;
    FG_REQUIRE(act >= FG_ACT_NONE && act <= FG_ACT_GELU, FG_ERR_INVALID_ARGUMENT,
               "%s: bad act %d", who, act);
    FG_REQUIRE(lddh >= C && lddz >= C, FG_ERR_SHAPE, "%s: lddh=%d or lddz=%d < C=%d", who, lddh,
               lddz, C);
    FG_REQUIRE(d_dH && d_dZ, FG_ERR_INVALID_ARGUMENT, "%s: dH and dZ are required", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const uint64_t n = (uint64_t)R * C;
    ckpt8_load_k<1><<<grid_of(n), kNT, 0, ctx->stream>>>(dtype, act, d_q, ldq, d_e, lde, n, C, d_dZ,
                                                         lddz, const_cast<void *>(d_dH), lddh);
    FG_LAUNCH_CHECK("act_bwd_ckpt8");
    return FG_OK;
}

FG_API int fg_matmul_bwd_ckpt8(fg_ctx *ctx, int dtype, int M, int N, int K, int act,
                               const int8_t *d_q, int ldq, const uint8_t *d_e, int lde,
                               const void *d_W, int ldw, const void *d_dZ, int lddz, void *d_Zr,
                               void *d_Xr, void *d_dX, int lddx, void *d_dW, int lddw,
                               void *d_dbias, int accumulate) {
    const char *who = "fg_matmul_bwd_ckpt8";
    if (int rc = check_q(who, dtype, M, K, d_q, ldq, d_e, lde)) return rc;
    FG_REQUIRE(act >= FG_ACT_NONE && act <= FG_ACT_GELU, FG_ERR_INVALID_ARGUMENT,
               "%s: bad act %d", who, act);
    FG_REQUIRE(M > 0 && N > 0, FG_ERR_SHAPE, "%s: bad shape M=%d N=%d", who, M, N);
    FG_REQUIRE(ldw >= N && lddz >= N && lddx >= K && lddw >= N, FG_ERR_SHAPE,
               "%s: a leading dimension is below its row length", who);
    FG_REQUIRE(d_W && d_dZ && d_dX && d_dW, FG_ERR_INVALID_ARGUMENT, "%s: NULL operand or output",
               who);
    FG_REQUIRE(d_Xr && (act == FG_ACT_NONE || d_Zr), FG_ERR_INVALID_ARGUMENT,
               "%s: Xr, and with an activation Zr, is required", who);
    FG_REQUIRE(d_Xr != d_Zr && d_Xr != d_dX, FG_ERR_INVALID_ARGUMENT,
               "%s: Xr must not be Zr or dX", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    void *zr = act == FG_ACT_NONE ? nullptr : d_Zr;
    if (int rc = fg_ckpt8_load(ctx, dtype, act, d_q, ldq, d_e, lde, M, K, zr, K, d_Xr, K))
        return rc;
    if (dtype == FG_DTYPE_F32)
        return fg_matmul_bwd_f32(ctx, M, N, K, (const float *)d_Xr, K, (const float *)d_W, ldw,
                                 (const float *)d_dZ, lddz, act, (const float *)zr, K,
                                 (float *)d_dX, lddx, (float *)d_dW, lddw, (float *)d_dbias,
                                 accumulate);
    return fg_matmul_bwd_x16(ctx, dtype, M, N, K, d_Xr, K, d_W, ldw, d_dZ, lddz, act, zr, K, d_dX,
                             lddx, d_dW, lddw, d_dbias, accumulate);
}
