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
//
// All three passes are bound by HBM.  A lane takes a 16-byte chunk of a row (a block
// is four lanes, eight in fp32) and, of the 8-bit form, the chunk's 8 or 4 bytes, so
// that every access of a wave is one stretch of memory: with 16 columns a lane, each
// store of a wave left gaps, and 2048 x 4096 fp32 there and back took 64 us.  Rows may
// start anywhere.  bf16 16384 x 4096: save 37 us, load of z and gelu(z) 48 us
// (6.9 TB/s), act_bwd 60 us (5.6 TB/s); 2048 x 4096 there and back 13.4 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "fg_act.h"
#include "fg_half.h"
#include "fg_internal.h"
#include "fg_rows.h"

namespace {

using fg::rows::apart;
using fg::rows::Chunk;
using fg::rows::Io;
using fg::rows::u32x2;
using fg::rows::u32x4;

constexpr int kNT = 256;
constexpr int kBlock = 32;  // columns per exponent byte
constexpr int kDeep = 4;    // chunks of a lane, loaded together
typedef u32x2 u32x2_byte __attribute__((aligned(1)));
typedef uint32_t u32_byte __attribute__((aligned(1)));

// Where a lane's chunks lie: 2^lshift lanes take kDeep chunks each of a row, and
// blockIdx.y the row's next 2^lshift * kDeep.
struct Tile {
    size_t row;
    int first, step;
    bool in;
    __device__ __forceinline__ Tile(int R, int lshift) {
        const int64_t r = ((int64_t)blockIdx.x << (8 - lshift)) + (threadIdx.x >> lshift);
        in = r < R;
        row = in ? (size_t)r : 0;
        step = 1 << lshift;
        first = (blockIdx.y << lshift) * kDeep + (threadIdx.x & (step - 1));
    }
};

// E signed bytes in one access; the bytes of the row's last, partial chunk in turn.
template <int E>
struct Bytes {
    uint32_t w[E / 4];
    __device__ __forceinline__ void load(const int8_t *row, int j, int nb, int C) {
        const int8_t *p = row + (size_t)j * E;
        if (j < nb) {
            if constexpr (E == 8) {
                const u32x2 v = *reinterpret_cast<const u32x2_byte *>(p);
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
            if constexpr (E == 8) *reinterpret_cast<u32x2_byte *>(p) = u32x2{w[0], w[1]};
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

// A kernel's arguments are one or two structs: with a dozen arguments the runtime takes
// up to 0.9 us more for a launch (layer norm backward of 64 rows, a call 5.4 us and 4.9).
template <class T>
struct Save {
    const T *x;
    int8_t *q;
    uint8_t *e;
    int ldx, ldq, lde, R, C, lshift;
};
template <class T>
struct Load {
    const int8_t *q;
    const uint8_t *e;
    const T *dh;  // ckpt8_load_k: z, h; act_bwd_ckpt8_k: dh, dz
    T *z, *h, *dz;
    int ldq, lde, lddh, ldz, ldh, lddz, R, C, lshift;
};

template <int DT>
__global__ __launch_bounds__(kNT) void ckpt8_save_k(const Save<typename Io<DT>::T> a) {
    const auto *__restrict__ x = a.x;
    int8_t *__restrict__ q = a.q;
    uint8_t *__restrict__ e = a.e;
    const int ldx = a.ldx, ldq = a.ldq, lde = a.lde, R = a.R, C = a.C, lshift = a.lshift;
    using IO = Io<DT>;
    constexpr int E = IO::E, kLanes = kBlock / E;  // lanes of a block
    const Tile t(R, lshift);
    if (!t.in) return;
    const auto *xr = x + t.row * ldx;
    const int nb = C / E, chunks = ((C - 1) / kBlock + 1) * kLanes;  // whole blocks of lanes
    u32x4 w[kDeep];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
        const int j = t.first + u * t.step;
        if (j < chunks) w[u] = Chunk<DT>::load(xr, j, nb, C);
    }
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
        const int j = t.first + u * t.step;
        if (j >= chunks) break;
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < E; ++k) m = max(m, __float_as_uint(IO::get(w[u], k)) & 0x7fffffffu);
        // The block's other lanes (all here: chunks come in whole blocks).
        m = max(m, (uint32_t)fg::smrow::dpp_i<fg::smrow::kDppSwap1>((int)m));
        m = max(m, (uint32_t)fg::smrow::dpp_i<fg::smrow::kDppSwap2>((int)m));
        if constexpr (kLanes == 8)
            m = max(m, (uint32_t)fg::smrow::dpp_i<fg::smrow::kDppHalfMirror>((int)m));
        const int b = max(1, (int)(m >> 23));
        Bytes<E> o;
#pragma unroll
        for (int k = 0; k < E; k += 4) {
            uint32_t p = 0;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float s =
                    __builtin_rintf(__builtin_amdgcn_ldexpf(IO::get(w[u], k + n), 133 - b));
                const int c = (int)__builtin_amdgcn_fmed3f(s, -127.0f, 127.0f);
                p |= ((uint32_t)c & 255u) << (8 * n);
            }
            o.w[k / 4] = b == 255 ? 0u : p;
        }
        o.store(q + t.row * ldq, j, nb, C);
        if (j % kLanes == 0) e[t.row * lde + j / kLanes] = (uint8_t)b;
    }
}

// Restored values: bytes and exponents of a lane's chunks, loaded together.
template <int E>
struct Kept {
    static constexpr int kLanes = kBlock / E;
    Bytes<E> q[kDeep];
    int b[kDeep];
    __device__ __forceinline__ Kept(const Tile &t, const int8_t *qr, const uint8_t *er, int nb,
                                    int chunks, int C) {
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const int j = t.first + u * t.step;
            if (j >= chunks) continue;
            q[u].load(qr, j, nb, C);
            b[u] = er[j / kLanes];
        }
    }
    __device__ __forceinline__ void values(int u, float (&v)[E]) const {
        // 2^(b - 133), exact (down to 2^-132; fp32 denormals are on).
        const float s =
            b[u] == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(1.0f, b[u] - 133);
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] = (float)q[u].get(k) * s;
    }
};

template <int DT, int ACT>
__global__ __launch_bounds__(kNT) void ckpt8_load_k(const Load<typename Io<DT>::T> a) {
    const int8_t *__restrict__ q = a.q;
    const uint8_t *__restrict__ e = a.e;
    const int ldq = a.ldq, lde = a.lde, R = a.R, C = a.C, lshift = a.lshift;
    auto *z = a.z, *h = a.h;
    const int ldz = a.ldz, ldh = a.ldh;
    constexpr int E = Io<DT>::E;
    const Tile t(R, lshift);
    if (!t.in) return;
    const int nb = C / E, chunks = (C - 1) / E + 1;
    const Kept<E> kept(t, q + t.row * ldq, e + t.row * lde, nb, chunks, C);
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
        const int j = t.first + u * t.step;
        if (j >= chunks) break;
        float v[E];
        kept.values(u, v);
        if (z) Chunk<DT>::store(z + t.row * ldz, j, nb, C, v);
        if (h) {
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = fg::act_fwd(ACT, v[k]);
            Chunk<DT>::store(h + t.row * ldh, j, nb, C, v);
        }
    }
}

template <int DT, int ACT>
__global__ __launch_bounds__(kNT) void act_bwd_ckpt8_k(const Load<typename Io<DT>::T> a) {
    const int8_t *__restrict__ q = a.q;
    const uint8_t *__restrict__ e = a.e;
    const int ldq = a.ldq, lde = a.lde, R = a.R, C = a.C, lshift = a.lshift;
    const auto *dh = a.dh;
    auto *dz = a.dz;
    const int lddh = a.lddh, lddz = a.lddz;
    using IO = Io<DT>;
    constexpr int E = IO::E;
    const Tile t(R, lshift);
    if (!t.in) return;
    const int nb = C / E, chunks = (C - 1) / E + 1;
    u32x4 w[kDeep];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
        const int j = t.first + u * t.step;
        if (j < chunks) w[u] = Chunk<DT>::load(dh + t.row * lddh, j, nb, C);
    }
    const Kept<E> kept(t, q + t.row * ldq, e + t.row * lde, nb, chunks, C);
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
        const int j = t.first + u * t.step;
        if (j >= chunks) break;
        float v[E];
        kept.values(u, v);
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] = IO::get(w[u], k) * fg::act_grad(ACT, v[k]);
        Chunk<DT>::store(dz + t.row * lddz, j, nb, C, v);
    }
}

struct Shape {
    dim3 grid;
    int lshift;
};
Shape shape_of(int dtype, int R, int C) {
    Shape s;
    const int E = dtype == FG_DTYPE_F32 ? 4 : 8;
    const int chunks = ((C - 1) / kBlock + 1) * (kBlock / E);  // whole blocks
    s.lshift = 3;  // (at least a block's lanes)
    while (s.lshift < 8 && (kDeep << s.lshift) < chunks) ++s.lshift;
    const int rows = kNT >> s.lshift;
    s.grid = dim3((R - 1) / rows + 1, (chunks - 1) / (kDeep << s.lshift) + 1);
    return s;
}

// f<DT, ACT>() for run-time codes.
template <class F>
void with_types(int dtype, int act, F f) {
    using std::integral_constant;
    auto with_act = [&](auto dt) {
        if (act == FG_ACT_RELU) f(dt, integral_constant<int, fg::kActRelu>{});
        else if (act == FG_ACT_GELU) f(dt, integral_constant<int, fg::kActGelu>{});
        else f(dt, integral_constant<int, fg::kActNone>{});
    };
    if (dtype == FG_DTYPE_F32) with_act(integral_constant<int, fg::kF32>{});
    else if (dtype == FG_DTYPE_BF16) with_act(integral_constant<int, fg::kBF16>{});
    else with_act(integral_constant<int, fg::kF16>{});
}

int check_q(const char *who, int dtype, int R, int C, const void *q, int ldq, const void *e,
            int lde) {
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape %d x %d", who, R, C);
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(ldq >= C, FG_ERR_SHAPE, "%s: ldq=%d < %d columns", who, ldq, C);
    FG_REQUIRE(lde >= (C - 1) / kBlock + 1, FG_ERR_SHAPE,
               "%s: lde=%d < %d exponents (one per 32 columns)", who, lde, (C - 1) / kBlock + 1);
    FG_REQUIRE(q && e, FG_ERR_INVALID_ARGUMENT, "%s: q and e are required", who);
    FG_REQUIRE(R == 0 || fg::rows::grid_holds(shape_of(dtype, R, C).grid.x, kNT),
               FG_ERR_OUT_OF_BOUNDS, "%s: %d rows of %d columns", who, R, C);
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
    FG_REQUIRE(apart(d_q, {d_x, d_e}) && apart(d_e, {d_x}), FG_ERR_INVALID_ARGUMENT,
               "%s: x, q and e must be apart", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const Shape s = shape_of(dtype, R, C);
    auto launch = [&](auto dt) {
        using T = typename Io<dt()>::T;
        ckpt8_save_k<dt()><<<s.grid, kNT, 0, ctx->stream>>>(
            {static_cast<const T *>(d_x), d_q, d_e, ldx, ldq, lde, R, C, s.lshift});
    };
    with_types(dtype, FG_ACT_NONE, [&](auto dt, auto) { launch(dt); });
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
    FG_REQUIRE(d_z != d_h, FG_ERR_INVALID_ARGUMENT, "%s: z is h", who);
    FG_REQUIRE((!d_z || ldz >= C) && (!d_h || ldh >= C), FG_ERR_SHAPE,
               "%s: ldz=%d or ldh=%d < C=%d", who, ldz, ldh, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_z, {d_q, d_e}) && apart(d_h, {d_q, d_e}), FG_ERR_INVALID_ARGUMENT,
               "%s: z or h is q or e", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const Shape s = shape_of(dtype, R, C);
    with_types(dtype, act, [&](auto dt, auto a) {
        using T = typename Io<dt()>::T;
        ckpt8_load_k<dt(), a()><<<s.grid, kNT, 0, ctx->stream>>>(
            {d_q, d_e, nullptr, static_cast<T *>(d_z), static_cast<T *>(d_h), nullptr, ldq, lde, 0,
             ldz, ldh, 0, R, C, s.lshift});
    });
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
    FG_REQUIRE(d_dZ != d_dH || lddz == lddh, FG_ERR_INVALID_ARGUMENT,
               "%s: dZ is dH, but lddz=%d, lddh=%d", who, lddz, lddh);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_dZ, {d_q, d_e}), FG_ERR_INVALID_ARGUMENT, "%s: dZ is q or e", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const Shape s = shape_of(dtype, R, C);
    with_types(dtype, act, [&](auto dt, auto a) {
        using T = typename Io<dt()>::T;
        act_bwd_ckpt8_k<dt(), a()><<<s.grid, kNT, 0, ctx->stream>>>(
            {d_q, d_e, static_cast<const T *>(d_dH), nullptr, nullptr, static_cast<T *>(d_dZ), ldq,
             lde, lddh, 0, 0, lddz, R, C, s.lshift});
    });
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
    FG_REQUIRE(d_Xr && (act != FG_ACT_GELU || d_Zr), FG_ERR_INVALID_ARGUMENT,
               "%s: Xr, and for GELU Zr, is required", who);
    auto free = [&](const void *r) {
        return apart(r, {d_q, d_e, d_W, d_dZ, d_dX, d_dW, d_dbias});
    };
    FG_REQUIRE(d_Xr != d_Zr && free(d_Xr) && free(d_Zr), FG_ERR_INVALID_ARGUMENT,
               "%s: Xr and Zr must not be an operand, an output or each other", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    // One pass restores z and act(z), 6 % of the call at bf16 2048 x 4096 x 4096 (8.6 us of
    // 148; fp32 26 us of 981), then the products as from kept activations: act(z) is
    // rounded to the type, which is what the matrix instructions take and what the forward
    // multiplied (in bf16 that is half of dW's error, 0.0024 normwise of fp64 where its
    // own rounding makes 0.0017; without it dW's product would take act(z) in two parts,
    // twice the work).  Nothing else is rounded before it is stored: dX 0.0017, with its
    // product rounded before act'(z) multiplies it 0.0023.
    // [act(z) > 0] == [z > 0] for ReLU, whose derivative then reads Xr.
    void *zr = act == FG_ACT_GELU ? d_Zr : nullptr;
    if (int rc = fg_ckpt8_load(ctx, dtype, act, d_q, ldq, d_e, lde, M, K, zr, K, d_Xr, K))
        return rc;
    const void *zs = act == FG_ACT_RELU ? d_Xr : zr;
    if (dtype == FG_DTYPE_F32)
        return fg_matmul_bwd_f32(ctx, M, N, K, (const float *)d_Xr, K, (const float *)d_W, ldw,
                                 (const float *)d_dZ, lddz, act, (const float *)zs, K,
                                 (float *)d_dX, lddx, (float *)d_dW, lddw, (float *)d_dbias,
                                 accumulate);
    // dW: TN K x N over M; dX: NT M x K over N.
    return fg::gemm16_dw_dx(ctx, dtype, K, N, M, d_Xr, K, d_dZ, lddz, d_dW, lddw, accumulate,
                            d_dbias, accumulate, M, K, N, d_dZ, lddz, d_W, ldw, act, zs, K, d_dX,
                            lddx, accumulate, true);
}
