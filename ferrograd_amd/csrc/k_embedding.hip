// k_embedding.hip -- embedding lookup with scaling and the table's gradient by
// sorted tokens, for gfx950.  The reference has no lookup: its inputs are
// dense, and only its labels are u32 (basic_loss.rs:91-133).
//
//   out[t][c] = scale * table[tokens[t]][c]       (NaN where tokens[t] >= V)
//   dtable[v][c] (=|+=) scale * sum of dout[t][c] over t with tokens[t] == v
//
// The gradient's sums run in fp32 in an order fixed by the tokens alone, so
// equal calls give equal bits (no atomics).  Tokens outside the table add to
// nothing.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fg_half.h"
#include "fg_internal.h"

namespace {

constexpr int kNT = 256;

__global__ __launch_bounds__(kNT) void emb_fwd(int dt, const uint32_t *tokens, int V, int C,
                                               const void *table, int ldt, float scale, void *out,
                                               int ldo) {
    const uint64_t t = blockIdx.x;
    const uint32_t v = tokens[t];
    const bool in = v < (uint32_t)V;
    for (int c = threadIdx.x; c < C; c += kNT)
        fg::store_from_f(out, dt, t * ldo + c,
                         in ? scale * fg::load_as_f(table, dt, (uint64_t)v * ldt + c)
                            : __builtin_nanf(""));
}

// order[k] = the k-th token position in (token, position) order, sorted[k] its
// token.  A thread counts the positions before its own.
__global__ __launch_bounds__(kNT) void emb_rank(const uint32_t *tokens, int T, uint32_t *order,
                                                uint32_t *sorted) {
    const int i = blockIdx.x * kNT + threadIdx.x;
    if (i >= T) return;
    const uint32_t mine = tokens[i];
    int before = 0;
    for (int j = 0; j < T; ++j) {
        const uint32_t o = tokens[j];
        before += (o < mine || (o == mine && j < i)) ? 1 : 0;
    }
    order[before] = (uint32_t)i;
    sorted[before] = mine;
}

// First position of `sorted` that holds a value >= v.
__device__ __forceinline__ int lower_bound(const uint32_t *sorted, int T, uint32_t v) {
    int lo = 0, n = T;
    while (n > 0) {
        const int h = n >> 1;
        if (sorted[lo + h] < v) {
            lo += h + 1;
            n -= h + 1;
        } else {
            n = h;
        }
    }
    return lo;
}

__global__ __launch_bounds__(kNT) void emb_bwd_row(int dt, const uint32_t *order,
                                                   const uint32_t *sorted, int T, int C,
                                                   const void *dout, int ldo, float scale,
                                                   void *dtable, int ldt, int accumulate) {
    const uint32_t v = blockIdx.x;
    const int k0 = lower_bound(sorted, T, v);
    if (accumulate && (k0 >= T || sorted[k0] != v)) return;
    for (int c = threadIdx.x; c < C; c += kNT) {
        float s = 0.0f;
        for (int k = k0; k < T && sorted[k] == v; ++k)
            s += fg::load_as_f(dout, dt, (uint64_t)order[k] * ldo + c);
        s *= scale;
        const uint64_t at = (uint64_t)v * ldt + c;
        fg::store_from_f(dtable, dt, at, accumulate ? fg::load_as_f(dtable, dt, at) + s : s);
    }
}

}  // namespace

namespace fg {
uint64_t embedding_bwd_ws_bytes(int T, int V, int C) {
    (void)V;
    (void)C;
    return std::max<uint64_t>(1, (uint64_t)T) * 8;
}
}  // namespace fg

FG_API int fg_embedding(fg_ctx *ctx, int dtype, const uint32_t *d_tokens, int T, int V, int C,
                        const void *d_table, int ldt, float scale, void *d_out, int ldo) {
    const char *who = "fg_embedding";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(T >= 0 && V > 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape T=%d V=%d C=%d", who, T, V,
               C);
    FG_REQUIRE(ldt >= C && ldo >= C, FG_ERR_SHAPE, "%s: ldt=%d or ldo=%d < C=%d", who, ldt, ldo,
               C);
    FG_REQUIRE(T == 0 || (d_tokens && d_table && d_out), FG_ERR_INVALID_ARGUMENT,
               "%s: tokens, table and out are required", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    if (T == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    emb_fwd<<<T, kNT, 0, ctx->stream>>>(dtype, d_tokens, V, C, d_table, ldt, scale, d_out, ldo);
    FG_LAUNCH_CHECK("emb_fwd");
    return FG_OK;
}

FG_API int fg_embedding_bwd(fg_ctx *ctx, int dtype, const uint32_t *d_tokens, int T, int V, int C,
                            const void *d_dout, int lddo, float scale, void *d_dtable, int lddt,
                            int accumulate) {
    const char *who = "fg_embedding_bwd";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(T >= 0 && V > 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape T=%d V=%d C=%d", who, T, V,
               C);
    FG_REQUIRE(lddo >= C && lddt >= C, FG_ERR_SHAPE, "%s: lddo=%d or lddt=%d < C=%d", who, lddo,
               lddt, C);
    FG_REQUIRE(d_dtable && (T == 0 || (d_tokens && d_dout)), FG_ERR_INVALID_ARGUMENT,
               "%s: tokens, dout and dtable are required", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_HIP(hipSetDevice(ctx->device));
    uint32_t *order = (uint32_t *)fg::workspace(ctx, fg::embedding_bwd_ws_bytes(T, V, C));
    if (!order) return FG_ERR_OUT_OF_MEMORY;
    uint32_t *sorted = order + T;
    if (T > 0) {
        emb_rank<<<(T + kNT - 1) / kNT, kNT, 0, ctx->stream>>>(d_tokens, T, order, sorted);
        FG_LAUNCH_CHECK("emb_rank");
    }
    emb_bwd_row<<<V, kNT, 0, ctx->stream>>>(dtype, order, sorted, T, C, d_dout, lddo, scale,
                                            d_dtable, lddt, accumulate);
    FG_LAUNCH_CHECK("emb_bwd_row");
    return FG_OK;
}
