// k_attention.hip -- entry points of attention over packed sequences with grouped
// heads, for prompts, single tokens over a cache, and training.  The kernels, and the
// mathematics, are in fg_attention_kernel.h.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fg_attention.h"
#include "fg_half.h"
#include "fg_internal.h"
#include "fg_rows.h"

namespace {

using fg::attn::Args;
using fg::rows::apart;

constexpr int kMaxD = 128;      // columns of a head
constexpr int kMaxSplits = 32;  // of a row's keys

// Few rows a sequence (single tokens).
bool few_rows(const Args &a) { return (int64_t)a.Tq * a.G <= (int64_t)a.n * fg::attn::kFewRows; }

// Whether few rows go to the kernel whose waves share out the keys, rather than to the
// one of 128 rows, of which most are idle.  fp32, always: the idle rows' products are what
// bounds the other (single tokens over caches of up to 8192, 16 heads of 128 over 4:
// 1 token 46 us and 96, 8 tokens 79 and 166, 64 tokens 340 and 698).  16 bits, where heads
// and sequences are few and rows lie on 16-byte boundaries (32 heads of 128 over 8: 1
// token 24 and 28, 8 tokens 32 and 33, of heads of 64 22 and 25); of more the other brings
// the bytes sooner (32 tokens 134 and 122, 64 tokens 233 and 224, 8 tokens off the
// boundaries 51 and 38).
bool few_kernel(int cus, int dtype, const Args &a, bool aligned) {
    return few_rows(a) &&
           (dtype == FG_DTYPE_F32 || (aligned && (int64_t)a.n * a.KV * 4 <= cus));
}

// Splits of each sequence's keys, from what the host knows, of no fewer than 512 keys in a
// sequence of average length: two workgroups for every CU, fp32's few rows four; eight
// where few rows have as many workgroups as CUs unsplit, since the sequences' lengths
// differ (up to 8192 at random, 32 heads of 128 over 8, two and eight a CU: 32 tokens 127
// us and 122, 64 tokens 238 and 224, 8 tokens 33 and 41).
int splits_of(int cus, int dtype, const Args &a, bool few) {
    const int per = few ? fg::attn::kFewRows : fg::attn::kRows;
    const int64_t tiles = std::max<int64_t>(a.n, ((int64_t)a.Tq * a.G + per - 1) / per) * a.KV;
    const int a_cu = few ? (dtype == FG_DTYPE_F32 ? 4 : 2) : few_rows(a) && tiles >= cus ? 8 : 2;
    const int64_t want = a_cu * (int64_t)cus / std::max<int64_t>(tiles, 1);
    const int64_t most = (int64_t)a.Tk / a.n / 512;
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxSplits}));
}

// Splits of a backward pass that sums over `all` rows (or keys) of n sequences, with
// `tiles` workgroups unsplit: for a sequence of average length as many as bring `fill`
// workgroups, of `least` at least; for the longest up to four times as many.
void bwd_splits(int fill, int least, int64_t tiles, int64_t all, int n, int &splits) {
    const int64_t want = fill / std::max<int64_t>(tiles, 1);
    const int64_t of = std::min<int64_t>({want, all / n / least, kMaxSplits});
    splits = of <= 1 ? 1 : (int)std::min<int64_t>({4 * of, all / 128, kMaxSplits});
}

// (A CU holds two workgroups, of fp32 one.)
void set_splits(int cus, int dtype, Args &a) {
    const int fill = dtype == FG_DTYPE_F32 ? cus : 2 * cus;
    const int64_t rows = (int64_t)a.Tq * a.G;
    const int64_t q_tiles = std::max<int64_t>(a.n, (rows - 1) / fg::attn::kRows + 1) * a.KV;
    const int64_t k_tiles = std::max<int64_t>(a.n, ((int64_t)a.Tk - 1) / fg::attn::kKeys + 1) * a.KV;
    // Many workgroups' splits pay for their sums' way through memory only where they are
    // long.  (8 heads of 128, bf16, in splits of 128 and unsplit: one sequence of 512 49 us
    // and 57, of 1024 67 and 91, four of 512 75 and 58.  fp32, heads of 64: four of 512
    // 139 and 153.)
    auto least = [&](int64_t tiles) {
        return dtype != FG_DTYPE_F32 && tiles * 4 > cus ? 512 : 128;
    };
    bwd_splits(fill, least(q_tiles), q_tiles, a.Tk, a.n, a.splits);
    bwd_splits(fill, least(k_tiles), k_tiles, rows, a.n, a.ksplits);
    // (Those are not spread over the XCDs evenly: one more than the CUs of one hold is a
    // second round.  fp32: 162 us where 7 / 8 are filled, 195 where all.)
    a.fill = fill - fill / 8;
}

// Work slots of the passes over rows, 128 a workgroup.
int q_slots(const Args &a) { return (int)((int64_t)a.Tq * a.G / fg::attn::kRows + a.n); }

// Floats of the backward's workspace.
struct BwdSpace {
    uint64_t rows, tiles, part = 0, kpart = 0;
    explicit BwdSpace(const Args &a) {
        const uint64_t all = (uint64_t)std::max(a.Tq, 1) * a.KV * a.G;
        rows = (3 * all + 3) / 4 * 4;
        tiles = 16 * (uint64_t)a.KV * q_slots(a);
        if (a.splits > 1) part = (a.splits * all * a.D + 3) / 4 * 4;
        if (a.ksplits > 1) kpart = 2 * (uint64_t)a.ksplits * a.KV * a.Tk * a.D;
    }
    uint64_t bytes() const { return (rows + tiles + part + kpart) * sizeof(float); }
};

// Floats of the forward's.
uint64_t fwd_space(const Args &a) {
    return a.splits > 1 ? (uint64_t)a.splits * a.Tq * a.KV * a.G * (a.D + 2) : 0;
}

Args args_of(const fg::AttentionShape &s) {
    Args a{};
    a.n = s.n;
    a.Tq = s.Tq;
    a.Tk = s.Tk;
    a.KV = s.kv_heads;
    a.G = s.heads / s.kv_heads;
    a.D = s.D;
    return a;
}

// Rows of 16-bit elements at 16-byte boundaries, a tile's within 32 bits of its first.
bool aligned(std::initializer_list<std::pair<const void *, int64_t>> rows) {
    for (const auto &r : rows)
        if (((uintptr_t)r.first & 15) || r.second % 8 || r.second >= 1 << 24) return false;
    return true;
}
bool whole_chunks(const Args &a) { return a.D == 64 || a.D == 128; }

// What both directions ask of their arguments.
int check(const char *who, int dtype, const Args &a, int heads, int kv_heads) {
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(a.n >= 0 && a.Tq >= 0 && a.Tk >= 0 && heads > 0 && kv_heads > 0 && a.D > 0,
               FG_ERR_SHAPE, "%s: bad shape n=%d Tq=%d Tk=%d heads=%d kv_heads=%d D=%d", who, a.n,
               a.Tq, a.Tk, heads, kv_heads, a.D);
    FG_REQUIRE(heads % kv_heads == 0, FG_ERR_SHAPE, "%s: %d heads are no multiple of %d key heads",
               who, heads, kv_heads);
    FG_REQUIRE(a.D <= kMaxD, FG_ERR_UNSUPPORTED, "%s: heads of %d columns, at most %d", who, a.D,
               kMaxD);
    const int64_t wide = (int64_t)heads * a.D, kv_wide = (int64_t)kv_heads * a.D;
    FG_REQUIRE(wide < INT32_MAX && a.ldq >= wide && a.ldk >= kv_wide && a.ldv >= kv_wide,
               FG_ERR_SHAPE, "%s: ldq=%lld, ldk=%lld or ldv=%lld too small for %d and %d heads", who,
               (long long)a.ldq, (long long)a.ldk, (long long)a.ldv, heads, kv_heads);
    FG_REQUIRE(a.scale > 0.0f && a.scale < INFINITY, FG_ERR_INVALID_ARGUMENT,
               "%s: scale must be positive and finite", who);
    // Rows of a key head are counted in 32 bits, and a grid holds the slots.
    const int64_t slots = (int64_t)a.Tq * (heads / kv_heads) / fg::attn::kFewRows + a.n;
    const int64_t kslots = (int64_t)a.Tk / fg::attn::kKeys + a.n;
    FG_REQUIRE((int64_t)a.Tq * (heads / kv_heads) < INT32_MAX - 256 && a.Tk < INT32_MAX - 256 &&
                   fg::rows::grid_holds(kv_heads * std::max(slots, kslots), 256),
               FG_ERR_OUT_OF_BOUNDS, "%s: %d sequences of %d rows and %d keys with %d heads", who,
               a.n, a.Tq, a.Tk, heads);
    return FG_OK;
}

}  // namespace

uint64_t fg::attention_ws_bytes(int cus, int dtype, const AttentionShape &s) {
    Args a = args_of(s);
    uint64_t most = 0;  // (whatever the rows' alignment)
    for (bool on : {false, true}) {
        a.splits = splits_of(cus, dtype, a, few_kernel(cus, dtype, a, on));
        most = std::max(most, fwd_space(a) * sizeof(float));
    }
    return most;
}

uint64_t fg::attention_bwd_ws_bytes(int cus, int dtype, const AttentionShape &s) {
    Args a = args_of(s);
    set_splits(cus, dtype, a);
    return BwdSpace(a).bytes();
}

int fg::attention_dispatches(int cus, int dtype, const AttentionShape &s) {
    return attention_ws_bytes(cus, dtype, s) ? 2 : 1;
}

int fg::attention_bwd_dispatches(int cus, int dtype, const AttentionShape &s) {
    Args a = args_of(s);
    set_splits(cus, dtype, a);
    return a.splits > 1 || a.ksplits > 1 ? 3 : 2;
}

FG_API int fg_attention(fg_ctx *ctx, int dtype, const void *d_q, int ldq, const void *d_k, int ldk,
                        const void *d_v, int ldv, const uint32_t *d_q_starts,
                        const uint32_t *d_k_starts, const uint32_t *d_k_lens, int n, int Tq, int Tk,
                        int heads, int kv_heads, int D, float scale, int causal, void *d_out,
                        int ldo, float *d_lse) {
    const char *who = "fg_attention";
    Args a{};
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.qs = d_q_starts;
    a.ks = d_k_starts;
    a.klens = d_k_lens;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.n = n;
    a.Tq = Tq;
    a.Tk = Tk;
    a.D = D;
    a.scale = scale;
    if (int rc = check(who, dtype, a, heads, kv_heads)) return rc;
    a.KV = kv_heads;
    a.G = heads / kv_heads;
    a.group = fg::attn::Div((uint32_t)a.G);
    a.causal = causal != 0;
    a.out = d_out;
    a.ldo = ldo;
    a.lse = d_lse;
    FG_REQUIRE(ldo >= heads * D, FG_ERR_SHAPE, "%s: ldo=%d < %d heads of %d", who, ldo, heads, D);
    // (What has no rows needs no memory.)
    FG_REQUIRE((Tq == 0 || (d_q && d_out)) && (Tk == 0 || (d_k && d_v)) && d_q_starts && d_k_starts,
               FG_ERR_INVALID_ARGUMENT, "%s: q, k, v, the starts and out are required", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_out, {d_q, d_k, d_v, d_q_starts, d_k_starts, d_k_lens, d_lse}) &&
                   apart(d_lse, {d_q, d_k, d_v, d_q_starts, d_k_starts, d_k_lens}),
               FG_ERR_INVALID_ARGUMENT, "%s: an output is another output or an input", who);
    if (n == 0 || Tq == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const bool on = aligned({{d_k, ldk}, {d_v, ldv}}), dma = on && whole_chunks(a);
    const bool few = few_kernel(ctx->cu_count, dtype, a, on);
    a.splits = splits_of(ctx->cu_count, dtype, a, few);
    if (a.splits > 1) {
        a.part = (float *)fg::workspace(ctx, fwd_space(a) * sizeof(float));
        if (!a.part) return FG_ERR_OUT_OF_MEMORY;
    }
    a.slots = (int)((int64_t)Tq * a.G / (few ? fg::attn::kFewRows : fg::attn::kRows) + n);
    auto launch = dtype == FG_DTYPE_F32    ? fg::attn::forward<fg::kF32>
                  : dtype == FG_DTYPE_BF16 ? fg::attn::forward<fg::kBF16>
                                           : fg::attn::forward<fg::kF16>;
    FG_HIP((hipError_t)launch(ctx->stream, a, few, dma));
    if (a.splits > 1) {
        auto join = dtype == FG_DTYPE_F32    ? fg::attn::combine<fg::kF32>
                    : dtype == FG_DTYPE_BF16 ? fg::attn::combine<fg::kBF16>
                                             : fg::attn::combine<fg::kF16>;
        FG_HIP((hipError_t)join(ctx->stream, a));
    }
    return FG_OK;
}

FG_API int fg_attention_bwd(fg_ctx *ctx, int dtype, const void *d_q, int ldq, const void *d_k,
                            int ldk, const void *d_v, int ldv, const void *d_out, int ldo,
                            const void *d_dout, int lddo, const float *d_lse,
                            const uint32_t *d_q_starts, const uint32_t *d_k_starts, int n, int Tq,
                            int Tk, int heads, int kv_heads, int D, float scale, int causal,
                            void *d_dq, int lddq, void *d_dk, int lddk, void *d_dv, int lddv,
                            int accumulate) {
    const char *who = "fg_attention_bwd";
    Args a{};
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.qs = d_q_starts;
    a.ks = d_k_starts;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.n = n;
    a.Tq = Tq;
    a.Tk = Tk;
    a.D = D;
    a.scale = scale;
    if (int rc = check(who, dtype, a, heads, kv_heads)) return rc;
    // (16 bits: lse enters the products' sums in units of 1 / scale.)
    FG_REQUIRE(dtype == FG_DTYPE_F32 || scale >= 0x1p-120f, FG_ERR_UNSUPPORTED,
               "%s: a scale of %g, in 16 bits at least 2^-120", who, (double)scale);
    a.KV = kv_heads;
    a.G = heads / kv_heads;
    a.group = fg::attn::Div((uint32_t)a.G);
    a.causal = causal != 0;
    a.out = const_cast<void *>(d_out);
    a.ldo = ldo;
    a.lse = const_cast<float *>(d_lse);
    a.dout = d_dout;
    a.lddo = lddo;
    a.dq = d_dq;
    a.lddq = lddq;
    a.dk = d_dk;
    a.lddk = lddk;
    a.dv = d_dv;
    a.lddv = lddv;
    a.accumulate = accumulate != 0;
    FG_REQUIRE(ldo >= heads * D && lddo >= heads * D && lddq >= heads * D, FG_ERR_SHAPE,
               "%s: ldo=%d, lddo=%d or lddq=%d < %d heads of %d", who, ldo, lddo, lddq, heads, D);
    FG_REQUIRE(lddk >= kv_heads * D && lddv >= kv_heads * D, FG_ERR_SHAPE,
               "%s: lddk=%d or lddv=%d < %d heads of %d", who, lddk, lddv, kv_heads, D);
    FG_REQUIRE((Tq == 0 || (d_q && d_out && d_dout && d_lse)) && (Tk == 0 || (d_k && d_v)) &&
                   d_q_starts && d_k_starts,
               FG_ERR_INVALID_ARGUMENT, "%s: q, k, v, out, dout, lse and the starts are required",
               who);
    FG_REQUIRE((Tq == 0 || d_dq) && (Tk == 0 || (d_dk && d_dv)), FG_ERR_INVALID_ARGUMENT,
               "%s: dq, dk and dv are required", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    for (const void *o : {(const void *)d_dq, (const void *)d_dk, (const void *)d_dv})
        FG_REQUIRE(apart(o, {d_q, d_k, d_v, d_out, d_dout, d_lse, d_q_starts, d_k_starts}),
                   FG_ERR_INVALID_ARGUMENT, "%s: an output is an input", who);
    FG_REQUIRE(apart(d_dq, {d_dk, d_dv}) && apart(d_dk, {d_dv}), FG_ERR_INVALID_ARGUMENT,
               "%s: an output is another output", who);
    if (n == 0 || (Tq == 0 && Tk == 0)) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    set_splits(ctx->cu_count, dtype, a);
    const BwdSpace need(a);
    float *ws = (float *)fg::workspace(ctx, need.bytes());
    if (!ws) return FG_ERR_OUT_OF_MEMORY;
    a.rows = ws;
    a.tiles = ws + need.rows;
    a.part = a.tiles + need.tiles;
    a.kpart = a.part + need.part;
    a.slots = q_slots(a);
    a.kslots = Tk / fg::attn::kKeys + n;
    const bool dma =
        whole_chunks(a) && aligned({{d_q, ldq}, {d_k, ldk}, {d_v, ldv}, {d_dout, lddo}});
    auto launch = dtype == FG_DTYPE_F32    ? fg::attn::backward<fg::kF32>
                  : dtype == FG_DTYPE_BF16 ? fg::attn::backward<fg::kBF16>
                                           : fg::attn::backward<fg::kF16>;
    FG_HIP((hipError_t)launch(ctx->stream, a, dma));
    return FG_OK;
}
