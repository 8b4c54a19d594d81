// k_logprobs.hip -- log probabilities of given tokens with the entropy and the most
// probable tokens of each row, and their gradient, for gfx950.  The reference answers
// with the softmax's values (crates/ferrograd-nn/src/op/softmax.rs:14-446) and its
// cross entropy (loss/basic_loss.rs:91-133).
//
// For a row x of C logits, z = scale * x, m = max z, s = sum exp(z - m):
//   lse = m + log(s),  logp = (z_token - m) - log(s)
//   entropy = log(s) + sum exp(z - m) (m - z) / s        (no difference of near values)
//   alternatives: the K largest x, the lower column first among equals
// Backward, from the gradients a of logp and b of entropy, p = exp(z - lse):
//   dx_c = scale * (a ([c = token] - p_c) - b p_c (z_c - lse + entropy))
// which needs no sum over the row again.
//
// Both are bound by HBM, and in 16 bits by the vector unit beside it: the forward reads
// a row once, with a running maximum and sums a thread that are raised together; the
// backward reads and writes each logit once.  fp32 4096 x 50257 with 5 alternatives: 155
// us, 5.3 TB/s (a large copy reaches 4.9); bf16 64 x 131072 with 20: 15, of which the
// splits' pass is 10.6 and their join 5 (8 in all without alternatives); backward, bf16
// 8192 x 32000, a quarter of the rows padding: 183 us, 5 TB/s.
//   Rows that have fewer logits above the others than alternatives are asked for take a
// pass an alternative: masked to 10 of their columns, with 20 alternatives, 64 x 131072 114
// us (15 with 1000 left) and 8192 x 32000 2.2 ms (0.12).
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

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
constexpr int kMaxTop = 32;   // alternatives: at most the 64 groups of threads
constexpr int kCands = 512;   // candidates for them kept at once

// A number's place among a row's, as an unsigned integer: -0 as +0, NaN below all.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Running maximum m of x * c (c = scale log2 e) and, of e = 2^(x c - m), the sums
// s of e and w of e (x c - m).
struct Stats {
    float m = -INFINITY, s = 0.0f, w = 0.0f;
    // To the maximum `to` (m: as it was).
    __device__ __forceinline__ void raise(float to) {
        if (!(to > m)) return;
        const float d = m - to, f = __builtin_amdgcn_exp2f(d);
        w = s > 0.0f ? f * (w + s * d) : w;  // (s = 0: no number yet, d may be -inf)
        s *= f;
        m = to;
    }
    // A value, with from = m (0 before the first number).  exp2 of -inf is 0, and so is
    // that value's share of w; NaN goes into s.
    __device__ __forceinline__ void add(float x, float c, float from) {
        const float d = __builtin_fmaf(x, c, -from), e = __builtin_amdgcn_exp2f(d);
        s += e;
        w = __builtin_fmaf(e, fmaxf(d, -1000.0f), w);
    }
    __device__ __forceinline__ float from() const { return m == -INFINITY ? 0.0f : m; }
};

// What a row's log probabilities are taken from: its maximum m times c, or where that
// product's rounding is not far below 1 or the product past fp32 (a row of nothing but
// masks of -1e10, or of the type's lowest number) the maximum logit itself, `raw`.
constexpr float kFar = 0x1p20f;
__device__ __forceinline__ bool is_raw(float m, float most) {
    return fabsf(m) >= kFar && fabsf(most) < INFINITY;
}
struct Base {
    float m;
    bool raw;
    // scale (x - max x)
    __device__ __forceinline__ float from_max(float x, float scale, float c) const {
        if (raw) return (x - m) * scale;
        const float d = __builtin_fmaf(x, c, -m) * kLn2;
        // (A finite logit so low that its product with c alone is past fp32.)
        return d == -INFINITY ? __builtin_fmaf(x, scale, -m * kLn2) : d;
    }
    __device__ __forceinline__ float lse(float scale, float log_s) const {
        return __builtin_fmaf(m, raw ? scale : kLn2, log_s);
    }
};

// Largest over a wave's 64 lanes (all active), the same in every lane, NaN left out.
__device__ __forceinline__ float wave_max(float v) {
    using namespace fg::smrow;
    v = fmaxf(v, dpp_f<kDppSwap1>(v));
    v = fmaxf(v, dpp_f<kDppSwap2>(v));
    v = fmaxf(v, dpp_f<kDppHalfMirror>(v));
    v = fmaxf(v, dpp_f<kDppMirror>(v));
    auto of = [&](int lane) {
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
    };
    return fmaxf(fmaxf(of(0), of(16)), fmaxf(of(32), of(48)));
}
// A value's place among a row's and its column as one number: larger is earlier.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int col) {
    return (uint64_t)key << 32 | (uint32_t)~col;
}
__device__ __forceinline__ int col_of(uint64_t place) { return (int)~(uint32_t)place; }
// How many of `all` come before v.
__device__ __forceinline__ int before_in(const uint64_t *all, int n, uint64_t v) {
    int before = 0;
#pragma unroll 8
    for (int k = 0; k < n; ++k) before += all[k] > v;
    return before;
}

struct Fwd {
    const void *x;
    const uint32_t *tokens;
    float *logp, *entropy, *lse;
    uint32_t *ids;
    float *tops;
    float scale;
    int ldx, C, K;
    // Rows in splits of their columns: [R][splits] of four statistics (Stats and the largest
    // logit), and of K places (place_of) in order.
    int splits;
    float *stats;
    uint64_t *best;
};

// A row's answers from its statistics, in thread 0.
__device__ __forceinline__ void write_answers(const Fwd &a, size_t r, const Stats &st, Base base,
                                              float log_s, float xt, bool inside, float c) {
    if (a.logp)
        a.logp[r] = inside ? base.from_max(xt, a.scale, c) - log_s : __builtin_nanf("");
    if (a.entropy) a.entropy[r] = log_s - kLn2 * (st.w / st.s);
    if (a.lse) a.lse[r] = base.lse(a.scale, log_s);
}
// The alternative at `place`: its column and log probability.
template <int DT>
__device__ __forceinline__ void write_top(const Fwd &a, size_t r, int place, int col,
                                          const typename Io<DT>::T *x, Base base, float log_s,
                                          float c) {
    if (a.ids) a.ids[r * a.K + place] = (uint32_t)col;
    if (a.tops)
        a.tops[r * a.K + place] = base.from_max(Io<DT>::load1(x, col), a.scale, c) - log_s;
}

// A row (or a split of its columns) a workgroup of NT threads, read once; for the
// alternatives the chunks of the threads that hold one (about as many as there are) are
// read again, by all threads.
//   The K-th largest of the maxima of 64 groups of threads is no more than the row's
// K-th largest value, so every alternative is among the values from it on: about as
// many as K where the large values lie anyhow.  Where they are more than fit (rows of
// few different values), the K are taken one after the other, a pass over the row each.
template <int DT, int NT>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(8))) void logprobs_fwd(
    const Fwd a) {
    using IO = Io<DT>;
    constexpr int E = IO::E, NW = NT / 64, kDeep = 4;
    __shared__ float sm[NW][3];
    __shared__ uint32_t keys[NT];
    __shared__ uint64_t cand[kCands];
    __shared__ int hot[NT];
    __shared__ uint32_t bound_s;
    __shared__ int count_s, hot_s;
    const size_t r = blockIdx.x;
    const int split = blockIdx.y;
    const auto *x = static_cast<const typename IO::T *>(a.x) + r * a.ldx;
    const int t = threadIdx.x, whole = a.C / E;
    const int j0 = (int)((int64_t)whole * split / a.splits);
    const int nb = (int)((int64_t)whole * (split + 1) / a.splits);
    const float c = a.scale * kLog2e;
    const int single = split == a.splits - 1 && t < a.C - whole * E ? whole * E + t : -1;
    const uint32_t token = a.tokens[r];
    const bool inside = token < (uint32_t)a.C;
    const float xt = inside ? IO::load1(x, (int)token) : 0.0f;
    Stats st;
    float big = -INFINITY;  // the thread's largest value
    auto take = [&](u32x4 w) {
        float b = IO::get(w, 0);
#pragma unroll
        for (int e = 1; e < E; ++e) b = fmaxf(b, IO::get(w, e));
        big = fmaxf(big, b);
        // Raised only by values 2^4 above the maximum, which are few after the first
        // chunks; the exact one comes at the end.
        if (__any(b * c > st.m + 4.0f)) st.raise(b * c);
        const float from = st.from();
#pragma unroll
        for (int e = 0; e < E; ++e) st.add(IO::get(w, e), c, from);
    };
    int j = j0 + t;
    for (; j + (kDeep - 1) * NT < nb; j += kDeep * NT) {
        u32x4 w[kDeep];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) w[u] = fg::rows::load<DT>(x, j + u * NT);
#pragma unroll
        for (int u = 0; u < kDeep; ++u) take(w[u]);
    }
    for (; j < nb; j += NT) take(fg::rows::load<DT>(x, j));
    if (single >= 0) {
        const float v = IO::load1(x, single);
        st.raise(v * c);
        st.add(v, c, st.from());
        big = fmaxf(big, v);
    }
    // (0: no number among the thread's values, or nothing above -inf.)
    const uint32_t mine = big > -INFINITY ? order_key(big) : 0u;
    const float top = wave_max(big);
    if ((t & 63) == 0) sm[t >> 6][0] = top;
    if (a.K) {
        keys[t] = mine;
        if (t == 0) count_s = hot_s = 0;
    }
    __syncthreads();
    float most = sm[0][0];
#pragma unroll
    for (int k = 1; k < NW; ++k) most = fmaxf(most, sm[k][0]);
    const float m = most * c;
    st.raise(m);
    const float s = fg::rows::wave_sum(st.s), w = fg::rows::wave_sum(st.w);
    if ((t & 63) == 0) {
        sm[t >> 6][1] = s;
        sm[t >> 6][2] = w;
    }
    if (a.K && t < 64) {
        uint32_t g = keys[t];
#pragma unroll
        for (int k = 1; k < NW; ++k) g = max(g, keys[k * 64 + t]);
        int before = 0;
#pragma unroll 16
        for (int k = 0; k < 64; ++k) {
            const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)g, k);
            before += o > g || (o == g && k < t);
        }
        if (before == a.K - 1) bound_s = g;
    }
    __syncthreads();
    st.m = m;
    st.s = sm[0][1];
    st.w = sm[0][2];
#pragma unroll
    for (int k = 1; k < NW; ++k) {
        st.s += sm[k][1];
        st.w += sm[k][2];
    }
    Base base{m, false};
    if (is_raw(m, most)) {
        // The sums again from the largest logit.
        base = {most, true};
        Stats again;
        for (int i = j0 + t; i < nb; i += NT) {
            const u32x4 v = fg::rows::load<DT>(x, i);
#pragma unroll
            for (int e = 0; e < E; ++e) again.add(IO::get(v, e) - most, c, 0.0f);
        }
        if (single >= 0) again.add(IO::load1(x, single) - most, c, 0.0f);
        const float s2 = fg::rows::wave_sum(again.s), w2 = fg::rows::wave_sum(again.w);
        __syncthreads();
        if ((t & 63) == 0) {
            sm[t >> 6][1] = s2;
            sm[t >> 6][2] = w2;
        }
        __syncthreads();
        st.s = sm[0][1];
        st.w = sm[0][2];
#pragma unroll
        for (int k = 1; k < NW; ++k) {
            st.s += sm[k][1];
            st.w += sm[k][2];
        }
    }
    const float log_s = logf(st.s);
    const size_t part = r * a.splits + split;
    if (t == 0) {
        if (a.splits > 1) {
            a.stats[4 * part] = st.m;
            a.stats[4 * part + 1] = st.s;
            a.stats[4 * part + 2] = st.w;
            a.stats[4 * part + 3] = most;
        } else {
            write_answers(a, r, st, base, log_s, xt, inside, c);
        }
    }
    if (!a.K) return;
    const uint32_t bound = bound_s;
    auto keep = [&](uint32_t key, int col) {
        if (key < bound) return;
        const int at = atomicAdd(&count_s, 1);
        if (at < kCands) cand[at] = place_of(key, col);
    };
    if (mine >= bound) hot[atomicAdd(&hot_s, 1)] = t;
    if (single >= 0) keep(order_key(IO::load1(x, single)), single);
    __syncthreads();
    const int per = nb > j0 ? (nb - j0 - 1) / NT + 1 : 0;  // chunks of a thread, at most
    for (int i = t; i < hot_s * per; i += NT) {
        const int k = i / per, at = j0 + hot[k] + (i - k * per) * NT;
        if (at >= nb) continue;
        const u32x4 v = fg::rows::load<DT>(x, at);
#pragma unroll
        for (int e = 0; e < E; ++e) keep(order_key(IO::get(v, e)), at * E + e);
    }
    __syncthreads();
    auto write = [&](int at, uint64_t place) {
        if (a.splits > 1) a.best[part * a.K + at] = place;
        else write_top<DT>(a, r, at, col_of(place), x, base, log_s, c);
    };
    const int n = count_s;
    if (n >= a.K && n <= kCands) {
        for (int i = t; i < n; i += NT) {
            const uint64_t v = cand[i];
            const int before = before_in(cand, n, v);
            if (before < a.K) write(before, v);
        }
        return;
    }
    uint64_t last = ~0ull;  // the place of the one before
    for (int k = 0; k < a.K; ++k) {
        uint64_t next = 0;
        auto see = [&](uint32_t key, int col) {
            const uint64_t v = place_of(key, col);
            if (v < last) next = max(next, v);
        };
        for (int i = j0 + t; i < nb; i += NT) {
            const u32x4 v = fg::rows::load<DT>(x, i);
#pragma unroll
            for (int e = 0; e < E; ++e) see(order_key(IO::get(v, e)), i * E + e);
        }
        if (single >= 0) see(order_key(IO::load1(x, single)), single);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) next = max(next, (uint64_t)__shfl_xor((long long)next, o));
        __syncthreads();
        if ((t & 63) == 0) cand[t >> 6] = next;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NW; ++q) next = max(next, cand[q]);
        last = next;
        if (t == 0) write(k, next);
    }
}

// A row's splits joined, their numbers all loaded at once: the statistics, and of the
// alternatives those from the largest of the splits' K-th on.
constexpr int kMaxSplits = 16, kJoinNT = 256;
template <int DT>
__global__ __launch_bounds__(kJoinNT) void logprobs_join(const Fwd a) {
    constexpr int kPer = kMaxSplits * kMaxTop / kJoinNT;
    __shared__ uint64_t cand[kMaxSplits * kMaxTop];
    __shared__ int count_s;
    const size_t r = blockIdx.x;
    const auto *x = static_cast<const typename Io<DT>::T *>(a.x) + r * a.ldx;
    const int t = threadIdx.x, lane = t & 63, all = a.splits * a.K;
    const float c = a.scale * kLog2e;
    const uint64_t *best = a.best + r * all;
    const bool on = lane < a.splits;
    const float *p = a.stats + 4 * (r * a.splits + (on ? lane : 0));
    Stats st;
    st.m = on ? p[0] : -INFINITY;
    st.s = on ? p[1] : 0.0f;
    st.w = on ? p[2] : 0.0f;
    const float largest = on ? p[3] : -INFINITY;
    uint64_t mine[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        mine[i] = t + i * kJoinNT < all ? best[t + i * kJoinNT] : 0;
    uint64_t bound = on && a.K ? best[lane * a.K + a.K - 1] : 0;
    const uint32_t token = a.tokens[r];
    const bool inside = token < (uint32_t)a.C;
    const float xt = inside ? Io<DT>::load1(x, (int)token) : 0.0f;
    if (t == 0) count_s = 0;
    Base base{wave_max(st.m), false};
    const bool raw = is_raw(st.m, largest);
    if (__any(raw)) {
        // All from the largest logits: the others' sums by the rounding of theirs times c.
        base = {wave_max(largest), true};
        const float r = raw || largest == -INFINITY ? 0.0f : __builtin_fmaf(largest, c, -st.m);
        const float d = (largest - base.m) * c - r, f = __builtin_amdgcn_exp2f(d);
        st.w = f > 0.0f ? f * (st.w + st.s * d) : 0.0f;
        st.s *= f;
    } else {
        st.raise(base.m);
    }
    st.s = fg::rows::wave_sum(st.s);
    st.w = fg::rows::wave_sum(st.w);
    const float log_s = logf(st.s);
    if (t == 0) write_answers(a, r, st, base, log_s, xt, inside, c);
    if (!a.K) return;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) bound = max(bound, (uint64_t)__shfl_xor((long long)bound, o));
    bound = (uint64_t)__shfl((long long)bound, 0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (t + i * kJoinNT < all && mine[i] >= bound) cand[atomicAdd(&count_s, 1)] = mine[i];
    __syncthreads();
    const int n = count_s;
    for (int i = t; i < n; i += kJoinNT) {
        const int before = before_in(cand, n, cand[i]);
        if (before < a.K) write_top<DT>(a, r, before, col_of(cand[i]), x, base, log_s, c);
    }
}

struct Bwd {
    const void *x;
    const uint32_t *tokens;
    const float *lse, *entropy, *dlogp, *dentropy;
    void *dx;
    float scale;
    int ldx, lddx, R, C, lshift;
};

// Elementwise over rows of 2^lshift lanes, kBwdDeep chunks a lane, loaded together.
// The columns past a row's whole chunks go one to a lane, so that dx may be x.  Rows of
// no gradient (padding) are written as zeros and not read.
constexpr int kBwdNT = 256, kBwdDeep = 4;
template <int DT>
__global__ __launch_bounds__(kBwdNT) void logprobs_bwd(const Bwd a) {
    using IO = Io<DT>;
    using T = typename IO::T;
    constexpr int E = IO::E;
    const int64_t row = ((int64_t)blockIdx.x << (8 - a.lshift)) + (threadIdx.x >> a.lshift);
    if (row >= a.R) return;
    const int step = 1 << a.lshift;
    const int lane = threadIdx.x & (step - 1);
    const int first = (blockIdx.y << a.lshift) * kBwdDeep + lane;
    const T *x = static_cast<const T *>(a.x) + (size_t)row * a.ldx;
    T *dx = static_cast<T *>(a.dx) + (size_t)row * a.lddx;
    const int nb = a.C / E;
    const int single = blockIdx.y == 0 && lane < a.C - nb * E ? nb * E + lane : -1;
    const float ga = a.dlogp ? a.dlogp[row] * a.scale : 0.0f;
    const float gb = a.dentropy ? a.dentropy[row] * a.scale : 0.0f;
    if (ga == 0.0f && gb == 0.0f) {
        const float zeros[E] = {};
#pragma unroll
        for (int u = 0; u < kBwdDeep; ++u)
            if (first + u * step < nb) fg::rows::store<DT>(dx, first + u * step, IO::pack(zeros));
        if (single >= 0) IO::store1(dx, single, 0.0f);
        return;
    }
    const float lse = a.lse[row], h = gb != 0.0f ? a.entropy[row] : 0.0f;
    const uint32_t token = a.tokens[row];
    // (A row with NaN, or of -inf alone, has no gradients.)
    const float gn = fabsf(lse) < INFINITY ? ga : __builtin_nanf("");
    auto grad = [&](float v, bool hot) {
        // z - lse rounded once, kept where its exponential is one of a probability: a masked
        // logit's may be -inf, and lse's own rounding may lie between it and the largest z.
        const float d = __builtin_amdgcn_fmed3f(__builtin_fmaf(v, a.scale, -lse), -1000.0f, 0.0f);
        const float o = -__builtin_amdgcn_exp2f(d * kLog2e) * __builtin_fmaf(gb, d + h, gn);
        return hot ? o + ga : o;
    };
    u32x4 w[kBwdDeep];
#pragma unroll
    for (int u = 0; u < kBwdDeep; ++u)
        if (first + u * step < nb) w[u] = fg::rows::load<DT>(x, first + u * step);
#pragma unroll
    for (int u = 0; u < kBwdDeep; ++u) {
        const int j = first + u * step;
        if (j >= nb) break;
        const uint32_t hot = token - (uint32_t)(j * E);
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = grad(IO::get(w[u], e), hot == (uint32_t)e);
        fg::rows::store<DT>(dx, j, IO::pack(o));
    }
    if (single >= 0) IO::store1(dx, single, grad(IO::load1(x, single), token == (uint32_t)single));
}

// Splits of each row's columns: of few long rows, as many as give every CU two
// workgroups, of at least 8192 columns (64 x 131072 bf16, 20 alternatives: unsplit 21 us,
// two a CU 14, four 19; splits of 4096 to 16384 columns alike).
int splits_of(int cus, int R, int C) {
    return std::max(1, std::min({2 * cus / R, C / 8192, kMaxSplits}));
}

template <int DT>
void launch_fwd(hipStream_t st, int R, const Fwd &a) {
    // A wave a row up to 8 chunks a lane, else four waves (8192 rows of bf16, a wave and
    // four: 2048 columns 8.6 and 13.6 us, 4096 14.6 and 18.1, 16384 44 and 42).
    if (a.C / Io<DT>::E <= 512) logprobs_fwd<DT, 64><<<R, 64, 0, st>>>(a);
    else logprobs_fwd<DT, 256><<<dim3(R, a.splits), 256, 0, st>>>(a);
    if (a.splits > 1) logprobs_join<DT><<<R, 256, 0, st>>>(a);
}

template <int DT>
void launch_bwd(hipStream_t st, Bwd a) {
    const int chunks = std::max(1, a.C / Io<DT>::E);
    a.lshift = 3;  // at least as many lanes as columns past the whole chunks
    while (a.lshift < 8 && (kBwdDeep << a.lshift) < chunks) ++a.lshift;
    const dim3 grid(((int64_t)a.R - 1) / (kBwdNT >> a.lshift) + 1,
                    (chunks - 1) / (kBwdDeep << a.lshift) + 1);
    logprobs_bwd<DT><<<grid, kBwdNT, 0, st>>>(a);
}

}  // namespace

FG_API int fg_token_logprobs(fg_ctx *ctx, int dtype, const void *d_logits, int ldx,
                             const uint32_t *d_tokens, int R, int C, float scale, float *d_logp,
                             float *d_entropy, float *d_lse, int top, uint32_t *d_top_ids,
                             float *d_top_logp) {
    const char *who = "fg_token_logprobs";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape R=%d C=%d", who, R, C);
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(ldx >= C, FG_ERR_SHAPE, "%s: ldx=%d < C=%d", who, ldx, C);
    FG_REQUIRE(top >= 0 && top <= kMaxTop && top <= C, FG_ERR_OUT_OF_BOUNDS,
               "%s: %d alternatives of %d columns, at most %d", who, top, C, kMaxTop);
    FG_REQUIRE(scale > 0.0f && scale < INFINITY, FG_ERR_INVALID_ARGUMENT,
               "%s: scale must be positive and finite", who);
    FG_REQUIRE(d_logits && d_tokens, FG_ERR_INVALID_ARGUMENT, "%s: logits and tokens are required",
               who);
    FG_REQUIRE((top > 0) == (d_top_ids || d_top_logp), FG_ERR_INVALID_ARGUMENT,
               "%s: %d alternatives, but %s for them", who, top,
               top > 0 ? "no output" : "an output");
    FG_REQUIRE(d_logp || d_entropy || d_lse || top, FG_ERR_INVALID_ARGUMENT, "%s: no output", who);
    FG_REQUIRE(fg::rows::grid_holds(R, 1024), FG_ERR_OUT_OF_BOUNDS, "%s: %d rows of %d columns",
               who, R, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_logp, {d_logits, d_tokens, d_entropy, d_lse, d_top_ids, d_top_logp}) &&
                   apart(d_entropy, {d_logits, d_tokens, d_lse, d_top_ids, d_top_logp}) &&
                   apart(d_lse, {d_logits, d_tokens, d_top_ids, d_top_logp}) &&
                   apart(d_top_ids, {d_logits, d_tokens, d_top_logp}) &&
                   apart(d_top_logp, {d_logits, d_tokens}),
               FG_ERR_INVALID_ARGUMENT, "%s: an output is another output or an input", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    Fwd a{d_logits, d_tokens, d_logp, d_entropy, d_lse, d_top_ids, d_top_logp, scale,
          ldx, C, top, splits_of(ctx->cu_count, R, C), nullptr, nullptr};
    if (a.splits > 1) {
        const uint64_t parts = (uint64_t)R * a.splits;
        a.best = (uint64_t *)fg::workspace(ctx, parts * (top * sizeof(uint64_t) + 4 * sizeof(float)));
        if (!a.best) return FG_ERR_OUT_OF_MEMORY;
        a.stats = (float *)(a.best + parts * top);
    }
    if (dtype == FG_DTYPE_F32) launch_fwd<fg::kF32>(ctx->stream, R, a);
    else if (dtype == FG_DTYPE_BF16) launch_fwd<fg::kBF16>(ctx->stream, R, a);
    else launch_fwd<fg::kF16>(ctx->stream, R, a);
    FG_LAUNCH_CHECK("logprobs_fwd");
    return FG_OK;
}

FG_API int fg_token_logprobs_bwd(fg_ctx *ctx, int dtype, const void *d_logits, int ldx,
                                 const uint32_t *d_tokens, int R, int C, float scale,
                                 const float *d_lse, const float *d_entropy, const float *d_dlogp,
                                 const float *d_dentropy, void *d_dlogits, int ldd) {
    const char *who = "fg_token_logprobs_bwd";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(R >= 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape R=%d C=%d", who, R, C);
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(ldx >= C && ldd >= C, FG_ERR_SHAPE, "%s: ldx=%d or ldd=%d < C=%d", who, ldx, ldd, C);
    FG_REQUIRE(scale > 0.0f && scale < INFINITY, FG_ERR_INVALID_ARGUMENT,
               "%s: scale must be positive and finite", who);
    FG_REQUIRE(d_logits && d_tokens && d_lse && d_dlogits && (d_dlogp || d_dentropy),
               FG_ERR_INVALID_ARGUMENT,
               "%s: logits, tokens, lse, dlogits and a gradient of logp or entropy are required",
               who);
    FG_REQUIRE(!d_dentropy || d_entropy, FG_ERR_INVALID_ARGUMENT,
               "%s: the entropy's gradient needs the entropy", who);
    FG_REQUIRE(d_dlogits != d_logits || ldd == ldx, FG_ERR_INVALID_ARGUMENT,
               "%s: dlogits is logits, but ldd=%d, ldx=%d", who, ldd, ldx);
    FG_REQUIRE(fg::rows::grid_holds(R, kBwdNT), FG_ERR_OUT_OF_BOUNDS, "%s: %d rows of %d columns",
               who, R, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_dlogits, {d_tokens, d_lse, d_entropy, d_dlogp, d_dentropy}),
               FG_ERR_INVALID_ARGUMENT, "%s: dlogits is an input but logits", who);
    if (R == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    const Bwd a{d_logits, d_tokens, d_lse, d_entropy, d_dlogp, d_dentropy, d_dlogits, scale,
                ldx, ldd, R, C, 0};
    if (dtype == FG_DTYPE_F32) launch_bwd<fg::kF32>(ctx->stream, a);
    else if (dtype == FG_DTYPE_BF16) launch_bwd<fg::kBF16>(ctx->stream, a);
    else launch_bwd<fg::kF16>(ctx->stream, a);
    FG_LAUNCH_CHECK("logprobs_bwd");
    return FG_OK;
}
