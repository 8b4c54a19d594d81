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
//
// Both are bound by HBM (the rows they read and write once): the lookup of 16384 rows
// of 4096 in bf16 takes 32.5 us, 5.6 TB/s.  The gradient:
//  * the positions in (token, position) order: one launch of workgroups that own
//    tokens (up to kOrderReads reads in all), a stable radix sort above; table rows are zeroed
//    beside either, which leave the memory idle;
//  * the sorted positions in units of equal length, so that a token that fills half
//    the batch is spread over the GPU as evenly as any other: a unit adds its runs
//    of equal tokens, writes the rows of runs that it holds whole, and leaves the
//    runs that cross its ends as fp32 partial sums; workgroups of the same launch
//    zero the rows of no token that are left;
//  * the crossing runs' partial sums are joined in order.
// 65536 tokens over 131072 rows of 2048 in bf16 (805 MB): sort 32 us, sums 137 at
// 4.7 TB/s, joins 8.  20011 tokens, four in ten of them one, over 50257 rows of 777 in
// fp32 (218 MB): order 25 with 93 MB of zeros, sums 25, joins 7.4.
// Small batches (own_launch) take one launch, whose workgroups own table rows and order
// their positions in LDS; the fewest tokens (kDirectMax) one of smaller workgroups, which
// only list theirs.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fg_half.h"
#include "fg_internal.h"
#include "fg_rows.h"

namespace {

using fg::rows::apart;
using fg::rows::Io;
using fg::rows::Tail;
using fg::rows::u32x4;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
using fg::rows::u32x2;
typedef u32x2 u32x2_any __attribute__((aligned(2)));

constexpr int kNT = 256;
constexpr int kDirectMax = 32;
constexpr int kOwnMax = 4096;
// Tokens that all of emb_order's workgroups read: 40960 a workgroup where there are 256,
// fewer where there are more (tables above 2^18 rows), more where a small table has fewer
// workgroups (3 for 2 rows, 51 for 50, 129 for 256), which may then take longer than the
// radix sort would (all of the gradient, bf16 rows of 256: 131072 tokens over 2 rows 92 us
// and 44, over 50 rows 81 and 38, over 256 rows 39 and 38; 40960 over 2 rows 41 and 34;
// 16384 over 2 rows 29 and 32).
// It takes 8.6 us for 8192 tokens, 15 for 16384, 22 for 32768 (as much again where zeros
// share the CUs); the radix sort's launches 24 or more for any of these.  All of the
// gradient, bf16, 32000 rows of 1024: 8192 tokens 25.7 us (radix sort 36.7), 16384 34.2
// (45.0), 32768 47.9 (54.6); 40900 tokens over 131072 rows 73.7 (75.9).
constexpr int64_t kOrderReads = 10 << 20;
// Workgroups of units (with 512 and 2048: 65536 tokens, 131072 rows of 2048 in bf16 177.5
// and 180.4 us, 177.1 with 1024; 20011 tokens, rows of 777 in fp32 67.4 and 60.6, 58.0).
constexpr int kUnitBlocks = 1024;
constexpr int kMaxTokens = 1 << 30;  // (positions a little past the last are 32-bit too)

// A kernel's arguments are one or two structs: with a dozen arguments the runtime takes
// up to 0.9 us more for a launch (layer norm backward of 64 rows, a call 5.4 us and 4.9).

// ------------------------------------------------------------------- lookup
template <class T>
struct Lookup {
    const uint32_t *tokens;
    const T *table;
    T *out;
    int count, V, C, ldt, ldo, lshift;
    float scale;
};
// 2^lshift lanes take a row, UNR chunks in flight a lane.
template <int DT>
__global__ __launch_bounds__(kNT) void emb_fwd(const Lookup<typename Io<DT>::T> a) {
    const uint32_t *__restrict__ tokens = a.tokens;
    const auto *__restrict__ table = a.table;
    auto *out = a.out;
    const int T = a.count, V = a.V, C = a.C, ldt = a.ldt, ldo = a.ldo, lshift = a.lshift;
    const float scale = a.scale;
    using IO = Io<DT>;
    constexpr int E = IO::E, UNR = 4;
    const int lanes = 1 << lshift, lane = threadIdx.x & (lanes - 1);
    const int64_t t = ((int64_t)blockIdx.x << (8 - lshift)) + (threadIdx.x >> lshift);
    if (t >= T) return;
    const uint32_t v = tokens[t];
    const bool in = v < (uint32_t)V;
    const auto *row = table + (size_t)(in ? v : 0) * ldt;
    auto *to = out + (size_t)t * ldo;
    const float k = in ? scale : __builtin_nanf("");
    const int nb = C / E, chunks = (C - 1) / E + 1;
    // (The product is rounded to fp32 and then to the type, here and in the oracle: kept
    // apart, or the compiler makes one rounding of both in one of the loops, and lanes
    // that share a column could differ.)
    auto out_of = [&](u32x4 w, float (&o)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            o[e] = in ? k * IO::get(w, e) : k;
            asm("" : "+v"(o[e]));
        }
    };
    int j = lane;
    float o[E];
    for (; j + (UNR - 1) * lanes < nb; j += UNR * lanes) {
        u32x4 w[UNR];
#pragma unroll
        for (int u = 0; u < UNR; ++u) w[u] = fg::rows::load<DT>(row, j + u * lanes);
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            out_of(w[u], o);
            fg::rows::store<DT>(to, j + u * lanes, IO::pack(o));
        }
    }
    for (; j < chunks; j += lanes) {
        const Tail<DT> tail(j, C);
        out_of(tail.load(row), o);
        tail.store(to, o);
    }
}

// --------------------------------------------------- few tokens: one launch
// (Zeros of 65 MB beside 64 tokens 13.9 us, as emb_bwd_own 16.8; but 64 tokens of 10 rows
// of 256 10.2 and 6.3, and 256 of which four in ten are one 33.7 and 16.3: a row's lanes
// walk the list from its first token to its last.)
// A workgroup owns `rows` table rows from blockIdx.x * rows on: it lists the
// positions of their tokens in order, then each group of 2^lshift lanes adds the
// rows of its own tokens.
template <class T>
struct Few {
    const uint32_t *tokens;
    const T *dout;
    T *dtable;
    int count, V, C, lddo, lddt, accumulate, rows, lshift;
    float scale;
};
template <int DT>
__global__ __launch_bounds__(kNT) void emb_bwd_few(const Few<typename Io<DT>::T> p) {
    const uint32_t *__restrict__ tokens = p.tokens;
    const auto *__restrict__ dout = p.dout;
    auto *dtable = p.dtable;
    const int T = p.count, V = p.V, C = p.C, lddo = p.lddo, lddt = p.lddt;
    const int accumulate = p.accumulate, rows = p.rows, lshift = p.lshift;
    const float scale = p.scale;
    using IO = Io<DT>;
    constexpr int E = IO::E;
    static_assert(kDirectMax <= kNT, "one token a thread");
    __shared__ uint32_t tok[kDirectMax + 8], at[kDirectMax + 8];  // (+ 8: read ahead)
    __shared__ int count[kNT / 64];
    const int lanes = 1 << lshift, lane = threadIdx.x & (lanes - 1);
    const int64_t v0 = (int64_t)blockIdx.x * rows;
    const int nrows = (int)min((int64_t)rows, V - v0);
    const uint32_t mine = threadIdx.x < (unsigned)T ? tokens[threadIdx.x] : 0xffffffffu;
    const bool hit = threadIdx.x < (unsigned)T && mine >= v0 && mine < v0 + nrows;
    const uint64_t mask = __ballot(hit);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) count[wave] = __popcll(mask);
    __syncthreads();
    int base = 0, n = 0;
#pragma unroll
    for (int w = 0; w < kNT / 64; ++w) {
        base += w < wave ? count[w] : 0;
        n += count[w];
    }
    if (hit) {
        const int k = base + __popcll(mask & ((1ull << (threadIdx.x & 63)) - 1));
        tok[k] = mine;
        at[k] = threadIdx.x;
    }
    __syncthreads();
    const int chunks = (C - 1) / E + 1;
    for (int r = threadIdx.x >> lshift; r < nrows; r += kNT >> lshift) {
        const uint32_t v = (uint32_t)(v0 + r);
        auto *to = dtable + (size_t)v * lddt;
        int first = n, last = -1;
        for (int k = 0; k < n; ++k)
            if (tok[k] == v) {
                first = min(first, k);
                last = k;
            }
        if (last < 0 && accumulate) continue;
        for (int j = lane; j < chunks; j += lanes) {
            const Tail<DT> at_j(j, C);
            float a[E];
#pragma unroll
            for (int e = 0; e < E; ++e) a[e] = 0.0f;
            for (int k = first; k <= last; k += 8) {
                u32x4 w[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const bool own = k + u <= last && tok[k + u] == v;
                    w[u] = u32x4{0u, 0u, 0u, 0u};
                    if (own) w[u] = at_j.load(dout + (size_t)at[k + u] * lddo);
                }
#pragma unroll
                for (int u = 0; u < 8; ++u)
#pragma unroll
                    for (int e = 0; e < E; ++e) a[e] += IO::get(w[u], e);
            }
            // (A row of no token is +0 whatever the scale.)
#pragma unroll
            for (int e = 0; e < E; ++e) a[e] = last < 0 ? 0.0f : a[e] * scale;
            if (accumulate) at_j.add(to, j, a);
            else at_j.store(to, a);
        }
    }
}

// -------------------------------------------------------------------- zeros
// Table rows that a launch zeroes beside its own work (whether tokens have them or
// not; what tokens do have is written by later launches).
struct Zero {
    char *base;
    uint64_t stride;           // bytes between rows
    int64_t row_bytes;         // even
    int first, count, lshift;  // rows; log2 of a row's lanes
};
__device__ __forceinline__ void zero_rows(const Zero &z, int block, int blocks) {
    const int lanes = 1 << z.lshift, lane = threadIdx.x & (lanes - 1);
    const int groups = blockDim.x >> z.lshift;
    const int64_t end = z.row_bytes & ~int64_t(15);
    for (int64_t r = (int64_t)block * groups + (threadIdx.x >> z.lshift); r < z.count;
         r += (int64_t)blocks * groups) {
        char *to = z.base + (uint64_t)(z.first + r) * z.stride;
        for (int64_t at = lane * 16; at < end; at += lanes * 16)
            __builtin_nontemporal_store(u32x4{0u, 0u, 0u, 0u},
                                        reinterpret_cast<fg::rows::u32x4_any *>(to + at));
        for (int64_t at = end + lane * 2; at < z.row_bytes; at += lanes * 2)
            *reinterpret_cast<uint16_t *>(to + at) = 0;
    }
}

// ------------------------------------------------------------------- sorting
// The positions of a workgroup's own tokens, `n` of them from v0 on, in (token, position)
// order.  Its waves take a run of the batch each and count the tokens below the
// workgroup's (where BELOW) and each of its own; the counts' prefix sums, by token and
// then by wave, are where a second reading places its positions: start(token, where,
// count) by a thread for each token, then place(where, position, key).  64 positions
// that hold none of its tokens, as most do, cost two comparisons.  Tokens outside the
// table count as V.  A wave's run of up to 512 (without BELOW, all of up to kOwnMax
// tokens) stays in registers between the readings.  idle() runs after the first, its
// memory accesses beside what follows.
constexpr int kOrderNT = 1024, kOrderWaves = kOrderNT / 64;
constexpr int kOrderBlocks = 256, kOrderBins = 1024;  // workgroups at least; tokens at most
struct OrderLds {
    uint32_t wbelow[kOrderWaves], wsum[kOrderWaves];
};
template <bool BELOW, class I, class S, class P>
__device__ __forceinline__ void order_own(const uint32_t *__restrict__ tokens, int T, uint32_t V,
                                          uint32_t v0, uint32_t n, int bins, OrderLds &lds,
                                          uint32_t *cnt,  // [wave][bins]
                                          I idle, S start, P place) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (An odd number of 64s: the waves' runs then begin in different memory channels.)
    const int per = (((T - 1) / kOrderNT + 1) | 1) * 64, i0 = wave * per, i1 = min(T, i0 + per);
    // Loads of a lane in flight; of a small batch, all.
    constexpr int kBatch = BELOW ? 8 : ((kOwnMax - 1) / kOrderNT + 1) | 1;
    uint32_t *mine = cnt + wave * bins;
    // f(its bin, its lanes) for each of the workgroup's tokens of 64 positions, in some
    // order.
    auto each = [&](uint32_t d, auto f) {
        uint64_t hits = __ballot(d < n);
        while (hits) {
            const uint32_t at =
                (uint32_t)__builtin_amdgcn_readlane((int)d, __ffsll((long long)hits) - 1);
            const uint64_t m = __ballot(d == at);
            f(at, m);
            hits &= ~m;
        }
    };
    uint32_t next[kBatch];
    auto load = [&](int i) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) next[u] = tokens[min(i + 64 * u + lane, T - 1)];
    };
    load(i0);
    auto scan = [&](auto f) {  // (next: the run's first)
        int i = i0;
        for (; BELOW && i + 64 * kBatch <= i1; i += 64 * kBatch) {
            uint32_t key[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) key[u] = min(next[u], V);
            load(i + 64 * kBatch);
#pragma unroll
            for (int u = 0; u < kBatch; ++u) f(key[u], i + 64 * u + lane);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int at = i + 64 * u + lane;
            if (i + 64 * u < i1) f(at < i1 ? min(next[u], V) : 0xffffffffu, at);
        }
    };
    for (int d = threadIdx.x; d < kOrderWaves * bins; d += kOrderNT) cnt[d] = 0;
    __syncthreads();
    uint32_t below = 0;
    scan([&](uint32_t key, int) {
        if constexpr (BELOW) below += (uint32_t)__popcll(__ballot(key < v0));
        each(key - v0, [&](uint32_t own, uint64_t m) {
            if (key - v0 == own && !(m & ((1ull << lane) - 1)))  // (one lane)
                atomicAdd(&mine[own], (uint32_t)__popcll(m));
        });
    });
    if (lane == 0) lds.wbelow[wave] = below;
    idle();
    __syncthreads();
    // A thread a bin.
    uint32_t total = 0;
    const uint32_t bin = threadIdx.x;
    if (bin < n)
        for (int w = 0; w < kOrderWaves; ++w) total += cnt[w * bins + bin];
    uint32_t incl = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 63) lds.wsum[wave] = incl;
    __syncthreads();
    uint32_t at = incl - total, all = 0;
    for (int w = 0; w < kOrderWaves; ++w) {
        at += lds.wbelow[w] + (w < wave ? lds.wsum[w] : 0u);
        all += lds.wsum[w];
    }
    if (bin < n) start(bin, at, total);
    if (all == 0) return;
    if (bin < n)
        for (int w = 0; w < kOrderWaves; ++w) {
            const uint32_t c = cnt[w * bins + bin];
            cnt[w * bins + bin] = at;
            at += c;
        }
    if (BELOW && per >= 64 * kBatch) load(i0);
    __syncthreads();
    scan([&](uint32_t key, int i) {
        const uint32_t d = key - v0;
        each(d, [&](uint32_t own, uint64_t m) {
            uint32_t to = 0;
            if (lane == 0) to = atomicAdd(&mine[own], (uint32_t)__popcll(m));
            to = (uint32_t)__builtin_amdgcn_readfirstlane((int)to);
            if (d == own) place(to + (uint32_t)__popcll(m & ((1ull << lane) - 1)), i, key);
        });
    });
}

// order[k] = the k-th position in (token, position) order, sorted[k] its token.
struct Order {
    const uint32_t *tokens;
    uint32_t *order, *sorted;
    int count, bins, blocks;
    uint32_t V;
};
__global__ __launch_bounds__(kOrderNT) void emb_order(const Order p, const Zero z) {
    __shared__ OrderLds lds;
    extern __shared__ uint32_t cnt[];
    if ((int)blockIdx.x >= p.blocks) {
        zero_rows(z, blockIdx.x - p.blocks, gridDim.x - p.blocks);
        return;
    }
    const uint32_t v0 = blockIdx.x * (uint32_t)p.bins, n = min((uint32_t)p.bins, p.V + 1 - v0);
    uint32_t *__restrict__ order = p.order, *__restrict__ sorted = p.sorted;
    order_own<true>(p.tokens, p.count, p.V, v0, n, p.bins, lds, cnt,
                    [] {}, [](uint32_t, uint32_t, uint32_t) {},
                    [&](uint32_t to, int i, uint32_t key) {
                        order[to] = (uint32_t)i;
                        sorted[to] = key;
                    });
}

// All of a small batch's gradient in one launch: a workgroup zeroes its own table rows
// beside the ordering of their positions in LDS (whose tokens are in registers by then:
// loads wait for the stores before them), then 2^lshift lanes take a row
// with tokens each, or all of them a share of a row of many tokens (kOwnMany), whose
// sums are added in order.
// (kOwnBlocks: fp32 448 tokens over 2568 rows of 42 8.8 us with 512, 6.2 with 256.)
constexpr int kOwnMany = 32, kOwnBlocks = 256;
template <int DT>
__global__ __launch_bounds__(kOrderNT) void emb_bwd_own(const Few<typename Io<DT>::T> p) {
    using IO = Io<DT>;
    constexpr int E = IO::E;
    __shared__ OrderLds lds;
    __shared__ uint32_t many[kOwnMax / kOwnMany], nfew, nmany;
    extern __shared__ uint32_t cnt[];
    uint32_t *first = cnt + kOrderWaves * p.rows, *few = first + p.rows + 1;
    uint32_t *list = few + p.rows;  // (few, many: rows, in any order)
    __shared__ f32x4 part[E / 4][kOrderNT];
    const auto *__restrict__ dout = p.dout;
    const uint32_t v0 = blockIdx.x * (uint32_t)p.rows, n = min((uint32_t)p.rows, p.V - v0);
    const int chunks = (p.C - 1) / E + 1, lanes = 1 << p.lshift, groups = kOrderNT >> p.lshift;
    const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> p.lshift;
    const int j = blockIdx.y * lanes + lane;
    const Tail<DT> at_j(min(j, chunks - 1), p.C);
    if (threadIdx.x == 0) nfew = nmany = 0;
    float a[E] = {};
    auto zero = [&] {
        if (!p.accumulate && j < chunks)
            for (uint32_t r = group; r < n; r += groups)
                at_j.store(p.dtable + (size_t)(v0 + r) * p.lddt, a);
    };
    order_own<false>(p.tokens, p.count, (uint32_t)p.V, v0, n, p.rows, lds, cnt, zero,
                     [&](uint32_t bin, uint32_t at, uint32_t count) {
                         first[bin] = at;
                         if (bin + 1 == n) first[n] = at + count;
                         if (count > kOwnMany) many[atomicAdd(&nmany, 1u)] = bin;
                         else if (count) few[atomicAdd(&nfew, 1u)] = bin;
                     },
                     [&](uint32_t to, int i, uint32_t) { list[to] = (uint32_t)i; });
    // (The zeros of a row are written before its sum, by whichever wave.)
    __threadfence_block();
    __syncthreads();
    // list[k0, k1) in order.
    auto sum = [&](uint32_t k0, uint32_t k1) {
#pragma unroll
        for (int e = 0; e < E; ++e) a[e] = 0.0f;
        for (uint32_t k = k0; k < k1; k += 8) {
            u32x4 w[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                w[u] = u32x4{0u, 0u, 0u, 0u};
                if (k + u < k1) w[u] = at_j.load(dout + (size_t)list[k + u] * p.lddo);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) a[e] += IO::get(w[u], e);
        }
    };
    auto put = [&](uint32_t bin) {
        auto *to = p.dtable + (size_t)(v0 + bin) * p.lddt;
#pragma unroll
        for (int e = 0; e < E; ++e) a[e] *= p.scale;
        if (p.accumulate) at_j.add(to, j, a);
        else at_j.store(to, a);
    };
    if (j < chunks)
        for (uint32_t h = group; h < nfew; h += groups) {
            const uint32_t bin = few[h];
            sum(first[bin], first[bin + 1]);
            put(bin);
        }
    for (uint32_t h = 0; h < nmany; ++h) {
        const uint32_t bin = many[h], k0 = first[bin], k1 = first[bin + 1];
        const uint32_t per = max(8u, (k1 - k0 - 1) / groups + 1), k = k0 + group * per;
        sum(min(k, k1), min(k + per, k1));
#pragma unroll
        for (int q = 0; q < E / 4; ++q)
            part[q][threadIdx.x] = f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
        __syncthreads();
        if (group == 0 && j < chunks) {
            const int used = (int)((k1 - k0 - 1) / per + 1);
#pragma unroll 4
            for (int g = 1; g < used; ++g)
#pragma unroll
                for (int e = 0; e < E; ++e) a[e] += part[e / 4][(g << p.lshift) + lane][e % 4];
            put(bin);
        }
        __syncthreads();
    }
}

// Stable radix sort, least significant digit first, of (token, position) pairs:
// tile b of the input counts its digits (radix_count: hist[tile][digit]), then
// places its pairs behind those of smaller digits and of earlier tiles
// (radix_place).  Tokens outside the table sort as V.
constexpr int kMaxBits = 11, kBins = 1 << kMaxBits;
constexpr int kTiles = 64;  // at most
constexpr int kSortNT = 1024;
struct Radix {
    const uint32_t *keys, *pos;
    uint32_t *hist, *keys_out, *pos_out;
    int count, per, shift, bits, tiles;
    uint32_t V;
};

__device__ __forceinline__ uint32_t key_of(uint32_t token, uint32_t V) { return min(token, V); }

__global__ __launch_bounds__(kSortNT) void radix_count(const Radix p, const Zero z) {
    const uint32_t *__restrict__ keys = p.keys;
    uint32_t *__restrict__ hist = p.hist;
    const int T = p.count, per = p.per, shift = p.shift, bits = p.bits, tiles = p.tiles;
    const uint32_t V = p.V;
    __shared__ uint32_t h[kBins];
    if ((int)blockIdx.x >= tiles) {
        zero_rows(z, blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += kSortNT) h[d] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * per, i1 = min((int64_t)T, i0 + per);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kSortNT)
        atomicAdd(&h[(key_of(keys[i], V) >> shift) & (bins - 1)], 1u);  // (counts: any order)
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortNT)
        hist[((size_t)blockIdx.x << bits) + d] = h[d];
}

// pos NULL: the pairs' positions are their own indices (the first pass).
__global__ __launch_bounds__(kSortNT) void radix_place(const Radix p, const Zero z) {
    const uint32_t *__restrict__ keys = p.keys, *__restrict__ pos = p.pos;
    const uint32_t *__restrict__ hist = p.hist;
    uint32_t *__restrict__ keys_out = p.keys_out, *__restrict__ pos_out = p.pos_out;
    const int T = p.count, per = p.per, shift = p.shift, bits = p.bits, tiles = p.tiles;
    const uint32_t V = p.V;
    if ((int)blockIdx.x >= tiles) {
        zero_rows(z, blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    constexpr int kWaves = kSortNT / 64;
    // Pairs of digit d in the tile's wave w; then where they go.
    __shared__ uint32_t cnt[kWaves][kBins];
    __shared__ uint32_t base[kBins];
    __shared__ uint32_t wsum[kWaves];
    const int bins = 1 << bits;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // Each wave takes a run of the tile, 64 pairs at a time; the first kHeld rounds'
    // pairs are loaded here and stay in registers.
    constexpr int kHeld = 4;
    const int64_t t0 = (int64_t)blockIdx.x * per, t1 = min((int64_t)T, t0 + per);
    const int run = (per + kWaves - 1) / kWaves;
    const int64_t i0 = t0 + (int64_t)wave * run, i1 = min(t1, i0 + run);
    auto key_at = [&](int64_t i) { return i + lane < i1 ? key_of(keys[i + lane], V) : 0u; };
    auto pos_at = [&](int64_t i) {
        return pos && i + lane < i1 ? pos[i + lane] : (uint32_t)(i + lane);
    };
    uint32_t hkey[kHeld], hpos[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        hkey[u] = key_at(i0 + 64 * u);
        hpos[u] = pos_at(i0 + 64 * u);
    }
    // base[d] = pairs of digit d in earlier tiles, and of smaller digits: thread
    // (g, d) adds the digit's counts of every G-th tile, the threads of a digit are
    // added in LDS (in cnt, which is cleared after), then a scan over the digits.
    constexpr int kOwn = kBins / kSortNT;  // digits of a thread in the scan
    const int G = max(1, kSortNT >> bits);
    for (int d0 = threadIdx.x; d0 < max(bins, kSortNT); d0 += kSortNT) {
        const int d = d0 & (bins - 1), g = d0 >> bits;
        uint32_t before = 0, all = 0;
        if (g < G) {
#pragma unroll 16
            for (int b = g; b < tiles; b += G) {
                const uint32_t c = hist[((size_t)b << bits) + d];
                all += c;
                before += b < (int)blockIdx.x ? c : 0u;
            }
            cnt[0][d0] = all;  // (G * bins <= 2 kSortNT = kBins values each)
            cnt[1][d0] = before;
        }
    }
    __syncthreads();
    uint32_t total[kOwn], mine = 0;
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
        const int d = threadIdx.x * kOwn + u;
        uint32_t before = 0, all = 0;
        if (d < bins) {
            for (int g = 0; g < G; ++g) {
                all += cnt[0][(g << bits) + d];
                before += cnt[1][(g << bits) + d];
            }
            base[d] = before;
        }
        total[u] = all;
        mine += all;
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    uint32_t excl = incl - mine;
    for (int w = 0; w < wave; ++w) excl += wsum[w];
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
        const int d = threadIdx.x * kOwn + u;
        if (d < bins) base[d] += excl;
        excl += total[u];
    }
    __syncthreads();
    for (int k = threadIdx.x; k < kWaves * bins; k += kSortNT) cnt[k >> bits][k & (bins - 1)] = 0;
    __syncthreads();
    // Lanes of a round with the lane's digit.
    auto same = [&](uint32_t d, bool in) {
        uint64_t m = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const uint64_t s = __ballot((d >> b) & 1u);
            m &= (d >> b) & 1u ? s : ~s;
        }
        return m;
    };
    auto count = [&](int64_t i, uint32_t key) {
        const bool in = i + lane < i1;
        const uint32_t d = (key >> shift) & (bins - 1);
        const uint64_t m = same(d, in);
        // (A wave's LDS accesses run in order: a round reads what the last one wrote.)
        if (in && lane == __ffsll((long long)m) - 1) cnt[wave][d] += (uint32_t)__popcll(m);
        __builtin_amdgcn_wave_barrier();
    };
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
        if (i0 + 64 * u < i1) count(i0 + 64 * u, hkey[u]);
    for (int64_t i = i0 + 64 * kHeld; i < i1; i += 64) count(i, key_at(i));
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortNT) {
        uint32_t at = base[d];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const uint32_t c = cnt[w][d];
            cnt[w][d] = at;
            at += c;
        }
    }
    __syncthreads();
    auto place = [&](int64_t i, uint32_t key, uint32_t p) {
        const bool in = i + lane < i1;
        const uint32_t d = (key >> shift) & (bins - 1);
        const uint64_t m = same(d, in);
        uint32_t to = 0;
        if (in) to = cnt[wave][d] + (uint32_t)__popcll(m & ((1ull << lane) - 1));
        __builtin_amdgcn_wave_barrier();
        if (in && lane == __ffsll((long long)m) - 1) cnt[wave][d] += (uint32_t)__popcll(m);
        __builtin_amdgcn_wave_barrier();
        if (in) {
            keys_out[to] = key;
            pos_out[to] = p;
        }
    };
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
        if (i0 + 64 * u < i1) place(i0 + 64 * u, hkey[u], hpos[u]);
    for (int64_t i = i0 + 64 * kHeld; i < i1; i += 64) place(i, key_at(i), pos_at(i));
}

// ---------------------------------------------------------------------- sums
// First of sorted[lo, hi) that is not below v.
__device__ __forceinline__ int lower_bound(const uint32_t *sorted, int lo, int hi, uint32_t v) {
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (sorted[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}
// The same by a whole wave, 64 probes at a time (all lanes; the same in each).
__device__ __forceinline__ int wave_lower_bound(const uint32_t *sorted, int T, uint32_t v) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, hi = T;  // the answer is in [lo, hi]
    while (lo < hi) {
        const int64_t step = (hi - lo + 63) / 64, at = lo + lane * step;
        const uint64_t below = __ballot(at < hi && sorted[at < hi ? at : lo] < v);
        const int n = __popcll(below);  // probes below v: the first n
        if (n == 0) return (int)lo;
        const int64_t last = lo + (int64_t)(n - 1) * step;  // is below
        hi = min(hi, last + step);
        lo = last + 1;
    }
    return (int)lo;
}

struct Sums {
    const uint32_t *order, *sorted;
    int T, V, C, lddo, lddt, accumulate;
    float scale;
    int P;            // sorted positions of a unit
    int units;        // units in all
    int lshift;       // log2 of a unit's lanes
    int unit_blocks;  // workgroups of units; those after them zero `zrows` rows each,
    int zrows;        // from zfirst on
    int zfirst;
    int64_t Cp;       // columns of a partial sum (rounded up to chunks)
    float *partial;   // [units][2][Cp]: the run that began before, the one that goes on
};

// WAVE: a unit's lanes fill whole waves, so that positions, tokens and rows' addresses
// are scalar.
template <int DT, bool WAVE>
__global__ __launch_bounds__(kNT) void emb_sums(const Sums p,
                                                const typename Io<DT>::T *__restrict__ dout,
                                                typename Io<DT>::T *dtable) {
    using IO = Io<DT>;
    constexpr int E = IO::E, UNR = 8;
    const int chunks = (p.C - 1) / E + 1;
    if ((int)blockIdx.x >= p.unit_blocks) {
        // Rows of no token.
        if (blockIdx.y > 0) return;
        __shared__ int used[kNT];
        __shared__ int range[2];
        const int64_t v0 = p.zfirst + (int64_t)(blockIdx.x - p.unit_blocks) * p.zrows;
        const int n = (int)min((int64_t)p.zrows, p.V - v0), wave = threadIdx.x >> 6;
        if (wave < 2) {
            const int at = wave_lower_bound(p.sorted, p.T, (uint32_t)(v0 + (wave ? n : 0)));
            if ((threadIdx.x & 63) == 0) range[wave] = at;
        }
        __syncthreads();
        // The rows' tokens are sorted[lo, hi): marked from there where a thread takes
        // one each, else (a frequent token is among them) searched for.
        const int lo = range[0], hi = range[1];
        if (hi - lo <= kNT) {
            used[threadIdx.x] = 0;
            __syncthreads();
            if (lo + (int)threadIdx.x < hi) used[p.sorted[lo + threadIdx.x] - (uint32_t)v0] = 1;
        } else if ((int)threadIdx.x < n) {
            const uint32_t v = (uint32_t)(v0 + threadIdx.x);
            const int k = lower_bound(p.sorted, lo, hi, v);
            used[threadIdx.x] = k < hi && p.sorted[k] == v;
        }
        __syncthreads();
        const float z[E] = {};
        const int lanes = 1 << p.lshift;
        for (int r = threadIdx.x >> p.lshift; r < n; r += kNT >> p.lshift) {
            if (used[r]) continue;
            auto *to = dtable + (size_t)(v0 + r) * p.lddt;
            for (int j = threadIdx.x & (lanes - 1); j < chunks; j += lanes)
                Tail<DT>(j, p.C).store(to, z);
        }
        return;
    }
    const int lanes = 1 << p.lshift;
    int unit = (int)(blockIdx.x << (8 - p.lshift)) + (int)(threadIdx.x >> p.lshift);
    if constexpr (WAVE) unit = __builtin_amdgcn_readfirstlane(unit);
    const int j = blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
    if (unit >= p.units || j >= chunks) return;
    const Tail<DT> at_j(j, p.C);
    const int k0 = unit * p.P, k1 = min(p.T, k0 + p.P);
    const uint32_t V = (uint32_t)p.V;
    const uint32_t *__restrict__ sorted = p.sorted, *__restrict__ order = p.order;
    // A run that began before the unit, or goes on after it, is a partial sum.
    bool head = k0 > 0 && sorted[k0 - 1] == sorted[k0];
    float a[E];
#pragma unroll
    for (int e = 0; e < E; ++e) a[e] = 0.0f;
    // Positions and tokens of the next UNR rows are loaded before this batch's rows
    // are added.
    uint32_t pos[UNR], tok[UNR + 1];
    auto index = [&](int k) {
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            pos[u] = order[min(k + u, k1 - 1)];
            tok[u] = sorted[min(k + u, p.T - 1)];
        }
        tok[UNR] = sorted[min(k + UNR, p.T - 1)];
    };
    index(k0);
    for (int k = k0; k < k1; k += UNR) {
        u32x4 w[UNR];
        uint32_t t[UNR + 1];
#pragma unroll
        for (int u = 0; u < UNR; ++u)
            w[u] = at_j.load(dout + (size_t)pos[u] * p.lddo);
#pragma unroll
        for (int u = 0; u <= UNR; ++u) t[u] = tok[u];
        if (k + UNR < k1) index(k + UNR);
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            if (k + u >= k1) break;
#pragma unroll
            for (int e = 0; e < E; ++e) a[e] += IO::get(w[u], e);
            const bool same = k + u + 1 < p.T && t[u + 1] == t[u];
            if (same && k + u + 1 < k1) continue;
            if (t[u] < V) {
                if (head || same) {  // (same: the run goes on in the next unit)
                    float *to = p.partial + ((size_t)unit * 2 + (head ? 0 : 1)) * p.Cp +
                                at_j.first;
#pragma unroll
                    for (int q = 0; q < E / 4; ++q)
                        *reinterpret_cast<f32x4_any *>(to + 4 * q) =
                            f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
                } else {
                    auto *to = dtable + (size_t)t[u] * p.lddt;
#pragma unroll
                    for (int e = 0; e < E; ++e) a[e] *= p.scale;
                    if (p.accumulate) at_j.add(to, j, a);
                    else at_j.store(to, a);
                }
            }
            head = false;
#pragma unroll
            for (int e = 0; e < E; ++e) a[e] = 0.0f;
        }
    }
}

// Joins the partial sums of a run that crosses units, 4 columns a lane.  Of a run of n
// units, the first S take a share of the columns each (S = 1 up to 16 units, so that a
// lane has one batch of loads), and in them S groups of lanes a share of the units each,
// added in order.  blockIdx.x: a unit but the last, blockIdx.y: 1024 columns.
constexpr int kJoinNT = 256, kJoinShare = 16;
template <int DT>
__global__ __launch_bounds__(kJoinNT) void emb_join(const Sums p, typename Io<DT>::T *dtable) {
    using IO = Io<DT>;
    __shared__ f32x4 sh[kJoinNT];
    const int u = blockIdx.x, lane = threadIdx.x & 63;
    const int64_t after = (int64_t)(u + 1 + lane) * p.P, before = (int64_t)(u - lane) * p.P - 1;
    const uint32_t v = p.sorted[(u + 1) * p.P - 1];
    // Units after u, and before it, that hold v as well: u's row of them, up to 64.
    auto ones = [](uint64_t m) { return m == ~0ull ? 64 : __ffsll((long long)~m) - 1; };
    const uint64_t on = __ballot(p.sorted[after < p.T ? after : 0] == v && after < p.T);
    const uint64_t back = __ballot(p.sorted[before > 0 ? before : 0] == v && before >= 0);
    int c = ones(on);
    const int b = ones(back);
    if (c == 0 || v >= (uint32_t)p.V || b == 64) return;
    if (c == 64) c = (wave_lower_bound(p.sorted, p.T, v + 1) - 1) / p.P - u;
    const int u0 = u - b, n = b + 1 + c;
    int sshift = 0;
    while (sshift < 6 && (kJoinShare << sshift) < n) ++sshift;
    if (b >> sshift) return;
    const int lshift = 8 - sshift, split = threadIdx.x >> lshift;
    const int per = (n + (1 << sshift) - 1) >> sshift;
    const int64_t col = ((int64_t)blockIdx.y * kJoinNT + (b << lshift) +
                         (threadIdx.x & ((1 << lshift) - 1))) * 4;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    if (col < p.Cp) {
        int k = split * per;
        const int end = min(n, k + per);
        const float *at = p.partial + (size_t)u0 * 2 * p.Cp + col;
        if (k == 0) {
            a = *reinterpret_cast<const f32x4 *>(at + p.Cp);
            ++k;
        }
#pragma unroll 16
        for (; k < end; ++k) a += *reinterpret_cast<const f32x4 *>(at + (size_t)k * 2 * p.Cp);
    }
    if (sshift) {
        sh[threadIdx.x] = a;
        __syncthreads();
        if (split != 0) return;
        const int used = (n - 1) / per + 1;
        for (int w = 1; w < used; ++w) a += sh[threadIdx.x + (w << lshift)];
    }
    if (col >= p.Cp) return;
    // The 4 columns in one access, or the row's last ones one by one.
    auto *to = dtable + (size_t)v * p.lddt + col;
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = a[e] * p.scale;
    const bool whole = col + 4 <= p.C;
    if (!whole) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.C) IO::store1(to, e, p.accumulate ? o[e] + IO::load1(to, e) : o[e]);
        return;
    }
    if constexpr (DT == fg::kF32) {
        auto *row = reinterpret_cast<f32x4_any *>(to);
        f32x4 r = {o[0], o[1], o[2], o[3]};
        if (p.accumulate) r += *row;
        *row = r;
    } else {
        auto *row = reinterpret_cast<u32x2_any *>(to);
        u32x4 w = {0u, 0u, 0u, 0u};
        if (p.accumulate) {
            const u32x2 was = *row;
            w[0] = was[0];
            w[1] = was[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += IO::get(w, e);
        }
        const float eight[8] = {o[0], o[1], o[2], o[3]};
        w = IO::pack(eight);
        *row = u32x2{w[0], w[1]};
    }
}

int log2_up(int64_t n) {
    int s = 0;
    while ((int64_t(1) << s) < n) ++s;
    return s;
}
// Lanes that take a row of `chunks` chunks: a power of two, at most a workgroup.
int lane_shift(int chunks) { return std::min(8, log2_up(chunks)); }

// Whether emb_bwd_own takes the batch: one workgroup reads all of a token's rows, 1 KB of
// each, so at most 1 MB; and at most 1024 workgroups order the batch each.  bf16, four
// tokens in ten one, 32000 rows of 1024: 1024 tokens 20.2 us (three launches 23.5), 2048
// 25.6 (25.0), 4096 37.2 (24.0); fp32 448 tokens, 2568 rows of 42 5.8 (12.7); 512 tokens,
// 2000000 rows of 16 37.8 (33.4).
bool own_launch(int dtype, int T, int V, int C) {
    const int64_t row = (int64_t)C * (dtype == FG_DTYPE_F32 ? 4 : 2);
    return T <= kOwnMax && V <= 1024 * kOrderBins && T * std::min<int64_t>(row, 1024) <= 1 << 20;
}

// How a gradient of T tokens over rows of C columns is laid out.
struct Plan {
    int P, units, lshift;
    int64_t Cp;
    int bins, blocks;              // of emb_order
    int passes, bits, tiles, per;  // of the radix sort (passes 0: emb_order)
    uint64_t sort_words, hist_words, partial_floats;
    uint64_t bytes() const {
        return 4 * (sort_words + hist_words) + 16 + 4 * partial_floats;
    }
};
Plan plan_of(int dtype, int T, int V, int C) {
    Plan p{};
    if (T <= kDirectMax || own_launch(dtype, T, V, C)) return p;
    const int E = dtype == FG_DTYPE_F32 ? 4 : 8, chunks = (C - 1) / E + 1;
    p.lshift = lane_shift(chunks);
    p.Cp = (int64_t)chunks * E;
    // About 1024 workgroups of units of 8 to 512 positions, and at most 4096 units (the
    // longest run joins as many).
    const int64_t tiles = (chunks - 1) / (1 << p.lshift) + 1;
    const int64_t lanes = ((int64_t)T << p.lshift) * tiles;  // with one position a unit
    p.P = 8;
    while (p.P < 512 && (lanes / p.P > kUnitBlocks * kNT || T / p.P > 4096)) p.P *= 2;
    p.units = (T - 1) / p.P + 1;
    p.partial_floats = (uint64_t)p.units * 2 * (uint64_t)p.Cp;
    p.sort_words = 2 * (uint64_t)T;
    p.bins = std::min(kOrderBins, V / kOrderBlocks + 1);  // (of keys 0 .. V)
    p.blocks = V / p.bins + 1;
    if ((int64_t)p.blocks * T > kOrderReads) {
        const int need = std::max(1, log2_up((int64_t)V + 1));  // of keys 0 .. V
        p.passes = (need - 1) / kMaxBits + 1;
        p.bits = (need - 1) / p.passes + 1;
        p.tiles = std::min(kTiles, (T - 1) / kSortNT + 1);
        p.per = (T - 1) / p.tiles + 1;
        p.sort_words *= 2;
        p.hist_words = ((uint64_t)p.tiles << p.bits);
    }
    return p;
}

int64_t fwd_blocks(int dtype, int T, int C) {
    const int rows = kNT >> lane_shift((C - 1) / (dtype == FG_DTYPE_F32 ? 4 : 8) + 1);
    return ((int64_t)T + rows - 1) / rows;
}

template <int DT>
int launch_fwd(fg_ctx *ctx, const uint32_t *tokens, int T, int V, int C, const void *table, int ldt,
               float scale, void *out, int ldo) {
    using Ty = typename Io<DT>::T;
    emb_fwd<DT><<<(unsigned)fwd_blocks(DT, T, C), kNT, 0, ctx->stream>>>(
        {tokens, static_cast<const Ty *>(table), static_cast<Ty *>(out), T, V, C, ldt, ldo,
         lane_shift((C - 1) / Io<DT>::E + 1), scale});
    FG_LAUNCH_CHECK("emb_fwd");
    return FG_OK;
}

template <int DT>
int launch_bwd(fg_ctx *ctx, const Plan &pl, void *ws, const uint32_t *tokens, int T, int V, int C,
               const void *dout, int lddo, float scale, void *dtable, int lddt, int accumulate) {
    using Ty = typename Io<DT>::T;
    const Ty *d = static_cast<const Ty *>(dout);
    Ty *g = static_cast<Ty *>(dtable);
    hipStream_t st = ctx->stream;
    const int chunks = (C - 1) / Io<DT>::E + 1;
    if (T <= kDirectMax) {
        const int lshift = lane_shift(chunks), at_once = kNT >> lshift;
        // Table rows of a workgroup: those it takes at once, more where the table is long.
        const int rows = (int)std::max<int64_t>(at_once, (V - 1) / (16 * ctx->cu_count) + 1);
        emb_bwd_few<DT><<<(V - 1) / rows + 1, kNT, 0, st>>>(
            {tokens, d, g, T, V, C, lddo, lddt, accumulate, rows, lshift, scale});
        FG_LAUNCH_CHECK("emb_bwd_few");
        return FG_OK;
    }
    uint32_t *order = (uint32_t *)ws, *sorted = order + T;
    if (own_launch(DT, T, V, C)) {
        const int lshift = std::min(6, log2_up(chunks)), tiles = ((chunks - 1) >> lshift) + 1;
        const int blocks = std::max(1, kOwnBlocks / tiles);
        const int rows = std::min(kOrderBins, (V - 1) / blocks + 1);
        const size_t lds = 4 * ((size_t)(kOrderWaves + 2) * rows + 1 + T);
        emb_bwd_own<DT><<<dim3((V - 1) / rows + 1, tiles), kOrderNT, lds, st>>>(
            {tokens, d, g, T, V, C, lddo, lddt, accumulate, rows, lshift, scale});
        FG_LAUNCH_CHECK("emb_bwd_own");
        return FG_OK;
    }
    // Zeroed beside the sort, which leaves the memory idle: what its launches have time
    // for; the whole table where that is most of it, or where few of its rows are
    // written again.  The rest goes beside the sums, without the rows of tokens.
    // (Measured with 256 workgroups ordering and a frequent token in both batches;
    // emb_order, MB for 20011 and 32768 tokens: 34 and 50 68.3 and 86.3 us in all, 59
    // and 90 60.0 and 79.7, 95 and 150 61.0 and 72.0, 142 and 220 70.0 and 77.0.)
    constexpr double kMB = 1 << 20;
    const double row_mb = (double)C * sizeof(Ty) / kMB, q = T / 8192.0;
    const double count_mb = 16.0, place_mb = 60.0, order_mb = 20.0 + 30.0 * q;
    const double sort_mb = pl.passes ? pl.passes * (count_mb + place_mb) : order_mb;
    int early = 0, done = 0;  // rows zeroed beside the sort; by the launches so far
    if (!accumulate) {
        const bool all = V * row_mb < 1.25 * sort_mb || T <= V / 8;
        early = all ? V : (int)(sort_mb / row_mb);
    }
    Zero z{(char *)dtable, (uint64_t)lddt * sizeof(Ty), (int64_t)C * (int64_t)sizeof(Ty), 0, 0,
           std::min(6, log2_up(std::max<int64_t>(1, (int64_t)C * (int64_t)sizeof(Ty) / 16)))};
    // Workgroups (1024 threads) of the next launch's share of them.
    auto share = [&](double mb) {
        z.first = done;
        z.count = std::min(early - done, (int)(early * (mb / sort_mb)) + 1);
        done += z.count;
        const int per = 1024 >> z.lshift;  // rows at once
        return z.count ? std::min(64 * ctx->cu_count, (z.count - 1) / per + 1) : 0;
    };
    if (pl.passes == 0) {
        const int zeros = share(order_mb);
        emb_order<<<pl.blocks + zeros, kOrderNT, 4 * kOrderWaves * pl.bins, st>>>(
            {tokens, order, sorted, T, pl.bins, pl.blocks, (uint32_t)V}, z);
        FG_LAUNCH_CHECK("emb_order");
    } else {
        // The passes go back and forth between two pairs of arrays and end in the first.
        uint32_t *pos[2] = {order, order + 2 * (size_t)T};
        uint32_t *key[2] = {sorted, sorted + 2 * (size_t)T};
        uint32_t *hist = order + 4 * (size_t)T;
        const uint32_t *kin = tokens, *pin = nullptr;
        for (int n = 0; n < pl.passes; ++n) {
            const int to = (pl.passes - 1 - n) & 1;
            const Radix r{kin, pin, hist, key[to], pos[to], T, pl.per, n * pl.bits, pl.bits,
                          pl.tiles, (uint32_t)V};
            int zeros = share(count_mb);
            radix_count<<<pl.tiles + zeros, kSortNT, 0, st>>>(r, z);
            FG_LAUNCH_CHECK("radix_count");
            // (The next pass's counts added up here by atomics, one launch fewer, took the
            // first pass from 8.5 to 21 us for 65536 tokens.)
            zeros = share(place_mb);
            radix_place<<<pl.tiles + zeros, kSortNT, 0, st>>>(r, z);
            FG_LAUNCH_CHECK("radix_place");
            kin = key[to];
            pin = pos[to];
        }
    }
    Sums s{};
    s.order = order;
    s.sorted = sorted;
    s.T = T;
    s.V = V;
    s.C = C;
    s.lddo = lddo;
    s.lddt = lddt;
    s.accumulate = accumulate;
    s.scale = scale;
    s.P = pl.P;
    s.units = pl.units;
    s.lshift = pl.lshift;
    s.Cp = pl.Cp;
    s.partial = (float *)ws + ((pl.sort_words + pl.hist_words + 3) & ~uint64_t(3));
    s.unit_blocks = ((pl.units - 1) >> (8 - pl.lshift)) + 1;
    int blocks = s.unit_blocks;
    s.zrows = 1;
    s.zfirst = done;
    if (!accumulate && done < V) {
        // Rows a workgroup zeroes: about 2048 workgroups, at most one row a thread.
        while (s.zrows < kNT && (V - done) / s.zrows > 2048) s.zrows *= 2;
        blocks += (V - done - 1) / s.zrows + 1;
    }
    const int tiles = (chunks - 1) / (1 << pl.lshift) + 1;
    auto sums = pl.lshift >= 6 ? emb_sums<DT, true> : emb_sums<DT, false>;
    sums<<<dim3(blocks, tiles), kNT, 0, st>>>(s, d, g);
    FG_LAUNCH_CHECK("emb_sums");
    if (pl.units > 1) {
        emb_join<DT><<<dim3(pl.units - 1, (unsigned)((pl.Cp / 4 - 1) / kJoinNT + 1)), kJoinNT, 0,
                       st>>>(s, g);
        FG_LAUNCH_CHECK("emb_join");
    }
    return FG_OK;
}

}  // namespace

namespace fg {
uint64_t embedding_bwd_ws_bytes(int dtype, int T, int V, int C) {
    return plan_of(dtype, T, V, C).bytes();
}
int embedding_bwd_dispatches(int dtype, int T, int V, int C) {
    const Plan p = plan_of(dtype, T, V, C);
    if (p.units == 0) return 1;
    return (p.passes ? 2 * p.passes : 1) + 1 + (p.units > 1 ? 1 : 0);
}
}  // namespace fg

FG_API int fg_embedding(fg_ctx *ctx, int dtype, const uint32_t *d_tokens, int T, int V, int C,
                        const void *d_table, int ldt, float scale, void *d_out, int ldo) {
    const char *who = "fg_embedding";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(T >= 0 && V > 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape T=%d V=%d C=%d", who, T, V,
               C);
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(ldt >= C && ldo >= C, FG_ERR_SHAPE, "%s: ldt=%d or ldo=%d < C=%d", who, ldt, ldo,
               C);
    FG_REQUIRE(T == 0 || (d_tokens && d_table && d_out), FG_ERR_INVALID_ARGUMENT,
               "%s: tokens, table and out are required", who);
    FG_REQUIRE(!d_out || d_out != d_table, FG_ERR_INVALID_ARGUMENT, "%s: out is the table", who);
    FG_REQUIRE(fg::rows::grid_holds(fwd_blocks(dtype, T, C), kNT), FG_ERR_OUT_OF_BOUNDS,
               "%s: %d rows of %d columns", who, T, C);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_out, {d_tokens}), FG_ERR_INVALID_ARGUMENT, "%s: out is the tokens", who);
    if (T == 0) return FG_OK;
    FG_HIP(hipSetDevice(ctx->device));
    auto launch = dtype == FG_DTYPE_F32    ? launch_fwd<fg::kF32>
                  : dtype == FG_DTYPE_BF16 ? launch_fwd<fg::kBF16>
                                           : launch_fwd<fg::kF16>;
    return launch(ctx, d_tokens, T, V, C, d_table, ldt, scale, d_out, ldo);
}

FG_API int fg_embedding_bwd(fg_ctx *ctx, int dtype, const uint32_t *d_tokens, int T, int V, int C,
                            const void *d_dout, int lddo, float scale, void *d_dtable, int lddt,
                            int accumulate) {
    const char *who = "fg_embedding_bwd";
    FG_REQUIRE(dtype >= FG_DTYPE_F32 && dtype <= FG_DTYPE_BF16, FG_ERR_INVALID_ARGUMENT,
               "%s: bad dtype %d", who, dtype);
    FG_REQUIRE(T >= 0 && V > 0 && C > 0, FG_ERR_SHAPE, "%s: bad shape T=%d V=%d C=%d", who, T, V,
               C);
    FG_REQUIRE(C <= fg::rows::kMaxCols, FG_ERR_OUT_OF_BOUNDS, "%s: %d columns, at most %d", who, C,
               fg::rows::kMaxCols);
    FG_REQUIRE(T <= kMaxTokens, FG_ERR_OUT_OF_BOUNDS, "%s: %d tokens, at most %d", who, T,
               kMaxTokens);
    FG_REQUIRE(lddo >= C && lddt >= C, FG_ERR_SHAPE, "%s: lddo=%d or lddt=%d < C=%d", who, lddo,
               lddt, C);
    FG_REQUIRE(d_dtable && (T == 0 || (d_tokens && d_dout)), FG_ERR_INVALID_ARGUMENT,
               "%s: tokens, dout and dtable are required", who);
    FG_REQUIRE(d_dtable != d_dout, FG_ERR_INVALID_ARGUMENT, "%s: dtable is dout", who);
    FG_REQUIRE(ctx, FG_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", who);
    FG_REQUIRE(apart(d_dtable, {d_tokens}), FG_ERR_INVALID_ARGUMENT, "%s: dtable is the tokens",
               who);
    FG_HIP(hipSetDevice(ctx->device));
    const Plan pl = plan_of(dtype, T, V, C);
    void *ws = nullptr;
    if (pl.units > 0 && !(ws = fg::workspace(ctx, pl.bytes()))) return FG_ERR_OUT_OF_MEMORY;
    auto launch = dtype == FG_DTYPE_F32    ? launch_bwd<fg::kF32>
                  : dtype == FG_DTYPE_BF16 ? launch_bwd<fg::kBF16>
                                           : launch_bwd<fg::kF16>;
    return launch(ctx, pl, ws, d_tokens, T, V, C, d_dout, lddo, scale, d_dtable, lddt, accumulate);
}
