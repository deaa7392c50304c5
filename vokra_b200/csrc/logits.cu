// logits.cu — the rules between a decoder's logits and the choice of a token
// (repetition, frequency and presence penalties, repeated n-grams, biases,
// grammar masks), written out (vkb_logits_process) or followed by log-softmax
// and the k best tokens of each row (vkb_logits_topk).
//
// Row r, token j with count c in the row's history:
//   x = logits[r][j]
//   c > 0: x = (x > 0 ? x / rep : x * rep) - (freq * c + pres)
//   x = x + bias[bias_row[r]][j]
//   j completes an n-gram of the history, or its mask bit is clear: x = -inf
// Every operation is one IEEE fp32 rounding in this order, so the values do
// not depend on which of the two entry points computes them.
//
// Bound: the arithmetic of the rules where they are all on, else HBM: one pass
// over the logits (and, for process, one write). The history is read once for
// each window, from L2. A CTA works on windows of 256 threads x NV 16-byte vectors of one row: the logits
// of the window are loaded first, the history is counted into a table of the
// window's tokens in shared memory while they arrive (integer adds: the order
// does not matter), and every rule is applied in registers. Rows start at any
// address: the vectors are those of the row's own 16-byte grid, and the few
// elements before and behind it are moved one by one.
#include "common.cuh"
#include <algorithm>

namespace vkb {
namespace {

constexpr int LG_THREADS = 256;
constexpr int WARPS = LG_THREADS / 32;
constexpr float L2E = 1.4426950408889634f;
constexpr uint32_t BANNED = 0x80000000u;  // in a count: the token completes an n-gram
constexpr int HASH_BITS = 12, HASH = 1 << HASH_BITS;  // slots of the second pass's table of a row's history
constexpr int TOPK_MAX = VKB_LOGITS_TOPK_MAX;
constexpr int CAND = 512;                 // candidate buffer of the selection
constexpr int PRUNE_AT = 144;             // candidates that are worth a pass over them

// 2^x on the special-function unit (relative error about 2^-22, -inf -> 0).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Rules {
    const int32_t* hist;
    int64_t hist_ld, hist_cols;
    const int32_t* hist_len;
    const float *rep, *freq, *pres;
    int ngram;
    const float* bias;
    int64_t bias_ld;
    const int32_t* bias_row;
    int n_bias;
    const uint32_t* mask;
    int64_t mask_ld;
    const int32_t* mask_row;
    int n_mask;
};

// What the rules are for one row.
struct RowRules {
    const int32_t* hist;
    int n_hist;
    float rep, freq, pres;
    const float* bias;
    const uint32_t* mask;
    __device__ RowRules(const Rules& R, int row) {
        hist = nullptr;
        n_hist = 0;
        if (R.hist) {
            hist = R.hist + (int64_t)row * R.hist_ld;
            const int64_t n = R.hist_len ? (int64_t)R.hist_len[row] : R.hist_cols;
            n_hist = (int)(n < 0 ? 0 : n > R.hist_cols ? R.hist_cols : n);
        }
        rep = R.rep ? R.rep[row] : 1.0f;
        freq = R.freq ? R.freq[row] : 0.0f;
        pres = R.pres ? R.pres[row] : 0.0f;
        const int b = R.bias ? (R.bias_row ? R.bias_row[row] : 0) : -1;
        bias = b >= 0 && b < R.n_bias ? R.bias + (int64_t)b * R.bias_ld : nullptr;
        const int m = R.mask ? (R.mask_row ? R.mask_row[row] : 0) : -1;
        mask = m >= 0 && m < R.n_mask ? R.mask + (int64_t)m * R.mask_ld : nullptr;
    }
};

// The penalties of a token that occurs c times.
__device__ __forceinline__ float penalized(const RowRules& rr, float x, uint32_t c) {
    x = x > 0.0f ? __fdiv_rn(x, rr.rep) : __fmul_rn(x, rr.rep);
    return __fsub_rn(x, __fadd_rn(__fmul_rn(rr.freq, (float)c), rr.pres));
}

// Whether id i of the history ends an n-gram whose first ngram - 1 ids are the history's last ones.
__device__ __forceinline__ bool ends_ngram(const RowRules& rr, int ngram, int i) {
    if (ngram <= 1 || i < ngram - 1) return false;
    for (int e = 1; e < ngram; ++e)
        if (rr.hist[i - e] != rr.hist[rr.n_hist - e]) return false;
    return true;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ float get(const uint4& u, int e) { return __uint_as_float((&u.x)[e]); }
};
template <> struct Vec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float get(const uint4& u, int e) {
        const uint32_t w = (&u.x)[e >> 1];
        return h2f((uint16_t)(e & 1 ? w >> 16 : w & 0xffffu));
    }
};
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__half* p, float x) { *p = __float2half_rn(x); }

// How often each token of a window occurs in the row's history, in shared memory (integer adds: the order does not
// matter), and a bit for each token that does, so that a look at the others costs a byte for eight.
template <int TOKENS>
struct History {
    static constexpr int BYTES = (TOKENS + TOKENS / 32) * 4;
    uint32_t *cnt, *bits;
    // Counts for the window at `lo`; ends with a barrier.
    __device__ __forceinline__ void count(const RowRules& rr, int ngram, uint32_t* smem, int lo, int vocab) {
        cnt = smem;
        bits = smem + TOKENS;
        const int first = max(lo, 0);
        const uint32_t width = (uint32_t)max(0, min(lo + TOKENS, vocab) - first);
        int id[4];
        auto fetch = [&](int base) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = base + k * LG_THREADS + (int)threadIdx.x;
                id[k] = i < rr.n_hist ? rr.hist[i] : -1;
            }
        };
        fetch(0);
        for (int i = threadIdx.x; i < BYTES / 16; i += LG_THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int base = 0; base < rr.n_hist; base += 4 * LG_THREADS) {
            if (base) fetch(base);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = id[k] - lo;
                const bool here = (uint32_t)id[k] - (uint32_t)first < width;
                const unsigned with = __ballot_sync(0xffffffffu, here);
                if (!here) continue;
                int times = 1;
                if (__popc(with) >= 8) {  // a loop of a few tokens would queue up at a few addresses: one lane adds for all equal ones
                    const unsigned same = __match_any_sync(with, t);
                    times = (int)(threadIdx.x & 31) == __ffs(same) - 1 ? __popc(same) : 0;
                }
                if (times) {
                    atomicAdd(&cnt[t], (uint32_t)times);
                    atomicOr(&bits[t >> 5], 1u << (t & 31));
                }
                if (ends_ngram(rr, ngram, base + k * LG_THREADS + (int)threadIdx.x)) atomicOr(&cnt[t], BANNED);
            }
        }
        __syncthreads();
    }
};

// The window's share of one thread: NV vectors of the row's 16-byte grid.
// j0(v) is the vocabulary index of vector v's first element (it may be
// negative, or the vector may end behind the row).
template <typename T, int NV>
struct Window {
    static constexpr int N = Vec<T>::N;
    [[maybe_unused]] static constexpr int TOKENS = LG_THREADS * NV * N;
    int lo;  // vocabulary index of the window's first slot
    int vocab;
    __device__ __forceinline__ int slot(int v) const { return (v * LG_THREADS + (int)threadIdx.x) * N; }
    __device__ __forceinline__ int j0(int v) const { return lo + slot(v); }
    __device__ __forceinline__ bool whole(int v) const { return j0(v) >= 0 && j0(v) + N <= vocab; }

    // logits as raw vectors; elements outside the row are -inf (whatever the rules make of them, they stay so)
    __device__ __forceinline__ void load1(const T* row, int v, uint4& raw) const {
        if (whole(v)) {
            raw = __ldcs(reinterpret_cast<const uint4*>(row + j0(v)));
        } else {
            T part[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int j = j0(v) + e;
                part[e] = j >= 0 && j < vocab ? row[j] : T(-INFINITY);
            }
            memcpy(&raw, part, 16);
        }
    }
    __device__ __forceinline__ void load(const T* row, uint4 (&raw)[NV]) const {
#pragma unroll
        for (int v = 0; v < NV; ++v) load1(row, v, raw[v]);
    }
    // The window's bias values and mask words, asked for before the history is counted. Through L1: where the bias row
    // does not share the logits' 16-byte grid, eight neighbouring words come one by one from the same line (past L1 that
    // was 8 times the traffic: 256 rows of 131071, 184 us).
    struct Extra {
        float bias[N];
        uint32_t mask[2];
    };
    __device__ __forceinline__ void fetch(const RowRules& rr, int v, Extra& x) const {
        if (rr.bias) {
            const float* b = rr.bias + j0(v);
            if (whole(v) && (reinterpret_cast<uintptr_t>(rr.bias + lo) & 15) == 0) {
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const float4 b4 = *reinterpret_cast<const float4*>(b + e);
                    x.bias[e] = b4.x;
                    x.bias[e + 1] = b4.y;
                    x.bias[e + 2] = b4.z;
                    x.bias[e + 3] = b4.w;
                }
            } else if (whole(v)) {
#pragma unroll
                for (int e = 0; e < N; ++e) x.bias[e] = b[e];
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) x.bias[e] = j0(v) + e >= 0 && j0(v) + e < vocab ? b[e] : 0.0f;
            }
        }
        if (rr.mask) {
            // bits j0 .. j0 + N - 1: they lie in one or two words
            const int first = min(max(j0(v), 0), vocab - 1), last = min(max(j0(v) + N - 1, 0), vocab - 1);
            x.mask[0] = rr.mask[first >> 5];
            x.mask[1] = rr.mask[last >> 5];
        }
    }
    // The rules on vector v.
    template <int TABLE>
    __device__ __forceinline__ void apply(const RowRules& rr, const History<TABLE>& hist, bool counted, const uint4& raw,
                                          const Extra& extra, int v, float (&x)[N]) const {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = Vec<T>::get(raw, e);
        uint32_t banned = 0;
        if (counted) {
            const int at = slot(v);
            uint32_t hit = (reinterpret_cast<const uint8_t*>(hist.bits)[at >> 3] >> (at & 7)) & ((1u << N) - 1);
            // one element of a lane at a time, so that lanes with one hit each, at whatever place, take one turn together
            while (hit) {
                const int which = __ffs(hit) - 1;
                hit &= hit - 1;
                float y = x[0];
#pragma unroll
                for (int e = 1; e < N; ++e) y = which == e ? x[e] : y;
                const uint32_t c = hist.cnt[at + which];
                y = penalized(rr, y, c & ~BANNED);
                banned |= (c >> 31) << which;
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] = which == e ? y : x[e];
            }
        }
        finish(rr, extra, v, banned, x);
    }
    // Bias and mask, after the penalties; `banned` has a bit for each element that an n-gram excludes.
    __device__ __forceinline__ void finish(const RowRules& rr, const Extra& extra, int v, uint32_t banned, float (&x)[N]) const {
        const int j = j0(v);
        if (rr.bias) {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = __fadd_rn(x[e], extra.bias[e]);
        }
        if (rr.mask) {
            const int first = min(max(j, 0), vocab - 1);
            const uint32_t bits = __funnelshift_r(extra.mask[0], extra.mask[1], first & 31);
            banned |= ~(bits << (first - j));  // (a bit of an element outside the row says nothing)
        }
        if (banned) {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = banned & (1u << e) ? -INFINITY : x[e];
        }
    }
};

// (Four blocks an SM: 14.8 to 16.4 us for 128 rows of 51866 in f32; five 17.9 and six 18.6, with spills.)
template <typename T, int NV>
__global__ void __launch_bounds__(LG_THREADS, 4) logits_process_kernel(const T* logits, int64_t ld, int vocab,
                                                                       Rules R, T* out, int64_t out_ld) {
    pdl_entry();
    using W = Window<T, NV>;
    extern __shared__ __align__(16) uint32_t lg_cnt[];
    const int row = blockIdx.y;
    const T* in = logits + (int64_t)row * ld;
    T* to = out + (int64_t)row * out_ld;
    const int shift = (int)(reinterpret_cast<uintptr_t>(in) / sizeof(T) % W::N);
    W w;
    w.vocab = vocab;
    w.lo = (int)blockIdx.x * W::TOKENS - shift;
    uint4 raw[NV];
    w.load(in, raw);
    const RowRules rr(R, row);
    typename W::Extra extra[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) w.fetch(rr, v, extra[v]);
    const bool counted = rr.n_hist > 0;
    History<W::TOKENS> hist;
    if (counted) hist.count(rr, R.ngram, lg_cnt, w.lo, vocab);
    const bool same_grid = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(to)) & 15) == 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float x[W::N];
        w.apply(rr, hist, counted, raw[v], extra[v], v, x);
        if (same_grid && w.whole(v)) {
            T part[W::N];
#pragma unroll
            for (int e = 0; e < W::N; ++e) store1(part + e, x[e]);
            uint4 u;
            memcpy(&u, part, 16);
            *reinterpret_cast<uint4*>(to + w.j0(v)) = u;
        } else {
#pragma unroll
            for (int e = 0; e < W::N; ++e)
                if (w.j0(v) + e >= 0 && w.j0(v) + e < vocab) store1(to + w.j0(v) + e, x[e]);
        }
    }
}

// ---------------------------------------------------------------------------
// Selection. A candidate is one 64-bit number that orders as (value, lower
// index first): the value's bits made monotonic above the complement of the
// index. 0 is below every candidate.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as +0
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_order(uint32_t o) {
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t cand_key(float x, int j) { return (uint64_t)order_bits(x) << 32 | (uint32_t)~j; }
__device__ __forceinline__ float cand_value(uint64_t c) { return from_order((uint32_t)(c >> 32)); }
__device__ __forceinline__ int cand_index(uint64_t c) { return (int)~(uint32_t)c; }

struct Select {
    uint64_t cand[CAND + 2];    // the candidates; the first `kept` are the best so far, in order
    uint64_t next[TOPK_MAX];
    float red[2 * (LG_THREADS / 32)];
    int n;
};

// Keeps the k best of the n candidates, in order: each
// thread counts how many candidates beat its own.
__device__ __forceinline__ void select_prune(Select& s, int k) {
    __syncthreads();
    const int n = s.n;
    if (threadIdx.x == 0) s.cand[n] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
        const uint64_t me = s.cand[i];
        int rank = 0;
#pragma unroll 4
        for (int o = 0; o < n; o += 2) {  // (behind the last one lies a 0: it beats none)
            const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(s.cand + o);
            rank += (c.x > me) + (c.y > me);
        }
        if (rank < k) s.next[rank] = me;
    }
    __syncthreads();
    const int kept = min(n, k);
    for (int i = threadIdx.x; i < kept; i += LG_THREADS) s.cand[i] = s.next[i];
    if (threadIdx.x == 0) s.n = kept;
    __syncthreads();
}

// The selection in two passes, with little between them: keeping the k best of a window (an earlier form) put a barrier
// and a candidate list into the pass over all logits, 185 us for 256 rows of 131071 (f16, k = 40) against 89 now.
// What bounds the first pass is the arithmetic of the rules, all of them on: 59 us, where the logits alone would take
// 10. The second one is a chain of short steps: 28 us for 256 rows, 12 for 5.
//
// The first pass: the rules on one window of a row, and what is left of it: the largest value of each
// segment (one 16-byte step of a warp: 32 * N tokens) and the sum of exp(x - largest) of each warp.
template <typename T, int NV>
__global__ void __launch_bounds__(LG_THREADS)
    logits_stats_kernel(const T* __restrict__ logits, int64_t ld, int vocab, Rules R, float* __restrict__ seg_max,
                        float* __restrict__ warp_sums) {
    pdl_entry();
    using W = Window<T, NV>;
    extern __shared__ __align__(16) uint32_t lg_cnt[];
    const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* in = logits + (int64_t)row * ld;
    const int shift = (int)(reinterpret_cast<uintptr_t>(in) / sizeof(T) % W::N);
    W w;
    w.vocab = vocab;
    w.lo = (int)blockIdx.x * W::TOKENS - shift;
    uint4 raw[NV];
    w.load(in, raw);
    const RowRules rr(R, row);
    typename W::Extra extra;
    w.fetch(rr, 0, extra);
    const bool counted = rr.n_hist > 0;
    History<W::TOKENS> hist;
    if (counted) hist.count(rr, R.ngram, lg_cnt, w.lo, vocab);
    // vector by vector: the sum is of exp(x - most), `most` the warp's largest value so far
    float most = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float x[W::N];
        w.apply(rr, hist, counted, raw[v], extra, v, x);
        if (v + 1 < NV) w.fetch(rr, v + 1, extra);
        float mine = -INFINITY;  // (fmaxf leaves out what is not a number)
#pragma unroll
        for (int e = 0; e < W::N; ++e) mine = fmaxf(mine, x[e]);
        mine = from_order(__reduce_max_sync(0xffffffffu, order_bits(mine)));
        if (lane == 0) seg_max[((int64_t)row * gridDim.x + blockIdx.x) * NV * WARPS + v * WARPS + warp] = mine;
        const float before = most;
        most = fmaxf(most, mine);
        if (most == INFINITY) {  // +inf shares its probability among the values that reach it
            if (before != INFINITY) sum = 0.0f;
#pragma unroll
            for (int e = 0; e < W::N; ++e) sum += x[e] == INFINITY ? 1.0f : 0.0f;
        } else if (most > -INFINITY) {
            sum *= ex2((before - most) * L2E);
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < W::N; ++e) part += ex2((x[e] - most) * L2E);  // (not one fma: most * log2(e) would be rounded)
            if (part != part) {  // something is not a number: it is never chosen and no part of the sum
                part = 0.0f;
#pragma unroll
                for (int e = 0; e < W::N; ++e) part += x[e] == x[e] ? ex2((x[e] - most) * L2E) : 0.0f;
            }
            sum += part;
        }
    }
    sum = warp_sum(sum);
    if (lane == 0) warp_sums[((int64_t)row * gridDim.x + blockIdx.x) * WARPS + warp] = sum;
}

// The second pass, one block a row: a value that the k best reach from the segments' largest values, then the few
// segments that reach it once more, a warp each. Segments ascend with the tokens.
template <typename T, int NV>
__global__ void __launch_bounds__(LG_THREADS)
    logits_pick_kernel(const T* __restrict__ logits, int64_t ld, int vocab, Rules R, int k, int windows,
                       const float* __restrict__ seg_max, const float* __restrict__ warp_sums, int32_t* __restrict__ ids,
                       float* __restrict__ logprob) {
    pdl_entry();
    constexpr int N = Vec<T>::N, SEG = 32 * N;
    __shared__ __align__(16) Select s;
    extern __shared__ __align__(16) uint32_t lg_hash[];  // [2][HASH]: token + 1 (0: none), how often it occurs
    uint32_t *keys = lg_hash, *counts = lg_hash + HASH;
    __shared__ uint32_t cnt_s[WARPS][SEG];
    __shared__ int list_s[LG_THREADS];
    __shared__ int list_n[WARPS];
    __shared__ int reach_s[2][3][WARPS];
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* in = logits + (int64_t)row * ld;
    const int shift = (int)(reinterpret_cast<uintptr_t>(in) / sizeof(T) % N);
    const RowRules rr(R, row);
    const int n_warp = windows * WARPS, n_seg = n_warp * NV;
    const float* maxima = seg_max + (int64_t)row * n_seg;
    const float* sums = warp_sums + (int64_t)row * n_warp;
    // The history as a table (open addressing): what a look-up finds does not depend on the order of the inserts. One that
    // is longer than half the table is counted anew for each segment.
    const bool hashed = rr.n_hist > 0 && rr.n_hist <= HASH / 2;
    auto slot_of = [](uint32_t t) { return (t * 2654435761u) >> (32 - HASH_BITS); };
    if (hashed) {
        for (int i = threadIdx.x; i < HASH / 2; i += LG_THREADS) reinterpret_cast<uint4*>(lg_hash)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        constexpr int AT_ONCE = 8;
        for (int base = 0; base < rr.n_hist; base += AT_ONCE * LG_THREADS) {
            int ids_now[AT_ONCE];
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                const int i = base + q * LG_THREADS + (int)threadIdx.x;
                ids_now[q] = i < rr.n_hist ? rr.hist[i] : -1;
            }
#pragma unroll 1
            for (int q = 0; q < AT_ONCE && base + q * LG_THREADS < rr.n_hist; ++q) {
                int id = ids_now[0];  // (rotated, not indexed: the array stays in registers)
#pragma unroll
                for (int o = 0; o + 1 < AT_ONCE; ++o) ids_now[o] = ids_now[o + 1];
                const bool here = id >= 0 && id < vocab;
                const unsigned with = __ballot_sync(0xffffffffu, here);
                if (!here) continue;
                const unsigned same = __match_any_sync(with, id);
                const bool ends = ends_ngram(rr, R.ngram, base + q * LG_THREADS + (int)threadIdx.x);
                if (lane != __ffs(same) - 1 && !ends) continue;
                uint32_t at = slot_of((uint32_t)id);
                for (int probe = 0; probe < HASH; ++probe, at = (at + 1) & (HASH - 1)) {
                    const uint32_t was = atomicCAS(&keys[at], 0u, (uint32_t)id + 1);
                    if (was == 0 || was == (uint32_t)id + 1) break;
                }
                if (lane == __ffs(same) - 1) atomicAdd(&counts[at], (uint32_t)__popc(same));
                if (ends) atomicOr(&counts[at], BANNED);
            }
        }
    } else if (rr.n_hist) {
        for (int i = lane; i < SEG; i += 32) cnt_s[warp][i] = 0;
    }
    if (threadIdx.x == 0) s.n = 0;

    // the row's largest value and sum, in a fixed order
    float M = -INFINITY, S = 0.0f;
    auto join = [&](float am, float as) {  // (M, S) += (am, as)
        if (am == -INFINITY) return;
        if (am > M) {
            S = M == -INFINITY || am == INFINITY ? 0.0f : S * ex2((M - am) * L2E);
            M = am;
        }
        S += am == M ? as : M == INFINITY ? 0.0f : as * ex2((am - M) * L2E);
    };
#pragma unroll 2
    for (int i = threadIdx.x; i < n_warp; i += LG_THREADS) {
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < NV; ++v) m = fmaxf(m, __ldcg(maxima + (i / WARPS * NV + v) * WARPS + i % WARPS));
        join(m, __ldcg(sums + i));
    }
    // The bound: what k segments' largest values reach, to the first 16 bits of their order (more would not spare a
    // segment often); with fewer than k segments above -inf, all of them.
    float bound = -INFINITY;
    {
        constexpr int KEPT = 4;  // of a thread's segments, in registers
        uint32_t key[KEPT];
#pragma unroll
        for (int i = 0; i < KEPT; ++i) {
            const int g = i * LG_THREADS + (int)threadIdx.x;
            key[i] = g < n_seg ? order_bits(__ldcg(maxima + g)) : 0;
        }
        uint32_t prefix = 0;
        for (int bit = 30; bit >= 16; bit -= 2) {  // two bits a turn: how many reach each of the three values above the prefix
            int reach[3] = {0, 0, 0};
            auto look = [&](uint32_t o) {
#pragma unroll
                for (uint32_t v = 1; v < 4; ++v) reach[v - 1] += o >= (prefix | v << bit);
            };
#pragma unroll
            for (int i = 0; i < KEPT; ++i) look(key[i]);
            for (int g = KEPT * LG_THREADS + (int)threadIdx.x; g < n_seg; g += LG_THREADS) look(order_bits(__ldcg(maxima + g)));
#pragma unroll
            for (int v = 0; v < 3; ++v) reach[v] = __reduce_add_sync(0xffffffffu, reach[v]);
            if (lane < 3) reach_s[bit >> 1 & 1][lane][warp] = lane == 0 ? reach[0] : lane == 1 ? reach[1] : reach[2];
            __syncthreads();  // (the other half of the array is written in the next turn)
            uint32_t most = 0;
#pragma unroll
            for (uint32_t v = 1; v < 4; ++v) {
                int all = 0;
#pragma unroll
                for (int o = 0; o < WARPS; ++o) all += reach_s[bit >> 1 & 1][v - 1][o];
                if (all >= k) most = v;
            }
            prefix |= most << bit;
        }
        if (prefix > order_bits(-INFINITY)) bound = from_order(prefix);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, M, o), os = __shfl_xor_sync(0xffffffffu, S, o);
        join(om, os);
    }
    __syncthreads();
    if (lane == 0) {
        s.red[warp] = M;
        s.red[WARPS + warp] = S;
    }
    __syncthreads();
    M = -INFINITY;
    S = 0.0f;
    for (int o = 0; o < WARPS; ++o) join(s.red[o], s.red[WARPS + o]);

    bool exact = false;  // the bound is the k-th best so far: only what exceeds it matters, for it would lose a tie
    // a value that is wanted; -inf never is
    auto wanted = [&](float x) { return exact ? x > bound : x >= bound && x > -INFINITY; };

    const bool lowers = rr.rep >= 1.0f && rr.freq >= 0.0f && rr.pres >= 0.0f;
    // segment g by one warp
    auto scan = [&](int g) {
        const int j = g * SEG + lane * N - shift;
        Window<T, 1> w;
        w.vocab = vocab;
        w.lo = j - (int)threadIdx.x * N;  // (the window whose vector 0 is this one)
        uint4 raw;
        w.load1(in, 0, raw);
        typename Window<T, 1>::Extra extra;
        w.fetch(rr, 0, extra);
        float x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = Vec<T>::get(raw, e);
        // which elements the history may matter for: where penalties only lower (every rounding keeps the order), those
        // that are wanted without them
        uint32_t look = 0, banned = 0;
        {
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = x[e];
            w.finish(rr, extra, 0, 0, y);
#pragma unroll
            for (int e = 0; e < N; ++e) look |= (!lowers || wanted(y[e]) ? 1u : 0u) << e;
        }
        if (!hashed && rr.n_hist && __any_sync(0xffffffffu, look)) {
            uint32_t* cnt = cnt_s[warp];
            const int lo = g * SEG - shift;
            for (int base = 0; base < rr.n_hist; base += 128) {
                int id[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = base + 32 * q + lane;
                    id[q] = i < rr.n_hist ? rr.hist[i] : -1;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const bool here = id[q] >= 0 && id[q] < vocab && id[q] >= lo && id[q] < lo + SEG;
                    const unsigned with = __ballot_sync(0xffffffffu, here);
                    if (!here) continue;
                    const unsigned same = __match_any_sync(with, id[q]);
                    if (lane == __ffs(same) - 1) atomicAdd(&cnt[id[q] - lo], (uint32_t)__popc(same));
                    if (ends_ngram(rr, R.ngram, base + 32 * q + lane)) atomicOr(&cnt[id[q] - lo], BANNED);
                }
            }
            __syncwarp();
        }
        if (rr.n_hist) {
            uint32_t todo = look;
            while (todo) {
                const int which = __ffs(todo) - 1;
                todo &= todo - 1;
                uint32_t c = 0;
                if (hashed) {
                    const uint32_t want = (uint32_t)(j + which) + 1;
                    uint32_t at = slot_of(want - 1), key = keys[at];
                    while (key != 0 && key != want) key = keys[at = (at + 1) & (HASH - 1)];  // (half of the table is empty)
                    if (key == want) c = counts[at];
                } else {
                    c = cnt_s[warp][lane * N + which];
                }
                if (!c) continue;
                float y = x[0];
#pragma unroll
                for (int e = 1; e < N; ++e) y = which == e ? x[e] : y;
                y = penalized(rr, y, c & ~BANNED);
                banned |= (c >> 31) << which;
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] = which == e ? y : x[e];
            }
            if (!hashed) {
                __syncwarp();
#pragma unroll
                for (int e = 0; e < N; ++e) cnt_s[warp][lane * N + e] = 0;
                __syncwarp();
            }
        }
        w.finish(rr, extra, 0, banned, x);
        uint32_t hit = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) hit |= (wanted(x[e]) ? 1u : 0u) << e;
        if (hit) {
            int at = atomicAdd(&s.n, __popc(hit));  // what there is no room for is only counted
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (hit & (1u << e)) {
                    if (at < CAND) s.cand[at] = cand_key(x[e], j + e);
                    ++at;
                }
        }
    };
    auto prune = [&] {
        select_prune(s, k);
        if (s.n == k) {
            bound = cand_value(s.cand[k - 1]);
            exact = true;
        }
    };

    for (int g0 = 0; g0 < n_seg; g0 += LG_THREADS) {
        // the segments of these that reach the bound, in order
        const int g = g0 + (int)threadIdx.x;
        const bool take = g < n_seg && wanted(__ldcg(maxima + g));
        const unsigned takers = __ballot_sync(0xffffffffu, take);
        __syncthreads();
        if (lane == 0) list_n[warp] = __popc(takers);
        __syncthreads();
        int at = __popc(takers & ((1u << lane) - 1)), n_list = 0;
        for (int o = 0; o < WARPS; ++o) {
            if (o < warp) at += list_n[o];
            n_list += list_n[o];
        }
        if (take) list_s[at] = g;
        __syncthreads();
        constexpr int ROUND = 2 * WARPS;
        for (int i = 0; i < n_list; i += ROUND) {
            const int have = s.n;  // (at rest: a barrier lies behind its last change)
            __syncthreads();
#pragma unroll
            for (int o = 0; o < ROUND; o += WARPS)
                if (i + o + warp < n_list) scan(list_s[i + o + warp]);
            __syncthreads();
            const int n = s.n;
            __syncthreads();
            if (n > CAND) {
                // many equal values: one segment after another, which always fits, the bound rising as soon as it can
                if (threadIdx.x == 0) s.n = have;
                __syncthreads();
                for (int o = 0; o < ROUND && i + o < n_list; ++o) {
                    if (warp == o % WARPS) scan(list_s[i + o]);
                    prune();
                }
            } else if (n >= PRUNE_AT) {
                prune();
            }
        }
    }
    static_assert(PRUNE_AT + SEG <= CAND && TOPK_MAX < PRUNE_AT, "one segment more always fits");
    prune();
    const float lse = logf(S);
    for (int i = threadIdx.x; i < k; i += LG_THREADS) {
        const bool have = i < s.n;
        const float x = have ? cand_value(s.cand[i]) : -INFINITY;
        ids[(int64_t)row * k + i] = have ? cand_index(s.cand[i]) : -1;
        logprob[(int64_t)row * k + i] = !have ? -INFINITY : M == INFINITY ? (x == INFINITY ? -lse : -INFINITY) : (x - M) - lse;
    }
}

Rules check_rules(const vkb_logits_rules* r, int64_t vocab) {
    Rules R{};
    if (!r) return R;
    if (r->hist_ld < 0) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: negative hist_ld");
    if (r->hist_cols < 0 || r->hist_cols > r->hist_ld) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: hist_cols must be in 0..hist_ld");
    if (r->hist_len_dev && !r->hist_dev) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: history lengths without a history");
    if (r->hist_ld > INT32_MAX) fail(VKB_ERROR_UNSUPPORTED_OP, "logits: history longer than 2^31 - 1");
    if (r->no_repeat_ngram < 0) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: negative no_repeat_ngram");
    if (r->bias_dev && (r->n_bias <= 0 || (r->n_bias > 1 && r->bias_ld < vocab)))
        fail(VKB_ERROR_INVALID_ARGUMENT, "logits: the bias table needs n_bias >= 1 rows of at least n_vocab values");
    if (r->mask_dev && (r->n_mask <= 0 || (r->n_mask > 1 && r->mask_ld < (vocab + 31) / 32)))
        fail(VKB_ERROR_INVALID_ARGUMENT, "logits: the mask table needs n_mask >= 1 rows of at least ceil(n_vocab / 32) words");
    R.hist = r->hist_ld > 0 ? r->hist_dev : nullptr;
    R.hist_ld = r->hist_ld;
    R.hist_cols = r->hist_cols ? r->hist_cols : r->hist_ld;
    R.hist_len = r->hist_len_dev;
    R.rep = r->repetition_dev;
    R.freq = r->frequency_dev;
    R.pres = r->presence_dev;
    R.ngram = r->no_repeat_ngram;
    R.bias = r->bias_dev;
    R.bias_ld = r->bias_ld;
    R.bias_row = r->bias_row_dev;
    R.n_bias = r->n_bias;
    R.mask = r->mask_dev;
    R.mask_ld = r->mask_ld;
    R.mask_row = r->mask_row_dev;
    R.n_mask = r->n_mask;
    return R;
}

void check_logits(const vkb_context* ctx, const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t ld) {
    if (!ctx) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: null context");
    if (dtype != VKB_DT_F32 && dtype != VKB_DT_F16) fail(VKB_ERROR_UNSUPPORTED_OP, "logits: dtype must be F32 or F16");
    if (n_rows < 0 || vocab <= 0) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: empty vocabulary or negative rows");
    if (vocab > (1 << 30)) fail(VKB_ERROR_UNSUPPORTED_OP, "logits: vocabulary above 2^30");
    if (n_rows > 1 && ld < vocab) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: ld below n_vocab");
    if (n_rows && !logits) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: null logits");
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == VKB_DT_F32 ? 4 : 2))
        fail(VKB_ERROR_INVALID_ARGUMENT, "logits: misaligned logits");
}

// 16-byte vectors of a thread. process, 128 rows of 51866 (f32): 2 vectors 17.2 us, 4 15.5 (14.8 to 16.4 with four blocks
// an SM); the same in f16: 1 vector 23.4, 2 21.3, 4 26. Selection, 256 rows of 131071 (f16): 2 vectors 108 us, 3 107, 4 104 (fewer looks at a history of 2048 tokens).
constexpr int NV_F32 = 4, NV_F16 = 2, NV_TOPK = 4;
constexpr int64_t ROWS_PER_LAUNCH = 32768;  // grid.y

// The rules of the rows from r0 on.
Rules rows_from(Rules R, int64_t r0) {
    if (R.hist) R.hist += r0 * R.hist_ld;
    for (const int32_t** p : {&R.hist_len, &R.bias_row, &R.mask_row})
        if (*p) *p += r0;
    for (const float** p : {&R.rep, &R.freq, &R.pres})
        if (*p) *p += r0;
    return R;
}

template <typename T, int NV>
void launch_process(vkb_context* ctx, const T* in, int64_t ld, int64_t n_rows, int vocab, const Rules& R0, T* out,
                    int64_t out_ld) {
    using W = Window<T, NV>;
    const unsigned windows = (unsigned)ceil_div((int64_t)vocab + W::N - 1, W::TOKENS);
    const size_t smem = R0.hist ? History<W::TOKENS>::BYTES : 0;
    for (int64_t r0 = 0; r0 < n_rows; r0 += ROWS_PER_LAUNCH) {
        const Rules R = rows_from(R0, r0);
        const unsigned rows = (unsigned)std::min<int64_t>(ROWS_PER_LAUNCH, n_rows - r0);
        launch_pdl(ctx, logits_process_kernel<T, NV>, dim3(windows, rows), LG_THREADS, smem, in + r0 * ld, ld, vocab, R,
                   out + r0 * out_ld, out_ld);
        VKB_CUDA(cudaGetLastError());
        ctx->count();
    }
}

template <typename T, int NV>
void launch_topk(vkb_context* ctx, const T* in, int64_t ld, int64_t n_rows, int vocab, const Rules& R0, int k,
                 int32_t* ids, float* logprob) {
    using W = Window<T, NV>;
    const int64_t windows = ceil_div((int64_t)vocab + W::N - 1, W::TOKENS);
    const size_t smem = R0.hist ? History<W::TOKENS>::BYTES : 0;
    for (int64_t r0 = 0; r0 < n_rows; r0 += ROWS_PER_LAUNCH) {
        const Rules R = rows_from(R0, r0);
        const int64_t rows = std::min<int64_t>(ROWS_PER_LAUNCH, n_rows - r0);
        const size_t maxima = (size_t)(rows * windows * NV * WARPS), sums = (size_t)(rows * windows * WARPS);
        ctx->ensure_workspace((maxima + sums) * sizeof(float));
        float* ws = ctx->workspace.as<float>();
        launch_pdl(ctx, logits_stats_kernel<T, NV>, dim3((unsigned)windows, (unsigned)rows), LG_THREADS, smem, in + r0 * ld,
                   ld, vocab, R, ws, ws + maxima);
        smem_optin(logits_pick_kernel<T, NV>, 2 * HASH * (int)sizeof(uint32_t));
        launch_pdl(ctx, logits_pick_kernel<T, NV>, dim3((unsigned)rows), LG_THREADS, R0.hist ? 2 * HASH * sizeof(uint32_t) : 0, in + r0 * ld, ld, vocab, R, k,
                   (int)windows, ws, ws + maxima, ids + r0 * k, logprob + r0 * k);
        VKB_CUDA(cudaGetLastError());
        ctx->count(2);
    }
}

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" {

vkb_status vkb_logits_process(vkb_context* ctx, const void* logits_dev, int32_t dtype, int64_t n_rows, int64_t n_vocab,
                              int64_t ld, const vkb_logits_rules* rules, void* out_dev, int64_t out_ld) {
    return guard([&] {
        check_logits(ctx, logits_dev, dtype, n_rows, n_vocab, ld);
        const Rules R = check_rules(rules, n_vocab);
        if (n_rows == 0) return;
        if (!out_dev || reinterpret_cast<uintptr_t>(out_dev) % (dtype == VKB_DT_F32 ? 4 : 2))
            fail(VKB_ERROR_INVALID_ARGUMENT, "logits_process: null or misaligned out");
        if (n_rows > 1 && out_ld < n_vocab) fail(VKB_ERROR_INVALID_ARGUMENT, "logits_process: out_ld below n_vocab");
        if (out_dev == logits_dev && n_rows > 1 && out_ld != ld)
            fail(VKB_ERROR_INVALID_ARGUMENT, "logits_process: in place needs out_ld == ld");
        NvtxRange nvtx_range("vkb.logits.process");
        const int v = (int)n_vocab;
        if (dtype == VKB_DT_F32)
            launch_process<float, NV_F32>(ctx, reinterpret_cast<const float*>(logits_dev), ld, n_rows, v, R,
                                     reinterpret_cast<float*>(out_dev), out_ld);
        else
            launch_process<__half, NV_F16>(ctx, reinterpret_cast<const __half*>(logits_dev), ld, n_rows, v, R,
                                      reinterpret_cast<__half*>(out_dev), out_ld);
    });
}

vkb_status vkb_logits_topk(vkb_context* ctx, const void* logits_dev, int32_t dtype, int64_t n_rows, int64_t n_vocab,
                           int64_t ld, const vkb_logits_rules* rules, int32_t k, int32_t* ids_dev, float* logprob_dev) {
    return guard([&] {
        check_logits(ctx, logits_dev, dtype, n_rows, n_vocab, ld);
        const Rules R = check_rules(rules, n_vocab);
        if (k < 1 || k > TOPK_MAX)
            fail(VKB_ERROR_INVALID_ARGUMENT, "logits_topk: k must be in 1.." + std::to_string(TOPK_MAX));
        if (n_rows == 0) return;
        if (!ids_dev || !logprob_dev) fail(VKB_ERROR_INVALID_ARGUMENT, "logits_topk: null outputs");
        NvtxRange nvtx_range("vkb.logits.topk");
        const int v = (int)n_vocab;
        if (dtype == VKB_DT_F32)
            launch_topk<float, NV_TOPK>(ctx, reinterpret_cast<const float*>(logits_dev), ld, n_rows, v, R, k, ids_dev,
                                  logprob_dev);
        else
            launch_topk<__half, NV_TOPK>(ctx, reinterpret_cast<const __half*>(logits_dev), ld, n_rows, v, R, k, ids_dev,
                                   logprob_dev);
    });
}

}  // extern "C"
