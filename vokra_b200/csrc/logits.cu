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
// Bound: HBM, one pass over the logits (and, for process, one write). A CTA
// works on windows of 256 threads x NV 16-byte vectors of one row: the logits
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
constexpr int TOPK_MAX = VKB_LOGITS_TOPK_MAX;
constexpr int CAND = 512;                 // candidate buffer of the selection
constexpr uint32_t BANNED = 0x80000000u;  // in a count: the token completes an n-gram

struct Rules {
    const int32_t* hist;
    int64_t hist_ld;
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
            const int64_t n = R.hist_len ? (int64_t)R.hist_len[row] : R.hist_ld;
            n_hist = (int)(n < 0 ? 0 : n > R.hist_ld ? R.hist_ld : n);
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

// The window's share of one thread: NV vectors of the row's 16-byte grid.
// j0(v) is the vocabulary index of vector v's first element (it may be
// negative, or the vector may end behind the row).
template <typename T, int NV>
struct Window {
    static constexpr int N = Vec<T>::N;
    static constexpr int TOKENS = LG_THREADS * NV * N;
    int lo;  // vocabulary index of the window's first slot
    int vocab;
    __device__ __forceinline__ int slot(int v) const { return (v * LG_THREADS + (int)threadIdx.x) * N; }
    __device__ __forceinline__ int j0(int v) const { return lo + slot(v); }
    __device__ __forceinline__ bool whole(int v) const { return j0(v) >= 0 && j0(v) + N <= vocab; }

    // logits as raw vectors; elements outside the row stay 0 and are skipped by every user
    __device__ __forceinline__ void load(const T* row, uint4 (&raw)[NV]) const {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            raw[v] = make_uint4(0, 0, 0, 0);
            if (whole(v)) {
                raw[v] = __ldcs(reinterpret_cast<const uint4*>(row + j0(v)));
            } else {
                T part[N];
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int j = j0(v) + e;
                    part[e] = j >= 0 && j < vocab ? row[j] : T(0.0f);
                }
                memcpy(&raw[v], part, 16);
            }
        }
    }
    // Counts the history's tokens of this window, and marks those that would complete an n-gram.
    __device__ __forceinline__ void count(const RowRules& rr, int ngram, uint32_t* cnt) const {
        for (int i = threadIdx.x; i < TOKENS / 4; i += LG_THREADS)
            reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int i = threadIdx.x; i < rr.n_hist; i += LG_THREADS) {
            const int id = rr.hist[i];
            if (id < 0 || id >= vocab || id < lo || id - lo >= TOKENS) continue;
            atomicAdd(&cnt[id - lo], 1u);
            // token i ends an n-gram whose first ngram - 1 tokens are the history's last ones
            if (ngram > 1 && i >= ngram - 1) {
                bool same = true;
                for (int e = 1; e < ngram && same; ++e) same = rr.hist[i - e] == rr.hist[rr.n_hist - e];
                if (same) atomicOr(&cnt[id - lo], BANNED);
            }
        }
        __syncthreads();
    }
    // The rules on vector v; `ok` has a bit for each element inside the row.
    __device__ __forceinline__ void apply(const RowRules& rr, const uint32_t* cnt, bool counted, const uint4& raw, int v,
                                          float (&x)[N], uint32_t& ok) const {
        const int j = j0(v);
        ok = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            x[e] = Vec<T>::get(raw, e);
            ok |= (j + e >= 0 && j + e < vocab ? 1u : 0u) << e;
        }
        uint32_t banned = 0;
        if (counted) {
#pragma unroll
            for (int e4 = 0; e4 < N; e4 += 4) {
                const uint4 c4 = *reinterpret_cast<const uint4*>(cnt + slot(v) + e4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t c = (&c4.x)[e];
                    if (c) {
                        float y = x[e4 + e];
                        y = y > 0.0f ? __fdiv_rn(y, rr.rep) : __fmul_rn(y, rr.rep);
                        const float n = (float)(c & ~BANNED);
                        x[e4 + e] = __fsub_rn(y, __fadd_rn(__fmul_rn(rr.freq, n), rr.pres));
                        banned |= (c >> 31) << (e4 + e);
                    }
                }
            }
        }
        if (rr.bias) {
            const float* b = rr.bias + j;
            if (ok == (1u << N) - 1 && (reinterpret_cast<uintptr_t>(b) & 15) == 0) {
#pragma unroll
                for (int e4 = 0; e4 < N; e4 += 4) {
                    const float4 b4 = __ldcg(reinterpret_cast<const float4*>(b + e4));
                    x[e4] = __fadd_rn(x[e4], b4.x);
                    x[e4 + 1] = __fadd_rn(x[e4 + 1], b4.y);
                    x[e4 + 2] = __fadd_rn(x[e4 + 2], b4.z);
                    x[e4 + 3] = __fadd_rn(x[e4 + 3], b4.w);
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (ok >> e & 1) x[e] = __fadd_rn(x[e], __ldcg(b + e));
            }
        }
        if (rr.mask && ok) {
            // bits j .. j + N - 1: they lie in one or two words of the mask
            const int first = j < 0 ? 0 : j, last = min(j + N, vocab) - 1;
            const uint32_t w0 = __ldcg(rr.mask + (first >> 5)), w1 = __ldcg(rr.mask + (last >> 5));
            const uint32_t bits = first >> 5 == last >> 5 ? w0 >> (first & 31) : __funnelshift_r(w0, w1, first & 31);
            banned |= ~(bits << (first - j)) & ok;
        }
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (banned >> e & 1) x[e] = -INFINITY;
    }
};

template <typename T, int NV>
__global__ void __launch_bounds__(LG_THREADS) logits_process_kernel(const T* logits, int64_t ld, int vocab,
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
    const bool counted = rr.n_hist > 0;
    if (counted) w.count(rr, R.ngram, lg_cnt);
    const bool same_grid = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(to)) & 15) == 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float x[W::N];
        uint32_t ok;
        w.apply(rr, lg_cnt, counted, raw[v], v, x, ok);
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
                if (ok >> e & 1) store1(to + w.j0(v) + e, x[e]);
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
    uint64_t cand[CAND];    // the candidates; the first `kept` are the best so far, in order
    uint64_t next[TOPK_MAX];
    float tmax[LG_THREADS];
    float red[2 * (LG_THREADS / 32)];
    int n, flag;
    float bound;            // values at or below it cannot be among the k best any more
};

// Keeps the k best of the n candidates, in order, and raises the bound: each
// thread counts how many candidates beat its own.
__device__ __forceinline__ void select_prune(Select& s, int k) {
    __syncthreads();
    const int n = s.n;
    for (int i = threadIdx.x; i < n; i += LG_THREADS) {
        const uint64_t me = s.cand[i];
        int rank = 0;
        for (int o = 0; o < n; ++o) rank += s.cand[o] > me;
        if (rank < k) s.next[rank] = me;
    }
    __syncthreads();
    const int kept = min(n, k);
    for (int i = threadIdx.x; i < kept; i += LG_THREADS) s.cand[i] = s.next[i];
    if (threadIdx.x == 0) {
        s.n = kept;
        if (kept == k) s.bound = cand_value(s.next[k - 1]);
    }
    __syncthreads();
}

// The k-th largest of the threads' own maxima: at least k values of the block
// reach it.
__device__ __forceinline__ float select_kth_max(Select& s, float mine, int k) {
    s.tmax[threadIdx.x] = mine;
    if (threadIdx.x == 0) s.red[0] = -INFINITY;
    __syncthreads();
    int above = 0, equal_before = 0;
    const float4* t4 = reinterpret_cast<const float4*>(s.tmax);
    for (int o = 0; o < LG_THREADS / 4; ++o) {
        const float4 t = t4[o];
        above += (t.x > mine) + (t.y > mine) + (t.z > mine) + (t.w > mine);
        const int b = 4 * o;
        equal_before += (t.x == mine && b < (int)threadIdx.x) + (t.y == mine && b + 1 < (int)threadIdx.x) +
                        (t.z == mine && b + 2 < (int)threadIdx.x) + (t.w == mine && b + 3 < (int)threadIdx.x);
    }
    if (above + equal_before == k - 1) s.red[0] = mine;
    __syncthreads();
    const float r = s.red[0];
    __syncthreads();
    return r;
}

// One block works on windows first, first + step, ... of a row and leaves its
// k best candidates, the largest value and the sum of exp(x - largest); the
// last block of the row to finish joins them.
template <typename T, int NV>
__global__ void __launch_bounds__(LG_THREADS)
    logits_topk_kernel(const T* __restrict__ logits, int64_t ld, int vocab, Rules R, int k, int windows_per_block,
                       uint64_t* part, float2* part_ms, unsigned* done, int32_t* __restrict__ ids,
                       float* __restrict__ logprob) {
    pdl_entry();
    using W = Window<T, NV>;
    extern __shared__ __align__(16) uint32_t lg_cnt[];
    __shared__ __align__(16) Select s;
    const int row = blockIdx.y, n_part = gridDim.x;
    const T* in = logits + (int64_t)row * ld;
    const int shift = (int)(reinterpret_cast<uintptr_t>(in) / sizeof(T) % W::N);
    const RowRules rr(R, row);
    const bool counted = rr.n_hist > 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        s.n = 0;
        s.bound = -INFINITY;
    }
    float m = -INFINITY, sum = 0.0f;  // of this thread's values
    constexpr float L2E = 1.4426950408889634f;
    const int n_windows = (vocab + shift + W::TOKENS - 1) / W::TOKENS;
    const int w0 = (int)blockIdx.x * windows_per_block, w1 = min(n_windows, w0 + windows_per_block);
    __syncthreads();
    for (int wi = w0; wi < w1; ++wi) {
        W w;
        w.vocab = vocab;
        w.lo = wi * W::TOKENS - shift;
        uint4 raw[NV];
        w.load(in, raw);
        if (counted) w.count(rr, R.ngram, lg_cnt);
        float x[NV][W::N];
        float mine = -INFINITY;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            uint32_t ok;
            w.apply(rr, lg_cnt, counted, raw[v], v, x[v], ok);
#pragma unroll
            for (int e = 0; e < W::N; ++e) {
                // outside the row, or not a number: never chosen and no part of the sum
                if (!(ok >> e & 1) || !(x[v][e] == x[v][e])) x[v][e] = -INFINITY;
                mine = fmaxf(mine, x[v][e]);
            }
        }
        // the running sum of exp(x - m); a largest value of +inf counts the values that reach it
        if (mine > m) {
            sum = m == -INFINITY || mine == INFINITY ? 0.0f : sum * exp2f((m - mine) * L2E);
            m = mine;
        }
        if (m == INFINITY) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < W::N; ++e) sum += x[v][e] == INFINITY ? 1.0f : 0.0f;
        } else if (m > -INFINITY) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < W::N; ++e) sum += exp2f((x[v][e] - m) * L2E);
        }
        // candidates: values above the bound. Windows ascend, so a value equal to the k-th best
        // has the higher index and loses.
        float bound = s.bound;
        int have = s.n;
        auto found = [&](bool at_bound) {  // how many of this window are above (or at) the bound
            int c = 0;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < W::N; ++e) c += at_bound ? x[v][e] >= bound : x[v][e] > bound;
            return c;
        };
        auto block_count = [&](int c) {
            if (threadIdx.x == 0) s.flag = 0;
            __syncthreads();
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0 && c) atomicAdd(&s.flag, c);
            __syncthreads();
            return s.flag;
        };
        if (!__syncthreads_or(mine > bound)) continue;
        bool at_bound = false;
        int c = block_count(found(false));
        if (have + c > CAND) {
            // too many (the first window, as a rule): the k-th largest of the threads' maxima bounds them
            const float kth = select_kth_max(s, mine, k);
            if (kth > bound) {
                bound = kth;
                at_bound = true;
                c = block_count(found(true));
            }
        }
        if (have + c <= CAND) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < W::N; ++e)
                    if (at_bound ? x[v][e] >= bound : x[v][e] > bound) {
                        const int at = atomicAdd(&s.n, 1);
                        s.cand[at] = cand_key(x[v][e], w.j0(v) + e);
                    }
            select_prune(s, k);
        } else {
            // many equal values: the window's best one after another, k times at most
            uint64_t below = ~0ull;
            for (int round = 0; round < k; ++round) {
                uint64_t best = 0;
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int e = 0; e < W::N; ++e) {
                        const uint64_t me = cand_key(x[v][e], w.j0(v) + e);
                        if (x[v][e] > -INFINITY && me < below && me > best) best = me;
                    }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
                    best = other > best ? other : best;
                }
                if (lane == 0) s.next[warp] = best;
                __syncthreads();
                if (threadIdx.x == 0) {
                    for (int o = 1; o < LG_THREADS / 32; ++o) best = s.next[o] > best ? s.next[o] : best;
                    s.next[0] = best;
                    if (best) s.cand[s.n++] = best;
                }
                __syncthreads();
                below = s.next[0];
                __syncthreads();
                if (!below) break;
            }
            select_prune(s, k);
        }
    }
    // the block's largest value and sum
    {
        const float bm = warp_max(m);
        float bs = m == -INFINITY ? 0.0f : m == bm ? sum : bm == INFINITY ? 0.0f : sum * exp2f((m - bm) * L2E);
        bs = warp_sum(bs);
        if (lane == 0) {
            s.red[warp] = bm;
            s.red[LG_THREADS / 32 + warp] = bs;
        }
        __syncthreads();
    }
    auto join = [&](float am, float as, float& M, float& S) {  // (M, S) += (am, as)
        if (am == -INFINITY) return;
        if (am > M) {
            S = M == -INFINITY || am == INFINITY ? 0.0f : S * exp2f((M - am) * L2E);
            M = am;
        }
        S += am == M ? as : M == INFINITY ? 0.0f : as * exp2f((am - M) * L2E);
    };
    float M = -INFINITY, S = 0.0f;
    for (int o = 0; o < LG_THREADS / 32; ++o) join(s.red[o], s.red[LG_THREADS / 32 + o], M, S);
    if (n_part > 1) {
        const int64_t p = (int64_t)row * n_part + blockIdx.x;
        for (int i = threadIdx.x; i < k; i += LG_THREADS) part[p * k + i] = i < s.n ? s.cand[i] : 0ull;
        if (threadIdx.x == 0) part_ms[p] = make_float2(M, S);
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            const unsigned before = atomicAdd(&done[row], 1u);
            s.flag = before == (unsigned)n_part - 1;
            if (s.flag) done[row] = 0;  // ready for the next call
        }
        __syncthreads();
        if (!s.flag) return;
        __threadfence();
        // the row's last block: joins the parts in order (the sum does not depend on who came last)
        M = -INFINITY;
        S = 0.0f;
        for (int o = 0; o < n_part; ++o) {
            const float2 ms = __ldcg(&part_ms[(int64_t)row * n_part + o]);
            join(ms.x, ms.y, M, S);
        }
        if (threadIdx.x == 0) {
            s.n = 0;
            s.bound = -INFINITY;
        }
        __syncthreads();
        const uint64_t* all = part + (int64_t)row * n_part * k;
        const int total = n_part * k, room = CAND - k;
        for (int c0 = 0; c0 < total; c0 += room) {
            for (int i = c0 + threadIdx.x; i < min(total, c0 + room); i += LG_THREADS) {
                const uint64_t c = __ldcg(all + i);
                if (c) s.cand[atomicAdd(&s.n, 1)] = c;
            }
            select_prune(s, k);
        }
    }
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
    if (r->hist_len_dev && !r->hist_dev) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: history lengths without a history");
    if (r->hist_ld > INT32_MAX) fail(VKB_ERROR_UNSUPPORTED_OP, "logits: history longer than 2^31 - 1");
    if (r->no_repeat_ngram < 0) fail(VKB_ERROR_INVALID_ARGUMENT, "logits: negative no_repeat_ngram");
    if (r->bias_dev && (r->n_bias <= 0 || (r->n_bias > 1 && r->bias_ld < vocab)))
        fail(VKB_ERROR_INVALID_ARGUMENT, "logits: the bias table needs n_bias >= 1 rows of at least n_vocab values");
    if (r->mask_dev && (r->n_mask <= 0 || (r->n_mask > 1 && r->mask_ld < (vocab + 31) / 32)))
        fail(VKB_ERROR_INVALID_ARGUMENT, "logits: the mask table needs n_mask >= 1 rows of at least ceil(n_vocab / 32) words");
    R.hist = r->hist_ld > 0 ? r->hist_dev : nullptr;
    R.hist_ld = r->hist_ld;
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

constexpr int64_t ROWS_PER_LAUNCH = 32768;  // grid.y, and the arrival counters of a selection

template <typename T, int NV>
void launch_process(vkb_context* ctx, const T* in, int64_t ld, int64_t n_rows, int vocab, const Rules& R0, T* out,
                    int64_t out_ld) {
    using W = Window<T, NV>;
    const unsigned windows = (unsigned)ceil_div((int64_t)vocab + W::N - 1, W::TOKENS);
    const size_t smem = R0.hist ? W::TOKENS * sizeof(uint32_t) : 0;
    for (int64_t r0 = 0; r0 < n_rows; r0 += ROWS_PER_LAUNCH) {
        Rules R = R0;
        if (R.hist) R.hist += r0 * R.hist_ld;
        for (const int32_t** p : {&R.hist_len, &R.bias_row, &R.mask_row})
            if (*p) *p += r0;
        for (const float** p : {&R.rep, &R.freq, &R.pres})
            if (*p) *p += r0;
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
    const size_t smem = R0.hist ? W::TOKENS * sizeof(uint32_t) : 0;
    for (int64_t r0 = 0; r0 < n_rows; r0 += ROWS_PER_LAUNCH) {
        Rules R = R0;
        if (R.hist) R.hist += r0 * R.hist_ld;
        for (const int32_t** p : {&R.hist_len, &R.bias_row, &R.mask_row})
            if (*p) *p += r0;
        for (const float** p : {&R.rep, &R.freq, &R.pres})
            if (*p) *p += r0;
        const int64_t rows = std::min<int64_t>(ROWS_PER_LAUNCH, n_rows - r0);
        // blocks of a row: enough for four on each SM, at most one a window
        const int64_t want = std::max<int64_t>(1, (4 * (int64_t)ctx->sm_count + rows - 1) / rows);
        const int64_t per = (windows + std::min(want, windows) - 1) / std::min(want, windows);
        const int64_t parts = (windows + per - 1) / per;
        uint64_t* part = nullptr;
        float2* part_ms = nullptr;
        if (parts > 1) {
            const size_t cand = (size_t)(rows * parts * k) * sizeof(uint64_t);
            ctx->ensure_workspace(cand + (size_t)(rows * parts) * sizeof(float2));
            part = ctx->workspace.as<uint64_t>();
            part_ms = reinterpret_cast<float2*>(ctx->workspace.as<uint8_t>() + cand);
        }
        launch_pdl(ctx, logits_topk_kernel<T, NV>, dim3((unsigned)parts, (unsigned)rows), LG_THREADS, smem, in + r0 * ld,
                   ld, vocab, R, k, (int)per, part, part_ms, ctx->tile_ctr.as<unsigned>(), ids + r0 * k,
                   logprob + r0 * k);
        VKB_CUDA(cudaGetLastError());
        ctx->count();
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
            launch_process<float, 4>(ctx, reinterpret_cast<const float*>(logits_dev), ld, n_rows, v, R,
                                     reinterpret_cast<float*>(out_dev), out_ld);
        else
            launch_process<__half, 4>(ctx, reinterpret_cast<const __half*>(logits_dev), ld, n_rows, v, R,
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
            launch_topk<float, 4>(ctx, reinterpret_cast<const float*>(logits_dev), ld, n_rows, v, R, k, ids_dev,
                                  logprob_dev);
        else
            launch_topk<__half, 4>(ctx, reinterpret_cast<const __half*>(logits_dev), ld, n_rows, v, R, k, ids_dev,
                                   logprob_dev);
    });
}

}  // extern "C"
