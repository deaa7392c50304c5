// bkv_prompt.cu — attention over the block-scaled 8-bit KV cache for many query
// rows a stream (prompts and chunks of them), 16-bit rows, on the fifth-generation
// tensor cores.
//
// Bound: three things that come to about the same at d_head 128: the products
// (2 x 2 x 256 x 128 x 128 operations a step at 8192 a cycle and SM: 2048 cycles),
// the exponentials (256 x 128 at 16 a cycle: 2048) and the shared memory that
// the products read. So a block keeps two tiles of 128 query rows (of one KV head:
// row = token * group + head) that share each K/V tile of 128 keys, and while one
// tile's softmax runs the other one's products do:
//   warps 0..3, 4..7  softmax of tile 0, 1: thread = row = its own lane of tensor
//                     memory, so a row's maximum and sum need no exchange
//   warps 8..11, 12..14  K, V pages from global memory, int8 -> f16 (exact), into
//                     shared memory with the 128-byte swizzle; V pages are stored
//                     channel by channel, which is the K-major operand of P.V, so
//                     nothing is transposed. The next tile's pages are in
//                     registers while this one is converted.
//   warp 15           issues the products: S = Q K^T from shared memory, O += P V
//                     with P (f16) in tensor memory, in S's own columns. It takes
//                     whichever tile is ready.
// Scales stay in fp32: a block's K scale multiplies its scores in the exponent's
// own multiply-add; its V scale is added to the exponent as a logarithm, so a
// weight comes out scaled at no cost, and the row's sum takes the 16 weights of
// a block times the inverse. The running maximum is that of score and logarithm
// together, over what the row itself sees: a block that it does not see, or whose
// scaled weights are small, takes no bits from the others. It (and O) is raised
// only when a half tile exceeds it by 2^8. Scales below 2^-60 count as 2^-60:
// their values, below 2^-53, are 0 in f16 all the same, and their weights stay
// above fp32's smallest number in the sum.
//
// Measured: 4 prompts of up to 2047 tokens over up to 12000 keys, 8 x 4 heads of
// 128: 680 us, 785 TFLOP/s, 47% of cuBLAS.
#include "bkv_attn.cuh"
#include "tc_ptx.cuh"
#include <algorithm>

namespace vkb {
namespace {

constexpr int ROWS = 256;           // query rows of a block, two tiles of 128
constexpr int KEYS = 128;           // keys of a step
constexpr int PAGES = KEYS / BKV_BLOCK;
constexpr int THREADS = 16 * 32;
constexpr uint32_t TMEM_COLS = 512;
constexpr float L2E = 1.4426950408889634f;
constexpr float RAISE = 8.0f;       // log2
constexpr float UP = 7.0f;          // log2: weights enter f16 times 2^7, below 2^15, and keep their bits down to 2^-21 of the maximum
constexpr float MIN_SCALE = 8.67361738e-19f;  // 2^-60
constexpr uint32_t POLLS = 1u << 24;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct StepScales {
    float k[PAGES];   // K scale * softmax scale * log2(e)
    float lw[PAGES];  // log2 of the V scale; -inf: the page is not there
    float iw[PAGES];  // the inverse of the V scale; 0 where the page is not there
    int missing;      // whether a page is not there
};

template <int D>
struct Smem {
    static constexpr int TILE = KEYS * D * 2;  // a tile of Q, K or V as f16
    static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE, SC = 6 * TILE;
    static constexpr int BARS = SC + 4 * (int)sizeof(StepScales);
    static constexpr int BYTES = 1024 + (BARS + 7) / 8 * 8 + 24 * 8;
};

// Byte offset of the 16-byte chunk `chunk` of row `row` in a block of rows of 128 bytes, swizzled.
__device__ __forceinline__ uint32_t sw128(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// 16 int8 as 16 f16, in order (two chunks).
__device__ __forceinline__ void to_f16(const uint4& v, uint4& a, uint4& b) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[8];
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = w[i] ^ 0x80808080u;
        const uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&lo), bias);
        const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&hi), bias);
        o[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
        o[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
    a = make_uint4(o[0], o[1], o[2], o[3]);
    b = make_uint4(o[4], o[5], o[6], o[7]);
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1) bkv_prompt_kernel(BkvAttn A, int* err) {
    pdl_entry();
    using M = Smem<D>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // The block's row tile: number x of all streams' tiles, found by every warp for itself. Of each 32 streams those with
    // the most keys come first, and of a stream its last tile, which sees the most: long blocks do not start last.
    // 8 prompts of up to 512 tokens, up to 8000 keys: 264 us with the streams as they come, 227.
    const int h = (int)(blockIdx.x % A.L.n_kv_head);
    int x = (int)(blockIdx.x / A.L.n_kv_head), s = -1, first_row = 0, n_q = 0, tile = 0;
    for (int base = 0; base < A.S.n_seq && s < 0; base += 32) {
        const int here = min(32, A.S.n_seq - base);
        int first = 0, n = 0, keys = 0;
        if (lane < here) {
            A.S.rows(base + lane, first, n);
            keys = A.S.keys(base + lane);
        }
        const int mine = (int)(((int64_t)n * A.group + ROWS - 1) / ROWS);
        int sum = mine;
        for (int o = 0; o < here; ++o) {
            const int other = __shfl_sync(0xffffffffu, keys, o), tiles = __shfl_sync(0xffffffffu, mine, o);
            if (other > keys || (other == keys && o < lane)) sum += tiles;
        }
        const unsigned found = __ballot_sync(0xffffffffu, x >= sum - mine && x < sum);
        if (found) {
            const int at = __ffs(found) - 1;
            s = base + at;
            first_row = __shfl_sync(0xffffffffu, first, at);
            n_q = __shfl_sync(0xffffffffu, n, at);
            tile = __shfl_sync(0xffffffffu, sum, at) - 1 - x;
        } else {
            x -= __reduce_add_sync(0xffffffffu, mine);
        }
    }
    if (s < 0) return;
    const int n_rows = n_q * A.group, row0 = tile * ROWS;
    const int n_keys = A.S.keys(s);
    // keys that row r sees: those up to its token's position
    auto limit_of = [&](int r) { return r < n_rows ? max(0, min(n_keys, n_keys - n_q + r / A.group + 1)) : 0; };
    const int n_half = (limit_of(min(n_rows, row0 + ROWS) - 1) + KEYS / 2 - 1) / (KEYS / 2), n_steps = (n_half + 1) / 2;

    extern __shared__ uint8_t raw_smem[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
    StepScales* scales = reinterpret_cast<StepScales*>(smem + M::SC);  // [4]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (M::BARS + 7) / 8 * 8);
    uint64_t *q_full = bars, *k_full = bars + 1, *v_full = bars + 3, *k_empty = bars + 5, *v_empty = bars + 7;
    uint64_t *s_full = bars + 9, *p_full = bars + 13, *pv_done = bars + 17;  // [tile * 2 + half]
    uint64_t* ended = bars + 21;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
    if (threadIdx.x == 0) {
        ptx::mbar_init(q_full, 256);
        ptx::mbar_init(ended, 1);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&k_full[i], 128);
            ptx::mbar_init(&v_full[i], 96);
            ptx::mbar_init(&k_empty[i], 1);
            ptx::mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&p_full[i], 128);
            ptx::mbar_init(&pv_done[i], 1);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 15) {
        ptx::tmem_alloc(tmem_slot, TMEM_COLS);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t S_COL = 0, O_COL = 256;  // S (and P) of tile t at 128 t, O at 256 + D t
    bool ok = true;

    if (warp < 8) {
        // ---- softmax and epilogue: thread = row
        const int t = warp >> 2, quarter = warp & 3;
        const int r = row0 + t * 128 + quarter * 32 + lane;
        const int tok = r / A.group, head = h * A.group + r % A.group;
        const int limit = r < n_rows ? limit_of(r) : INT32_MAX;  // (a row that is not there masks nothing and is not written)
        bool bad;  // the row is NaN
        {
            const __half* q = reinterpret_cast<const __half*>(A.q) + (int64_t)(first_row + tok) * A.q_ld + (int64_t)head * D;
            uint8_t* to = smem + M::Q + t * M::TILE;
            const int row = quarter * 32 + lane;
            uint4 v[D / 8];
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                v[i] = r < n_rows ? __ldcg(reinterpret_cast<const uint4*>(q) + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint4*>(to + (i >> 3) * (128 * 128) + sw128(row, i & 7)) = v[i];
            // A row with an infinity or NaN (exponent bits all 1) that sees a key is NaN, though its scores may all be -inf;
            // one in front of the first key is 0, whatever it holds. (The sum is set behind the loop: in front of it 694 us
            // for four prompts instead of 687.)
            uint32_t odd = 0;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) odd |= ((&v[i].x)[e] & 0x7c007c00u) + 0x04000400u;
            bad = odd & 0x80008000u && limit > 0;
            ptx::fence_proxy_async_smem();
            ptx::mbar_arrive(q_full);
        }
        const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_at = at + S_COL + 128 * t, o_at = at + O_COL + D * t;
        float m = -INFINITY, l = 0.0f;  // running maximum of the scaled weights less UP (log2 units), sum
        for (int i = 0; i < n_half && ok; ++i) {
            const int j = i >> 1, half = i & 1;
            if (!ptx::mbar_wait(&s_full[2 * t + half], j & 1)) { ok = false; break; }
            ptx::tc_fence_after();
            const StepScales& sc = scales[j & 3];
            const int left = limit - i * (KEYS / 2);  // the row sees the half's first `left` keys
            const bool masked = __any_sync(0xffffffffu, left < KEYS / 2) || sc.missing;
            uint32_t v[2][32];  // the row's scores
            ptx::tmem_ld32(s_at + 64 * half, v[0]);
            ptx::tmem_ld32(s_at + 64 * half + 32, v[1]);
            ptx::tmem_ld_wait_for(v[0]);
            ptx::tmem_ld_wait_for(v[1]);
            float mx = -INFINITY;
#pragma unroll
            for (int b = 0; b < PAGES / 2; ++b) {
                uint32_t* x = v[b >> 1] + 16 * (b & 1);
                const int page = half * (PAGES / 2) + b;
                if (masked) {
                    const int n = sc.iw[page] == 0.0f ? 0 : left - 16 * b;  // of the page's tokens the row sees the first n
#pragma unroll
                    for (int c = 0; c < 16; ++c) x[c] = c < n ? x[c] : __float_as_uint(-INFINITY);
                }
                float bm = -INFINITY;
#pragma unroll
                for (int c = 0; c < 16; ++c) bm = fmaxf(bm, __uint_as_float(x[c]));
                mx = fmaxf(mx, fmaf(bm, sc.k[page], sc.lw[page]));
            }
            const bool raise = mx > m + (RAISE + UP);
            const float m_new = raise ? mx - UP : m;
            const float m_use = m_new == -INFINITY ? 0.0f : m_new;
            const float corr = raise ? ex2(m - m_use) : 1.0f;
            if (i > 0 && __any_sync(0xffffffffu, corr != 1.0f)) {
                // O has to be at rest: the last half's P.V is complete
                if (!ptx::mbar_wait(&pv_done[2 * t + ((i - 1) & 1)], ((i - 1) >> 1) & 1)) { ok = false; break; }
                ptx::tc_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < D; c0 += 16) {
                    uint32_t o[16];
                    ptx::tmem_ld16(o_at + c0, o);
                    ptx::tmem_ld_wait_for(o);
#pragma unroll
                    for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
                    ptx::tmem_st16(o_at + c0, o);
                }
            }
            l *= corr;
            m = m_new;
            // P over S, 64 columns of scores (all in registers by now) becoming 32 of f16 pairs
#pragma unroll
            for (int c0 = 0; c0 < 2; ++c0) {
                uint32_t p[16];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint32_t* x = v[c0] + 16 * b;
                    const int page = half * (PAGES / 2) + 2 * c0 + b;
                    const float k = sc.k[page], add = sc.lw[page] - m_use;
                    const float2 k2 = make_float2(k, k), add2 = make_float2(add, add);
                    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        float2 y = __ffma2_rn(make_float2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), k2, add2);
                        y.x = ex2(y.x);
                        y.y = ex2(y.y);
                        sum = __fadd2_rn(sum, y);
                        const __half2 hp = __floats2half2_rn(y.x, y.y);
                        p[8 * b + (c >> 1)] = *reinterpret_cast<const uint32_t*>(&hp);
                    }
                    l = fmaf(sum.x + sum.y, sc.iw[page], l);
                }
                ptx::tmem_st16(s_at + 64 * half + 16 * c0, p);
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            ptx::mbar_arrive(&p_full[2 * t + half]);
        }
        if (ok && n_half > 0 && !ptx::mbar_wait(&pv_done[2 * t + ((n_half - 1) & 1)], ((n_half - 1) >> 1) & 1)) ok = false;
        if (ok) {
            ptx::tc_fence_after();
            if (bad) l = __uint_as_float(0x7fc00000u);
            const float fin = 1.0f / l;
            __half* to = reinterpret_cast<__half*>(A.out) + (int64_t)(first_row + tok) * A.out_ld + (int64_t)head * D;
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t o[32];
                if (n_steps > 0) {
                    ptx::tmem_ld32(o_at + c0, o);
                    ptx::tmem_ld_wait();
                }
                if (r < n_rows) {
                    __align__(16) __half2 y[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        y[c] = l == 0.0f ? __floats2half2_rn(0.0f, 0.0f)
                                         : __floats2half2_rn(__uint_as_float(o[2 * c]) * fin, __uint_as_float(o[2 * c + 1]) * fin);
#pragma unroll
                    for (int c = 0; c < 4; ++c) reinterpret_cast<uint4*>(to + c0)[c] = reinterpret_cast<const uint4*>(y)[c];
                }
            }
        }
    } else if (warp < 15) {
        // ---- warps 8..11: K, 12..14: V, in pieces of 16 bytes; the next step's are in registers while this one's are
        // converted
        const bool is_v = warp >= 12;
        const int tid = threadIdx.x - (is_v ? 384 : 256);
        constexpr int PIECES = PAGES * D;                   // of K or V of a step
        constexpr int NK = PIECES / 128, NV = (PIECES + 95) / 96;
        const int n_pages = (n_keys + BKV_BLOCK - 1) / BKV_BLOCK;
        const int8_t* arena = (is_v ? A.L.v : A.L.k) + (int64_t)h * (BKV_BLOCK * D);
        const int64_t page_bytes = (int64_t)A.L.n_kv_head * (BKV_BLOCK * D);
        auto ids_of = [&](int j) {  // lane i < 8: page i of step j
            const int p = j * PAGES + lane;
            return j < n_steps && lane < PAGES && p < n_pages ? (int)A.S.page(s, p, A.L.n_pages) : -1;
        };
        // K: two neighbouring tokens' four pieces of one 64-channel block lie in eight neighbouring lanes, whose chunks of the
        // swizzled operand are in eight different banks; the lane bits are piece (2), token (1), block (D = 128), token (3)
        constexpr int BLK = D / 64;
        const int k_tok = ((tid >> 2) & 1) | (tid / (8 * BLK) & 7) << 1, k_blk = tid >> 3 & (BLK - 1), k_grp = 4 * k_blk + (tid & 3);
        const int8_t* mine = arena + (is_v ? 0 : k_tok * D + 16 * k_grp);
        uint4 raw[NV];
        auto load = [&](int ids) {  // (a page that is not there reads page 0: its scores are masked)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int piece = min(tid + (is_v ? 96 : 128) * i, PIECES - 1);
                const int id = max(__shfl_sync(0xffffffffu, ids, piece / D), 0);
                if (is_v || i < NK)
                    raw[i] = __ldcg(reinterpret_cast<const uint4*>(mine + id * page_bytes + (is_v ? 16 * (piece % D) : 0)));
            }
        };
        float ks = 0.0f, vs = 0.0f;
        auto load_scales = [&](int id) {
            ks = id >= 0 ? __ldcg(A.L.ks + (int64_t)id * A.L.n_kv_head + h) : 0.0f;
            vs = id >= 0 ? __ldcg(A.L.vs + (int64_t)id * A.L.n_kv_head + h) : 0.0f;
        };
        int ids = ids_of(0), ids_next = ids_of(1);
        load(ids);
        if (warp == 8) load_scales(ids);
        uint64_t *empty = is_v ? v_empty : k_empty, *full = is_v ? v_full : k_full;
        for (int j = 0; j < n_steps && ok; ++j) {
            const int st = j & 1;
            if (!ptx::mbar_wait(&empty[st], ((j >> 1) & 1) ^ 1)) { ok = false; break; }
            if (!is_v) {
                // token = row of the operand, channels in blocks of 64
                const int row = 16 * (tid / D) + k_tok;
                uint8_t* to = smem + M::K + st * M::TILE + k_blk * (KEYS * 128);
                uint8_t* to_a = to + sw128(row, 2 * (tid & 3));
                uint8_t* to_b = to + sw128(row, 2 * (tid & 3) + 1);
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    uint4 a, b;
                    to_f16(raw[i], a, b);
                    *reinterpret_cast<uint4*>(to_a + i * (16 * (128 / D) * 128)) = a;  // whole pages on: the swizzle is the same
                    *reinterpret_cast<uint4*>(to_b + i * (16 * (128 / D) * 128)) = b;
                }
            } else {
                // channel = row of the operand, keys in blocks of 64
                uint8_t* to = smem + M::V + st * M::TILE;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int piece = tid + 96 * i, page = piece / D, ch = piece % D;
                    if (piece >= PIECES) break;
                    uint4 a, b;
                    to_f16(raw[i], a, b);
                    uint8_t* blk = to + (page >> 2) * (D * 128);
                    *reinterpret_cast<uint4*>(blk + sw128(ch, 2 * (page & 3))) = a;
                    *reinterpret_cast<uint4*>(blk + sw128(ch, 2 * (page & 3) + 1)) = b;
                }
            }
            if (warp == 8) {
                // (scales[j & 3] was last read for step j - 4, which ended before K's buffer of step j - 2 came free)
                StepScales& sc = scales[j & 3];
                const unsigned there = __ballot_sync(0xffffffffu, ids >= 0);
                if (lane < PAGES) {
                    const float w = fmaxf(vs, MIN_SCALE);
                    sc.k[lane] = fmaxf(ks * (A.scale * L2E), 1e-37f);  // above 0: a masked -inf stays -inf
                    sc.lw[lane] = ids >= 0 ? log2f(w) : -INFINITY;
                    sc.iw[lane] = ids >= 0 ? 1.0f / w : 0.0f;
                }
                const int valid = min(PAGES, n_pages - j * PAGES);
                if (lane == 0) sc.missing = (there & ((1u << valid) - 1)) != (1u << valid) - 1;
                __syncwarp();
            }
            ptx::fence_proxy_async_smem();
            ptx::mbar_arrive(&full[st]);
            ids = ids_next;
            if (j + 1 < n_steps) {
                load(ids);
                if (warp == 8) load_scales(ids);
            }
            ids_next = ids_of(j + 2);
        }
    } else if (n_steps > 0) {
        // ---- the products, by the whole warp in step. Half i of a tile's keys has its scores in half i % 2 of the tile's
        // columns, so S of the next half is made while this one's softmax runs. Tile t is at S of half s_at[t] and P.V of
        // half pv_at[t]
        constexpr uint32_t idesc_s = ptx::idesc_f16_f32(128, KEYS / 2), idesc_o = ptx::idesc_f16_f32(128, D);
        const uint64_t q_desc = ptx::sdesc_sw128(ptx::smem_u32(smem + M::Q)), k_desc = ptx::sdesc_sw128(ptx::smem_u32(smem + M::K)),
                       v_desc = ptx::sdesc_sw128(ptx::smem_u32(smem + M::V));  // + bytes / 16: another place
        auto ready = [&](uint64_t* bar, uint32_t parity) { return __any_sync(0xffffffffu, ptx::mbar_test(bar, parity)) != 0; };
        int s_at[2] = {0, 0}, pv_at[2] = {0, 0};
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(q_full, 0));
        uint32_t polls = 0;
        while (ok && (pv_at[0] < n_half || pv_at[1] < n_half)) {
            bool moved = false;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (pv_at[t] < s_at[t]) {
                    const int i = pv_at[t], half = i & 1, st = (i >> 1) & 1;
                    if (ready(&p_full[2 * t + half], (i >> 1) & 1) && ready(&v_full[st], (i >> 2) & 1)) {
                        ptx::tc_fence_after();
                        const uint64_t b = v_desc + (st * M::TILE + half * (D * 128)) / 16;
#pragma unroll
                        for (int kk = 0; kk < KEYS / 32; ++kk)
                            ptx::mma_f16_ts_warp(tmem + O_COL + D * t, tmem + S_COL + 128 * t + 64 * half + kk * 8, b + kk * 32 / 16,
                                                 idesc_o, (i > 0 || kk > 0) ? 1u : 0u);
                        ptx::mma_commit_warp(&pv_done[2 * t + half]);
                        ++pv_at[t];
                        if (half && pv_at[t ^ 1] > i) ptx::mma_commit_warp(&v_empty[st]);
                        moved = true;
                    }
                }
                if (s_at[t] < n_half) {
                    const int i = s_at[t], half = i & 1, st = (i >> 1) & 1;
                    // the columns held P of half i - 2: that P.V must be complete
                    if (ready(&k_full[st], (i >> 2) & 1) && (i < 2 || (pv_at[t] > i - 2 && ready(&pv_done[2 * t + half], ((i >> 1) - 1) & 1)))) {
                        ptx::tc_fence_after();
                        const uint64_t a = q_desc + t * (M::TILE / 16), b = k_desc + (st * M::TILE + half * (KEYS / 2 * 128)) / 16;
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            ptx::mma_f16_ss_warp(tmem + S_COL + 128 * t + 64 * half, a + ((kk >> 2) * (128 * 128) + (kk & 3) * 32) / 16,
                                                 b + ((kk >> 2) * (KEYS * 128) + (kk & 3) * 32) / 16, idesc_s, kk > 0 ? 1u : 0u);
                        ptx::mma_commit_warp(&s_full[2 * t + half]);
                        ++s_at[t];
                        if (half && s_at[t ^ 1] > i) ptx::mma_commit_warp(&k_empty[st]);
                        moved = true;
                    }
                }
            }
            if (moved) {
                polls = 0;
            } else {
                __nanosleep(20);
                if (++polls == POLLS) ok = false;
            }
        }
    }
    if (!ok) atomicExch(err, 1);
    __syncwarp();
    if (warp == 15) {
        // The last commit of all: products and arrivals (the last steps' buffers are given back to nobody) that are under
        // way, where a wait gave up too, end before the block does.
        ptx::mma_commit_warp(ended);
        ptx::mbar_wait(ended, 0);
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 15) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, TMEM_COLS);
    }
}

int64_t most_tiles(const BkvAttn& a) { return (int64_t)a.S.n_tok * a.group / ROWS + a.S.n_seq; }

template <int D>
void launch(vkb_context* ctx, const BkvAttn& a) {
    auto kern = bkv_prompt_kernel<D>;
    static_assert(Smem<D>::BYTES <= 227 * 1024, "shared memory of one block");
    smem_optin(kern, Smem<D>::BYTES);
    // (at most) as many row tiles: the rows of all streams, and one begun tile for each
    const int64_t blocks = most_tiles(a) * a.L.n_kv_head;
    if (blocks > INT32_MAX) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv_attention: too many rows");
    launch_pdl(ctx, kern, dim3((unsigned)blocks), THREADS, Smem<D>::BYTES, a, ctx->err_flag.as<int>());
    VKB_CUDA(cudaGetLastError());
    ctx->count();
}

}  // namespace

bool bkv_prompt_takes(const vkb_context* ctx, const BkvAttn& a) {
    if (!a.q_f16 || !a.out_f16 || (a.d_head != 64 && a.d_head != 128)) return false;
    if ((uintptr_t)a.q % 16 || (uintptr_t)a.out % 16 || a.q_ld % 8 || a.out_ld % 8) return false;
    // A wave of these blocks takes the time of its longest stream whatever the rows. The other kernel's time grows with the
    // rows, by tiles of 16 (all heads), and has a fixed part that counts with few keys: what this one needs to be the faster
    // is tiles for each of its waves, more of them the more keys there are, up to as many as make the two grow alike.
    // Microseconds here and there, one stream, group 4, 8 KV heads:
    //   d_head 128, 1000 keys:  128 tiles 35 and 33, 256 tiles 35 and 41
    //               2000        256 tiles 55 and 51, 512 tiles 55 and 76
    //               4000        256 tiles 96 and 74, 512 tiles 95 and 117
    //               64000       256 tiles 1294 and 659, 512 tiles 1292 and 1295, 1024 tiles 1294 and 2534
    //   d_head 64,  1000        128 tiles 29 and 28, 256 tiles 30 and 33
    //               4000        512 tiles 82 and 80, 1024 tiles 84 and 131
    //               64000       512 tiles 1146 and 780, 1024 tiles 1147 and 1518
    // Up to 512 keys: 500 keys, 16 rows 16 and 20; 64 rows 20 and 20. Where the longest stream is not known the table's
    // width stands for it, which matters below the upper limit only (1.7 times the time at worst: 1000 keys).
    if ((int64_t)a.max_q * a.group < 64) return false;
    const int64_t pages = a.max_kv > 0 ? std::min<int64_t>(a.S.ld, ((int64_t)a.max_kv + BKV_BLOCK - 1) / BKV_BLOCK) : a.S.ld;
    if (pages <= 32) return true;
    const int64_t blocks = most_tiles(a) * a.L.n_kv_head, waves = (blocks + ctx->sm_count - 1) / ctx->sm_count;
    const int64_t tiles = ((int64_t)a.S.n_tok * a.group + 15) / 16 * a.L.n_kv_head;
    return tiles >= waves * (a.d_head == 64 ? std::min<int64_t>(4 * pages, 768) : std::min<int64_t>(2 * pages, 512));
}

void run_bkv_prompt(vkb_context* ctx, const BkvAttn& a) {
    if (a.d_head == 64) launch<64>(ctx, a);
    else launch<128>(ctx, a);
}

}  // namespace vkb
