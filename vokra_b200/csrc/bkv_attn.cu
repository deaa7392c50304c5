// bkv_attn.cu — attention over the block-scaled 8-bit KV cache for few query
// rows a stream: decode steps, tokens to check, short chunks.
//
// Bound: HBM (2 d_head bytes a key and KV head). A warp takes 64 keys = 4 pages
// at a time from a ring of its own in shared memory, filled by bulk copies that
// run ahead over the ends of its items; pages are contiguous, and neither K nor
// V is ever transposed or shuffled. What makes that work is that the order of
// keys and channels inside a matrix product is free as long as both operands
// agree:
//  - lane (g, c) = (lane / 4, lane % 4). Column n of score tile t is token
//    2t + n % 2 of page n / 2, so that lane c's columns (2c, 2c + 1) of all 8
//    tiles are the 16 tokens of page c: one K scale and one V scale a lane.
//  - a lane reads 16 neighbouring channels of a K row: two k steps (m16n8k32,
//    int8) of Q.K. q is made int8 planes in the same order: p1 + p2 / 254 (+
//    p3 / 254^2) units of 1/127 of the row's largest. The products are exact
//    in 32-bit integers; two planes hold q to 2^-16 of that largest, three to
//    2^-24. K is never converted, which was a third of the instructions.
//  - V is stored channel by channel, so 16 bytes of (page c, channel 8i + g) are
//    the 16 tokens whose weights the lane holds: four k steps of P.V (m16n8k16).
//    int8 -> f16 is exact (a byte permute into 1024 + u, minus 1152). The V scale
//    multiplies the weights in fp32; they enter divided by the row's `frame`, a
//    power of two near the row's largest product of weight and V scale so far, so
//    that f16 holds what counts whatever the scales, and times 2^14, so that a
//    weight keeps its bits down to 2^-28 of the row's largest. The frame falls with the weights when
//    the row's maximum rises, and blocks that the row does not see are no part of it.
//
// Tiles of 8 query rows (SPLIT) hold p1 in rows 0..7 of the 16-row operand and
// p2 in rows 8..15, likewise the high and low f16 parts of the weights: 2^-21
// at the price of one product. 32-bit rows take the third plane in a second
// one. Tiles of 16 rows (16-bit rows, more than 8 a stream and KV head) take
// two products for the planes and one f16 part of the weights.
//
// Measured: 64 streams of up to 448 keys, 20 heads of 64, f32, 28.9 us; one stream
// of 131071 keys, 8 x 4 heads of 128, f16, 59 us (4.6 TB/s); 48 streams of up to
// 8191 keys with up to 4 rows, 8 x 4 heads of 128, f16, 100 us (4.2 TB/s).
//
// The (stream, KV head, row tile, 64 keys) steps of the whole call are one
// sequence, cut into equal contiguous shares for the blocks and their warps, so
// ragged lengths balance themselves (an item counts a few steps more than it has,
// for its query rows and its join). A warp finishes an item that lies in its
// share alone; parts of shared items are joined in order, first within the
// block, then by the last block of the item to arrive.
#include "bkv_attn.cuh"
#include "tc_ptx.cuh"
#include <algorithm>
#include <cfloat>

namespace vkb {
namespace {

constexpr int BKV_SEQ_PER_LAUNCH = 512;
constexpr float W_UP = 16384.0f;  // weights over the frame are below 2, their f16 forms below 2^15
constexpr float MIN_FRAME = FLT_MIN * W_UP;
constexpr float L2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four values y (in units of 1/127 of the row's largest) as int8 words: the nearest whole numbers, then 254 times
// what they leave, and so on; y becomes what is left behind the word, times 254.
__device__ __forceinline__ uint32_t take_plane(float (&y)[4]) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int q = __float2int_rn(y[e]);
        w |= (uint32_t)(q & 0xff) << (8 * e);
        y[e] = (y[e] - (float)q) * 254.0f;
    }
    return w;
}

// Four int8 (one word) as two f16 pairs: bytes 0, 1 and bytes 2, 3.
__device__ __forceinline__ void s8x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias), y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// What the f16 pair leaves of (a, b), as an f16 pair.
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pack_f16(a - h.x, b - h.y);
}

struct AttnArgs : BkvAttn {
    int q_vec, out_vec;
    float* warp_o;    // [blocks * AW][2][rows][D]: a warp's parts of items that it shares with others
    float2* warp_ml;  // [blocks * AW][2][rows]: their maximum and sum; the part's rows are divided by that sum
    float* block_o;   // [blocks][2][rows][D]: the same of a block
    float2* block_ml;
    unsigned* arrived;  // [blocks], 0 at rest: blocks that have left their part of the item that starts in block i
    int* err;
};

// What a block knows of the streams: the running number of steps in front of
// each (pre[n_seq] is the total), keys, first row.
struct Streams {
    int64_t pre[BKV_SEQ_PER_LAUNCH + 1];
    int keys[BKV_SEQ_PER_LAUNCH];
    int first[BKV_SEQ_PER_LAUNCH];
    int n_q[BKV_SEQ_PER_LAUNCH];
    int extra;  // steps that an item counts for beside its own
};

template <int D>
struct Ring {
    // Warps of a block, one block an SM, and the ring's slots of each. 64 streams of up to 448 keys, 20 heads of 64:
    // 12 warps x 4 slots 29.3 us, 16 x 3 34.8 (spills), 8 x 5 33.2; one stream of 131071 keys, 8 heads of 128: 8 x 3
    // 73 us, 10 x 2 93, 12 x 2 81 (before the int8 scores).
    static constexpr int AW = D <= 64 ? 12 : D <= 128 ? 8 : 4;
    static constexpr int PAGE = BKV_BLOCK * D;
    static constexpr int STRIDE = PAGE + 32;    // pages of a slot: the 32 bytes spread a quad's V loads over the banks
    static constexpr int SLOT = 4 * STRIDE;     // the K or the V of 64 keys
    static constexpr int SLOTS = D <= 64 ? 4 : 3;
    static constexpr int META = 8;
    static constexpr int WARP = SLOTS * SLOT + META * 4 * (int)sizeof(int) + SLOTS * (int)sizeof(uint64_t) + 8;
    static constexpr int WARP_BYTES = (WARP + 15) / 16 * 16;
};

template <int TR, int AW>
__device__ __forceinline__ void load_streams(const AttnArgs& A, Streams& st, int extra) {
    __shared__ int64_t sums[AW];
    const int n = A.S.n_seq, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t carry = 0;
    if (threadIdx.x == 0) {
        st.pre[0] = 0;
        st.extra = extra;
    }
    for (int base = 0; base < n; base += 32 * AW) {
        const int s = base + (int)threadIdx.x;
        int64_t x = 0;
        if (s < n) {
            int first, rows;
            A.S.rows(s, first, rows);
            const int keys = A.S.keys(s);
            st.keys[s] = keys;
            st.first[s] = first;
            st.n_q[s] = rows;
            x = (int64_t)A.L.n_kv_head * ((rows * A.group + TR - 1) / TR) * (max(1, (keys + 63) / 64) + extra);
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        int64_t all = 0;
#pragma unroll
        for (int w = 0; w < AW; ++w) {
            if (w < warp) x += sums[w];
            all += sums[w];
        }
        if (s < n) st.pre[s + 1] = carry + x;
        carry += all;
        __syncthreads();
    }
}

// A place in the sequence of steps (stream, KV head, row tile, 64 keys).
template <int TR>
struct Walk {
    int64_t u;      // the step
    int s, h, tile, ch;
    int tiles, chunks;
    int seen;       // steps of the item in which some row sees a key

    __device__ __forceinline__ void stream(const AttnArgs& A, const Streams& st) {
        tiles = (st.n_q[s] * A.group + TR - 1) / TR;
        chunks = max(1, (st.keys[s] + 63) / 64) + st.extra;
    }
    __device__ __forceinline__ void item(const AttnArgs& A, const Streams& st) {
        const int last_tok = min(st.n_q[s] * A.group, (tile + 1) * TR) - 1;
        const int keys = max(0, st.keys[s] - st.n_q[s] + last_tok / A.group + 1);
        seen = (keys + 63) / 64;
    }
    __device__ __forceinline__ void seek(const AttnArgs& A, const Streams& st, int64_t to) {
        u = to;
        int lo = 0, hi = A.S.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (st.pre[mid] <= to) lo = mid;
            else hi = mid - 1;
        }
        s = lo;
        while (st.pre[s + 1] <= to) ++s;
        stream(A, st);
        const int64_t in_seq = to - st.pre[s];
        const int64_t i = in_seq >> 32 ? in_seq / chunks : (uint32_t)in_seq / (uint32_t)chunks;
        ch = (int)(in_seq - i * chunks);
        h = (int)(i >> 32 ? i / tiles : (uint32_t)i / (uint32_t)tiles);
        tile = (int)(i - (int64_t)h * tiles);
        item(A, st);
    }
    // On to the item's next step, or (past its end) to the next item, if there is one before `end`.
    __device__ __forceinline__ void next_item(const AttnArgs& A, const Streams& st, int64_t end) {
        ch = 0;
        if (++tile == tiles) {
            tile = 0;
            if (++h == A.L.n_kv_head) {
                h = 0;
                if (u < end) {
                    ++s;
                    while (st.pre[s + 1] <= u) ++s;
                    stream(A, st);
                }
            }
        }
        item(A, st);
    }
    // The next step that has keys to load; false: none before `end`.
    __device__ __forceinline__ bool to_loaded(const AttnArgs& A, const Streams& st, int64_t end) {
        while (u < end && ch >= seen) {
            u += chunks - ch;
            next_item(A, st, end);
        }
        return u < end;
    }
    __device__ __forceinline__ void step(const AttnArgs& A, const Streams& st, int64_t end) {
        ++u;
        if (++ch == chunks) next_item(A, st, end);
    }
};

// A part of an item that several warps share.
struct Part {
    int64_t u0;  // the item's first step
    int chunks;  // its steps; 0: no part
    int s, h, tile;
    int head;    // the first one of its item in the block
};

__device__ __forceinline__ void store_pair(const AttnArgs& A, int64_t at, float y0, float y1) {
    if (A.out_f16) {
        __half* p = reinterpret_cast<__half*>(A.out) + at;
        if (A.out_vec) {
            *reinterpret_cast<__half2*>(p) = __floats2half2_rn(y0, y1);
        } else {
            p[0] = __float2half_rn(y0);
            p[1] = __float2half_rn(y1);
        }
    } else {
        float* p = reinterpret_cast<float*>(A.out) + at;
        if (A.out_vec) {
            *reinterpret_cast<float2*>(p) = make_float2(y0, y1);
        } else {
            p[0] = y0;
            p[1] = y1;
        }
    }
}

// Joins rows r and (if it is not negative) r2 of `n` parts, in order, a warp for both at once: their loads are one round
// trip. Part i's rows are o(i) and their (max, sum) ml(i). To the output, or (to_o) to another part. The parts are averages,
// and `share`, a power of two at or below 1 / keys, keeps their sum one: it holds whatever fp32 values V has.
template <int D, class FO, class FM>
__device__ __forceinline__ void join_rows(const AttnArgs& A, int n, int r, int r2, int64_t row_at, int tile_row0, int h, float share,
                                          FO o, FM ml, float* to_o, float2* to_ml) {
    const int lane = threadIdx.x & 31;
    constexpr int C = D / 32;  // channels of a lane, as pairs 64 apart (one alone for D = 32, three for D = 96)
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, y[2][C];
#pragma unroll
    for (int i = 0; i < 2 * C; ++i) y[i / C][i % C] = 0.0f;
    auto ch = [&](int i) { return C == 1 ? lane : C % 2 ? lane + 32 * i : 64 * (i / 2) + 2 * lane + i % 2; };
    // parts at a time: 2, 4, 8: 48 ragged streams 121, 123, 128 us; one of 131071 keys 60.9, 58.0, 58.7
    constexpr int U = C <= 4 ? 4 : 2;
    for (int p0 = 0; p0 < n; p0 += U) {
        float2 x[2][U];
        float v[2][U][C];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int p = 0; p < U; ++p) {
                const bool real = p0 + p < n && (k == 0 || r2 >= 0);
                const int rk = real && k ? r2 : r;
                x[k][p] = real ? __ldcg(ml(p0 + p) + rk) : make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int i = 0; i < C; ++i) v[k][p][i] = 0.0f;
                if (real) {
                    const float* row = o(p0 + p) + rk * D;
#pragma unroll
                    for (int i = 0; i < C; i += C % 2 ? 1 : 2) {
                        if constexpr (C % 2) {
                            v[k][p][i] = __ldcg(row + ch(i));
                        } else {
                            const float2 f = __ldcg(reinterpret_cast<const float2*>(row + ch(i)));
                            v[k][p][i] = f.x;
                            v[k][p][i + 1] = f.y;
                        }
                    }
                }
            }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int p = 0; p < U; ++p) {
                const float m_new = fmaxf(m[k], x[k][p].x);
                const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                const float a = ex2(m[k] - m_use), b = ex2(x[k][p].x - m_use);
                const float lb = x[k][p].y * b, part = lb * share;
                l[k] = l[k] * a + lb;
#pragma unroll
                for (int i = 0; i < C; ++i) y[k][i] = y[k][i] * a + v[k][p][i] * part;
                m[k] = m_new;
            }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int rk = k ? r2 : r;
        if (rk < 0) continue;
        const float inv = l[k] == 0.0f ? 0.0f : 1.0f / (l[k] * share);
        if (to_o) {
#pragma unroll
            for (int i = 0; i < C; ++i) to_o[rk * D + ch(i)] = y[k][i] * inv;
            if (lane == 0) to_ml[rk] = make_float2(m[k], l[k]);
        } else {
            const int row = tile_row0 + rk, tok = row / A.group, head = h * A.group + row % A.group;
            const int64_t at = (row_at + tok) * A.out_ld + (int64_t)head * D;
#pragma unroll
            for (int i = 0; i < C; i += C % 2 ? 1 : 2) {
                if constexpr (C % 2) {
                    if (A.out_f16) reinterpret_cast<__half*>(A.out)[at + ch(i)] = __float2half_rn(y[k][i] * inv);
                    else reinterpret_cast<float*>(A.out)[at + ch(i)] = y[k][i] * inv;
                } else {
                    store_pair(A, at + ch(i), y[k][i] * inv, y[k][i + 1] * inv);
                }
            }
        }
    }
}

template <int D, bool SPLIT, bool P3>
__global__ void __launch_bounds__(32 * Ring<D>::AW, 1) bkv_attn_kernel(AttnArgs A) {
    pdl_entry();
    constexpr int TR = SPLIT ? 8 : 16;       // query rows of a tile
    constexpr int NR = SPLIT ? 1 : 2;        // of them in this lane's hands
    constexpr int KW = D / 16;               // 32-bit words of a K row a lane holds = k steps of Q.K
    constexpr int NT = D / 8;                // channel tiles of P.V
    using R = Ring<D>;
    constexpr int AW = R::AW;
    constexpr int EXTRA = SPLIT ? 1 : 3;
    extern __shared__ __align__(16) uint8_t smem[];
    Streams& st = *reinterpret_cast<Streams*>(smem);
    __shared__ Part parts[2 * AW];
    __shared__ int last_one[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    uint8_t* mine = smem + (sizeof(Streams) + 15) / 16 * 16 + (size_t)warp * R::WARP_BYTES;
    int* meta = reinterpret_cast<int*>(mine + R::SLOTS * R::SLOT);  // [META][4] ids of a step's pages
    uint64_t* full = reinterpret_cast<uint64_t*>(meta + R::META * 4);
    if (lane == 0) {
        for (int i = 0; i < R::SLOTS; ++i) ptx::mbar_init(&full[i], 1);
        ptx::fence_mbar_init();
    }
    if (lane < 2) parts[2 * warp + lane].chunks = 0;
    load_streams<TR, AW>(A, st, 0);
    __syncthreads();
    // An item costs its query rows and its join too, as much as EXTRA steps. They are counted, behind its own steps, once
    // there is a step for every warp; else short items gather in a few blocks. 48 ragged streams of up to 8191 keys, 16
    // rows: 124 us without them (one block 250 thousand cycles, the others 150 to 210), 97 with 2 to 4; 256 streams of up
    // to 448 keys, 8 rows: 80 us without, 62 with one, 64 with two. From two steps a warp on: 64 streams of up to 448 keys
    // 28.8 -> 27.6, from one on also 8 streams of up to 2000 keys 19.6 -> 17.2.
    if (st.pre[A.S.n_seq] >= (int64_t)AW * gridDim.x) {
        __syncthreads();
        load_streams<TR, AW>(A, st, EXTRA);
        __syncthreads();
    }
    const int64_t total = st.pre[A.S.n_seq];
    // Equal shares for the blocks and their warps. Few steps go to as many blocks, a warp in each, not to the warps of
    // few blocks: 5 streams of up to 100 keys, 20 heads of 64, 12.0 us instead of 15.9; one of up to 1000 keys, 8 heads
    // of 128, 13.3 instead of 18.0.
    const int64_t n_block = min((int64_t)gridDim.x, total);
    if (blockIdx.x >= n_block) return;
    const int64_t block_begin = blockIdx.x * total / n_block, block_end = (blockIdx.x + 1) * total / n_block;
    // warps without a step are the block's last ones: an item's warps follow one another
    const int64_t share = (block_end - block_begin) / AW;
    const int rest = (int)((block_end - block_begin) % AW);
    const int64_t u_begin = block_begin + warp * share + min(warp, rest), u_end = u_begin + share + (warp < rest ? 1 : 0);
    bool ok = true;

    if (u_begin < u_end) {
        // ---- the loads run ahead of the products by R::SLOTS halves of a step, over the ends of items
        Walk<TR> ld;
        ld.seek(A, st, u_begin);
        Walk<TR> w = ld;
        bool more = ld.to_loaded(A, st, u_end);
        int ids = -1, ids_s = -1, ids_b = 0;  // lane i: page 32 * ids_b + i of stream ids_s
        int page = -1;
        int op = 0;  // the next half step to load: even K, odd V
        int h_now = 0;
        auto issue = [&]() {
            const int slot = op % R::SLOTS;
            if (!(op & 1)) {
                if (!more) return;
                if (ld.s != ids_s || ld.ch >> 3 != ids_b) {
                    ids_s = ld.s;
                    ids_b = ld.ch >> 3;
                    const int p = 32 * ids_b + lane;
                    ids = p < (st.keys[ids_s] + BKV_BLOCK - 1) / BKV_BLOCK ? (int)A.S.page(ids_s, p, A.L.n_pages) : -1;
                }
                page = __shfl_sync(0xffffffffu, ids, 4 * (ld.ch & 7) + c);
                h_now = ld.h;
                if (lane < 4) meta[((op >> 1) & (R::META - 1)) * 4 + lane] = page;
                else page = -1;
                ld.step(A, st, u_end);
                more = ld.to_loaded(A, st, u_end);
            }
            const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) ptx::mbar_expect_tx(&full[slot], (uint32_t)__popc(there) * R::PAGE);
            __syncwarp();
            if (page >= 0) {
                const int64_t at = ((int64_t)page * A.L.n_kv_head + h_now) * R::PAGE;
                ptx::bulk_load(mine + slot * R::SLOT + lane * R::STRIDE, (op & 1 ? A.L.v : A.L.k) + at, R::PAGE, &full[slot]);
            }
            ++op;
        };
#pragma unroll 1
        for (int i = 0; i < R::SLOTS; ++i) issue();
        int done = 0;  // half steps consumed

        while (w.u < u_end && ok) {
            const int s = w.s, h = w.h, tile = w.tile, chunks = w.chunks, c0 = w.ch;
            const int64_t u0 = w.u - c0;
            const int c1 = (int)min((int64_t)chunks, c0 + (u_end - w.u));
            const int n_keys = st.keys[s], n_q = st.n_q[s], first_row = st.first[s];
            const int c_last = min(c1, w.seen);

            // ---- the tile's query rows as int8 planes, in the order of the K loads
            uint32_t qa[KW / 2][4];
            uint32_t qb[KW / 2][SPLIT ? 2 : 4];  // the third plane (SPLIT, 32-bit rows), or the second one of 16 rows
            float row_fac[NR];  // multiplies a score: scale * log2(e) * the units of the planes
            float row_down = 1.0f;  // so does this (a row of 32 bits: a tile has one a lane)
            int limit[NR];      // keys that the row sees
            if (c0 < c_last)
#pragma unroll
            for (int half_row = 0; half_row < NR; ++half_row) {
                const int r = tile * TR + half_row * 8 + g;
                const int tok = r / A.group, head = h * A.group + r % A.group;
                const bool real = tok < n_q;
                // word i of the lane: 4 channels of the 64-channel part i / 4 (or of what is left behind them)
                auto channel = [&](int i) { return 64 * (i >> 2) + 4 * ((i >> 2) < KW / 4 ? 4 : KW & 3) * c + 4 * (i & 3); };
                const int64_t at = (int64_t)(first_row + (real ? tok : 0)) * A.q_ld + (int64_t)head * D;
                float x[KW][4];
                if (A.q_f16) {
                    const __half* p = reinterpret_cast<const __half*>(A.q) + at;
                    if (A.q_vec) {
                        uint2 v[KW];
#pragma unroll
                        for (int i = 0; i < KW; ++i) v[i] = __ldcg(reinterpret_cast<const uint2*>(p + channel(i)));
#pragma unroll
                        for (int i = 0; i < KW; ++i) {
                            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&v[i].x));
                            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&v[i].y));
                            x[i][0] = f0.x;
                            x[i][1] = f0.y;
                            x[i][2] = f1.x;
                            x[i][3] = f1.y;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < KW; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[i][e] = __half2float(p[channel(i) + e]);
                    }
                } else {
                    const float* p = reinterpret_cast<const float*>(A.q) + at;
                    if (A.q_vec) {
#pragma unroll
                        for (int i = 0; i < KW; ++i) {
                            const float4 v = __ldcg(reinterpret_cast<const float4*>(p + channel(i)));
                            x[i][0] = v.x;
                            x[i][1] = v.y;
                            x[i][2] = v.z;
                            x[i][3] = v.w;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < KW; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[i][e] = p[channel(i) + e];
                    }
                }
                float amax = 0.0f;
                bool number = true;
#pragma unroll
                for (int i = 0; i < KW; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        amax = fmaxf(amax, fabsf(x[i][e]));
                        number &= x[i][e] == x[i][e];
                    }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                number = (__ballot_sync(0xffffffffu, number) >> (4 * g) & 15) == 15;
                // Small rows (of 32 bits) are taken times 2^64: their scores need not be small, for K reaches FLT_MAX.
                if constexpr (P3) {
                    const bool small = amax < 0x1p-60f;
                    row_down = small ? 0x1p-64f : 1.0f;
                    if (small) {
                        amax *= 0x1p64f;
#pragma unroll
                        for (int i = 0; i < KW; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[i][e] *= 0x1p64f;
                    }
                }
                // planes: q = amax / 127 * (p1 + p2 / 254 + p3 / 254^2). Two of them hold it to 2^-16 of the row's
                // largest, three to 2^-24.
                const float unit = amax > 0.0f ? 127.0f / amax : 0.0f;
                limit[half_row] = real ? max(0, min(n_keys, n_keys - n_q + tok + 1)) : 0;
                row_fac[half_row] = amax * (1.0f / (127.0f * (P3 ? 64516.0f : 254.0f))) * (A.scale * L2E);
                // NaN where q has an infinity or NaN; a row in front of the first key is 0, whatever it holds
                if (!(number && amax < INFINITY)) row_fac[half_row] = limit[half_row] > 0 ? __uint_as_float(0x7fc00000u) : 0.0f;
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    float y[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = x[i][e] * unit;
                    const uint32_t p1 = take_plane(y), p2 = take_plane(y);
                    const int a = 2 * (i & 1);
                    if constexpr (SPLIT) {
                        qa[i / 2][a] = p1;
                        qa[i / 2][a + 1] = p2;
                        qb[i / 2][i & 1] = P3 ? take_plane(y) : 0;
                    } else {
                        qa[i / 2][a + half_row] = p1;
                        qb[i / 2][a + half_row] = p2;
                    }
                }
            }

            float m[NR], l[NR];
            float o[NT][4];
            float frame[NR];  // O is in units of frame / W_UP
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                m[i] = -INFINITY;
                l[i] = 0.0f;
                frame[i] = MIN_FRAME;
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;

            for (int ch = c0; ch < c_last; ++ch) {
                // ---- scores
                int slot = done % R::SLOTS;
                if (!ptx::mbar_wait(&full[slot], (done / R::SLOTS) & 1)) {
                    ok = false;
                    break;
                }
                const int id = meta[((done >> 1) & (R::META - 1)) * 4 + c];  // this lane's page
                const bool there = id >= 0;
                float ks = 0.0f, vs = 0.0f;
                if (there) {
                    const int64_t at = (int64_t)id * A.L.n_kv_head + h;
                    ks = __ldcg(A.L.ks + at);
                    vs = __ldcg(A.L.vs + at);
                }
                const uint8_t* kp = mine + slot * R::SLOT + (g >> 1) * R::STRIDE + (g & 1) * D;
                int sc[8][4], sd[8][P3 || !SPLIT ? 4 : 1];
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[t][e] = 0;
                        if constexpr (P3 || !SPLIT) sd[t][e] = 0;
                    }
                // four tiles side by side, so that independent products are under way
#pragma unroll
                for (int t0 = 0; t0 < 8; t0 += 4)
#pragma unroll
                    for (int part = 0; part < (KW + 3) / 4; ++part) {
                        uint32_t kw[4][4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const uint8_t* at = kp + 2 * (t0 + t) * D + 64 * part;
                            if (part < KW / 4) {
                                const uint4 v4 = *reinterpret_cast<const uint4*>(at + 16 * c);
                                kw[t][0] = v4.x;
                                kw[t][1] = v4.y;
                                kw[t][2] = v4.z;
                                kw[t][3] = v4.w;
                            } else {
                                const uint2 v2 = *reinterpret_cast<const uint2*>(at + 8 * c);
                                kw[t][0] = v2.x;
                                kw[t][1] = v2.y;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < (part < KW / 4 ? 2 : 1); ++i)
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const uint32_t* qf = qa[2 * part + i];
                                const uint32_t* qg = qb[2 * part + i];
                                mma16832(sc[t0 + t], qf[0], qf[1], qf[2], qf[3], kw[t][2 * i], kw[t][2 * i + 1]);
                                if constexpr (!SPLIT) mma16832(sd[t0 + t], qg[0], qg[1], qg[2], qg[3], kw[t][2 * i], kw[t][2 * i + 1]);
                                else if constexpr (P3) mma16832(sd[t0 + t], qg[0], 0, qg[1], 0, kw[t][2 * i], kw[t][2 * i + 1]);
                            }
                    }
                __syncwarp();
                ++done;
                issue();  // into the slot that has just been read

                // ---- softmax step. Lane c holds tokens 0..15 of page 4 ch + c: x[row][token]
                const int key0 = 64 * ch + 16 * c;
                float w_scale[NR];
                float corr_o[NR];
                float x[NR][16];
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    float f = ks * row_fac[i];
                    if constexpr (P3) f *= row_down;
                    if (f < 1e-37f) f = 1e-37f;  // above 0: a masked token's -inf stays -inf (and NaN stays NaN)
                    float mx = -INFINITY;
#pragma unroll
                    for (int t = 0; t < 8; ++t)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            // |p1 . k| <= 127 * 127 * 256: 254 of them fit 32 bits
                            float y;
                            if constexpr (!SPLIT) y = (float)(sc[t][2 * i + e] * 254 + sd[t][2 * i + e]);
                            else if constexpr (P3) y = fmaf((float)(sc[t][e] * 254 + sc[t][2 + e]), 254.0f, (float)sd[t][e]);
                            else y = (float)(sc[t][e] * 254 + sc[t][2 + e]);
                            x[i][2 * t + e] = y;
                        }
                    const int left = there ? limit[i] - key0 : 0;  // of the lane's tokens the row sees the first `left`
                    if (__any_sync(0xffffffffu, left < 16)) {
#pragma unroll
                        for (int t = 0; t < 16; ++t)
                            if (t >= left) x[i][t] = -INFINITY;
                    }
#pragma unroll
                    for (int t = 0; t < 16; ++t) mx = fmaxf(mx, x[i][t]);
                    mx *= f;
                    const float mine_max = mx;  // of the lane's page
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float m_new = fmaxf(m[i], mx);
                    const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                    const float corr = ex2(m[i] - m_use);
                    m[i] = m_new;
                    float sum = 0.0f;
#pragma unroll
                    for (int t = 0; t < 16; ++t) {
                        x[i][t] = ex2(fmaf(x[i][t], f, -m_use));
                        sum += x[i][t];
                    }
                    l[i] = fmaf(l[i], corr, sum);
                    float w_max = ex2(mine_max - m_use) * vs;
                    w_max = fmaxf(w_max, __shfl_xor_sync(0xffffffffu, w_max, 1));
                    w_max = fmaxf(w_max, __shfl_xor_sync(0xffffffffu, w_max, 2));
                    const float old = frame[i] * corr;
                    frame[i] = __uint_as_float(__float_as_uint(fmaxf(fmaxf(old, w_max), MIN_FRAME)) & 0x7f800000u);
                    const float inv = __uint_as_float(0x7f000000u - __float_as_uint(frame[i]));
                    corr_o[i] = old * inv;
                    w_scale[i] = fminf(vs * inv * W_UP, FLT_MAX);  // (finite: a hidden page's weights are 0 times this)
                }
                bool turn = corr_o[0] != 1.0f;
                if constexpr (NR == 2) turn |= corr_o[1] != 1.0f;
                if (__any_sync(0xffffffffu, turn)) {
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        o[i][0] *= corr_o[0];
                        o[i][1] *= corr_o[0];
                        o[i][2] *= corr_o[NR - 1];
                        o[i][3] *= corr_o[NR - 1];
                    }
                }
                // ---- weights as f16 operands: k step t holds tokens 4t .. 4t + 3 of each lane's page
                uint32_t pa[4][4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        const float y0 = x[i][4 * t] * w_scale[i], y1 = x[i][4 * t + 1] * w_scale[i], y2 = x[i][4 * t + 2] * w_scale[i],
                                    y3 = x[i][4 * t + 3] * w_scale[i];
                        const uint32_t h0 = pack_f16(y0, y1), h1 = pack_f16(y2, y3);
                        if constexpr (SPLIT) {
                            pa[t][0] = h0;
                            pa[t][1] = pack_rest(y0, y1, h0);
                            pa[t][2] = h1;
                            pa[t][3] = pack_rest(y2, y3, h1);
                        } else {
                            pa[t][i] = h0;
                            pa[t][2 + i] = h1;
                        }
                    }
                }
                // ---- O += P.V
                slot = done % R::SLOTS;
                if (!ptx::mbar_wait(&full[slot], (done / R::SLOTS) & 1)) {
                    ok = false;
                    break;
                }
                const uint8_t* vp = mine + slot * R::SLOT + c * R::STRIDE + g * BKV_BLOCK;
#pragma unroll
                for (int i0 = 0; i0 < NT; i0 += 4) {
                    uint32_t vw[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 v4 = *reinterpret_cast<const uint4*>(vp + 8 * (i0 + i) * BKV_BLOCK);
                        vw[i][0] = v4.x;
                        vw[i][1] = v4.y;
                        vw[i][2] = v4.z;
                        vw[i][3] = v4.w;
                    }
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t b0, b1;
                            s8x4_to_f16(vw[i][t], b0, b1);
                            mma16816(o[i0 + i], pa[t][0], pa[t][1], pa[t][2], pa[t][3], b0, b1);
                        }
                }
                __syncwarp();
                ++done;
                issue();
            }

            // ---- the item's rows: finished, or a part of them
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            }
            const bool alone = c0 == 0 && c1 == chunks;
            const int which = w.u == u_begin ? 0 : 1;
            const int64_t part = ((int64_t)blockIdx.x * AW + warp) * 2 + which;
            if (!alone && lane == 0) parts[2 * warp + which] = Part{u0, chunks, s, h, tile, warp == 0 || c0 == 0};
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int r = tile * TR + i * 8 + g;
                const int tok = r / A.group, head = h * A.group + r % A.group;
                if (tok >= n_q) continue;
                const float fin = l[i] == 0.0f ? 0.0f : frame[i] * (1.0f / W_UP) / l[i];
                const int64_t at = (int64_t)(first_row + tok) * A.out_ld + (int64_t)head * D + 2 * c;
                float* po = A.warp_o + (part * TR + i * 8 + g) * D + 2 * c;
                if (!alone && c == 0) A.warp_ml[part * TR + i * 8 + g] = make_float2(m[i], l[i]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float y0, y1;
                    if constexpr (SPLIT) {
                        y0 = (o[n][0] + o[n][2]) * fin;
                        y1 = (o[n][1] + o[n][3]) * fin;
                    } else {
                        y0 = o[n][2 * i] * fin;
                        y1 = o[n][2 * i + 1] * fin;
                    }
                    if (alone) store_pair(A, at + 8 * n, y0, y1);
                    else *reinterpret_cast<float2*>(po + 8 * n) = make_float2(y0, y1);
                }
            }
            w.u += c1 - c0;
            w.ch = c1;
            if (c1 == chunks) w.next_item(A, st, u_end);
        }
        // a wait that gave up: the copies still under way end before the block does
        for (int i = done; !ok && i < op; ++i) ptx::mbar_wait(&full[i % R::SLOTS], (i / R::SLOTS) & 1);
    }
    if (!ok && lane == 0) atomicExch(A.err, 1);
    __syncthreads();

    auto share_of = [&](int s) { return __uint_as_float((uint32_t)(95 + __clz(max(st.keys[s], 1))) << 23); };  // 2^-bits(keys)
    // ---- parts of one item within the block, then what the block shares with others
    // lane i: whether part i is the block's first one of its item (the second part of a warp starts its item)
    const unsigned heads = __ballot_sync(
        0xffffffffu, lane < 2 * AW && parts[min(lane, 2 * AW - 1)].chunks && parts[min(lane, 2 * AW - 1)].head);
    static_assert(2 * AW <= 32, "a lane for each part");
    Part open[2];
    int n_open = 0;
    int job = warp;
    for (unsigned left = heads; left; left &= left - 1) {  // the rows of all items in turn, one warp each
        const int i = __ffs(left) - 1;
        const Part p = parts[i];
        const bool whole = p.u0 >= block_begin && p.u0 + p.chunks <= block_end;
        if (!whole) open[n_open++] = p;
        const int rows = min(TR, st.n_q[p.s] * A.group - p.tile * TR);
        if (job < rows) {
            int n = 1;  // the warps behind the first one have their part of the item at the start of their range
            while (i / 2 + n < AW && parts[2 * (i / 2 + n)].chunks && parts[2 * (i / 2 + n)].u0 == p.u0) ++n;
            const int64_t to = ((int64_t)blockIdx.x * 2 + (i == 0 ? 0 : 1)) * TR;
            auto nth = [&](int j) { return ((int64_t)blockIdx.x * AW * 2 + (j ? 2 * (i / 2 + j) : i)) * TR; };
            while (job < rows) {
                const int second = job + AW < rows ? job + AW : -1;
                join_rows<D>(A, n, job, second, st.first[p.s], p.tile * TR, p.h, share_of(p.s), [&](int j) { return A.warp_o + nth(j) * D; },
                            [&](int j) { return A.warp_ml + nth(j); }, whole ? nullptr : A.block_o + to * D,
                            whole ? nullptr : A.block_ml + to);
                job += second < 0 ? AW : 2 * AW;
            }
        }
        job -= rows;
    }
    if (n_open == 0) return;
    auto block_of = [&](int64_t u) { return (int)(((u + 1) * n_block + total - 1) / total) - 1; };  // whose share has step u
    __syncthreads();
    if (threadIdx.x < n_open) {
        const Part p = open[threadIdx.x];
        const int first = block_of(p.u0), n = block_of(p.u0 + p.chunks - 1) - first + 1;
        __threadfence();  // the block's parts, written before the barrier, come before its arrival
        const unsigned before = atomicAdd(&A.arrived[first], 1u);
        last_one[threadIdx.x] = before == (unsigned)n - 1;
        if (before == (unsigned)n - 1) A.arrived[first] = 0;  // at rest again
        __threadfence();
    }
    __syncthreads();
    for (int k = 0; k < n_open; ++k) {
        if (!last_one[k]) continue;
        const Part p = open[k];
        const int64_t first = block_of(p.u0);
        const int n = block_of(p.u0 + p.chunks - 1) - (int)first + 1;
        const int rows = min(TR, st.n_q[p.s] * A.group - p.tile * TR);
        // the item starts somewhere in its first block's range, and at the start of every other one's
        auto nth = [&](int b) { return ((first + b) * 2 + (b == 0 && p.u0 != first * total / n_block ? 1 : 0)) * TR; };
        for (int r = warp; r < rows; r += 2 * AW)
            join_rows<D>(A, n, r, r + AW < rows ? r + AW : -1, st.first[p.s], p.tile * TR, p.h, share_of(p.s), [&](int b) { return A.block_o + nth(b) * D; },
                        [&](int b) { return A.block_ml + nth(b); }, nullptr, nullptr);
    }
}

template <int D, bool SPLIT, bool P3>
void launch_attn(vkb_context* ctx, AttnArgs A) {
    constexpr int TR = SPLIT ? 8 : 16, AW = Ring<D>::AW;
    constexpr int SMEM = ((int)sizeof(Streams) + 15) / 16 * 16 + AW * Ring<D>::WARP_BYTES;
    static_assert(SMEM <= 227 * 1024 - 2048, "shared memory of one block");
    const size_t blocks = (size_t)ctx->sm_count;
    const size_t warp_o = blocks * AW * 2 * TR * D * sizeof(float), block_o = blocks * 2 * TR * D * sizeof(float);
    const size_t warp_ml = blocks * AW * 2 * TR * sizeof(float2), block_ml = blocks * 2 * TR * sizeof(float2);
    ctx->ensure_workspace(warp_o + block_o + warp_ml + block_ml);
    uint8_t* ws = ctx->workspace.as<uint8_t>();
    A.warp_o = reinterpret_cast<float*>(ws);
    A.block_o = reinterpret_cast<float*>(ws + warp_o);
    A.warp_ml = reinterpret_cast<float2*>(ws + warp_o + block_o);
    A.block_ml = reinterpret_cast<float2*>(ws + warp_o + block_o + warp_ml);
    A.arrived = ctx->tile_ctr.as<unsigned>();
    A.err = ctx->err_flag.as<int>();
    auto kern = bkv_attn_kernel<D, SPLIT, P3>;
    smem_optin(kern, SMEM);
    const BkvStreams all = A.S;
    for (int s0 = 0; s0 < all.n_seq; s0 += BKV_SEQ_PER_LAUNCH) {
        A.S.n_seq = std::min(all.n_seq - s0, BKV_SEQ_PER_LAUNCH);
        A.S.start = all.start + s0;
        A.S.len = all.len + s0;
        A.S.table = all.table + (int64_t)s0 * all.ld;
        launch_pdl(ctx, kern, dim3((unsigned)blocks), 32 * AW, SMEM, A);
        VKB_CUDA(cudaGetLastError());
        ctx->count();
    }
}

}  // namespace

void run_bkv_attn(vkb_context* ctx, const BkvAttn& a) {
    AttnArgs A{};
    static_cast<BkvAttn&>(A) = a;
    A.q_vec = (uintptr_t)a.q % (a.q_f16 ? 8 : 16) == 0 && a.q_ld % 4 == 0;
    A.out_vec = (uintptr_t)a.out % (a.out_f16 ? 4 : 8) == 0 && a.out_ld % 2 == 0;
    with_bkv_head(a.d_head, [&](auto D) {
        if (!a.q_f16 || !a.out_f16) launch_attn<decltype(D)::value, true, true>(ctx, A);
        else if ((int64_t)a.max_q * a.group <= 8) launch_attn<decltype(D)::value, true, false>(ctx, A);
        else launch_attn<decltype(D)::value, false, false>(ctx, A);
    });
}

}  // namespace vkb

using namespace vkb;

extern "C" vkb_status vkb_bkv_attention(vkb_context* ctx, const vkb_bkv_cache* cache, int32_t layer,
                                        const vkb_bkv_batch* batch, int32_t n_head, const void* q_dev, int64_t q_ld,
                                        int32_t q_dtype, float scale, void* out_dev, int64_t out_ld, int32_t out_dtype) {
    return guard([&] {
        BkvAttn a{};
        a.L = bkv_layer(ctx, cache, layer);
        a.S = bkv_streams(batch);
        if (n_head <= 0 || n_head % cache->n_kv_head)
            fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: n_head must be a multiple of n_kv_head");
        for (int dt : {q_dtype, out_dtype})
            if (dt != VKB_DT_F32 && dt != VKB_DT_F16) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv_attention: q and out must be F32 or F16");
        a.d_head = cache->d_head;
        const int64_t width = (int64_t)n_head * a.d_head;
        if (q_ld < width || out_ld < width) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: row stride below n_head*d_head");
        if (!(scale > 0.0f) || scale > 2.0e38f)  // (times log2(e) it is finite)
            fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: scale must be positive and at most 2e38");
        if (batch->n_seq == 0 || batch->n_tok == 0) return;
        if (!q_dev || !out_dev) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: null q/out");
        a.group = n_head / cache->n_kv_head;
        a.n_head = n_head;
        a.max_q = std::max(1, std::min(batch->max_q, batch->n_tok));
        a.max_kv = batch->max_kv;
        if ((int64_t)batch->n_tok * a.group > INT32_MAX / 2) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv_attention: too many rows");
        a.q_f16 = q_dtype == VKB_DT_F16;
        a.out_f16 = out_dtype == VKB_DT_F16;
        if ((uintptr_t)q_dev % (a.q_f16 ? 2 : 4) || (uintptr_t)out_dev % (a.out_f16 ? 2 : 4))
            fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: misaligned q/out");
        a.q = q_dev;
        a.q_ld = q_ld;
        a.scale = scale;
        a.out = out_dev;
        a.out_ld = out_ld;
        NvtxRange nvtx_range("vkb.bkv.attention");
        if (bkv_prompt_takes(ctx, a)) run_bkv_prompt(ctx, a);
        else run_bkv_attn(ctx, a);
    });
}
