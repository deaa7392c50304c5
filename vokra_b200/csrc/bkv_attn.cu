// bkv_attn.cu — attention over the block-scaled 8-bit KV cache for few query
// rows a stream: decode steps, tokens to check, short chunks.
//
// Bound: HBM (2 d_head bytes a key and KV head). A warp takes 64 keys = 4 pages
// at a time and feeds m16n8k16 tensor-core products straight from global
// memory: no shared memory, no transpose, and every 16-byte load is used whole.
// What makes that work is that the order of keys and channels inside a product
// is free as long as both operands agree:
//  - lane (g, c) = (lane / 4, lane % 4). Column n of the score tile t is token
//    2t + n % 2 of page n / 2, so that lane c's columns (2c, 2c + 1) of all 8
//    tiles are the 16 tokens of page c: one K scale, one V scale and one page
//    id a lane and step.
//  - a K row is loaded as 16 neighbouring channels a lane (D = 64: a quad reads
//    the 64 bytes of a key, a warp 4 x 128 bytes), which are four k steps of the
//    Q.K product; q is kept in the same order.
//  - V is stored channel by channel, so 16 bytes at (page c, channel 8i + g) are
//    the 16 tokens whose weights the lane holds: four k steps of the P.V product.
// int8 -> f16 is exact (a byte permute into 1024 + u, minus 1152). The K scale
// multiplies the scores, the V scale the weights, both in fp32; weights enter
// the product divided by a running power of two above the V scales, so that f16
// holds them whatever the scale.
//
// SPLIT tiles (8 query rows) hold the high f16 part of q in rows 0..7 of the
// 16-row operand and the low part in rows 8..15, likewise for the weights: the
// products are accurate to about 2^-21 at the price of one. Tiles of 16 rows
// have one f16 part. Up to 8 rows SPLIT costs nothing more and is taken always.
//
// The (stream, KV head, row tile, 64 keys) steps of the whole call are one
// sequence, cut into equal contiguous ranges, one a warp, so ragged lengths
// balance themselves. A warp finishes an item that lies in its range alone;
// the others leave partial rows that bkv_combine_kernel joins in order.
#include "bkv.cuh"
#include <algorithm>

namespace vkb {
namespace {

constexpr int AW = 4;  // warps of a block
constexpr float L2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

struct AttnArgs {
    BkvLayer L;
    BkvStreams S;
    int group, n_head;
    const void* q;
    int64_t q_ld;
    float scale;
    void* out;
    int64_t out_ld;
    int q_f16, out_f16, q_vec;
    float* part_o;   // [warps][2][rows][D]
    float2* part_ml; // [warps][2][rows]
    int4* todo;      // [warps]: the item that starts in the warp's range and goes on behind it (stream, head,
                     // tile, further warps * 2 + slot of its first part); stream -1: none
};

__device__ __forceinline__ int64_t steps_of(const AttnArgs& A, int s, int tile_rows, int& tiles, int& chunks) {
    int first, n;
    A.S.rows(s, first, n);
    tiles = (n * A.group + tile_rows - 1) / tile_rows;
    chunks = max(1, (A.S.keys(s) + 63) / 64);
    return (int64_t)A.L.n_kv_head * tiles * chunks;
}

// Running steps in front of each stream, in shared memory: pre[n_seq] is the total.
template <int TR>
__device__ __forceinline__ void stream_prefix(const AttnArgs& A, int64_t* pre) {
    __shared__ int64_t warp_sum_s[32];
    __shared__ int64_t carry_s;
    const int n = A.S.n_seq, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        carry_s = 0;
        pre[0] = 0;
    }
    __syncthreads();
    for (int base = 0; base < n; base += blockDim.x) {
        const int s = base + (int)threadIdx.x;
        int tiles, chunks;
        int64_t x = s < n ? steps_of(A, s, TR, tiles, chunks) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_sum_s[warp] = x;
        __syncthreads();
        int64_t before = carry_s;
        for (int w = 0; w < warp; ++w) before += warp_sum_s[w];
        if (s < n) pre[s + 1] = before + x;
        __syncthreads();
        if ((int)threadIdx.x == blockDim.x - 1) carry_s = before + x;
        __syncthreads();
    }
}

template <int D, bool SPLIT>
__global__ void __launch_bounds__(32 * AW, D <= 64 ? 3 : D <= 128 ? 2 : 1) bkv_attn_kernel(AttnArgs A) {
    pdl_entry();
    constexpr int TR = SPLIT ? 8 : 16;       // query rows of a tile
    constexpr int NR = SPLIT ? 1 : 2;        // of them in this lane's hands
    constexpr int KW = D / 16;               // 32-bit words of a K row a lane holds = k steps of Q.K
    constexpr int NT = D / 8;                // channel tiles of P.V
    extern __shared__ int64_t pre[];         // [n_seq + 1]
    stream_prefix<TR>(A, pre);
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int64_t n_warps = (int64_t)gridDim.x * AW;
    const int64_t me = (int64_t)blockIdx.x * AW + (threadIdx.x >> 5);
    const int64_t total = pre[A.S.n_seq];
    const int64_t per = (total + n_warps - 1) / n_warps;
    const int64_t u_begin = min(total, me * per), u_end = min(total, u_begin + per);
    if (lane == 0) A.todo[me] = make_int4(-1, 0, 0, 0);
    if (u_begin == u_end) return;

    // the stream of the first step
    int s;
    {
        int lo = 0, hi = A.S.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= u_begin) lo = mid;
            else hi = mid - 1;
        }
        s = lo;
    }
    int64_t u = u_begin;
    while (u < u_end) {
        while (pre[s + 1] <= u) ++s;
        int tiles, chunks;
        steps_of(A, s, TR, tiles, chunks);
        int first_row, n_q;
        A.S.rows(s, first_row, n_q);
        const int64_t in_seq = u - pre[s];
        const int item = (int)(in_seq / chunks);
        const int c0 = (int)(in_seq % chunks);
        const int c1 = (int)min((int64_t)chunks, c0 + (u_end - u));
        const int h = item / tiles, tile = item % tiles;
        const int n_keys = A.S.keys(s);

        // ---- the tile's query rows: f16 operands in the order of the K loads
        uint32_t qa[KW][4];
        float row_fac[NR];  // multiplies a score: 2^e * scale * log2(e)
        int limit[NR];      // keys that the row sees
#pragma unroll
        for (int half_row = 0; half_row < NR; ++half_row) {
            const int r = tile * TR + half_row * 8 + g;
            const int tok = r / A.group, head = h * A.group + r % A.group;
            const bool real = tok < n_q;
            float x[KW * 4];
            float amax = 0.0f;
            if (real) {
                const int64_t at = (int64_t)(first_row + tok) * A.q_ld + (int64_t)head * D;
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    // word w of the lane: 4 channels of the 64-channel part w / 4 (or of what is left behind them)
                    const int part = w >> 2;
                    constexpr int LEFT = KW & 3;  // words of the last, shorter part
                    const int words = part < KW / 4 ? 4 : LEFT;
                    const int d = 64 * part + 4 * words * c + 4 * (w & 3);
                    if (A.q_f16) {
                        const __half* p = reinterpret_cast<const __half*>(A.q) + at + d;
                        if (A.q_vec) {
                            const uint2 v = __ldcg(reinterpret_cast<const uint2*>(p));
                            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
                            const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
                            x[4 * w] = a.x;
                            x[4 * w + 1] = a.y;
                            x[4 * w + 2] = b.x;
                            x[4 * w + 3] = b.y;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[4 * w + e] = __half2float(p[e]);
                        }
                    } else {
                        const float* p = reinterpret_cast<const float*>(A.q) + at + d;
                        if (A.q_vec) {
                            const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
                            x[4 * w] = v.x;
                            x[4 * w + 1] = v.y;
                            x[4 * w + 2] = v.z;
                            x[4 * w + 3] = v.w;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[4 * w + e] = p[e];
                        }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < KW * 4; ++i) x[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < KW * 4; ++i) amax = fmaxf(amax, fabsf(x[i]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // the row as values below 2 times 2^e: f16 holds it whatever its size
            uint32_t e = __float_as_uint(amax) & 0x7f800000u;
            e = e == 0 || e == 0x7f800000u ? 0x3f800000u : min(e, 0x7e800000u);  // zero and infinity stay as they are
            const float pow2 = __uint_as_float(e), inv2 = __uint_as_float(0x7f000000u - e);
            row_fac[half_row] = pow2 * (A.scale * L2E);
            limit[half_row] = real ? max(0, min(n_keys, n_keys - n_q + tok + 1)) : 0;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const float y0 = x[4 * w] * inv2, y1 = x[4 * w + 1] * inv2, y2 = x[4 * w + 2] * inv2, y3 = x[4 * w + 3] * inv2;
                const uint32_t h0 = pack_f16(y0, y1), h1 = pack_f16(y2, y3);
                if constexpr (SPLIT) {
                    qa[w][0] = h0;
                    qa[w][1] = pack_rest(y0, y1, h0);
                    qa[w][2] = h1;
                    qa[w][3] = pack_rest(y2, y3, h1);
                } else {
                    qa[w][half_row] = h0;
                    qa[w][2 + half_row] = h1;
                }
            }
        }

        float m[NR], l[NR];
        float o[NT][4];
        float frame = __uint_as_float(0x00800000u);  // power of two at or above half of every V scale so far
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;

        // no row of the tile sees a key from here on
        int seen = limit[0];
        if constexpr (NR == 2) seen = max(seen, limit[1]);
        seen = __reduce_max_sync(0xffffffffu, seen);
        const int c_last = min(c1, (seen + 63) / 64);

        int64_t next_page = c0 < c_last ? A.S.page(s, 4 * c0 + c, A.L.n_pages) : -1;
        for (int ch = c0; ch < c_last; ++ch) {
            const int64_t page = next_page;
            if (ch + 1 < c_last) next_page = A.S.page(s, 4 * (ch + 1) + c, A.L.n_pages);
            const bool there = page >= 0 && 64 * ch + 16 * c < seen;  // a page behind the last seen key may hold anything
            const int64_t head_at = (there ? page : 0) * A.L.n_kv_head + h;
            const int64_t k_head = __shfl_sync(0xffffffffu, head_at, g >> 1);  // lane g / 2 holds page g / 2
            const int8_t* kp = A.L.k + k_head * (BKV_BLOCK * D) + (g & 1) * D;
            const int8_t* vp = A.L.v + head_at * (BKV_BLOCK * D) + g * BKV_BLOCK;
            const float ks = there ? A.L.ks[head_at] : 0.0f;
            const float vs = there ? A.L.vs[head_at] : 0.0f;

            // ---- scores
            float sc[8][4];
#pragma unroll
            for (int t = 0; t < 8; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[t][e] = 0.0f;
                uint32_t kw[KW];
#pragma unroll
                for (int part = 0; part < KW / 4; ++part) {
                    const uint4 v4 = __ldcg(reinterpret_cast<const uint4*>(kp + 2 * t * D + 64 * part + 16 * c));
                    kw[4 * part] = v4.x;
                    kw[4 * part + 1] = v4.y;
                    kw[4 * part + 2] = v4.z;
                    kw[4 * part + 3] = v4.w;
                }
                if constexpr ((KW & 3) == 2) {
                    const uint2 v2 = __ldcg(reinterpret_cast<const uint2*>(kp + 2 * t * D + 64 * (KW / 4) + 8 * c));
                    kw[KW - 2] = v2.x;
                    kw[KW - 1] = v2.y;
                }
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    uint32_t b0, b1;
                    s8x4_to_f16(kw[w], b0, b1);
                    mma16816(sc[t], qa[w][0], qa[w][1], qa[w][2], qa[w][3], b0, b1);
                }
            }

            // ---- softmax step. Lane c holds tokens 0..15 of page 4 ch + c: x[row][token]
            const int key0 = 64 * ch + 16 * c;
            float w_scale;
            float corr_o[NR];
            float x[NR][16];
            {
                // the V scales' frame
                float vmax = fmaxf(vs, __shfl_xor_sync(0xffffffffu, vs, 1));
                vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
                const float pow2 = fmaxf(frame, __uint_as_float(__float_as_uint(vmax) & 0x7f800000u));
                const float inv = __uint_as_float(0x7f000000u - __float_as_uint(pow2));
                w_scale = vs * inv;
#pragma unroll
                for (int i = 0; i < NR; ++i) corr_o[i] = frame * inv;
                frame = pow2;
            }
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const float f = ks * row_fac[i];
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float y = SPLIT ? sc[t][e] + sc[t][2 + e] : sc[t][2 * i + e];
                        y *= f;
                        if (!there || key0 + 2 * t + e >= limit[i]) y = -INFINITY;
                        x[i][2 * t + e] = y;
                        mx = fmaxf(mx, y);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float m_new = fmaxf(m[i], mx);
                const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                const float corr = ex2(m[i] - m_use);
                m[i] = m_new;
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < 16; ++t) {
                    x[i][t] = ex2(x[i][t] - m_use);
                    sum += x[i][t];
                }
                l[i] = fmaf(l[i], corr, sum);
                corr_o[i] *= corr;
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
            // ---- weights as f16 operands: k step t' holds tokens 4t' .. 4t' + 3 of each lane's page
            uint32_t pa[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const float y0 = x[i][4 * t] * w_scale, y1 = x[i][4 * t + 1] * w_scale, y2 = x[i][4 * t + 2] * w_scale,
                                y3 = x[i][4 * t + 3] * w_scale;
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
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint4 v4 = __ldcg(reinterpret_cast<const uint4*>(vp + 8 * i * BKV_BLOCK));
                const uint32_t vw[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    uint32_t b0, b1;
                    s8x4_to_f16(vw[t], b0, b1);
                    mma16816(o[i], pa[t][0], pa[t][1], pa[t][2], pa[t][3], b0, b1);
                }
            }
        }

        // ---- the item's rows: finished, or left for the combine kernel
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        const bool alone = c0 == 0 && c1 == chunks;
        const int64_t slot = me * 2 + (u == u_begin ? 0 : 1);
        if (!alone && c0 == 0 && lane == 0) A.todo[me] = 
            make_int4(s, h, tile, (int)((u + chunks - 1) / per - me) * 2 + (u == u_begin ? 0 : 1));
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = tile * TR + i * 8 + g;
            const int tok = r / A.group, head = h * A.group + r % A.group;
            if (tok >= n_q) continue;
            const float fin = alone ? (l[i] > 0.0f ? frame / l[i] : 0.0f) : frame;
            const int64_t at = (int64_t)(first_row + tok) * A.out_ld + (int64_t)head * D + 2 * c;
            float* po = A.part_o + (slot * TR + i * 8 + g) * D + 2 * c;
            if (!alone && c == 0) A.part_ml[slot * TR + i * 8 + g] = make_float2(m[i], l[i]);
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
                if (!alone) {
                    *reinterpret_cast<float2*>(po + 8 * n) = make_float2(y0, y1);
                } else if (A.out_f16) {
                    __half* p = reinterpret_cast<__half*>(A.out) + at + 8 * n;
                    p[0] = __float2half_rn(y0);
                    p[1] = __float2half_rn(y1);
                } else {
                    float* p = reinterpret_cast<float*>(A.out) + at + 8 * n;
                    p[0] = y0;
                    p[1] = y1;
                }
            }
        }
        u += c1 - c0;
    }
}

// Joins the parts of one item that several warps of the attention shared: block
// b has the item that starts in warp b's range. A warp takes a row at a time.
constexpr int CW = 8;
template <int D, bool SPLIT>
__global__ void __launch_bounds__(32 * CW) bkv_combine_kernel(AttnArgs A) {
    pdl_entry();
    constexpr int TR = SPLIT ? 8 : 16;
    constexpr int V = D / 32;  // channels of a lane
    const int64_t w0 = blockIdx.x;
    const int4 t = A.todo[w0];
    if (t.x < 0) return;
    const int s = t.x, h = t.y, tile = t.z, last = t.w >> 1;  // the parts of warps w0 .. w0 + last
    int first_row, n_q;
    A.S.rows(s, first_row, n_q);
    __shared__ float so[CW][D];
    __shared__ float2 sml[CW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = 0; r < TR; ++r) {
        const int row = tile * TR + r, tok = row / A.group, head = h * A.group + row % A.group;
        if (tok >= n_q) break;
        float m = -INFINITY, l = 0.0f, acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
#pragma unroll 4
        for (int p = warp; p <= last; p += CW) {
            const int64_t slot = (w0 + p) * 2 + (p == 0 ? t.w & 1 : 0);  // a later part starts its warp's range
            const float2 ml = __ldcg(&A.part_ml[slot * TR + r]);
            const float* po = A.part_o + (slot * TR + r) * D + lane;
            float y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = __ldcg(po + 32 * i);
            if (ml.x == -INFINITY) continue;
            const float m_new = fmaxf(m, ml.x);
            const float a = ex2(m - m_new), b = ex2(ml.x - m_new);
            l = l * a + ml.y * b;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = acc[i] * a + y[i] * b;
            m = m_new;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) so[warp][lane + 32 * i] = acc[i];
        if (lane == 0) sml[warp] = make_float2(m, l);
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += blockDim.x) {
            float M = -INFINITY, Lr = 0.0f, O = 0.0f;
            for (int w = 0; w < CW; ++w) M = fmaxf(M, sml[w].x);
            for (int w = 0; w < CW; ++w) {
                if (sml[w].x == -INFINITY) continue;
                const float f = ex2(sml[w].x - M);
                Lr += sml[w].y * f;
                O += so[w][d] * f;
            }
            const float y = Lr > 0.0f ? O / Lr : 0.0f;
            const int64_t at = (int64_t)(first_row + tok) * A.out_ld + (int64_t)head * D + d;
            if (A.out_f16) reinterpret_cast<__half*>(A.out)[at] = __float2half_rn(y);
            else reinterpret_cast<float*>(A.out)[at] = y;
        }
        __syncthreads();
    }
}

template <int D, bool SPLIT>
void launch_attn(vkb_context* ctx, AttnArgs A) {
    constexpr int TR = SPLIT ? 8 : 16;
    const unsigned blocks = (unsigned)(ctx->sm_count * (D <= 64 ? 3 : D <= 128 ? 2 : 1));
    const size_t warps = (size_t)blocks * AW;
    const size_t o_bytes = warps * 2 * TR * D * sizeof(float), ml_bytes = warps * 2 * TR * sizeof(float2);
    ctx->ensure_workspace(o_bytes + ml_bytes + warps * sizeof(int4));
    uint8_t* ws = ctx->workspace.as<uint8_t>();
    A.part_o = reinterpret_cast<float*>(ws);
    A.part_ml = reinterpret_cast<float2*>(ws + o_bytes);
    A.todo = reinterpret_cast<int4*>(ws + o_bytes + ml_bytes);
    const size_t smem = (size_t)(A.S.n_seq + 1) * sizeof(int64_t);
    auto kern = bkv_attn_kernel<D, SPLIT>;
    if (smem > 40 * 1024) smem_optin(kern, 72 * 1024);
    launch_pdl(ctx, kern, dim3(blocks), 32 * AW, smem, A);
    VKB_CUDA(cudaGetLastError());
    ctx->count();
    launch_pdl(ctx, bkv_combine_kernel<D, SPLIT>, dim3((unsigned)warps), 32 * CW, 0, A);
    VKB_CUDA(cudaGetLastError());
    ctx->count();
}

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" vkb_status vkb_bkv_attention(vkb_context* ctx, const vkb_bkv_cache* cache, int32_t layer,
                                        const vkb_bkv_batch* batch, int32_t n_head, const void* q_dev, int64_t q_ld,
                                        int32_t q_dtype, float scale, void* out_dev, int64_t out_ld, int32_t out_dtype) {
    return guard([&] {
        AttnArgs A{};
        A.L = bkv_layer(ctx, cache, layer);
        A.S = bkv_streams(batch);
        if (n_head <= 0 || n_head % cache->n_kv_head)
            fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: n_head must be a multiple of n_kv_head");
        for (int dt : {q_dtype, out_dtype})
            if (dt != VKB_DT_F32 && dt != VKB_DT_F16) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv_attention: q and out must be F32 or F16");
        const int64_t width = (int64_t)n_head * cache->d_head;
        if (q_ld < width || out_ld < width) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: row stride below n_head*d_head");
        if (!(scale > 0.0f) || scale > 3.0e38f) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: scale must be positive and finite");
        if (batch->n_seq == 0 || batch->n_tok == 0) return;
        if (!q_dev || !out_dev) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: null q/out");
        A.group = n_head / cache->n_kv_head;
        A.n_head = n_head;
        if ((int64_t)batch->n_tok * A.group > INT32_MAX / 2) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv_attention: too many rows");
        A.q_f16 = q_dtype == VKB_DT_F16;
        A.out_f16 = out_dtype == VKB_DT_F16;
        if ((uintptr_t)q_dev % (A.q_f16 ? 2 : 4) || (uintptr_t)out_dev % (A.out_f16 ? 2 : 4))
            fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_attention: misaligned q/out");
        A.q = q_dev;
        A.q_ld = q_ld;
        A.q_vec = (uintptr_t)q_dev % (A.q_f16 ? 8 : 16) == 0 && q_ld % 4 == 0;
        A.scale = scale;
        A.out = out_dev;
        A.out_ld = out_ld;
        NvtxRange nvtx_range("vkb.bkv.attention");
        const bool split = !A.q_f16 || !A.out_f16 || (int64_t)batch->max_q * A.group <= 8;
        with_bkv_head(cache->d_head, [&](auto D) {
            if (split) launch_attn<decltype(D)::value, true>(ctx, A);
            else launch_attn<decltype(D)::value, false>(ctx, A);
        });
    });
}
