// bkv.cu — a paged KV cache in 8 bits with one fp32 scale for each block of 16
// tokens and head: its checks, append and read-back.
//
// A page is one block: K as [16][d_head] (a token's channels together), V as
// [d_head][16] (a channel's tokens together), which is how the attention's
// matrix instructions take the two, so neither is ever transposed on the way.
//
// append, block by block: s' = max(s, amax * (1/127)) with s = 0 where the block's
// first slot is among the new tokens; the block's earlier quants become
// rint(q * (s / s')) where s' > s, the new ones rint(x * (1 / s')). All in
// IEEE fp32, so the stored bytes are defined to the bit. NaN counts as 0, and a
// block with an infinity has the scale FLT_MAX * (1/127): 127 stands for it.
//
// Bound: HBM, then the conversions. One warp holds one block of one head and
// side: each lane owns d_head / 32 neighbouring channels of all 16 tokens, so a
// token's row is one coalesced load, the maximum is one warp reduction, and a V
// block goes out as 16-byte stores without a transpose. Measured, 8 streams with
// about 8500 new tokens in all, 8 heads of 128, f16: append 23.5 us (52 MB:
// 2.2 TB/s; 27 with the rows asked for behind the page's id and the status), read
// as f32 15.5 us (87 MB: 5.6 TB/s). Rounding by a magic number with an integer
// maximum, a branch for whole blocks, or a path of their own: 55, 42 and 29 us.
#include "bkv.cuh"
#include <cfloat>
#include <algorithm>

namespace vkb {

BkvLayer bkv_layer(const vkb_context* ctx, const vkb_bkv_cache* c, int layer) {
    if (!ctx || !c) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: null context or cache");
    if (c->n_layer <= 0 || c->n_kv_head <= 0 || c->d_head <= 0 || c->n_pages <= 0)
        fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: every axis of the cache must be > 0");
    if (c->n_pages > INT32_MAX) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv: more than 2^31 - 1 pages");
    if (c->n_kv_head > 32768) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv: more than 32768 heads");
    if (layer < 0 || layer >= c->n_layer) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: layer out of range");
    if (!c->k_dev || !c->v_dev || !c->k_scale_dev || !c->v_scale_dev)
        fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: null arena");
    with_bkv_head(c->d_head, [](auto) {});
    if (((uintptr_t)c->k_dev | (uintptr_t)c->v_dev) & 15) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: arenas must be 16-byte aligned");
    if (((uintptr_t)c->k_scale_dev | (uintptr_t)c->v_scale_dev) & 3) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: misaligned scales");
    const int64_t heads = (int64_t)layer * c->n_pages * c->n_kv_head;
    const int64_t block = (int64_t)BKV_BLOCK * c->d_head;
    return BkvLayer{reinterpret_cast<int8_t*>(c->k_dev) + heads * block, reinterpret_cast<int8_t*>(c->v_dev) + heads * block,
                    c->k_scale_dev + heads, c->v_scale_dev + heads, c->n_pages, c->n_kv_head};
}

BkvStreams bkv_streams(const vkb_bkv_batch* b) {
    if (!b) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: null batch");
    if (b->n_seq < 0 || b->n_tok < 0 || b->max_q < 0 || b->max_kv < 0) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: negative count in the batch");
    if (b->n_seq > VKB_BKV_MAX_SEQ)
        fail(VKB_ERROR_UNSUPPORTED_OP, "bkv: more than " + std::to_string(VKB_BKV_MAX_SEQ) + " streams in one call");
    if (b->n_seq && (!b->tok_start_dev || !b->kv_len_dev || !b->table_dev))
        fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: null array in the batch");
    if (b->table_ld <= 0 && b->n_seq) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv: table_ld must be > 0");
    if (b->table_ld > INT32_MAX / BKV_BLOCK) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv: streams of 2^31 tokens or more");
    return BkvStreams{b->n_seq, b->n_tok, b->tok_start_dev, b->kv_len_dev, b->table_dev, b->table_ld};
}

namespace {

template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_row(const T* p, float (&x)[N]) {
    constexpr int BYTES = N * (int)sizeof(T);
    if constexpr (VEC && BYTES % 16 == 0) {
        __align__(16) T part[N];
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i)
            reinterpret_cast<uint4*>(part)[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)part[i];
    } else if constexpr (VEC && BYTES == 8) {
        const uint2 u = __ldcg(reinterpret_cast<const uint2*>(p));
        T part[N];
        memcpy(part, &u, 8);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)part[i];
    } else if constexpr (VEC && BYTES == 4) {
        const uint32_t u = __ldcg(reinterpret_cast<const uint32_t*>(p));
        T part[N];
        memcpy(part, &u, 4);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)part[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)p[i];
    }
}

// N bytes at p (aligned to N where N is a power of two).
template <int N>
__device__ __forceinline__ void store_bytes(int8_t* p, const int8_t (&b)[N]) {
    if constexpr (N == 2) {
        uint16_t u;
        memcpy(&u, b, 2);
        *reinterpret_cast<uint16_t*>(p) = u;
    } else if constexpr (N == 4) {
        uint32_t u;
        memcpy(&u, b, 4);
        *reinterpret_cast<uint32_t*>(p) = u;
    } else if constexpr (N == 8) {
        uint2 u;
        memcpy(&u, b, 8);
        *reinterpret_cast<uint2*>(p) = u;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = b[i];
    }
}
template <int N>
__device__ __forceinline__ void load_bytes(const int8_t* p, int8_t (&b)[N]) {
    if constexpr (N == 2) {
        const uint16_t u = *reinterpret_cast<const uint16_t*>(p);
        memcpy(b, &u, 2);
    } else if constexpr (N == 4) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
        memcpy(b, &u, 4);
    } else if constexpr (N == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        memcpy(b, &u, 8);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) b[i] = p[i];
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, const T (&x)[N]) {
    constexpr int BYTES = N * (int)sizeof(T);
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(x)[i];
    } else if constexpr (BYTES == 8) {
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(x);
    } else if constexpr (BYTES == 4) {
        *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(x);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = x[i];
    }
}

// One value of a block: nearest whole number of scales, NaN as 0.
__device__ __forceinline__ int8_t quant(float x, float inv) {
    const float y = x * inv;
    return y == y ? (int8_t)__float2int_rn(fminf(fmaxf(y, -127.0f), 127.0f)) : (int8_t)0;
}

constexpr int APPEND_WARPS = 4;
constexpr float SCALE = 1.0f / 127.0f;  // rounded to fp32: part of the definition

// grid (2 * n_kv_head / 4, pages of a stream, streams); warp = one head and side.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(32 * APPEND_WARPS)
    bkv_append_kernel(BkvLayer L, BkvStreams S, const T* __restrict__ k, int64_t k_ld, const T* __restrict__ v,
                      int64_t v_ld, const int32_t* __restrict__ status) {
    pdl_entry();
    constexpr int C = D / 32;  // channels of a lane
    const int lane = threadIdx.x & 31;
    const int job = (int)blockIdx.x * APPEND_WARPS + (int)(threadIdx.x >> 5);
    if (job >= 2 * L.n_kv_head) return;
    const int refused = status ? *status : 0;  // (looked at behind the loads, which do not depend on it)
    const bool is_v = job >= L.n_kv_head;
    const int h = is_v ? job - L.n_kv_head : job;
    const int s = blockIdx.z;
    int first_row, n_new;
    S.rows(s, first_row, n_new);
    if (n_new == 0) return;
    const int n_keys = S.keys(s);
    const int pos0 = n_keys - n_new;  // position of the stream's first new token
    const int p_begin = max(pos0, 0) / BKV_BLOCK, p_end = (n_keys + BKV_BLOCK - 1) / BKV_BLOCK;
    for (int p = p_begin + (int)blockIdx.y; p < p_end; p += gridDim.y) {
        const int64_t id = S.page(s, p, L.n_pages);
        const int t0 = max(pos0 - p * BKV_BLOCK, 0);                   // first new slot
        const int t1 = min(n_keys - p * BKV_BLOCK, BKV_BLOCK);         // behind the last one
        const int64_t ld = is_v ? v_ld : k_ld;
        const T* src = (is_v ? v : k) + (int64_t)(first_row + p * BKV_BLOCK - pos0) * ld + h * D + lane * C;
        float x[BKV_BLOCK][C];
#pragma unroll
        for (int t = 0; t < BKV_BLOCK; ++t) load_row<T, C, VEC>(src + min(max(t, t0), t1 - 1) * ld, x[t]);
        if (id < 0 || refused != 0) continue;
        const int64_t head = id * L.n_kv_head + h;
        float* sp = (is_v ? L.vs : L.ks) + head;
        int8_t* q = (is_v ? L.v : L.k) + head * (BKV_BLOCK * D);
        const float s_old = t0 > 0 ? *sp : 0.0f;
        float amax = 0.0f;  // (a new row that stands in for another one changes nothing)
#pragma unroll
        for (int t = 0; t < BKV_BLOCK; ++t)
#pragma unroll
            for (int c = 0; c < C; ++c) amax = fmaxf(amax, fabsf(x[t][c]));
        amax = fminf(warp_max(amax), FLT_MAX);
        const float s_new = fmaxf(s_old, amax * SCALE);
        const float inv = s_new > 0.0f ? __fdiv_rn(1.0f, s_new) : 0.0f;
        const bool grown = t0 > 0 && s_new > s_old;
        const float ratio = grown ? __fdiv_rn(s_old, s_new) : 1.0f;
        if (lane == 0 && (t0 == 0 || grown)) *sp = s_new;
        if (!is_v) {
#pragma unroll
            for (int t = 0; t < BKV_BLOCK; ++t) {
                int8_t* row = q + t * D + lane * C;
                int8_t b[C];
                if (t < t0) {
                    if (!grown) continue;
                    load_bytes<C>(row, b);
#pragma unroll
                    for (int c = 0; c < C; ++c) b[c] = (int8_t)__float2int_rn((float)b[c] * ratio);
                } else if (t < t1) {
#pragma unroll
                    for (int c = 0; c < C; ++c) b[c] = quant(x[t][c], inv);
                } else {
                    continue;
                }
                store_bytes<C>(row, b);
            }
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                uint4* at = reinterpret_cast<uint4*>(q + (int64_t)(lane * C + c) * BKV_BLOCK);
                int8_t b[BKV_BLOCK];
                uint4 u = make_uint4(0, 0, 0, 0);
                if (t0 > 0 || t1 < BKV_BLOCK) u = *at;
                memcpy(b, &u, 16);
#pragma unroll
                for (int t = 0; t < BKV_BLOCK; ++t) {
                    if (t < t0) {
                        if (grown) b[t] = (int8_t)__float2int_rn((float)b[t] * ratio);
                    } else if (t < t1) {
                        b[t] = quant(x[t][c], inv);
                    }
                }
                memcpy(&u, b, 16);
                *at = u;
            }
        }
    }
}

// The values of each stream's last rows, [row][n_kv_head][d_head]; same shape of work.
template <typename T, int D>
__global__ void __launch_bounds__(32 * APPEND_WARPS)
    bkv_read_kernel(BkvLayer L, BkvStreams S, T* __restrict__ k, T* __restrict__ v) {
    pdl_entry();
    constexpr int C = D / 32;
    const int lane = threadIdx.x & 31;
    const int job = (int)blockIdx.x * APPEND_WARPS + (int)(threadIdx.x >> 5);
    if (job >= 2 * L.n_kv_head) return;
    const bool is_v = job >= L.n_kv_head;
    const int h = is_v ? job - L.n_kv_head : job;
    const int s = blockIdx.z;
    int first_row, n_rows;
    S.rows(s, first_row, n_rows);
    const int n_keys = S.keys(s);
    const int pos0 = n_keys - n_rows;
    T* out = (is_v ? v : k) + (int64_t)h * D + lane * C;
    const int64_t ld = (int64_t)L.n_kv_head * D;
    // rows in front of the stream's first position are zero
    for (int i = (int)blockIdx.y; i < -pos0 && i < n_rows; i += gridDim.y)
#pragma unroll
        for (int c = 0; c < C; ++c) out[(int64_t)(first_row + i) * ld + c] = T(0.0f);
    const int p_begin = max(pos0, 0) / BKV_BLOCK, p_end = (n_keys + BKV_BLOCK - 1) / BKV_BLOCK;
    for (int p = p_begin + (int)blockIdx.y; p < p_end; p += gridDim.y) {
        const int64_t id = S.page(s, p, L.n_pages);
        const int t0 = max(pos0 - p * BKV_BLOCK, 0), t1 = min(n_keys - p * BKV_BLOCK, BKV_BLOCK);
        const int64_t head = id * L.n_kv_head + h;
        const float scale = id < 0 ? 0.0f : (is_v ? L.vs : L.ks)[head];
        const int8_t* q = (is_v ? L.v : L.k) + (id < 0 ? 0 : head * (BKV_BLOCK * D));
        T* to = out + (int64_t)(first_row + p * BKV_BLOCK - pos0) * ld;
        int8_t b[BKV_BLOCK][C];
        if (is_v) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint4 u = *reinterpret_cast<const uint4*>(q + (int64_t)(lane * C + c) * BKV_BLOCK);
                int8_t part[BKV_BLOCK];
                memcpy(part, &u, 16);
#pragma unroll
                for (int t = 0; t < BKV_BLOCK; ++t) b[t][c] = part[t];
            }
        } else {
#pragma unroll
            for (int t = 0; t < BKV_BLOCK; ++t) load_bytes<C>(q + t * D + lane * C, b[t]);
        }
#pragma unroll
        for (int t = 0; t < BKV_BLOCK; ++t)
            if (t >= t0 && t < t1) {
                __align__(16) T part[C];
#pragma unroll
                for (int c = 0; c < C; ++c) part[c] = (T)(id < 0 ? 0.0f : (float)b[t][c] * scale);
                store_row<T, C>(to + (int64_t)t * ld, part);
            }
    }
}

dim3 block_grid(const BkvLayer& L, const vkb_bkv_batch* b) {
    const int pages = std::max(1, std::min(ceil_div(b->max_q, BKV_BLOCK) + 1, 4096));
    return dim3((unsigned)ceil_div(2 * L.n_kv_head, APPEND_WARPS), (unsigned)pages, (unsigned)b->n_seq);
}

template <typename T, int D>
void launch_append(vkb_context* ctx, const BkvLayer& L, const vkb_bkv_batch* b, const void* k, int64_t k_ld, const void* v,
                   int64_t v_ld) {
    constexpr int C = D / 32, BYTES = C * (int)sizeof(T);
    constexpr int ALIGN = BYTES % 16 == 0 ? 16 : BYTES % 8 == 0 ? 8 : BYTES % 4 == 0 ? 4 : (int)sizeof(T);
    const bool vec = !(((uintptr_t)k | (uintptr_t)v) % ALIGN) && !((k_ld * (int64_t)sizeof(T)) % ALIGN) &&
                     !((v_ld * (int64_t)sizeof(T)) % ALIGN);
    auto kern = vec ? bkv_append_kernel<T, D, true> : bkv_append_kernel<T, D, false>;
    launch_pdl(ctx, kern, block_grid(L, b), 32 * APPEND_WARPS, 0, L, bkv_streams(b), reinterpret_cast<const T*>(k), k_ld,
               reinterpret_cast<const T*>(v), v_ld, b->status_dev);
    VKB_CUDA(cudaGetLastError());
    ctx->count();
}

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" {

vkb_status vkb_bkv_append(vkb_context* ctx, const vkb_bkv_cache* cache, int32_t layer, const vkb_bkv_batch* batch,
                          const void* k_dev, int64_t k_ld, const void* v_dev, int64_t v_ld, int32_t dtype) {
    return guard([&] {
        const BkvLayer L = bkv_layer(ctx, cache, layer);
        bkv_streams(batch);
        const int64_t width = (int64_t)cache->n_kv_head * cache->d_head;
        if (dtype != VKB_DT_F32 && dtype != VKB_DT_F16) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv_append: dtype must be F32 or F16");
        if (batch->n_seq == 0 || batch->n_tok == 0) return;
        if (!k_dev || !v_dev) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_append: null k/v");
        if (((uintptr_t)k_dev | (uintptr_t)v_dev) % (dtype == VKB_DT_F32 ? 4 : 2))
            fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_append: misaligned k/v");
        if (k_ld < width || v_ld < width) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_append: row stride below n_kv_head*d_head");
        NvtxRange nvtx_range("vkb.bkv.append");
        with_bkv_head(cache->d_head, [&](auto D) {
            if (dtype == VKB_DT_F32) launch_append<float, decltype(D)::value>(ctx, L, batch, k_dev, k_ld, v_dev, v_ld);
            else launch_append<__half, decltype(D)::value>(ctx, L, batch, k_dev, k_ld, v_dev, v_ld);
        });
    });
}

vkb_status vkb_bkv_read(vkb_context* ctx, const vkb_bkv_cache* cache, int32_t layer, const vkb_bkv_batch* batch,
                        void* k_dev, void* v_dev, int32_t dtype) {
    return guard([&] {
        const BkvLayer L = bkv_layer(ctx, cache, layer);
        const BkvStreams S = bkv_streams(batch);
        if (dtype != VKB_DT_F32 && dtype != VKB_DT_F16) fail(VKB_ERROR_UNSUPPORTED_OP, "bkv_read: dtype must be F32 or F16");
        if (batch->n_seq == 0 || batch->n_tok == 0) return;
        if (!k_dev || !v_dev) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_read: null k/v");
        if (((uintptr_t)k_dev | (uintptr_t)v_dev) & 15) fail(VKB_ERROR_INVALID_ARGUMENT, "bkv_read: outputs must be 16-byte aligned");
        NvtxRange nvtx_range("vkb.bkv.read");
        with_bkv_head(cache->d_head, [&](auto D) {
            constexpr int d = decltype(D)::value;
            if (dtype == VKB_DT_F32)
                launch_pdl(ctx, bkv_read_kernel<float, d>, block_grid(L, batch), 32 * APPEND_WARPS, 0, L, S,
                           reinterpret_cast<float*>(k_dev), reinterpret_cast<float*>(v_dev));
            else
                launch_pdl(ctx, bkv_read_kernel<__half, d>, block_grid(L, batch), 32 * APPEND_WARPS, 0, L, S,
                           reinterpret_cast<__half*>(k_dev), reinterpret_cast<__half*>(v_dev));
            VKB_CUDA(cudaGetLastError());
            ctx->count();
        });
    });
}

}  // extern "C"
