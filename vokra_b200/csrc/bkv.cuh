// bkv.cuh — what the kernels of the block-scaled 8-bit KV cache share.
#pragma once
#include "common.cuh"

namespace vkb {

constexpr int BKV_BLOCK = VKB_BKV_BLOCK;

// One layer of the cache, as the kernels see it.
struct BkvLayer {
    int8_t* k;         // [n_pages][n_kv_head][16][d_head]
    int8_t* v;         // [n_pages][n_kv_head][d_head][16]
    float* ks;         // [n_pages][n_kv_head]
    float* vs;
    int64_t n_pages;
    int n_kv_head;
};

// The streams of a call.
struct BkvStreams {
    int n_seq, n_tok;
    const int32_t* start;  // [n_seq + 1]
    const int32_t* len;    // [n_seq]
    const int32_t* table;  // [n_seq][ld]
    int64_t ld;

    __device__ __forceinline__ int keys(int s) const {
        const int64_t n = len[s], cap = ld * BKV_BLOCK;
        return (int)(n < 0 ? 0 : n > cap ? cap : n);
    }
    // First row of a stream and its row count, inside [0, n_tok].
    __device__ __forceinline__ void rows(int s, int& first, int& n) const {
        first = min(max(start[s], 0), n_tok);
        n = max(0, min(start[s + 1], n_tok) - first);
    }
    // Page id of the stream's p-th page; -1 where it has none inside the arena.
    __device__ __forceinline__ int64_t page(int s, int64_t p, int64_t n_pages) const {
        if (p >= ld) return -1;
        const int64_t id = table[(int64_t)s * ld + p];
        return id >= 0 && id < n_pages ? id : -1;
    }
};

BkvLayer bkv_layer(const vkb_context* ctx, const vkb_bkv_cache* c, int layer);
BkvStreams bkv_streams(const vkb_bkv_batch* b);

// Calls f(std::integral_constant<int, D>{}) for a head size that the cache takes.
template <class F>
inline void with_bkv_head(int d_head, F&& f) {
    switch (d_head) {
        case 32: f(std::integral_constant<int, 32>{}); break;
        case 64: f(std::integral_constant<int, 64>{}); break;
        case 96: f(std::integral_constant<int, 96>{}); break;
        case 128: f(std::integral_constant<int, 128>{}); break;
        case 256: f(std::integral_constant<int, 256>{}); break;
        default: fail(VKB_ERROR_UNSUPPORTED_OP, "bkv: d_head must be 32, 64, 96, 128 or 256 (got " + std::to_string(d_head) + ")");
    }
}

}  // namespace vkb
