// bkv_attn.cuh — the two attention kernels of the block-scaled KV cache.
#pragma once
#include "bkv.cuh"

namespace vkb {

// One call of vkb_bkv_attention.
struct BkvAttn {
    BkvLayer L;
    BkvStreams S;
    int d_head, group, n_head, max_q;
    int max_kv;  // tokens of the longest stream; 0: not known
    const void* q;
    int64_t q_ld;
    float scale;
    void* out;
    int64_t out_ld;
    int q_f16, out_f16;
};

// Few rows a stream and KV head: bound by the cache's bytes (bkv_attn.cu).
void run_bkv_attn(vkb_context* ctx, const BkvAttn& a);
// Many rows: bound by the tensor cores (bkv_prompt.cu). True where it takes the call's types, sizes and alignment
// and has enough row tiles to be the faster one.
bool bkv_prompt_takes(const vkb_context* ctx, const BkvAttn& a);
void run_bkv_prompt(vkb_context* ctx, const BkvAttn& a);

}  // namespace vkb
