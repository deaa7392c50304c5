// pages.cu — the pages of a paged cache, managed on the device: forking, freeing
// and growing streams (with copy on write), and compaction. Tables, lengths and
// reference counts are device arrays, so a beam-search step goes from the
// chosen parents to the attention without a word from the host.
//
// Bound: HBM. The copies of pages dominate (all layers of K, V and scales); the
// tables are read and written once. Which page is taken is fixed by the
// definition (lowest free pages, streams in order), so results do not depend
// on the order in which blocks run; counts are integer adds.
//
// Measured: advance of 64 streams of up to 447 tokens that all fork, 32 layers of
// 20 heads of 64, 34 us (fork 4, plan 9, copies 17: 54 MB each way, 6.2 TB/s);
// compaction that moves 1.1 GB (2 layers, pages of 33 KB), 412 us (count 3, plan 6,
// moves 390: 5.7 TB/s).
#include "common.cuh"
#include <algorithm>

namespace vkb {
namespace {

constexpr int PT = 256;     // threads of the wide kernels
constexpr int PLAN = 1024;  // threads of the planning block
constexpr int COPY_BYTES = 64 * 1024;  // bytes of a page that one block moves: at half of that the loads of a thread in flight
                                       // were one (33 KB a page and layer, 34000 pages: 524 us)
constexpr int CHUNK = 4 * PLAN;        // pages that a planning block looks at

struct Planes {
    int n_layer, n;
    uint8_t* base[VKB_PAGES_MAX_PLANES];
    int64_t page[VKB_PAGES_MAX_PLANES];
    int64_t layer[VKB_PAGES_MAX_PLANES];
    int unit[VKB_PAGES_MAX_PLANES];  // bytes moved at a time: 16, 4 or 1
};

struct State {
    int32_t *table, *len, *refs;
};

struct Pool {
    int64_t n_pages, ld;
    int n_seq, page_tokens;
    int32_t* status;
};

// Scratch of one call. info[0]: why the call cannot be done (0: it can);
// info[1]: pages moved or taken; info[2]: pages in use.
struct Plan {
    int32_t* info;
    int32_t* base;    // [n_seq] length after the fork
    int32_t* first;   // [n_seq] the stream's first entry of `fresh`; compaction: pages in use of each chunk
    int2* copy;       // [n_seq] (source, destination) of a stream's copied page, or (-1, -1)
    int32_t* fresh;   // [n_pages] free pages in order; compaction: destinations
    int32_t* moved;   // [n_pages] compaction: sources
    int32_t* map;     // [n_pages] compaction: where a moved page goes
};

// Sum over the block's threads before this one; `total` over all. Threads: PLAN.
__device__ __forceinline__ int block_scan(int x, int& total) {
    __shared__ int warps[PLAN / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    if (lane == 31) warps[warp] = y;
    __syncthreads();
    if (warp == 0) {
        int w = warps[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += z;
        }
        warps[lane] = w;
    }
    __syncthreads();
    const int before = warp ? warps[warp - 1] : 0;
    total = warps[PLAN / 32 - 1];
    __syncthreads();
    return before + y - x;
}

__device__ __forceinline__ int pages_of(int64_t tokens, int page_tokens) {
    return (int)((tokens + page_tokens - 1) / page_tokens);
}

// The forked tables, the lengths before they grow, and how many tables list each page.
__global__ void __launch_bounds__(PT) pages_fork_kernel(Pool P, const int32_t* __restrict__ parent, State from, State to,
                                                        Plan W) {
    pdl_entry();
    const int s = blockIdx.y;
    const int p = parent ? parent[s] : s;
    int len = 0;
    if (p >= P.n_seq) {
        if (threadIdx.x == 0) atomicMax(&W.info[0], VKB_PAGES_BAD_INPUT);
    } else if (p >= 0) {
        len = from.len[p];
        if (len < 0 || len > P.ld * P.page_tokens) {
            if (threadIdx.x == 0) atomicMax(&W.info[0], VKB_PAGES_BAD_INPUT);
            len = 0;
        }
    }
    const int have = pages_of(len, P.page_tokens);
    if (blockIdx.x == 0 && threadIdx.x == 0) W.base[s] = p >= 0 && p < P.n_seq ? len : -1;
    for (int64_t i = (int64_t)blockIdx.x * PT + threadIdx.x; i < P.ld; i += (int64_t)gridDim.x * PT) {
        int id = -1;
        if (i < have) {
            id = from.table[(int64_t)p * P.ld + i];
            if (id < 0 || id >= P.n_pages) {
                atomicMax(&W.info[0], VKB_PAGES_BAD_INPUT);
                id = -1;
            } else {
                atomicAdd(&to.refs[id], 1);
            }
        }
        to.table[(int64_t)s * P.ld + i] = id;
    }
}

// One block: what each stream takes, the free pages, and the tables with them.
__global__ void __launch_bounds__(PLAN) pages_plan_kernel(Pool P, const int32_t* __restrict__ n_new, State from, State to,
                                                          Plan W) {
    pdl_entry();
    __shared__ int why, found_s;
    const int t = threadIdx.x;
    if (t == 0) why = W.info[0];
    __syncthreads();
    int taken = 0;
    for (int s0 = 0; s0 < P.n_seq; s0 += PLAN) {
        const int s = s0 + t;
        int need = 0;
        int2 copy = make_int2(-1, -1);
        if (s < P.n_seq) {
            const int base = W.base[s];
            const int grow = base >= 0 && n_new ? n_new[s] : 0;
            if (grow < 0) {
                atomicMax(&why, VKB_PAGES_BAD_INPUT);
            } else if (base >= 0) {
                const int have = pages_of(base, P.page_tokens);
                const int64_t want = ((int64_t)base + grow + P.page_tokens - 1) / P.page_tokens;
                if (want > P.ld) {
                    atomicMax(&why, VKB_PAGES_TABLE_FULL);
                } else {
                    need = (int)want - have;
                    if (grow > 0 && base % P.page_tokens) {
                        const int last = to.table[(int64_t)s * P.ld + have - 1];
                        if (last >= 0 && to.refs[last] > 1) {
                            copy.x = last;
                            ++need;
                        }
                    }
                }
            }
        }
        int total;
        const int before = block_scan(need, total);
        if (s < P.n_seq) {
            W.first[s] = taken + before;
            W.copy[s] = copy;
        }
        taken += total;
        if (taken > P.n_pages) break;  // more than there are (a stream takes ld at most, so no sum passes n_seq * ld < 2^31)
    }
    __syncthreads();
    if (why == 0 && taken > 0) {
        int found = 0;
        for (int64_t i0 = 0; i0 < P.n_pages && found < taken; i0 += 4 * PLAN) {
            int free4 = 0, n = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t i = i0 + 4 * t + e;
                if (i < P.n_pages && to.refs[i] == 0 && from.refs[i] == 0) {
                    free4 |= 1 << e;
                    ++n;
                }
            }
            int total;
            int at = found + block_scan(n, total);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (free4 >> e & 1) {
                    if (at < taken) W.fresh[at] = (int)(i0 + 4 * t + e);
                    ++at;
                }
            found += total;
        }
        if (t == 0) found_s = found;
        __syncthreads();
        if (t == 0 && found_s < taken) why = VKB_PAGES_EXHAUSTED;
    }
    __syncthreads();
    if (why) {
        if (t == 0) {
            W.info[0] = why;
            atomicMax(P.status, why);
        }
        return;
    }
    // a warp hands a stream its pages
    const int lane = t & 31;
    for (int s = t >> 5; s < P.n_seq; s += PLAN / 32) {
        const int base = W.base[s];
        const int grow = base >= 0 && n_new ? n_new[s] : 0;
        const int len = max(base, 0);
        const int have = pages_of(len, P.page_tokens), want = pages_of((int64_t)len + grow, P.page_tokens);
        int at = W.first[s];
        int32_t* row = to.table + (int64_t)s * P.ld;
        const int src = W.copy[s].x;
        if (src >= 0) {
            if (lane == 0) {
                const int dst = W.fresh[at];
                W.copy[s].y = dst;
                row[have - 1] = dst;
                to.refs[dst] = 1;
                atomicSub(&to.refs[src], 1);
            }
            ++at;
        }
        for (int i = lane; i < want - have; i += 32) {
            const int id = W.fresh[at + i];
            row[have + i] = id;
            to.refs[id] = 1;
        }
        if (lane == 0) to.len[s] = len + grow;
    }
}

// Moves part `part` of `parts` of one page of one layer.
__device__ __forceinline__ void move_page(const Planes& A, int layer, int64_t src, int64_t dst, int part, int parts) {
    for (int p = 0; p < A.n; ++p) {
        const uint8_t* from = A.base[p] + layer * A.layer[p] + src * A.page[p];
        uint8_t* to = A.base[p] + layer * A.layer[p] + dst * A.page[p];
        const int64_t n = A.page[p] / A.unit[p];
        const int64_t lo = n * part / parts, hi = n * (part + 1) / parts;
        if (A.unit[p] == 16) {
            constexpr int U = 8;
            for (int64_t i = lo + threadIdx.x; i < hi; i += U * PT) {
                uint4 v[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u * PT < hi) v[u] = __ldcs(reinterpret_cast<const uint4*>(from) + i + u * PT);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u * PT < hi) __stcs(reinterpret_cast<uint4*>(to) + i + u * PT, v[u]);
            }
        } else if (A.unit[p] == 4) {
            for (int64_t i = lo + threadIdx.x; i < hi; i += PT)
                reinterpret_cast<uint32_t*>(to)[i] = reinterpret_cast<const uint32_t*>(from)[i];
        } else {
            for (int64_t i = lo + threadIdx.x; i < hi; i += PT) to[i] = from[i];
        }
    }
}

// The copied last pages; or, when the call cannot be done, the old state.
__global__ void __launch_bounds__(PT) pages_copy_kernel(Pool P, Planes A, State from, State to, Plan W, int parts) {
    pdl_entry();
    if (W.info[0] != 0) {
        const int64_t step = (int64_t)gridDim.x * gridDim.y * PT;
        const int64_t first = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * PT + threadIdx.x;
        for (int64_t i = first; i < P.n_seq * P.ld; i += step) to.table[i] = from.table[i];
        for (int64_t i = first; i < P.n_seq; i += step) to.len[i] = from.len[i];
        for (int64_t i = first; i < P.n_pages; i += step) to.refs[i] = from.refs[i];
        return;
    }
    const int2 c = W.copy[blockIdx.y];
    if (c.x < 0) return;
    for (int j = blockIdx.x; j < A.n_layer * parts; j += gridDim.x) move_page(A, j / parts, c.x, c.y, j % parts, parts);
}

// Pages in use of each chunk.
__global__ void __launch_bounds__(PLAN) compact_count_kernel(Pool P, const int32_t* __restrict__ refs, Plan W) {
    pdl_entry();
    int used = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t i = (int64_t)blockIdx.x * CHUNK + e * PLAN + threadIdx.x;
        used += __syncthreads_count(i < P.n_pages && refs[i] > 0);
    }
    if (threadIdx.x == 0) W.first[blockIdx.x] = used;
}

// One block a chunk: which of its pages are holes before the number in use, and which are in use behind it. The place of
// each in its list is a count of pages in use: holes before page i are i - used(i), moves before it used(i) - used(n).
__global__ void __launch_bounds__(PLAN) compact_plan_kernel(Pool P, const int32_t* __restrict__ refs, Plan W, int32_t* n_used) {
    pdl_entry();
    const int t = threadIdx.x, chunks = gridDim.x, me = blockIdx.x;
    __shared__ int before_s, total_s;
    if (t == 0) before_s = total_s = 0;
    __syncthreads();
    for (int c = t; c < chunks; c += PLAN) {
        const int u = W.first[c];
        atomicAdd(&total_s, u);
        if (c < me) atomicAdd(&before_s, u);
    }
    __syncthreads();
    const int n = total_s;  // pages in use: they become pages 0 .. n - 1
    // used(n): whole chunks before n, and the part of the one that n lies in
    __shared__ int below_s;
    if (t == 0) below_s = 0;
    __syncthreads();
    const int at = n / CHUNK;
    for (int c = t; c < at; c += PLAN) atomicAdd(&below_s, W.first[c]);
    int part = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t i = (int64_t)at * CHUNK + e * PLAN + t;
        part += __syncthreads_count(i < n && refs[i] > 0);
    }
    __syncthreads();
    const int below = below_s + part;
    int live = 0, mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t i = (int64_t)me * CHUNK + 4 * t + e;
        if (i < P.n_pages && refs[i] > 0) {
            live |= 1 << e;
            ++mine;
        }
    }
    int total;
    int used = before_s + block_scan(mine, total);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t i = (int64_t)me * CHUNK + 4 * t + e;
        if (i >= P.n_pages) break;
        const bool in_use = live >> e & 1;
        if (i < n && !in_use) W.fresh[i - used] = (int)i;
        if (i >= n && in_use) {
            W.map[i] = used - below;
            W.moved[used - below] = (int)i;
        }
        used += in_use;
    }
    if (me == 0 && t == 0) {
        W.info[1] = n - below;
        W.info[2] = n;
        if (n_used) *n_used = n;
    }
}

// The moved pages of every layer, the tables that list them, and the counts.
__global__ void __launch_bounds__(PT) compact_move_kernel(Pool P, Planes A, State from, State to, Plan W, int parts) {
    pdl_entry();
    const int moves = W.info[1], used = W.info[2];
    const int64_t step = (int64_t)gridDim.x * PT, first = (int64_t)blockIdx.x * PT + threadIdx.x;
    for (int64_t i = first; i < P.n_seq * P.ld; i += step) {
        const int id = from.table[i];
        to.table[i] = id < used || id >= P.n_pages || from.refs[id] <= 0 ? id : W.fresh[W.map[id]];
    }
    for (int64_t i = first; i < P.n_seq; i += step) to.len[i] = from.len[i];
    // a free page before `used` takes its count from the page that comes to it
    for (int64_t i = first; i < P.n_pages; i += step) {
        const int r = from.refs[i];
        if (i >= used) to.refs[i] = 0;
        else if (r > 0) to.refs[i] = r;
    }
    for (int64_t i = first; i < moves; i += step) to.refs[W.fresh[i]] = from.refs[W.moved[i]];
    const int64_t jobs = (int64_t)moves * A.n_layer * parts;
    for (int64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
        const int64_t k = j / parts;
        const int i = (int)(k / A.n_layer);
        move_page(A, (int)(k % A.n_layer), W.moved[i], W.fresh[i], (int)(j % parts), parts);
    }
}

Planes check_planes(const vkb_page_pool* p) {
    if (p->n_layer <= 0) fail(VKB_ERROR_INVALID_ARGUMENT, "pages: n_layer must be > 0");
    if (p->n_planes < 0 || p->n_planes > VKB_PAGES_MAX_PLANES)
        fail(VKB_ERROR_INVALID_ARGUMENT, "pages: n_planes must be in 0.." + std::to_string(VKB_PAGES_MAX_PLANES));
    if (p->n_planes && !p->planes) fail(VKB_ERROR_INVALID_ARGUMENT, "pages: null planes");
    Planes A{};
    A.n_layer = p->n_layer;
    A.n = p->n_planes;
    for (int i = 0; i < A.n; ++i) {
        const vkb_page_plane& q = p->planes[i];
        if (!q.base_dev || q.page_bytes <= 0 || (p->n_layer > 1 && q.layer_bytes < q.page_bytes * p->n_pages))
            fail(VKB_ERROR_INVALID_ARGUMENT, "pages: plane " + std::to_string(i) + " is null, or its layers overlap");
        A.base[i] = reinterpret_cast<uint8_t*>(q.base_dev);
        A.page[i] = q.page_bytes;
        A.layer[i] = q.layer_bytes;
        const uint64_t all = (uint64_t)(uintptr_t)q.base_dev | (uint64_t)q.page_bytes | (p->n_layer > 1 ? (uint64_t)q.layer_bytes : 0);
        A.unit[i] = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    }
    return A;
}

Pool check_pool(const vkb_context* ctx, const vkb_page_pool* p) {
    if (!ctx || !p) fail(VKB_ERROR_INVALID_ARGUMENT, "pages: null context or pool");
    if (p->n_pages <= 0 || p->n_pages > INT32_MAX) fail(VKB_ERROR_INVALID_ARGUMENT, "pages: n_pages must be in 1..2^31-1");
    if (p->n_seq <= 0 || p->n_seq > 65535) fail(VKB_ERROR_INVALID_ARGUMENT, "pages: n_seq must be in 1..65535");
    if (p->page_tokens <= 0 || p->table_ld <= 0 || p->table_ld > INT32_MAX / p->page_tokens)
        fail(VKB_ERROR_INVALID_ARGUMENT, "pages: page_tokens and table_ld must be > 0, a stream below 2^31 tokens");
    if (p->n_seq * p->table_ld > INT32_MAX - 65536) fail(VKB_ERROR_UNSUPPORTED_OP, "pages: tables of 2^31 entries");
    return Pool{p->n_pages, p->table_ld, p->n_seq, p->page_tokens, p->status_dev};
}

bool overlap(const void* a, const void* b, int64_t bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (uintptr_t)bytes && y < x + (uintptr_t)bytes;
}

void check_states(const Pool& P, const vkb_page_state* a, const vkb_page_state* b) {
    if (!a || !b || !a->table_dev || !a->len_dev || !a->refs_dev || !b->table_dev || !b->len_dev || !b->refs_dev)
        fail(VKB_ERROR_INVALID_ARGUMENT, "pages: null state");
    if (overlap(a->table_dev, b->table_dev, P.n_seq * P.ld * 4) || overlap(a->len_dev, b->len_dev, P.n_seq * 4ll) ||
        overlap(a->refs_dev, b->refs_dev, P.n_pages * 4))
        fail(VKB_ERROR_INVALID_ARGUMENT, "pages: the two states must not overlap");
}

Plan make_plan(vkb_context* ctx, const Pool& P) {
    const size_t seq = ((size_t)std::max<int64_t>(P.n_seq, P.n_pages / CHUNK + 1) + 3) & ~(size_t)3, pages = ((size_t)P.n_pages + 3) & ~(size_t)3;
    ctx->ensure_workspace((16 + 4 * seq + 3 * pages) * 4);
    int32_t* w = ctx->workspace.as<int32_t>();
    Plan W;
    W.info = w;
    W.copy = reinterpret_cast<int2*>(w + 16);
    W.base = w + 16 + 2 * seq;
    W.first = W.base + seq;
    W.fresh = W.first + seq;
    W.moved = W.fresh + pages;
    W.map = W.moved + pages;
    return W;
}

// Blocks that share one page of one layer.
int page_parts(const Planes& A) {
    int64_t bytes = 0;
    for (int i = 0; i < A.n; ++i) bytes += A.page[i];
    return (int)std::min<int64_t>(1024, std::max<int64_t>(1, (bytes + COPY_BYTES - 1) / COPY_BYTES));
}

State state_of(const vkb_page_state* s) { return State{s->table_dev, s->len_dev, s->refs_dev}; }

}  // namespace
}  // namespace vkb

using namespace vkb;

extern "C" {

vkb_status vkb_pages_advance(vkb_context* ctx, const vkb_page_pool* pool, const int32_t* parent_dev,
                             const int32_t* n_new_dev, const vkb_page_state* from, const vkb_page_state* to) {
    return guard([&] {
        const Pool P = check_pool(ctx, pool);
        const Planes A = check_planes(pool);
        check_states(P, from, to);
        if (!P.status) fail(VKB_ERROR_INVALID_ARGUMENT, "pages_advance: null status");
        NvtxRange nvtx_range("vkb.pages.advance");
        const Plan W = make_plan(ctx, P);
        const State a = state_of(from), b = state_of(to);
        VKB_CUDA(cudaMemsetAsync(W.info, 0, 16 * sizeof(int32_t), ctx->stream));
        VKB_CUDA(cudaMemsetAsync(b.refs, 0, (size_t)P.n_pages * 4, ctx->stream));
        const unsigned wide = (unsigned)std::min<int64_t>(64, (P.ld + PT - 1) / PT);
        launch_pdl(ctx, pages_fork_kernel, dim3(wide, (unsigned)P.n_seq), PT, 0, P, parent_dev, a, b, W);
        launch_pdl(ctx, pages_plan_kernel, dim3(1), PLAN, 0, P, n_new_dev, a, b, W);
        const int parts = page_parts(A);
        const unsigned per = (unsigned)std::min<int64_t>((int64_t)A.n_layer * parts, 512);
        launch_pdl(ctx, pages_copy_kernel, dim3(per, (unsigned)P.n_seq), PT, 0, P, A, a, b, W, parts);
        VKB_CUDA(cudaGetLastError());
        ctx->count(3);
    });
}

vkb_status vkb_pages_compact(vkb_context* ctx, const vkb_page_pool* pool, const vkb_page_state* from,
                             const vkb_page_state* to, int32_t* n_used_dev) {
    return guard([&] {
        const Pool P = check_pool(ctx, pool);
        const Planes A = check_planes(pool);
        check_states(P, from, to);
        NvtxRange nvtx_range("vkb.pages.compact");
        const Plan W = make_plan(ctx, P);
        const State a = state_of(from), b = state_of(to);
        const unsigned chunks = (unsigned)((P.n_pages + CHUNK - 1) / CHUNK);
        launch_pdl(ctx, compact_count_kernel, dim3(chunks), PLAN, 0, P, a.refs, W);
        launch_pdl(ctx, compact_plan_kernel, dim3(chunks), PLAN, 0, P, a.refs, W, n_used_dev);
        launch_pdl(ctx, compact_move_kernel, dim3((unsigned)(8 * ctx->sm_count)), PT, 0, P, A, a, b, W, page_parts(A));
        VKB_CUDA(cudaGetLastError());
        ctx->count(3);
    });
}

}  // extern "C"
