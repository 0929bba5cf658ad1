// Trees of drafted tokens: their masks and positions from the draft that each one follows, and the acceptance of a path of them once the model has drawn a token
// behind every draft.
//
// A sequence's drafts are its new tokens of a step (wf_paged_plan), in an order in which every draft stands behind the one that it follows; the first one is the
// token drawn last, which is not in the cache yet.  Draft i sees j where j = i or j stands on the way from i up to a draft that follows none: with up_k the 2^k-th
// step up, seen_{k+1}(i) = seen_k(i) | seen_k(up_k(i)), up_{k+1}(i) = up_k(up_k(i)), so that a tree of depth d takes log2 d rounds.
//
// Acceptance: a draft fits where its token is the one that was drawn behind the draft that it follows (of equal siblings the first one does); the path goes from
// the first draft to the one that fits behind it, and on.  With the tokens drawn from the model's own distribution, so is the path.  The keys and values of the
// path's drafts, of all layers, then move up to where the path would have put them, and pages behind the last of them go back on the free list.
#include <cuda_fp16.h>

#include "attn_chunks.cuh"
#include "wf_bitnet.h"

namespace wf {

namespace {

typedef unsigned long long u64;

constexpr int TR_MAX = 256;                            // drafts of a sequence
constexpr int TR_WORDS = TR_MAX / 64;

struct TreePlanParams {
    const int32_t *parents, *offsets, *seq;
    int rows, tokens, max_nodes;
    u64* mask;
    int32_t* positions;
};

// A sequence's share of the token list, whatever stands in `offsets`
__device__ __forceinline__ void tr_span(const int32_t* offsets, int b, int tokens, int& first, int& n) {
    first = min(max(offsets[b], 0), tokens);
    n = min(max(offsets[b + 1], first), tokens) - first;
}

// A block per sequence, a thread per draft.  A chain of latencies: a launch, the offsets, the parents, a few rounds of two barriers, the stores.  8 trees of 60: 3.3 us; 256 of
// 256: 6.2.
template <int W>
__global__ void __launch_bounds__(64 * W) tree_plan_kernel(const __grid_constant__ TreePlanParams p) {
    __shared__ u64 seen_s[64 * W][W];
    __shared__ int up_s[64 * W];
    const int i = threadIdx.x;
    pdl_wait_prior();
    pdl_launch_dependents();
    int first, n;
    tr_span(p.offsets, blockIdx.x, p.tokens, first, n);
    const int len = p.seq[blockIdx.x], front = p.offsets[0], end = min(max(p.offsets[p.rows], 0), p.tokens);
    const bool fits = n <= p.max_nodes && len >= 0 && len <= 0x7fffffff - TR_MAX;
    if (fits) {
        int up = -1;
        u64 seen[W];
#pragma unroll
        for (int w = 0; w < W; ++w) seen[w] = w == i >> 6 ? 1ull << (i & 63) : 0ull;
        if (i < n) {
            up = p.parents[first + i];
            if (up < 0 || up >= i) up = -1;            // a draft can only follow one in front of it
        }
        while (__syncthreads_or(up >= 0)) {
            up_s[i] = up;
#pragma unroll
            for (int w = 0; w < W; ++w) seen_s[i][w] = seen[w];
            __syncthreads();
            if (up >= 0) {
#pragma unroll
                for (int w = 0; w < W; ++w) seen[w] |= seen_s[up][w];
                up = up_s[up];
            }
        }
        if (i < n) {
            int depth = -1;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                depth += __popcll(seen[w]);
                p.mask[(size_t)(first + i) * W + w] = seen[w];
            }
            p.positions[first + i] = len + depth;
        }
    } else {
        for (int k = i; k < n; k += 64 * W) {
            for (int w = 0; w < W; ++w) p.mask[(size_t)(first + k) * W + w] = 0ull;
            p.positions[first + k] = -1;
        }
    }
    auto nothing = [&](int from, int to) {             // rows of no sequence
        for (int k = from + blockIdx.x * 64 * W + i; k < to; k += gridDim.x * 64 * W) {
            for (int w = 0; w < W; ++w) p.mask[(size_t)k * W + w] = 0ull;
            p.positions[k] = 0;
        }
    };
    nothing(0, min(front, end));
    nothing(end, p.tokens);
}

struct AcceptParams {
    const int32_t *parents, *tokens, *targets, *offsets, *seq;
    int rows, n_tokens;
    int32_t *accepted, *path, *next;
    // the cache
    unsigned char* pool;
    float* scales;                                     // int8 pools
    int layers, kv_heads, page_size, max_pages, row_bytes;
    const int32_t* table;
    int max_blocks;
    int32_t* free_pages;
    int pool_pages;
    const int32_t* free_count;
    int32_t *lens_out, *count_out, *status;
};

constexpr int AC_WARPS = 4;                            // sequences of a block: few, so that a small batch has an SM each

// A warp per sequence.  Which draft fits behind each one is settled by all lanes at once (the lowest of them, by atomicMin: the result has no order); the path is
// then a chase through shared memory.
__global__ void __launch_bounds__(AC_WARPS * 32) tree_accept_kernel(const __grid_constant__ AcceptParams p) {
    __shared__ int want_s[AC_WARPS][TR_MAX], first_s[AC_WARPS][TR_MAX], path_s[AC_WARPS][TR_MAX];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x * AC_WARPS + warp;
    int *want = want_s[warp], *behind = first_s[warp], *path = path_s[warp];
    pdl_wait_prior();
    pdl_launch_dependents();
    if (b < p.rows) {
        int first, n;
        tr_span(p.offsets, b, p.n_tokens, first, n);
        int kept = 0, last = -1;
        if (n > 0 && n <= TR_MAX) {
            int up[TR_WORDS * 2], tok[TR_WORDS * 2];
#pragma unroll
            for (int k = 0; k < TR_WORDS * 2; ++k) {
                const int j = k * 32 + lane;
                up[k] = j < n ? p.parents[first + j] : -1;
                tok[k] = j < n ? p.tokens[first + j] : 0;
                if (j < n) { want[j] = p.targets[first + j]; behind[j] = TR_MAX; }
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < TR_WORDS * 2; ++k) {
                const int j = k * 32 + lane;
                if (j < n && up[k] >= 0 && up[k] < j && want[up[k]] == tok[k]) atomicMin(&behind[up[k]], j);
            }
            __syncwarp();
            int at = 0;                                // every lane takes the same steps
            do {
                if (lane == 0) path[kept] = at;
                ++kept;
                last = at;
                at = behind[at];
            } while (at < TR_MAX);
            __syncwarp();
        }
        for (int k = lane; k < n; k += 32) p.path[first + k] = k < kept ? path[k] : -1;
        if (lane == 0) {
            p.accepted[b] = kept;
            p.next[b] = kept ? want[last] : -1;
        }
    }
    const int front = p.offsets[0], end = p.rows ? min(max(p.offsets[p.rows], 0), p.n_tokens) : 0;
    auto nothing = [&](int from, int to) {             // rows of no sequence
        for (int k = from + blockIdx.x * blockDim.x + threadIdx.x; k < to; k += gridDim.x * blockDim.x) p.path[k] = -1;
    };
    nothing(0, min(front, end));
    nothing(end, p.n_tokens);
}

__device__ __forceinline__ int ac_blocks(int tokens, int page) { return (int)(((unsigned)tokens + page - 1) / page); }

// pages that sequence b hands back, or the bits of why it cannot (negative)
__device__ __forceinline__ int ac_freed(const AcceptParams& p, int b) {
    int first, n;
    tr_span(p.offsets, b, p.n_tokens, first, n);
    const int len = p.seq[b];
    if (len < 0 || n > TR_MAX || len > 0x7fffffff - n) return -WF_PLAN_LENGTH;
    const int old = ac_blocks(len + n, p.page_size);
    return old > p.max_blocks ? -WF_PLAN_BLOCKS : old - ac_blocks(len + p.accepted[b], p.page_size);
}

// Moves, and one block (the last) for the free list.  Every block first sums what all sequences hand back, for nothing is done where that does not fit.  A thread
// owns 16 bytes of a head's row in one layer and takes the path's tokens in order: it reads token k from its draft's place path[k] >= k and writes it to place k, which
// only tokens behind k can still be read from.  Four tokens are under way at a time.  With the acceptance 9.6 us for 8 sequences of 60 drafts and 30 layers of 5 heads, 16 for 64 and
// 32 layers of 8 (33 MB): chains of loads, two waves of blocks (one, with two pieces a thread: the same).
constexpr int AC_THREADS = 256;
__global__ void __launch_bounds__(AC_THREADS) tree_move_kernel(const __grid_constant__ AcceptParams p, int per_row) {
    __shared__ int path_s[TR_MAX], sum_s[AC_THREADS / 32], flag_s[AC_THREADS / 32];
    __shared__ unsigned src_s[TR_MAX], dst_s[TR_MAX];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait_prior();
    pdl_launch_dependents();
    const bool last = blockIdx.x == gridDim.x - 1;
    const int count = *p.free_count;
    const int per = (p.rows + AC_THREADS - 1) / AC_THREADS, r0 = tid * per, r1 = min(p.rows, r0 + per);
    int status = count < 0 || count > p.pool_pages ? WF_PLAN_COUNT : 0, mine = 0;              // (at most 8192 x 256 pages)
    for (int r = r0; r < r1; ++r) {
        const int f = ac_freed(p, r);
        if (f < 0) status |= -f; else mine += f;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += y; }
    status = (int)__reduce_or_sync(0xffffffffu, (unsigned)status);
    if (lane == 31) { sum_s[warp] = incl; flag_s[warp] = status; }
    __syncthreads();
    int total = 0, before = incl - mine;
#pragma unroll
    for (int w = 0; w < AC_THREADS / 32; ++w) { if (w < warp) before += sum_s[w]; total += sum_s[w]; status |= flag_s[w]; }
    if ((long long)count + total > p.pool_pages) status |= WF_PLAN_PAGES;
    if (last) {
        for (int r = r0; r < r1; ++r) {
            int first, n;
            tr_span(p.offsets, r, p.n_tokens, first, n);
            const int len = p.seq[r], kept = p.accepted[r];
            p.lens_out[r] = status ? (int)((unsigned)len + n) : len + kept;
            if (!status) {
                const int from = ac_blocks(len + kept, p.page_size), to = ac_blocks(len + n, p.page_size);
                for (int k = from; k < to; ++k) p.free_pages[count + before++] = p.table[(size_t)r * p.max_blocks + k];
            }
        }
        if (tid == 0) { *p.status = status; *p.count_out = count + (status ? 0 : total); }
        return;
    }
    if (status) return;
    const int b = blockIdx.x / per_row, part = blockIdx.x - b * per_row;
    const int kept = p.accepted[b], len = p.seq[b];
    int first, n;
    tr_span(p.offsets, b, p.n_tokens, first, n);
    int moved = 0;
    for (int k = tid; k < kept; k += AC_THREADS) {
        int j = p.path[first + k];
        if (j < k || j >= n) j = k;                    // (where offsets do not rise, another sequence may have written there: no place outside this one's drafts is looked up)
        path_s[k] = j;
        const int from = len + j, to = len + k;
        const int fp = p.table[(size_t)b * p.max_blocks + from / p.page_size], tp = p.table[(size_t)b * p.max_blocks + to / p.page_size];
        const bool ok = fp >= 0 && fp < p.max_pages && tp >= 0 && tp < p.max_pages;
        src_s[k] = ok ? (unsigned)fp : 0xffffffffu;
        dst_s[k] = (unsigned)tp;
        moved |= j != k;
    }
    if (!__syncthreads_or(moved)) return;
    int k0 = 0;
    while (path_s[k0] == k0) ++k0;                     // the path's start that is in place already (a draft behind it moves)
    const int pieces = p.row_bytes / 16, rows = p.layers * 2 * p.kv_heads;
    const int x = part * AC_THREADS + tid;
    if (x < rows * pieces) {
        const int row = x / pieces, c = x - row * pieces;              // row: (layer, K | V, head)
        auto at = [&](unsigned page, int pos) { return reinterpret_cast<uint4*>(p.pool + (((size_t)page * rows + row) * p.page_size + pos % p.page_size) * p.row_bytes) + c; };
        for (int k = k0; k < kept; k += 4) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k + u < kept && src_s[k + u] != 0xffffffffu) v[u] = *at(src_s[k + u], len + path_s[k + u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k + u < kept && src_s[k + u] != 0xffffffffu) *at(dst_s[k + u], len + k + u) = v[u];
        }
    } else if (p.scales && x < rows * pieces + rows) {
        const int row = x - rows * pieces;
        auto at = [&](unsigned page, int pos) { return p.scales + ((size_t)page * rows + row) * p.page_size + pos % p.page_size; };
        for (int k = k0; k < kept; k += 4) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k + u < kept && src_s[k + u] != 0xffffffffu) v[u] = *at(src_s[k + u], len + path_s[k + u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k + u < kept && src_s[k + u] != 0xffffffffu) *at(dst_s[k + u], len + k + u) = v[u];
        }
    }
}

}  // namespace

}  // namespace wf

using namespace wf;

extern "C" int wf_tree_plan(const int32_t* parents, const int32_t* offsets, const int32_t* seq_lens, int rows, int tokens, int max_nodes, uint64_t* mask, int32_t* positions, void* stream) {
    const char* who = "wf_tree_plan";
    if (rows < 0 || tokens < 0 || max_nodes <= 0) { set_error("%s: bad size (%d sequences, %d tokens, trees of %d)", who, rows, tokens, max_nodes); return WF_ERR_INVALID; }
    if (max_nodes > TR_MAX) { set_error("%s: a tree has at most %d drafts (got %d)", who, TR_MAX, max_nodes); return WF_ERR_UNSUPPORTED; }
    if (tokens > 1 << 30 || rows > 1 << 20) { set_error("%s: at most 2^30 tokens and 2^20 sequences", who); return WF_ERR_UNSUPPORTED; }
    if (tokens == 0) return WF_OK;
    if (!mask || !positions || !offsets || (rows > 0 && (!parents || !seq_lens))) { set_error("%s: null pointer", who); return WF_ERR_INVALID; }
    if ((uintptr_t)mask & 7) { set_error("%s: the mask must be 8-byte aligned", who); return WF_ERR_INVALID; }
    const int words = (max_nodes + 63) / 64;
    TreePlanParams p = {};
    p.parents = parents; p.offsets = offsets; p.seq = seq_lens; p.rows = rows; p.tokens = tokens; p.max_nodes = max_nodes;
    p.mask = (u64*)mask; p.positions = positions;
    if (rows == 0) {                                   // no sequence: rows of none
        if (int rc = cuda_check(cudaMemsetAsync(mask, 0, (size_t)tokens * words * 8, (cudaStream_t)stream), who)) return rc;
        return cuda_check(cudaMemsetAsync(positions, 0, (size_t)tokens * 4, (cudaStream_t)stream), who);
    }
    cudaStream_t s = (cudaStream_t)stream;
    const dim3 grid((unsigned)rows);
    switch (words) {
        case 1: return launch_check(launch_pdl(tree_plan_kernel<1>, grid, 64, 0, s, p), who);
        case 2: return launch_check(launch_pdl(tree_plan_kernel<2>, grid, 128, 0, s, p), who);
        case 3: return launch_check(launch_pdl(tree_plan_kernel<3>, grid, 192, 0, s, p), who);
        default: return launch_check(launch_pdl(tree_plan_kernel<4>, grid, 256, 0, s, p), who);
    }
}

extern "C" int wf_tree_accept(const int32_t* parents, const int32_t* tokens, const int32_t* targets, const int32_t* offsets, const int32_t* seq_lens, int rows, int n_tokens,
                              const wf_kv_layout* kv, const int32_t* block_table, int max_blocks, int32_t* free_pages, int pool_pages, const int32_t* free_count, int32_t* accepted,
                              int32_t* path, int32_t* next_tokens, int32_t* lens_out, int32_t* free_count_out, int32_t* status, void* stream) {
    const char* who = "wf_tree_accept";
    if (rows < 0 || n_tokens < 0 || max_blocks < 0 || pool_pages < 0) { set_error("%s: negative size", who); return WF_ERR_INVALID; }
    if (!kv || !kv->pool) { set_error("%s: null kv layout/pool", who); return WF_ERR_INVALID; }
    if (kv->max_pages <= 0 || kv->layers <= 0 || kv->kv_heads <= 0 || kv->page_size <= 0 || kv->head_dim <= 0) { set_error("%s: bad kv layout", who); return WF_ERR_INVALID; }
    const int es = kv->dtype == WF_F32 ? 4 : kv->dtype == WF_BF16 ? 2 : kv->dtype == WF_I8 ? 1 : 0;
    if (!es) { set_error("%s: pool must be f32, bf16 or int8", who); return WF_ERR_UNSUPPORTED; }
    if ((long long)kv->head_dim * es % 16 || kv->head_dim > 1 << 16) { set_error("%s: a head's row must be a multiple of 16 bytes (head_dim %d)", who, kv->head_dim); return WF_ERR_UNSUPPORTED; }
    if (rows > 8192) { set_error("%s: at most 8192 sequences (got %d)", who, rows); return WF_ERR_UNSUPPORTED; }
    if (n_tokens > 1 << 30 || pool_pages > 1 << 30) { set_error("%s: at most 2^30 tokens, and a free list of 2^30 entries", who); return WF_ERR_UNSUPPORTED; }
    if (!offsets || !free_count || !free_count_out || !status || (rows > 0 && (!seq_lens || !accepted || !next_tokens || !lens_out)) || (n_tokens > 0 && (!path || !parents || !tokens || !targets)) ||
        (rows > 0 && max_blocks > 0 && !block_table) || (pool_pages > 0 && !free_pages)) { set_error("%s: null pointer", who); return WF_ERR_INVALID; }
    if ((uintptr_t)kv->pool & 15) { set_error("%s: the pool must be 16-byte aligned", who); return WF_ERR_INVALID; }
    AcceptParams p = {};
    p.parents = parents; p.tokens = tokens; p.targets = targets; p.offsets = offsets; p.seq = seq_lens; p.rows = rows; p.n_tokens = n_tokens;
    p.accepted = accepted; p.path = path; p.next = next_tokens;
    p.pool = (unsigned char*)kv->pool; p.scales = kv_scales_of(kv); p.layers = kv->layers; p.kv_heads = kv->kv_heads; p.page_size = kv->page_size; p.max_pages = kv->max_pages;
    p.row_bytes = kv->head_dim * es;
    p.table = block_table; p.max_blocks = max_blocks; p.free_pages = free_pages; p.pool_pages = pool_pages; p.free_count = free_count;
    p.lens_out = lens_out; p.count_out = free_count_out; p.status = status;
    const long long items = (long long)p.layers * 2 * p.kv_heads * (p.row_bytes / 16 + (p.scales ? 1 : 0)), per_row = (items + AC_THREADS - 1) / AC_THREADS;
    if (items > 1 << 30 || per_row * rows + 1 > 0x7fffffffll) { set_error("%s: too many layers and heads", who); return WF_ERR_UNSUPPORTED; }
    cudaStream_t s = (cudaStream_t)stream;
    if (rows > 0 || n_tokens > 0)
        if (int rc = launch_check(launch_pdl(tree_accept_kernel, dim3((unsigned)(rows > 0 ? (rows + AC_WARPS - 1) / AC_WARPS : 1)), AC_WARPS * 32, 0, s, p), who)) return rc;
    return launch_check(launch_pdl(tree_move_kernel, dim3((unsigned)(per_row * rows + 1)), AC_THREADS, 0, s, p, (int)per_row), who);
}
