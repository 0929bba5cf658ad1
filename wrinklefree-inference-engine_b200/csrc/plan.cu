// Block tables and slot maps of a step, built on the GPU from the lengths of its requests, and the way back of a finished request's pages.
//
// The free list is the stack of sgl_kernel.kvcache.PageAllocator (tests/test_kv_cache_cpp.py:44-70 of the reference) in device memory: pages come off its
// end, request after request and block after block, and a step that cannot be served as a whole takes nothing.  With p tokens a page, request b of s_b
// cached and n_b new tokens needs ceil((s_b + n_b) / p) - ceil(s_b / p) pages; two exclusive sums over the requests say where its tokens lie in the step's
// flat token list and where its pages lie in the stack.
//
// One launch, and no block waits for another: every block sums over all requests for itself (8 bytes each, from L2 for all but the first) into shared
// memory and then takes its share of the tokens, four to a thread, and of the new pages, each finding its request by bisection.  What one block writes no
// other reads: a token's page comes from the stack, or from a table entry that was there before the step.
//
// A chain of latencies: a launch, the lengths, the sums (two barriers), a bisection in shared memory, a page, the stores: 3.3 us for 32 requests, 3.9 for 256 with
// 24576 token slots, 7.8 for 2048 with 524288 (8.5 MB, 1.3 at the copy rate); a release of 512 requests 3.5.
#include "kernels.cuh"
#include "wf_bitnet.h"

namespace wf {

namespace {

constexpr int PL_THREADS = 512;                       // at most
constexpr int PL_MAX_ROWS = 8192;                     // four numbers of every request: 128 KB of shared memory

struct PlanParams {
    const int32_t *seq, *fresh;    // cached and new tokens of each request
    const uint8_t* done;           // release: requests that hand their pages back
    int32_t* table;
    int32_t* free_pages;
    const int32_t* free_count;
    int rows, max_blocks, pool_pages, page, cap;
    uint32_t mul, shift;           // x / page = x * mul >> shift for x below 2^31
    int32_t *positions, *token_rows, *pages, *slots, *offsets, *lens_out, *count_out, *status;
};

__device__ __forceinline__ int pl_div(const PlanParams& p, int x) { return (int)((unsigned long long)(unsigned)x * p.mul >> p.shift); }
__device__ __forceinline__ int pl_blocks(const PlanParams& p, int x) { return x > 0 ? pl_div(p, x - 1) + 1 : 0; }
__device__ __forceinline__ long long pl_warp_scan(long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long y = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += y; }
    return v;
}
// the last i of [0, n) with first[i] <= x (first[0] == 0 <= x)
__device__ __forceinline__ int pl_find(const int* first, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (first[mid] <= x) lo = mid; else hi = mid; }
    return lo;
}

// Sums over the requests.  tok[i], blk[i]: tokens and pages in front of request i (entry `rows`: all of them); seq[i], old[i]: its cached tokens and their pages.
// Returns the status, the same in every thread; with a status the sums mean nothing.
template <bool RELEASE>
__device__ __forceinline__ int pl_sums(const PlanParams& p, int count, int* tok, int* blk, int* seq, int* old) {
    __shared__ long long w_tok[32], w_blk[32];
    __shared__ int w_status[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    const int per = (p.rows + blockDim.x - 1) / blockDim.x, r0 = tid * per, r1 = min(p.rows, r0 + per);
    int status = count < 0 || count > p.pool_pages ? WF_PLAN_COUNT : 0;
    long long nt = 0, nb = 0;
    for (int r = r0; r < r1; ++r) {
        const int s = p.seq[r];
        seq[r] = s;
        if (RELEASE) {
            if (s < 0) status |= WF_PLAN_LENGTH;
            const int have = p.done[r] ? pl_blocks(p, s) : 0;
            if (have > p.max_blocks) status |= WF_PLAN_BLOCKS;
            blk[r] = have;
            nb += have;
        } else {
            const int n = p.fresh[r];
            if (s < 0 || n < 0 || s > 0x7fffffff - n) status |= WF_PLAN_LENGTH;
            else {
                const int before = pl_blocks(p, s), after = pl_blocks(p, s + n), need = after - before;
                old[r] = before;
                if (after > p.max_blocks) status |= WF_PLAN_BLOCKS;
                tok[r] = n;
                blk[r] = need;
                nt += n;
                nb += need;
            }
        }
    }
    const long long it = RELEASE ? 0 : pl_warp_scan(nt, lane), ib = pl_warp_scan(nb, lane);
    status = (int)__reduce_or_sync(0xffffffffu, (unsigned)status);
    if (lane == 31) { w_tok[warp] = it; w_blk[warp] = ib; w_status[warp] = status; }
    __syncthreads();
    long long bt = it - nt, bb = ib - nb, at = 0, ab = 0;
    for (int w = 0; w < nw; ++w) { if (w == warp) { bt += at; bb += ab; } at += w_tok[w]; ab += w_blk[w]; status |= w_status[w]; }
    if (RELEASE ? count + ab > p.pool_pages : ab > count) status |= WF_PLAN_PAGES;
    if (!RELEASE && at > p.cap) status |= WF_PLAN_TOKENS;
    if (!status) {                                     // every sum is below 2^31 now
        int t = (int)bt, b = (int)bb;
        for (int r = r0; r < r1; ++r) {
            const int nb_r = blk[r];
            blk[r] = b;
            b += nb_r;
            if (!RELEASE) { const int nt_r = tok[r]; tok[r] = t; t += nt_r; }
        }
        if (tid == 0) { blk[p.rows] = (int)ab; if (!RELEASE) tok[p.rows] = (int)at; }
    }
    __syncthreads();
    return status;
}

__global__ void __launch_bounds__(PL_THREADS) paged_plan_kernel(const __grid_constant__ PlanParams p) {
    extern __shared__ int pl_smem[];
    int *tok = pl_smem, *blk = tok + p.rows + 1, *seq = blk + p.rows + 1, *old = seq + p.rows + 1;
    pdl_wait_prior();
    pdl_launch_dependents();
    const int count = *p.free_count, status = pl_sums<false>(p, count, tok, blk, seq, old);
    const int total = status || !p.rows ? 0 : tok[p.rows], n_pages = status || !p.rows ? 0 : blk[p.rows];
    const int first = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
    if (blockIdx.x == gridDim.x - 1) {
        for (int r = threadIdx.x; r < p.rows; r += blockDim.x) {
            p.offsets[r] = status ? 0 : tok[r];
            p.lens_out[r] = seq[r] + (status ? 0 : tok[r + 1] - tok[r]);
        }
        if (threadIdx.x == 0) { p.offsets[p.rows] = total; *p.count_out = count - n_pages; *p.status = status; }
    }
    for (int q = first; q < (p.cap + 3) / 4; q += step) {
        int pos[4] = {0, 0, 0, 0}, row[4] = {-1, -1, -1, -1}, page[4] = {-1, -1, -1, -1}, slot[4] = {0, 0, 0, 0};
        if (4 * q < total) {
            int r = pl_find(tok, p.rows, 4 * q);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = 4 * q + k;
                if (t >= total) break;
                while (t >= tok[r + 1]) ++r;           // requests without new tokens are passed over
                pos[k] = seq[r] + (t - tok[r]);
                const int b = pl_div(p, pos[k]), fresh = b - old[r];
                row[k] = r;
                slot[k] = pos[k] - b * p.page;
                page[k] = fresh < 0 ? p.table[(size_t)r * p.max_blocks + b] : p.free_pages[count - 1 - (blk[r] + fresh)];
            }
        }
        if (4 * q + 4 <= p.cap) {
            reinterpret_cast<int4*>(p.positions)[q] = make_int4(pos[0], pos[1], pos[2], pos[3]);
            reinterpret_cast<int4*>(p.token_rows)[q] = make_int4(row[0], row[1], row[2], row[3]);
            reinterpret_cast<int4*>(p.pages)[q] = make_int4(page[0], page[1], page[2], page[3]);
            reinterpret_cast<int4*>(p.slots)[q] = make_int4(slot[0], slot[1], slot[2], slot[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (4 * q + k < p.cap) { p.positions[4 * q + k] = pos[k]; p.token_rows[4 * q + k] = row[k]; p.pages[4 * q + k] = page[k]; p.slots[4 * q + k] = slot[k]; }
        }
    }
    for (int k = first; k < n_pages; k += step) {
        const int r = pl_find(blk, p.rows, k);
        p.table[(size_t)r * p.max_blocks + old[r] + (k - blk[r])] = p.free_pages[count - 1 - k];
    }
}

__global__ void __launch_bounds__(PL_THREADS) paged_release_kernel(const __grid_constant__ PlanParams p) {
    extern __shared__ int pl_smem[];
    int *blk = pl_smem, *seq = blk + p.rows + 1;
    pdl_wait_prior();
    pdl_launch_dependents();
    const int count = *p.free_count, status = pl_sums<true>(p, count, nullptr, blk, seq, nullptr);
    const int n_pages = status || !p.rows ? 0 : blk[p.rows];
    if (blockIdx.x == gridDim.x - 1) {
        for (int r = threadIdx.x; r < p.rows; r += blockDim.x) p.lens_out[r] = !status && p.done[r] ? 0 : seq[r];
        if (threadIdx.x == 0) *p.count_out = count + n_pages;
    }
    for (int k = blockIdx.x * blockDim.x + threadIdx.x; k < n_pages; k += gridDim.x * blockDim.x) {
        const int r = pl_find(blk, p.rows, k);
        p.free_pages[count + k] = p.table[(size_t)r * p.max_blocks + (k - blk[r])];
    }
}

int pl_check(const char* who, PlanParams& p) {
    if (p.rows < 0 || p.max_blocks < 0 || p.pool_pages < 0 || p.cap < 0) { set_error("%s: negative size", who); return WF_ERR_INVALID; }
    if (p.page <= 0) { set_error("%s: page_size must be positive (got %d)", who, p.page); return WF_ERR_INVALID; }
    if (p.cap > 1 << 30) { set_error("%s: max_tokens is at most 2^30 (got %d)", who, p.cap); return WF_ERR_UNSUPPORTED; }
    if (p.pool_pages > 1 << 30) { set_error("%s: a free list is at most 2^30 entries (got %d)", who, p.pool_pages); return WF_ERR_UNSUPPORTED; }      // what a block's step adds to an index fits too
    if (p.rows > PL_MAX_ROWS) { set_error("%s: at most %d requests (got %d)", who, PL_MAX_ROWS, p.rows); return WF_ERR_UNSUPPORTED; }
    // with 2^(l-1) < page <= 2^l, mul = ceil(2^(31+l) / page) is below 2^32 and exceeds 2^(31+l) / page by less than 1: x * mul / 2^(31+l) is above x / page by less
    // than 2^-l <= 1 / page, which does not reach the next whole number
    uint32_t l = 0;
    while (l < 31 && (1u << l) < (uint32_t)p.page) ++l;
    p.shift = 31 + l;
    p.mul = (uint32_t)(((1ull << p.shift) + p.page - 1) / p.page);
    return WF_OK;
}

DevMade g_pl_attr;

int pl_attrs() {
    return g_pl_attr.once([]() -> int {
        if (cuda_check(cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * (PL_MAX_ROWS + 1) * 4), "wf_paged_plan")) return WF_ERR_CUDA;
        return cuda_check(cudaFuncSetAttribute(paged_release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * (PL_MAX_ROWS + 1) * 4), "wf_paged_release");
    });
}
// A thread per request, as long as a block of so few threads an SM has all items.  512 threads: 256 requests and 24576 tokens 4.5 us, 256 threads 3.9, 1024 7.2; 2048
// requests and 524288 tokens 7.7, 256 threads 9.4, 1024 8.4, 512 twice on every SM 11.3; 512 requests' release 3.5, 256 threads 3.9, 1024 4.3.
int pl_threads(const PlanParams& p, long long items) {
    int t = 128;
    while (t < PL_THREADS && (p.rows > t || items > (long long)t * sm_count())) t *= 2;
    return t;
}
int pl_grid(const PlanParams& p, long long items) {
    const long long t = pl_threads(p, items), n = (items + t - 1) / t;
    return n < 1 ? 1 : n > sm_count() ? sm_count() : (int)n;
}

}  // namespace

}  // namespace wf

using namespace wf;

extern "C" int wf_paged_plan(const int32_t* seq_lens, const int32_t* new_lens, int rows, int32_t* block_table, int max_blocks, const int32_t* free_pages, int pool_pages,
                             const int32_t* free_count, int page_size, int max_tokens, int32_t* positions, int32_t* token_rows, int32_t* pages, int32_t* slots, int32_t* offsets,
                             int32_t* lens_out, int32_t* free_count_out, int32_t* status, void* stream) {
    PlanParams p = {};
    p.seq = seq_lens; p.fresh = new_lens; p.table = block_table; p.free_pages = (int32_t*)free_pages; p.free_count = free_count;
    p.rows = rows; p.max_blocks = max_blocks; p.pool_pages = pool_pages; p.page = page_size; p.cap = max_tokens;
    p.positions = positions; p.token_rows = token_rows; p.pages = pages; p.slots = slots; p.offsets = offsets; p.lens_out = lens_out; p.count_out = free_count_out; p.status = status;
    if (int rc = pl_check("wf_paged_plan", p)) return rc;
    if (!free_count || !offsets || !free_count_out || !status || (rows > 0 && (!seq_lens || !new_lens || !lens_out)) || (rows > 0 && max_blocks > 0 && !block_table) ||
        (pool_pages > 0 && !free_pages) || (max_tokens > 0 && (!positions || !token_rows || !pages || !slots))) { set_error("wf_paged_plan: null pointer"); return WF_ERR_INVALID; }
    if (((uintptr_t)positions | (uintptr_t)token_rows | (uintptr_t)pages | (uintptr_t)slots) & 15) { set_error("wf_paged_plan: the token maps must be 16-byte aligned"); return WF_ERR_INVALID; }
    if (int rc = pl_attrs()) return rc;
    const long long items = ((long long)max_tokens + 3) / 4;
    return launch_check(launch_pdl(paged_plan_kernel, pl_grid(p, items), pl_threads(p, items), 4 * (rows + 1) * 4, (cudaStream_t)stream, p), "wf_paged_plan");
}

extern "C" int wf_paged_release(const uint8_t* done, const int32_t* seq_lens, int rows, const int32_t* block_table, int max_blocks, int32_t* free_pages, int pool_pages,
                                const int32_t* free_count, int page_size, int32_t* lens_out, int32_t* free_count_out, void* stream) {
    PlanParams p = {};
    p.seq = seq_lens; p.done = done; p.table = (int32_t*)block_table; p.free_pages = free_pages; p.free_count = free_count;
    p.rows = rows; p.max_blocks = max_blocks; p.pool_pages = pool_pages; p.page = page_size;
    p.lens_out = lens_out; p.count_out = free_count_out;
    if (int rc = pl_check("wf_paged_release", p)) return rc;
    if (!free_count || !free_count_out || (rows > 0 && (!done || !seq_lens || !lens_out)) || (rows > 0 && max_blocks > 0 && !block_table) || (pool_pages > 0 && !free_pages)) {
        set_error("wf_paged_release: null pointer");
        return WF_ERR_INVALID;
    }
    const long long most = (long long)rows * max_blocks;
    const long long items = most < pool_pages ? most : pool_pages;
    if (int rc = pl_attrs()) return rc;
    return launch_check(launch_pdl(paged_release_kernel, pl_grid(p, items), pl_threads(p, items), 2 * (rows + 1) * 4, (cudaStream_t)stream, p), "wf_paged_release");
}
