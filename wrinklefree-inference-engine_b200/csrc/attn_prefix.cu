// Decode attention of a batch whose sequences share a long prefix: the prefix's keys and values are read once for all of them.
//
// Softmax over (prefix, own) keys is the merge of two: each part leaves its running maximum m, sum l of 2^(s - m) and weighted values o, and the row's result is
// sum o_i 2^(m_i - M) / sum l_i 2^(m_i - M).  The own part is paged decode attention (attn.cu) with its chunks left unmerged.  The prefix part is a dense
// product per key/value head, B * H / Hkv rows of queries against the prefix's keys, cut over the keys into splits.
#include "attn_chunks.cuh"
#include "wf_bitnet.h"

namespace wf {

namespace {

struct PxParams {
    const __nv_bfloat16* q;        // [B][H][AT_D]
    const void* pool;
    const float* scales;           // int8 pool
    const int32_t* table;          // pages of the prefix
    int prefix, B, H, Hkv, G;
    int layers, layer, page_size;
    int splits, split_keys;        // keys of a split
    float scale_log2e;
    float *part_o, *part_ml;       // [splits][B][H][AT_D], [splits][B][H][2]
    int wait_first;                // the kernel before is not this call's own
};

constexpr int PX_SIMPLE_WARPS = 4;
// a warp per row and split: a lane per key for the scores, then a lane per 4 output columns
__global__ void __launch_bounds__(PX_SIMPLE_WARPS * 32) prefix_attn_kernel(const __grid_constant__ PxParams p) {
    const int lane = threadIdx.x & 31, row = blockIdx.x * PX_SIMPLE_WARPS + (threadIdx.x >> 5), split = blockIdx.y;
    pdl_wait_prior();
    pdl_launch_dependents();
    if (row >= p.B * p.H) return;
    const int kvh = row % p.H / p.G, j0 = split * p.split_keys, j1 = min(p.prefix, j0 + p.split_keys);
    const __nv_bfloat16* q = p.q + (size_t)row * AT_D;
    auto place = [&](int j, int kv) -> size_t {
        const int pg = j / p.page_size;
        return ((((size_t)p.table[pg] * p.layers + p.layer) * 2 + kv) * p.Hkv + kvh) * p.page_size + (j - pg * p.page_size);
    };
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int b = j0; b < j1; b += 32) {
        const int j = b + lane;
        float s = -INFINITY;
        if (j < j1) {
            const size_t at = place(j, 0);
            float dot = 0.f;
            for (int c = 0; c < AT_D; ++c) {
                const float k = p.scales ? (float)((int)((const uint8_t*)p.pool)[at * AT_D + c] - 128) : __bfloat162float(((const __nv_bfloat16*)p.pool)[at * AT_D + c]);
                dot = fmaf(__bfloat162float(q[c]), k, dot);
            }
            s = (p.scales ? dot * p.scales[at] : dot) * p.scale_log2e;
        }
        const float mn = fmaxf(m, warp_max(s)), f = m == -INFINITY ? 0.f : exp2f(m - mn), e = s == -INFINITY ? 0.f : exp2f(s - mn);
        m = mn;
        l = l * f + e;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] *= f;
        for (int i = 0; i < min(32, j1 - b); ++i) {
            const size_t at = place(b + i, 1);
            const float w = __shfl_sync(0xffffffffu, e, i) * (p.scales ? p.scales[at] : 1.f);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float v = p.scales ? (float)((int)((const uint8_t*)p.pool)[at * AT_D + 4 * lane + c] - 128) : __bfloat162float(((const __nv_bfloat16*)p.pool)[at * AT_D + 4 * lane + c]);
                o[c] = fmaf(w, v, o[c]);
            }
        }
    }
    l = warp_sum(l);
    const size_t at = (size_t)split * p.B * p.H + row;
    *reinterpret_cast<float4*>(p.part_o + at * AT_D + 4 * lane) = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) { p.part_ml[at * 2] = m; p.part_ml[at * 2 + 1] = l; }
}

struct PxMerge {
    AttnChunks own;                // part_o null: no own keys
    const int32_t* seq_lens;
    const float *part_o, *part_ml;
    int splits, rows, H;
    void* out;
    int out_dtype;
};

// A warp per row (sequence and head), a lane per part for the maxima and factors and per 4 columns for the values.
constexpr int PX_MERGE_WARPS = 4;
__global__ void __launch_bounds__(PX_MERGE_WARPS * 32) prefix_merge_kernel(const __grid_constant__ PxMerge p) {
    const int lane = threadIdx.x & 31, row = blockIdx.x * PX_MERGE_WARPS + (threadIdx.x >> 5);
    pdl_wait_prior();
    pdl_launch_dependents();
    if (row >= p.rows) return;
    int own = 0;
    if (p.own.part_o) {
        const int nblocks = (p.seq_lens[row / p.H] + AT_BLK - 1) / AT_BLK;
        const int cb = chunk_blocks_of(nblocks, p.own.chunk_blocks, p.own.max_chunks, p.own.min_cb);
        own = (nblocks + cb - 1) / cb;
    }
    auto slot = [&](int i) -> size_t { return i < p.splits ? (size_t)i * p.rows + row : (size_t)row * p.own.max_chunks + (i - p.splits); };
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const int n = p.splits + own;
    for (int b = 0; b < n; b += 32) {
        const int i = b + lane;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (i < n) ml = reinterpret_cast<const float2*>(i < p.splits ? p.part_ml : p.own.part_ml)[slot(i)];
        const float mn = fmaxf(M, warp_max(ml.x)), r = M == -INFINITY ? 0.f : exp2f(M - mn), f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mn);
        M = mn;
        L = L * r + warp_sum(ml.y * f);
        o.x *= r; o.y *= r; o.z *= r; o.w *= r;
        for (int k = 0; k < min(32, n - b); ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            const float4 v = reinterpret_cast<const float4*>((b + k < p.splits ? p.part_o : p.own.part_o) + slot(b + k) * AT_D)[lane];
            o.x = fmaf(fk, v.x, o.x); o.y = fmaf(fk, v.y, o.y); o.z = fmaf(fk, v.z, o.z); o.w = fmaf(fk, v.w, o.w);
        }
    }
    const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;      // no key: zeros; NaN stays
    o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
    if (p.out_dtype == WF_BF16) reinterpret_cast<uint2*>(p.out)[(size_t)row * 32 + lane] = make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
    else reinterpret_cast<float4*>(p.out)[(size_t)row * 32 + lane] = o;
}

// splits of the prefix and their keys
void px_cut(int B, int H, int Hkv, int prefix, int* splits, int* keys) {
    const int most = (prefix + 127) / 128;
    const int want = most < 16 ? most : 16;
    *keys = ((most + want - 1) / want) * 128;
    *splits = (prefix + *keys - 1) / *keys;
}

size_t px_bytes(int B, int H, int Hkv, int prefix) {
    if (prefix <= 0) return 0;
    int splits, keys;
    px_cut(B, H, Hkv, prefix, &splits, &keys);
    return ((size_t)splits * B * H * (AT_D + 2) * sizeof(float) + 255) / 256 * 256;      // the own chunks' vectors follow
}

}  // namespace

}  // namespace wf

using namespace wf;

extern "C" size_t wf_prefix_attn_workspace_bytes(int B, int H, int kv_heads, int head_dim, int max_seq, int prefix_len) {
    if (B <= 0 || H <= 0 || kv_heads <= 0) return 0;
    return px_bytes(B, H, kv_heads, prefix_len) + (max_seq > 0 ? wf_attn_workspace_bytes(B, H, head_dim, max_seq) : 0);
}

extern "C" int wf_paged_prefix_attn(const void* q, const wf_kv_layout* kv, int layer, const int32_t* prefix_table, int prefix_len, const int32_t* block_table, int max_blocks,
                                    const int32_t* seq_lens, int B, int H, float scale, void* out, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "wf_paged_prefix_attn";
    if (prefix_len < 0 || max_blocks < 0 || B < 0) { set_error("%s: negative size", who); return WF_ERR_INVALID; }
    const bool pointers = B == 0 || (q && out && (prefix_len == 0 || prefix_table) && (max_blocks == 0 || (block_table && seq_lens)));
    if (int rc = check_decode_attn(kv, layer, H, out_dtype, pointers, who)) return rc;
    if (B == 0) return WF_OK;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kv->pool) & 15) { set_error("%s: q, out and the pool must be 16-byte aligned", who); return WF_ERR_INVALID; }
    const size_t mine = px_bytes(B, H, kv->kv_heads, prefix_len), need = wf_prefix_attn_workspace_bytes(B, H, kv->kv_heads, AT_D, max_blocks * kv->page_size, prefix_len);
    if (need && (!workspace || workspace_bytes < need)) { set_error("%s: workspace too small (%zu < %zu)", who, workspace_bytes, need); return WF_ERR_INVALID; }
    if ((uintptr_t)workspace & 15) { set_error("%s: the workspace must be 16-byte aligned", who); return WF_ERR_INVALID; }
    cudaStream_t s = (cudaStream_t)stream;
    PxMerge g = {};
    g.seq_lens = seq_lens; g.rows = B * H; g.H = H; g.out = out; g.out_dtype = out_dtype;
    if (max_blocks > 0)
        if (int rc = attn_decode_chunks(q, kv->pool, kv->layers, layer, kv->kv_heads, kv->page_size, block_table, max_blocks, seq_lens, B, H, scale, (char*)workspace + mine, workspace_bytes - mine,
                                        kv_scales_of(kv), &g.own, s)) return rc;
    if (prefix_len > 0) {
        PxParams p;
        p.q = (const __nv_bfloat16*)q; p.pool = kv->pool; p.scales = kv_scales_of(kv); p.table = prefix_table;
        p.prefix = prefix_len; p.B = B; p.H = H; p.Hkv = kv->kv_heads; p.G = H / kv->kv_heads;
        p.layers = kv->layers; p.layer = layer; p.page_size = kv->page_size;
        p.scale_log2e = scale * 1.4426950408889634f;
        px_cut(B, H, kv->kv_heads, prefix_len, &p.splits, &p.split_keys);
        p.part_o = (float*)workspace;
        p.part_ml = p.part_o + (size_t)p.splits * B * H * AT_D;
        p.wait_first = max_blocks == 0;
        g.part_o = p.part_o; g.part_ml = p.part_ml; g.splits = p.splits;
        if (int rc = launch_check(launch_pdl(prefix_attn_kernel, dim3((B * H + PX_SIMPLE_WARPS - 1) / PX_SIMPLE_WARPS, p.splits), PX_SIMPLE_WARPS * 32, 0, s, p), "prefix_attn")) return rc;
    }
    return launch_check(launch_pdl(prefix_merge_kernel, dim3((g.rows + PX_MERGE_WARPS - 1) / PX_MERGE_WARPS), PX_MERGE_WARPS * 32, 0, s, g), "prefix_merge");
}
