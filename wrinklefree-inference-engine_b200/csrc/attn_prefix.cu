// Decode attention of a batch whose sequences share a long prefix: the prefix's keys and values are read once for all of them.
//
// Softmax over (prefix, own) keys is the merge of two: each part leaves its running maximum m, sum l of 2^(s - m) and weighted values o, and the row's result is
// sum o_i 2^(m_i - M) / sum l_i 2^(m_i - M).  The own part is paged decode attention (attn.cu) with its chunks left unmerged.  The prefix part is a dense
// product per key/value head, B * H / Hkv rows of queries against the prefix's keys, cut over the keys into splits.  The first part is bound by memory, the
// second by the tensor cores' operand reads and the exponentials between their products: with a bf16 pool the prefix part is launched first and keeps to 161 KB of
// shared memory and 2/3 of the registers, so that blocks of the own part run beside it on the same SMs (128 sequences, 32 and 8 heads, a prefix of 32768 and up to 512
// own tokens: 101 us against 119 one after the other, the own part first; 64 of 20 and 5 heads, 8192 and 300: 24.7 and 29.0; 256 of 32 and 8, 2048 and 128: 43.7 and 50.3;
// 4 of 20 and 5, 2048 and 300: 10.5 and 11.1; 64 of 32 and 8 behind 512: 17.0 and 20.2, behind 65536: 99 and 109).  These are replays over the same inputs, medians of one
// run; another GPU gave 92 for the first, and a call that finds its inputs changed takes 117.
// With an int8 pool the prefix part needs all of an SM's shared memory and registers, and the own part goes first.
//
// Operands have 8 bits: weights go into the value product as bf16, with an int8 pool after the value's scale (the own part and paged_decode_attn have 11 bits of them there).
#include "attn_px.cuh"

namespace wf {

namespace {

struct PxParams {
    static constexpr bool TREE = false;
    const __nv_bfloat16* q;        // [B][H][AT_D]
    const void* pool;
    const float* scales;           // int8 pool
    const int32_t* table;          // pages of the prefix
    int prefix, B, H, Hkv, G;
    int layers, layer, page_size, max_pages;
    int splits, split_keys;        // keys of a split
    float scale_log2e;
    float *part_o, *part_ml;       // [splits][Hkv][AT_D / 4][rows][4], [splits][Hkv][rows][2], rows = B * G up to the next multiple of 32
    int rows_p;                    // those rows
    int box, stages;               // keys per TMA box (a power of two that divides the page); key and value tiles in flight (bf16 pools)
    int behind_own;                // the kernel before is this call's own part, which has waited for what both read
    int* err;                      // the wait word

    struct Walk {};
    __device__ __forceinline__ PxWork first(Walk&) const {
        PxWork w;
        w.rows = B * G;
        const int pairs = (w.rows + 2 * PX_ROWS - 1) / (2 * PX_ROWS), pr = blockIdx.x % pairs, split = blockIdx.x / pairs / Hkv;
        w.kvh = blockIdx.x / pairs % Hkv;
        w.row0 = pr * 2 * PX_ROWS;
        w.key0 = split * split_keys;
        w.key1 = min(prefix, w.key0 + split_keys);
        w.first = 0;
        w.part = split * Hkv + w.kvh;
        w.part_row0 = 0;
        w.ctx = 0;
        w.narrow = 0;
        w.table = table;
        return w;
    }
};

template <bool I8>
__maxnreg__(I8 ? PX_REGS8 : PX_REGS) __global__ void prefix_attn_tc_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ PxParams p) {
    extern __shared__ unsigned char smem_raw[];
    px_block<I8>(tmap, p, smem_raw, [&] { if (!p.behind_own) pdl_wait_prior(); });
    if (p.behind_own) pdl_wait_prior();                   // whoever waits for this kernel has waited for that one
}

DevMade g_px_attr;

struct PxMerge {
    AttnChunks own;                // part_o null: no own keys
    const int32_t* seq_lens;
    const float *part_o, *part_ml; // as in PxParams
    int splits, rows, rows_p, Hkv, G, H;
    void* out;
    int out_dtype;
};

// Bound by a few rounds of latency: of 128 sequences with 9 splits of 2.1 MB 8 us, of which the launch takes 2.  A thread per row and 4 C columns: neighbouring
// threads are neighbouring rows, as the prefix part's results lie.  The results of several parts, with their maxima and sums, are under way at a time; the first own
// chunks' too, before it is known how many of them there are (every slot is memory of the workspace).
constexpr int PX_MERGE = 128;
template <int C>
__global__ void __launch_bounds__(PX_MERGE, 4) prefix_merge_kernel(const __grid_constant__ PxMerge p) {
    constexpr int AT_ONCE = C == 1 ? 8 : C == 2 ? 9 : 4, OWN = C == 1 ? 4 : 2;
    const int kvh = blockIdx.x % p.Hkv, r = blockIdx.x / p.Hkv * PX_MERGE + threadIdx.x, c0 = blockIdx.y * C;
    pdl_wait_prior();
    pdl_launch_dependents();
    if (r >= p.rows) return;
    const int b = r / p.G, row = b * p.H + kvh * p.G + (r - b * p.G);
    const size_t next = (size_t)p.Hkv * p.rows_p;         // from a split to the next
    const float2 *ml = reinterpret_cast<const float2*>(p.part_ml) + (size_t)kvh * p.rows_p + r, *oml = reinterpret_cast<const float2*>(p.own.part_ml) + (size_t)row * p.own.max_chunks;
    const float4* v = reinterpret_cast<const float4*>(p.part_o) + ((size_t)kvh * 32 + c0) * p.rows_p + r;
    const float4* w = reinterpret_cast<const float4*>(p.own.part_o) + (size_t)row * p.own.max_chunks * 32 + c0;
    const float2 none = make_float2(-INFINITY, 0.f);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = -INFINITY, L = 0.f;
    float4 o[C];
#pragma unroll
    for (int k = 0; k < C; ++k) o[k] = zero;
    auto join = [&](auto& x, auto& y) {                   // parts with their maxima and sums x, and values y
        constexpr int N = sizeof(x) / sizeof(x[0]);
        float m = M;
#pragma unroll
        for (int u = 0; u < N; ++u) m = fmaxf(m, x[u].x);
        const float f0 = M == -INFINITY ? 0.f : exp2f(M - m);
        L *= f0;
#pragma unroll
        for (int k = 0; k < C; ++k) { o[k].x *= f0; o[k].y *= f0; o[k].z *= f0; o[k].w *= f0; }
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const float f = x[u].x == -INFINITY ? 0.f : exp2f(x[u].x - m);
            L = fmaf(x[u].y, f, L);
#pragma unroll
            for (int k = 0; k < C; ++k) {
                o[k].x = fmaf(f, y[u][k].x, o[k].x); o[k].y = fmaf(f, y[u][k].y, o[k].y); o[k].z = fmaf(f, y[u][k].z, o[k].z); o[k].w = fmaf(f, y[u][k].w, o[k].w);
            }
        }
        M = m;
    };
    int own = 0;
    const int slots = p.own.part_o ? p.own.max_chunks : 0;
    const int len = slots ? p.seq_lens[b] : 0;
    float2 ox[OWN];
    float4 oy[OWN][C];
#pragma unroll
    for (int u = 0; u < OWN; ++u) {
        ox[u] = u < slots ? oml[u] : none;
#pragma unroll
        for (int k = 0; k < C; ++k) oy[u][k] = u < slots ? w[(size_t)u * 32 + k] : zero;
    }
    for (int i = 0; i < p.splits; i += AT_ONCE) {
        float2 x[AT_ONCE];
        float4 y[AT_ONCE][C];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            x[u] = i + u < p.splits ? ml[(i + u) * next] : none;
#pragma unroll
            for (int k = 0; k < C; ++k) y[u][k] = i + u < p.splits ? v[(i + u) * next * 32 + (size_t)k * p.rows_p] : zero;
        }
        join(x, y);
    }
    if (slots) {
        const int nblocks = (len + AT_BLK - 1) / AT_BLK;
        const int cb = chunk_blocks_of(nblocks, p.own.chunk_blocks, p.own.max_chunks, p.own.min_cb);
        own = min((nblocks + cb - 1) / cb, slots);        // (a length beyond the table's)
    }
#pragma unroll
    for (int u = 0; u < OWN; ++u)
        if (u >= own) {
            ox[u] = none;
#pragma unroll
            for (int k = 0; k < C; ++k) oy[u][k] = zero;
        }
    join(ox, oy);
    for (int i = OWN; i < own; i += OWN) {
#pragma unroll
        for (int u = 0; u < OWN; ++u) {
            ox[u] = i + u < own ? oml[i + u] : none;
#pragma unroll
            for (int k = 0; k < C; ++k) oy[u][k] = i + u < own ? w[(size_t)(i + u) * 32 + k] : zero;
        }
        join(ox, oy);
    }
    const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;      // no key: zeros; NaN stays
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const float4 y = make_float4(o[k].x * inv, o[k].y * inv, o[k].z * inv, o[k].w * inv);
        const size_t at = (size_t)row * 32 + c0 + k;
        if (p.out_dtype == WF_BF16) reinterpret_cast<uint2*>(p.out)[at] = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
        else reinterpret_cast<float4*>(p.out)[at] = y;
    }
}

int px_rows_p(int B, int G) { return (B * G + 31) / 32 * 32; }

struct PxCut { int splits, keys; size_t bytes; };      // splits of the prefix, their keys, and the bytes of the partial results

// In units of a hundredth of what two tiles take a block (1.95 us): a block costs 300 beside its tiles (queries in, results out), and every split what the
// merge reads of it.  Twice or half of the latter moves 64 sequences over 8192 keys by -0.2 and +1.8 us of 22.8, 4 over 2048 not at all.
PxCut px_cut(int B, int H, int Hkv, int prefix) {
    if (prefix <= 0) return PxCut{0, 0, 0};
    const int G = H / Hkv, sms = sm_count(), tiles = (int)(((long long)prefix + 2 * PX_KEYS - 1) / (2 * PX_KEYS));       // pairs of tiles: one for each group
    const long long rows = (long long)B * G, units = Hkv * ((rows + 2 * PX_ROWS - 1) / (2 * PX_ROWS));
    int best = 1;
    long long least = -1;
    // more than two blocks an SM are for those who have them without splits
    for (int n = 1; n <= tiles && (n == 1 || units * n <= 2 * sms); ++n) {
        const long long waves = (units * n + sms - 1) / sms, cost = waves * ((tiles + n - 1) / n + 3) * 100 + n * (5 + rows * Hkv / 60);
        if (least < 0 || cost < least) { least = cost; best = n; }
    }
    PxCut c;
    c.keys = (tiles + best - 1) / best * 2 * PX_KEYS;
    c.splits = (int)(((long long)prefix + c.keys - 1) / c.keys);
    c.bytes = ((size_t)c.splits * Hkv * px_rows_p(B, G) * (AT_D + 2) * sizeof(float) + 255) / 256 * 256;                // the own chunks' vectors follow
    return c;
}

// what the call refuses for its size alone, and has no workspace for (the last one: a grid's third dimension)
const char* px_too_large(int B, int H, int prefix, bool own) {
    return prefix > 1 << 30 ? "a prefix is at most 2^30 tokens" : (long long)B * H > 1 << 24 ? "at most 2^24 rows of queries" : own && B > 65535 ? "at most 65535 sequences with keys of their own" : nullptr;
}

}  // namespace

}  // namespace wf

using namespace wf;

extern "C" size_t wf_prefix_attn_workspace_bytes(int B, int H, int kv_heads, int max_seq, int prefix_len) {
    if (B <= 0 || H <= 0 || kv_heads <= 0 || px_too_large(B, H, prefix_len, max_seq > 0)) return 0;
    return px_cut(B, H, kv_heads, prefix_len).bytes + attn_chunks_bytes(B, H, kv_heads, max_seq);
}

extern "C" int wf_paged_prefix_attn(const void* q, const wf_kv_layout* kv, int layer, const int32_t* prefix_table, int prefix_len, const int32_t* block_table, int max_blocks,
                                    const int32_t* seq_lens, int B, int H, float scale, void* out, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "wf_paged_prefix_attn";
    if (prefix_len < 0 || max_blocks < 0 || B < 0 || H <= 0) { set_error("%s: bad size (B %d, H %d, prefix %d, blocks %d)", who, B, H, prefix_len, max_blocks); return WF_ERR_INVALID; }
    if (const char* why = px_too_large(B, H, prefix_len, max_blocks > 0)) { set_error("%s: %s (%d sequences, %d heads, a prefix of %d)", who, why, B, H, prefix_len); return WF_ERR_UNSUPPORTED; }
    const bool pointers = B == 0 || (q && out && (prefix_len == 0 || prefix_table) && (max_blocks == 0 || (block_table && seq_lens)));
    if (int rc = check_decode_attn(kv, layer, H, out_dtype, pointers, who)) return rc;
    if (B == 0) return WF_OK;
    // (a warp asks for pages a few blocks behind the last one)
    if ((long long)max_blocks * kv->page_size > 0x80000000ll - 4096) { set_error("%s: a row of block_table holds at most 2^31 - 4096 tokens", who); return WF_ERR_UNSUPPORTED; }
    if (int rc = check_wait_word(who)) return rc;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kv->pool) & 15) { set_error("%s: q, out and the pool must be 16-byte aligned", who); return WF_ERR_INVALID; }
    const PxCut cut = px_cut(B, H, kv->kv_heads, prefix_len);
    const size_t mine = cut.bytes, need = mine + attn_chunks_bytes(B, H, kv->kv_heads, max_blocks * kv->page_size);
    if (need && (!workspace || workspace_bytes < need)) { set_error("%s: workspace too small (%zu < %zu)", who, workspace_bytes, need); return WF_ERR_INVALID; }
    if ((uintptr_t)workspace & 15) { set_error("%s: the workspace must be 16-byte aligned", who); return WF_ERR_INVALID; }
    cudaStream_t s = (cudaStream_t)stream;
    PxMerge g = {};
    g.seq_lens = seq_lens; g.Hkv = kv->kv_heads; g.G = H / kv->kv_heads; g.H = H; g.rows = B * g.G; g.rows_p = px_rows_p(B, g.G); g.out = out; g.out_dtype = out_dtype;
    auto own_part = [&](bool beside) -> int {
        return attn_decode_chunks(q, kv->pool, kv->layers, layer, kv->kv_heads, kv->page_size, block_table, max_blocks, seq_lens, B, H, scale, (char*)workspace + mine, workspace_bytes - mine,
                                  kv_scales_of(kv), beside, &g.own, s);
    };
    const bool own_first = max_blocks > 0 && kv->dtype == WF_I8;
    if (own_first)
        if (int rc = own_part(false)) return rc;
    if (prefix_len > 0) {
        PxParams p = {};
        p.q = (const __nv_bfloat16*)q; p.pool = kv->pool; p.scales = kv_scales_of(kv); p.table = prefix_table;
        p.prefix = prefix_len; p.B = B; p.H = H; p.Hkv = kv->kv_heads; p.G = H / kv->kv_heads;
        p.layers = kv->layers; p.layer = layer; p.page_size = kv->page_size; p.max_pages = kv->max_pages;
        p.scale_log2e = scale * 1.4426950408889634f;
        p.splits = cut.splits; p.split_keys = cut.keys;
        p.part_o = (float*)workspace;
        p.rows_p = g.rows_p;
        p.behind_own = own_first;
        p.part_ml = p.part_o + (size_t)p.splits * p.Hkv * p.rows_p * AT_D;
        g.part_o = p.part_o; g.part_ml = p.part_ml; g.splits = p.splits;
        const int rows = g.rows, pairs = (rows + 2 * PX_ROWS - 1) / (2 * PX_ROWS);
        const bool i8 = p.scales != nullptr;
        p.box = 16;
        while (p.box < PX_KEYS && kv->page_size % (2 * p.box) == 0) p.box *= 2;
        p.stages = (PX_SMEM_USE - (rows <= PX_ROWS ? 1 : 2) * PX_QTILE) / (2 * PX_TILE);
        p.err = tc_wait_word();
        if (!p.err) { set_error("%s: no wait word", who); return WF_ERR_CUDA; }
        CUtensorMap tm;
        if (int rc = px_encode(&tm, kv, p.box, who)) return rc;
        if (int rc = g_px_attr.once([&]() -> int {
                return cuda_check(cudaFuncSetAttribute(prefix_attn_tc_kernel<false>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared), who) ||
                               cuda_check(cudaFuncSetAttribute(prefix_attn_tc_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM), who) ||
                               cuda_check(cudaFuncSetAttribute(prefix_attn_tc_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM8), who) ? WF_ERR_CUDA : WF_OK;
            })) return rc;
        const dim3 grid((unsigned)(pairs * p.Hkv * p.splits));
        const cudaError_t e = i8 ? launch_pdl(prefix_attn_tc_kernel<true>, grid, PX_THREADS8, PX_SMEM8, s, tm, p) : launch_pdl(prefix_attn_tc_kernel<false>, grid, PX_THREADS, PX_SMEM, s, tm, p);
        if (int rc = launch_check(e, "prefix_attn_tc")) return rc;
    }
    if (max_blocks > 0 && !own_first)
        if (int rc = own_part(prefix_len > 0)) return rc;
    const unsigned blocks = (unsigned)((g.rows + PX_MERGE - 1) / PX_MERGE) * g.Hkv;
    // one wave of four blocks an SM, with as many columns a thread as that takes (128 sequences of 32 and 8 heads, prefix 32768: 97.2 us with 8, 98.9 with 4, 1.7 waves)
    if (blocks * 32 <= 4 * (unsigned)sm_count()) return launch_check(launch_pdl(prefix_merge_kernel<1>, dim3(blocks, 32), PX_MERGE, 0, s, g), "prefix_merge");
    if (blocks * 16 <= 4 * (unsigned)sm_count()) return launch_check(launch_pdl(prefix_merge_kernel<2>, dim3(blocks, 16), PX_MERGE, 0, s, g), "prefix_merge");
    return launch_check(launch_pdl(prefix_merge_kernel<4>, dim3(blocks, 8), PX_MERGE, 0, s, g), "prefix_merge");
}
