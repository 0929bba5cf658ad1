// Attention of drafted tokens over the paged cache: every sequence brings up to 256 new tokens that are in the cache already, and each of them sees the tokens in front
// of the drafts and those drafts that its mask names.
//
// A sequence's n drafts of G query heads are n G rows per key/value head, which share every key: a dense product (attn_px.cuh), of which only the tiles that reach the
// drafts look at masks.  Rows stand in tiles of 256; a tile's keys are cut into splits where there are SMs for them, and the splits' results joined as the chunks of
// decode attention are (running maximum m, sum l of 2^(s - m), weighted values o; the result is sum o_i 2^(m_i - M) / sum l_i 2^(m_i - M)).
//
// The host knows neither lengths nor drafts, so every block works out the cut for itself, in a warp, from the sequences' lengths: the shortest split t for which the
// number of blocks stays within what was launched.  Sequences with one split are written straight to the output, the others in parts of the workspace that the
// second kernel joins.
//
// A row that sees no key gets zeros.  A value that is not finite under a key that a row does not see would make it NaN (0 times it): such rows, found by their result, are
// computed again key by key.
#include <algorithm>

#include "attn_px.cuh"

namespace wf {

namespace {

constexpr int TX_WORDS = 4;                            // words of a mask: 256 drafts
constexpr int TX_ROWS = 2 * PX_ROWS;                   // rows of a block
constexpr int TX_SPAN = 2 * PX_KEYS;                   // keys are cut in steps of two tiles, one for each group of a block
constexpr int TX_COST1 = 5, TX_COST2 = 7;              // of such a step, for one group of rows and for two
constexpr int TX_REGS = 168;                           // 384 threads of an SM's 65536

__device__ __forceinline__ int tx_warp_sum(int v) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)v); }

// what the two kernels read of a sequence
struct TxSeq { int first, n, ctx, keys, rows, tiles; };

struct TxParams {
    static constexpr bool TREE = true;
    const __nv_bfloat16* q;        // [T][H][AT_D]
    const void* pool;
    const float* scales;           // int8 pool
    const int32_t *block_table, *seq_lens, *offsets;
    const u64* mask;               // [T][words]
    int words, max_blocks, B, T, H, Hkv, G;
    int layers, layer, page_size, max_pages;
    float scale_log2e;
    int sms, blocks;               // of the GPU; launched
    int32_t* cut;                  // [B][2]: splits, and the first part, of sequences with more than one
    float *part_o, *part_ml;       // [parts][AT_D / 4][rows_p][4], [parts][rows_p][2]
    int parts, rows_p;
    void* out;
    int out_dtype;
    int box, stages;
    int* err;

    __device__ __forceinline__ TxSeq seq(int b) const {
        TxSeq s;
        s.first = min(max(offsets[b], 0), T);
        s.n = min(max(offsets[b + 1], s.first), T) - s.first;
        const int len = seq_lens[b];
        if (s.n > 64 * words || len < 0) s.n = 0;      // more drafts than the masks have bits for: not taken
        const int room = max_blocks * page_size;       // (below 2^31 - 4096)
        s.ctx = min(max(len, 0), room);
        s.keys = min(room - s.ctx, s.n) + s.ctx;
        s.rows = s.keys > 0 ? s.n * G : 0;
        s.tiles = (s.keys + TX_SPAN - 1) / TX_SPAN;
        return s;
    }
    static __device__ __forceinline__ int tiles_of_rows(int rows) { return (rows + TX_ROWS - 1) / TX_ROWS; }
    static __device__ __forceinline__ int cost(const TxSeq& s) { return s.tiles * (s.rows > PX_ROWS ? TX_COST2 : TX_COST1); }
    // splits of a sequence for splits of cost t, and the steps that each has
    static __device__ __forceinline__ int splits(const TxSeq& s, int t, int& steps) {
        if (!s.rows) return 0;
        const int c = cost(s), n = t >= c ? 1 : min(s.tiles, (c + t - 1) / t);
        steps = (s.tiles + n - 1) / n;
        return (s.tiles + steps - 1) / steps;
    }
    __device__ __forceinline__ int units(const TxSeq& s) const { return tiles_of_rows(s.rows) * Hkv; }

    // In one warp: this block's share
    __device__ __forceinline__ PxWork find() const {
        const int lane = threadIdx.x & 31;
        long long total = 0;
        int all = 0, rows = 0;
        for (int b = lane; b < B; b += 32) {
            const TxSeq s = seq(b);
            total += (long long)cost(s) * units(s);
            all += units(s);
            rows += s.rows;
        }
        all = tx_warp_sum(all);
        rows = tx_warp_sum(rows);
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        PxWork w = {};
        if (all > blocks || rows > T * G) return w;    // (offsets that do not rise)
        const int target = min(blocks, all <= sms ? sms : all + sms);
        int t = max((int)((total + target - 1) / target), 1);
        for (int i = 0;; ++i) {
            int n = 0, steps;
            for (int b = lane; b < B; b += 32) { const TxSeq s = seq(b); n += splits(s, t, steps) * units(s); }
            n = tx_warp_sum(n);
            if (n <= target) break;
            t = i < 4 ? max(t + 1, (int)((long long)t * n / target)) : 0x7fffffff;
        }
        int before = 0, part = 0;
        for (int b0 = 0; b0 < B; b0 += 32) {
            const int b = b0 + lane;
            TxSeq s = {};
            int steps = 1, k = 0, n = 0;
            if (b < B) { s = seq(b); k = splits(s, t, steps); n = k * units(s); }
            const int np = k > 1 ? n : 0;
            int in = n, ip = np;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, in, o), y = __shfl_up_sync(0xffffffffu, ip, o);
                if (lane >= o) { in += x; ip += y; }
            }
            const int at = (int)blockIdx.x - before - (in - n);
            const unsigned mine = __ballot_sync(0xffffffffu, at >= 0 && at < n);
            if (mine) {
                const int who = __ffs(mine) - 1;
                if (lane == who) {
                    const int row_tiles = tiles_of_rows(s.rows), rt = at % row_tiles, kvh = at / row_tiles % Hkv, split = at / row_tiles / Hkv;
                    w.rows = s.rows;
                    w.row0 = rt * TX_ROWS;
                    w.kvh = kvh;
                    w.key0 = split * steps * TX_SPAN;
                    w.key1 = min(s.keys, w.key0 + steps * TX_SPAN);
                    w.first = s.first;
                    w.ctx = s.ctx;
                    w.part = k > 1 ? part + ip - np + at : -1;
                    w.part_row0 = w.row0;
                    w.table = block_table + (size_t)b * max_blocks;
                    if (k > 1 && w.part >= parts) w.rows = 0;
                    if (at == 0) { cut[2 * b] = k; cut[2 * b + 1] = part + ip - np; }
                }
                return w;                              // lane `who` has it
            }
            before += __shfl_sync(0xffffffffu, in, 31);
            part += __shfl_sync(0xffffffffu, ip, 31);
        }
        return w;
    }

    template <typename Wait>
    __device__ __forceinline__ PxWork work(Wait wait) const {
        __shared__ PxWork w_s;
        if (threadIdx.x == 0) w_s.rows = 0;
        __syncthreads();
        wait();
        if (threadIdx.x >> 5 == 8) {
            const PxWork w = find();
            if (w.rows > 0) w_s = w;                   // one lane at most
        }
        __syncthreads();
        return w_s;
    }

    __device__ __forceinline__ void store2(const PxWork& w, int r, int c, float x, float y) const {
        const size_t at = (((size_t)w.first + r / G) * H + w.kvh * G + r % G) * AT_D + c;
        if (out_dtype == WF_BF16) reinterpret_cast<uint32_t*>(out)[at / 2] = pack_bf16x2(x, y);
        else reinterpret_cast<float2*>(out)[at / 2] = make_float2(x, y);
    }
    __device__ __forceinline__ void store64(const PxWork& w, int r, int c, const uint32_t (&o)[64], float inv) const {
        const size_t at = (((size_t)w.first + r / G) * H + w.kvh * G + r % G) * AT_D + c;
        auto v = [&](int i) { return __uint_as_float(o[i]) * inv; };
        if (out_dtype == WF_BF16) {
            uint4* y = reinterpret_cast<uint4*>(out) + at / 8;
#pragma unroll
            for (int i = 0; i < 64; i += 8)
                y[i / 8] = make_uint4(pack_bf16x2(v(i), v(i + 1)), pack_bf16x2(v(i + 2), v(i + 3)), pack_bf16x2(v(i + 4), v(i + 5)), pack_bf16x2(v(i + 6), v(i + 7)));
        } else {
            float4* y = reinterpret_cast<float4*>(out) + at / 4;
#pragma unroll
            for (int i = 0; i < 64; i += 4) y[i / 4] = make_float4(v(i), v(i + 1), v(i + 2), v(i + 3));
        }
    }

    // Row r's weighted values of columns c and c + 1 again, by the whole warp (c is the lane's own), over the keys that it sees alone; m: its maximum
    template <bool I8>
    __device__ __forceinline__ float2 row_again(const PxWork& w, int r, float m, float, int c) const {
        const int lane = threadIdx.x & 31;
        float2 sum = make_float2(0.f, 0.f);
        if (m == -INFINITY) return sum;
        const u64* sees = mask + (size_t)(w.first + r / G) * words;
        const uint2 qw = *(reinterpret_cast<const uint2*>(q + (((size_t)w.first + r / G) * H + w.kvh * G + r % G) * AT_D) + lane);
        const float x[4] = {bf16lo(qw.x), bf16hi(qw.x), bf16lo(qw.y), bf16hi(qw.y)};
        for (int j = w.key0; j < w.key1; ++j) {
            const int d = j - w.ctx;
            if (d >= 0 && !(sees[d >> 6] >> (d & 63) & 1ull)) continue;
            const int page = w.table[j / page_size];
            float k[4] = {0.f, 0.f, 0.f, 0.f}, v0 = 0.f, v1 = 0.f;
            if (page >= 0 && page < max_pages) {       // what is no page reads as zeros
                const size_t kr = ((((size_t)page * layers + layer) * 2) * Hkv + w.kvh) * page_size + j % page_size, vr = kr + (size_t)Hkv * page_size;
                if (I8) {
                    const uchar4 a = *(reinterpret_cast<const uchar4*>(reinterpret_cast<const uint8_t*>(pool) + kr * AT_D) + lane);
                    const uchar2 b = *reinterpret_cast<const uchar2*>(reinterpret_cast<const uint8_t*>(pool) + vr * AT_D + c);
                    const float ks = scales[kr], vs = scales[vr];
                    k[0] = ((int)a.x - 128) * ks; k[1] = ((int)a.y - 128) * ks; k[2] = ((int)a.z - 128) * ks; k[3] = ((int)a.w - 128) * ks;
                    v0 = ((int)b.x - 128) * vs; v1 = ((int)b.y - 128) * vs;
                } else {
                    const uint2 a = *(reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(pool) + kr * AT_D) + lane);
                    const uint32_t b = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const __nv_bfloat16*>(pool) + vr * AT_D + c);
                    k[0] = bf16lo(a.x); k[1] = bf16hi(a.x); k[2] = bf16lo(a.y); k[3] = bf16hi(a.y);
                    v0 = bf16lo(b); v1 = bf16hi(b);
                }
            }
            const float s = warp_sum(x[0] * k[0] + x[1] * k[1] + x[2] * k[2] + x[3] * k[3]);
            const float e = exp2f((scale_log2e == 0.f ? 0.f : s * scale_log2e) - m);
            sum.x = fmaf(e, v0, sum.x);
            sum.y = fmaf(e, v1, sum.y);
        }
        return sum;
    }
};

template <bool I8>
__maxnreg__(I8 ? PX_REGS8 : TX_REGS) __global__ void tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ TxParams p) {
    extern __shared__ unsigned char smem_raw[];
    px_block<I8>(tmap, p, smem_raw, [] { pdl_wait_prior(); });
}

// Joins the splits, and writes zeros where no sequence has a row.  A thread per row and four columns; neighbouring threads are neighbouring rows, as the parts lie.  Which
// sequence a row belongs to is found ahead of the wait: the kernel before has waited for the offsets.
constexpr int TX_MERGE = 128, TX_AHEAD = 4;
__global__ void __launch_bounds__(TX_MERGE) tree_merge_kernel(const __grid_constant__ TxParams p) {
    const int kvh = blockIdx.x % p.Hkv, c4 = blockIdx.y;
    const long long x = (long long)(blockIdx.x / p.Hkv) * TX_MERGE + threadIdx.x;
    const int t = (int)(x / p.G), g = (int)(x - (long long)t * p.G);
    int lo = 0, hi = p.B;
    const bool in = t < p.T;
    TxSeq s = {};
    if (in) {
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (p.offsets[mid] <= t) lo = mid; else hi = mid; }
        s = p.seq(lo);
    }
    const bool live = in && s.rows > 0 && t >= s.first && t < s.first + s.n;
    pdl_wait_prior();
    pdl_launch_dependents();
    if (!in) return;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
        const int r = (t - s.first) * p.G + g, tiles = TxParams::tiles_of_rows(s.rows), stride = tiles * p.Hkv;
        const int n = p.cut[2 * lo], part0 = p.cut[2 * lo + 1] + kvh * tiles + r / TX_ROWS, local = r % TX_ROWS;
        if (n == 1) return;                            // written already
        if (n > 1 && part0 >= 0 && n <= p.parts && part0 + (long long)(n - 1) * stride < p.parts) {
            float M = -INFINITY, L = 0.f;
            for (int i = 0; i < n; i += TX_AHEAD) {
                float2 ml[TX_AHEAD];
                float4 v[TX_AHEAD];
#pragma unroll
                for (int u = 0; u < TX_AHEAD; ++u) {
                    const size_t part = (size_t)(part0 + min(i + u, n - 1) * stride);
                    ml[u] = reinterpret_cast<const float2*>(p.part_ml)[part * p.rows_p + local];
                    v[u] = reinterpret_cast<const float4*>(p.part_o)[(part * 32 + c4) * p.rows_p + local];
                    if (i + u >= n) ml[u] = make_float2(-INFINITY, 0.f);
                }
                float m = M;
#pragma unroll
                for (int u = 0; u < TX_AHEAD; ++u) m = fmaxf(m, ml[u].x);
                const float f0 = M == -INFINITY ? 0.f : exp2f(M - m);
                L *= f0; y.x *= f0; y.y *= f0; y.z *= f0; y.w *= f0;
#pragma unroll
                for (int u = 0; u < TX_AHEAD; ++u) {
                    if (ml[u].x == -INFINITY) continue;
                    const float f = exp2f(ml[u].x - m);
                    L = fmaf(ml[u].y, f, L);
                    y.x = fmaf(f, v[u].x, y.x); y.y = fmaf(f, v[u].y, y.y); y.z = fmaf(f, v[u].z, y.z); y.w = fmaf(f, v[u].w, y.w);
                }
                M = m;
            }
            const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;      // no key: zeros; NaN stays
            y.x *= inv; y.y *= inv; y.z *= inv; y.w *= inv;
        }
    }
    const size_t at = ((size_t)t * p.H + kvh * p.G + g) * 32 + c4;
    if (p.out_dtype == WF_BF16) reinterpret_cast<uint2*>(p.out)[at] = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
    else reinterpret_cast<float4*>(p.out)[at] = y;
}

DevMade g_tx_attr;

struct TxSize { int blocks, parts, rows_p; size_t bytes; };

// Row tiles are at most T G / 256 + B; as many blocks as those and one more an SM (or an SM each), of which at most twice the blocks beyond one a tile have a part
TxSize tx_size(int B, int T, int H, int Hkv, int words) {
    const int G = H / Hkv, sms = sm_count();
    const long long units = Hkv * std::min((long long)B * ((64ll * words * G + TX_ROWS - 1) / TX_ROWS), (long long)T * G / TX_ROWS + B);
    TxSize z;
    z.blocks = (int)(units <= sms ? sms : units + sms);
    z.parts = 2 * sms;
    z.rows_p = std::min(TX_ROWS, (64 * words * G + 31) / 32 * 32);
    z.bytes = ((size_t)B * 8 + 255) / 256 * 256 + (size_t)z.parts * z.rows_p * (AT_D + 2) * sizeof(float);
    return z;
}

// what the call refuses for its size alone, and has no workspace for
const char* tx_too_large(int B, int T, int H, int Hkv, int words) {
    return words > TX_WORDS ? "at most 256 drafts a sequence (4 words of mask)" : (long long)T * H > 1 << 24 ? "at most 2^24 rows of queries" : B > 1 << 16 ? "at most 65536 sequences"
         : ((long long)T * (H / Hkv) / TX_ROWS + B) * Hkv > 1 << 22 ? "too many sequences and heads" : nullptr;
}

}  // namespace

}  // namespace wf

using namespace wf;

extern "C" size_t wf_tree_attn_workspace_bytes(int B, int tokens, int H, int kv_heads, int mask_words) {
    if (B <= 0 || tokens <= 0 || H <= 0 || kv_heads <= 0 || mask_words <= 0 || tx_too_large(B, tokens, H, kv_heads, mask_words)) return 0;
    return tx_size(B, tokens, H, kv_heads, mask_words).bytes;
}

extern "C" int wf_paged_tree_attn(const void* q, const wf_kv_layout* kv, int layer, const int32_t* block_table, int max_blocks, const int32_t* seq_lens, const int32_t* offsets,
                                  const uint64_t* mask, int mask_words, int B, int tokens, int H, float scale, void* out, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "wf_paged_tree_attn";
    if (max_blocks < 0 || B < 0 || tokens < 0 || H <= 0 || mask_words <= 0) { set_error("%s: bad size (B %d, %d tokens, H %d, blocks %d, %d words of mask)", who, B, tokens, H, max_blocks, mask_words); return WF_ERR_INVALID; }
    if (kv && kv->kv_heads > 0)                        // (ahead of the pointers: there is no memory for what is refused)
        if (const char* why = tx_too_large(B, tokens, H, kv->kv_heads, mask_words)) { set_error("%s: %s (%d sequences, %d tokens, %d heads)", who, why, B, tokens, H); return WF_ERR_UNSUPPORTED; }
    const bool pointers = tokens == 0 || (q && out && mask && (B == 0 || (seq_lens && offsets && (max_blocks == 0 || block_table))));
    if (int rc = check_decode_attn(kv, layer, H, out_dtype, pointers, who)) return rc;
    if (tokens == 0) return WF_OK;
    if ((long long)max_blocks * kv->page_size > 0x80000000ll - 4096) { set_error("%s: a row of block_table holds at most 2^31 - 4096 tokens", who); return WF_ERR_UNSUPPORTED; }
    if (int rc = check_wait_word(who)) return rc;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kv->pool) & 15) { set_error("%s: q, out and the pool must be 16-byte aligned", who); return WF_ERR_INVALID; }
    if ((uintptr_t)mask & 7) { set_error("%s: the mask must be 8-byte aligned", who); return WF_ERR_INVALID; }
    cudaStream_t s = (cudaStream_t)stream;
    if (B == 0) return cuda_check(cudaMemsetAsync(out, 0, (size_t)tokens * H * AT_D * (out_dtype == WF_BF16 ? 2 : 4), s), who);
    const TxSize z = tx_size(B, tokens, H, kv->kv_heads, mask_words);
    if (!workspace || workspace_bytes < z.bytes) { set_error("%s: workspace too small (%zu < %zu)", who, workspace_bytes, z.bytes); return WF_ERR_INVALID; }
    if ((uintptr_t)workspace & 15) { set_error("%s: the workspace must be 16-byte aligned", who); return WF_ERR_INVALID; }
    TxParams p = {};
    p.q = (const __nv_bfloat16*)q; p.pool = kv->pool; p.scales = kv_scales_of(kv);
    p.block_table = block_table; p.seq_lens = seq_lens; p.offsets = offsets; p.mask = (const u64*)mask; p.words = mask_words;
    p.max_blocks = max_blocks; p.B = B; p.T = tokens; p.H = H; p.Hkv = kv->kv_heads; p.G = H / kv->kv_heads;
    p.layers = kv->layers; p.layer = layer; p.page_size = kv->page_size; p.max_pages = kv->max_pages;
    p.scale_log2e = scale * 1.4426950408889634f;
    p.sms = sm_count(); p.blocks = z.blocks;
    p.cut = (int32_t*)workspace;
    p.part_o = (float*)((char*)workspace + ((size_t)B * 8 + 255) / 256 * 256);
    p.part_ml = p.part_o + (size_t)z.parts * z.rows_p * AT_D;
    p.parts = z.parts; p.rows_p = z.rows_p;
    p.out = out; p.out_dtype = out_dtype;
    p.box = 16;
    while (p.box < PX_KEYS && kv->page_size % (2 * p.box) == 0) p.box *= 2;
    p.stages = PX_STAGES8;
    p.err = tc_wait_word();
    if (!p.err) { set_error("%s: no wait word", who); return WF_ERR_CUDA; }
    CUtensorMap tm;
    if (int rc = px_encode(&tm, kv, p.box, who)) return rc;
    if (int rc = g_tx_attr.once([&]() -> int {
            return cuda_check(cudaFuncSetAttribute(tree_attn_tc_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM_FULL + 1024), who) ||
                           cuda_check(cudaFuncSetAttribute(tree_attn_tc_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM8_FULL), who) ? WF_ERR_CUDA : WF_OK;
        })) return rc;
    const cudaError_t e = p.scales ? launch_pdl(tree_attn_tc_kernel<true>, dim3((unsigned)z.blocks), PX_THREADS8, PX_SMEM8_FULL, s, tm, p)
                                   : launch_pdl(tree_attn_tc_kernel<false>, dim3((unsigned)z.blocks), PX_THREADS, PX_SMEM_FULL + 1024, s, tm, p);
    if (int rc = launch_check(e, "tree_attn_tc")) return rc;
    const long long rows = (long long)tokens * p.G;
    return launch_check(launch_pdl(tree_merge_kernel, dim3((unsigned)((rows + TX_MERGE - 1) / TX_MERGE) * p.Hkv, 32), TX_MERGE, 0, s, p), "tree_merge");
}
