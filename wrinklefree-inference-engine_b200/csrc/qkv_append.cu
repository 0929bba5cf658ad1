// What lies between the projection of a step's tokens and their attention, in one pass: RMS norm of every query and key head, rotation by the token's position,
// queries out, keys and values into the paged cache at the tokens' pages and slots.
//
// With x a head of D numbers, g its gain and r = sqrt(mean x^2 + eps): y = x g / r, then of the first R dims every pair (a, b) -> (a cos - b sin, a sin + b cos),
// pairs (i, i + R/2) or (2i, 2i + 1), cos and sin from the tables' row of the position.  All of it in float, rounded once to bf16; an int8 pool then has
// round(127 y / max |y|) of those bf16 values, as wf_kv_scatter makes of them.
//
// Bound by memory: (2 H + 4 Hkv) D 2 bytes a token are read and written once.  D / 8 lanes have a head, each the 8 numbers of four pairs, so that the rotation is a
// lane's own business: with pairs (i, i + R/2) lane l < R/8 has 4l.. and R/2 + 4l.. of the head (8 bytes each), the others 8 in a row.  A warp has a token, where there are
// many, and asks for the next heads ahead of working on these: 16384 tokens of 32 + 8 heads 73.5 us (5.5 TB/s; the bytes alone 62), in blocks of 256 threads 79 (the last ones run
// alone), of 64 76; without the loads ahead 88, with twice as many heads a time 87, with half a token 84, with warps that go on from token to token 94.
#include "attn_chunks.cuh"
#include "kv8.cuh"
#include "wf_bitnet.h"

namespace wf {

namespace {

struct AppendParams {
    const __nv_bfloat16* qkv;
    long long ld;                                      // elements from a token to the next
    int T, H, Hkv;
    unsigned char* pool;
    float* scales;                                     // int8 pool
    int layers, layer, page_size, max_pages;
    const int32_t *positions, *pages, *slots;
    const void *cos_tab, *sin_tab;                     // [max_pos][rot / 2]
    int tab_bf16, rot, max_pos;
    const void *q_norm, *k_norm;                       // [D], or null
    int norm_bf16;
    float eps;
    __nv_bfloat16* q_out;
    int chunk, chunks;                                 // heads of a warp's share of a token, and shares of a token
};

constexpr int QA_THREADS = 128;
constexpr int QA_AHEAD = 2;                            // rounds of heads whose loads are under way while as many are worked on

__device__ __forceinline__ void qa_load4(const void* tab, int bf16, size_t at, float (&v)[4]) {
    if (bf16) {
        const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(tab) + at);
        v[0] = bf16lo(w.x); v[1] = bf16hi(w.x); v[2] = bf16lo(w.y); v[3] = bf16hi(w.y);
    } else {
        const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(tab) + at);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    }
}

// two floats at a time
typedef unsigned long long u64;
__device__ __forceinline__ u64 qa_pair(float a, float b) { u64 v; asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); return v; }
__device__ __forceinline__ float qa_lo(u64 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float qa_hi(u64 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ u64 qa_mul(u64 a, u64 b) { u64 v; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b)); return v; }
__device__ __forceinline__ u64 qa_fma(u64 a, u64 b, u64 c) { u64 v; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c)); return v; }

// A warp takes `chunk` heads of one token, 32 / (D / 8) at a time.
template <int D, bool I8, bool PAIRS>
__global__ void __launch_bounds__(QA_THREADS) norm_rope_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;
    const int lane = threadIdx.x & 31, l = lane % LANES, sub = lane / LANES;
    const long long warp = (long long)blockIdx.x * (QA_THREADS / 32) + (threadIdx.x >> 5);
    pdl_wait_prior();
    pdl_launch_dependents();
    if (warp >= (long long)p.T * p.chunks) return;
    const int t = (int)(warp / p.chunks), h0 = (int)(warp - (long long)t * p.chunks) * p.chunk, heads = p.H + 2 * p.Hkv, h1 = min(heads, h0 + p.chunk);
    const int pos = p.positions[t], page = p.pages[t], slot = p.slots[t];
    const bool turned = l < p.rot / 8;
    const int c0 = !PAIRS && turned ? 4 * l : 8 * l, c1 = !PAIRS && turned ? p.rot / 2 + 4 * l : 8 * l + 4;
    const __nv_bfloat16* src = p.qkv + (size_t)t * p.ld;
    uint2 in[QA_AHEAD][2], ahead[QA_AHEAD][2];             // this round's heads, and the next one's
    auto ask = [&](int hb) {
#pragma unroll
        for (int u = 0; u < QA_AHEAD; ++u) {
            const int h = hb + u * AT_ONCE + sub;
            ahead[u][0] = ahead[u][1] = make_uint2(0u, 0u);
            if (h < h1) {
                ahead[u][0] = *reinterpret_cast<const uint2*>(src + (size_t)h * D + c0);
                ahead[u][1] = *reinterpret_cast<const uint2*>(src + (size_t)h * D + c1);
            }
        }
    };
    ask(h0);
    const bool bad = pos < 0 || pos >= p.max_pos;
    const bool held = !bad && page >= 0 && page < p.max_pages && slot >= 0 && slot < p.page_size;
    // what belongs to the lane's pairs, two pairs in a word: (0, 1) and (2, 3); of gains the pairs' first and second numbers'
    u64 cs[2], sn[2], minus_sn[2], ga[2][2], gb[2][2];
    {
        float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
        if (turned && !bad) {
            qa_load4(p.cos_tab, p.tab_bf16, (size_t)pos * (p.rot / 2) + 4 * l, c);
            qa_load4(p.sin_tab, p.tab_bf16, (size_t)pos * (p.rot / 2) + 4 * l, s);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) { cs[k] = qa_pair(c[2 * k], c[2 * k + 1]); sn[k] = qa_pair(s[2 * k], s[2 * k + 1]); minus_sn[k] = qa_pair(-s[2 * k], -s[2 * k + 1]); }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const void* gain = w ? p.k_norm : p.q_norm;
        float a[4] = {1.f, 1.f, 1.f, 1.f}, b[4] = {1.f, 1.f, 1.f, 1.f};
        if (gain) { qa_load4(gain, p.norm_bf16, c0, a); qa_load4(gain, p.norm_bf16, c1, b); }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            ga[w][k] = !PAIRS ? qa_pair(a[2 * k], a[2 * k + 1]) : k ? qa_pair(b[0], b[2]) : qa_pair(a[0], a[2]);
            gb[w][k] = !PAIRS ? qa_pair(b[2 * k], b[2 * k + 1]) : k ? qa_pair(b[1], b[3]) : qa_pair(a[1], a[3]);
        }
    }
    __nv_bfloat16* const q = p.q_out + (size_t)t * p.H * D;
    const size_t row0 = held ? ((size_t)page * p.layers + p.layer) * 2 * p.Hkv * p.page_size + slot : 0;       // the keys' first head's; values' heads follow the keys'
    const bool norms = p.q_norm || p.k_norm;
    for (int hb = h0; hb < h1; hb += AT_ONCE * QA_AHEAD) {
#pragma unroll
        for (int u = 0; u < QA_AHEAD; ++u) { in[u][0] = ahead[u][0]; in[u][1] = ahead[u][1]; }
        ask(hb + AT_ONCE * QA_AHEAD);
#pragma unroll
        for (int u = 0; u < QA_AHEAD; ++u) {
            const int h = hb + u * AT_ONCE + sub, which = h < p.H ? 0 : h < p.H + p.Hkv ? 1 : 2;     // query, key, value
            if (hb + u * AT_ONCE >= h1) break;
            uint2 o0 = in[u][0], o1 = in[u][1];
            u64 a[2], b[2];                                // the lane's pairs
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t one = k ? o0.y : o0.x, two = k ? o1.y : o1.x, even = k ? o1.x : o0.x, odd = k ? o1.y : o0.y;
                a[k] = PAIRS ? qa_pair(bf16lo(even), bf16lo(odd)) : qa_pair(bf16lo(one), bf16hi(one));
                b[k] = PAIRS ? qa_pair(bf16hi(even), bf16hi(odd)) : qa_pair(bf16lo(two), bf16hi(two));
            }
            float inv = 1.f;
            if (norms && hb + u * AT_ONCE < p.H + p.Hkv) { // (not for values alone)
                const u64 sq = qa_fma(b[1], b[1], qa_fma(b[0], b[0], qa_fma(a[1], a[1], qa_mul(a[0], a[0]))));
                float ss = qa_lo(sq) + qa_hi(sq);
#pragma unroll
                for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                inv = rsqrtf(ss * (1.f / D) + p.eps);
            }
            if (which < 2) {
                if (which ? p.k_norm != nullptr : p.q_norm != nullptr) {
                    const u64 inv2 = qa_pair(inv, inv);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        a[k] = qa_mul(qa_mul(a[k], inv2), which ? ga[1][k] : ga[0][k]);
                        b[k] = qa_mul(qa_mul(b[k], inv2), which ? gb[1][k] : gb[0][k]);
                    }
                }
                if (turned) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const u64 x = qa_fma(a[k], cs[k], qa_mul(b[k], minus_sn[k])), y = qa_fma(a[k], sn[k], qa_mul(b[k], cs[k]));
                        a[k] = x; b[k] = y;
                    }
                }
                if (PAIRS) {
                    o0 = make_uint2(pack_bf16x2(qa_lo(a[0]), qa_lo(b[0])), pack_bf16x2(qa_hi(a[0]), qa_hi(b[0])));
                    o1 = make_uint2(pack_bf16x2(qa_lo(a[1]), qa_lo(b[1])), pack_bf16x2(qa_hi(a[1]), qa_hi(b[1])));
                } else {
                    o0 = make_uint2(pack_bf16x2(qa_lo(a[0]), qa_hi(a[0])), pack_bf16x2(qa_lo(a[1]), qa_hi(a[1])));
                    o1 = make_uint2(pack_bf16x2(qa_lo(b[0]), qa_hi(b[0])), pack_bf16x2(qa_lo(b[1]), qa_hi(b[1])));
                }
                if (bad) o0 = o1 = make_uint2(0x7fff7fffu, 0x7fff7fffu);       // NaN: there is no such position
            }
            if (which == 0) {
                if (h < h1) {
                    *reinterpret_cast<uint2*>(q + (size_t)h * D + c0) = o0;
                    *reinterpret_cast<uint2*>(q + (size_t)h * D + c1) = o1;
                }
            }
            if (I8) {
                float am = 0.f;
                const float y[8] = {bf16lo(o0.x), bf16hi(o0.x), bf16lo(o0.y), bf16hi(o0.y), bf16lo(o1.x), bf16hi(o1.x), bf16lo(o1.y), bf16hi(o1.y)};
#pragma unroll
                for (int k = 0; k < 8; ++k) am = fmaxf(am, fabsf(y[k]));
#pragma unroll
                for (int o = LANES / 2; o; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
                if (which > 0 && h < h1 && held) {
                    const float inv = kv8_inv(am);
                    const size_t row = row0 + (size_t)(h - p.H) * p.page_size;
                    uchar4 a, b;
                    a.x = kv8_store(y[0], inv); a.y = kv8_store(y[1], inv); a.z = kv8_store(y[2], inv); a.w = kv8_store(y[3], inv);
                    b.x = kv8_store(y[4], inv); b.y = kv8_store(y[5], inv); b.z = kv8_store(y[6], inv); b.w = kv8_store(y[7], inv);
                    *reinterpret_cast<uchar4*>(p.pool + row * D + c0) = a;
                    *reinterpret_cast<uchar4*>(p.pool + row * D + c1) = b;
                    if (l == 0) p.scales[row] = kv8_scale(am);
                }
            } else if (which > 0 && h < h1 && held) {
                const size_t row = row0 + (size_t)(h - p.H) * p.page_size;
                __nv_bfloat16* kv = reinterpret_cast<__nv_bfloat16*>(p.pool) + row * D;
                *reinterpret_cast<uint2*>(kv + c0) = o0;
                *reinterpret_cast<uint2*>(kv + c1) = o1;
            }
        }
    }
}

template <int D, bool I8>
cudaError_t qa_launch(const AppendParams& p, bool pairs, unsigned blocks, cudaStream_t s) {
    return pairs ? launch_pdl(norm_rope_append_kernel<D, I8, true>, dim3(blocks), QA_THREADS, 0, s, p) : launch_pdl(norm_rope_append_kernel<D, I8, false>, dim3(blocks), QA_THREADS, 0, s, p);
}

}  // namespace

}  // namespace wf

using namespace wf;

extern "C" int wf_norm_rope_kv_append(const void* qkv, long long row_stride, int tokens, int H, const wf_kv_layout* kv, int layer, const int32_t* positions, const int32_t* pages,
                                      const int32_t* slots, const void* cos_tab, const void* sin_tab, int table_dtype, int rot, int max_pos, const void* q_norm, const void* k_norm,
                                      int norm_dtype, float eps, int interleaved, void* q_out, void* stream) {
    const char* who = "wf_norm_rope_kv_append";
    if (tokens < 0 || H <= 0) { set_error("%s: bad size (%d tokens, %d heads)", who, tokens, H); return WF_ERR_INVALID; }
    if (!kv || !kv->pool) { set_error("%s: null kv layout/pool", who); return WF_ERR_INVALID; }
    if (kv->max_pages <= 0 || kv->layers <= 0 || kv->kv_heads <= 0 || kv->page_size <= 0 || kv->head_dim <= 0) { set_error("%s: bad kv layout", who); return WF_ERR_INVALID; }
    if (kv->dtype != WF_BF16 && kv->dtype != WF_I8) { set_error("%s: pool must be bf16 or int8", who); return WF_ERR_UNSUPPORTED; }
    const int D = kv->head_dim;
    if (D != 64 && D != 128 && D != 256) { set_error("%s: head_dim must be 64, 128 or 256 (got %d)", who, D); return WF_ERR_UNSUPPORTED; }
    if (kv->dtype == WF_I8 && D != 128) { set_error("%s: int8 pools need head_dim 128 (got %d)", who, D); return WF_ERR_UNSUPPORTED; }
    if (layer < 0 || layer >= kv->layers) { set_error("%s: layer %d out of range", who, layer); return WF_ERR_INVALID; }
    if (rot < 0 || rot > D || max_pos < 0) { set_error("%s: %d rotated dims of %d, %d positions", who, rot, D, max_pos); return WF_ERR_INVALID; }
    if (rot % 8) { set_error("%s: the rotated dims must be a multiple of 8 (got %d)", who, rot); return WF_ERR_UNSUPPORTED; }
    if (table_dtype != WF_F32 && table_dtype != WF_BF16) { set_error("%s: tables must be f32 or bf16", who); return WF_ERR_INVALID; }
    if ((q_norm || k_norm) && norm_dtype != WF_F32 && norm_dtype != WF_BF16) { set_error("%s: gains must be f32 or bf16", who); return WF_ERR_INVALID; }
    if (!(eps >= 0.f) || !(eps < INFINITY)) { set_error("%s: eps must not be negative (got %g)", who, (double)eps); return WF_ERR_INVALID; }
    const long long heads = (long long)H + 2ll * kv->kv_heads;
    if (heads > 1 << 20 || tokens > 1 << 30) { set_error("%s: at most 2^20 heads and 2^30 tokens", who); return WF_ERR_UNSUPPORTED; }
    if (tokens > 1 && row_stride < heads * D) { set_error("%s: row stride %lld below %lld numbers", who, row_stride, heads * D); return WF_ERR_INVALID; }
    if (tokens == 0) return WF_OK;
    if (!qkv || !positions || !pages || !slots || !q_out || (rot && (!cos_tab || !sin_tab))) { set_error("%s: null pointer", who); return WF_ERR_INVALID; }
    if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)kv->pool | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)cos_tab | (uintptr_t)sin_tab) & 15) {
        set_error("%s: qkv, q_out, the pool, tables and gains must be 16-byte aligned", who);
        return WF_ERR_INVALID;
    }
    if (tokens > 1 && row_stride % 4) { set_error("%s: the row stride must be a multiple of 4 (got %lld)", who, row_stride); return WF_ERR_INVALID; }
    AppendParams p = {};
    p.qkv = (const __nv_bfloat16*)qkv; p.ld = row_stride; p.T = tokens; p.H = H; p.Hkv = kv->kv_heads;
    p.pool = (unsigned char*)kv->pool; p.scales = kv_scales_of(kv); p.layers = kv->layers; p.layer = layer; p.page_size = kv->page_size; p.max_pages = kv->max_pages;
    p.positions = positions; p.pages = pages; p.slots = slots;
    p.cos_tab = cos_tab; p.sin_tab = sin_tab; p.tab_bf16 = table_dtype == WF_BF16; p.rot = rot; p.max_pos = max_pos;
    p.q_norm = q_norm; p.k_norm = k_norm; p.norm_bf16 = norm_dtype == WF_BF16; p.eps = eps; p.q_out = (__nv_bfloat16*)q_out;
    // a warp takes as many heads of a token as leave every SM 32 warps
    const int at_once = 256 / D;
    p.chunk = at_once * QA_AHEAD;
    while (p.chunk < heads && (long long)tokens * ((heads + 2 * p.chunk - 1) / (2 * p.chunk)) >= 32ll * sm_count()) p.chunk *= 2;
    while (p.chunk > at_once && (long long)tokens * ((heads + p.chunk - 1) / p.chunk) < 8ll * sm_count()) p.chunk /= 2;
    p.chunks = (int)((heads + p.chunk - 1) / p.chunk);
    const long long blocks = ((long long)tokens * p.chunks + QA_THREADS / 32 - 1) / (QA_THREADS / 32);
    if (blocks > 0x7fffffffll) { set_error("%s: too many tokens and heads", who); return WF_ERR_UNSUPPORTED; }
    cudaStream_t s = (cudaStream_t)stream;
    const bool i8 = p.scales != nullptr;
    const cudaError_t e = D == 64 ? qa_launch<64, false>(p, interleaved, (unsigned)blocks, s)
                        : D == 128 ? (i8 ? qa_launch<128, true>(p, interleaved, (unsigned)blocks, s) : qa_launch<128, false>(p, interleaved, (unsigned)blocks, s))
                                   : qa_launch<256, false>(p, interleaved, (unsigned)blocks, s);
    return launch_check(e, who);
}
