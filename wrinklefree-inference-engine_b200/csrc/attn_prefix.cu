// Decode attention of a batch whose sequences share a long prefix: the prefix's keys and values are read once for all of them.
//
// Softmax over (prefix, own) keys is the merge of two: each part leaves its running maximum m, sum l of 2^(s - m) and weighted values o, and the row's result is
// sum o_i 2^(m_i - M) / sum l_i 2^(m_i - M).  The own part is paged decode attention (attn.cu) with its chunks left unmerged.  The prefix part is a dense
// product per key/value head, B * H / Hkv rows of queries against the prefix's keys, cut over the keys into splits.
#include "attn_chunks.cuh"
#include "gemm_tc_common.cuh"
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
    int box, stages;               // keys per TMA box (a power of two that divides the page); key and value tiles in flight
    int* err;                      // the wait word
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

// ---- the prefix part on the tensor cores (bf16 pools)
//
// A block owns one key/value head, a range of 128-key tiles and up to 256 query rows (a row = a sequence and one of the query heads that share the key/value
// head).  Two softmax groups of four warps, a thread per row, take turns with the tensor cores, each with 128 TMEM columns of scores, overwritten in place by
// the weights in bf16, and 128 columns of output:
//   * more than 128 rows: a group per tile of 128 rows, and every key tile serves both;
//   * up to 128 rows: both groups have the same rows and every other key tile; their results are joined in shared memory at the end.
// Warp 8 loads keys and values by TMA (128 keys x 64 dims a box row of 128 bytes, a box per run of keys inside a page); one thread of warp 9 issues S = Q K^T
// (both operands in shared memory) and O += P V (P in TMEM).  The output is rescaled only when a row's maximum has grown by more than 2^8 since the scale
// was last fixed (exact: the sum carries the same scale).
// Every wait is bounded: one that runs out leaves a code in the device's wait word, and the block waits for its copies and products and leaves.
constexpr int PX_KEYS = 128, PX_ROWS = 128;
constexpr int PX_HALF = 128 * 128;                     // bytes of 128 rows x 64 bf16
constexpr int PX_TILE = 2 * PX_HALF;
constexpr int PX_RING = 7 * PX_TILE;                   // queries of one or two tiles, then three or two stages of keys and of values
constexpr int PX_SMEM = PX_RING + 1024;
constexpr int PX_THREADS = 10 * 32;
constexpr unsigned long long PX_LIMIT_NS = 1000000000ull;
constexpr float PX_LAZY = 8.f;

__device__ __forceinline__ uint64_t px_desc(uint32_t saddr, uint32_t lbo) {       // 128-byte rows, 128B swizzle, 8-row groups 1024 bytes apart
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D f32, A and B bf16, 128 x 128; b_mn: B is MN-major
constexpr uint32_t px_idesc(int b_mn) { return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | (16u << 17) | (8u << 24); }
__device__ __forceinline__ void px_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void px_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void px_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool px_wait(uint64_t* bar, uint32_t parity) {
    for (int i = 0; i < 64; ++i) if (mbar_try_wait(bar, parity)) return true;
    unsigned long long t0, t1;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    do {
        if (mbar_try_wait(bar, parity)) return true;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t1));
    } while (t1 - t0 < PX_LIMIT_NS);
    return false;
}
__device__ __forceinline__ bool px_wait_warp(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, px_wait(bar, parity)); }   // one answer, and the warp together again
__device__ __forceinline__ uint64_t px_pair(uint32_t a, uint32_t b) { uint64_t v; asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(a), "r"(b)); return v; }
__device__ __forceinline__ void px_unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t px_fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t v; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c)); return v; }
__device__ __forceinline__ uint64_t px_add2(uint64_t a, uint64_t b) { uint64_t v; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b)); return v; }
__device__ __forceinline__ float px_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint4 px_ldcg(const uint4* a) {
    uint4 r;
    asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(a));
    return r;
}

__global__ void __launch_bounds__(PX_THREADS, 1) prefix_attn_tc_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ PxParams p) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_full[2], k_full[3], k_empty[3], v_full[3], v_empty[3], v_fixed, s_full[2], p_full[2], o_full[2], drained;
    __shared__ uint32_t tmem_base_s;
    __shared__ float2 other_ml[PX_ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rows = p.B * p.G, pairs = (rows + 2 * PX_ROWS - 1) / (2 * PX_ROWS);
    const int pr = blockIdx.x % pairs, kvh = blockIdx.x / pairs % p.Hkv, split = blockIdx.x / pairs / p.Hkv;
    const int row0 = pr * 2 * PX_ROWS;
    const bool alt = rows - row0 <= PX_ROWS;              // one tile of rows: the groups take every other key tile
    const int key0 = split * p.split_keys, key1 = min(p.prefix, key0 + p.split_keys);
    const int nt = (key1 - key0 + PX_KEYS - 1) / PX_KEYS;
    const int fix_row = key1 - key0 - (nt - 1) * PX_KEYS;  // rows of the last value tile from here on hold no key: zeroed (a weight of zero times NaN is NaN)
    const int nst = p.stages;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_s = base, k_s = base + (7 - 2 * nst) * PX_TILE, v_s = k_s + nst * PX_TILE;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) { mbar_init(&q_full[i], 4); mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1); }
        for (int i = 0; i < 3; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
        mbar_init(&v_fixed, 1);
        mbar_init(&drained, 1);
        fence_mbar_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    if (p.wait_first) pdl_wait_prior();
    pdl_launch_dependents();

    if (warp == 8) {
        // ------------------------------------------------------------ producer
        bool ok = true;
        int issued[2] = {0, 0};                           // tiles of keys and of values under way or landed
        int st = 0, lap = 0;
        for (int i = 0; i < nt && ok; ++i) {
            const int j = key0 + i * PX_KEYS + lane * p.box;
            const bool mine = lane * p.box < PX_KEYS && j < key1;
            const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine));
            int slot = 0, block = 0;
            if (mine) {
                const int pg = j / p.page_size;
                slot = j - pg * p.page_size;
                block = ((ldcg_i32(p.table + pg) * p.layers + p.layer) * 2) * p.Hkv + kvh;
            }
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                uint64_t* full = kv ? &v_full[st] : &k_full[st];
                if (lap && !px_wait_warp(kv ? &v_empty[st] : &k_empty[st], (uint32_t)((lap & 1) ^ 1))) { ok = false; break; }
                if (lane == 0) mbar_expect_tx(full, boxes * (uint32_t)(2 * p.box * 128));
                __syncwarp();
                if (mine) {
                    const uint32_t dst = (kv ? v_s : k_s) + st * PX_TILE + lane * p.box * 128;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                     ::"r"(dst + h * PX_HALF), "l"(&tmap), "r"(h * 64), "r"(slot), "r"(block + kv * p.Hkv), "r"(smem_u32(full)) : "memory");
                }
                __syncwarp();
                issued[kv] = i + 1;
            }
            if (ok && i == nt - 1 && fix_row < PX_KEYS) {
                if (!px_wait_warp(&v_full[st], (uint32_t)(lap & 1))) { ok = false; break; }
                for (int c = lane; c < (PX_KEYS - fix_row) * 16; c += 32) {
                    const int h = c / ((PX_KEYS - fix_row) * 8), r = c - h * (PX_KEYS - fix_row) * 8;
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v_s + st * PX_TILE + h * PX_HALF + (fix_row * 8 + r) * 16), "r"(0u) : "memory");
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_fixed);
            }
            if (++st == nst) { st = 0; ++lap; }
        }
        if (!ok) {                                        // the block leaves early, but not before its copies have landed
            if (lane == 0) *(volatile int*)p.err = 16;
            for (int kv = 0; kv < 2; ++kv)
                for (int i = max(0, issued[kv] - nst); i < issued[kv]; ++i) px_wait_warp(kv ? &v_full[i % nst] : &k_full[i % nst], (uint32_t)((i / nst) & 1));
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMA issuer
        uint32_t elected;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
        if (elected) {
            const uint32_t idesc_s = px_idesc(0), idesc_o = px_idesc(1);
            uint32_t np[2] = {0, 0};                      // weight tiles consumed per group
            bool ok = true, q_ready[2] = {false, false};
            int kst = 0, klap = 0, vst = 0, vlap = 0;
            auto scores = [&](int t) {                    // of the key tile in stage kst, for group t
                const int qt = alt ? 0 : t;
                if (!q_ready[qt]) { if (!px_wait(&q_full[qt], 0)) return false; q_ready[qt] = true; }
                tc_fence_after();
                const uint64_t qd = px_desc(q_s + qt * PX_TILE, 16), kd = px_desc(k_s + kst * PX_TILE, 16);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint64_t off = (uint64_t)((ks >> 2) * (PX_HALF >> 4) + (ks & 3) * 2);
                    px_mma_ss(tmem + t * 256, qd + off, kd + off, idesc_s, ks ? 1u : 0u);
                }
                px_commit(&s_full[t]);
                return true;
            };
            auto values = [&](int t, bool last) {         // with the value tile in stage vst
                if (!px_wait(&p_full[t], np[t] & 1)) return false;
                tc_fence_after();
                const uint64_t vd = px_desc(v_s + vst * PX_TILE, PX_HALF);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) px_mma_ts(tmem + t * 256 + 128, tmem + t * 256 + ks * 8, vd + (uint64_t)(ks * 128), idesc_o, np[t] || ks ? 1u : 0u);   // 16 keys = 2048 bytes
                ++np[t];
                if (last) px_commit(&o_full[t]);
                return true;
            };
            for (int i = -1; i < nt && ok; ++i) {
                const bool more = i + 1 < nt;
                if (more && !px_wait(&k_full[kst], (uint32_t)(klap & 1))) { ok = false; break; }
                auto next_k = [&]() { px_commit(&k_empty[kst]); if (++kst == nst) { kst = 0; ++klap; } };
                if (alt && more) { ok = scores((i + 1) & 1); if (ok) next_k(); }
                if (i >= 0 && ok) ok = px_wait(&v_full[vst], (uint32_t)(vlap & 1)) && !(i == nt - 1 && fix_row < PX_KEYS && !px_wait(&v_fixed, 0));
                if (alt) {
                    if (i >= 0 && ok) ok = values(i & 1, i >= nt - 2);
                } else {
                    for (int t = 0; t < 2 && ok; ++t) {
                        if (i >= 0) ok = values(t, i == nt - 1);
                        if (more && ok) ok = scores(t);
                    }
                }
                if (!ok) break;
                if (i >= 0) { px_commit(&v_empty[vst]); if (++vst == nst) { vst = 0; ++vlap; } }
                if (more && !alt) next_k();
            }
            if (!ok) *(volatile int*)p.err = 17;
            px_commit(&drained);                          // nor while a product still reads shared memory or TMEM
            px_wait(&drained, 0);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax: a thread per row
        const int t = warp >> 2, tr = (warp & 3) * 32 + lane, r = row0 + (alt ? 0 : t * PX_ROWS) + tr;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_t = tmem + t * 256 + lane_base, o_t = s_t + 128;
        const bool r_ok = r < rows;
        const int b = r_ok ? r / p.G : 0, row = b * p.H + kvh * p.G + (r_ok ? r - b * p.G : 0);
        const int tiles = alt ? (nt - t + 1) / 2 : nt;
        const bool flat = p.scale_log2e == 0.f;           // zero queries: every score is 0, but for the masked ones
        const float unit = flat ? 1.f : fabsf(p.scale_log2e);       // a negative scale turns the queries' signs
        if (t == 0 || !alt) {
            // the row's query into the swizzled operand tile (zero where there is no row)
            const uint32_t qrow = q_s + t * PX_TILE + tr * 128, sign = p.scale_log2e < 0.f ? 0x80008000u : 0u;
            const uint4* src = reinterpret_cast<const uint4*>(p.q + (size_t)row * AT_D);
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (r_ok && !flat) v = px_ldcg(src + c);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(qrow + (c >> 3) * PX_HALF + (((c & 7) ^ (tr & 7)) << 4)), "r"(v.x ^ sign), "r"(v.y ^ sign), "r"(v.z ^ sign),
                             "r"(v.w ^ sign) : "memory");
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);
        }
        float m_ref = -INFINITY, l = 0.f;                 // scores in units of log 2
        bool ok = true;
        for (int it = 0; it < tiles && ok; ++it) {
            if (!px_wait_warp(&s_full[t], it & 1)) { ok = false; break; }     // also: every earlier product of this group is done
            tc_fence_after();
            uint32_t s[128];
            TC_LD32(s_t, (s + 0));
            TC_LD32(s_t + 32, (s + 32));
            TC_LD32(s_t + 64, (s + 64));
            TC_LD32(s_t + 96, (s + 96));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if ((alt ? 2 * it + t : it) == nt - 1 && fix_row < PX_KEYS) {
#pragma unroll
                for (int c = 0; c < 128; ++c) if (c >= fix_row) s[c] = 0xff800000u;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 128; c += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k) mx4[k] = fmaxf(fmaxf(mx4[k], __uint_as_float(s[c + k])), __uint_as_float(s[c + 4 + k]));
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * unit;
            float corr = 1.f;
            if (mx > m_ref + PX_LAZY) {                   // also the first time anything is seen
                corr = m_ref == -INFINITY ? 0.f : px_ex2(m_ref - mx);
                m_ref = mx;
                l *= corr;
            }
            const uint32_t nm = __float_as_uint(m_ref == -INFINITY ? 0.f : -m_ref);
            const uint64_t nm2 = px_pair(nm, nm), unit2 = px_pair(__float_as_uint(unit), __float_as_uint(unit));
            uint64_t ls[2] = {0ull, 0ull};
#pragma unroll
            for (int c = 0; c < 64; ++c) {                // columns (2c, 2c + 1) go to s[c], an entry whose score has been read
                float e0, e1;
                px_unpair(px_fma2(px_pair(s[2 * c], s[2 * c + 1]), unit2, nm2), e0, e1);
                e0 = px_ex2(e0); e1 = px_ex2(e1);
                ls[c & 1] = px_add2(ls[c & 1], px_pair(__float_as_uint(e0), __float_as_uint(e1)));
                s[c] = pack_bf16x2(e0, e1);
            }
            float l0, l1;
            px_unpair(px_add2(ls[0], ls[1]), l0, l1);
            l += l0 + l1;
            TC_ST32(s_t, (s + 0));
            TC_ST32(s_t + 32, (s + 32));
            if (it > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
                for (int c = 0; c < AT_D; c += 32) {
                    uint32_t o[32];
                    TC_LD32(o_t + c, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                    TC_ST32(o_t + c, o);
                }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t]);
        }
        // ---- the group's output: alone, or with that of the other group, whose half lies in the ring by then
        if (ok && tiles > 0) ok = px_wait_warp(&o_full[t], 0);
        bool joined = false;
        if (alt) {
            if (t == 1) {
                if (ok) ok = px_wait_warp(&o_full[0], 0);  // the ring is read by neither group's products any more
                other_ml[tr] = ok && tiles > 0 ? make_float2(m_ref, l) : make_float2(-INFINITY, 0.f);
            }
            if (t == 1 && ok && tiles > 0) {
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < AT_D; c += 32) {
                    uint32_t o[32];
                    __syncwarp();
                    TC_LD32(o_t + c, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(k_s + (((c + k) >> 2) * PX_ROWS + tr) * 16), "r"(o[k]), "r"(o[k + 1]), "r"(o[k + 2]), "r"(o[k + 3]) : "memory");
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            joined = t == 0 && nt > 1;
        }
        if (ok && (t == 0 || !alt)) {
            tc_fence_after();
            float f0 = 1.f, f1 = 0.f;
            if (joined) {
                const float2 ml = other_ml[tr];
                const float m = fmaxf(m_ref, ml.x);
                f0 = m_ref == -INFINITY ? 0.f : px_ex2(m_ref - m);
                f1 = ml.x == -INFINITY ? 0.f : px_ex2(ml.x - m);
                l = l * f0 + ml.y * f1;
                m_ref = m;
            }
            const size_t at = (size_t)split * p.B * p.H + row;
#pragma unroll 1
            for (int c = 0; c < AT_D; c += 32) {
                uint32_t o[32];
                __syncwarp();
                TC_LD32(o_t + c, o);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float4 v = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
                    if (joined) {
                        float4 w;
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(w.x), "=f"(w.y), "=f"(w.z), "=f"(w.w) : "r"(k_s + (((c + k) >> 2) * PX_ROWS + tr) * 16) : "memory");
                        v.x = fmaf(v.x, f0, w.x * f1); v.y = fmaf(v.y, f0, w.y * f1); v.z = fmaf(v.z, f0, w.z * f1); v.w = fmaf(v.w, f0, w.w * f1);
                    }
                    if (r_ok) *reinterpret_cast<float4*>(p.part_o + at * AT_D + c + k) = v;
                }
            }
            if (r_ok) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m_ref, l);
        }
        if (!ok && lane == 0) *(volatile int*)p.err = 18;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
    if (!p.wait_first) pdl_wait_prior();                  // the own part's kernel: whoever waits for this one has waited for that one
}

DevOnce g_px_attr;

// [128][slot][page, layer, K | V, head], boxes of `box` slots x 64
int px_encode(CUtensorMap* tm, const wf_kv_layout* kv, int box) {
    if (!tc_encoder()) gemm_tc_init_attrs();
    EncodeTiledFn fn = tc_encoder();
    if (!fn) { set_error("wf_paged_prefix_attn: cuTensorMapEncodeTiled unavailable"); return WF_ERR_CUDA; }
    const cuuint64_t gdim[3] = {AT_D, (cuuint64_t)kv->page_size, (cuuint64_t)kv->max_pages * kv->layers * 2 * kv->kv_heads};
    const cuuint64_t gstride[2] = {AT_D * 2, (cuuint64_t)kv->page_size * AT_D * 2};
    const cuuint32_t bx[3] = {64, (cuuint32_t)box, 1}, es[3] = {1, 1, 1};
    const CUresult cr = fn(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, kv->pool, gdim, gstride, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) { set_error("wf_paged_prefix_attn: tensor map failed (%d)", (int)cr); return WF_ERR_CUDA; }
    return WF_OK;
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
    const int tiles = (prefix + PX_KEYS - 1) / PX_KEYS;
    const long long rows = (long long)B * (H / Hkv), units = Hkv * ((rows + 2 * PX_ROWS - 1) / (2 * PX_ROWS));
    int best = 1;
    long long least = -1;
    for (int n = 1; n <= tiles && n <= 148; ++n) {
        const long long waves = (units * n + sm_count() - 1) / sm_count(), cost = waves * ((tiles + n - 1) / n + 3) * 100 + n * 20;
        if (least < 0 || cost < least) { least = cost; best = n; }
    }
    *keys = (tiles + best - 1) / best * PX_KEYS;
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
    if (int rc = check_wait_word(who)) return rc;
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
        PxParams p = {};
        p.q = (const __nv_bfloat16*)q; p.pool = kv->pool; p.scales = kv_scales_of(kv); p.table = prefix_table;
        p.prefix = prefix_len; p.B = B; p.H = H; p.Hkv = kv->kv_heads; p.G = H / kv->kv_heads;
        p.layers = kv->layers; p.layer = layer; p.page_size = kv->page_size;
        p.scale_log2e = scale * 1.4426950408889634f;
        px_cut(B, H, kv->kv_heads, prefix_len, &p.splits, &p.split_keys);
        p.part_o = (float*)workspace;
        p.part_ml = p.part_o + (size_t)p.splits * B * H * AT_D;
        p.wait_first = max_blocks == 0;
        g.part_o = p.part_o; g.part_ml = p.part_ml; g.splits = p.splits;
        if (!p.scales) {
            const int rows = B * p.G;
            p.box = 16;
            while (p.box < PX_KEYS && kv->page_size % (2 * p.box) == 0) p.box *= 2;
            p.stages = rows <= PX_ROWS ? 3 : 2;
            p.err = tc_wait_word();
            if (!p.err) { set_error("%s: no wait word", who); return WF_ERR_CUDA; }
            CUtensorMap tm;
            if (int rc = px_encode(&tm, kv, p.box)) return rc;
            if (g_px_attr.need() && cuda_check(cudaFuncSetAttribute(prefix_attn_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PX_SMEM), who)) return WF_ERR_CUDA;
            const int pairs = (rows + 2 * PX_ROWS - 1) / (2 * PX_ROWS);
            if (int rc = launch_check(launch_pdl(prefix_attn_tc_kernel, dim3((unsigned)(pairs * p.Hkv * p.splits)), PX_THREADS, PX_SMEM, s, tm, p), "prefix_attn_tc")) return rc;
        } else
            if (int rc = launch_check(launch_pdl(prefix_attn_kernel, dim3((B * H + PX_SIMPLE_WARPS - 1) / PX_SIMPLE_WARPS, p.splits), PX_SIMPLE_WARPS * 32, 0, s, p), "prefix_attn")) return rc;
    }
    return launch_check(launch_pdl(prefix_merge_kernel, dim3((g.rows + PX_MERGE_WARPS - 1) / PX_MERGE_WARPS), PX_MERGE_WARPS * 32, 0, s, g), "prefix_merge");
}
