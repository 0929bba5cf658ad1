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
    int layers, layer, page_size, max_pages;
    int splits, split_keys;        // keys of a split
    float scale_log2e;
    float *part_o, *part_ml;       // [splits][Hkv][AT_D / 4][rows][4], [splits][Hkv][rows][2], rows = B * G up to the next multiple of 32
    int rows_p;                    // those rows
    int box, stages;               // keys per TMA box (a power of two that divides the page); key and value tiles in flight
    int behind_own;                // the kernel before is this call's own part, which has waited for what both read
    int* err;                      // the wait word
};

// ---- the prefix part on the tensor cores
//
// A block owns one key/value head, a range of 64-key tiles and up to 256 query rows (a row = a sequence and one of the query heads that share the key/value
// head).  Two softmax groups of four warps, a thread per row, each have two score buffers of 64 TMEM columns, which their weights (bf16) overwrite in place, and
// 128 columns of output; the scores of a group's next tile are under way while a tile's weights are computed:
//   * more than 128 rows: a group per 128 rows, and every tile serves both;
//   * up to 128 rows: both groups have the same rows and every other tile; their results are joined in shared memory at the end.
// Warp 8 loads keys and values by TMA into rings of 64-key tiles (a box of 64 dims per run of keys inside a page); one thread of warps 9 and 10 each issues a
// group's S = Q K^T (both operands in shared memory) and O += P V (P in TMEM): a wait of one group leaves the other's products running.  The output is rescaled
// only when a row's maximum has grown by more than 2^8 since the scale was last fixed (exact: the sum carries the same scale).
// Weights are rounded to bf16, as the products' operands (off by 2^-8 of a weight at most; sums, maxima and outputs are fp32).
// Every wait is bounded: one that runs out leaves a code in the device's wait word, and the block waits for its copies and products and leaves.
//
// What bounds it: with 256 rows a 64-key tile takes 1720 clocks, of which the tensor core works for 1280 (S reads 4 KB of queries and 2 KB of keys in 48 clocks where
// its products take 32; P V is bound by its products, 2 x 256) and the special function units for 768; the rest are the waits between a group's products and its
// softmax, 150 clocks and more each beside the products' reads.  128 sequences, 32 and 8 heads, 32768 keys (69 GFLOP): 63 us in place, 1.1 PFLOP/s, 65 % of a library
// product's rate.  Two threads a row, tiles of 128 keys (one score buffer a group, whose
// softmax and products wait for one another), one issuing thread for both groups: 4 to 22 % slower.
constexpr int PX_KEYS = 64, PX_ROWS = 128;             // keys of a tile, rows of a group
constexpr int PX_QHALF = PX_ROWS * 128, PX_QTILE = 2 * PX_QHALF;       // bytes of 128 rows x 64 bf16, and of both halves of the dims
constexpr int PX_HALF = PX_KEYS * 128, PX_TILE = 2 * PX_HALF;          // the same of a tile of keys or values
constexpr int PX_SMEM_USE = 160 * 1024;                // queries of one or two groups, then rings of four or three tiles of keys and of values (five of six: as fast)
constexpr int PX_SMEM = PX_SMEM_USE + 1024;
constexpr int PX_STAGES = 4;
// A block of the own part wants 64 KB and 168 registers a thread of the same SM.  Registers are had from quarters of an SM, three warps of this kernel and one of that
// on each: (3 x 112 + 168) x 32 of 16384.  The softmax warps take 16 of what the others leave (at 112 for all they spill, 84 us instead of 73).
constexpr int PX_THREADS = 12 * 32, PX_REGS = 112, PX_REGS_SOFTMAX = 128, PX_REGS_OTHERS = 80;         // (warp 11 only fills its warpgroup)
static_assert(2 * PX_REGS_SOFTMAX + PX_REGS_OTHERS == 3 * PX_REGS, "the softmax warpgroups take what the third one gives");
// int8 pools: a ring of tiles as they lie in the pool, and one of converted tiles with their scales
constexpr int PX_RAW = 3, PX_RAW_TILE = 2 * PX_KEYS * AT_D, PX_SC = 2 * PX_KEYS * 4, PX_STAGES8 = 3;
constexpr int PX_CONV = 4;                             // converting warps (eight: as fast, at 34.4 us for 31 sequences of 64 and 8 heads over 16003 keys)
constexpr int PX_SMEM8_USE = 2 * PX_QTILE + PX_STAGES8 * 2 * PX_TILE + PX_RAW * PX_RAW_TILE + PX_STAGES8 * PX_SC;
constexpr int PX_SMEM8 = PX_SMEM8_USE + 1024;
constexpr int PX_THREADS8 = (11 + PX_CONV) * 32, PX_REGS8 = 128;
static_assert(PX_SMEM <= 226 * 1024 && PX_SMEM8 <= 226 * 1024, "one block's shared memory");
constexpr unsigned long long PX_LIMIT_NS = 1000000000ull;
constexpr float PX_LAZY = 8.f;

__device__ __forceinline__ uint64_t px_desc(uint32_t saddr, uint32_t lbo) {       // 128-byte rows, 128B swizzle, 8-row groups 1024 bytes apart
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D f32, A and B bf16, 128 x n; b_mn: B is MN-major
constexpr uint32_t px_idesc(int n, int b_mn) { return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24); }
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
__device__ __forceinline__ uint64_t px_mul2(uint64_t a, uint64_t b) { uint64_t v; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b)); return v; }
__device__ __forceinline__ uint64_t px_add2(uint64_t a, uint64_t b) { uint64_t v; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b)); return v; }
__device__ __forceinline__ float px_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float px_max(float a, float b) { float y; asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }     // NaN stays NaN
// 2^x of two numbers on the multiply-add units: x = i + f, |f| <= 1/2, by adding 1.5 * 2^23; 2^f by its minimax polynomial of degree 3 (Remez; off by 7.5e-5 at
// most, a 50th of what the rounding of a weight to bf16 may be); i goes into the exponent.  Below 2^-126: 2^-126 or less.  The special function unit gives 16 values a
// clock and SM; one pair in PX_POLY takes this way: 74.4 us for a prefix of 32768 under 128 sequences with one in 8, 71.5 in 4, 71.7 in 3, 72.3 in 2, 79 without.
constexpr int PX_POLY = 4;
__device__ __forceinline__ void px_exp2_poly(uint64_t x, float& e0, float& e1) {
    const uint64_t magic = px_pair(0x4b400000u, 0x4b400000u), minus_magic = px_pair(0xcb400000u, 0xcb400000u), minus1 = px_pair(0xbf800000u, 0xbf800000u);
    constexpr float c0 = 0.9999280571937561f, c1 = 0.6932609677314758f, c2 = 0.2426111251115799f, c3 = 0.0551716685295105f;
    float x0, x1;
    px_unpair(x, x0, x1);
    x = px_pair(__float_as_uint(px_max(x0, -126.f)), __float_as_uint(px_max(x1, -126.f)));
    const uint64_t t = px_add2(x, magic), f = px_fma2(px_add2(t, minus_magic), minus1, x);
    uint64_t y = px_fma2(px_pair(__float_as_uint(c3), __float_as_uint(c3)), f, px_pair(__float_as_uint(c2), __float_as_uint(c2)));
    y = px_fma2(y, f, px_pair(__float_as_uint(c1), __float_as_uint(c1)));
    y = px_fma2(y, f, px_pair(__float_as_uint(c0), __float_as_uint(c0)));
    e0 = __uint_as_float((uint32_t)y + ((uint32_t)t << 23));
    e1 = __uint_as_float((uint32_t)(y >> 32) + ((uint32_t)(t >> 32) << 23));
}
template <int N> __device__ __forceinline__ void px_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void px_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 px_ldcg(const uint4* a) {
    uint4 r;
    asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(a));
    return r;
}

template <bool I8>
__maxnreg__(I8 ? PX_REGS8 : PX_REGS) __global__ void prefix_attn_tc_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ PxParams p) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_full[2], kv_full[PX_STAGES], kv_empty[PX_STAGES], tail_full, raw_full[PX_RAW], raw_empty[PX_RAW], s_full[2][2], p_full[2][2], o_full[2], o_end[2], drained[2];
    __shared__ uint32_t tmem_base_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rows = p.B * p.G, pairs = (rows + 2 * PX_ROWS - 1) / (2 * PX_ROWS);
    const int pr = blockIdx.x % pairs, kvh = blockIdx.x / pairs % p.Hkv, split = blockIdx.x / pairs / p.Hkv;
    const int row0 = pr * 2 * PX_ROWS;
    const bool alt = rows - row0 <= PX_ROWS;              // the groups have the same rows and every other tile
    const int key0 = split * p.split_keys, key1 = min(p.prefix, key0 + p.split_keys);
    const int nt = (key1 - key0 + PX_KEYS - 1) / PX_KEYS;
    const int fix_row = key1 - key0 - (nt - 1) * PX_KEYS;  // rows of the last value tile from here on hold no key: zeroed (a weight of zero times NaN is NaN)
    const int nst = p.stages, hop = alt ? 2 : 1;           // tiles of a ring; from one tile of a group to its next
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_s = base, k_s = I8 ? base + 2 * PX_QTILE : base + PX_SMEM_USE - 2 * nst * PX_TILE, v_s = k_s + nst * PX_TILE;
    const uint32_t raw_s = v_s + nst * PX_TILE, sc_s = raw_s + PX_RAW * PX_RAW_TILE;       // int8: the pool's tiles; 64 scales of keys and 64 of values of every converted tile

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4); mbar_init(&o_full[i], 1); mbar_init(&o_end[i], 1); mbar_init(&drained[i], 1);
            for (int u = 0; u < 2; ++u) { mbar_init(&s_full[i][u], 1); mbar_init(&p_full[i][u], 4); }
        }
        for (int u = 0; u < PX_STAGES; ++u) { mbar_init(&kv_full[u], I8 ? PX_CONV : 1); mbar_init(&kv_empty[u], alt ? 1 : 2); }
        for (int u = 0; u < PX_RAW; ++u) { mbar_init(&raw_full[u], 1); mbar_init(&raw_empty[u], PX_CONV); }
        mbar_init(&tail_full, 1);
        fence_mbar_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 8 * 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap) : "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    if (!p.behind_own) pdl_wait_prior();
    pdl_launch_dependents();

    if (!I8 && warp == 11) {
        if (!I8) px_regs_dec<PX_REGS_OTHERS>();
    } else if (warp == 8) {
        if (!I8) px_regs_dec<PX_REGS_OTHERS>();
        // ------------------------------------------------------------ producer: lanes 0..3 the boxes of keys, 4..7 of values
        const int kv = lane >> 2 & 1, off = (lane & 3) * p.box;
        const int depth = I8 ? PX_RAW : nst, step = I8 ? PX_RAW_TILE : PX_TILE;
        const uint32_t ring = (I8 ? raw_s + kv * PX_KEYS * AT_D : kv ? v_s : k_s) + off * 128;
        uint64_t *const fulls = I8 ? raw_full : kv_full, *const empties = I8 ? raw_empty : kv_empty;
        auto here = [&](int i) { return lane < 8 && off < PX_KEYS && key0 + i * PX_KEYS + off < key1; };       // this lane's box of tile i holds keys
        auto page_of = [&](int i) { return here(i) ? ldcg_i32(p.table + (key0 + i * PX_KEYS + off) / p.page_size) : 0; };
        bool ok = true;
        int st = 0, lap = 0, i = 0;
        int page = page_of(0), page1 = page_of(1), page2 = page_of(2), page3 = page_of(3);      // a tile's entry is asked for four tiles ahead
        for (; i < nt; ++i) {
            const int next = page_of(i + 4);
            const bool mine = here(i), tail = !I8 && i == nt - 1 && fix_row < PX_KEYS;
            const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine));
            uint64_t* full = tail ? &tail_full : &fulls[st];
            if (lap && !px_wait_warp(&empties[st], (uint32_t)((lap & 1) ^ 1))) { ok = false; break; }
            if (lane == 0) mbar_expect_tx(full, boxes * (uint32_t)((I8 ? 1 : 2) * p.box * 128));
            __syncwarp();
            if (mine) {
                const int slot = (key0 + i * PX_KEYS + off) % p.page_size, block = ((page * p.layers + p.layer) * 2 + kv) * p.Hkv + kvh;
#pragma unroll
                for (int h = 0; h < (I8 ? 1 : 2); ++h)
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                 ::"r"(ring + st * step + h * PX_HALF), "l"(&tmap), "r"(h * 64), "r"(slot), "r"(block), "r"(smem_u32(full)) : "memory");
            }
            __syncwarp();
            page = page1; page1 = page2; page2 = page3; page3 = next;
            // the other tiles wait until the queries are there, which would queue behind them (the ring's first filling takes all SMs' bandwidth)
            if (i == 1) { px_wait_warp(&q_full[0], 0); if (!alt) px_wait_warp(&q_full[1], 0); }
            if (tail) {                                    // its keyless value rows are cleared before the tile is handed on
                ok = px_wait_warp(&tail_full, 0);
                for (int c = lane; ok && c < (PX_KEYS - fix_row) * 16; c += 32) {
                    const int h = c / ((PX_KEYS - fix_row) * 8), r = c - h * (PX_KEYS - fix_row) * 8;
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v_s + st * PX_TILE + h * PX_HALF + (fix_row * 8 + r) * 16), "r"(0u) : "memory");
                }
                fence_proxy_async();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(&kv_full[st]);
            }
            if (++st == depth) { st = 0; ++lap; }
        }
        if (!ok) {                                        // the block leaves early, but not before its copies have landed
            if (lane == 0) *(volatile int*)p.err = 16;
            for (int u = max(0, i - depth); u < i; ++u)
                if (I8 || u < nt - 1 || fix_row == PX_KEYS) px_wait_warp(&fulls[u % depth], (uint32_t)((u / depth) & 1));
        }
    } else if (I8 && warp >= 11) {
        // ------------------------------------------------------------ converters: codes to bf16 in the operands' layout, scales beside them
        // A thread takes 16 codes of a row at a time.  A quarter of a warp takes four pieces of rows r and r ^ 5: both the swizzled pieces that it reads and those
        // that it writes lie in different banks.
        const int x = tid - 11 * 32, w = warp - 11;
        const int pc = (lane & 3) + 4 * (lane >> 3 & 1), flip = lane >> 2 & 1 ? 5 : 0;
        const int skv = x >> 6, sj = x & 63;               // this thread's scale: of keys or values, of which key
        auto page_of = [&](int i) { const int j = key0 + i * PX_KEYS + sj; return i < nt && j < key1 ? ldcg_i32(p.table + j / p.page_size) : -1; };
        auto scale_of = [&](int i, int page) {
            float v = 0.f;
            if (page >= 0 && page < p.max_pages)           // what is no page reads as zeros, as the copies do
                asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p.scales + ((((size_t)page * p.layers + p.layer) * 2 + skv) * p.Hkv + kvh) * p.page_size + (key0 + i * PX_KEYS + sj) % p.page_size));
            return v;
        };
        bool ok = true;
        int st = 0, lap = 0, rs = 0, rlap = 0;
        // a scale is asked for one tile ahead, its page two tiles before that
        int page1 = page_of(1), page2 = page_of(2);
        float sc = scale_of(0, page_of(0));
        for (int i = 0; i < nt; ++i) {
            const float sc_next = scale_of(i + 1, page1);
            page1 = page2; page2 = page_of(i + 3);
            if (!px_wait_warp(&raw_full[rs], (uint32_t)(rlap & 1)) || (lap && !px_wait_warp(&kv_empty[st], (uint32_t)((lap & 1) ^ 1)))) { ok = false; break; }
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(sc_s + st * PX_SC + x * 4), "f"(sc) : "memory");
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                uint32_t y[4][4];
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const int row = 2 * ((lane >> 4) | w << 1 | it << 3) ^ flip;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(y[it][0]), "=r"(y[it][1]), "=r"(y[it][2]), "=r"(y[it][3])
                                 : "r"(raw_s + rs * PX_RAW_TILE + kv * PX_KEYS * AT_D + row * 128 + ((pc ^ (row & 7)) << 4)) : "memory");
                }
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const int row = 2 * ((lane >> 4) | w << 1 | it << 3) ^ flip;
                    uint32_t o[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {          // a byte below the exponent of 2^23 is 2^23 + code + 128
                        const uint64_t off2 = px_pair(0xcb000080u, 0xcb000080u);
                        float a, b;
                        px_unpair(px_add2(px_pair(__byte_perm(y[it][k], 0x4b000000u, 0x7440), __byte_perm(y[it][k], 0x4b000000u, 0x7441)), off2), a, b);
                        o[2 * k] = pack_bf16x2(a, b);
                        px_unpair(px_add2(px_pair(__byte_perm(y[it][k], 0x4b000000u, 0x7442), __byte_perm(y[it][k], 0x4b000000u, 0x7443)), off2), a, b);
                        o[2 * k + 1] = pack_bf16x2(a, b);
                    }
                    const uint32_t dst = (kv ? v_s : k_s) + st * PX_TILE + (pc >> 2) * PX_HALF + row * 128;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + ((((pc & 3) * 2 + k) ^ (row & 7)) << 4)), "r"(o[4 * k]), "r"(o[4 * k + 1]), "r"(o[4 * k + 2]),
                                     "r"(o[4 * k + 3]) : "memory");
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&kv_full[st]); mbar_arrive(&raw_empty[rs]); }
            sc = sc_next;
            if (++st == nst) { st = 0; ++lap; }
            if (++rs == PX_RAW) { rs = 0; ++rlap; }
        }
        if (!ok && lane == 0) *(volatile int*)p.err = 19;
    } else if (warp == 9 || warp == 10) {
        if (!I8) px_regs_dec<PX_REGS_OTHERS>();
        // ------------------------------------------------------------ a group's products
        const int t = warp - 9, tiles = alt ? (nt - t + 1) / 2 : nt;
        uint32_t elected;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
        constexpr uint32_t idesc_s = px_idesc(PX_KEYS, 0), idesc_o = px_idesc(AT_D, 1);
        const uint64_t qd = px_desc(q_s + (alt ? 0 : t) * PX_QTILE, 16), kd0 = px_desc(k_s, 16), vd0 = px_desc(v_s, PX_HALF);
        const uint32_t s_t = tmem + t * 256, o_t = s_t + 128;
        int kst = alt ? t : 0, vst = kst;
        uint32_t par = 0;
        bool ok = px_wait_warp(&q_full[alt ? 0 : t], 0);
        for (int n = -1; n < tiles && ok; ++n) {
            if (n + 1 < tiles) {                          // the next tile's scores, into the buffer that the values before last have left
                if (!px_wait_warp(&kv_full[kst], par)) { ok = false; break; }
                tc_fence_after();
                if (elected) {
                    const uint64_t kd = kd0 + (uint64_t)(kst * (PX_TILE >> 4));
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        px_mma_ss(s_t + ((n + 1) & 1) * PX_KEYS, qd + (uint64_t)((ks >> 2) * (PX_QHALF >> 4) + (ks & 3) * 2), kd + (uint64_t)((ks >> 2) * (PX_HALF >> 4) + (ks & 3) * 2), idesc_s,
                                  ks ? 1u : 0u);
                    px_commit(&s_full[t][(n + 1) & 1]);
                }
                __syncwarp();
                if ((kst += hop) >= nst) { kst -= nst; par ^= 1; }
            }
            if (n >= 0) {
                if (!px_wait_warp(&p_full[t][n & 1], (uint32_t)((n >> 1) & 1))) { ok = false; break; }
                tc_fence_after();
                if (elected) {
                    const uint64_t vd = vd0 + (uint64_t)(vst * (PX_TILE >> 4));
#pragma unroll
                    for (int ks = 0; ks < PX_KEYS / 16; ++ks) px_mma_ts(o_t, s_t + (n & 1) * PX_KEYS + ks * 8, vd + (uint64_t)(ks * 128), idesc_o, n || ks ? 1u : 0u);   // 16 keys = 2048 bytes
                    px_commit(n == tiles - 1 ? &o_end[t] : &o_full[t]);
                    px_commit(&kv_empty[vst]);
                }
                __syncwarp();
                if ((vst += hop) >= nst) vst -= nst;
            }
        }
        if (!ok && lane == 0) *(volatile int*)p.err = 17;
        __syncwarp();
        if (elected) px_commit(&drained[t]);              // nor while a product still reads shared memory or TMEM
        px_wait_warp(&drained[t], 0);
    } else {
        if (!I8) px_regs_inc<PX_REGS_SOFTMAX>();
        // ------------------------------------------------------------ softmax: a thread per row
        const int t = warp >> 2, tr = (warp & 3) * 32 + lane, r = row0 + (alt ? 0 : t * PX_ROWS) + tr;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_t = tmem + t * 256 + lane_base, o_t = s_t + 128;
        const bool r_ok = r < rows;
        const int tiles = alt ? (nt - t + 1) / 2 : nt;
        const bool idle = r - lane >= rows;               // none of the warp's rows exists: it only keeps the others company
        const bool flat = p.scale_log2e == 0.f;           // zero queries: every score is 0, but for the masked ones
        const float unit = flat ? 1.f : fabsf(p.scale_log2e);       // a negative scale turns the queries' signs
        if (t == 0 || !alt) {
            // the warp's 32 queries into the swizzled operand tile (zero where there is no row): two whole rows a load, all loads under way together
            const uint32_t sign = p.scale_log2e < 0.f ? 0x80008000u : 0u;
            const int q0 = (warp & 3) * 32 + (lane >> 4), c = lane & 15;
            int x = row0 + (alt ? 0 : t * PX_ROWS) + q0, xb = x / p.G, xg = x - xb * p.G;
            uint4 v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i, x += 2) {
                v[i] = make_uint4(0u, 0u, 0u, 0u);
                if (x < rows && !flat) v[i] = px_ldcg(reinterpret_cast<const uint4*>(p.q + ((size_t)xb * p.H + kvh * p.G + xg) * AT_D) + c);
                for (xg += 2; xg >= p.G; xg -= p.G) ++xb;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(q_s + t * PX_QTILE + (c >> 3) * PX_QHALF + (q0 + 2 * i) * 128 + (((c & 7) ^ ((q0 + 2 * i) & 7)) << 4)),
                             "r"(v[i].x ^ sign), "r"(v[i].y ^ sign), "r"(v[i].z ^ sign), "r"(v[i].w ^ sign) : "memory");
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);
        }
        float m_ref = -INFINITY, l = 0.f;                 // scores in units of log 2
        int sst = alt ? t : 0;                             // int8: the converted tile that holds the scales
        bool ok = true;
        for (int n = 0; n < tiles && ok; ++n) {
            const uint32_t s_n = s_t + (n & 1) * PX_KEYS;
            if (!px_wait_warp(&s_full[t][n & 1], (uint32_t)((n >> 1) & 1))) { ok = false; break; }
            tc_fence_after();
            if (idle) {
                if (lane == 0) mbar_arrive(&p_full[t][n & 1]);
                continue;
            }
            uint32_t s[PX_KEYS];
            TC_LD32(s_n, (s + 0));
            TC_LD32(s_n + 32, (s + 32));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            const uint32_t sc_n = sc_s + (I8 ? sst * PX_SC : 0);
            if (I8) {                                     // the keys' scales; those of keys that are none are 0
#pragma unroll
                for (int c = 0; c < PX_KEYS; c += 4) {
                    uint32_t k[4];
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(k[0]), "=r"(k[1]), "=r"(k[2]), "=r"(k[3]) : "r"(sc_n + c * 4) : "memory");
                    const uint64_t a = px_mul2(px_pair(s[c], s[c + 1]), px_pair(k[0], k[1])), b = px_mul2(px_pair(s[c + 2], s[c + 3]), px_pair(k[2], k[3]));
                    s[c] = (uint32_t)a; s[c + 1] = (uint32_t)(a >> 32); s[c + 2] = (uint32_t)b; s[c + 3] = (uint32_t)(b >> 32);
                }
                if ((sst += hop) >= nst) sst -= nst;
            }
            if (n * hop + (alt ? t : 0) == nt - 1 && fix_row < PX_KEYS) {
#pragma unroll
                for (int c = 0; c < PX_KEYS; ++c) if (c >= fix_row) s[c] = 0xff800000u;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < PX_KEYS; c += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k) mx4[k] = px_max(px_max(mx4[k], __uint_as_float(s[c + k])), __uint_as_float(s[c + 4 + k]));
            const float mx = px_max(px_max(mx4[0], mx4[1]), px_max(mx4[2], mx4[3])) * unit;
            float corr = 1.f;
            if (!(mx <= m_ref + PX_LAZY)) {               // also the first time anything is seen, and NaN
                corr = m_ref == -INFINITY ? 0.f : px_ex2(m_ref - mx);
                m_ref = mx;
                l *= corr;
            }
            // a row with a score of +inf or NaN has no weights but NaN
            const uint32_t nm = __float_as_uint(m_ref == -INFINITY ? 0.f : m_ref == INFINITY ? __uint_as_float(0x7fc00000u) : -m_ref);
            const uint64_t nm2 = px_pair(nm, nm), unit2 = px_pair(__float_as_uint(unit), __float_as_uint(unit));
            uint64_t ls[2] = {0ull, 0ull};
            uint32_t vs[4];
#pragma unroll
            for (int c = 0; c < PX_KEYS / 2; ++c) {       // columns (2c, 2c + 1) go to s[c], an entry whose score has been read
                const uint64_t x = px_fma2(px_pair(s[2 * c], s[2 * c + 1]), unit2, nm2);
                float e0, e1;
                if (c % PX_POLY == PX_POLY - 1) {
                    px_exp2_poly(x, e0, e1);
                } else {
                    px_unpair(x, e0, e1);
                    e0 = px_ex2(e0); e1 = px_ex2(e1);
                }
                ls[c & 1] = px_add2(ls[c & 1], px_pair(__float_as_uint(e0), __float_as_uint(e1)));
                if (I8) {                                 // the values' scales go into the weights
                    if (!(c & 1)) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(vs[0]), "=r"(vs[1]), "=r"(vs[2]), "=r"(vs[3]) : "r"(sc_n + PX_KEYS * 4 + c * 8) : "memory");
                    px_unpair(px_mul2(px_pair(__float_as_uint(e0), __float_as_uint(e1)), px_pair(vs[2 * (c & 1)], vs[2 * (c & 1) + 1])), e0, e1);
                }
                s[c] = pack_bf16x2(e0, e1);
            }
            TC_ST32(s_n, s);
            if (n > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
                if (!px_wait_warp(&o_full[t], (uint32_t)((n - 1) & 1))) { ok = false; break; }      // the scores above came behind all values but the last tile's
                tc_fence_after();
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
            if (lane == 0) mbar_arrive(&p_full[t][n & 1]);
            float l0, l1;
            px_unpair(px_add2(ls[0], ls[1]), l0, l1);
            l += l0 + l1;
        }
        // ---- the group's output.  Groups of the same rows hand each other a half of the columns through the ring, when no product reads it any more, and each
        // finishes the half that it keeps
        const bool joined = alt && nt > 1;
        if (ok && tiles > 0) ok = px_wait_warp(&o_end[t], 0);
        if (joined && ok) ok = px_wait_warp(&o_end[1 - t], 0);
        tc_fence_after();
        const uint32_t ml_s = k_s + 2 * PX_ROWS * 256 + tr * 8;
        const uint32_t mine = k_s + (uint32_t)t * PX_ROWS * 256 + tr * 16, theirs = k_s + (uint32_t)(1 - t) * PX_ROWS * 256 + tr * 16;
        if (joined && ok && !idle) {
            uint32_t o[64];
            TC_LD32(o_t + (1 - t) * 64, (o + 0));
            TC_LD32(o_t + (1 - t) * 64 + 32, (o + 32));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int k = 0; k < 64; k += 4)
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(mine + (k >> 2) * PX_ROWS * 16), "r"(o[k]), "r"(o[k + 1]), "r"(o[k + 2]), "r"(o[k + 3]) : "memory");
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(ml_s + t * PX_ROWS * 8), "f"(m_ref), "f"(l) : "memory");
        }
        if (joined) asm volatile("bar.sync 1, 256;" ::: "memory");
        if (ok && !idle && (t == 0 || joined || !alt)) {
            const size_t part = (size_t)split * p.Hkv + kvh;
            float4* dst = reinterpret_cast<float4*>(p.part_o) + part * 32 * p.rows_p + r;      // rows side by side: a warp's stores are whole lines
            float f0 = 1.f, f1 = 0.f;
            if (joined) {
                float2 ml;
                asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "r"(ml_s + (1 - t) * PX_ROWS * 8) : "memory");
                const float m = fmaxf(m_ref, ml.x);
                f0 = m_ref == -INFINITY ? 0.f : px_ex2(m_ref - m);
                f1 = ml.x == -INFINITY ? 0.f : px_ex2(ml.x - m);
                l = l * f0 + ml.y * f1;
                m_ref = m;
            }
#pragma unroll 1
            for (int c = joined ? t * 64 : 0; c < (joined ? t * 64 + 64 : AT_D); c += 64) {
                uint32_t o[64];
                __syncwarp();
                TC_LD32(o_t + c, (o + 0));
                TC_LD32(o_t + c + 32, (o + 32));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (joined) {
#pragma unroll
                    for (int k = 0; k < 64; k += 4) {
                        float4 w;
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(w.x), "=f"(w.y), "=f"(w.z), "=f"(w.w) : "r"(theirs + (k >> 2) * PX_ROWS * 16) : "memory");
                        o[k] = __float_as_uint(fmaf(__uint_as_float(o[k]), f0, w.x * f1));
                        o[k + 1] = __float_as_uint(fmaf(__uint_as_float(o[k + 1]), f0, w.y * f1));
                        o[k + 2] = __float_as_uint(fmaf(__uint_as_float(o[k + 2]), f0, w.z * f1));
                        o[k + 3] = __float_as_uint(fmaf(__uint_as_float(o[k + 3]), f0, w.w * f1));
                    }
                }
#pragma unroll
                for (int k = 0; k < 64; k += 4)
                    if (r_ok) dst[(size_t)((c + k) >> 2) * p.rows_p] = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
            }
            if (r_ok && (t == 0 || !alt)) reinterpret_cast<float2*>(p.part_ml)[part * p.rows_p + r] = make_float2(m_ref, l);
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
    if (p.behind_own) pdl_wait_prior();                   // whoever waits for this kernel has waited for that one
}

DevMade g_px_attr;

// [128][slot][page, layer, K | V, head], boxes of `box` slots x 128 bytes
int px_encode(CUtensorMap* tm, const wf_kv_layout* kv, int box) {
    EncodeTiledFn fn = tc_encoder();
    if (!fn) { set_error("wf_paged_prefix_attn: cuTensorMapEncodeTiled unavailable"); return WF_ERR_CUDA; }
    const cuuint64_t gdim[3] = {AT_D, (cuuint64_t)kv->page_size, (cuuint64_t)kv->max_pages * kv->layers * 2 * kv->kv_heads};
    const int es_ = kv->dtype == WF_I8 ? 1 : 2;
    const cuuint64_t gstride[2] = {(cuuint64_t)AT_D * es_, (cuuint64_t)kv->page_size * AT_D * es_};
    const cuuint32_t bx[3] = {(cuuint32_t)(128 / es_), (cuuint32_t)box, 1}, es[3] = {1, 1, 1};
    const CUresult cr = fn(tm, es_ == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, kv->pool, gdim, gstride, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) { set_error("wf_paged_prefix_attn: tensor map failed (%d)", (int)cr); return WF_ERR_CUDA; }
    return WF_OK;
}

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
        p.stages = i8 ? PX_STAGES8 : (PX_SMEM_USE - (rows <= PX_ROWS ? 1 : 2) * PX_QTILE) / (2 * PX_TILE);
        p.err = tc_wait_word();
        if (!p.err) { set_error("%s: no wait word", who); return WF_ERR_CUDA; }
        CUtensorMap tm;
        if (int rc = px_encode(&tm, kv, p.box)) return rc;
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
