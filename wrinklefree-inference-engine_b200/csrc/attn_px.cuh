// Dense attention of many query rows over paged keys and values on the tensor cores, one block: what the shared-prefix part (attn_prefix.cu) and the attention of
// drafted tokens (attn_tree.cu) have in common.
//
// A block owns one key/value head, a range of 64-key tiles and up to 256 query rows (a row = a sequence and one of the query heads that share the key/value
// head).  Two softmax groups of four warps, a thread per row, each have two score buffers of 64 TMEM columns, which their weights (bf16) overwrite in place, and
// 128 columns of output; the scores of a group's next tile are under way while a tile's weights are computed:
//   * more than 128 rows: a group per 128 rows, and every tile serves both;
//   * up to 128 rows: both groups have the same rows and every other tile; their results are joined at the end: a thread's lane of tensor memory is
//     that of the other group's thread with the same row too, and each finishes a half of the columns.
// Warps 8 and 11 load keys and values by TMA into rings of 64-key tiles (a box of 64 dims per run of keys inside a page; of int8 pools warp 8 both, into a ring of codes from which two
// sets of four warps convert every other tile: one set took 3300 clocks a tile, two 1700, of which a set's own 2000 of 4000 are the conversion); one thread of warps 9 and 10 each issues a
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
#pragma once
#include "attn_chunks.cuh"
#include "gemm_tc_common.cuh"
#include "wf_bitnet.h"

namespace wf {

namespace {

typedef unsigned long long u64;

// a block's share: query rows [row0, rows) of one key/value head, against keys [key0, key1) of a table's pages
struct PxWork {
    int rows, row0, kvh, key0, key1;
    int first;                     // the token of row 0
    int part, part_row0;           // where its results go, and the row that stands there first (part < 0: straight into the output)
    int ctx;                       // trees: keys in front of the drafts
    int narrow;                    // trees: no share of the call has rows of a second group, whose queries' place is one more tile's
    const int32_t* table;
};

constexpr int PX_KEYS = 64, PX_ROWS = 128;             // keys of a tile, rows of a group
constexpr int PX_QHALF = PX_ROWS * 128, PX_QTILE = 2 * PX_QHALF;       // bytes of 128 rows x 64 bf16, and of both halves of the dims
constexpr int PX_HALF = PX_KEYS * 128, PX_TILE = 2 * PX_HALF;          // the same of a tile of keys or values
constexpr int PX_SMEM_USE = 160 * 1024;                // queries of one or two groups, then rings of four or three tiles of keys and of values (five of six: as fast)
constexpr int PX_SMEM = PX_SMEM_USE + 1024;
constexpr int PX_STAGES = 4;
constexpr int PX_SMEM_FULL = 224 * 1024, PX_STAGES_FULL = 6;           // the same of a block that shares its SM with no other
// A block of the own part wants 64 KB and 168 registers a thread of the same SM.  Registers are had from quarters of an SM, three warps of this kernel and one of that
// on each: (3 x 112 + 168) x 32 of 16384.  The softmax warps take 16 of what the others leave (at 112 for all they spill, 84 us instead of 73).
constexpr int PX_THREADS = 12 * 32, PX_REGS = 112, PX_REGS_SOFTMAX = 128, PX_REGS_OTHERS = 80;         // (with int8 pools warp 11 only fills its warpgroup)
static_assert(2 * PX_REGS_SOFTMAX + PX_REGS_OTHERS == 3 * PX_REGS, "the softmax warpgroups take what the third one gives");
// int8 pools: a ring of tiles as they lie in the pool, and one of converted tiles with their scales
constexpr int PX_RAW = 3, PX_RAW_TILE = 2 * PX_KEYS * AT_D, PX_SC = 2 * PX_KEYS * 4, PX_STAGES8 = 3;
constexpr int PX_CONV = 4;                             // converting warps of a tile; two such sets take the tiles in turn
constexpr int PX_CONV0 = 12;                           // the first of them
constexpr int PX_SMEM8_USE = 2 * PX_QTILE + PX_STAGES8 * 2 * PX_TILE + PX_RAW * PX_RAW_TILE + PX_STAGES8 * PX_SC;
constexpr int PX_SMEM8 = PX_SMEM8_USE + 1024, PX_SMEM8_FULL = PX_SMEM8 + PX_SC;      // (a tile instead of the second group's queries)
constexpr int PX_THREADS8 = (PX_CONV0 + 2 * PX_CONV) * 32, PX_REGS8 = 96, PX_REGS8_SOFTMAX = 128, PX_REGS8_OTHERS = 72;
static_assert(2 * PX_REGS8_SOFTMAX + 3 * PX_REGS8_OTHERS <= 5 * PX_REGS8, "the softmax warpgroups take what the three others give");
static_assert(PX_SMEM <= 226 * 1024 && PX_SMEM8 <= 226 * 1024 && PX_SMEM_FULL + 1024 <= 226 * 1024, "one block's shared memory");
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
// most, a 50th of what the rounding of a weight to bf16 may be); i goes into the exponent.  Below 2^-126: 0.  The special function unit gives 16 values a
// clock and SM; one pair in PX_POLY takes this way: 74.4 us for a prefix of 32768 under 128 sequences with one in 8, 71.5 in 4, 71.7 in 3, 72.3 in 2, 79 without.
// Int8 pools: none, for their conversion wants the issue slots (31 sequences of 25 drafts over 8000: 193 us, with one in 4 204, in 2 218).
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
    // what is left below 2^-126 becomes 0, so that hidden keys and those of -inf scores have no weight at all
    uint64_t z;
    asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(z) : "l"(px_pair(__float_as_uint(e0), __float_as_uint(e1))), "l"(0ull));
    px_unpair(z, e0, e1);
}
template <int N> __device__ __forceinline__ void px_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void px_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 px_ldcg(const uint4* a) {
    uint4 r;
    asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(a));
    return r;
}

// which of the keys [rel, rel + 64) a row sees, rel counted from its first draft: all in front of it, of the drafts those in the row's words; of them the first n
__device__ __forceinline__ u64 px_sight(const u64* words, int count, int rel, int n) {
    auto word = [&](int i) { return words && i < count ? words[i] : 0ull; };
    u64 see;
    if (rel >= 0) {
        see = word(rel >> 6) >> (rel & 63);
        if (rel & 63) see |= word((rel >> 6) + 1) << (64 - (rel & 63));
    } else {
        see = rel <= -64 ? ~0ull : word(0) << -rel | ((1ull << -rel) - 1ull);
    }
    return n < 64 ? see & ((1ull << n) - 1ull) : see;
}

// such a share, and what follows from it
struct PxSeg : PxWork {
    bool alt;                      // the groups have the same rows and every other tile
    int nt, fix_row;               // tiles; rows of the last value tile from here on hold no key: zeroed (a weight of zero times NaN is NaN)
    int nst, hop;                  // tiles of a ring; from one tile of a group to its next
    uint32_t q_s, k_s, v_s, raw_s, sc_s;       // int8: the pool's tiles; 64 scales of keys and 64 of values of every converted tile
};
template <bool I8, typename P>
__device__ __forceinline__ PxSeg px_seg(const PxWork& w, const P& p, uint32_t base) {
    constexpr bool TREE = P::TREE;
    PxSeg g;
    static_cast<PxWork&>(g) = w;
    g.alt = w.rows - w.row0 <= PX_ROWS;
    g.nt = (w.key1 - w.key0 + PX_KEYS - 1) / PX_KEYS;
    g.fix_row = w.key1 - w.key0 - (g.nt - 1) * PX_KEYS;
    const int queries = TREE && w.narrow ? 1 : 2;
    if constexpr (I8 || TREE) g.nst = (I8 ? PX_STAGES8 + 1 : PX_STAGES_FULL) + 1 - queries;
    else g.nst = p.stages;
    g.hop = g.alt ? 2 : 1;
    g.q_s = base;
    g.k_s = I8 || TREE ? base + queries * PX_QTILE : base + PX_SMEM_USE - 2 * g.nst * PX_TILE;
    g.v_s = g.k_s + g.nst * PX_TILE;
    g.raw_s = g.v_s + g.nst * PX_TILE;
    g.sc_s = g.raw_s + PX_RAW * PX_RAW_TILE;
    return g;
}

// a place in a ring and the parity of its lap
struct PxAt {
    int st = 0;
    uint32_t par = 0;
    __device__ __forceinline__ void step(int n, int size) { st += n; while (st >= size) { st -= size; par ^= 1u; } }
    __device__ __forceinline__ void leap(int n, int size) { st += n; const int laps = st / size; st -= laps * size; par ^= (uint32_t)laps & 1u; }
    __device__ __forceinline__ PxAt after(int n, int size) const { PxAt a = *this; a.step(n, size); return a; }
};

// A block's work: one share (the shared prefix), or, for trees, shares one after another.  Between two of those nothing is drained: warp 8 says what comes next as soon as it has
// asked for a share's last keys, and each role takes it up when it is through with its own part, the rings and their phases running on.
template <bool I8, typename P, typename Wait>
__device__ __forceinline__ void px_block(const CUtensorMap& tmap, const P& p, unsigned char* smem_raw, Wait wait) {
    constexpr bool TREE = P::TREE, FULL = TREE;            // FULL: the block has its SM to itself
    constexpr int STAGES = TREE ? PX_STAGES_FULL : PX_STAGES;
    constexpr int TAKERS = I8 ? 2 + 8 + 2 * PX_CONV : 3 + 8;        // warps that are told of a share
    __shared__ __align__(8) uint64_t q_full[3], kv_full[STAGES], kv_empty[STAGES], tail_full[2], raw_full[PX_RAW], raw_empty[PX_RAW], s_full[2][2], p_full[2][2], o_full[2], o_end[2], drained[2],
        joint, w_full[2], w_empty[2];
    __shared__ uint32_t tmem_base_s;
    __shared__ PxWork w_s[2];
    __shared__ typename P::Walk walk_s;
    __shared__ int failed_s;
    __shared__ uint32_t hidden_s[TREE ? 4 : 1][8];         // of the shares of late, a bit for each draft whose values are not all finite
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    if (tid == 0) {
        failed_s = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&kv_full[i], I8 ? PX_CONV : 2); mbar_init(&kv_empty[i], 2); }
        for (int i = 0; i < PX_RAW; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], PX_CONV); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4); mbar_init(&o_full[i], 1); mbar_init(&o_end[i], 1); mbar_init(&drained[i], 1); mbar_init(&w_full[i], 1); mbar_init(&w_empty[i], TAKERS);
            for (int k = 0; k < 2; ++k) { mbar_init(&s_full[i][k], 1); mbar_init(&p_full[i][k], 4); }
        }
        mbar_init(&q_full[2], 4);
        for (int i = 0; i < 2; ++i) mbar_init(&tail_full[i], 1);
        mbar_init(&joint, 8);
        fence_mbar_init();
    }
    if (TREE) wait();
    if (warp == 8) {
        typename P::Walk walk;
        const PxWork w = p.first(walk);
        if (lane == 0) { w_s[0] = w; walk_s = walk; }
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
    if (!TREE) wait();                                     // (a tree's block has waited for its lengths)
    pdl_launch_dependents();
    auto fail = [&](int code) { if (lane == 0) { *(volatile int*)p.err = code; *(volatile int*)&failed_s = 1; } };
    // A role's part of the shares; run(share, its number): whether all went well
    auto shares = [&](auto run) {
        if constexpr (!TREE) {
            run(px_seg<I8>(w_s[0], p, base), 0);
        } else {
            for (int sh = 0;; ++sh) {
                PxWork& said = w_s[sh & 1];
                const uint32_t par = (uint32_t)(sh >> 1 & 1);
                if (sh > 0) {
                    if (warp == 8) {                       // what comes next: said where all have taken up the share before last
                        typename P::Walk walk = walk_s;
                        PxWork w = p.next(walk);           // (the same in all lanes)
                        if (!px_wait_warp(&w_empty[sh & 1], par ^ 1u)) { fail(20); break; }
                        if (*(volatile int*)&failed_s) w.rows = 0;
                        if (lane == 0) { said = w; walk_s = walk; mbar_arrive(&w_full[sh & 1]); }
                        __syncwarp();
                    } else if (!px_wait_warp(&w_full[sh & 1], par)) { fail(21); break; }
                } else if (warp == 8 && lane == 0) mbar_arrive(&w_full[0]);
                const PxWork w = said;
                __syncwarp();
                if (warp != 8 && lane == 0) mbar_arrive(&w_empty[sh & 1]);
                if (w.rows <= 0 || !run(px_seg<I8>(w, p, base), sh)) break;
            }
        }
    };

    if (warp >= 8) { if (I8) px_regs_dec<PX_REGS8_OTHERS>(); else if (!FULL) px_regs_dec<PX_REGS_OTHERS>(); }
    if (warp == 8 || (!I8 && warp == 11)) {
        PxAt at_ring;
        int depth = 1;
        int tails = 0;                                     // tiles of values that were looked at before they were handed on: they take two barriers in turn
        shares([&](const PxSeg& g, int sh) {
        const int kvh = g.kvh, key0 = g.key0, key1 = g.key1, nt = g.nt, fix_row = g.fix_row, nst = g.nst;
        const uint32_t k_s = g.k_s, v_s = g.v_s, raw_s = g.raw_s;
        const int32_t* table = g.table;
        if (TREE && !I8 && warp == 11) {                   // (who was told of this share has told that it is through with the one three before)
            if (lane < 8) hidden_s[sh & 3][lane] = 0u;
            __syncwarp();
        }
        // ------------------------------------------------------------ producers: warp 8 the boxes of keys and warp 11 those of values, lanes 0..3 (int8: warp 8 all, 4..7 the values')
        const int kv = I8 ? lane >> 2 & 1 : warp == 11, off = (lane & 3) * p.box;
        depth = I8 ? PX_RAW : nst;
        const int tile_bytes = I8 ? PX_RAW_TILE : PX_TILE;
        const uint32_t ring = (I8 ? raw_s + kv * PX_KEYS * AT_D : kv ? v_s : k_s) + off * 128;
        uint64_t *const fulls = I8 ? raw_full : kv_full, *const empties = I8 ? raw_empty : kv_empty;
        const bool boxed = lane < (I8 ? 8 : 4) && off < PX_KEYS;
        // this lane's box: its place in a page, and that page's among the range's.  The warp holds 32 entries of the table from `held` on, and the 32 behind them
        const int first_page = key0 / p.page_size, pages = (key1 - 1) / p.page_size - first_page + 1, per_page = p.layers * 2 * p.Hkv, block0 = (p.layer * 2 + kv) * p.Hkv + kvh;
        int slot = key0 - first_page * p.page_size + off, at = 0, held = 0;
        auto entry = [&](int i) { return i < pages ? (int)min((unsigned)ldcg_i32(table + first_page + i), (unsigned)p.max_pages) : 0; };       // what is no page reads as zeros: behind the last
        int entries = entry(lane), behind = entry(32 + lane);
        bool ok = true;
        int waiting = 0, first_st = 0;                     // such tiles whose copies have been asked for, and the place of the first of them
        auto hand_on = [&](int i) {                        // tile i
            const uint32_t v = v_s + first_st * PX_TILE;
            const int st = first_st, rows = i == nt - 1 ? fix_row : PX_KEYS;
            if (++first_st == depth) first_st = 0;
            --waiting;
            if (!px_wait_warp(&tail_full[tails & 1], (uint32_t)(tails >> 1 & 1))) return false;
            ++tails;
            // rows without a key are cleared
            for (int c = lane; c < (PX_KEYS - rows) * 16; c += 32) {
                const int h = c / ((PX_KEYS - rows) * 8), r = c - h * (PX_KEYS - rows) * 8;
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + h * PX_HALF + (rows * 8 + r) * 16), "r"(0u) : "memory");
            }
            if constexpr (TREE) {
                // Values of drafts that are not finite become 0 (a weight of 0 times them is NaN for rows that do not see them), and their drafts are noted: rows that do see
                // them get them at the end
                const int first = key0 + i * PX_KEYS - g.ctx, r0 = max(-first, 0), n16 = (rows - r0) * 8;
                auto place = [&](int c) { const int h = c >= n16; return v + h * PX_HALF + (r0 * 8 + c - h * n16) * 16; };
                for (int c0 = lane; c0 < 2 * n16; c0 += 4 * 32) {
                    uint32_t y[4][4], odd = 0;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        y[u][0] = y[u][1] = y[u][2] = y[u][3] = 0u;
                        if (c0 + u * 32 < 2 * n16)
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(y[u][0]), "=r"(y[u][1]), "=r"(y[u][2]), "=r"(y[u][3]) : "r"(place(c0 + u * 32)) : "memory");
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u)            // an exponent of ones carries into the sign's place
#pragma unroll
                        for (int k = 0; k < 4; ++k) odd |= (y[u][k] & 0x7f807f80u) + 0x00800080u;
                    if (!(odd & 0x80008000u)) continue;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint32_t any = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t top = ((y[u][k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                            any |= top;
                            y[u][k] &= ~((top >> 15) * 0xffffu);
                        }
                        if (any) {
                            const int c = c0 + u * 32, d = first + ((r0 * 8 + c - (c >= n16) * n16) >> 3);
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(place(c)), "r"(y[u][0]), "r"(y[u][1]), "r"(y[u][2]), "r"(y[u][3]) : "memory");
                            if (d < 256) atomicOr(&hidden_s[sh & 3][d >> 5], 1u << (d & 31));
                        }
                    }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&kv_full[st]);
            return true;
        };
        for (int i = 0; i < nt; ++i) {
            const int st = at_ring.st;
            while (slot >= p.page_size) { slot -= p.page_size; ++at; }
            const int lead = __shfl_sync(0xffffffffu, at, 0);              // (box 0 is the first)
            if (lead - held >= 32) { entries = behind; held += 32; behind = entry(held + 32 + lane); }
            const int page0 = __shfl_sync(0xffffffffu, entries, (at - held) & 31), page1 = __shfl_sync(0xffffffffu, behind, (at - held) & 31), page = at - held < 32 ? page0 : page1;
            const int reach = TREE ? key0 + (i + 1) * PX_KEYS - g.ctx : 0;         // trees: the tile's last drafts
            const bool mine = boxed && key0 + i * PX_KEYS + off < key1, tail = !I8 && kv && ((i == nt - 1 && fix_row < PX_KEYS) || reach > 0);
            const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine));
            if (tail && waiting == 2 && !hand_on(i - 2)) { ok = false; break; }
            uint64_t* full = tail ? &tail_full[(tails + waiting) & 1] : &fulls[st];
            if (!px_wait_warp(&empties[st], at_ring.par ^ 1u)) { ok = false; break; }       // (the first lap finds every place empty)
            if (lane == 0) mbar_expect_tx(full, boxes * (uint32_t)((I8 ? 1 : 2) * p.box * 128));
            __syncwarp();
            if (mine) {
                const int block = page * per_page + block0;
#pragma unroll
                for (int h = 0; h < (I8 ? 1 : 2); ++h)
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                 ::"r"(ring + st * tile_bytes + h * PX_HALF), "l"(&tmap), "r"(h * 64), "r"(slot), "r"(block), "r"(smem_u32(full)) : "memory");
            }
            __syncwarp();
            slot += PX_KEYS;
            // the first share's other tiles wait until the queries are there, which would queue behind them (the ring's first filling takes all SMs' bandwidth); not a tree's bf16
            // tiles, whose block has more shares to come (48 sequences of 12 drafts: 134 us, waiting 136; over int8 pools waiting took 31 sequences of 25 from 205 to 200 when it was tried)
            if (i == 1 && sh == 0 && (!TREE || I8)) { px_wait_warp(&q_full[g.alt ? 2 : 0], 0); if (!g.alt) px_wait_warp(&q_full[1], 0); }
            at_ring.step(1, depth);
            if (tail && !waiting++) first_st = st;
        }
        while (waiting) ok = hand_on(nt - waiting) && ok;
        if (!ok) fail(16);
        return ok;
        });
        // a block that leaves early does so only when its copies have landed (places never used: the phase before the first)
        for (int u = 0; u < depth; ++u, at_ring.step(1, depth)) px_wait_warp(&(I8 ? raw_full : kv_full)[at_ring.st], at_ring.par ^ 1u);
    } else if (I8 && warp == 11) {                        // only fills its warpgroup
    } else if (I8 && warp >= PX_CONV0) {
        PxAt raw0, kv0;                                    // where a share begins in either ring
        shares([&](const PxSeg& g, int) {
        const int kvh = g.kvh, key0 = g.key0, key1 = g.key1, nt = g.nt, nst = g.nst;
        const uint32_t k_s = g.k_s, v_s = g.v_s, raw_s = g.raw_s, sc_s = g.sc_s;
        const int32_t* table = g.table;
        // ------------------------------------------------------------ converters: codes to bf16 in the operands' layout, scales beside them; every other tile a set of four warps
        // A thread takes 16 codes of a row at a time.  A quarter of a warp takes four pieces of rows r and r ^ 5: both the swizzled pieces that it reads and those
        // that it writes lie in different banks.
        const int set = (warp - PX_CONV0) / PX_CONV, x = tid - (PX_CONV0 + set * PX_CONV) * 32, w = (warp - PX_CONV0) % PX_CONV;
        const int pc = (lane & 3) + 4 * (lane >> 3 & 1), flip = lane >> 2 & 1 ? 5 : 0;
        const int skv = x >> 6, sj = x & 63;               // this thread's scale: of keys or values, of which key
        // a scale is asked for a tile of this set ahead, its page two; their places are counted on from tile to tile
        const int page_size = p.page_size, per_page = p.layers * 2 * p.Hkv, block0 = (p.layer * 2 + skv) * p.Hkv + kvh;
        int key = key0 + set * PX_KEYS + sj, at = key / page_size, slot = key - at * page_size;
        int page_now = key < key1 ? ldcg_i32(table + at) : -1, slot_now = slot;
        auto next_page = [&]() { key += 2 * PX_KEYS; slot += 2 * PX_KEYS; while (slot >= page_size) { slot -= page_size; ++at; } return key < key1 ? ldcg_i32(table + at) : -1; };
        auto scale_at = [&](int page, int s) {
            float v = 0.f;
            if (page >= 0 && page < p.max_pages)           // what is no page reads as zeros, as the copies do
                asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p.scales + (size_t)(page * per_page + block0) * page_size + s));
            return v;
        };
        float sc = scale_at(page_now, slot_now);
        int page1 = next_page(), slot1 = slot;
        int page2 = next_page(), slot2 = slot;
        bool ok = true;
        PxAt raw = raw0.after(set, PX_RAW), kvt = kv0.after(set, nst);
        for (int i = set; i < nt; i += 2) {
            const float sc_next = scale_at(page1, slot1);
            page1 = page2; slot1 = slot2;
            page2 = next_page(); slot2 = slot;
            const int rs = raw.st, st = kvt.st;
            // The tile before in this place of either ring was the other set's: a phase of its barriers is told from the one two before only once that tile is converted
            if (!px_wait_warp(&raw_empty[rs], raw.par ^ 1u) || !px_wait_warp(&raw_full[rs], raw.par) || !px_wait_warp(&kv_empty[st], kvt.par ^ 1u)) { ok = false; break; }
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
            kvt.step(2, nst);
            raw.step(2, PX_RAW);
        }
        raw0.leap(nt, PX_RAW);
        kv0.leap(nt, nst);
        if (!ok) fail(19);
        return ok;
        });
    } else if (warp == 9 || warp == 10) {
        PxAt kv0;                                          // where a share begins in the ring
        int tile0 = 0;                                     // tiles of the group's in the shares before: its buffers go on in turn
        uint32_t q_alt = 0, q_two = 0;                     // parities of the shares of one group's rows and of two groups' (who waits for a barrier waits for all of its phases)
        uint32_t elected;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
        shares([&](const PxSeg& g, int) {
        const int nt = g.nt, nst = g.nst, hop = g.hop;
        const uint32_t q_s = g.q_s, k_s = g.k_s, v_s = g.v_s;
        const bool alt = g.alt;
        // ------------------------------------------------------------ a group's products
        const int t = warp - 9, tiles = alt ? (nt - t + 1) / 2 : nt;
        constexpr uint32_t idesc_s = px_idesc(PX_KEYS, 0), idesc_o = px_idesc(AT_D, 1);
        const uint64_t qd = px_desc(q_s + (alt ? 0 : t) * PX_QTILE, 16), kd0 = px_desc(k_s, 16), vd0 = px_desc(v_s, PX_HALF);
        const uint32_t s_t = tmem + t * 256, o_t = s_t + 128;
        PxAt kt = kv0, vt = kv0.after(alt ? t : 0, nst);
        // The other group's tiles are looked at and given back too: who waits for some of a barrier's phases alone takes the phase two before for the one it waits for
        int seen = 0;
        auto pass_by = [&](int upto) {
            for (; seen < upto; ++seen, kt.step(1, nst)) {
                if (!px_wait_warp(&kv_full[kt.st], kt.par)) return false;
                if (lane == 0) mbar_arrive(&kv_empty[kt.st]);
                __syncwarp();
            }
            return true;
        };
        bool ok = px_wait_warp(&q_full[alt ? 2 : t], alt ? q_alt : q_two);
        if (alt) q_alt ^= 1u; else q_two ^= 1u;
        for (int n = -1; n < tiles && ok; ++n) {
            const int now = tile0 + n, next = now + 1;
            if (n + 1 < tiles) {                          // the next tile's scores, into the buffer that the values before last have left
                if (!pass_by(alt ? 2 * (n + 1) + t : n + 1) || !px_wait_warp(&kv_full[kt.st], kt.par)) { ok = false; break; }
                tc_fence_after();
                if (elected) {
                    const uint64_t kd = kd0 + (uint64_t)(kt.st * (PX_TILE >> 4));
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        px_mma_ss(s_t + (next & 1) * PX_KEYS, qd + (uint64_t)((ks >> 2) * (PX_QHALF >> 4) + (ks & 3) * 2), kd + (uint64_t)((ks >> 2) * (PX_HALF >> 4) + (ks & 3) * 2), idesc_s,
                                  ks ? 1u : 0u);
                    px_commit(&s_full[t][next & 1]);
                }
                __syncwarp();
                kt.step(1, nst);
                ++seen;
            }
            if (n >= 0) {
                if (!px_wait_warp(&p_full[t][now & 1], (uint32_t)(now >> 1 & 1))) { ok = false; break; }
                tc_fence_after();
                if (elected) {
                    const uint64_t vd = vd0 + (uint64_t)(vt.st * (PX_TILE >> 4));
#pragma unroll
                    for (int ks = 0; ks < PX_KEYS / 16; ++ks) px_mma_ts(o_t, s_t + (now & 1) * PX_KEYS + ks * 8, vd + (uint64_t)(ks * 128), idesc_o, n || ks ? 1u : 0u);   // 16 keys = 2048 bytes
                    px_commit(n == tiles - 1 ? &o_end[t] : &o_full[t]);
                    px_commit(&kv_empty[vt.st]);
                }
                __syncwarp();
                vt.step(hop, nst);
            }
        }
        ok = ok && pass_by(nt);
        if (tiles == 0 && elected) px_commit(&o_end[t]);
        __syncwarp();
        kv0.leap(nt, nst);
        tile0 += tiles;
        if (!ok) fail(17);
        return ok;
        });
        __syncwarp();
        if (elected) px_commit(&drained[warp - 9]);       // nor while a product still reads shared memory or TMEM
        px_wait_warp(&drained[warp - 9], 0);
    } else {
        if (I8) px_regs_inc<PX_REGS8_SOFTMAX>(); else if (!FULL) px_regs_inc<PX_REGS_SOFTMAX>();
        PxAt kv0;                                          // as the products'
        int tile0 = 0;
        uint32_t o_par = 0;                                // the parity of the shares' o_full before
        shares([&](const PxSeg& w, int sh) {
        const int rows = w.rows, kvh = w.kvh, row0 = w.row0, key0 = w.key0, key1 = w.key1, nt = w.nt, fix_row = w.fix_row, nst = w.nst, hop = w.hop;
        const uint32_t q_s = w.q_s, sc_s = w.sc_s;
        const bool alt = w.alt;
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
                if (x < rows && !flat) v[i] = px_ldcg(reinterpret_cast<const uint4*>(p.q + ((size_t)(w.first + xb) * p.H + kvh * p.G + xg) * AT_D) + c);
                for (xg += 2; xg >= p.G; xg -= p.G) ++xb;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(q_s + t * PX_QTILE + (c >> 3) * PX_QHALF + (q0 + 2 * i) * 128 + (((c & 7) ^ ((q0 + 2 * i) & 7)) << 4)),
                             "r"(v[i].x ^ sign), "r"(v[i].y ^ sign), "r"(v[i].z ^ sign), "r"(v[i].w ^ sign) : "memory");
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[alt ? 2 : t]);
        }
        const u64* mask_row = nullptr;                     // the row's drafts
        if constexpr (TREE) mask_row = r_ok ? p.mask + (size_t)(w.first + r / p.G) * p.words : nullptr;
        float m_ref = -INFINITY, l = 0.f;                 // scores in units of log 2
        PxAt sc_at = kv0.after(alt ? t : 0, nst);          // int8: the converted tile that holds the scales
        bool ok = true;
        for (int n = 0; n < tiles && ok; ++n) {
            const int buf = (tile0 + n) & 1;
            const uint32_t s_n = s_t + buf * PX_KEYS;
            if (!px_wait_warp(&s_full[t][buf], (uint32_t)((tile0 + n) >> 1 & 1))) { ok = false; break; }
            tc_fence_after();
            if (idle) {
                if (lane == 0) mbar_arrive(&p_full[t][buf]);
                continue;
            }
            uint32_t s[PX_KEYS];
            TC_LD32(s_n, (s + 0));
            TC_LD32(s_n + 32, (s + 32));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            const uint32_t sc_n = sc_s + (I8 ? sc_at.st * PX_SC : 0);
            if (I8) {                                     // the keys' scales; those of keys that are none are 0
#pragma unroll
                for (int c = 0; c < PX_KEYS; c += 4) {
                    uint32_t k[4];
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(k[0]), "=r"(k[1]), "=r"(k[2]), "=r"(k[3]) : "r"(sc_n + c * 4) : "memory");
                    const uint64_t a = px_mul2(px_pair(s[c], s[c + 1]), px_pair(k[0], k[1])), b = px_mul2(px_pair(s[c + 2], s[c + 3]), px_pair(k[2], k[3]));
                    s[c] = (uint32_t)a; s[c + 1] = (uint32_t)(a >> 32); s[c + 2] = (uint32_t)b; s[c + 3] = (uint32_t)(b >> 32);
                }
                sc_at.step(hop, nst);
            }
            const int tile = n * hop + (alt ? t : 0);
            if constexpr (TREE) {                         // a tile that reaches the drafts: those that the row's mask has, and no key behind the last one
                const int at = key0 + tile * PX_KEYS;
                if (at + PX_KEYS > w.ctx) {
                    const u64 see = px_sight(mask_row, p.words, at - w.ctx, key1 - at);
#pragma unroll
                    for (int c = 0; c < PX_KEYS; ++c) if (!((uint32_t)(see >> (c & 32)) >> (c & 31) & 1u)) s[c] = 0xff800000u;
                }
            } else if (tile == nt - 1 && fix_row < PX_KEYS) {
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
            if (!(mx <= m_ref + PX_LAZY)) {               // also the first time anything is seen, and NaN, which stays: who joins parts takes -inf for one without weights
                const float top = px_max(m_ref, mx);
                corr = m_ref == -INFINITY ? 0.f : px_ex2(m_ref - top);
                m_ref = top;
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
                if (!I8 && c % PX_POLY == PX_POLY - 1) {
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
            if constexpr (TREE && I8) {                    // a hidden key has no weight, whatever its values' scale
                const int at = key0 + tile * PX_KEYS;
                if (at + PX_KEYS > w.ctx) {
                    const u64 see = px_sight(mask_row, p.words, at - w.ctx, key1 - at);
#pragma unroll
                    for (int c = 0; c < PX_KEYS / 2; ++c) {
                        const uint32_t two = (uint32_t)(see >> (2 * c & 32)) >> (2 * c & 31);
                        s[c] &= (two & 1u) * 0xffffu | (two & 2u) * 0x7fff8000u;
                    }
                }
            }
            TC_ST32(s_n, s);
            if (n > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
                if (!px_wait_warp(&o_full[t], o_par ^ (uint32_t)((n - 1) & 1))) { ok = false; break; }      // the scores above came behind all values but the last tile's
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
            if (lane == 0) mbar_arrive(&p_full[t][buf]);
            float l0, l1;
            px_unpair(px_add2(ls[0], ls[1]), l0, l1);
            l += l0 + l1;
        }
        if (tiles > 0) o_par ^= (uint32_t)(tiles - 1) & 1u;
        tile0 += tiles;
        kv0.leap(nt, nst);
        // ---- the group's output.  Groups of the same rows tell each other their maxima and sums, and each finishes a half of the columns: its lanes of tensor memory are the
        // other's too
        const bool joined = alt && nt > 1;
        if (ok) ok = px_wait_warp(&o_end[t], (uint32_t)(sh & 1));
        tc_fence_after();
        if (joined) {                                      // (by way of tensor memory, where the group's scores were)
            if (ok && !idle) {
                asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(s_t), "f"(m_ref), "f"(l) : "memory");
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            tc_fence_before();
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&joint);
            if (ok) ok = px_wait_warp(&joint, 0);
            tc_fence_after();
        }
        if (ok && !idle && (t == 0 || joined || !alt)) {
            float4* dst = reinterpret_cast<float4*>(p.part_o) + (size_t)w.part * 32 * p.rows_p + (r - w.part_row0);      // rows side by side: a warp's stores are whole lines
            float f0 = 1.f, f1 = 0.f;
            if (joined) {
                float2 ml;
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "r"(tmem + (1 - t) * 256 + lane_base) : "memory");
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                const float m = px_max(m_ref, ml.x);      // (-inf is no weight in either group; a maximum that is NaN stays)
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
                    const uint32_t theirs = tmem + (1 - t) * 256 + 128 + lane_base + c;
#pragma unroll
                    for (int h = 0; h < 64; h += 32) {
                        uint32_t x[32];
                        TC_LD32(theirs + h, x);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[h + k] = __float_as_uint(fmaf(__uint_as_float(o[h + k]), f0, __uint_as_float(x[k]) * f1));
                    }
                }
                if constexpr (TREE && !I8) {               // drafts' values that are not finite, for the rows that see them
                    uint32_t noted = 0;
#pragma unroll
                    for (int k = 0; k < 8; ++k) noted |= hidden_s[sh & 3][k];
                    unsigned rows_of = noted ? __ballot_sync(0xffffffffu, r_ok && m_ref != -INFINITY && p.sees_any(w, r, hidden_s[sh & 3])) : 0u;
                    for (; rows_of; rows_of &= rows_of - 1u) {
                        const int who = __ffs(rows_of) - 1;
                        const float2 v = p.hidden_values(w, r - lane + who, hidden_s[sh & 3], __shfl_sync(0xffffffffu, m_ref, who), c + 2 * lane);
#pragma unroll
                        for (int k = 0; k < 64; ++k) {
                            const float x = __shfl_sync(0xffffffffu, k & 1 ? v.y : v.x, k >> 1);
                            if (lane == who) o[k] = __float_as_uint(__uint_as_float(o[k]) + x);
                        }
                    }
                }
                if constexpr (TREE) {
                    if (w.part < 0) {
                        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;      // no key: zeros; NaN stays
                        if (r_ok) p.store64(w, r, c, o, inv);
                        continue;
                    }
                }
#pragma unroll
                for (int k = 0; k < 64; k += 4)
                    if (r_ok) dst[(size_t)((c + k) >> 2) * p.rows_p] = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
            }
            if (r_ok && (t == 0 || !alt) && (!TREE || w.part >= 0)) reinterpret_cast<float2*>(p.part_ml)[(size_t)w.part * p.rows_p + (r - w.part_row0)] = make_float2(m_ref, l);
        }
        if (TREE && joined && ok) {                       // nor does a group go on while the other still reads its results
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&joint);
            ok = px_wait_warp(&joint, 1);
        }
        if (!ok) fail(18);
        return ok;
        });
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
}


// [128][slot][page, layer, K | V, head], boxes of `box` slots x 128 bytes
inline int px_encode(CUtensorMap* tm, const wf_kv_layout* kv, int box, const char* who) {
    if (((long long)kv->max_pages + 1) * kv->layers * 2 * kv->kv_heads > 0x7fffffffll) { set_error("%s: a pool of at most 2^31 heads' rows of pages", who); return WF_ERR_UNSUPPORTED; }
    EncodeTiledFn fn = tc_encoder();
    if (!fn) { set_error("%s: cuTensorMapEncodeTiled unavailable", who); return WF_ERR_CUDA; }
    const cuuint64_t gdim[3] = {AT_D, (cuuint64_t)kv->page_size, (cuuint64_t)kv->max_pages * kv->layers * 2 * kv->kv_heads};
    const int es_ = kv->dtype == WF_I8 ? 1 : 2;
    const cuuint64_t gstride[2] = {(cuuint64_t)AT_D * es_, (cuuint64_t)kv->page_size * AT_D * es_};
    const cuuint32_t bx[3] = {(cuuint32_t)(128 / es_), (cuuint32_t)box, 1}, es[3] = {1, 1, 1};
    const CUresult cr = fn(tm, es_ == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, kv->pool, gdim, gstride, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) { set_error("%s: tensor map failed (%d)", who, (int)cr); return WF_ERR_CUDA; }
    return WF_OK;
}

}  // namespace

}  // namespace wf
