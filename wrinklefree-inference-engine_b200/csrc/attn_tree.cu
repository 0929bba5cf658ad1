// Attention of drafted tokens over the paged cache: every sequence brings up to 256 new tokens that are in the cache already, and each of them sees the tokens in front
// of the drafts and those drafts that its mask names.
//
// A sequence's n drafts of G query heads are n G rows per key/value head, which share every key: a dense product (attn_px.cuh), of which only the tiles that reach the
// drafts look at masks.  Rows stand in tiles of 256; where several blocks share a tile's keys, their results are joined as the chunks of decode attention are (running maximum m, sum l of 2^(s - m), weighted values o; the result is sum o_i 2^(m_i - M) / sum l_i 2^(m_i - M)).
//
// The host knows neither lengths nor drafts.  The work of all sequences, key/value heads and row tiles lies on one line, a block an SM takes an equal stretch of it
// (every block sums over the sequences for itself, in a warp), and so a row tile's keys lie with one block or with several that follow one another.  A tile that one block has
// is written straight to the output; of the others every block has at most two, one that it ends and one that it begins, whose results go to its two parts of the
// workspace, and the second kernel joins them.  (A block per tile and split instead, in waves, with 10 us a block before its first product and behind its last, against 4 us from
// one tile to the next: 48 sequences of 12 drafts over up to 4096 keys 177 us instead of 134, 8 of 250 over up to 16384 with 64 heads 670 instead of 629, 31 of 25 over int8 241
// instead of 213; with what came since, 193.)
//
// Bound by the memory where rows are few (the 48: 0.73 us for a tile of 64 keys an SM, 6.4 TB/s), by a tile's softmax and the products' turns on the tensor cores where there are
// 256 (1500 of 2000 clocks are exponentials, maxima and sums), by the conversion of codes for int8 pools (1650).
//
// A row that sees no key gets zeros.  A value that is not finite under a key that a row does not see would make it NaN (0 times it): among the drafts' values the warp that loads them
// looks for such ones, puts zeros there and notes the drafts; rows that do see them get them at the end.  (Rows found by their
// NaN and computed again key by key would keep the block's other roles waiting for longer than their limit behind long contexts.)
#include <algorithm>

#include "attn_px.cuh"

namespace wf {

namespace {

constexpr int TX_WORDS = 4;                            // words of a mask: 256 drafts
constexpr int TX_ROWS = 2 * PX_ROWS;                   // rows of a block
constexpr int TX_SPAN = 2 * PX_KEYS;                   // keys are cut in steps of two tiles, one for each group of a block
constexpr int TX_COST1 = 5, TX_COST2 = 7;              // of such a step, for one group of rows and for two
constexpr int TX_COST0 = 10;                           // of a row tile itself, its queries and results: 3 to 4 us
constexpr int TX_LEAST = 2;                            // steps of a block at least, where there are so few
constexpr int TX_SNAP = 3;                             // fewer steps than this of a tile's start or end are left to the neighbour
constexpr int TX_REGS = 168;                           // 384 threads of an SM's 65536

// what the two kernels read of a sequence
struct TxSeq { int first, n, ctx, keys, rows, tiles; };
// A part of a row tile that several blocks have, for the second kernel.  Two of a block: 2 c of the tile that it ends (or has a middle of), 2 c + 1 of the one that it begins.
struct __align__(16) TxPart {
    long long tile;                // the row tile's place on the line (none: no such part)
    int row, rows, kvh;            // row 0 of the tile among all T G rows, rows of the tile, key/value head
    int behind;                    // of one that begins: the blocks behind that may have parts
    int pad[2];
};

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
    int blocks;
    TxPart* parts;                 // [2 blocks]
    int* live;                     // whether there is any work
    float *part_o, *part_ml;       // [parts][AT_D / 4][rows_p][4], [parts][rows_p][2]
    int rows_p;
    void* out;
    int out_dtype;
    int box;
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
    static __device__ __forceinline__ int cost(const TxSeq& s) { return TX_COST0 + s.tiles * (s.rows > PX_ROWS ? TX_COST2 : TX_COST1); }
    __device__ __forceinline__ int units(const TxSeq& s) const { return tiles_of_rows(s.rows) * Hkv; }
    // Blocks that share a line so long, and where the stretch of one begins
    __device__ __forceinline__ int sharers(long long all) const { return (int)min((long long)blocks, max(all / (TX_LEAST * TX_COST1), 1ll)); }
    static __device__ __forceinline__ long long begin_of(long long all, int n, int c) { return all * c / n; }
    // the first step of a row tile that lies x or more behind its start
    static __device__ __forceinline__ int step_at(const TxSeq& s, long long x) {
        const int each = s.rows > PX_ROWS ? TX_COST2 : TX_COST1;
        if (x <= TX_COST0) return 0;
        if (x >= cost(s)) return s.tiles;
        const int i = ((int)x - TX_COST0 + each - 1) / each, snap = min(TX_SNAP, s.tiles / 2);
        return i < snap ? 0 : i > s.tiles - snap ? s.tiles : i;
    }

    // A block's way along the line, in one warp: its stretch, and the row tile that comes next (sequence b's number u, from `at` on, its steps from s0 on)
    // and the rest of the row tile that the block before begins, which comes last: blocks begin with whole tiles, so that those of the same keys read them at a time.
    struct Walk { long long to, at, all; int n, b, u, s0, narrow; TxSeq s; PxWork late; };
    __device__ __forceinline__ PxWork first(Walk& k) const {
        const int lane = threadIdx.x & 31;
        long long mine = 0;
        int rows = 0;
        bool wide = false;
        for (int b = lane; b < B; b += 32) { const TxSeq q = seq(b); mine += (long long)cost(q) * units(q); rows += min(q.rows, T * G); wide = wide || q.rows > PX_ROWS; }
        long long all = mine, total_rows = rows;
#pragma unroll
        for (int o = 16; o; o >>= 1) { all += __shfl_xor_sync(0xffffffffu, all, o); total_rows += __shfl_xor_sync(0xffffffffu, total_rows, o); }
        if (total_rows > (long long)T * G) all = 0;    // (offsets that do not rise)
        if (blockIdx.x == 0 && lane == 0) *live = all > 0;
        if (lane < 2) parts[2 * blockIdx.x + lane].tile = -1;
        __syncwarp();
        PxWork none = {};
        const int n = sharers(all);
        k.b = B;
        k.late.rows = 0;
        k.narrow = !__any_sync(0xffffffffu, wide);
        if (!all || (int)blockIdx.x >= n) return none;
        k.all = all;
        k.n = n;
        const long long from = begin_of(all, n, blockIdx.x);
        k.to = begin_of(all, n, blockIdx.x + 1);
        long long before = 0;
        for (int b0 = 0; b0 < B; b0 += 32) {           // the sequence that the stretch begins in
            long long in = 0;
            if (b0 + lane < B) { const TxSeq q = seq(b0 + lane); in = (long long)cost(q) * units(q); }
            const long long own = in;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const long long y = __shfl_up_sync(0xffffffffu, in, o); if (lane >= o) in += y; }
            const unsigned here = __ballot_sync(0xffffffffu, own > 0 && from < before + in);
            if (here) {
                const int who = __ffs(here) - 1;
                k.b = b0 + who;
                k.at = before + __shfl_sync(0xffffffffu, in - own, who);
                break;
            }
            before += __shfl_sync(0xffffffffu, in, 31);
        }
        k.s = seq(k.b);
        const long long each = cost(k.s);
        k.u = (int)((from - k.at) / each);
        k.at += k.u * each;
        k.s0 = step_at(k.s, from - k.at);
        return next(k);
    }
    __device__ __forceinline__ PxWork next(Walk& k) const {
        while (k.b < B && k.at < k.to) {
            PxWork w;
            const int s0 = k.s0, s1 = step_at(k.s, k.to - k.at), u = k.u, b = k.b;
            const TxSeq s = k.s;
            const long long tile = k.at;
            k.at += cost(s);
            k.s0 = 0;
            if (++k.u == units(s)) {                   // on to the next sequence that has work
                k.u = 0;
                const int lane = threadIdx.x & 31;
                unsigned here = 0;
                for (++k.b; k.b < B; k.b += 32) {
                    here = __ballot_sync(0xffffffffu, k.b + lane < B && seq(k.b + lane).rows > 0);
                    if (here) { k.b += __ffs(here) - 1; break; }
                }
                if (k.b < B) k.s = seq(k.b);
            }
            if (s1 > s0) {
                const int row_tiles = tiles_of_rows(s.rows);
                w.rows = s.rows;
                w.row0 = u % row_tiles * TX_ROWS;
                w.kvh = u / row_tiles;
                w.key0 = s0 * TX_SPAN;
                w.key1 = min(s.keys, s1 * TX_SPAN);
                w.first = s.first;
                w.ctx = s.ctx;
                w.part = s0 > 0 ? 2 * blockIdx.x : s1 < s.tiles ? 2 * blockIdx.x + 1 : -1;
                if (w.part >= 0) {                     // (all lanes: the same)
                    TxPart t;
                    t.tile = tile; t.row = s.first * G + w.row0; t.rows = min(s.rows - w.row0, TX_ROWS); t.kvh = w.kvh;
                    t.behind = s0 > 0 ? 0 : min((int)((tile + cost(s) - 1) * k.n / k.all), k.n - 1) - (int)blockIdx.x;
                    parts[w.part] = t;
                }
                w.part_row0 = w.row0;
                w.narrow = k.narrow;
                w.table = block_table + (size_t)b * max_blocks;
                if (s0 == 0) return w;
                k.late = w;                            // (the first of the stretch alone begins behind a tile's start)
            }
        }
        PxWork w = k.late;
        k.late.rows = 0;
        return w;
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

    // whether row r sees any of the drafts noted
    __device__ __forceinline__ bool sees_any(const PxWork& w, int r, const uint32_t* noted) const {
        const u64* sees = mask + (size_t)(w.first + r / G) * words;
        u64 any = 0;
        for (int i = 0; i < words; ++i) any |= sees[i] & ((u64)noted[2 * i + 1] << 32 | noted[2 * i]);
        return any != 0;
    }
    // Row r's weighted values of columns c and c + 1, by the whole warp (c is the lane's own), of those drafts and of the values among them that are not finite; m: its maximum
    __device__ __forceinline__ float2 hidden_values(const PxWork& w, int r, const uint32_t* noted, float m, int c) const {
        const int lane = threadIdx.x & 31;
        float2 sum = make_float2(0.f, 0.f);
        const u64* sees = mask + (size_t)(w.first + r / G) * words;
        const uint2 qw = *(reinterpret_cast<const uint2*>(q + (((size_t)w.first + r / G) * H + w.kvh * G + r % G) * AT_D) + lane);
        const float x[4] = {bf16lo(qw.x), bf16hi(qw.x), bf16lo(qw.y), bf16hi(qw.y)};
        for (int i = 0; i < words; ++i)
            for (u64 which = sees[i] & ((u64)noted[2 * i + 1] << 32 | noted[2 * i]); which; which &= which - 1ull) {
                const int j = w.ctx + i * 64 + __ffsll((long long)which) - 1, page = w.table[j / page_size];      // (of a page: what is none reads as zeros)
                const size_t kr = ((((size_t)page * layers + layer) * 2) * Hkv + w.kvh) * page_size + j % page_size, vr = kr + (size_t)Hkv * page_size;
                const uint2 a = *(reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(pool) + kr * AT_D) + lane);
                const uint32_t b = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const __nv_bfloat16*>(pool) + vr * AT_D + c);
                const float s = warp_sum(x[0] * bf16lo(a.x) + x[1] * bf16hi(a.x) + x[2] * bf16lo(a.y) + x[3] * bf16hi(a.y));
                const float e = exp2f((scale_log2e == 0.f ? 0.f : s * scale_log2e) - m);
                if (!isfinite(bf16lo(b))) sum.x += e * bf16lo(b);
                if (!isfinite(bf16hi(b))) sum.y += e * bf16hi(b);
            }
        return sum;
    }
};

template <bool I8>
__maxnreg__(I8 ? PX_REGS8 : TX_REGS) __global__ void tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ TxParams p) {
    extern __shared__ unsigned char smem_raw[];
    px_block<I8>(tmap, p, smem_raw, [] { pdl_wait_prior(); });
}

// Joins the parts of row tiles that several blocks had, and writes zeros where no sequence has a row.  What there is to join the first kernel's blocks have written down; every
// block here counts it for itself and takes its share.  A piece is 32 rows (a lane each: the parts lie so) of one key/value head and 32 columns, all of a part's columns under way
// together.  Of tiles of a few parts a block takes eight pieces, a warp each; of tiles of many it takes one, its warps every eighth of the parts, and they meet in shared memory.
// Bound by latency: 6 us from the last part to the last row.  (A block for every 32 rows and 16 columns of the output, most of which had nothing to do: 250 us of 8 sequences of 250
// drafts with 64 heads, where one block zeroed the rows of no sequence 130.)  Which sequence a token belongs to is found ahead of the wait: the kernel before has waited for the offsets.
constexpr int TX_MERGE = 256, TX_MERGE_COLS = 8;       // (columns by fours)
constexpr int TX_PIECES = 32 / TX_MERGE_COLS;          // of the columns
constexpr int TX_FEW = 4;                              // parts that a warp takes alone
__global__ void __launch_bounds__(TX_MERGE, 2) tree_merge_kernel(const __grid_constant__ TxParams p) {
    constexpr int WARPS = TX_MERGE / 32;
    __shared__ float2 ml_s[WARPS][32];
    __shared__ float4 o_s[WARPS][TX_MERGE_COLS][32];
    extern __shared__ TxPart part_s[];                     // [2 blocks]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto lives = [&](int t) {
        int lo = 0, hi = p.B;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (p.offsets[mid] <= t) lo = mid; else hi = mid; }
        const TxSeq s = p.seq(lo);
        return s.rows > 0 && t >= s.first && t < s.first + s.n;
    };
    // a lane looks at a token, the warp writes the zeros; every warp of the grid has one in as many tokens as there are warps
    const long long warps = (long long)gridDim.x * WARPS, t0 = (long long)warp * gridDim.x + blockIdx.x;
    long long t = t0 + lane * warps;
    bool dead = t < p.T && !lives((int)t);
    pdl_wait_prior();
    pdl_launch_dependents();
    for (int i = tid; i < 2 * p.blocks * (int)(sizeof(TxPart) / 16); i += TX_MERGE) reinterpret_cast<uint4*>(part_s)[i] = px_ldcg(reinterpret_cast<const uint4*>(p.parts) + i);
    const bool any = ldcg_i32(p.live) != 0;
    const long long row16 = (long long)p.H * AT_D / (p.out_dtype == WF_BF16 ? 8 : 4);        // 16 bytes each
    for (long long from = t0; from < p.T; from += 32 * warps) {
        for (unsigned who = __ballot_sync(0xffffffffu, t < p.T && (dead || !any)); who; who &= who - 1u) {
            uint4* y = reinterpret_cast<uint4*>(p.out) + (from + (__ffs(who) - 1) * warps) * row16;
            for (int i = lane; i < row16; i += 32) y[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        t += 32 * warps;
        dead = t < p.T && !lives((int)t);
    }
    if (!any) return;
    __syncthreads();
    // the items of a tile are its first block's: thread c's
    __shared__ int sums[WARPS], found[2];
    int items = 0;
    if (tid < p.blocks) {
        const TxPart& tile = part_s[2 * tid + 1];
        const int pieces = (tile.rows + 31) / 32 * TX_PIECES;
        if (tile.tile >= 0) items = tile.behind < TX_FEW ? (pieces + WARPS - 1) / WARPS : pieces;
    }
    int before = items;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += y; }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { if (w < warp) before += sums[w]; all += sums[w]; }
    before -= items;
    for (int item = blockIdx.x; item < all; item += gridDim.x) {
        if (item >= before && item < before + items) { found[0] = tid; found[1] = item - before; }
        __syncthreads();
        const int c = found[0], local = found[1];
        const TxPart tile = part_s[2 * c + 1];
        const bool few = tile.behind < TX_FEW;
        const int piece = few ? local * WARPS + warp : local, col = piece % TX_PIECES * TX_MERGE_COLS, r = piece / TX_PIECES * 32 + lane;
        float M = -INFINITY, L = 0.f;
        float4 y[TX_MERGE_COLS];
#pragma unroll
        for (int i = 0; i < TX_MERGE_COLS; ++i) y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < tile.rows) {
#pragma unroll 2
            for (int i = few ? 0 : warp; i <= tile.behind; i += few ? 1 : WARPS) {
                const int part = i ? 2 * (c + i) : 2 * c + 1;
                if (part_s[part].tile != tile.tile) continue;      // (what is left of a tile's keys to a block can be nothing)
                const float2 ml = reinterpret_cast<const float2*>(p.part_ml)[(size_t)part * p.rows_p + r];
                float4 v[TX_MERGE_COLS];
#pragma unroll
                for (int k = 0; k < TX_MERGE_COLS; ++k) v[k] = reinterpret_cast<const float4*>(p.part_o)[((size_t)part * 32 + col + k) * p.rows_p + r];
                // a part of nothing (-inf) has no weight, whatever stands there; a maximum that is NaN is none of those, and stays NaN to the end
                const float m = px_max(M, ml.x), f0 = M == -INFINITY ? 0.f : exp2f(M - m), f1 = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
                const bool nothing = ml.x == -INFINITY;
                L = nothing ? L : L * f0 + ml.y * f1;
#pragma unroll
                for (int k = 0; k < TX_MERGE_COLS; ++k) {
                    if (nothing) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    y[k].x = y[k].x * f0 + f1 * v[k].x; y[k].y = y[k].y * f0 + f1 * v[k].y; y[k].z = y[k].z * f0 + f1 * v[k].z; y[k].w = y[k].w * f0 + f1 * v[k].w;
                }
                M = m;
            }
        }
        const int row = tile.row + r;
        const size_t at = ((size_t)(row / p.G) * p.H + tile.kvh * p.G + row % p.G) * 32 + col;
        auto store = [&](int k, float4 o, float l) {
            const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;          // no key: zeros; NaN stays
            o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
            if (p.out_dtype == WF_BF16) reinterpret_cast<uint2*>(p.out)[at + k] = make_uint2(pack_bf16x2(o.x, o.y), pack_bf16x2(o.z, o.w));
            else reinterpret_cast<float4*>(p.out)[at + k] = o;
        };
        if (few) {
            if (r < tile.rows) {
#pragma unroll
                for (int k = 0; k < TX_MERGE_COLS; ++k) store(k, y[k], L);
            }
            __syncthreads();
            continue;
        }
        ml_s[warp][lane] = make_float2(M, L);
#pragma unroll
        for (int k = 0; k < TX_MERGE_COLS; ++k) o_s[warp][k][lane] = y[k];
        __syncthreads();
        if (r < tile.rows) {                           // a warp finishes four columns
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) m = px_max(m, ml_s[w][lane].x);
            float l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float2 ml = ml_s[w][lane];
                if (ml.x == -INFINITY) continue;
                const float f = exp2f(ml.x - m);
                const float4 v = o_s[w][warp][lane];
                l = fmaf(ml.y, f, l);
                o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
            }
            store(warp, o, l);
        }
        __syncthreads();
    }
}
static_assert(TX_MERGE / 32 == TX_MERGE_COLS, "a warp for every four columns of a piece");

DevMade g_tx_attr;

struct TxSize { int blocks, rows_p; size_t head, bytes; };

TxSize tx_size(int H, int Hkv, int words) {
    TxSize z;
    z.blocks = std::min(sm_count(), TX_MERGE);
    z.rows_p = std::min(TX_ROWS, (64 * words * (H / Hkv) + 31) / 32 * 32);
    z.head = 256 + (size_t)2 * z.blocks * sizeof(TxPart);
    z.bytes = z.head + (size_t)2 * z.blocks * z.rows_p * (AT_D + 2) * sizeof(float);
    return z;
}

// what the call refuses for its size alone, and has no workspace for
const char* tx_too_large(int B, int T, int H, int Hkv, int words) {
    return words > TX_WORDS ? "at most 256 drafts a sequence (4 words of mask)" : (long long)T * H > 1 << 24 ? "at most 2^24 rows of queries" : B > 1 << 16 ? "at most 65536 sequences"
         : nullptr;
}

}  // namespace

}  // namespace wf

using namespace wf;

extern "C" size_t wf_tree_attn_workspace_bytes(int B, int tokens, int H, int kv_heads, int mask_words) {
    if (B <= 0 || tokens <= 0 || H <= 0 || kv_heads <= 0 || mask_words <= 0 || tx_too_large(B, tokens, H, kv_heads, mask_words)) return 0;
    return tx_size(H, kv_heads, mask_words).bytes;
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
    const TxSize z = tx_size(H, kv->kv_heads, mask_words);
    if (!workspace || workspace_bytes < z.bytes) { set_error("%s: workspace too small (%zu < %zu)", who, workspace_bytes, z.bytes); return WF_ERR_INVALID; }
    if ((uintptr_t)workspace & 15) { set_error("%s: the workspace must be 16-byte aligned", who); return WF_ERR_INVALID; }
    TxParams p = {};
    p.q = (const __nv_bfloat16*)q; p.pool = kv->pool; p.scales = kv_scales_of(kv);
    p.block_table = block_table; p.seq_lens = seq_lens; p.offsets = offsets; p.mask = (const u64*)mask; p.words = mask_words;
    p.max_blocks = max_blocks; p.B = B; p.T = tokens; p.H = H; p.Hkv = kv->kv_heads; p.G = H / kv->kv_heads;
    p.layers = kv->layers; p.layer = layer; p.page_size = kv->page_size; p.max_pages = kv->max_pages;
    p.scale_log2e = scale * 1.4426950408889634f;
    p.blocks = z.blocks;
    p.live = (int*)workspace;
    p.parts = (TxPart*)((char*)workspace + 256);
    p.part_o = (float*)((char*)workspace + z.head);
    p.part_ml = p.part_o + (size_t)2 * z.blocks * z.rows_p * AT_D;
    p.rows_p = z.rows_p;
    p.out = out; p.out_dtype = out_dtype;
    p.box = 16;
    while (p.box < PX_KEYS && kv->page_size % (2 * p.box) == 0) p.box *= 2;
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
    const long long rows = (long long)tokens * p.G, items = std::max((rows + 31) / 32 * p.Hkv * TX_PIECES, (tokens + TX_MERGE - 1ll) / TX_MERGE);
    return launch_check(launch_pdl(tree_merge_kernel, dim3((unsigned)std::min(items, 2ll * z.blocks)), TX_MERGE, 2 * z.blocks * sizeof(TxPart), s, p), "tree_merge");
}
