// What a request asks of its logits before a token is drawn: penalties for tokens that were there before, biases, and a grammar's mask, in one pass.
//
// With c the times that token v was drawn (or drafted) and "seen" for those and the prompt's: y = x / r where x > 0 and x r elsewhere for seen tokens, then
// y - f c - p [c > 0], then + bias, then -inf where the grammar does not allow v; in float, rounded once to the logits' type.  Entries that nothing of it concerns are
// copied as they are (left alone where the result goes over the logits).
//
// A block has a run of a sequence's logits, row after row.  It first notes the tokens there that the history, the drafts or a bias concerns: a bitmap, the number of them in
// front of each word of it, and so the place of each token's own word (times drawn, whether seen) in a list as long as there are such tokens.  All of it are whole numbers whose
// order of arrival does not show.  Meanwhile the first logits are on their way: each warp moves chunks of 2 KB (of 512 bytes where there are few) through a ring of two in shared memory,
// changes its listed tokens there, a lane each, and masks on the way out.  A draft's own past, which differs from row to row, is the common bits of its mask and of a set
// of drafts for each listed token.
//
// Bound by memory: each logit is read and written once; masked vectors are not read.  32 trees of 60 drafts over 128256 tokens in bf16, histories of 2000, a grammar that hides a
// third: 187 us, 4.7 TB/s of the 890 MB that have to move (a third of the rows is hardly read; 191 where a warp asks for its next chunk only behind this one, 916 without rings and lists); one row of them in float 10, latencies.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "wf_bitnet.h"

namespace wf {

namespace {

constexpr int LG_WARPS = 12, LG_THREADS = 32 * LG_WARPS;
constexpr int LG_CHUNK = 2048, LG_STAGES = 2;          // bytes of a warp's chunk, and chunks of its ring
constexpr int LG_SHORT = 512;                          // bytes of a chunk where there is little to read, and warps would have none
constexpr int lg_ring(int bytes) { return LG_WARPS * LG_STAGES * (bytes + 16); }
constexpr int LG_SLICE = 131072, LG_ENTRIES = 8192;    // columns that a block's bitmap has, and entries of a list, at most
constexpr int LG_BLOCKS = 2;                           // blocks of an SM
constexpr int LG_TABLE_COST = 28;                      // what a block's table takes, in chunks' times
constexpr int LG_MIN_RUN = 2;                          // chunks of a block at least
constexpr int LG_NODES = 256;                          // drafts of a sequence at most: a thread each
static_assert(LG_NODES <= LG_THREADS, "");
constexpr uint32_t LG_SEEN = 0x80000000u, LG_DRAFT = 0x40000000u, LG_TIMES = 0x3fffffffu;      // of an entry's word: in the history, a draft, times drawn

struct LogitsParams {
    wf_logits_args a;
    int slice, groups;             // columns of a slice (a multiple of a chunk; nearly always all there are), and blocks of each slice
    int run;                       // chunks of a block
    int entries, tables;
};

template <typename T> struct LgType;
template <> struct LgType<float> {
    static __device__ __forceinline__ float get(const float& v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct LgType<__nv_bfloat16> {
    static __device__ __forceinline__ float get(const __nv_bfloat16& v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct LgType<__half> {
    static __device__ __forceinline__ float get(const __half& v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ void lg_async16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }

template <typename T, int BYTES>
__global__ void __launch_bounds__(LG_THREADS, LG_BLOCKS) process_logits_kernel(const __grid_constant__ LogitsParams p) {
    constexpr int E = 16 / (int)sizeof(T), CHUNK = BYTES / (int)sizeof(T), GROUPS = CHUNK / 32, VECS = BYTES / 512;
    extern __shared__ __align__(16) unsigned char lg_smem[];
    __shared__ uint32_t mask_s[LG_WARPS][LG_STAGES][GROUPS];
    __shared__ int warp_n[LG_WARPS], found[4];
    __shared__ float bias_s[LG_THREADS];
    const wf_logits_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, words = p.slice / 32;
    uint32_t* entry = reinterpret_cast<uint32_t*>(lg_smem + lg_ring(BYTES));          // [entries]
    uint32_t* touched = entry + p.entries;             // [words] a bit per token that has an entry
    uint32_t* same = touched + words;                  // [drafts][2 words of mask] the drafts of the same token, by one of them
    uint16_t* bias = reinterpret_cast<uint16_t*>(same + 128 * a.mask_words * a.mask_words);    // [entries] the place of its bias among the sequence's, from 1
    uint16_t* token_of = bias + (a.bias_ids ? p.entries : 0);          // [entries] the token, from the first column's (mod 2^16: a chunk's tokens are near one another)
    uint16_t* front = token_of + p.entries;            // [words + 1] entries in front of a word's first
    uint8_t* draft_of = reinterpret_cast<uint8_t*>(front + words + 2);         // [entries] the draft that stands for the token
    const int slice = blockIdx.x / p.groups, group = blockIdx.x - slice * p.groups;
    const int s_lo = slice * p.slice, s_hi = min(a.vocab, s_lo + p.slice), per_row = (s_hi - s_lo + CHUNK - 1) / CHUNK;
    pdl_wait_prior();
    pdl_launch_dependents();
    // this block's sequence (a.sequences: rows behind the last one, a.sequences + 1: in front of the first one), its rows first .. end, and its run of their chunks
    int b, first, end, part;
    if (a.offsets) {
        int before = 0;                                // runs of the sequences in front
        b = -1;
        for (int s0 = 0; s0 <= a.sequences + 1; s0 += LG_THREADS) {
            const int s = s0 + tid;
            int from = 0, to = 0;
            if (s <= a.sequences) {
                from = a.sequences > 0 ? min(max(a.offsets[s], 0), a.rows) : 0;
                to = s < a.sequences ? max(min(a.offsets[s + 1], a.rows), from) : a.rows;
            } else if (s == a.sequences + 1 && a.sequences > 0) {
                to = min(max(a.offsets[0], 0), a.rows);
            }
            const int n = (int)(((long long)(to - from) * per_row + p.run - 1) / p.run);
            int in = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int z = __shfl_up_sync(0xffffffffu, in, o); if (lane >= o) in += z; }
            if (lane == 31) warp_n[warp] = in;
            __syncthreads();
            int total = 0, base = before;
#pragma unroll
            for (int w = 0; w < LG_WARPS; ++w) { if (w < warp) base += warp_n[w]; total += warp_n[w]; }
            const int at = group - base - (in - n);
            if (at >= 0 && at < n) { found[0] = s; found[1] = from; found[2] = to; found[3] = at; }
            before += total;
            __syncthreads();
            if (group < before) { b = found[0]; first = found[1]; end = found[2]; part = found[3]; break; }
        }
        if (b < 0) return;                             // (the same in all threads)
    } else {
        const int parts = (per_row + p.run - 1) / p.run;
        b = first = group / parts;
        end = b + 1;
        part = group - b * parts;
        if (b >= a.rows) return;
    }
    const bool none = b >= a.sequences, tables = !none && p.tables, masked = !none && a.allowed, in_place = a.logits == a.out;
    if (in_place && !tables && !masked) return;
    // its first row and chunk there, how many chunks, and the columns that they have
    const long long at0 = (long long)part * p.run;
    const int row0 = first + (int)(at0 / per_row), col0 = (int)(at0 % per_row);
    const int chunks = (int)min((long long)p.run, (long long)(end - first) * per_row - at0);
    const bool one_row = col0 + chunks <= per_row;
    const int lo = one_row ? s_lo + col0 * CHUNK : s_lo, hi = one_row ? min(s_hi, lo + chunks * CHUNK) : s_hi;
    const uint32_t ring = smem_u32(lg_smem) + warp * LG_STAGES * (BYTES + 16);
    T* const ring_p = reinterpret_cast<T*>(lg_smem + warp * LG_STAGES * (BYTES + 16));
    constexpr int STEP = (BYTES + 16) / (int)sizeof(T);

    // a warp's chunks are every twelfth of the block's
    struct Chunk { int left, row, col; };              // chunks of the block from this one on (none: 0 or less), its row and place there
    auto step = [&](Chunk& c) { c.left -= LG_WARPS; c.col += LG_WARPS; while (c.col >= per_row) { c.col -= per_row; ++c.row; } };
    auto from_of = [&](const Chunk& c) { return s_lo + c.col * CHUNK; };
    auto in_of = [&](const Chunk& c) { return reinterpret_cast<const T*>(a.logits) + (size_t)c.row * a.row_stride + from_of(c); };
    Chunk ahead{chunks - warp, row0, col0 + warp};     // the chunk whose mask is asked for next
    while (ahead.col >= per_row) { ahead.col -= per_row; ++ahead.row; }
    Chunk asked = ahead, now = ahead;                  // whose logits are; the one to change
    // the mask's word of this lane's 32 tokens; bits behind the last token are 0
    auto mask_of = [&](const Chunk& c) -> uint32_t {
        const int n = s_hi - from_of(c) - lane * 32;
        if (c.left <= 0 || lane >= GROUPS || n <= 0) return 0u;
        const uint32_t valid = n < 32 ? (1u << n) - 1u : ~0u;
        return masked ? reinterpret_cast<const uint32_t*>(a.allowed)[(size_t)c.row * a.allowed_stride + (from_of(c) >> 5) + lane] & valid : valid;
    };
    // Asks for a chunk: its 16-byte vectors from the boundary at or in front of its first token on (a row may begin anywhere), but for those that the mask hides
    auto ask = [&](const Chunk& c, uint32_t word, int stage) {
        if (lane < GROUPS) mask_s[warp][stage][lane] = word;
        if (c.left > 0 && !in_place) {
            const T* x = in_of(c);
            const int off = (int)((uintptr_t)x % 16 / sizeof(T)), n = min(CHUNK, s_hi - from_of(c));
            const uint32_t dst = ring + stage * (BYTES + 16);
            if (off == 0 && n == CHUNK) {              // the usual case: a vector's bits lie in one word, and words a whole number of lanes apart
                const T* xl = x + lane * E;
#pragma unroll
                for (int u = 0; u < VECS; ++u) {
                    const uint32_t bits = masked ? __shfl_sync(0xffffffffu, word, u * E + lane * E / 32) >> (lane * E & 31) & ((1u << E) - 1u) : 1u;
                    if (bits) lg_async16(dst + lane * 16 + u * 512, xl + u * 32 * E);
                }
            } else
#pragma unroll
            for (int u = 0; u < VECS + 1; ++u) {
                const int vec = u * 32 + lane, t0 = vec * E - off;             // its first token; in an aligned row the others are in the same word
                const uint32_t w0 = __shfl_sync(0xffffffffu, word, max(t0, 0) / 32), w1 = __shfl_sync(0xffffffffu, word, min(t0 + E - 1, CHUNK - 1) / 32);
                if (t0 < n && (!masked || (off ? (w0 | w1) != 0u : (w0 >> (t0 & 31) & ((1u << E) - 1u)) != 0u))) lg_async16(dst + vec * 16, x + t0);
                if (u == VECS - 1 && !off) break;                               // (the last vector only where the row begins inside one)
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint32_t next[LG_STAGES];                          // a chunk's mask is asked for a ring ahead of its logits
#pragma unroll
    for (int i = 0; i < LG_STAGES; ++i) { next[i] = mask_of(ahead); step(ahead); }
#pragma unroll
    for (int i = 0; i < LG_STAGES - 1; ++i) {
        ask(asked, next[i], i);
        step(asked);
        next[i] = mask_of(ahead);
        step(ahead);
    }
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (tables) {
        // what comes from memory is asked for at once: the first biases and the drafts, a thread each, lengths and weights
        const int n_b = a.bias_ids ? a.bias_width : 0, n_nodes = a.node_mask ? min(end - first, 64 * a.mask_words) : 0;
        const int32_t *h = a.history + (size_t)b * a.history_stride, *ids = a.bias_ids + (size_t)b * a.bias_width;
        const int my_id = tid < n_b ? ids[tid] : -1, my_node = tid < n_nodes ? a.node_tokens[first + tid] : -1;
        const float my_bias = tid < n_b ? a.bias_values[(size_t)b * a.bias_width + tid] : 0.f;
        if (a.repetition) rep = a.repetition[b];
        if (a.frequency) freq = a.frequency[b];
        if (a.presence) pres = a.presence[b];
        const int n_h = !a.history ? 0 : min(max(a.history_lens ? a.history_lens[b] : a.history_width, 0), a.history_width), drawn = a.prompt_lens ? a.prompt_lens[b] : 0;
        const int used = (hi - lo + 31) / 32;          // words of the bitmap
        for (int i = tid; i < (p.entries + used + 3) / 4; i += LG_THREADS) reinterpret_cast<uint4*>(entry)[i] = make_uint4(0u, 0u, 0u, 0u);      // (and the bitmap behind it)
        for (int i = tid; a.bias_ids && i < p.entries / 8; i += LG_THREADS) reinterpret_cast<uint4*>(bias)[i] = make_uint4(0u, 0u, 0u, 0u);
        auto history = [&](auto token) {               // every token of it that lies in the run's columns, with its place
            const int n4 = (uintptr_t)h % 16 ? 0 : n_h / 4;
            auto in = [&](int v, int i) { if (v >= lo && v < hi) token(v - lo, i); };
            for (int i = tid; i < n4; i += LG_THREADS * 4) {
                int4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = i + u * LG_THREADS < n4 ? reinterpret_cast<const int4*>(h)[i + u * LG_THREADS] : make_int4(-1, -1, -1, -1);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int k = 4 * (i + u * LG_THREADS);
                    in(v[u].x, k); in(v[u].y, k + 1); in(v[u].z, k + 2); in(v[u].w, k + 3);
                }
            }
            for (int i = 4 * n4 + tid; i < n_h; i += LG_THREADS) in(h[i], i);
        };
        auto biases = [&](auto each) {
            if (my_id >= lo && my_id < hi) each(my_id - lo, tid);
            for (int i = tid + LG_THREADS; i < n_b; i += LG_THREADS) { const int v = ids[i]; if (v >= lo && v < hi) each(v - lo, i); }
        };
        auto touch = [&](int v) {
            const uint32_t bit = 1u << (v & 31);
            if (!(*(volatile uint32_t*)&touched[v >> 5] & bit)) atomicOr(&touched[v >> 5], bit);
        };
        const bool draft = my_node >= lo && my_node < hi;
        bias_s[tid] = my_bias;
        __syncthreads();
        history([&](int v, int) { touch(v); });
        if (draft) touch(my_node - lo);
        biases([&](int v, int) { touch(v); });
        __syncthreads();
        {                                              // entries in front of every word
            const int each = (used + LG_THREADS - 1) / LG_THREADS, w0 = min(used, tid * each), w1 = min(used, w0 + each);
            int n = 0;
            for (int w = w0; w < w1; ++w) n += __popc(touched[w]);
            int in = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int z = __shfl_up_sync(0xffffffffu, in, o); if (lane >= o) in += z; }
            if (lane == 31) warp_n[warp] = in;
            __syncthreads();
            int at = in - n;
#pragma unroll
            for (int w = 0; w < LG_WARPS; ++w) if (w < warp) at += warp_n[w];
            for (int w = w0; w < w1; ++w) { front[w] = (uint16_t)at; at += __popc(touched[w]); }
            if (tid == LG_THREADS - 1) front[used] = (uint16_t)at;
        }
        for (int i = tid; i < n_nodes * 2 * a.mask_words; i += LG_THREADS) same[i] = 0u;
        __syncthreads();
        auto place = [&](int v) {
            const int e = front[v >> 5] + __popc(touched[v >> 5] & ((1u << (v & 31)) - 1u));
            token_of[e] = (uint16_t)v;
            return e;
        };
        history([&](int v, int i) {
            uint32_t* e = &entry[place(v)];
            if (!(*(volatile uint32_t*)e & LG_SEEN)) atomicOr(e, LG_SEEN);
            if (i >= drawn) atomicAdd(e, 1u);
        });
        int my_entry = -1;
        if (draft) {                                   // drafts of the same token: the one whose number is left, whichever, stands for all
            my_entry = place(my_node - lo);
            atomicOr(&entry[my_entry], LG_DRAFT);
            draft_of[my_entry] = (uint8_t)tid;
        }
        bool more;                                     // of biases of the same token the last one counts: those that find an earlier one there write again
        do {
            more = false;
            biases([&](int v, int i) { const int e = place(v); if (bias[e] <= i) { bias[e] = (uint16_t)(i + 1); more = true; } });
        } while (__syncthreads_or(more));
        if (a.node_mask) {
            if (draft) atomicOr(&same[draft_of[my_entry] * 2 * a.mask_words + (tid >> 5)], 1u << (tid & 31));
            __syncthreads();
        }
    }
    uint4 neg;                                         // -inf all over
    {
        alignas(16) T q[E];
#pragma unroll
        for (int i = 0; i < E; ++i) q[i] = LgType<T>::put(-INFINITY);
        neg = *reinterpret_cast<const uint4*>(q);
    }
    auto change = [&](int stage) {
        const T* x = in_of(now);
        const int from = from_of(now), n = min(CHUNK, s_hi - from), off = in_place ? 0 : (int)((uintptr_t)x % 16 / sizeof(T));
        T* y = reinterpret_cast<T*>(a.out) + (size_t)now.row * a.out_stride + from;
        T* s = in_place ? y : ring_p + stage * STEP + off;                     // the chunk's tokens
        const uint32_t* keep_s = mask_s[warp][stage];
        int e0 = 0, e1 = 0;                            // its entries
        if (tables) { e0 = front[(from - lo) >> 5]; e1 = front[(from - lo + n + 31) >> 5]; }
        asm volatile("cp.async.wait_group %0;" ::"n"(LG_STAGES - 1) : "memory");
        __syncwarp();
        for (int e = e0 + lane; e < e1; e += 32) {
            const int v = (uint16_t)(token_of[e] - (from - lo));
            const uint32_t w = entry[e], biased = a.bias_ids ? bias[e] : 0;
            uint32_t times = w & LG_TIMES;
            if (!(keep_s[v >> 5] >> (v & 31) & 1u)) continue;
            if (w & LG_DRAFT) {                        // drafts of this token in the row's own past
                const uint32_t* past = reinterpret_cast<const uint32_t*>(a.node_mask + (size_t)now.row * a.mask_words);
                for (int i = 0; i < 2 * a.mask_words; ++i) times += __popc(same[draft_of[e] * 2 * a.mask_words + i] & past[i]);
            }
            const bool seen = times || (w & LG_SEEN);
            float z = LgType<T>::get(s[v]);
            if (seen) z = z > 0.f ? __fdiv_rn(z, rep) : z * rep;
            z -= freq * (float)times + (times ? pres : 0.f);
            if (biased) z += biased <= LG_THREADS ? bias_s[biased - 1] : a.bias_values[(size_t)b * a.bias_width + biased - 1];
            if (seen || biased) s[v] = LgType<T>::put(z);              // (else a draft that is not in this row's past)
        }
        __syncwarp();
        auto one = [&](int v) {
            if (!(keep_s[v >> 5] >> (v & 31) & 1u)) y[v] = LgType<T>::put(-INFINITY);
            else if (!in_place) y[v] = s[v];
        };
        constexpr uint32_t ALL = (1u << E) - 1u;
        if (!masked && in_place) {
        } else if (!in_place && off == 0 && n == CHUNK && !((uintptr_t)y & 15)) {              // the usual case
            const uint32_t keep_l = masked && lane < GROUPS ? keep_s[lane] : 0u;
            const T* sl = s + lane * E;
            T* yl = y + lane * E;
#pragma unroll
            for (int u = 0; u < VECS; ++u) {
                const uint32_t keep = masked ? __shfl_sync(0xffffffffu, keep_l, u * E + lane * E / 32) >> (lane * E & 31) & ALL : ALL;
                alignas(16) T q[E];
                if (keep == 0u) { *reinterpret_cast<uint4*>(yl + u * 32 * E) = neg; continue; }
                *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(sl + u * 32 * E);
                if (keep != ALL) {
#pragma unroll
                    for (int i = 0; i < E; ++i) if (!(keep >> i & 1u)) q[i] = LgType<T>::put(-INFINITY);
                }
                *reinterpret_cast<uint4*>(yl + u * 32 * E) = *reinterpret_cast<const uint4*>(q);
            }
        } else if (!in_place && (((uintptr_t)x ^ (uintptr_t)y) & 15)) {        // the rows lie differently to 16 bytes
            for (int v = lane; v < n; v += 32) one(v);
        } else {
            const int lead = (int)((uintptr_t)y % 16 / sizeof(T)), va = min(n, lead ? E - lead : 0), ve = va + (n - va) / E * E;
#pragma unroll
            for (int u = 0; u < VECS; ++u) {
                const int v = va + (u * 32 + lane) * E;
                if (v >= ve) break;
                uint32_t keep = ALL;
                if (masked) {
                    keep = keep_s[v >> 5] >> (v & 31);
                    if ((v & 31) + E > 32) keep |= keep_s[(v >> 5) + 1] << (32 - (v & 31));
                    keep &= ALL;
                }
                if (in_place && keep == ALL) continue;
                alignas(16) T q[E];
                if (keep) *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(s + v);
                if (keep != ALL) {
#pragma unroll
                    for (int i = 0; i < E; ++i) if (!(keep >> i & 1u)) q[i] = LgType<T>::put(-INFINITY);
                }
                *reinterpret_cast<uint4*>(y + v) = *reinterpret_cast<const uint4*>(q);
            }
            if (lane < va) one(lane);
            if (ve + lane < n) one(ve + lane);
        }
        __syncwarp();                                  // the stage is free
    };
    while (now.left > 0) {
#pragma unroll
        for (int stage = 0; stage < LG_STAGES; ++stage) {
            if (now.left <= 0) break;
            constexpr int LAST = LG_STAGES - 1;
            const int free = (stage + LAST) % LG_STAGES;               // (left by the chunk before)
            ask(asked, next[free], free);
            step(asked);
            next[free] = mask_of(ahead);
            step(ahead);
            change(stage);
            step(now);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

DevMade g_lg_attr;
// entries of words, and of biases and drafts where there are any; bitmap, fronts; the drafts' sets
int lg_smem_bytes(int bytes, int slice, int entries, int mask_words, bool biases) {
    return lg_ring(bytes) + entries * (6 + (biases ? 2 : 0) + (mask_words ? 1 : 0)) + slice / 8 + slice / 16 + 4 + 512 * mask_words * mask_words;
}

template <typename T>
cudaError_t lg_launch(const LogitsParams& p, int bytes, dim3 grid, cudaStream_t s) {
    const size_t smem = (size_t)lg_smem_bytes(bytes, p.slice, p.entries, p.a.mask_words, p.a.bias_ids != nullptr);
    return bytes == LG_SHORT ? launch_pdl(process_logits_kernel<T, LG_SHORT>, grid, LG_THREADS, smem, s, p) : launch_pdl(process_logits_kernel<T, LG_CHUNK>, grid, LG_THREADS, smem, s, p);
}
template <typename T>
int lg_attrs(const char* who) {
    auto set = [&](auto kernel, int bytes) { return cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, lg_smem_bytes(bytes, LG_SLICE, LG_ENTRIES, LG_NODES / 64, true)), who); };
    return set(process_logits_kernel<T, LG_SHORT>, LG_SHORT) || set(process_logits_kernel<T, LG_CHUNK>, LG_CHUNK) ? WF_ERR_CUDA : WF_OK;
}

// How many chunks a block takes.  The time of a run in units of what a chunk takes at the memory's rate over all blocks (about 0.19 us): every round of blocks costs its
// table, and its chunks at least half of that each (what one block alone moves); all of them the memory's rate; and the last block ends half a run behind the others.
int lg_run(long long rows, long long seqs, long long per_row, long long wave, bool tables, bool whole_rows) {
    const long long all = rows * per_row, own = (rows + seqs - 1) / seqs * per_row;           // of all, and of a sequence on average
    long long best = 0, least = 0;
    auto look = [&](long long run) {
        if (run < LG_MIN_RUN || run > 1 << 30) return;
        const long long groups = whole_rows ? (per_row + run - 1) / run * rows : (all + run - 1) / run + (own % run ? seqs / 2 : 0), rounds = (groups + wave - 1) / wave;
        const long long cost = 2 * rounds * (tables ? LG_TABLE_COST : 4) + std::max(rounds * run, 2 * all / wave) + run;
        if (!best || cost < least) { best = run; least = cost; }
    };
    for (int k = 1; k <= 16; ++k) look((4 * all + k * wave - 1) / (k * wave));
    for (int k = 1; k <= 16; ++k) look((own + k - 1) / k);
    return best ? (int)best : LG_MIN_RUN;
}

// whether rows of the one have bytes of rows of the other (rows of the same stride may lie between each other)
bool lg_overlap(uintptr_t x, uintptr_t y, const wf_logits_args& a, int es) {
    const unsigned long long row = (unsigned long long)a.vocab * es, sx = (unsigned long long)a.row_stride * es, sy = (unsigned long long)a.out_stride * es, n = a.rows - 1;
    if (x + n * sx + row <= y || y + n * sy + row <= x) return false;
    if (n == 0 || sx != sy) return true;
    const unsigned long long off = (x > y ? x - y : y - x) % sx;
    return off < row || sx - off < row;
}

}  // namespace

}  // namespace wf

using namespace wf;

extern "C" int wf_process_logits(const wf_logits_args* args, void* stream) {
    const char* who = "wf_process_logits";
    if (!args) { set_error("%s: null args", who); return WF_ERR_INVALID; }
    LogitsParams p = {};
    p.a = *args;
    wf_logits_args& a = p.a;
    if (a.rows < 0 || a.vocab <= 0 || a.sequences < 0) { set_error("%s: bad shape [%d, %d] of %d sequences", who, a.rows, a.vocab, a.sequences); return WF_ERR_INVALID; }
    if (a.vocab > 1 << 30 || a.rows > 1 << 30) { set_error("%s: at most 2^30 columns and rows (got %d, %d)", who, a.vocab, a.rows); return WF_ERR_UNSUPPORTED; }
    if (a.dtype != WF_F32 && a.dtype != WF_BF16 && a.dtype != WF_F16) { set_error("%s: logits must be f32, bf16 or f16", who); return WF_ERR_INVALID; }
    if (a.rows > 1 && (a.row_stride < a.vocab || a.out_stride < a.vocab)) { set_error("%s: row strides %lld, %lld below %d columns", who, a.row_stride, a.out_stride, a.vocab); return WF_ERR_INVALID; }
    if (!a.offsets && a.sequences != a.rows) { set_error("%s: %d rows of %d sequences want offsets", who, a.rows, a.sequences); return WF_ERR_INVALID; }
    if (a.sequences > 65534) { set_error("%s: at most 65534 sequences (got %d)", who, a.sequences); return WF_ERR_UNSUPPORTED; }
    if (a.history_width < 0 || a.bias_width < 0 || a.mask_words < 0) { set_error("%s: negative width", who); return WF_ERR_INVALID; }
    if (a.history_width > 1 << 29) { set_error("%s: a history is at most 2^29 tokens (got %d)", who, a.history_width); return WF_ERR_UNSUPPORTED; }
    if (a.bias_width > 65535) { set_error("%s: at most 65535 biases a sequence (got %d)", who, a.bias_width); return WF_ERR_UNSUPPORTED; }
    if (a.mask_words > LG_NODES / 64) { set_error("%s: at most %d drafts a sequence (got %d words of mask)", who, LG_NODES, a.mask_words); return WF_ERR_UNSUPPORTED; }
    if (a.rows == 0) return WF_OK;
    if (a.history_width == 0) a.history = nullptr;
    if (a.bias_width == 0) a.bias_ids = nullptr;
    if (a.mask_words == 0) a.node_mask = nullptr;
    if (!a.node_mask) a.mask_words = 0;
    if (!a.logits || !a.out || (a.bias_ids && !a.bias_values) || (a.node_mask && !a.node_tokens)) { set_error("%s: null pointer", who); return WF_ERR_INVALID; }
    if (a.history && a.history_stride < a.history_width && a.sequences > 1) { set_error("%s: history stride %lld below its width %d", who, a.history_stride, a.history_width); return WF_ERR_INVALID; }
    if (a.allowed && a.rows > 1 && a.allowed_stride < (a.vocab + 31) / 32) { set_error("%s: mask stride %lld below its %d words", who, a.allowed_stride, (a.vocab + 31) / 32); return WF_ERR_INVALID; }
    if (a.logits == a.out && a.rows > 1 && a.row_stride != a.out_stride) { set_error("%s: the same memory with row strides %lld and %lld", who, a.row_stride, a.out_stride); return WF_ERR_INVALID; }
    const int es = a.dtype == WF_F32 ? 4 : 2;
    if (a.logits != a.out && lg_overlap((uintptr_t)a.logits, (uintptr_t)a.out, a, es)) { set_error("%s: out overlaps the logits without being them", who); return WF_ERR_INVALID; }
    if ((uintptr_t)a.logits % es || (uintptr_t)a.out % es) { set_error("%s: logits are not aligned to their type", who); return WF_ERR_INVALID; }
    if ((uintptr_t)a.node_mask & 7) { set_error("%s: the drafts' masks must be 8-byte aligned", who); return WF_ERR_INVALID; }
    // Entries of a list are at most what the sequence brings, and at most the columns of a slice
    const long long brings = (a.history ? a.history_width : 0ll) + (a.bias_ids ? a.bias_width : 0) + (a.node_mask ? 64 * a.mask_words : 0);
    p.tables = brings > 0;
    // short chunks where the others would not give every warp of an SM one
    const int bytes = (long long)a.rows * a.vocab * es < (long long)LG_WARPS * sm_count() * LG_CHUNK ? LG_SHORT : LG_CHUNK, chunk = bytes / es;
    const long long most = brings > LG_ENTRIES ? LG_ENTRIES : LG_SLICE;
    p.slice = (int)((a.vocab < most ? a.vocab : most) + 511) / 512 * 512;
    const long long slices = ((long long)a.vocab + p.slice - 1) / p.slice, per_row = (p.slice + chunk - 1) / chunk;
    const long long seqs = a.offsets ? a.sequences + 2ll : a.sequences;            // (and the rows behind the last one, and in front of the first)
    const int full = lg_smem_bytes(bytes, p.slice, (int)(std::min(brings, (long long)p.slice) + 7) / 8 * 8, a.mask_words, a.bias_ids != nullptr);
    const long long wave = std::max((full + 6144 <= 113 * 1024 ? LG_BLOCKS : 1) * sm_count() / slices, 1ll);
    p.run = lg_run(a.rows, a.offsets && a.sequences ? a.sequences : seqs, per_row, wave, p.tables, !a.offsets);
    const long long all = a.rows * per_row;
    const long long groups = a.offsets ? (all + p.run - 1) / p.run + seqs : (per_row + p.run - 1) / p.run * seqs;        // every sequence's last run may be short
    const long long columns = a.offsets ? p.slice : std::min((long long)p.slice, (long long)p.run * chunk);
    p.entries = (int)(std::min(brings, columns) + 7) / 8 * 8;
    if (groups * slices > 0x7fffffffll || groups > 0x7fffffffll) { set_error("%s: too many rows and columns (%d, %d)", who, a.rows, a.vocab); return WF_ERR_UNSUPPORTED; }
    p.groups = (int)groups;
    if (int rc = g_lg_attr.once([&]() -> int { return lg_attrs<float>(who) || lg_attrs<__nv_bfloat16>(who) || lg_attrs<__half>(who) ? WF_ERR_CUDA : WF_OK; })) return rc;
    const dim3 grid((unsigned)(groups * slices));
    cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = a.dtype == WF_F32 ? lg_launch<float>(p, bytes, grid, s) : a.dtype == WF_BF16 ? lg_launch<__nv_bfloat16>(p, bytes, grid, s) : lg_launch<__half>(p, bytes, grid, s);
    return launch_check(e, who);
}
