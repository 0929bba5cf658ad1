// What a request asks of its logits before a token is drawn: penalties for tokens that were there before, biases, and a grammar's mask, in one pass.
//
// With c the times that token v was drawn (or drafted) and "seen" for those and the prompt's: y = x / r where x > 0 and x r elsewhere for seen tokens, then
// y - f c - p [c > 0], then + bias, then -inf where the grammar does not allow v; in float, rounded once to the logits' type.  Entries that nothing of it concerns are
// copied as they are (left alone where the result goes over the logits).
//
// A block has a slice of the vocabulary of one sequence: it counts the sequence's history into a table in shared memory (whole numbers: the order of the atomics does not
// show) and then takes its share of the sequence's rows, a warp or several to a row.  Rows of drafted tokens differ by what each one's own past adds, up to 256
// tokens: those of the slice stand in a short list of the warp's, and in a bitmap beside the table's.  Only where a bitmap or the mask has something to say is an
// entry more than copied.
//
// Bound by memory: each logit is read and written once; a masked vector is not read at all.
#include <cuda_fp16.h>

#include "common.cuh"
#include "wf_bitnet.h"

namespace wf {

namespace {

typedef unsigned long long u64;

constexpr int LG_THREADS = 256, LG_WARPS = LG_THREADS / 32;
constexpr int LG_SLICE = 4096;                         // tokens of a slice at most
constexpr int LG_NODES = 256;                          // drafts of a sequence at most
constexpr int LG_AHEAD = 4;                            // vectors of a lane under way together
constexpr uint32_t LG_SEEN = 0x80000000u;

struct LogitsParams {
    wf_logits_args a;
    int slice, row_parts;
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

// n <= 32 bits from bit `at` of the words on
__device__ __forceinline__ uint32_t lg_bits(const uint32_t* w, int at, int n) {
    uint32_t v = w[at >> 5] >> (at & 31);
    if ((at & 31) + n > 32) v |= w[(at >> 5) + 1] << (32 - (at & 31));
    return n < 32 ? v & ((1u << n) - 1u) : v;
}

template <typename T>
__global__ void __launch_bounds__(LG_THREADS) process_logits_kernel(const __grid_constant__ LogitsParams p) {
    constexpr int E = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) uint32_t lg_smem[];
    __shared__ uint32_t past_bits[LG_WARPS][LG_SLICE / 32];
    __shared__ uint16_t past_list[LG_WARPS][LG_NODES];
    const wf_logits_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t* count = lg_smem;                         // [slice] drawn so often; LG_SEEN: there before
    uint32_t* touched = count + p.slice;               // [slice / 32] a bit per entry that the history or a bias concerns
    uint16_t* bias_at = reinterpret_cast<uint16_t*>(touched + p.slice / 32);      // [slice] its bias, from 1
    const int lo = blockIdx.x * p.slice, hi = min(a.vocab, lo + p.slice);
    const int b = blockIdx.y;
    pdl_wait_prior();
    pdl_launch_dependents();
    int r0, r1;                                        // this block's rows
    if (a.offsets) {
        const int end = a.sequences > 0 ? min(max(a.offsets[a.sequences], 0), a.rows) : 0;
        r0 = b < a.sequences ? min(max(a.offsets[b], 0), a.rows) : end;
        r1 = b < a.sequences ? max(min(a.offsets[b + 1], a.rows), r0) : a.rows;
    } else {
        r0 = min(b, a.rows);
        r1 = b < a.sequences ? min(b + 1, a.rows) : a.rows;
    }
    const int first = r0, per = (r1 - r0 + p.row_parts - 1) / p.row_parts;
    r0 += min(r1 - r0, per * (int)blockIdx.z);
    r1 = min(r1, r0 + per);
    if (r0 >= r1) return;
    const bool none = b >= a.sequences;                // rows behind the last sequence
    if (none && a.out == a.logits) return;
    const bool tables = !none && (a.history || a.bias_ids);
    if (tables) {
        for (int i = tid; i < p.slice + p.slice / 32 + p.slice / 2; i += LG_THREADS) lg_smem[i] = 0u;
        __syncthreads();
        if (a.history) {
            const int32_t* h = a.history + (size_t)b * a.history_stride;
            const int n = min(max(a.history_lens ? a.history_lens[b] : a.history_width, 0), a.history_width), drawn = a.prompt_lens ? a.prompt_lens[b] : 0;
            for (int i = tid; i < n; i += LG_THREADS) {
                const int v = h[i];
                if (v < lo || v >= hi) continue;
                if (i >= drawn) atomicAdd(&count[v - lo], 1u);
                atomicOr(&count[v - lo], LG_SEEN);
                atomicOr(&touched[(v - lo) >> 5], 1u << ((v - lo) & 31));
            }
        }
        if (a.bias_ids) {
            // entries of an id in order: the last one counts, and it is the one that no later one of the same id follows
            for (int i = tid; i < a.bias_width; i += LG_THREADS) {
                const int v = a.bias_ids[(size_t)b * a.bias_width + i];
                if (v < lo || v >= hi) continue;
                bool last = true;
                for (int j = i + 1; j < a.bias_width && last; ++j) last = a.bias_ids[(size_t)b * a.bias_width + j] != v;
                if (last) {
                    bias_at[v - lo] = (uint16_t)(i + 1);
                    atomicOr(&touched[(v - lo) >> 5], 1u << ((v - lo) & 31));
                }
            }
        }
    }
    const bool nodes = !none && a.node_mask;
    if (nodes)
        for (int i = lane; i < p.slice / 32; i += 32) past_bits[warp][i] = 0u;
    __syncthreads();
    const float rep = !none && a.repetition ? a.repetition[b] : 1.f, freq = !none && a.frequency ? a.frequency[b] : 0.f, pres = !none && a.presence ? a.presence[b] : 0.f;
    const int rows = r1 - r0, of_row = rows >= LG_WARPS ? 1 : rows >= 4 ? 2 : rows >= 2 ? 4 : 8;       // warps of a row
    const int share = p.slice / of_row;
    for (int unit = warp; unit < rows * of_row; unit += LG_WARPS) {
        const int row = r0 + unit / of_row, slo = lo + unit % of_row * share, shi = min(hi, slo + share);
        if (slo >= shi) continue;
        int past = 0;
        if (nodes) {                                   // what this draft's own past adds in the slice
            for (int w = 0; w < a.mask_words; ++w) {
                const u64 seen = a.node_mask[(size_t)row * a.mask_words + w];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int j = w * 64 + half * 32 + lane;
                    int v = -1;
                    if ((seen >> (half * 32 + lane) & 1) && first + j < a.rows) v = a.node_tokens[first + j];
                    const bool in = v >= slo && v < shi;
                    const unsigned who = __ballot_sync(0xffffffffu, in);
                    if (in) {
                        past_list[warp][past + __popc(who & ((1u << lane) - 1u))] = (uint16_t)(v - lo);
                        atomicOr(&past_bits[warp][(v - lo) >> 5], 1u << ((v - lo) & 31));
                    }
                    past += __popc(who);
                }
            }
            __syncwarp();
        }
        const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.row_stride;
        T* y = reinterpret_cast<T*>(a.out) + (size_t)row * a.out_stride;
        const uint32_t* ok = !none && a.allowed ? reinterpret_cast<const uint32_t*>(a.allowed) + (size_t)row * a.allowed_stride : nullptr;
        const bool in_place = (const void*)x == (const void*)y;
        auto concerned = [&](int v, int n) -> uint32_t { return (tables ? lg_bits(touched, v - lo, n) : 0u) | (past ? lg_bits(past_bits[warp], v - lo, n) : 0u); };
        auto value = [&](float z, int v) -> float {
            const uint32_t c0 = tables ? count[v - lo] : 0u;
            uint32_t c = c0 & ~LG_SEEN;
            for (int i = 0; i < past; ++i) c += past_list[warp][i] == (uint16_t)(v - lo);
            if (c0 | c) z = z > 0.f ? __fdiv_rn(z, rep) : z * rep;
            z -= freq * (float)c + (c ? pres : 0.f);
            if (tables && a.bias_ids) {
                const int i = bias_at[v - lo];
                if (i) z += a.bias_values[(size_t)b * a.bias_width + i - 1];
            }
            return z;
        };
        auto one = [&](int v) {
            const bool keep = !ok || (ok[v >> 5] >> (v & 31) & 1u);
            const bool work = concerned(v, 1);
            if (keep && !work && in_place) return;
            y[v] = !keep ? LgType<T>::put(-INFINITY) : work ? LgType<T>::put(value(LgType<T>::get(x[v]), v)) : x[v];
        };
        // vectors between the row's 16-byte boundaries, entries one by one in front of and behind them (all of them where the two rows lie differently to it)
        const int off = (int)((uintptr_t)(x + slo) % 16 / sizeof(T));
        int va = min(shi, slo + (off ? E - off : 0)), ve = va + (shi - va) / E * E;
        if (((uintptr_t)x ^ (uintptr_t)y) & 15) va = ve = shi;
        for (int v = slo + lane; v < va; v += 32) one(v);
        for (int v = ve + lane; v < shi; v += 32) one(v);
        for (int v = va + lane * E; v < ve; v += 32 * E * LG_AHEAD) {
            uint32_t keep[LG_AHEAD], work[LG_AHEAD];
            uint4 q[LG_AHEAD];
#pragma unroll
            for (int u = 0; u < LG_AHEAD; ++u) {
                const int at = v + u * 32 * E;
                keep[u] = at >= ve ? 0u : ok ? lg_bits(ok, at, E) : (1u << E) - 1u;
            }
#pragma unroll
            for (int u = 0; u < LG_AHEAD; ++u) {
                const int at = v + u * 32 * E;
                work[u] = keep[u] ? concerned(at, E) : 0u;
                if (keep[u] && (work[u] || !in_place || keep[u] != (1u << E) - 1u)) q[u] = *reinterpret_cast<const uint4*>(x + at);
            }
#pragma unroll
            for (int u = 0; u < LG_AHEAD; ++u) {
                const int at = v + u * 32 * E;
                if (at >= ve) break;
                if (in_place && !work[u] && keep[u] == (1u << E) - 1u) continue;
                if (keep[u] != (1u << E) - 1u) {
                    alignas(16) T e[E];
                    *reinterpret_cast<uint4*>(e) = keep[u] ? q[u] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                    for (int k = 0; k < E; ++k)
                        if (!(keep[u] >> k & 1u)) e[k] = LgType<T>::put(-INFINITY);
                    q[u] = *reinterpret_cast<const uint4*>(e);
                }
                *reinterpret_cast<uint4*>(y + at) = q[u];
                for (uint32_t m = work[u] & keep[u]; m; m &= m - 1u) {         // few: read again, and stored behind their vector by the thread that stored it
                    const int v1 = at + __ffs(m) - 1;
                    y[v1] = LgType<T>::put(value(LgType<T>::get(x[v1]), v1));
                }
            }
        }
        if (past) {
            __syncwarp();
            for (int i = lane; i < past; i += 32) past_bits[warp][past_list[warp][i] >> 5] = 0u;
            __syncwarp();
        }
    }
}

template <typename T>
cudaError_t lg_launch(const LogitsParams& p, dim3 grid, cudaStream_t s) {
    return launch_pdl(process_logits_kernel<T>, grid, LG_THREADS, (size_t)p.slice * 4 + p.slice / 8 + p.slice * 2, s, p);
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
    if (a.bias_width > 65535) { set_error("%s: at most 65535 biases a sequence (got %d)", who, a.bias_width); return WF_ERR_UNSUPPORTED; }
    if (a.mask_words > LG_NODES / 64) { set_error("%s: at most %d drafts a sequence (got %d words of mask)", who, LG_NODES, a.mask_words); return WF_ERR_UNSUPPORTED; }
    if (a.rows == 0) return WF_OK;
    if (a.history_width == 0) a.history = nullptr;
    if (a.bias_width == 0) a.bias_ids = nullptr;
    if (a.mask_words == 0) a.node_mask = nullptr;
    if (!a.logits || !a.out || (a.bias_ids && !a.bias_values) || (a.node_mask && !a.node_tokens)) { set_error("%s: null pointer", who); return WF_ERR_INVALID; }
    if (a.history && a.history_stride < a.history_width && a.sequences > 1) { set_error("%s: history stride %lld below its width %d", who, a.history_stride, a.history_width); return WF_ERR_INVALID; }
    if (a.allowed && a.rows > 1 && a.allowed_stride < (a.vocab + 31) / 32) { set_error("%s: mask stride %lld below its %d words", who, a.allowed_stride, (a.vocab + 31) / 32); return WF_ERR_INVALID; }
    if (a.logits == a.out && a.rows > 1 && a.row_stride != a.out_stride) { set_error("%s: the same memory with row strides %lld and %lld", who, a.row_stride, a.out_stride); return WF_ERR_INVALID; }
    const int es = a.dtype == WF_F32 ? 4 : 2;
    if ((uintptr_t)a.logits % es || (uintptr_t)a.out % es) { set_error("%s: logits are not aligned to their type", who); return WF_ERR_INVALID; }
    if ((uintptr_t)a.node_mask & 7) { set_error("%s: the drafts' masks must be 8-byte aligned", who); return WF_ERR_INVALID; }
    // slices as wide as leave the GPU two blocks an SM, and shares of a sequence's rows where even whole sequences do not
    p.slice = LG_SLICE;
    const long long groups = (long long)a.sequences + (a.offsets ? 1 : 0);
    auto blocks = [&](int slice) { return ((long long)a.vocab + slice - 1) / slice * groups; };
    while (p.slice > 512 && blocks(p.slice) < 2ll * sm_count()) p.slice /= 2;
    p.row_parts = 1;
    const long long most = a.offsets ? ((long long)a.rows + a.sequences) / (a.sequences + 1) : 1;      // rows of a sequence, about
    while (p.row_parts < 32 && p.row_parts * 2 * LG_WARPS <= most && blocks(p.slice) * p.row_parts < 4ll * sm_count()) p.row_parts *= 2;
    const dim3 grid((unsigned)((a.vocab + p.slice - 1) / p.slice), (unsigned)(groups ? groups : 1), (unsigned)p.row_parts);
    cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = a.dtype == WF_F32 ? lg_launch<float>(p, grid, s) : a.dtype == WF_BF16 ? lg_launch<__nv_bfloat16>(p, grid, s) : lg_launch<__half>(p, grid, s);
    return launch_check(e, who);
}
