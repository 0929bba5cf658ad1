// Log probabilities of given tokens, with the entropy of their distributions and the most likely alternatives, from a batch's logits in ONE pass.
//
// With z = x / T, m the row's largest logit, a_i = (x_i - m) / T (in log 2), s = sum 2^a_i and t = sum a_i 2^a_i:
//   log p(tok) = (x_tok - m) / T - ln 2 log2 s,   H = -sum p ln p = ln 2 (log2 s - t / s);
// both sums follow the running maximum (s' = s r, t' = (t + s log2 r) r, r = 2^((m - m') / T)).  Logits of -inf have probability 0 and add nothing; differences
// are taken before the scale, so that rows masked with a type's lowest value come out right too.
//
// The k largest (k <= 64) come out of the same pass.  An alternative is a 64-bit key, the number in an order-preserving form above the complement of its index, so
// that keys differ and ties go to the lowest index.  A bound, which k entries are known to reach, keeps almost all entries out: the k-th largest of the threads'
// running maxima (of the ceil(k / 16) + 1 largest of each warp), taken after rounds 1, 4, 16, ... of loads.  What reaches it goes to a buffer of the block, some
// k (1 + 3 log4 rounds) entries of a row in no special order; at the end a thread per candidate counts the larger ones: its place.  A row that fills the
// buffer (rising, or of few different numbers) is read again: then every warp sorts what may belong to its k largest into a list of them (bitonic, by shuffles),
// and the lists are merged.  Entries of -inf are not collected: where there are fewer than k others, the lowest of their indices are looked up at the end.
//
// A row is one block, or a cluster of 2 to 8 for few rows, whose results meet in distributed shared memory: one launch, no workspace.
//
// Bound by memory where there is much to read: 2000 rows of 128256 in float 153 us, 6.7 TB/s.  A small call is a chain of latencies: one row 3.9 us without
// alternatives, 6.1 with one, 8.3 with 20 (bounds, ranks and the meeting of the blocks, a barrier or two each); 64 rows in bf16 with five 11.1, of which 2.5 are its
// bytes.
#include <cuda_fp16.h>

#include "logprobs.cuh"

namespace wf {

namespace {

constexpr int LP_THREADS = 512, LP_WARPS = LP_THREADS / 32;
constexpr int LP_CAND = 2048;                         // candidates of a block
// Blocks' lists of up to so many keys are joined by counting (n^2 / 32 reads of shared memory an SM), longer ones by bisection in each other list (a chain of reads):
// of one row of 128256, eight lists of 20 take 8.5 us counted and 9.4 otherwise, of 24 9.0 and 9.6, of 32 10.5 and 10.2, of 64 21.0 and 13.8; of 33 rows of 32000, four
// lists of 24 take 7.6 and 7.8, of 32 8.0 both, of 64 10.8 and 9.2; of 64 rows, two lists of 24 8.1 both, of 32 8.5 and 8.2.
constexpr int LP_FEW = 20;
constexpr int LP_PEND = 64;                           // entries of a warp's buffer where a row is read again
constexpr float LP_LN2 = 0.6931471805599453f, LP_LOG2E = 1.4426950408889634f;
constexpr float LP_FLOOR = -1000.f;                   // 2^LP_FLOOR is 0: what lies below (also -inf) is brought up to it, so that 0 times it is 0

struct LpParams {
    const void* logits;
    long long ld;
    const int32_t* tokens;
    int V, k, parts;                // parts: blocks a row
    float inv_t;
    float *logprob, *entropy, *top_logprob;
    int32_t* top_id;
};

typedef unsigned long long u64;

__device__ __forceinline__ float lp_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float lp_max_nan(float a, float b) { float y; asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }   // NaN stays NaN
__device__ __forceinline__ u64 lp_key(float x, int i) {
    const uint32_t b = __float_as_uint(x + 0.f);      // -0 and 0 are the same number
    return ((u64)(b ^ ((uint32_t)((int)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float lp_value(u64 key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ u64 lp_shfl_xor(u64 v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ u64 lp_max(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 lp_min(u64 a, u64 b) { return a < b ? a : b; }
// a bitonic sequence over the lanes -> descending
__device__ __forceinline__ u64 lp_bitonic(u64 v, int lane) {
#pragma unroll
    for (int o = 16; o; o >>= 1) { const u64 w = lp_shfl_xor(v, o); v = lane & o ? lp_min(v, w) : lp_max(v, w); }
    return v;
}
__device__ __forceinline__ u64 lp_sort(u64 v, int lane) {      // descending
#pragma unroll
    for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
        for (int o = n >> 1; o; o >>= 1) {
            const u64 w = lp_shfl_xor(v, o);
            const bool up = ((lane & n) == 0 || n == 32) == ((lane & o) == 0);      // this lane keeps the larger
            v = up ? lp_max(v, w) : lp_min(v, w);
        }
    return v;
}
// R x 32 sorted keys (position r * 32 + lane) take in 32 more sorted ones
template <int R>
__device__ __forceinline__ void lp_merge32(u64 (&list)[R], u64 more, int lane) {
    u64 v = __shfl_sync(0xffffffffu, more, 31 - lane);
    list[R - 1] = lp_bitonic(lp_max(list[R - 1], v), lane);    // the larger half of (last 32 of the list, the new ones) stays
    if (R == 2) {
        v = __shfl_sync(0xffffffffu, list[1], 31 - lane);
        const u64 hi = lp_max(list[0], v), lo = lp_min(list[0], v);
        list[0] = lp_bitonic(hi, lane);
        list[R - 1] = lp_bitonic(lo, lane);
    }
}
// the R x 32 largest of two sorted lists, the second in memory
template <int R>
__device__ __forceinline__ void lp_merge(u64 (&list)[R], const u64 (&other)[R], int lane) {
    if (R == 1) {
        const u64 v = __shfl_sync(0xffffffffu, other[0], 31 - lane);
        list[0] = lp_bitonic(lp_max(list[0], v), lane);
    } else {                                           // max with the reversed other list is bitonic over 64 positions
        const u64 a = lp_max(list[0], __shfl_sync(0xffffffffu, other[R - 1], 31 - lane)), b = lp_max(list[R - 1], __shfl_sync(0xffffffffu, other[0], 31 - lane));
        list[0] = lp_bitonic(lp_max(a, b), lane);
        list[R - 1] = lp_bitonic(lp_min(a, b), lane);
    }
}

// The n entries of a warp's buffer into its list, both in shared memory; the list's k-th key is returned and offered to the block's other warps
template <int R>
__device__ __noinline__ u64 lp_flush(u64* list, const u64* pend, int n, int k, u64* bound_s) {
    const int lane = threadIdx.x & 31;
    u64 l[R];
    __syncwarp();
#pragma unroll
    for (int r = 0; r < R; ++r) l[r] = list[r * 32 + lane];
    for (int i = 0; i < n; i += 32) lp_merge32<R>(l, lp_sort(i + lane < n ? pend[i + lane] : 0, lane), lane);
#pragma unroll
    for (int r = 0; r < R; ++r) list[r * 32 + lane] = l[r];
    const u64 kth = __shfl_sync(0xffffffffu, l[(k - 1) >> 5 ? R - 1 : 0], (k - 1) & 31);
    if (lane == 0 && kth) atomicMax(bound_s, kth);
    __syncwarp();
    return kth;
}

struct Sums { float m, s, t; };
// the sums of two parts of a row
__device__ __forceinline__ Sums lp_join(const Sums& a, const Sums& b, float c) {
    Sums o;
    o.m = fmaxf(a.m, b.m);
    const float da = a.m == o.m ? 0.f : lp_max_nan((a.m - o.m) * c, LP_FLOOR), db = b.m == o.m ? 0.f : lp_max_nan((b.m - o.m) * c, LP_FLOOR);
    const float ra = lp_ex2(da), rb = lp_ex2(db);
    o.s = fmaf(a.s, ra, b.s * rb);
    o.t = fmaf(fmaf(a.s, da, a.t), ra, fmaf(b.s, db, b.t) * rb);
    return o;
}

// read once, by an ordinary load: the logits are the work of the kernel before
__device__ __forceinline__ uint4 lp_load(const uint4* a) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(a));
    return r;
}

template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4& w, float* x) { x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w); }
    static __device__ __forceinline__ float one(float v) { return v; }
};
template <> struct LpVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& w, float* x) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = bf16lo(u[i]); x[2 * i + 1] = bf16hi(u[i]); }
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <> struct LpVec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& w, float* x) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i])); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
};

template <typename V>
__device__ __forceinline__ V lp_peer(const V* local, int rank) {       // the same shared-memory address in block `rank` of this cluster
    uint32_t ra;
    V v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(local)), "r"(rank));
    if (sizeof(V) == 8) { u64 w; asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(w) : "r"(ra) : "memory"); v = *reinterpret_cast<const V*>(&w); }
    else { uint32_t w; asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(ra) : "memory"); v = *reinterpret_cast<const V*>(&w); }
    return v;
}

// A block's part of a row, entry by entry: every warp's k largest into its list, then all into list 0.  pend: LP_PEND entries a warp
template <typename T, int R>
__device__ __noinline__ void lp_again(const T* x, int i0, int i1, int k, u64 bound, u64* lists, u64* pend, u64* bound_s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 *const list = lists + warp * R * 32, *const buf = pend + warp * LP_PEND;
    int npend = 0;
    for (int r = 0; r < R; ++r) list[r * 32 + lane] = 0;
    if (threadIdx.x == 0) *bound_s = bound;
    __syncthreads();
    for (int b = i0 + warp * 32; b < i1; b += LP_THREADS) {
        const int i = b + lane;
        const float v = i < i1 ? LpVec<T>::one(x[i]) : -INFINITY;
        const u64 key = lp_key(v, i);
        bound = lp_max(bound, *reinterpret_cast<volatile u64*>(bound_s));
        const bool in = v > -INFINITY && key > bound;
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        if (!who) continue;
        if (npend + __popc(who) > LP_PEND) { bound = lp_max(bound, lp_flush<R>(list, buf, npend, k, bound_s)); npend = 0; }
        if (in) buf[npend + __popc(who & ((1u << lane) - 1))] = key;
        npend += __popc(who);
    }
    if (npend) lp_flush<R>(list, buf, npend, k, bound_s);
    __syncthreads();
    for (int half = LP_WARPS >> 1; half; half >>= 1) {
        if (warp < half) {
            u64 mine[R], other[R];
#pragma unroll
            for (int r = 0; r < R; ++r) { mine[r] = list[r * 32 + lane]; other[r] = list[(half * R + r) * 32 + lane]; }
            lp_merge<R>(mine, other, lane);
#pragma unroll
            for (int r = 0; r < R; ++r) list[r * 32 + lane] = mine[r];
        }
        __syncthreads();
    }
}

// R: 32-key parts of the lists of alternatives (0: none wanted)
template <typename T, int R>
__global__ void __launch_bounds__(LP_THREADS, 2) token_logprobs_kernel(const __grid_constant__ LpParams p) {
    constexpr int VN = LpVec<T>::N, VECS = 16 / VN, RL = R ? R : 1;      // 16 entries a thread and round, the next round's under way
    constexpr int TOPS = LP_TOP_MAX / LP_WARPS + 1;
    __shared__ u64 cand[R ? LP_CAND : 1];
    __shared__ u64 lists[R ? LP_WARPS * RL * 32 : 1];
    __shared__ u64 bound_s;
    __shared__ uint32_t tops[LP_WARPS * TOPS], bound_v;
    __shared__ int ncand, ranks[R ? 8 * LP_FEW : 1];
    __shared__ float part[LP_WARPS][3];
    static_assert(!R || (LP_CAND >= LP_WARPS * LP_PEND && LP_CAND >= 8 * LP_TOP_MAX), "the candidates' space is used again");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cs = p.parts, rank = blockIdx.x % cs, row = blockIdx.x / cs;
    if (R && tid == 0) { bound_v = 0; ncand = 0; }
    if (R && tid < p.k) lists[tid] = 0;
    if (R && tid < 8 * LP_FEW) ranks[tid] = 0;
    if (R) __syncthreads();
    pdl_wait_prior();
    pdl_launch_dependents();
    const T* x = reinterpret_cast<const T*>(p.logits) + (long long)row * p.ld;
    const float c = p.inv_t * LP_LOG2E;
    const int head = min(p.V, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));       // entries in front of the first whole vector
    const int nvec = (p.V - head) / VN, tail = p.V - head - nvec * VN;
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    const int v0 = (int)((long long)nvec * rank / cs), v1 = (int)((long long)nvec * (rank + 1) / cs);
    const uint4 none = make_uint4(0, 0, 0, 0);
    uint4 w[VECS];
    auto load = [&](int b) {
#pragma unroll
        for (int u = 0; u < VECS; ++u) { const int i = b + u * LP_THREADS + tid; w[u] = i < v1 ? lp_load(xv + i) : none; }
    };
    load(v0);
    // the given token's logit, under way while the row is read
    float x_tok = __uint_as_float(0x7fc00000u);
    if (rank == 0 && tid == 0) { const int tok = p.tokens[row]; if (tok >= 0 && tok < p.V) x_tok = LpVec<T>::one(x[tok]); }

    Sums q = {-INFINITY, 0.f, 0.f};
    float bound_x = -INFINITY;                         // entries below are not among the k largest
    // the k-th largest of the threads' numbers, in its ordered form: of each warp's ceil(k / 16) + 1 largest; 0 where there are not so many above -inf
    auto kth_of = [&](float m) {
        const int each = (p.k + LP_WARPS - 1) / LP_WARPS + 1;
        uint32_t mine = m > -INFINITY ? (uint32_t)(lp_key(m, 0) >> 32) : 0;
        for (int r = 0; r < each; ++r) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
            if (lane == __ffs(__ballot_sync(0xffffffffu, mine == top)) - 1) mine = 0;
            if (lane == 0) tops[r * LP_WARPS + warp] = top;
        }
        __syncthreads();
        const int n = each * LP_WARPS;
        if (tid < n) {
            const uint32_t top = tops[tid];
            int larger = 0;
#pragma unroll 8
            for (int i = 0; i < n; ++i) larger += tops[i] >= top + (i >= tid ? 1u : 0u);      // equal ones: the first counts as larger
            if (larger == p.k - 1) bound_v = top;
        }
        __syncthreads();
        return bound_v;
    };
    auto value_of = [](uint32_t ordered) { return ordered ? lp_value((u64)ordered << 32) : -INFINITY; };
    // entry j of n has index i0 + (j / VN) * stride + j % VN
    auto offer = [&](auto& v, int n, int i0, int stride) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < n && v[j] >= bound_x && v[j] > -INFINITY) {
                const int at = atomicAdd(&ncand, 1);
                if (at < LP_CAND) cand[R ? at : 0] = lp_key(v[j], i0 + (j / VN) * stride + j % VN);
            }
    };
    auto add = [&](auto& v, int n, float m) {
        if (m > q.m) {
            const float d = lp_max_nan((q.m - m) * c, LP_FLOOR), r = lp_ex2(d);
            q.t = fmaf(q.s, d, q.t) * r;
            q.s *= r;
            q.m = m;
        }
        const float m0 = q.m == -INFINITY ? 0.f : q.m;
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < n) {
                const float a = lp_max_nan((v[j] - m0) * c, LP_FLOOR), e = lp_ex2(a);
                q.s += e;
                q.t = fmaf(a, e, q.t);
            }
    };

    for (int b = v0, round = 1; b < v1; b += LP_THREADS * VECS, ++round) {
        float v[16];
#pragma unroll
        for (int u = 0; u < VECS; ++u) {
            LpVec<T>::get(w[u], v + u * VN);
            if (b + u * LP_THREADS + tid >= v1) {
#pragma unroll
                for (int j = 0; j < VN; ++j) v[u * VN + j] = -INFINITY;
            }
        }
        load(b + LP_THREADS * VECS);
        float m = v[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) m = fmaxf(m, v[j]);
        if (R) {
            if (!(round & (round - 1)) && (round & 0x55555555)) bound_x = value_of(kth_of(fmaxf(m, q.m)));
            if (m >= bound_x && m > -INFINITY) offer(v, 16, head + (b + tid) * VN, LP_THREADS * VN);
        }
        add(v, 16, m);
    }
    // the entries beside the whole vectors, one a lane: those in front belong to the first block, those behind to the last, as where a block reads its part again
    if (warp == 0 && (rank == 0 || rank == cs - 1)) {
        float v[16];
        const int i = lane < 16 ? lane : head + nvec * VN + lane - 16;
        v[0] = (lane < 16 ? rank == 0 && lane < head : rank == cs - 1 && lane - 16 < tail) ? LpVec<T>::one(x[i]) : -INFINITY;
        if (R) offer(v, 1, i, 0);
        add(v, 1, v[0]);
    }

    // ---- a row's parts together: lanes, warps, blocks of the cluster
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const Sums other = {__shfl_xor_sync(0xffffffffu, q.m, o), __shfl_xor_sync(0xffffffffu, q.s, o), __shfl_xor_sync(0xffffffffu, q.t, o)};
        q = lp_join(q, other, c);
    }
    if (lane == 0) { part[warp][0] = q.m; part[warp][1] = q.s; part[warp][2] = q.t; }
    __syncthreads();
    auto sums_of = [&](int n) {                        // the first n parts, in every lane of a warp
        Sums a = {-INFINITY, 0.f, 0.f};
        if (lane < n) a = {part[lane][0], part[lane][1], part[lane][2]};
#pragma unroll
        for (int o = LP_WARPS / 2; o; o >>= 1) {
            const Sums other = {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)};
            a = lp_join(a, other, c);
        }
        a.m = __shfl_sync(0xffffffffu, a.m, 0); a.s = __shfl_sync(0xffffffffu, a.s, 0); a.t = __shfl_sync(0xffffffffu, a.t, 0);
        return a;
    };
    // the k largest of the first n candidates into list 0, a thread for each: its place is how many are larger
    auto place = [&](int n) {
        for (int i = tid; i < n; i += LP_THREADS) {
            const u64 key = cand[R ? i : 0];
            int at = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) at += cand[R ? j : 0] > key;
            if (at < p.k) lists[R ? at : 0] = key;
        }
        __syncthreads();
    };
    if (warp == 0) q = sums_of(LP_WARPS);
    if (R) {
        int n = ncand;
        if (n > LP_CAND) {
            const int i0 = rank ? head + v0 * VN : 0, i1 = rank == cs - 1 ? p.V : head + v1 * VN;
            lp_again<T, RL>(x, i0, i1, p.k, bound_v ? ((u64)bound_v << 32) - 1 : 0, lists, cand, &bound_s);
        } else {
            if (n > 128) {                             // only those that reach the bound of all of them
                u64 mine[LP_CAND / LP_THREADS], top = 0;
#pragma unroll
                for (int r = 0; r < LP_CAND / LP_THREADS; ++r) { mine[r] = r * LP_THREADS + tid < n ? cand[r * LP_THREADS + tid] : 0; top = lp_max(top, mine[r]); }
                const uint32_t least = kth_of(top ? lp_value(top) : -INFINITY);
                if (tid == 0) ncand = 0;
                __syncthreads();
#pragma unroll
                for (int r = 0; r < LP_CAND / LP_THREADS; ++r)
                    if (mine[r] && (uint32_t)(mine[r] >> 32) >= least) cand[atomicAdd(&ncand, 1)] = mine[r];
                __syncthreads();
                n = ncand;
            }
            place(n);
        }
    }
    if (cs > 1) {
        __syncthreads();
        if (tid == 0) { part[0][0] = q.m; part[0][1] = q.s; part[0][2] = q.t; }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank == 0) {
            Sums mine = {0.f, 0.f, 0.f};
            if (warp == 0 && lane < cs) mine = {lp_peer(&part[0][0], lane), lp_peer(&part[0][1], lane), lp_peer(&part[0][2], lane)};
            const int of = R ? tid / p.k : 0, own = R ? tid - of * p.k : 0;
            if (R && tid < cs * p.k) cand[tid] = lp_peer(&lists[own], of);         // at most 8 x 64
            __syncwarp();
            if (warp == 0 && lane < cs) { part[lane][0] = mine.m; part[lane][1] = mine.s; part[lane][2] = mine.t; }
            __syncthreads();
            if (R && p.k <= LP_FEW) {
                // a key's place is how many are larger, counted by as many threads as there are for each (places beyond the keys that there are hold 0 already)
                const int n = cs * p.k, per = LP_THREADS / n, i = tid / per;
                if (i < n) {
                    const u64 key = cand[i];
                    int at = 0;
#pragma unroll 4
                    for (int j = tid - i * per; j < n; j += per) at += cand[j] > key;
                    if (at) atomicAdd(&ranks[i], at);
                }
                __syncthreads();
                if (tid < n && ranks[tid] < p.k) lists[ranks[tid]] = cand[tid];
                __syncthreads();
            } else if (R) {
                // every block's list is sorted: a key's place is its own plus, of each other list, how many are larger
                if (tid < p.k) lists[tid] = 0;         // (read by the copies above)
                __syncthreads();
                const u64 key = tid < cs * p.k ? cand[tid] : 0;
                int at = own;
                for (int r = 0; key && r < cs; ++r) {
                    if (r == of) continue;
                    int lo = 0, hi = p.k;
                    while (lo < hi) { const int mid = (lo + hi) >> 1; if (cand[r * p.k + mid] > key) lo = mid + 1; else hi = mid; }
                    at += lo;
                }
                if (key && at < p.k) lists[at] = key;
                __syncthreads();
            }
            if (warp == 0) q = sums_of(cs);
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (rank) {                                        // nobody leaves while its shared memory may be read
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            return;
        }
    }
    if (warp) return;
    const float ls = log2f(q.s), nan = __uint_as_float(0x7fc00000u);
    // not ln 2 ((x - m) c - ls): the lowest float under a mask times log2 e is beyond float
    auto log_p = [&](float v) { return fmaf(v - q.m, p.inv_t, -LP_LN2 * ls); };
    const bool empty = q.m == -INFINITY, bad = !(q.s >= 0.f) || q.m == INFINITY;     // no entry above -inf; NaN or +inf among them
    if (lane == 0) {
        p.entropy[row] = bad ? nan : empty ? 0.f : fmaxf(LP_LN2 * (ls - q.t / q.s), 0.f);
        p.logprob[row] = bad || x_tok != x_tok ? nan : empty ? -INFINITY : log_p(x_tok);
    }
    if (R) {
        int have = 0;
#pragma unroll
        for (int r = 0; r < RL; ++r) {
            const int at = r * 32 + lane;
            const u64 key = at < p.k ? lists[at] : 0;
            have += __popc(__ballot_sync(0xffffffffu, key != 0));
            if (!key) continue;
            p.top_id[(size_t)row * p.k + at] = (int)~(uint32_t)key;
            p.top_logprob[(size_t)row * p.k + at] = bad ? nan : log_p(lp_value(key));
        }
        for (int b = 0; have < p.k && b < p.V; b += 32) {      // the others are -inf: the lowest indices of those
            const bool low = b + lane < p.V && LpVec<T>::one(x[b + lane]) == -INFINITY;
            const uint32_t who = __ballot_sync(0xffffffffu, low);
            const int at = have + __popc(who & ((1u << lane) - 1));
            if (low && at < p.k) { p.top_id[(size_t)row * p.k + at] = b + lane; p.top_logprob[(size_t)row * p.k + at] = bad ? nan : -INFINITY; }
            have += __popc(who);
        }
        for (int at = have + lane; at < p.k; at += 32) { p.top_id[(size_t)row * p.k + at] = -1; p.top_logprob[(size_t)row * p.k + at] = nan; }
    }
}

template <typename T, int R>
cudaError_t lp_launch(const LpParams& p, int n, cudaStream_t s) {
    const int cs = p.parts;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n * cs);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cs; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cs > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, R>, p);
}
template <typename T>
cudaError_t lp_launch(const LpParams& p, int n, cudaStream_t s) {
    return p.k == 0 ? lp_launch<T, 0>(p, n, s) : p.k <= 32 ? lp_launch<T, 1>(p, n, s) : lp_launch<T, 2>(p, n, s);
}

}  // namespace

int launch_token_logprobs(const void* logits, int dtype, int n, int V, long long ld, const int32_t* tokens, int k, float temperature, float* logprob, float* entropy,
                          float* top_logprob, int32_t* top_id, cudaStream_t s) {
    if (n < 0 || V <= 0) { set_error("wf_token_logprobs: bad shape [%d, %d]", n, V); return WF_ERR_INVALID; }
    if (V > 1 << 30) { set_error("wf_token_logprobs: at most 2^30 columns (got %d)", V); return WF_ERR_UNSUPPORTED; }       // indices of a step beyond the last column fit too
    if (n > 1 && ld < V) { set_error("wf_token_logprobs: row stride %lld below %d columns", ld, V); return WF_ERR_INVALID; }
    if (k < 0 || k > V) { set_error("wf_token_logprobs: top (%d) of %d", k, V); return WF_ERR_INVALID; }
    if (k > LP_TOP_MAX) { set_error("wf_token_logprobs: top is at most %d (got %d)", LP_TOP_MAX, k); return WF_ERR_UNSUPPORTED; }
    if (!(temperature > 0.f) || !(1.f / temperature * LP_LOG2E < INFINITY) || !(1.f / temperature > 0.f)) { set_error("wf_token_logprobs: temperature must be positive (got %g)", (double)temperature); return WF_ERR_INVALID; }
    if (n == 0) return WF_OK;
    if (!logits || !tokens || !logprob || !entropy || (k > 0 && (!top_logprob || !top_id))) { set_error("wf_token_logprobs: null pointer"); return WF_ERR_INVALID; }
    const int es = dtype == 0 ? 4 : 2;
    if ((uintptr_t)logits % es) { set_error("wf_token_logprobs: logits are not aligned to their type"); return WF_ERR_INVALID; }
    LpParams p;
    p.logits = logits; p.ld = ld; p.tokens = tokens; p.V = V; p.k = k; p.inv_t = 1.f / temperature;
    p.logprob = logprob; p.entropy = entropy; p.top_logprob = top_logprob; p.top_id = top_id;
    // blocks of a row: as many as there are SMs for, while every thread of them has two vectors to read.  One row of 128256 in float with 20 alternatives, lists
    // joined by bisection: 9.4 us, 10.9 on four blocks, 13.3 on two, 16.7 on one.  Two blocks an SM: 37 rows with 5 alternatives 16.3 for 12.1, 64 rows of 32064 7.8 for 6.9, 75 rows of 128256 15.8 for 15.4
    // (with 20 alternatives 19.2 for 20.1); four: 64 rows in bf16 18.3 for 11.3.
    int cs = 1;
    while (cs < 8 && (long long)n * cs * 2 <= sm_count() && (long long)V * es >= 16LL * LP_THREADS * cs * 2) cs *= 2;
    p.parts = cs;
    cudaError_t e;
    if (dtype == 0) e = lp_launch<float>(p, n, s);
    else if (dtype == 1) e = lp_launch<__nv_bfloat16>(p, n, s);
    else if (dtype == 2) e = lp_launch<__half>(p, n, s);
    else { set_error("wf_token_logprobs: logits must be f32, bf16 or f16"); return WF_ERR_INVALID; }
    return launch_check(e, "wf_token_logprobs");
}

}  // namespace wf

extern "C" int wf_token_logprobs(const void* logits, int dtype, int rows, int vocab, long long row_stride, const int32_t* tokens, int top, float temperature, float* logprob,
                                 float* entropy, float* top_logprob, int32_t* top_id, void* stream) {
    return wf::launch_token_logprobs(logits, dtype, rows, vocab, row_stride, tokens, top, temperature, logprob, entropy, top_logprob, top_id, (cudaStream_t)stream);
}
