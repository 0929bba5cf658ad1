// The tensor-level ops under torch's dispatcher, natively: argument checks, output tensors and the launches of one call without a pass through Python.
//   sgl_kernel::bitnet_gemv_cpu / bitnet_gemm_cpu / bitnet_quantize_activations_cpu and their aliases (schemas: sgl_kernel/_ops.py; the names are the
//   reference's, docs/research/sglang_optimization_plan.md:59-75): CUDA kernels of those ops;
//   wf_native::linear, wf_native::mlp: the calls behind BitNetLinearNative and bitnet_mlp_forward (several launches each);
//   wf_native::paged_decode_attn, paged_prefix_attn, paged_plan, paged_release, token_logprobs: the functions of these names in wf_bitnet.ops.
// A call through ctypes spent 20 us of host time on what takes the GPU 6 (one token, 2560 x 2560), and the feed-forward op waited twice for a copy of
// its weight scales to the device; here a call costs about 8 us and the scales travel as kernel parameters.
#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <utility>

#include "wf_bitnet.h"

namespace {

using at::Tensor;

// wf_bitnet._lib.WfError, as the calls through ctypes raise it: callers tell a failed launch from a bad argument by its type
[[noreturn]] void raise_wf_error(const std::string& msg) {
    if (Py_IsInitialized()) {
        pybind11::gil_scoped_acquire gil;
        const pybind11::object type = pybind11::module_::import("wf_bitnet._lib").attr("WfError");
        PyErr_SetString(type.ptr(), msg.c_str());
        throw pybind11::error_already_set();
    }
    TORCH_CHECK(false, msg);
}

void check(int rc) {          // the Python side's mapping of the C status
    if (rc == 0) return;
    const char* msg = wf_last_error();
    TORCH_CHECK_VALUE(rc != -1, msg);
    TORCH_CHECK_NOT_IMPLEMENTED(rc != -2, msg);
    raise_wf_error(msg);
}

void need_gpu(std::initializer_list<const Tensor*> ts) {
    if (!wf_bitnet_available()) raise_wf_error("no compute-capability-10.x CUDA device visible; the BitNet kernels are sm_100a-only and there is no CPU fallback");
    for (const Tensor* t : ts) TORCH_CHECK_VALUE(t->is_cuda(), "expected a CUDA tensor (the B200 BitNet ops have no CPU path)");
}

void* stream() { return (void*)c10::cuda::getCurrentCUDAStream().stream(); }

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t);
    }
    return -1;
}

// Scratch per device and stream, grown to the largest request.  zeroed: the split-K workspace that kernels leave zero; its contents are only ever
// touched by launches on that stream.  The map itself is never destroyed: tensors outlive the CUDA context at exit otherwise.
Tensor workspace(const Tensor& like, int64_t bytes, bool zeroed) {
    static std::mutex& mu = *new std::mutex;
    static auto& all = *new std::map<std::tuple<int, void*, bool>, Tensor>;
    const auto key = std::make_tuple((int)like.get_device(), stream(), zeroed);
    std::lock_guard<std::mutex> lk(mu);
    Tensor& t = all[key];
    if (!t.defined() || t.numel() < bytes) {
        const auto opt = like.options().dtype(at::kByte);
        bytes = std::max<int64_t>(bytes, 1 << 20);
        t = zeroed ? at::zeros({bytes}, opt) : at::empty({bytes}, opt);
    }
    return t;
}

Tensor bitnet_gemv(const Tensor& packed_weights, const Tensor& activations, double scale) {
    need_gpu({&packed_weights, &activations});
    const c10::cuda::CUDAGuard guard(packed_weights.device());
    TORCH_CHECK_VALUE(packed_weights.dim() == 2, "packed_weights must be 2-D");
    const Tensor p = packed_weights.contiguous(), x = activations.contiguous();
    const int N = (int)p.size(0), K = (int)p.size(1) * 4;
    Tensor y = at::empty({N}, p.options().dtype(at::kFloat));
    const size_t need = wf_bitnet_gemm_workspace_bytes(1, N, K);
    Tensor ws = workspace(p, (int64_t)need, true);
    check(wf_bitnet_gemv((const uint8_t*)p.data_ptr(), (const int8_t*)x.data_ptr(), (float)scale, N, K, (float*)y.data_ptr(), ws.data_ptr(), (size_t)ws.numel(), stream()));
    return y;
}

Tensor bitnet_gemm(const Tensor& packed_weights, const Tensor& activations, double scale) {
    need_gpu({&packed_weights, &activations});
    const c10::cuda::CUDAGuard guard(packed_weights.device());
    TORCH_CHECK_VALUE(packed_weights.dim() == 2 && activations.dim() >= 1, "packed_weights must be 2-D");
    const Tensor p = packed_weights.contiguous(), x = activations.contiguous();
    const int M = (int)x.size(0), N = (int)p.size(0), K = (int)p.size(1) * 4;
    Tensor y = at::empty({M, N}, p.options().dtype(at::kFloat));
    const size_t need = wf_bitnet_gemm_workspace_bytes(M, N, K);
    Tensor ws;
    if (need) ws = workspace(p, (int64_t)need, true);
    check(wf_bitnet_gemm((const uint8_t*)p.data_ptr(), (const int8_t*)x.data_ptr(), (float)scale, M, N, K, (float*)y.data_ptr(), need ? ws.data_ptr() : nullptr,
                         need ? (size_t)ws.numel() : 0, stream()));
    return y;
}

struct Quant { Tensor q, scale, rowsum; };

// x2: [M, K] contiguous
Quant quantize(const Tensor& x2, bool per_token) {
    const int M = (int)x2.size(0), K = (int)x2.size(1);
    const int dt = code_of(x2.scalar_type());
    Quant o;
    o.q = at::empty({M, K}, x2.options().dtype(at::kChar));
    o.scale = at::empty({per_token ? M : 1}, x2.options().dtype(at::kFloat));
    o.rowsum = at::empty({std::max(M, 1) + 1}, x2.options().dtype(at::kInt));       // the last entry: the per-tensor absmax cell
    check(wf_act_quant_i8(x2.data_ptr(), dt, M, K, K, per_token ? 1 : 0, (int8_t*)o.q.data_ptr(), (float*)o.scale.data_ptr(), (int32_t*)o.rowsum.data_ptr(),
                          (int32_t*)o.rowsum.data_ptr() + std::max(M, 1), stream()));
    return o;
}

std::tuple<Tensor, Tensor> bitnet_quantize_activations(const Tensor& activations) {
    need_gpu({&activations});
    const c10::cuda::CUDAGuard guard(activations.device());
    const Tensor x2 = (activations.dim() == 1 ? activations.reshape({1, -1}) : activations.reshape({-1, activations.size(-1)})).contiguous();
    Quant o = quantize(x2, false);
    return {o.q.reshape(activations.sizes()), o.scale};
}

void fill_linear(wf_linear_args& a, const Tensor& w, bool tile, int N, int K, const Quant& x, Tensor& out, int out_dtype, Tensor& ws) {
    memset(&a, 0, sizeof a);
    const int M = (int)x.q.size(0);
    a.w = (const uint8_t*)w.data_ptr(); a.w_layout = tile ? 1 : 0; a.N = N; a.K = K;
    a.q = (const int8_t*)x.q.data_ptr(); a.M = M; a.ldq = K;
    a.rowsum = (const int32_t*)x.rowsum.data_ptr();
    a.act_scale = (const float*)x.scale.data_ptr(); a.act_scale_per_token = x.scale.numel() > 1 || M == 1 ? 1 : 0;
    a.nseg = 1; a.seg_end[0] = N;
    a.host_scale = 1.f;
    a.out_mode = 3; a.out_dtype = out_dtype;
    a.out = out.data_ptr(); a.ldo = (int)out.size(1);
    size_t need = M > 8 ? wf_bitnet_gemm_workspace_bytes(M, N, K) : wf_linear_workspace_bytes(M, N, K);
    if (need) {
        need += 4 * (size_t)((N + 15) / 16) + 256;
        ws = workspace(w, (int64_t)need, true);
        a.workspace = ws.data_ptr(); a.workspace_bytes = (size_t)ws.numel();
    }
}

// y [M, N] float = w_scale * W x, x [M, K] quantised with one scale for all of it; w: tile (tile = true) or packed layout
Tensor linear(const Tensor& x, const Tensor& w, bool tile, int64_t N, int64_t K, const Tensor& w_scale) {
    need_gpu({&x, &w, &w_scale});
    const c10::cuda::CUDAGuard guard(w.device());
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == K, "activations.shape[-1] != in_features");
    const Tensor x2 = x.contiguous(), wc = w.contiguous(), sc = w_scale.contiguous();
    TORCH_CHECK_VALUE(sc.scalar_type() == at::kFloat && sc.numel() >= 1, "w_scale must be float32");
    Quant q = quantize(x2, false);
    Tensor out = at::empty({x2.size(0), N}, x2.options().dtype(at::kFloat)), ws;
    wf_linear_args a;
    fill_linear(a, wc, tile, (int)N, (int)K, q, out, 0, ws);
    a.w_scale = (const float*)sc.data_ptr();
    check(wf_ternary_linear(&a, stream()));
    return out;
}

// quantise -> [gate | up] with relu(gate)^2 * up -> norm + quantise -> down; x [M, K], y bf16 [M, down rows]
Tensor mlp(const Tensor& x, const Tensor& gate_up_tile, int64_t N2, const Tensor& down_w, double gate_scale, double up_scale, double down_scale, const Tensor& norm, double eps) {
    need_gpu({&x, &gate_up_tile, &down_w, &norm});
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor x2 = x.contiguous(), dw = down_w.contiguous(), g = norm.contiguous();
    TORCH_CHECK_VALUE(dw.dim() == 2, "packed weights must be 2-D");
    const int M = (int)x2.size(0), K = (int)x2.size(1), F = (int)N2 / 2, D = (int)dw.size(0);
    TORCH_CHECK_VALUE(dw.size(1) * 4 == F, "activations.shape[-1] != in_features");
    TORCH_CHECK_VALUE(g.scalar_type() == at::kBFloat16 && g.numel() >= F, "ffn_sub_norm must have one weight per feed-forward row");
    Quant q = quantize(x2, true);
    const auto bf = x2.options().dtype(at::kBFloat16);
    Tensor h = at::empty({M, F}, bf), ws, ws2;
    wf_linear_args a;
    fill_linear(a, gate_up_tile, true, (int)N2, K, q, h, 1, ws);
    const float gu[2] = {(float)gate_scale, (float)up_scale};
    a.nseg = 2; a.epi_flags = 2;
    check(wf_ternary_linear_scales(&a, gu, stream()));
    Quant q2;
    q2.q = at::empty({M, F}, x2.options().dtype(at::kChar));
    q2.scale = at::empty({M}, x2.options().dtype(at::kFloat));
    q2.rowsum = at::empty({M}, x2.options().dtype(at::kInt));
    check(wf_rmsnorm_quant(h.data_ptr(), g.data_ptr(), (float)eps, M, F, nullptr, (int8_t*)q2.q.data_ptr(), (float*)q2.scale.data_ptr(), (int32_t*)q2.rowsum.data_ptr(), stream()));
    Tensor y = at::empty({M, D}, bf);
    fill_linear(a, dw, false, D, F, q2, y, 1, ws2);
    const float ds[1] = {(float)down_scale};
    check(wf_ternary_linear_scales(&a, ds, stream()));
    return y;
}

Tensor paged_decode_attn(const Tensor& q, const Tensor& pool, int64_t max_pages, int64_t layers, int64_t kv_heads, int64_t page_size, int64_t head_dim, int64_t kv_dtype,
                         int64_t layer, const Tensor& block_table, const Tensor& seq_lens, double scale, at::ScalarType out_dtype) {
    need_gpu({&q, &block_table, &seq_lens});
    const c10::cuda::CUDAGuard guard(q.device());
    TORCH_CHECK_VALUE(q.dim() == 3 && block_table.dim() == 2, "q must be [B, H, D] and block_table [B, blocks]");
    const Tensor qc = q.contiguous();
    const int B = (int)q.size(0), H = (int)q.size(1), D = (int)q.size(2), blocks = (int)block_table.size(1);
    Tensor out = at::empty({B, H, D}, q.options().dtype(out_dtype));
    wf_kv_layout kv;
    memset(&kv, 0, sizeof kv);
    kv.pool = pool.data_ptr();
    kv.max_pages = (int)max_pages; kv.layers = (int)layers; kv.kv_heads = (int)kv_heads; kv.page_size = (int)page_size; kv.head_dim = (int)head_dim; kv.dtype = (int)kv_dtype;
    Tensor ws = workspace(q, (int64_t)wf_attn_workspace_bytes(B, H, D, blocks * (int)page_size), false);
    check(wf_paged_decode_attn(qc.data_ptr(), &kv, (int)layer, (const int32_t*)block_table.data_ptr(), blocks, (const int32_t*)seq_lens.data_ptr(), B, H, (float)scale, out.data_ptr(),
                               code_of(out_dtype), ws.data_ptr(), (size_t)ws.numel(), stream()));
    return out;
}

// an int32 tensor of `dim` dimensions on the device of `like`
void need_i32(const Tensor& t, int64_t dim, const Tensor& like, const char* name) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt, name, " must be int32");
    TORCH_CHECK_VALUE(t.dim() == dim, name, " must have ", dim, " dimension", dim == 1 ? "" : "s");
    TORCH_CHECK_VALUE(t.device() == like.device(), name, " must be on ", like.device());
}
int to_int(int64_t v, const char* name) {
    TORCH_CHECK_VALUE(v >= 0 && v <= 0x7fffffff, name, " out of range");
    return (int)v;
}

// A contiguous tensor in new memory of the current device and stream, straight from torch's allocator: an at::empty takes 1.6 us, most of it on its way there
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
    size_t bytes = c10::elementSize(type);
    for (int64_t s : sizes) bytes *= (size_t)s;
    auto* from = c10::cuda::CUDACachingAllocator::get();
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(c10::Storage::use_byte_size_t(), bytes, from->allocate(bytes), from, true), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                     c10::scalarTypeToTypeMeta(type));
    impl->set_sizes_contiguous(sizes);
    return Tensor(std::move(impl));
}

// A contiguous tensor over part of `buf`, `at` entries of its own type from the start: the outputs of a call share one allocation (1.6 us each otherwise, and a
// slice through the dispatcher 0.9 us)
Tensor part_of(const Tensor& buf, at::ScalarType type, int64_t at, at::IntArrayRef sizes) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buf.storage()), buf.key_set(), c10::scalarTypeToTypeMeta(type));
    impl->set_storage_offset(at);
    impl->set_sizes_contiguous(sizes);
    return Tensor(std::move(impl));
}

Tensor paged_prefix_attn(const Tensor& q, const Tensor& pool, int64_t max_pages, int64_t layers, int64_t kv_heads, int64_t page_size, int64_t head_dim, int64_t kv_dtype,
                         int64_t layer, const Tensor& prefix_table, int64_t prefix_len, const Tensor& block_table, const Tensor& seq_lens, double scale, at::ScalarType out_dtype) {
    need_gpu({&q, &pool, &prefix_table, &block_table, &seq_lens});
    const c10::cuda::CUDAGuard guard(q.device());
    TORCH_CHECK_VALUE(q.dim() == 3 && q.scalar_type() == at::kBFloat16, "q must be bf16 [B, H, D]");
    TORCH_CHECK_VALUE(q.size(2) == head_dim, "q has heads of ", q.size(2), ", the cache of ", head_dim);
    TORCH_CHECK_VALUE(pool.device() == q.device(), "the cache must be on ", q.device());
    need_i32(prefix_table, 1, q, "prefix_table");
    need_i32(block_table, 2, q, "block_table");
    need_i32(seq_lens, 1, q, "seq_lens");
    TORCH_CHECK_VALUE(block_table.size(0) == q.size(0) && seq_lens.size(0) == q.size(0), "block_table and seq_lens must have a row for each of ", q.size(0), " sequences");
    TORCH_CHECK_VALUE(prefix_len >= 0 && prefix_len <= prefix_table.size(0) * page_size, "prefix_len (", prefix_len, ") beyond the ", prefix_table.size(0), " pages of prefix_table");
    Tensor qc = q.contiguous();
    if ((uintptr_t)qc.data_ptr() & 15) qc = qc.clone();
    const Tensor pt = prefix_table.contiguous(), bt = block_table.contiguous(), sl = seq_lens.contiguous();
    const int B = (int)q.size(0), H = (int)q.size(1), D = (int)q.size(2), blocks = to_int(bt.size(1), "block_table"), pre = to_int(prefix_len, "prefix_len");
    to_int(bt.size(1) * page_size, "block_table");
    wf_kv_layout kv;
    memset(&kv, 0, sizeof kv);
    kv.pool = pool.data_ptr();
    kv.max_pages = (int)max_pages; kv.layers = (int)layers; kv.kv_heads = (int)kv_heads; kv.page_size = (int)page_size; kv.head_dim = (int)head_dim; kv.dtype = (int)kv_dtype;
    // memory of this call's own: calls on other streams and captured graphs do not share it (none for sizes that the call refuses)
    const int64_t bytes = (int64_t)wf_prefix_attn_workspace_bytes(B, H, kv.kv_heads, blocks * kv.page_size, pre);
    Tensor out = fresh({bytes || (blocks == 0 && pre == 0) ? B : 0, H, D}, out_dtype), ws = fresh({bytes}, at::kByte);
    check(wf_paged_prefix_attn(qc.data_ptr(), &kv, (int)layer, (const int32_t*)pt.data_ptr(), pre, (const int32_t*)bt.data_ptr(), blocks, (const int32_t*)sl.data_ptr(), B, H, (float)scale,
                               out.data_ptr(), code_of(out_dtype), ws.data_ptr(), (size_t)ws.numel(), stream()));
    return out;
}

// rows, positions, pages, slots [max_tokens], offsets [B + 1], lens [B], free_count [1], status [1]: views of one buffer
std::vector<Tensor> paged_plan(const Tensor& seq_lens, const Tensor& new_lens, Tensor block_table, const Tensor& free_pages, const Tensor& free_count, int64_t page_size,
                               int64_t max_tokens) {
    need_gpu({&seq_lens, &new_lens, &block_table, &free_pages, &free_count});
    const c10::cuda::CUDAGuard guard(block_table.device());
    need_i32(block_table, 2, block_table, "block_table");
    need_i32(seq_lens, 1, block_table, "seq_lens");
    need_i32(new_lens, 1, block_table, "new_lens");
    need_i32(free_pages, 1, block_table, "free_pages");
    need_i32(free_count, 1, block_table, "free_count");
    const int64_t B = block_table.size(0);
    TORCH_CHECK_VALUE(seq_lens.size(0) == B && new_lens.size(0) == B, "seq_lens and new_lens must have an entry for each of the ", B, " rows of block_table");
    TORCH_CHECK_VALUE(free_count.size(0) == 1, "free_count must have one entry");
    TORCH_CHECK_VALUE(block_table.is_contiguous(), "block_table must be contiguous (it is written in place)");
    const Tensor sl = seq_lens.contiguous(), nl = new_lens.contiguous(), fp = free_pages.contiguous();
    const int rows = to_int(B, "block_table"), cap = to_int(max_tokens, "max_tokens"), page = to_int(page_size, "page_size");
    const int64_t cap4 = cap > 1 << 30 ? 0 : (max_tokens + 3) / 4 * 4;      // every map starts on 16 bytes (the call refuses more than 2^30 tokens)
    const Tensor buf = fresh({4 * cap4 + 2 * B + 3}, at::kInt);
    const int64_t at[8] = {0, cap4, 2 * cap4, 3 * cap4, 4 * cap4, 4 * cap4 + B + 1, 4 * cap4 + 2 * B + 1, 4 * cap4 + 2 * B + 2};
    const int64_t len[8] = {max_tokens, max_tokens, max_tokens, max_tokens, B + 1, B, 1, 1};
    int32_t* base = (int32_t*)buf.data_ptr();
    check(wf_paged_plan((const int32_t*)sl.data_ptr(), (const int32_t*)nl.data_ptr(), rows, (int32_t*)block_table.data_ptr(), to_int(block_table.size(1), "block_table"),
                        (const int32_t*)fp.data_ptr(), to_int(fp.size(0), "free_pages"), (const int32_t*)free_count.data_ptr(), page, cap, base + at[1], base, base + at[2], base + at[3],
                        base + at[4], base + at[5], base + at[6], base + at[7], stream()));
    std::vector<Tensor> out;
    out.reserve(8);
    for (int i = 0; i < 8; ++i) out.push_back(part_of(buf, at::kInt, at[i], {len[i]}));
    return out;
}

std::tuple<Tensor, Tensor> paged_release(const Tensor& done, const Tensor& seq_lens, const Tensor& block_table, Tensor free_pages, const Tensor& free_count, int64_t page_size) {
    need_gpu({&done, &seq_lens, &block_table, &free_pages, &free_count});
    const c10::cuda::CUDAGuard guard(block_table.device());
    need_i32(block_table, 2, block_table, "block_table");
    need_i32(seq_lens, 1, block_table, "seq_lens");
    need_i32(free_pages, 1, block_table, "free_pages");
    need_i32(free_count, 1, block_table, "free_count");
    const int64_t B = block_table.size(0);
    TORCH_CHECK_VALUE(done.scalar_type() == at::kBool && done.dim() == 1 && done.device() == block_table.device(), "done must be bool [B] on ", block_table.device());
    TORCH_CHECK_VALUE(done.size(0) == B && seq_lens.size(0) == B, "done and seq_lens must have an entry for each of the ", B, " rows of block_table");
    TORCH_CHECK_VALUE(free_count.size(0) == 1, "free_count must have one entry");
    TORCH_CHECK_VALUE(free_pages.is_contiguous(), "free_pages must be contiguous (it is written in place)");
    const Tensor dn = done.contiguous(), sl = seq_lens.contiguous(), bt = block_table.contiguous();
    const Tensor buf = fresh({B + 1}, at::kInt);
    Tensor lens = part_of(buf, at::kInt, 0, {B}), count = part_of(buf, at::kInt, B, {1});
    check(wf_paged_release((const uint8_t*)dn.data_ptr(), (const int32_t*)sl.data_ptr(), to_int(B, "block_table"), (const int32_t*)bt.data_ptr(), to_int(bt.size(1), "block_table"),
                           (int32_t*)free_pages.data_ptr(), to_int(free_pages.size(0), "free_pages"), (const int32_t*)free_count.data_ptr(), to_int(page_size, "page_size"),
                           (int32_t*)lens.data_ptr(), (int32_t*)count.data_ptr(), stream()));
    return {lens, count};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t top, double temperature) {
    need_gpu({&logits, &tokens});
    const c10::cuda::CUDAGuard guard(logits.device());
    TORCH_CHECK_VALUE(logits.dim() == 2, "logits must be [rows, vocab]");
    need_i32(tokens, 1, logits, "tokens");
    TORCH_CHECK_VALUE(tokens.size(0) == logits.size(0), "tokens must have an entry for each of the ", logits.size(0), " rows of logits");
    const int dt = code_of(logits.scalar_type());
    const Tensor x = logits.stride(1) == 1 || logits.size(1) <= 1 ? logits : logits.contiguous(), tk = tokens.contiguous();
    const int n = to_int(x.size(0), "rows"), V = to_int(x.size(1), "vocab"), k = to_int(top, "top");
    const int64_t ld = n > 1 ? x.stride(0) : V;
    const Tensor& y = ld < V ? x.contiguous() : x;         // rows that overlap (an expanded row)
    const int64_t m = n, kk = k > 64 || k > V ? 0 : k, mk = m * kk;        // (the call refuses more)
    const Tensor buf = fresh({2 * (m + mk)}, at::kFloat);
    Tensor lp = part_of(buf, at::kFloat, 0, {m}), ent = part_of(buf, at::kFloat, m, {m}), tlp = part_of(buf, at::kFloat, 2 * m, {m, kk}), tid = part_of(buf, at::kInt, 2 * m + mk, {m, kk});
    check(wf_token_logprobs(y.data_ptr(), dt, n, V, ld < V ? V : ld, (const int32_t*)tk.data_ptr(), k, (float)temperature, (float*)lp.data_ptr(), (float*)ent.data_ptr(),
                            (float*)tlp.data_ptr(), (int32_t*)tid.data_ptr(), stream()));
    return {lp, ent, tlp, tid};
}

}  // namespace

TORCH_LIBRARY(wf_native, m) {
    m.def("linear(Tensor x, Tensor w, bool tile, int N, int K, Tensor w_scale) -> Tensor");
    m.def("mlp(Tensor x, Tensor gate_up_tile, int N2, Tensor down_w, float gate_scale, float up_scale, float down_scale, Tensor norm, float eps) -> Tensor");
    m.def("paged_decode_attn(Tensor q, Tensor pool, int max_pages, int layers, int kv_heads, int page_size, int head_dim, int kv_dtype, int layer, Tensor block_table, "
          "Tensor seq_lens, float scale, ScalarType out_dtype) -> Tensor");
    m.def("paged_prefix_attn(Tensor q, Tensor pool, int max_pages, int layers, int kv_heads, int page_size, int head_dim, int kv_dtype, int layer, Tensor prefix_table, "
          "int prefix_len, Tensor block_table, Tensor seq_lens, float scale, ScalarType out_dtype) -> Tensor");
    m.def("paged_plan(Tensor seq_lens, Tensor new_lens, Tensor(a!) block_table, Tensor free_pages, Tensor free_count, int page_size, int max_tokens) -> Tensor[]");
    m.def("paged_release(Tensor done, Tensor seq_lens, Tensor block_table, Tensor(a!) free_pages, Tensor free_count, int page_size) -> (Tensor, Tensor)");
    m.def("token_logprobs(Tensor logits, Tensor tokens, int top, float temperature) -> (Tensor, Tensor, Tensor, Tensor)");
}
// CPU: the same functions, for their errors (a missing GPU, a tensor that is not on it).  Autograd: passed through, so that the outputs are plain tensors
// whatever the inputs require, as behind the calls through ctypes.
#define WF_NATIVE_IMPL(key)                    \
    TORCH_LIBRARY_IMPL(wf_native, key, m) {    \
        m.impl("linear", linear);              \
        m.impl("mlp", mlp);                    \
        m.impl("paged_decode_attn", paged_decode_attn); \
        m.impl("paged_prefix_attn", paged_prefix_attn); \
        m.impl("paged_plan", paged_plan);      \
        m.impl("paged_release", paged_release); \
        m.impl("token_logprobs", token_logprobs); \
    }
WF_NATIVE_IMPL(CUDA)
WF_NATIVE_IMPL(CPU)
TORCH_LIBRARY_IMPL(wf_native, Autograd, m) {
    m.impl("linear", torch::CppFunction::makeFallthrough());
    m.impl("mlp", torch::CppFunction::makeFallthrough());
    m.impl("paged_decode_attn", torch::CppFunction::makeFallthrough());
    m.impl("paged_prefix_attn", torch::CppFunction::makeFallthrough());
    m.impl("paged_plan", torch::CppFunction::makeFallthrough());
    m.impl("paged_release", torch::CppFunction::makeFallthrough());
    m.impl("token_logprobs", torch::CppFunction::makeFallthrough());
}
TORCH_LIBRARY_IMPL(sgl_kernel, CUDA, m) {
    m.impl("bitnet_gemv_cpu", bitnet_gemv);
    m.impl("bitnet_gemv", bitnet_gemv);
    m.impl("bitnet_gemm_cpu", bitnet_gemm);
    m.impl("bitnet_gemm", bitnet_gemm);
    m.impl("bitnet_quantize_activations_cpu", bitnet_quantize_activations);
    m.impl("bitnet_quantize_activations", bitnet_quantize_activations);
}
