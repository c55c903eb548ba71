// torch.Tensor front end of the ring-attention forward.
//
// The reference's include/attention_api.cuh (lines 1-30) includes torch/extension.h and defines CHECK_CUDA /
// CHECK_CONTIGUOUS / CHECK_INPUT but declares no operator; this file is the operator those checks were written
// for.  Every function validates its tensors with CHECK_INPUT, takes the current torch CUDA stream, and calls the
// extern "C" entry points of ring_attention_b200.h.  Nothing is computed here and there is no fallback: a CPU
// tensor or a missing library is an error.  Forward only (the reference has no backward pass).
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>

#include <vector>

#include "../../include/attention_api.cuh"

namespace {

void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
    CHECK_INPUT(q);
    CHECK_INPUT(k);
    CHECK_INPUT(v);
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k, v must be [batch, heads, rows, dim]");
    TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q must be float16 or bfloat16");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k, v must share a dtype");
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
    TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
                "q and k must agree in batch, heads and dim");
    TORCH_CHECK(q.get_device() == k.get_device() && q.get_device() == v.get_device(), "q, k, v must be on one device");
}

void check_status(int status, const char* what) {
    TORCH_CHECK(status == RING_OK, what, " failed (", status, "): ", ring_last_error_string());
}

float default_scale(const at::Tensor& q, double softmax_scale) {
    return softmax_scale > 0.0 ? static_cast<float>(softmax_scale)
                               : 1.0f / std::sqrt(static_cast<float>(q.size(3)));
}

// One Q shard against one K/V shard (the flash inner loop of csrc/ring_attention.cu:536-609 plus :621-664).
std::vector<at::Tensor> block_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double softmax_scale,
                                      bool causal, int64_t q_off, int64_t k_off) {
    check_qkv(q, k, v);
    const c10::cuda::CUDAGuard guard(q.device());
    auto out = at::empty(q.sizes(), q.options().dtype(at::kFloat));
    auto lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    check_status(ring_attention_block_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr<float>(),
                                          lse.data_ptr<float>(), static_cast<int>(q.size(0)), static_cast<int>(q.size(1)),
                                          static_cast<int>(q.size(2)), static_cast<int>(k.size(2)),
                                          static_cast<int>(q.size(3)), default_scale(q, softmax_scale), causal ? 1 : 0,
                                          q_off, k_off, /*merge=*/0, q.scalar_type() == at::kBFloat16 ? 1 : 0,
                                          at::cuda::getCurrentCUDAStream().stream()),
                 "ring_attention_block_fwd");
    return {out, lse};
}

// The ring forward of one rank (set_params_fprop + run_ring_fwd, csrc/ring_attention.cu:361-395, 669-704).
// `ctx` is the address of a RingCtx made by ring_ctx_create / ring_ctx_create_local; `seqlens` holds the rows of
// every rank's shard (the reference's seqlen[], :706).  Asynchronous on the current stream.
std::vector<at::Tensor> ring_forward(int64_t ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                     std::vector<int64_t> seqlens, int64_t mype, double softmax_scale, bool causal) {
    check_qkv(q, k, v);
    TORCH_CHECK(ctx != 0, "ctx must be the address of a ring context");
    const int npes = static_cast<int>(seqlens.size());
    TORCH_CHECK(npes >= 1 && mype >= 0 && mype < npes, "mype must index seqlens");
    TORCH_CHECK(seqlens[mype] == q.size(2) && q.size(2) == k.size(2), "seqlens[mype] must equal the local rows of q and k");
    const c10::cuda::CUDAGuard guard(q.device());
    auto out = at::empty(q.sizes(), q.options().dtype(at::kFloat));
    auto lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    std::vector<int> h_seqlen(seqlens.begin(), seqlens.end());

    Ring_fwd_params params{};
    params.mype = static_cast<int>(mype);
    params.npes = npes;
    params.h_seqlen = h_seqlen.data();
    params.dim = static_cast<int>(q.size(3));
    params.softmax_scale = default_scale(q, softmax_scale);
    params.q_ptr = q.data_ptr();
    params.k_ptr = k.data_ptr();
    params.v_ptr = v.data_ptr();
    params.out_ptr = out.data_ptr<float>();
    params.batch = static_cast<int>(q.size(0));
    params.heads = static_cast<int>(q.size(1));
    params.lse_ptr = lse.data_ptr<float>();
    params.causal = causal ? 1 : 0;
    params.is_bf16 = q.scalar_type() == at::kBFloat16 ? 1 : 0;
    params.stream = at::cuda::getCurrentCUDAStream().stream();
    check_status(ring_attention_fwd(reinterpret_cast<RingCtx*>(ctx), &params), "ring_attention_fwd");
    return {out, lse};
}

// In-place merge of a partial result into the running one (csrc/ring_attention.cu:439-443, 597-598, 621-633).
void lse_merge_(at::Tensor& o_acc, at::Tensor& lse_acc, const at::Tensor& o_part, const at::Tensor& lse_part) {
    CHECK_INPUT(o_acc);
    CHECK_INPUT(lse_acc);
    CHECK_INPUT(o_part);
    CHECK_INPUT(lse_part);
    TORCH_CHECK(o_acc.scalar_type() == at::kFloat && lse_acc.scalar_type() == at::kFloat &&
                    o_part.scalar_type() == at::kFloat && lse_part.scalar_type() == at::kFloat,
                "merge operands must be float32");
    TORCH_CHECK(o_acc.sizes() == o_part.sizes() && lse_acc.sizes() == lse_part.sizes(), "merge operands must agree in shape");
    TORCH_CHECK(o_acc.dim() >= 2 && lse_acc.numel() * o_acc.size(-1) == o_acc.numel(), "lse must have one entry per row of o");
    const c10::cuda::CUDAGuard guard(o_acc.device());
    check_status(ring_lse_merge(o_acc.data_ptr<float>(), lse_acc.data_ptr<float>(), o_part.data_ptr<float>(),
                                lse_part.data_ptr<float>(), lse_acc.numel(), static_cast<int>(o_acc.size(-1)),
                                at::cuda::getCurrentCUDAStream().stream()),
                 "ring_lse_merge");
}

// ---- paged K/V cache ------------------------------------------------------------------------------------------------
// Strides are taken from the tensors; a dimension of one element has no stride that matters (torch leaves any there).
int64_t stride_of(const at::Tensor& x, int64_t d) { return x.size(d) == 1 ? 0 : x.stride(d); }

void check_strided(const at::Tensor& x, const char* what, int64_t dims, at::ScalarType type, const at::Device& device) {
    TORCH_CHECK(x.device().is_cuda(), what, " must be a CUDA tensor");
    TORCH_CHECK(x.dim() == dims, what, " must have ", dims, " dimensions, got ", x.dim());
    TORCH_CHECK(x.scalar_type() == type, what, " has dtype ", x.scalar_type(), ", expected ", type);
    TORCH_CHECK(x.device() == device, what, " is on ", x.device(), ", expected ", device);
    TORCH_CHECK(x.size(dims - 1) <= 1 || x.stride(dims - 1) == 1, "the last dimension of ", what, " must be contiguous");
}

void check_distinct(const at::Tensor& x, const char* what) {
    for (int64_t d = 0; d < x.dim(); ++d)
        TORCH_CHECK(x.size(d) <= 1 || x.stride(d) != 0, what, " is written to and must not be an expanded tensor");
}

int to_int(int64_t x, const char* what) {
    TORCH_CHECK(x >= INT32_MIN && x <= INT32_MAX, what, " does not fit 32 bits");
    return static_cast<int>(x);
}

template <class P>
void fill_cache(P& p, const at::Tensor& k_cache, const at::Tensor* v_cache, const at::Tensor& page_table, const at::Tensor& kv_lens) {
    TORCH_CHECK(k_cache.scalar_type() == at::kHalf || k_cache.scalar_type() == at::kBFloat16, "k_cache must be float16 or bfloat16");
    check_strided(k_cache, "k_cache", 4, k_cache.scalar_type(), k_cache.device());
    p.k_cache = k_cache.data_ptr();
    p.k_page_stride = stride_of(k_cache, 0);
    p.k_head_stride = stride_of(k_cache, 1);
    p.k_place_stride = stride_of(k_cache, 2);
    if (v_cache) {
        check_strided(*v_cache, "v_cache", 4, k_cache.scalar_type(), k_cache.device());
        TORCH_CHECK(v_cache->sizes() == k_cache.sizes(), "k_cache and v_cache must both be [pages, kv_heads, page_size, dim]");
        p.v_cache = v_cache->data_ptr();
        p.v_page_stride = stride_of(*v_cache, 0);
        p.v_head_stride = stride_of(*v_cache, 1);
        p.v_place_stride = stride_of(*v_cache, 2);
    }
    p.num_pages = to_int(k_cache.size(0), "the number of pages");
    p.kv_heads = to_int(k_cache.size(1), "kv_heads");
    p.page_size = to_int(k_cache.size(2), "page_size");
    p.dim = to_int(k_cache.size(3), "dim");
    check_strided(page_table, "page_table", 2, at::kInt, k_cache.device());
    p.page_table = page_table.data_ptr<int>();
    p.table_stride = stride_of(page_table, 0);
    p.batch = to_int(page_table.size(0), "batch");
    p.max_pages = to_int(page_table.size(1), "max_pages");
    check_strided(kv_lens, "kv_lens", 1, at::kInt, k_cache.device());
    TORCH_CHECK(kv_lens.size(0) == p.batch, "kv_lens must have one entry per row of page_table");
    p.kv_lens = kv_lens.data_ptr<int>();
    p.stream = at::cuda::getCurrentCUDAStream(k_cache.get_device()).stream();
}

void fill_tokens(Ring_paged_params& p, int64_t tokens, const c10::optional<at::Tensor>& cu_seqlens, int64_t max_new, const at::Device& device) {
    p.tokens = to_int(tokens, "the number of tokens");
    p.max_new = to_int(max_new, "max_new");
    if (cu_seqlens) {
        check_strided(*cu_seqlens, "cu_seqlens", 1, at::kInt, device);
        TORCH_CHECK(cu_seqlens->size(0) == p.batch + 1, "cu_seqlens must have batch + 1 entries");
        p.cu_seqlens = cu_seqlens->data_ptr<int>();
    }
}

void fill_weights(Ring_paged_params& p, const at::Tensor& weights, const at::Device& device) {
    check_strided(weights, "weights", 3, at::kFloat, device);
    TORCH_CHECK(weights.size(0) == p.batch && weights.size(1) == p.kv_heads, "weights must be [batch, kv_heads, places]");
    check_distinct(weights, "weights");
    p.weights = weights.data_ptr<float>();
    p.weights_batch_stride = stride_of(weights, 0);
    p.weights_head_stride = stride_of(weights, 1);
    p.weights_len = to_int(weights.size(2), "the places of weights");
}

void fill_queries(Ring_paged_params& p, const at::Tensor& q, const at::Tensor& k_cache, const c10::optional<double>& softmax_scale, bool causal,
                  int64_t window, int64_t sinks) {
    check_strided(q, "q", 3, k_cache.scalar_type(), k_cache.device());
    TORCH_CHECK(q.size(2) == p.dim, "q must be [tokens, heads, dim] with the cache's dim");
    p.q = q.data_ptr();
    p.q_token_stride = stride_of(q, 0);
    p.q_head_stride = stride_of(q, 1);
    p.heads = to_int(q.size(1), "heads");
    p.softmax_scale = softmax_scale ? static_cast<float>(*softmax_scale) : 1.0f / std::sqrt(static_cast<float>(p.dim));
    p.causal = causal ? 1 : 0;
    p.window = to_int(window, "window");
    p.sinks = to_int(sinks, "sinks");
    p.is_bf16 = q.scalar_type() == at::kBFloat16 ? 1 : 0;
}

// Scratch from torch's allocator for the current stream: calls that overlap get memory of their own, and nothing is kept.
c10::DataPtr take_workspace(Ring_paged_params& p, int64_t bytes, const char* what) {
    TORCH_CHECK(bytes >= 0, what, " failed (", bytes, "): ", ring_last_error_string());
    if (bytes == 0) return {};
    c10::DataPtr w = c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(bytes));
    p.workspace = w.get();
    p.workspace_bytes = bytes;
    return w;
}

void paged_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
                  const at::Tensor& page_table, const at::Tensor& kv_lens, const c10::optional<at::Tensor>& cu_seqlens,
                  const c10::optional<at::Tensor>& weights) {
    Ring_paged_params p{};
    fill_cache(p, k_cache, &v_cache, page_table, kv_lens);
    check_distinct(k_cache, "k_cache");
    check_distinct(v_cache, "v_cache");
    check_strided(k, "k", 3, k_cache.scalar_type(), k_cache.device());
    check_strided(v, "v", 3, k_cache.scalar_type(), k_cache.device());
    TORCH_CHECK(k.size(1) == p.kv_heads && k.size(2) == p.dim && v.sizes() == k.sizes(), "k and v must both be [tokens, kv_heads, dim]");
    p.k_new = k.data_ptr();
    p.v_new = v.data_ptr();
    p.k_new_token_stride = stride_of(k, 0);
    p.k_new_head_stride = stride_of(k, 1);
    p.v_new_token_stride = stride_of(v, 0);
    p.v_new_head_stride = stride_of(v, 1);
    fill_tokens(p, k.size(0), cu_seqlens, 0, k_cache.device());
    if (weights) fill_weights(p, *weights, k_cache.device());
    const c10::cuda::CUDAGuard guard(k_cache.device());
    check_status(ring_paged_append(&p), "ring_paged_append");
}

std::tuple<at::Tensor, at::Tensor> paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                                   const at::Tensor& page_table, const at::Tensor& kv_lens,
                                                   const c10::optional<at::Tensor>& cu_seqlens, int64_t max_new,
                                        const c10::optional<double>& softmax_scale, bool causal, int64_t window, int64_t sinks, bool fp32_out) {
    Ring_paged_params p{};
    fill_cache(p, k_cache, &v_cache, page_table, kv_lens);
    fill_queries(p, q, k_cache, softmax_scale, causal, window, sinks);
    fill_tokens(p, q.size(0), cu_seqlens, max_new, k_cache.device());
    const c10::cuda::CUDAGuard guard(k_cache.device());
    at::Tensor out(at::detail::empty_cuda(q.sizes(), fp32_out ? at::kFloat : q.scalar_type(), q.device(), c10::nullopt));
    at::Tensor lse(at::detail::empty_cuda({q.size(0), q.size(1)}, at::kFloat, q.device(), c10::nullopt));
    p.out = out.data_ptr();
    p.out_token_stride = out.stride(0);
    p.out_head_stride = out.stride(1);
    p.out_fp32 = fp32_out ? 1 : 0;
    p.lse = lse.data_ptr<float>();
    const c10::DataPtr workspace = take_workspace(p, ring_paged_attention_workspace(&p), "ring_paged_attention_fwd");
    check_status(ring_paged_attention_fwd(&p), "ring_paged_attention_fwd");
    return {out, lse};
}

void paged_weights_(const at::Tensor& weights, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& lse,
                    const at::Tensor& page_table, const at::Tensor& kv_lens, const c10::optional<at::Tensor>& cu_seqlens, int64_t max_new,
                    const c10::optional<double>& softmax_scale, bool causal, int64_t window, int64_t sinks) {
    Ring_paged_params p{};
    fill_cache(p, k_cache, nullptr, page_table, kv_lens);
    fill_queries(p, q, k_cache, softmax_scale, causal, window, sinks);
    fill_tokens(p, q.size(0), cu_seqlens, max_new, k_cache.device());
    fill_weights(p, weights, k_cache.device());
    check_strided(lse, "lse", 2, at::kFloat, k_cache.device());
    TORCH_CHECK(lse.is_contiguous() && lse.size(0) == q.size(0) && lse.size(1) == q.size(1), "lse must be a contiguous [tokens, heads]");
    p.lse = lse.data_ptr<float>();
    const c10::cuda::CUDAGuard guard(k_cache.device());
    const c10::DataPtr workspace = take_workspace(p, ring_paged_weights_workspace(&p), "ring_paged_weights");
    check_status(ring_paged_weights(&p), "ring_paged_weights");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> paged_evict(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& weights,
                                    const at::Tensor& page_table, const at::Tensor& kv_lens, const at::Tensor& dst_table, int64_t budget,
                                    int64_t first, int64_t recent) {
    Ring_evict_params p{};
    fill_cache(p, k_cache, &v_cache, page_table, kv_lens);
    check_distinct(k_cache, "k_cache");
    check_distinct(v_cache, "v_cache");
    check_strided(weights, "weights", 3, at::kFloat, k_cache.device());
    TORCH_CHECK(weights.size(0) == p.batch && weights.size(1) == p.kv_heads, "weights must be [batch, kv_heads, places]");
    p.weights = weights.data_ptr<float>();
    p.weights_batch_stride = stride_of(weights, 0);
    p.weights_head_stride = stride_of(weights, 1);
    p.weights_len = to_int(weights.size(2), "the places of weights");
    check_strided(dst_table, "dst_table", 2, at::kInt, k_cache.device());
    TORCH_CHECK(dst_table.size(0) == p.batch, "dst_table must have one row per row of page_table");
    p.dst_table = dst_table.data_ptr<int>();
    p.dst_stride = stride_of(dst_table, 0);
    p.dst_pages = to_int(dst_table.size(1), "the pages of dst_table");
    p.budget = to_int(budget, "budget");
    p.first = to_int(first, "first");
    p.recent = to_int(recent, "recent");
    const int64_t places = dst_table.size(1) * p.page_size;
    TORCH_CHECK(budget >= 1 && budget <= places, "budget must be positive and fit the pages of dst_table (", places, " places), got ", budget);
    const c10::cuda::CUDAGuard guard(k_cache.device());
    at::Tensor new_lens(at::detail::empty_cuda({p.batch}, at::kInt, k_cache.device(), c10::nullopt));
    at::Tensor new_weights(at::detail::empty_cuda({p.batch, p.kv_heads, places}, at::kFloat, k_cache.device(), c10::nullopt));
    at::Tensor kept(at::detail::empty_cuda({p.batch, p.kv_heads, budget}, at::kInt, k_cache.device(), c10::nullopt));
    p.new_lens = new_lens.data_ptr<int>();
    p.new_weights = new_weights.data_ptr<float>();
    p.new_weights_batch_stride = new_weights.stride(0);
    p.new_weights_head_stride = new_weights.stride(1);
    p.new_weights_len = to_int(places, "the places of dst_table");
    p.kept = kept.data_ptr<int>();
    check_status(ring_paged_evict(&p), "ring_paged_evict");
    return {new_lens, new_weights, kept};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "torch.Tensor front end of the B200 ring-attention forward";
    m.def("block_forward", &block_forward, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("softmax_scale") = 0.0,
          py::arg("causal") = false, py::arg("q_off") = 0, py::arg("k_off") = 0,
          "Attention of one Q shard against one K/V shard: returns (out fp32, lse fp32)");
    m.def("ring_forward", &ring_forward, py::arg("ctx"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("seqlens"),
          py::arg("mype"), py::arg("softmax_scale") = 0.0, py::arg("causal") = false,
          "Ring-attention forward of rank mype: returns (out fp32, lse fp32)");
    m.def("lse_merge_", &lse_merge_, "Merge (o_part, lse_part) into (o_acc, lse_acc) in place");
    m.def("paged_append", &paged_append, "Write new K and V rows to their places in the pages");
    m.def("paged_attention", &paged_attention, "Attention of new tokens over the paged cache: returns (out, lse)");
    m.def("paged_weights_", &paged_weights_, "Add the new tokens' attention to the weights of the cached places");
    m.def("paged_evict", &paged_evict, "Keep the heaviest places: returns (new_lens, new_weights, kept)");
}
