// Host side of the paged-cache operators: argument checks, kernel choice, launches (see ring_attention_b200.h).
//
// Nothing here allocates (beyond the library's one-time per-device set-up), waits for the GPU or keeps state between calls.
#include <cmath>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/ring_attention_b200.h"
#include "host_common.h"
#include "kernel_traits.h"
#include "paged_cache.cuh"
#include "paged_chunk.cuh"
#include "paged_plan.cuh"
#include "paged_rows.cuh"
#include "paged_weights.cuh"

using namespace ring_host;

namespace {

constexpr int64_t kMaxInt = 0x7fffffff;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

#define PAGED_REQUIRE(cond, ...) \
    do {                         \
        if (!(cond)) return fail(RING_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
    } while (0)

template <class P>
int check_cache(const P& p) {
    PAGED_REQUIRE(p.dim == 64 || p.dim == 128, "dim must be 64 or 128, got %d", p.dim);
    PAGED_REQUIRE(p.page_size >= 8 && (p.page_size & (p.page_size - 1)) == 0, "page_size must be a power of two >= 8, got %d", p.page_size);
    PAGED_REQUIRE(p.num_pages >= 1 && p.kv_heads >= 1, "num_pages and kv_heads must be positive");
    PAGED_REQUIRE(p.max_pages >= 1 && static_cast<int64_t>(p.max_pages) * p.page_size <= (int64_t(1) << 30),
                  "max_pages must be positive and max_pages * page_size at most 2^30");
    PAGED_REQUIRE(p.batch >= 1 && p.batch <= 65535, "batch must be in [1, 65535], got %d", p.batch);
    PAGED_REQUIRE(static_cast<int64_t>(p.batch) * p.kv_heads <= 65535, "batch * kv_heads must not exceed 65535");
    PAGED_REQUIRE(p.page_table && p.kv_lens, "null page_table or kv_lens");
    PAGED_REQUIRE(p.table_stride >= p.max_pages || p.batch == 1, "table_stride is smaller than max_pages");
    PAGED_REQUIRE(p.k_cache, "null k_cache");
    PAGED_REQUIRE(aligned16(p.k_cache) && aligned16(p.v_cache), "cache base pointers must be 16-byte aligned");
    const int64_t st = p.k_page_stride | p.k_head_stride | p.k_place_stride | p.v_page_stride | p.v_head_stride | p.v_place_stride;
    PAGED_REQUIRE((st & 7) == 0, "cache strides must be multiples of 8 elements");
    PAGED_REQUIRE(p.k_page_stride >= 0 && p.k_head_stride >= 0 && p.k_place_stride >= 0 && p.v_page_stride >= 0 &&
                      p.v_head_stride >= 0 && p.v_place_stride >= 0, "cache strides must not be negative");
    // rows of an expanded tensor are one memory: written twice by append, and not a tensor map's either
    PAGED_REQUIRE((p.num_pages == 1 || (p.k_page_stride && (!p.v_cache || p.v_page_stride))) &&
                      (p.kv_heads == 1 || (p.k_head_stride && (!p.v_cache || p.v_head_stride))) && p.k_place_stride &&
                      (!p.v_cache || p.v_place_stride), "cache strides of 0 (an expanded tensor) are not supported");
    return RING_OK;
}

template <class P>
void cache_args(const P& p, ring::PagedArgs* a) {
    *a = ring::PagedArgs{};
    a->k = p.k_cache;
    a->v = p.v_cache;
    a->k_page = p.k_page_stride;
    a->k_head = p.k_head_stride;
    a->k_place = p.k_place_stride;
    a->v_page = p.v_page_stride;
    a->v_head = p.v_head_stride;
    a->v_place = p.v_place_stride;
    a->num_pages = p.num_pages;
    a->page_shift = __builtin_ctz(static_cast<unsigned>(p.page_size));
    a->kv_heads = p.kv_heads;
    a->table = p.page_table;
    a->table_stride = p.table_stride;
    a->max_pages = p.max_pages;
    a->capacity = p.max_pages * p.page_size;
    a->batch = p.batch;
    a->lens = p.kv_lens;
}

int check_tokens(const Ring_paged_params& p) {
    PAGED_REQUIRE(p.tokens >= 0 && p.max_new >= 0, "tokens and max_new must not be negative");
    PAGED_REQUIRE(p.cu_seqlens || p.tokens % p.batch == 0, "without cu_seqlens tokens must be a multiple of batch (%d of %d)", p.tokens, p.batch);
    return RING_OK;
}

int check_weights(const Ring_paged_params& p) {
    PAGED_REQUIRE(p.weights_len >= static_cast<int64_t>(p.max_pages) * p.page_size, "weights_len must be at least max_pages * page_size");
    PAGED_REQUIRE(p.weights_batch_stride >= 0 && p.weights_head_stride >= 0, "weights strides must not be negative");
    // rows are added to without atomics: two of them in one memory would lose sums
    const int64_t places = static_cast<int64_t>(p.max_pages) * p.page_size;
    PAGED_REQUIRE((p.batch == 1 || p.weights_batch_stride >= places) && (p.kv_heads == 1 || p.weights_head_stride >= places),
                  "rows of weights overlap");
    return RING_OK;
}

// Sizes of a query operand; `pointers` = false leaves the addresses out (the workspace question).
int check_queries(const Ring_paged_params& p, bool pointers) {
    int rc = check_tokens(p);
    if (rc) return rc;
    PAGED_REQUIRE(p.heads >= 1 && p.heads % p.kv_heads == 0, "heads (%d) must be a positive multiple of kv_heads (%d)", p.heads, p.kv_heads);
    PAGED_REQUIRE(static_cast<int64_t>(p.tokens) * p.heads <= kMaxInt - 1024, "tokens * heads must stay below 2^31");
    PAGED_REQUIRE(p.softmax_scale > 0.f && std::isfinite(p.softmax_scale), "softmax_scale must be positive and finite");
    PAGED_REQUIRE(p.window >= 0 && p.sinks >= 0, "window and sinks must not be negative");
    PAGED_REQUIRE(p.causal || p.window == 0, "a window needs causal = 1");
    if (pointers && p.tokens > 0) {
        PAGED_REQUIRE(p.q && p.lse, "null q or lse");
        PAGED_REQUIRE(aligned16(p.q), "q must be 16-byte aligned");
        PAGED_REQUIRE(((p.q_token_stride | p.q_head_stride) & 7) == 0 && p.q_token_stride >= 0 && p.q_head_stride >= 0,
                      "q strides must be non-negative multiples of 8 elements");
        PAGED_REQUIRE((p.tokens == 1 || p.q_token_stride) && (p.heads == 1 || p.q_head_stride), "q strides of 0 (an expanded tensor) are not supported");
    }
    return RING_OK;
}

// x / d = (umulhi(x, mul) + x) >> shift for 0 <= x < 2^31: mul = floor(2^32 (2^shift - d) / d) + 1 with 2^shift >= d the least such.
void quotient_of(int d, uint32_t* mul, uint32_t* shift) {
    *shift = 0;
    while ((uint64_t(1) << *shift) < static_cast<uint64_t>(d)) ++*shift;
    *mul = static_cast<uint32_t>((uint64_t(1) << 32) * ((uint64_t(1) << *shift) - d) / d + 1);
}

void query_args(const Ring_paged_params& p, ring::PagedArgs* a) {
    cache_args(p, a);
    a->cu = p.cu_seqlens;
    a->uniform_new = p.cu_seqlens ? 0 : p.tokens / p.batch;
    a->tokens = p.tokens;
    a->q = p.q;
    a->q_token = p.q_token_stride;
    a->q_head = p.q_head_stride;
    a->heads = p.heads;
    a->group = p.kv_heads ? p.heads / p.kv_heads : 0;
    if (a->group) quotient_of(a->group, &a->group_mul, &a->group_shift);
    a->out_fp32 = p.out_fp32;
    a->out = p.out;
    a->out_token = p.out_token_stride;
    a->out_head = p.out_head_stride;
    a->lse = p.lse;
    a->scale = p.softmax_scale;
    a->scale_log2 = p.softmax_scale * 1.4426950408889634f;
    a->causal = p.causal ? 1 : 0;
    a->window = p.window < (1 << 30) ? p.window : 1 << 30;  // no sequence is longer: the same mask, and no sum overflows
    a->sinks = p.sinks < (1 << 30) ? p.sinks : 1 << 30;
    a->weights = p.weights;
    a->w_batch = p.weights_batch_stride;
    a->w_head = p.weights_head_stride;
}

int max_new_of(const Ring_paged_params& p) {
    if (!p.cu_seqlens) return p.tokens / p.batch;
    return p.max_new > 0 && p.max_new < p.tokens ? p.max_new : p.tokens;
}

template <class Kernel>
int set_smem(Kernel kernel, int bytes, bool* done) {
    std::lock_guard<std::mutex> lock(g_dev_mutex);
    if (!*done) {
        RING_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        *done = true;
    }
    return RING_OK;
}

// Every kernel here is launched so that its CTAs may be set up while the kernel before it in the stream still runs; each waits
// (griddepcontrol.wait) for that kernel's end and its memory before it reads or writes anything.
template <class... Params, class... Args>
int launch(void (*kernel)(Params...), dim3 grid, dim3 block, int smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    RING_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return RING_OK;
}

int check_workspace(const Ring_paged_params& p, int64_t need) {
    PAGED_REQUIRE(p.workspace && (reinterpret_cast<uintptr_t>(p.workspace) & 255) == 0, "workspace must be 256-byte aligned and not null");
    PAGED_REQUIRE(p.workspace_bytes >= need, "workspace holds %lld bytes, %lld are needed", (long long)p.workspace_bytes, (long long)need);
    return RING_OK;
}

// ---- attention -----------------------------------------------------------------------------------------------------
struct AttentionPlan {
    int unit_rows;
    int rows;  // rows a unit of the few-rows kernel is expected to have
    int grid;
    int64_t o_bytes, lse_bytes, cut_bytes;
    int64_t bytes() const { return o_bytes + lse_bytes + cut_bytes; }
};

int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

// Which kernel, by the query rows per K/V head (new tokens x group).  Microseconds for 16 sequences of 8192 places, 8 K/V heads,
// bf16, pages of 64 (16-row units / 32-row units of the few-rows kernel / the 256-row tcgen05 kernel):
//   D = 128   16 rows 101 / 123 / 104    24 rows 179 / 128 / 106    32 rows 181 / 131 / 107    64 rows 340 / 248 / 110
//   D = 64    16 rows  53 /  56 /  99    24 rows  75 /  58 / 100    32 rows  76 /  59 / 100    64 rows 173 / 100 / 100
// At D = 128 the 32-row units spill, so there the tcgen05 kernel takes over at 17 rows, at D = 64 at 33.
AttentionPlan attention_plan(const Ring_paged_params& p, int sm_count) {
    AttentionPlan r;
    const int64_t rows = static_cast<int64_t>(max_new_of(p)) * (p.heads / p.kv_heads);
    r.unit_rows = rows <= 16 ? 16 : (rows <= 32 && p.dim == 64 ? 32 : 256);
    r.rows = static_cast<int>(rows < 1 ? 1 : (rows < r.unit_rows ? rows : r.unit_rows));
    r.grid = r.unit_rows <= 32 ? 2 * sm_count : sm_count;  // two CTAs of the few-rows kernel fit an SM, one of the other
    r.o_bytes = round256(int64_t(2) * r.grid * r.unit_rows * p.dim * 4);
    r.lse_bytes = round256(int64_t(2) * r.grid * r.unit_rows * 4);
    r.cut_bytes = round256(int64_t(r.grid) * 32);
    return r;
}

template <int D, bool kBf16, int MT>
int launch_rows(const ring::PagedArgs& a, const AttentionPlan& plan, DeviceState* st, cudaStream_t stream) {
    using T = ring::PagedRowsTraits<D, kBf16, MT>;
    auto kernel = &ring::ring_paged_rows_kernel<T>;
    int rc = set_smem(kernel, T::kSmem, &st->paged_attr_set[(MT - 1) * 4 + (D == 128) * 2 + kBf16]);
    if (rc) return rc;
    if ((rc = launch(kernel, dim3(plan.grid), dim3(T::kThreads), T::kSmem, stream, a))) return rc;
    return launch(&ring::ring_paged_join_kernel<D, kBf16, 4>, dim3(plan.grid, plan.rows < 8 ? plan.rows : 8), dim3(128), 0, stream, a, plan.unit_rows);
}

// The cache as a 4-D map [pages, kv_heads, page_size, dim]: a box is 64 columns of min(page_size, 128) places of one page and head,
// 128-byte swizzle.  Page num_pages reads as zeros.
int cache_map(CUtensorMap* tm, const ring::PagedArgs& a, const void* base, int64_t page, int64_t head, int64_t place, int dim, bool bf16) {
    EncodeTiledFn enc = nullptr;
    int rc = encode_fn(&enc);
    if (rc) return rc;
    const int page_size = 1 << a.page_shift;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(page_size), static_cast<cuuint64_t>(a.kv_heads),
                                static_cast<cuuint64_t>(a.num_pages)};
    // a dimension of one element may come with any stride
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(place) * 2, static_cast<cuuint64_t>(a.kv_heads == 1 ? dim : head) * 2,
                                   static_cast<cuuint64_t>(a.num_pages == 1 ? dim : page) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(page_size < 128 ? page_size : 128), 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims,
                           strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RING_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return RING_OK;
}

template <int D, bool kBf16, bool kWindow>
int launch_chunk(const ring::PagedArgs& a, const AttentionPlan& plan, DeviceState* st, cudaStream_t stream) {
    using T = Ring_fwd_traits<D, 256, 128, 12, typename std::conditional<kBf16, __nv_bfloat16, __half>::type>;
    auto kernel = &ring::ring_paged_chunk_kernel<T, kWindow>;
    int rc = set_smem(kernel, T::kSmemSize, &st->paged_attr_set[8 + kWindow * 20 + (D == 128) * 2 + kBf16]);
    if (rc) return rc;
    CUtensorMap tk, tv;
    if ((rc = cache_map(&tk, a, a.k, a.k_page, a.k_head, a.k_place, D, kBf16))) return rc;
    if ((rc = cache_map(&tv, a, a.v, a.v_page, a.v_head, a.v_place, D, kBf16))) return rc;
    if ((rc = launch(kernel, dim3(plan.grid), dim3(T::kNThreads), T::kSmemSize, stream, tk, tv, a))) return rc;
    return launch(&ring::ring_paged_join_kernel<D, kBf16, 1>, dim3(plan.grid, 16), dim3(128), 0, stream, a, plan.unit_rows);
}

template <int D, bool kBf16>
int launch_attention(const ring::PagedArgs& a, const AttentionPlan& plan, DeviceState* st, cudaStream_t stream) {
    if (plan.unit_rows == 256)
        return a.window > 0 ? launch_chunk<D, kBf16, true>(a, plan, st, stream) : launch_chunk<D, kBf16, false>(a, plan, st, stream);
    if constexpr (D == 64) {
        if (plan.unit_rows == 32) return launch_rows<D, kBf16, 2>(a, plan, st, stream);
    }
    return launch_rows<D, kBf16, 1>(a, plan, st, stream);
}

// ---- weights -------------------------------------------------------------------------------------------------------
struct WeightsPlan {
    bool chunk;      // many query rows: the tcgen05 form
    int row_tiles;   // rows form: tiles of 8 query rows held in registers
    int grid;
    int64_t part_bytes, cut_bytes;
    int64_t bytes() const { return part_bytes + cut_bytes; }
};

// Which form, by the query rows per K/V head.  Microseconds for 16 sequences of 8192 places, 8 K/V heads, bf16 (rows form holding 8 / 16 /
// 32 rows in registers, chunk form):
//   D = 128    8 rows 59 / 66 / 77 / 135    16 rows 97 / 67 / 77 / 136    24 rows 124 / 133 / 78 / 136    32 rows 151 / 141 / 79 / 136
//             40 rows 178 / 181 / 190 / 136    64 rows 262 / 239 / 211 / 136
//   D = 64     8 rows 38 / 45 / 58 / 133    16 rows 54 / 45 / 58 / 133    24 rows 67 / 72 / 58 / 133    32 rows 80 / 73 / 58 / 133
//             40 rows 94 / 95 / 111 / 133    64 rows 135 / 120 / 116 / 133
// One rule for both, although at D = 64 the rows forms stay ahead to about 64 rows.
WeightsPlan weights_plan(const Ring_paged_params& p, int sm_count) {
    WeightsPlan r;
    const int64_t group = p.heads / p.kv_heads, rows = max_new_of(p) * group;
    r.chunk = rows > 32 && group <= 128;  // a query tile of the chunk form holds whole tokens of at most 128 heads
    r.row_tiles = rows <= 8 ? 1 : (rows <= 16 ? 2 : 4);
    r.grid = r.chunk ? sm_count : 2 * sm_count;
    r.part_bytes = r.chunk ? round256(int64_t(2) * r.grid * 256 * 4) : 0;
    r.cut_bytes = r.chunk ? round256(int64_t(r.grid) * 32) : 0;
    return r;
}

template <int D, bool kBf16, int NT>
int launch_weights_rows(const ring::PagedArgs& a, const WeightsPlan& plan, DeviceState* st, cudaStream_t stream) {
    using T = ring::PagedWeightsRowsTraits<D, kBf16, NT>;
    auto kernel = &ring::ring_paged_weights_rows_kernel<T>;
    int rc = set_smem(kernel, T::kSmem, &st->paged_attr_set[16 + (NT >> 1) * 4 + (D == 128) * 2 + kBf16]);
    if (rc) return rc;
    return launch(kernel, dim3(plan.grid), dim3(T::kThreads), T::kSmem, stream, a);
}

// The queries as a 4-D map [tokens, kv_heads, group, dim]: a box is 64 columns of all heads of a group for `row_tokens` tokens.
int query_map(CUtensorMap* tm, const ring::PagedArgs& a, int dim, bool bf16) {
    EncodeTiledFn enc = nullptr;
    int rc = encode_fn(&enc);
    if (rc) return rc;
    const int64_t head = a.heads == 1 ? dim : a.q_head, token = a.tokens == 1 ? dim : a.q_token;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(a.group), static_cast<cuuint64_t>(a.kv_heads),
                                static_cast<cuuint64_t>(a.tokens)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(head) * 2, static_cast<cuuint64_t>(head) * a.group * 2, static_cast<cuuint64_t>(token) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(a.group), 1, static_cast<cuuint32_t>(a.row_tokens)};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(a.q), dims,
                           strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RING_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return RING_OK;
}

template <int D, bool kBf16>
int launch_weights(const ring::PagedArgs& a, const WeightsPlan& plan, DeviceState* st, cudaStream_t stream) {
    if (!plan.chunk) {
        if (plan.row_tiles == 1) return launch_weights_rows<D, kBf16, 1>(a, plan, st, stream);
        if (plan.row_tiles == 2) return launch_weights_rows<D, kBf16, 2>(a, plan, st, stream);
        return launch_weights_rows<D, kBf16, 4>(a, plan, st, stream);
    }
    using T = ring::PagedWeightsTraits<D, typename std::conditional<kBf16, __nv_bfloat16, __half>::type>;
    auto kernel = &ring::ring_paged_weights_chunk_kernel<T>;
    int rc = set_smem(kernel, T::kSmemSize, &st->paged_attr_set[12 + (D == 128) * 2 + kBf16]);
    if (rc) return rc;
    CUtensorMap tk, tq;
    if ((rc = cache_map(&tk, a, a.k, a.k_page, a.k_head, a.k_place, D, kBf16))) return rc;
    if ((rc = query_map(&tq, a, D, kBf16))) return rc;
    if ((rc = launch(kernel, dim3(plan.grid), dim3(T::kNThreads), T::kSmemSize, stream, tk, tq, a))) return rc;
    return launch(&ring::ring_paged_weights_join_kernel, dim3(plan.grid), dim3(256), 0, stream, a);
}

// What the workspace questions look at.
int check_sizes(const Ring_paged_params* params, DeviceState** st) {
    if (!params) return fail(RING_ERR_INVALID_ARGUMENT, "null params");
    PAGED_REQUIRE(params->dim == 64 || params->dim == 128, "dim must be 64 or 128, got %d", params->dim);
    PAGED_REQUIRE(params->batch >= 1 && params->kv_heads >= 1, "batch and kv_heads must be positive");
    const int rc = check_queries(*params, false);
    return rc ? rc : device_state(st);
}

}  // namespace

extern "C" {

int ring_paged_append(const Ring_paged_params* params) {
    if (!params) return fail(RING_ERR_INVALID_ARGUMENT, "null params");
    const Ring_paged_params& p = *params;
    int rc;
    if ((rc = check_cache(p)) || (rc = check_tokens(p))) return rc;
    if (p.weights && (rc = check_weights(p))) return rc;
    if (p.tokens == 0) return RING_OK;
    PAGED_REQUIRE(p.v_cache, "null v_cache");
    PAGED_REQUIRE(p.k_new && p.v_new, "null k_new or v_new");
    PAGED_REQUIRE(aligned16(p.k_new) && aligned16(p.v_new), "k_new and v_new must be 16-byte aligned");
    PAGED_REQUIRE(((p.k_new_token_stride | p.k_new_head_stride | p.v_new_token_stride | p.v_new_head_stride) & 7) == 0 &&
                      p.k_new_token_stride >= 0 && p.k_new_head_stride >= 0 && p.v_new_token_stride >= 0 && p.v_new_head_stride >= 0,
                  "k_new and v_new strides must be non-negative multiples of 8 elements");
    ring::PagedAppendArgs args;
    cache_args(p, &args.a);
    args.a.cu = p.cu_seqlens;
    args.a.uniform_new = p.cu_seqlens ? 0 : p.tokens / p.batch;
    args.a.tokens = p.tokens;
    args.a.weights = p.weights;
    args.a.w_batch = p.weights_batch_stride;
    args.a.w_head = p.weights_head_stride;
    args.k_new = p.k_new;
    args.v_new = p.v_new;
    args.k_token = p.k_new_token_stride;
    args.k_head = p.k_new_head_stride;
    args.v_token = p.v_new_token_stride;
    args.v_head = p.v_new_head_stride;
    // one pass of the unrolled loop covers 4 * (256 / dim) heads: a warp per pass while there are few tokens
    const int per_pass = 4 * 256 / p.dim;
    args.head_parts = (p.kv_heads + per_pass - 1) / per_pass;
    const int64_t warps = static_cast<int64_t>(p.tokens) * args.head_parts;
    PAGED_REQUIRE((warps + 7) / 8 <= kMaxInt, "too many tokens");
    const int blocks = static_cast<int>((warps + 7) / 8);
    cudaStream_t stream = static_cast<cudaStream_t>(p.stream);
    return launch(p.dim == 128 ? &ring::ring_paged_append_kernel<128> : &ring::ring_paged_append_kernel<64>, dim3(blocks), dim3(256), 0,
                  stream, args);
}

int64_t ring_paged_attention_workspace(const Ring_paged_params* params) {
    DeviceState* st = nullptr;
    const int rc = check_sizes(params, &st);
    return rc ? rc : attention_plan(*params, st->sm_count).bytes();
}

int64_t ring_paged_weights_workspace(const Ring_paged_params* params) {
    DeviceState* st = nullptr;
    const int rc = check_sizes(params, &st);
    return rc ? rc : weights_plan(*params, st->sm_count).bytes();
}

int ring_paged_attention_fwd(const Ring_paged_params* params) {
    if (!params) return fail(RING_ERR_INVALID_ARGUMENT, "null params");
    const Ring_paged_params& p = *params;
    int rc;
    if ((rc = check_cache(p)) || (rc = check_queries(p, true))) return rc;
    if (p.tokens == 0) return RING_OK;
    PAGED_REQUIRE(p.v_cache && p.out, "null v_cache or out");
    PAGED_REQUIRE(aligned16(p.out), "out must be 16-byte aligned");
    const int out_unit = p.out_fp32 ? 3 : 7;
    PAGED_REQUIRE(((p.out_token_stride | p.out_head_stride) & out_unit) == 0 && p.out_token_stride >= 0 && p.out_head_stride >= 0,
                  "out strides must be non-negative multiples of 16 bytes");
    PAGED_REQUIRE((p.tokens == 1 || p.out_token_stride >= p.dim) && (p.heads == 1 || p.out_head_stride >= p.dim), "rows of out overlap");
    DeviceState* st = nullptr;
    if ((rc = device_state(&st))) return rc;
    const AttentionPlan plan = attention_plan(p, st->sm_count);
    if ((rc = check_workspace(p, plan.bytes()))) return rc;
    ring::PagedArgs a;
    query_args(p, &a);
    char* ws = static_cast<char*>(p.workspace);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_lse = reinterpret_cast<float*>(ws + plan.o_bytes);
    a.cut = reinterpret_cast<int4*>(ws + plan.o_bytes + plan.lse_bytes);
    a.unit_rows = plan.unit_rows;
    a.unit_shift = __builtin_ctz(static_cast<unsigned>(plan.unit_rows));
    a.many_tiles = (static_cast<int64_t>(max_new_of(p)) * a.group + plan.unit_rows - 1) / plan.unit_rows > 4;
    // in blocks: about 7 thousand clocks of lookups, first loads and write-out against 3 thousand a block of 256 rows, and 3 thousand
    // against 1.4 thousand of the few-rows kernel
    a.start_cost = plan.unit_rows == 256 ? 4 : 2;
    a.min_blocks = a.start_cost + (plan.unit_rows == 256 ? 2 : 1);
    a.status = plan.unit_rows == 256 ? st->d_status : nullptr;
    cudaStream_t stream = static_cast<cudaStream_t>(p.stream);
    if (p.dim == 128)
        return p.is_bf16 ? launch_attention<128, true>(a, plan, st, stream) : launch_attention<128, false>(a, plan, st, stream);
    return p.is_bf16 ? launch_attention<64, true>(a, plan, st, stream) : launch_attention<64, false>(a, plan, st, stream);
}

int ring_paged_weights(const Ring_paged_params* params) {
    if (!params) return fail(RING_ERR_INVALID_ARGUMENT, "null params");
    const Ring_paged_params& p = *params;
    int rc;
    if ((rc = check_cache(p)) || (rc = check_queries(p, true)) || (rc = check_weights(p))) return rc;
    if (p.tokens == 0) return RING_OK;
    PAGED_REQUIRE(p.weights, "null weights");
    DeviceState* st = nullptr;
    if ((rc = device_state(&st))) return rc;
    ring::PagedArgs a;
    query_args(p, &a);
    const WeightsPlan plan = weights_plan(p, st->sm_count);
    if (plan.bytes() > 0) {
        if ((rc = check_workspace(p, plan.bytes()))) return rc;
        a.part_lse = static_cast<float*>(p.workspace);
        a.cut = reinterpret_cast<int4*>(static_cast<char*>(p.workspace) + plan.part_bytes);
    }
    a.status = st->d_status;
    if (plan.chunk) {
        a.row_tokens = 128 / a.group;
        quotient_of(a.row_tokens, &a.tokens_mul, &a.tokens_shift);
    }
    a.unit_rows = 1 << 30;  // one unit holds all rows of its sequence
    a.unit_shift = 30;
    a.many_tiles = plan.chunk;
    // in blocks, from one case of each form: 1024 tokens over 8192 places 102.4 / 99.2 / 98.7 us with 1 / 2 / 3, 16 single tokens (rows
    // form) 36.1 / 36.8 / 37.6
    a.start_cost = plan.chunk ? 3 : 1;
    a.min_blocks = a.start_cost + 1;
    cudaStream_t stream = static_cast<cudaStream_t>(p.stream);
    if (p.dim == 128) return p.is_bf16 ? launch_weights<128, true>(a, plan, st, stream) : launch_weights<128, false>(a, plan, st, stream);
    return p.is_bf16 ? launch_weights<64, true>(a, plan, st, stream) : launch_weights<64, false>(a, plan, st, stream);
}

int ring_paged_evict(const Ring_evict_params* params) {
    if (!params) return fail(RING_ERR_INVALID_ARGUMENT, "null params");
    const Ring_evict_params& p = *params;
    int rc;
    if ((rc = check_cache(p))) return rc;
    PAGED_REQUIRE(p.v_cache, "null v_cache");
    PAGED_REQUIRE(p.budget >= 1 && p.first >= 0 && p.recent >= 0 && static_cast<int64_t>(p.first) + p.recent <= p.budget,
                  "budget must be positive and first + recent at most budget (budget %d, first %d, recent %d)", p.budget, p.first, p.recent);
    PAGED_REQUIRE(p.dst_table && p.dst_pages >= 1 && static_cast<int64_t>(p.dst_pages) * p.page_size >= p.budget,
                  "dst_table must name pages for %d places", p.budget);
    PAGED_REQUIRE(p.dst_stride >= p.dst_pages || p.batch == 1, "dst_stride is smaller than dst_pages");
    PAGED_REQUIRE(p.dst_table != p.page_table, "dst_table must name pages of its own, not the source's");
    PAGED_REQUIRE(p.weights && p.new_weights && p.kept && p.new_lens, "null weights, new_weights, kept or new_lens");
    PAGED_REQUIRE(p.weights != p.new_weights, "new_weights must not be weights");
    PAGED_REQUIRE(p.new_lens != p.kv_lens, "new_lens must not be kv_lens");
    PAGED_REQUIRE(p.weights_len >= static_cast<int64_t>(p.max_pages) * p.page_size, "weights_len must be at least max_pages * page_size");
    PAGED_REQUIRE(p.new_weights_len >= p.budget, "new_weights_len must be at least budget");
    // loops over these step past their end by up to a block: far from where 32 bits turn over
    PAGED_REQUIRE(p.new_weights_len <= (1 << 30) && p.budget <= (1 << 30), "budget and new_weights_len must not exceed 2^30");
    PAGED_REQUIRE(p.weights_batch_stride >= 0 && p.weights_head_stride >= 0 && p.new_weights_batch_stride >= 0 &&
                      p.new_weights_head_stride >= 0, "weights strides must not be negative");
    PAGED_REQUIRE((p.batch == 1 || p.new_weights_batch_stride >= p.new_weights_len) &&
                      (p.kv_heads == 1 || p.new_weights_head_stride >= p.new_weights_len), "rows of new_weights overlap");
    ring::PagedEvictArgs e;
    cache_args(p, &e.a);
    e.a.weights = const_cast<float*>(p.weights);
    e.a.w_batch = p.weights_batch_stride;
    e.a.w_head = p.weights_head_stride;
    e.dst_table = p.dst_table;
    e.dst_stride = p.dst_stride;
    e.dst_pages = p.dst_pages;
    e.budget = p.budget;
    e.first = p.first;
    e.recent = p.recent;
    e.new_weights = p.new_weights;
    e.nw_batch = p.new_weights_batch_stride;
    e.nw_head = p.new_weights_head_stride;
    e.nw_len = p.new_weights_len;
    e.kept = p.kept;
    e.new_lens = p.new_lens;
    cudaStream_t stream = static_cast<cudaStream_t>(p.stream);
    if ((rc = launch(&ring::ring_paged_select_kernel, dim3(p.batch * p.kv_heads), dim3(ring::kSelectThreads), 0, stream, e))) return rc;
    const int per_block = 8 * 4 * (p.dim == 128 ? 1 : 2);
    const dim3 grid((p.budget + per_block - 1) / per_block, p.batch * p.kv_heads);
    if (p.dim == 128) return launch(&ring::ring_paged_gather_kernel<128>, grid, dim3(256), 0, stream, e);
    return launch(&ring::ring_paged_gather_kernel<64>, grid, dim3(256), 0, stream, e);
}

}  // extern "C"
