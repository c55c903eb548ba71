// Paged-cache kernels that move rows: append and eviction.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "paged_plan.cuh"
#include "paged_rows.cuh"
#include "ptx_sm100.cuh"

namespace ring {

struct PagedAppendArgs {
    PagedArgs a;
    const void* k_new;
    const void* v_new;
    int64_t k_token, k_head, v_token, v_head;
    int head_parts;  // warps per token: each takes a share of the heads
};

// The sequence that holds packed row t (or -1): the last b with cu[b] <= t, by one warp, 32 candidates a step.
__device__ __forceinline__ int seq_of_token(const PagedArgs& a, int t) {
    if (!a.cu) return t / a.uniform_new;
    const int lane = threadIdx.x & 31;
    int lo = 0, n = a.batch;  // the answer is in [lo, lo + n) or there is none
    while (n > 32) {
        const int step = (n + 31) / 32;
        const int i = lane * step;
        const bool ge = i < n && a.cu[lo + i] <= t;
        const unsigned m = __ballot_sync(0xffffffffu, ge);
        if (!m) return -1;
        const int k = 31 - __clz(m);
        lo += k * step;
        n = min(step, n - k * step);
    }
    const unsigned m = __ballot_sync(0xffffffffu, lane < n && a.cu[lo + lane] <= t);
    if (!m) return -1;
    const int b = lo + 31 - __clz(m);
    return t < a.cu[b + 1] ? b : -1;
}

// K and V rows of the new tokens to their places.  Moves 8 D bytes per token and head and does nothing else: bound by latency for
// a decoding step, by HBM for prompts.  A warp takes one token's rows of a share of the heads; its loads of the new rows do
// not wait for the lookups (cu_seqlens, length, page id) that give the destination.  Measured: 24 831 rows of 16 heads, D = 128: 64 us,
// 6.4 TB/s (0.98 of the measured copy rate); 32 rows of 8 heads: 2.5 us in a graph.
template <int D>
__global__ void __launch_bounds__(256) ring_paged_append_kernel(const PagedAppendArgs p) {
    const PagedArgs& a = p.a;
    constexpr int kChunks = D / 8;          // 16-byte chunks per row
    constexpr int kHeads = 32 / kChunks;    // heads one warp-wide access covers
    constexpr int kUnroll = 4;
    const int lane = threadIdx.x & 31;
    const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int t = static_cast<int>(w / p.head_parts);
    const int part = static_cast<int>(w % p.head_parts);
    if (t >= a.tokens) return;
    ptx::griddep_wait();
    const int per = (a.kv_heads + p.head_parts - 1) / p.head_parts;
    const int h_begin = part * per, h_end = min(a.kv_heads, h_begin + per);
    const int ch = (lane % kChunks) * 8, hl = lane / kChunks;
    const uint16_t* kn = static_cast<const uint16_t*>(p.k_new) + t * p.k_token + ch;
    const uint16_t* vn = static_cast<const uint16_t*>(p.v_new) + t * p.v_token + ch;
    uint16_t* kc = static_cast<uint16_t*>(const_cast<void*>(a.k)) + ch;
    uint16_t* vc = static_cast<uint16_t*>(const_cast<void*>(a.v)) + ch;
    int page = -2, slot = 0, b = 0, place = 0;
    for (int h0 = h_begin; h0 < h_end; h0 += kHeads * kUnroll) {
        uint4 kr[kUnroll], vr[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = h0 + u * kHeads + hl;
            if (h < h_end) {
                kr[u] = *reinterpret_cast<const uint4*>(kn + h * p.k_head);
                vr[u] = *reinterpret_cast<const uint4*>(vn + h * p.v_head);
            }
        }
        if (page == -2) {
            page = -1;
            b = seq_of_token(a, t);
            if (b >= 0 && b < a.batch) {
                const SeqView s = seq_view(a, b);
                place = s.pos + (t - s.q0);
                if (t >= s.q0 && t < s.q0 + s.n && place >= 0) page = page_of(a, b, place >> a.page_shift);
            }
            slot = place & ((1 << a.page_shift) - 1);
        }
        if (page < 0) return;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int h = h0 + u * kHeads + hl;
            if (h < h_end) {
                *reinterpret_cast<uint4*>(kc + page * a.k_page + slot * a.k_place + h * a.k_head) = kr[u];
                *reinterpret_cast<uint4*>(vc + page * a.v_page + slot * a.v_place + h * a.v_head) = vr[u];
                if (a.weights && ch == 0) a.weights[b * a.w_batch + h * a.w_head + place] = 0.f;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ eviction
struct PagedEvictArgs {
    PagedArgs a;  // cache, table, lengths, weights
    const int* dst_table;
    int64_t dst_stride;
    int dst_pages;
    int budget, first, recent;
    float* new_weights;
    int64_t nw_batch, nw_head;
    int nw_len;
    int* kept;
    int* new_lens;
};

__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xffffffffu;          // NaN: the largest
    const uint32_t u = __float_as_uint(w + 0.f);  // -0 becomes +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Which places stay: one CTA per (sequence, K/V head).  The key of the last place that fits is found by radix
// selection, three histograms of 11, 11 and 10 bits over the candidates' keys (integer counts: no order of atomics
// can change them); the kept places are then written in order with a running prefix, equal keys from the lowest place up.
// Measured: 128 rows of up to 8192 weights 14 us, four of 1100 8.9 us (latency of the passes).
constexpr int kSelectThreads = 1024;
constexpr int kSelectBins = 2048;
constexpr int kSelectPer = 4;  // consecutive places per thread in the last pass

__device__ __forceinline__ uint32_t select_prefix(uint32_t v, uint32_t* warp_sum, uint32_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    if (warp == 0) {
        uint32_t y = warp_sum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        warp_sum[lane] = y;
    }
    __syncthreads();
    const uint32_t before = warp ? warp_sum[warp - 1] : 0u;
    *total = warp_sum[31];
    __syncthreads();
    return before + x - v;  // exclusive
}

__global__ void __launch_bounds__(kSelectThreads) ring_paged_select_kernel(const PagedEvictArgs p) {
    const PagedArgs& a = p.a;
    __shared__ uint32_t hist[kSelectBins];
    __shared__ uint32_t warp_sum[32];
    __shared__ uint32_t found_digit, found_above;
    ptx::griddep_wait();
    ptx::griddep_launch();
    const int tid = threadIdx.x;
    const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
    const int len = min(max(a.lens[b], 0), a.capacity);
    const int m = min(len, p.budget);
    int* kept = p.kept + (static_cast<int64_t>(b) * a.kv_heads + h) * p.budget;
    const float* w = a.weights + b * a.w_batch + h * a.w_head;
    float* nw = p.new_weights + b * p.nw_batch + h * p.nw_head;
    if (h == 0 && tid == 0) p.new_lens[b] = m;
    for (int i = m + tid; i < p.nw_len; i += kSelectThreads) nw[i] = 0.f;
    for (int i = m + tid; i < p.budget; i += kSelectThreads) kept[i] = -1;
    if (len <= p.budget) {
        for (int i = tid; i < m; i += kSelectThreads) {
            kept[i] = i;
            nw[i] = w[i];
        }
        return;
    }
    for (int i = tid; i < p.first; i += kSelectThreads) {
        kept[i] = i;
        nw[i] = w[i];
    }
    for (int i = tid; i < p.recent; i += kSelectThreads) {
        kept[p.budget - p.recent + i] = len - p.recent + i;
        nw[p.budget - p.recent + i] = w[len - p.recent + i];
    }
    const uint32_t need = p.budget - p.first - p.recent;
    if (need == 0) return;
    const int c0 = p.first, c1 = len - p.recent;  // candidates, more than `need`

    uint32_t prefix = 0, left = need;  // key bits found so far; how many are still to come from keys with this prefix
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10;
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
        for (int i = tid; i < kSelectBins; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        for (int j = c0 + tid; j < c1; j += kSelectThreads) {
            const uint32_t key = weight_key(w[j]);
            const bool in = pass == 0 || (key >> (shift + bits)) == prefix;
            if (in) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // bins from the top: thread t owns bins top - 2t and top - 2t - 1
        const int top = kSelectBins - 1 - 2 * tid;
        const uint32_t n0 = hist[top], n1 = hist[top - 1];
        uint32_t all;
        const uint32_t above = select_prefix(n0 + n1, warp_sum, &all);
        if (above < left && left <= above + n0) {
            found_digit = top;
            found_above = above;
        } else if (above + n0 < left && left <= above + n0 + n1) {
            found_digit = top - 1;
            found_above = above + n0;
        }
        __syncthreads();
        prefix = (prefix << bits) | found_digit;
        left -= found_above;
        __syncthreads();
    }
    // keys above `prefix` stay, and the first `left` of the equal ones
    uint32_t gt_done = 0, eq_done = 0;
    for (int base = c0; base < c1; base += kSelectThreads * kSelectPer) {
        const int j0 = base + tid * kSelectPer;
        uint32_t key[kSelectPer];
        float val[kSelectPer];
        uint32_t gt = 0, eq = 0;
#pragma unroll
        for (int u = 0; u < kSelectPer; ++u) {
            const bool in = j0 + u < c1;
            val[u] = in ? w[j0 + u] : 0.f;
            key[u] = weight_key(val[u]);
            gt += in && key[u] > prefix;
            eq += in && key[u] == prefix;
        }
        uint32_t all;
        const uint32_t before = select_prefix(gt << 16 | eq, warp_sum, &all);
        uint32_t g = gt_done + (before >> 16), e = eq_done + (before & 0xffffu);
#pragma unroll
        for (int u = 0; u < kSelectPer; ++u) {
            if (j0 + u < c1) {
                const bool is_gt = key[u] > prefix, is_eq = key[u] == prefix;
                if (is_gt || (is_eq && e < left)) {
                    const uint32_t at = p.first + g + min(e, left);
                    kept[at] = j0 + u;
                    nw[at] = val[u];
                }
                g += is_gt;
                e += is_eq;
            }
        }
        gt_done += all >> 16;
        eq_done += all & 0xffffu;
    }
}

// The kept rows of K and V to their new places: 8 D bytes read and written per place and head, bound by HBM.  A warp moves
// `kUnroll` sets of rows with all their loads in flight (K in one half of the lanes, V in the other at D = 128).  Measured: 4096 rows
// of 16 x 8 heads, D = 128: 90 us, 5.9 TB/s.
template <int D>
__global__ void __launch_bounds__(256) ring_paged_gather_kernel(const PagedEvictArgs p) {
    const PagedArgs& a = p.a;
    constexpr int kChunks = D / 8;
    constexpr int kLanes = 2 * kChunks;     // lanes per place: its K row, then its V row
    constexpr int kPlaces = 32 / kLanes;    // places per warp-wide access
    constexpr int kUnroll = 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int bh = blockIdx.y, b = bh / a.kv_heads, h = bh % a.kv_heads;
    const bool is_v = (lane % kLanes) >= kChunks;
    const int64_t page_stride = is_v ? a.v_page : a.k_page, place_stride = is_v ? a.v_place : a.k_place;
    uint16_t* base = static_cast<uint16_t*>(const_cast<void*>(is_v ? a.v : a.k)) + h * (is_v ? a.v_head : a.k_head) + (lane % kChunks) * 8;
    const int j0 = (blockIdx.x * 8 + warp) * kPlaces * kUnroll + lane / kLanes;
    const int mask = (1 << a.page_shift) - 1;
    ptx::griddep_wait();
    const int* kept = p.kept + static_cast<int64_t>(bh) * p.budget;
    int from[kUnroll], to[kUnroll], src[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int j = j0 + u * kPlaces;
        from[u] = j < p.budget ? kept[j] : -1;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int j = j0 + u * kPlaces;
        src[u] = to[u] = -1;
        if (from[u] >= 0) {
            src[u] = page_of(a, b, from[u] >> a.page_shift);
            const int pi = j >> a.page_shift;
            if (pi < p.dst_pages) to[u] = p.dst_table[static_cast<int64_t>(b) * p.dst_stride + pi];
            if (to[u] >= a.num_pages) to[u] = -1;
        }
    }
    uint4 row[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
        if (src[u] >= 0 && to[u] >= 0)
            row[u] = *reinterpret_cast<const uint4*>(base + src[u] * page_stride + (from[u] & mask) * place_stride);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
        if (src[u] >= 0 && to[u] >= 0)
            *reinterpret_cast<uint4*>(base + to[u] * page_stride + ((j0 + u * kPlaces) & mask) * place_stride) = row[u];
}

}  // namespace ring
