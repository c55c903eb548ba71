// What the paged-cache kernels share: their argument block, the view of one sequence, and the plan that deals the work
// of a ragged batch out to CTAs on the device.
//
// The lengths of the sequences live on the device and no call waits for them, so the host cannot size a grid by them.  The
// attention kernels therefore run a fixed grid of resident CTAs; each computes the total number of key blocks that all units
// (sequence, K/V head, tile of query rows) have to visit, takes its equal share [c T / n, (c + 1) T / n) of that list, and
// walks the units in it.  A unit that a share boundary cuts leaves normalised partials with their LSE in the
// workspace, which a second small kernel joins (the algebra of lse_merge.cuh over many partials).  So a batch of one long
// sequence and thirty short ones keeps every SM equally busy, and a single sequence is cut as finely as there are CTAs.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace ring {

struct PagedArgs {
    const void* k;
    const void* v;
    int64_t k_page, k_head, k_place, v_page, v_head, v_place;  // strides in elements
    int num_pages, page_shift, kv_heads;
    const int* table;
    int64_t table_stride;
    int max_pages, capacity;  // capacity = max_pages << page_shift
    int batch;
    const int* lens;
    const int* cu;  // or null: uniform_new tokens each
    int uniform_new, tokens;
    const void* q;
    int64_t q_token, q_head;
    int heads, group;  // group = heads / kv_heads
    int out_fp32;
    void* out;
    int64_t out_token, out_head;
    float* lse;  // [tokens, heads]
    float scale, scale_log2;
    int causal, window, sinks;
    int unit_rows;    // query rows (token-major, then head of the group) per unit
    int many_tiles;   // hint: a sequence may have many tiles, sum its blocks with a warp instead of a thread
    int min_blocks;   // key blocks a CTA should at least get
    float* weights;
    int64_t w_batch, w_head;
    // workspace of the attention kernels: part_o [2 * grid][unit_rows][D], part_lse [2 * grid][unit_rows], cut [grid]
    float* part_o;
    float* part_lse;
    int4* cut;  // two int4 per CTA: {sequence, kv head, first row, rows}, {parts, first token row, 0, 0}
    int* status;
};

struct SeqView {
    int q0;   // first packed row
    int n;    // new tokens
    int len;  // places, the new ones included
};

__device__ __forceinline__ SeqView seq_view(const PagedArgs& a, int b) {
    SeqView s;
    if (a.cu) {
        s.q0 = min(max(a.cu[b], 0), a.tokens);
        s.n = max(min(a.cu[b + 1], a.tokens) - s.q0, 0);
    } else {
        s.q0 = b * a.uniform_new;
        s.n = a.uniform_new;
    }
    s.len = min(max(a.lens[b], 0), a.capacity);
    return s;
}

// Page id holding places [i, i + 1) * page_size of sequence b, or -1 if there is none.
__device__ __forceinline__ int page_of(const PagedArgs& a, int b, int i) {
    if (i < 0 || i >= a.max_pages) return -1;
    const int id = a.table[static_cast<int64_t>(b) * a.table_stride + i];
    return (id >= 0 && id < a.num_pages) ? id : -1;
}

// Places a token of the sequence sees: [0, hi) without [sinks, lo).
__device__ __forceinline__ int token_hi(const PagedArgs& a, const SeqView& s, int token) {
    return a.causal ? min(max(s.len - s.n + token + 1, 0), s.len) : s.len;
}
__device__ __forceinline__ int token_lo(const PagedArgs& a, const SeqView& s, int token) {
    return a.window > 0 ? max(s.len - s.n + token - a.window + 1, 0) : 0;
}

// The key blocks of BN places a tile of query rows has to visit: blocks [0, sink) and then [first, ...), count in all.
// At least one, so that a tile that sees nothing is still visited and writes its empty rows.
struct TileBlocks {
    int count, sink, first;
    __device__ __forceinline__ int block(int i) const { return i < sink ? i : i - sink + first; }
};

template <int BN>
__device__ __forceinline__ TileBlocks tile_blocks(const PagedArgs& a, const SeqView& s, int row0, int rows) {
    const int t0 = row0 / a.group, t1 = (row0 + rows - 1) / a.group;
    const int hi = token_hi(a, s, t1), lo = token_lo(a, s, t0);
    TileBlocks r;
    r.sink = 0;
    r.first = 0;
    const int last = (hi + BN - 1) / BN;
    if (lo > 0) {
        r.sink = (min(a.sinks, hi) + BN - 1) / BN;
        r.first = max(lo / BN, r.sink);
    }
    r.count = max(r.sink + max(last - r.first, 0), 1);
    return r;
}

__device__ __forceinline__ int seq_tiles(const PagedArgs& a, const SeqView& s) {
    return (s.n * a.group + a.unit_rows - 1) / a.unit_rows;
}
__device__ __forceinline__ int tile_rows(const PagedArgs& a, const SeqView& s, int tile) {
    return min(a.unit_rows, s.n * a.group - tile * a.unit_rows);
}

// One unit's piece in a CTA's share.
struct Segment {
    int b, h, tile;
    int first, count;  // index of the first of the unit's blocks to visit, and how many
    int unit_blocks;
    int tiles;   // of the sequence
    int valid;
};

struct PlanShared {
    int64_t warp_sum[33];
    int64_t total;  // key blocks per K/V head, over all sequences
    int found_b;
    int64_t found_before;
    int64_t found_own;
    Segment seg;
    int active;       // CTAs that have a share
    int64_t x0, x1;   // this CTA's share
};

// Sum of the sequence's tile blocks (one K/V head), by one warp (all lanes call it, all get the sum).
template <int BN>
__device__ __forceinline__ int64_t seq_blocks_warp(const PagedArgs& a, const SeqView& s) {
    const int tiles = seq_tiles(a, s);
    int64_t sum = 0;
    for (int t = threadIdx.x & 31; t < tiles; t += 32)
        sum += tile_blocks<BN>(a, s, t * a.unit_rows, tile_rows(a, s, t)).count;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}
template <int BN>
__device__ __forceinline__ int64_t seq_blocks_thread(const PagedArgs& a, const SeqView& s) {
    const int tiles = seq_tiles(a, s);
    int64_t sum = 0;
    for (int t = 0; t < tiles; ++t) sum += tile_blocks<BN>(a, s, t * a.unit_rows, tile_rows(a, s, t)).count;
    return sum;
}

// Exclusive prefix over the block's threads; *total receives the sum.  Every thread calls it.
template <int kThreads>
__device__ __forceinline__ int64_t block_prefix(PlanShared& p, int64_t v, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) p.warp_sum[warp] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        const int64_t y = p.warp_sum[w];
        if (w < warp) before += y;
        all += y;
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// This thread's sequence of the chunk starting at b0: its blocks per K/V head (0 past the batch).
// kSlots sequences per chunk: one per thread, or one per warp when sequences may have many tiles.
template <int BN, int kThreads>
__device__ __forceinline__ int64_t chunk_blocks(const PagedArgs& a, int b0, int* b_out) {
    int64_t own = 0;
    int b;
    if (a.many_tiles) {
        b = b0 + (threadIdx.x >> 5);
        if (b < a.batch) {
            own = seq_blocks_warp<BN>(a, seq_view(a, b));
            if (threadIdx.x & 31) own = 0;
        }
        if (threadIdx.x & 31) b = -1;
    } else {
        b = b0 + threadIdx.x;
        if (b < a.batch) own = seq_blocks_thread<BN>(a, seq_view(a, b));
    }
    *b_out = b;
    return own;
}

// Computes this CTA's share and its first segment into `p` (all threads call it; ends in a __syncthreads).
template <int BN, int kThreads>
__device__ void plan_start(const PagedArgs& a, PlanShared& p, int cta, int ctas) {
    const int step = a.many_tiles ? kThreads / 32 : kThreads;
    const bool single = a.batch <= step;
    int64_t total = 0, own = 0, before = 0, chunk_total = 0;
    int b = 0;
    for (int b0 = 0; b0 < a.batch; b0 += step) {
        own = chunk_blocks<BN, kThreads>(a, b0, &b);
        before = block_prefix<kThreads>(p, own, &chunk_total);
        total += chunk_total;
    }
    const int64_t all = total * a.kv_heads;
    int64_t want = (all + a.min_blocks - 1) / a.min_blocks;
    const int active = static_cast<int>(want < ctas ? want : ctas);
    int64_t x0 = 0, x1 = 0;
    if (cta < active) {
        x0 = all * cta / active;
        x1 = all * (cta + 1) / active;
    }
    if (threadIdx.x == 0) {
        p.total = total;
        p.active = active;
        p.x0 = x0;
        p.x1 = x1;
        p.found_b = -1;
        p.seg.valid = 0;
    }
    __syncthreads();
    if (x0 >= x1) return;  // CTA-uniform
    // the sequence whose units hold block x0
    int64_t done = 0;
    for (int b0 = 0; b0 < a.batch; b0 += step) {
        if (!single) {
            own = chunk_blocks<BN, kThreads>(a, b0, &b);
            before = block_prefix<kThreads>(p, own, &chunk_total);
        }
        const int64_t lo = (done + before) * a.kv_heads, hi = lo + own * a.kv_heads;
        if (own > 0 && x0 >= lo && x0 < hi) {
            p.found_b = b;
            p.found_before = lo;
            p.found_own = own;
        }
        done += chunk_total;
        if (done * a.kv_heads > x0) break;  // CTA-uniform
    }
    __syncthreads();
    // the head and the tile within it: one warp
    if (threadIdx.x < 32) {
        const int fb = p.found_b;
        const SeqView s = seq_view(a, fb);
        const int h = static_cast<int>((x0 - p.found_before) / p.found_own);
        int64_t rest = (x0 - p.found_before) - h * p.found_own;
        const int tiles = seq_tiles(a, s);
        for (int t0 = 0; t0 < tiles; t0 += 32) {
            const int t = t0 + threadIdx.x;
            int c = t < tiles ? tile_blocks<BN>(a, s, t * a.unit_rows, tile_rows(a, s, t)).count : 0;
            int x = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (threadIdx.x >= o) x += y;
            }
            const int sum = __shfl_sync(0xffffffffu, x, 31);
            if (rest < sum) {
                if (c > 0 && rest >= x - c && rest < x) {
                    Segment g;
                    g.b = fb;
                    g.h = h;
                    g.tile = t;
                    g.tiles = tiles;
                    g.unit_blocks = c;
                    g.first = static_cast<int>(rest) - (x - c);
                    const int64_t left = x1 - x0;
                    g.count = static_cast<int>(left < c - g.first ? left : c - g.first);
                    g.valid = 1;
                    p.seg = g;
                }
                break;
            }
            rest -= sum;
        }
    }
    __syncthreads();
}

// The segment after `g` in a share that has `left` blocks remaining behind g.  One thread.
template <int BN>
__device__ __forceinline__ Segment plan_next(const PagedArgs& a, Segment g, int64_t left) {
    g.valid = 0;
    if (left <= 0) return g;
    SeqView s;
    if (g.tile + 1 < g.tiles) {
        ++g.tile;
        s = seq_view(a, g.b);
    } else if (g.h + 1 < a.kv_heads) {
        ++g.h;
        g.tile = 0;
        s = seq_view(a, g.b);
    } else {
        g.h = 0;
        g.tile = 0;
        do {
            if (++g.b >= a.batch) return g;
            s = seq_view(a, g.b);
        } while (s.n == 0);
        g.tiles = seq_tiles(a, s);
    }
    g.unit_blocks = tile_blocks<BN>(a, s, g.tile * a.unit_rows, tile_rows(a, s, g.tile)).count;
    g.first = 0;
    g.count = static_cast<int>(left < g.unit_blocks ? left : g.unit_blocks);
    g.valid = 1;
    return g;
}

// Where a segment's result goes: -1 = the unit is whole, straight to the output; else its partial slot.
__device__ __forceinline__ int partial_slot(const Segment& g, int cta) {
    if (g.count == g.unit_blocks) return -1;
    return g.first > 0 ? 2 * cta : 2 * cta + 1;
}

// CTA `cta` notes the unit that begins in its share and ends behind it (parts = 0: there is none).
__device__ __forceinline__ void note_cut(const PagedArgs& a, const PlanShared& p, const Segment& g, int cta, int64_t x_seg, int row0,
                                         int rows, int q0) {
    // the unit ends at block x_seg - first + unit_blocks; the CTA that holds its last block is the largest c with
    // all * c / active <= that block
    const int64_t all = p.total * a.kv_heads;
    const int64_t last = x_seg - g.first + g.unit_blocks - 1;
    int64_t c = last * p.active / all;
    while (c + 1 < p.active && all * (c + 1) / p.active <= last) ++c;
    while (c > 0 && all * c / p.active > last) --c;
    a.cut[2 * cta] = make_int4(g.b, g.h, row0, rows);
    a.cut[2 * cta + 1] = make_int4(static_cast<int>(c) - cta + 1, q0, 0, 0);
}

}  // namespace ring
