// What the paged-cache kernels share: their argument block, the view of one sequence, and the plan that deals the work
// of a ragged batch out to CTAs on the device.
//
// The lengths of the sequences live on the device and no call waits for them, so the host cannot size a grid by them.  The
// kernels therefore run a fixed grid of resident CTAs; each computes the total cost of all units (sequence, K/V head, tile: of
// query rows for attention, of places for the weights), takes its equal share [c T / n, (c + 1) T / n) of that list, and
// walks the units in it.  A unit costs its blocks plus a constant for starting it: without the constant the CTA that got
// a batch's short sequences and idle slots finished last (b32 ragged to 8192, 8 K/V heads: busiest SM 1.35 times the mean).  A unit
// that a share boundary cuts leaves partials in the workspace, which a second small kernel joins.  So a batch of one long
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
    uint32_t group_mul, group_shift;  // x / group = (umulhi(x, mul) + x) >> shift for 0 <= x < 2^31
    int out_fp32;
    void* out;
    int64_t out_token, out_head;
    float* lse;  // [tokens, heads]
    float scale, scale_log2;
    int causal, window, sinks;
    int unit_rows, unit_shift;  // query rows (token-major, then head of the group) per unit, a power of two
    int many_tiles;   // hint: a sequence may have many tiles, sum its blocks with a warp instead of a thread
    int min_blocks;   // cost a CTA should at least get
    int start_cost;   // cost of starting a unit, in blocks
    float* weights;
    int64_t w_batch, w_head;
    int row_tokens;   // weights, chunk form: tokens per tile of query rows
    uint32_t tokens_mul, tokens_shift;  // x / row_tokens, as group_mul
    // workspace.  Attention: part_o [2 * grid][unit_rows][D], part_lse [2 * grid][unit_rows], cut [grid];
    // weights, chunk form: part_lse [2 * grid][256] (sums), cut [grid]
    float* part_o;
    float* part_lse;
    int4* cut;  // two int4 per CTA: {sequence, kv head, first row, rows}, {parts, first token row, 0, 0}
    int* status;
};

__device__ __forceinline__ int div_group(const PagedArgs& a, int x) {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(x), a.group_mul) + static_cast<uint32_t>(x)) >> a.group_shift);
}

__device__ __forceinline__ int div_tokens(const PagedArgs& a, int x) {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(x), a.tokens_mul) + static_cast<uint32_t>(x)) >> a.tokens_shift);
}

struct SeqView {
    int q0;   // first packed row
    int n;    // new tokens
    int len;  // places that exist: at most what the table's pages hold
    int pos;  // place of the first new token, by the length as given (a place behind the table's pages does not exist)
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
    const int given = max(a.lens[b], 0);
    s.len = min(given, a.capacity);
    s.pos = given - s.n;
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
    return a.causal ? min(max(s.pos + token + 1, 0), s.len) : s.len;
}
__device__ __forceinline__ int token_lo(const PagedArgs& a, const SeqView& s, int token) {
    // at most len, or the blocks of a window far behind the table's pages would lie where 32 bits turn over
    return a.window > 0 ? min(max(s.pos + token - a.window + 1, 0), s.len) : 0;
}

// The key blocks of BN places a tile of query rows has to visit: blocks [0, sink) and then [first, ...), count in all.
// At least one, so that a tile that sees nothing is still visited and writes its empty rows.
struct TileBlocks {
    int count, sink, first;
    __device__ __forceinline__ int block(int i) const { return i < sink ? i : i - sink + first; }
};

template <int BN>
__device__ __forceinline__ TileBlocks tile_blocks(const PagedArgs& a, const SeqView& s, int row0, int rows) {
    const int t0 = div_group(a, row0), t1 = div_group(a, row0 + rows - 1);
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
    return (s.n * a.group + a.unit_rows - 1) >> a.unit_shift;
}
__device__ __forceinline__ int tile_rows(const PagedArgs& a, const SeqView& s, int tile) {
    return min(a.unit_rows, s.n * a.group - tile * a.unit_rows);
}

// What the attention kernels deal out: tiles of unit_rows query rows, with the BN-place key blocks each has to visit.
template <int BN>
struct AttentionUnits {
    static __device__ __forceinline__ int tiles(const PagedArgs& a, const SeqView& s) { return seq_tiles(a, s); }
    static __device__ __forceinline__ int blocks(const PagedArgs& a, const SeqView& s, int tile) {
        return tile_blocks<BN>(a, s, tile * a.unit_rows, tile_rows(a, s, tile)).count;
    }
};

// One unit's piece in a CTA's share.
struct Segment {
    int b, h, tile;
    int tiles;        // of the sequence
    int first, count; // index of the first of the unit's blocks to visit, and how many
    int unit_blocks;
    int valid;
    int64_t begin;    // where the unit begins in the list of costs
};

// A CTA's share [x0, x1) of the list of costs: quot + 1 for the first rem shares, quot for the others.
struct Share {
    int64_t quot, rem;
    int active;   // CTAs that have a share
    int64_t x0, x1;
};

// List positions may pass 32 bits (a very long prompt), and a 64-bit division is a long piece of code that every launch would
// fetch: x / n for n < 2^15 goes digit by digit, quotients by other list positions are found by halving.
__device__ __forceinline__ int64_t div_small(int64_t x, uint32_t n) {
    if ((x >> 32) == 0) return static_cast<uint32_t>(x) / n;
    int64_t q = 0;
    uint32_t r = 0;
#pragma unroll 1
    for (int sh = 48; sh >= 0; sh -= 16) {
        const uint32_t cur = r << 16 | static_cast<uint32_t>((x >> sh) & 0xffff);
        q = q << 16 | (cur / n);
        r = cur % n;
    }
    return q;
}

__device__ __forceinline__ int64_t share_begin(const Share& sh, int c) { return c * sh.quot + (c < sh.rem ? c : sh.rem); }

__device__ __forceinline__ Share make_share(const PagedArgs& a, int64_t all, int cta, int ctas) {
    Share r;
    r.active = all >= static_cast<int64_t>(a.min_blocks) * ctas
                   ? ctas
                   : (static_cast<int>(all) + a.min_blocks - 1) / a.min_blocks;
    r.quot = r.rem = r.x0 = r.x1 = 0;
    if (cta < r.active) {
        r.quot = div_small(all, r.active);
        r.rem = all - r.quot * r.active;
        r.x0 = share_begin(r, cta);
        r.x1 = share_begin(r, cta + 1);
    }
    return r;
}

// Cost of the sequence's units for one K/V head: by one thread, or by a warp (all its lanes call it and get the sum).
template <class U>
__device__ __forceinline__ int64_t seq_cost_thread(const PagedArgs& a, const SeqView& s) {
    const int tiles = U::tiles(a, s);
    int64_t sum = 0;
    for (int t = 0; t < tiles; ++t) sum += U::blocks(a, s, t) + a.start_cost;
    return sum;
}
template <class U>
__device__ __forceinline__ int64_t seq_cost_warp(const PagedArgs& a, const SeqView& s) {
    const int tiles = U::tiles(a, s);
    int64_t sum = 0;
    for (int t = threadIdx.x & 31; t < tiles; t += 32) sum += U::blocks(a, s, t) + a.start_cost;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// The piece of a unit that begins at `g.begin` (g.b, h, tile, tiles, unit_blocks set) inside [from, x1).
__device__ __forceinline__ void cut_unit(const PagedArgs& a, Segment& g, int64_t from, int64_t x1) {
    const int64_t blocks0 = g.begin + a.start_cost;
    g.first = from > blocks0 ? static_cast<int>(from - blocks0) : 0;
    const int64_t end = x1 - blocks0;
    g.count = static_cast<int>(end < g.unit_blocks ? end : g.unit_blocks) - g.first;
    g.valid = g.count > 0;
}

// The segment after `g` in the share.  Every thread that needs it works it out.
template <class U>
__device__ __forceinline__ Segment plan_next(const PagedArgs& a, const Share& sh, Segment g) {
    const int64_t at = g.begin + a.start_cost + g.unit_blocks;  // where the next unit begins
    g.valid = 0;
    if (g.first + g.count < g.unit_blocks || at >= sh.x1) return g;
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
            g.tiles = U::tiles(a, s);
        } while (g.tiles == 0);
    }
    g.begin = at;
    g.unit_blocks = U::blocks(a, s, g.tile);
    cut_unit(a, g, at, sh.x1);
    return g;
}

// The first segment of the share: x0 lies in sequence b, whose list begins at `before` and costs `own` per head.  Called by a
// whole warp, which gets the result in every lane.
template <class U>
__device__ __forceinline__ Segment first_segment(const PagedArgs& a, const Share& sh, int b, int64_t before, int64_t own) {
    const int lane = threadIdx.x & 31;
    const SeqView s = seq_view(a, b);
    Segment g;
    g.b = b;
    const int64_t rel = sh.x0 - before;
    g.h = 0;
    for (int step = 1 << (31 - __clz(a.kv_heads)); step; step >>= 1)
        if (g.h + step < a.kv_heads && (g.h + step) * own <= rel) g.h += step;
    g.tiles = U::tiles(a, s);
    int64_t at = before + g.h * own;  // list position of the tiles looked at
    g.tile = 0;
    g.begin = at;
    g.unit_blocks = 0;
    for (int t0 = 0; t0 < g.tiles; t0 += 32) {
        const int t = t0 + lane;
        const int c = t < g.tiles ? U::blocks(a, s, t) + a.start_cost : 0;
        int x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, c > 0 && sh.x0 < at + x);
        if (hit) {
            const int l = __ffs(hit) - 1;
            g.tile = t0 + l;
            g.unit_blocks = __shfl_sync(0xffffffffu, c, l) - a.start_cost;
            g.begin = at + __shfl_sync(0xffffffffu, x - c, l);
            break;
        }
        at += __shfl_sync(0xffffffffu, x, 31);
    }
    cut_unit(a, g, sh.x0, sh.x1);
    return g;
}

struct PlanShared {
    int64_t warp_sum[32];
    int found_b;
    int64_t found_before, found_own;
    // for kernels whose warps have no registers to spare for them: the share, and the current and the next segment
    Share share;
    Segment seg[2];
};

// This CTA's share and its first segment (all threads call it and get the same; `p` is scratch).
template <class U, int kThreads>
__device__ __forceinline__ Segment plan_start(const PagedArgs& a, PlanShared& p, Share& sh, int cta, int ctas) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Segment none;
    none.valid = 0;
    if (a.batch <= 32) {
        // every warp works it out for itself: no barrier on the way to the first load
        int64_t own = 0;
        if (a.many_tiles) {
            for (int b = 0; b < a.batch; ++b) {
                const int64_t c = seq_cost_warp<U>(a, seq_view(a, b));
                if (lane == b) own = c;
            }
        } else if (lane < a.batch) {
            own = seq_cost_thread<U>(a, seq_view(a, lane));
        }
        int64_t x = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        sh = make_share(a, __shfl_sync(0xffffffffu, x, 31) * a.kv_heads, cta, ctas);
        if (sh.x0 >= sh.x1) return none;
        const unsigned hit = __ballot_sync(0xffffffffu, own > 0 && sh.x0 < x * a.kv_heads);
        const int b = __ffs(hit) - 1;
        return first_segment<U>(a, sh, b, __shfl_sync(0xffffffffu, x - own, b) * a.kv_heads, __shfl_sync(0xffffffffu, own, b));
    }
    // larger batches: a sequence per thread (per warp if they may have many tiles), prefix sums over the CTA
    const int step = a.many_tiles ? kThreads / 32 : kThreads;
    int64_t total = 0;
    auto chunk = [&](int b0, int* b_out, int64_t* own_out, int64_t* chunk_total) {
        int64_t own = 0;
        int b;
        if (a.many_tiles) {
            b = b0 + warp;
            if (b < a.batch) own = seq_cost_warp<U>(a, seq_view(a, b));
            if (lane) own = 0;
        } else {
            b = b0 + threadIdx.x;
            if (b < a.batch) own = seq_cost_thread<U>(a, seq_view(a, b));
        }
        int64_t x = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) p.warp_sum[warp] = x;
        __syncthreads();
        int64_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            const int64_t y = p.warp_sum[w];
            if (w < warp) before += y;
            all += y;
        }
        *b_out = b;
        *own_out = own;
        *chunk_total = all;
        return before + x - own;
    };
    int b = 0;
    int64_t own = 0, chunk_total = 0;
    for (int b0 = 0; b0 < a.batch; b0 += step) {
        chunk(b0, &b, &own, &chunk_total);
        total += chunk_total;
    }
    sh = make_share(a, total * a.kv_heads, cta, ctas);
    if (sh.x0 >= sh.x1) return none;  // CTA-uniform
    int64_t done = 0;
    for (int b0 = 0; b0 < a.batch && done * a.kv_heads <= sh.x0; b0 += step) {
        const int64_t before = chunk(b0, &b, &own, &chunk_total);
        const int64_t lo = (done + before) * a.kv_heads;
        if (own > 0 && sh.x0 >= lo && sh.x0 < lo + own * a.kv_heads) {
            p.found_b = b;
            p.found_before = lo;
            p.found_own = own;
        }
        done += chunk_total;
    }
    __syncthreads();
    return first_segment<U>(a, sh, p.found_b, p.found_before, p.found_own);
}

// Where a segment's result goes: -1 = the unit is whole, straight to the output; else its partial slot.
__device__ __forceinline__ int partial_slot(const Segment& g, int cta) {
    if (g.count == g.unit_blocks) return -1;
    return g.first > 0 ? 2 * cta : 2 * cta + 1;
}

// The CTA, `cta` or a later one, whose share holds list position x.
__device__ __forceinline__ int cta_of(const Share& sh, int cta, int64_t x) {
    int c = cta;
    for (int step = 1 << (31 - __clz(sh.active)); step; step >>= 1)
        if (c + step < sh.active && share_begin(sh, c + step) <= x) c += step;
    return c;
}

// CTA `cta` notes the unit whose first block is in its share and whose last is not: the pieces in between lie in the shares up to
// the one with the unit's last block.
__device__ __forceinline__ void note_cut(const PagedArgs& a, const Share& sh, const Segment& g, int cta, int row0, int rows, int q0) {
    const int last = cta_of(sh, cta, g.begin + a.start_cost + g.unit_blocks - 1);
    a.cut[2 * cta] = make_int4(g.b, g.h, row0, rows);
    a.cut[2 * cta + 1] = make_int4(last - cta + 1, q0, 0, 0);
}

}  // namespace ring
