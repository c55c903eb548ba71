// Paged attention for many query rows (chunks of a prompt, many drafted tokens): bound by the tensor pipe.
//
// The block kernel's machinery (block_attention.cuh: two 128-row Q tiles per CTA, S = Q K^T and O += P V on tcgen05 with
// accumulators in TMEM, P read from TMEM, one S buffer that the tiles use in turn, lazy rescale, bounded waits), with what a
// paged cache needs:
//   * query rows are (token, head of the group) pairs of ONE K/V head, packed token-major, so every K/V block that is loaded
//     serves the whole group; the softmax warps fetch them (any token and head strides) and store them swizzled;
//   * a K/V block of 128 places is gathered page by page: one TMA box of min(page, 128) places per lane of the loader
//     warp; pages that nobody sees are fetched from behind the last page, which reads as zeros without traffic;
//   * V rows that no row of the unit sees are zeroed in shared memory on the blocks at the edges (0 x NaN is not 0);
//   * a CTA walks an equal share of all units' blocks (paged_plan.cuh), with running phase counters across units; a unit that a
//     share boundary cuts leaves normalised fp32 partials; the loader warp runs ahead into the next unit.
// P is rounded to the inputs' type as in the block kernel (at most 2^-8 of it for bf16, 2^-11 for fp16); sums and statistics are fp32.
//
// Measured: 2048 tokens over 32768 places, 32 / 8 heads, D = 128, bf16: 1.04 ms in a steady loop (1.03 PFLOP/s, 0.61 of the measured
// cuBLAS burst rate; 0.87 ms, 1.22 PFLOP/s from idle), about 3 thousand clocks a block of 2 x 128 rows by 128 places as in the block kernel,
// bound by its S-buffer chain.  At D = 64 the same takes 0.74 ms (0.67 PFLOP/s; its exponentials need 0.46 ms of the MUFU).  With a window of
// 4096 + 4: 160 us at D = 128, 143 at 64.  4 chunks of 130-515 tokens over 1500-6001 places, 16 heads: 114 us; a quarter of its rows are
// padding of the last tiles and joining the cut units takes 14 us.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "kernel_traits.h"
#include "paged_plan.cuh"
#include "paged_rows.cuh"
#include "ptx_sm100.cuh"

namespace ring {

// Values of the device status word (continuing the block kernel's).
enum PagedDeviceStatus : int {
    kDevPagedLoad = 131,
    kDevPagedMmaQ = 132,
    kDevPagedMmaKV = 133,
    kDevPagedMmaS = 134,
    kDevPagedMmaP = 135,
    kDevPagedSoftmaxS = 136,
    kDevPagedSoftmaxO = 137,
};

namespace ptx {
__device__ __forceinline__ void fence_proxy_async_cta() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Named barrier that also tells every thread whether any of them brought `pred`.
__device__ __forceinline__ bool bar_any(int id, int threads, bool pred) {
    uint32_t any;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.u32 p, %3, 0;\n\t"
        "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}"
        : "=r"(any)
        : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(pred))
        : "memory");
    return any != 0;
}
}  // namespace ptx

// A window's edge, or a page that does not exist: the scores of block col0 that nobody may see are overwritten where they are, in TMEM,
// 32 columns at a time.  By a warp; lo is the thread's row's lower limit.  A call, so that its registers are not the main loop's:
// as one more mask on the 128 scores in registers it cost every block 8 %.
template <bool kWindow>
__device__ __noinline__ void hide_scores(const PagedArgs& a, uint32_t t_s, int b, int col0, int lo) {
    using namespace ptx;
    const int lane = threadIdx.x & 31;
    const int per_block = a.page_shift >= 7 ? 1 : 128 >> a.page_shift;
    const uint32_t have = __ballot_sync(0xffffffffu, lane < per_block && page_of(a, b, (col0 >> a.page_shift) + lane) >= 0);
#pragma unroll 1
    for (int w = 0; w < 128; w += 32) {
        // 32 columns a word: all without [sink, from), and only in pages that exist
        auto below = [&](int n) { return n <= w ? 0u : (n >= w + 32 ? 0xffffffffu : (1u << (n - w)) - 1u); };
        uint32_t see = kWindow ? below(a.sinks - col0) | ~below(lo - col0) : 0xffffffffu;
#pragma unroll 1
        for (int v = 0; v < 32; v += 8)
            if (!((have >> ((w + v) >> min(a.page_shift, 7))) & 1u)) see &= ~(0xffu << v);
        uint32_t x[32];
        tmem_ld_x32(t_s + w, x);
        tmem_wait_ld();
#pragma unroll
        for (int v = 0; v < 32; ++v)
            if (!((see >> v) & 1u)) x[v] = 0xff800000u;  // -inf
        tmem_st_x32(t_s + w, x);
    }
    tmem_wait_st();
}

// kWindow: the call has a window (its limits held across the main loop cost every block 8 %).
template <class T, bool kWindow>
__global__ void __launch_bounds__(T::kNThreads, 1)
ring_paged_chunk_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ PagedArgs a) {
    using namespace ptx;
    constexpr int D = T::kHeadDim;
    constexpr int BN = T::kBlockN;
    constexpr int kStages = T::kStages;
    constexpr int kTileBytes = T::kTileBytes;
    constexpr int kBoxBytes = T::kBoxBytes;
    constexpr int kBoxes = T::kBoxesPerTile;
    // The block kernel's split, although every warp follows the plan here: ptxas spills 216 bytes a thread. With 208 / 88 the softmax
    // spills in its main loop (2048 tokens over 32768 places: 1341 us against 1071 at the time).
    constexpr int kSoftmaxRegs = 216, kProducerRegs = 72;
    static_assert(256 * kSoftmaxRegs + 128 * kProducerRegs <= 384 * 168, "what the CTA was launched with");
    constexpr uint32_t kIdescQK = umma_idesc_f16(128, BN, false, false, T::kIsBf16);
    constexpr uint32_t kIdescPV = umma_idesc_f16(128, D, false, true, T::kIsBf16);

    extern __shared__ uint8_t smem_raw[];
    __shared__ PlanShared plan;
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_addr);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + T::kSmemTiles);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + T::kNumBarriers);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* prior_error = reinterpret_cast<volatile int*>(tmem_slot + 2);
    // Block n & 7: a page of it that somebody sees does not exist.  The loader is less than eight blocks ahead of the softmax (a V
    // slot is free only when its block's product is done), and its store is ordered before the block's scores by the barriers between.
    volatile int* gap = reinterpret_cast<volatile int*>(tmem_slot + 3);
    static_assert(T::kNumBarriers * 8 + 12 + 32 <= 256 && T::kVStages < 7, "tail of shared memory, depth of the V ring");

    const uint32_t bar0 = smem_u32(bars);
    auto bar_q_full = [&](int t) { return bar0 + 8u * t; };
    auto bar_kv_full = [&](int s) { return bar0 + 8u * (2 + s); };
    auto bar_kv_empty = [&](int s) { return bar0 + 8u * (2 + kStages + s); };
    auto bar_s_full = [&](int t) { return bar0 + 8u * (2 + 2 * kStages + t); };
    auto bar_p_full = [&](int t) { return bar0 + 8u * (4 + 2 * kStages + t); };
    auto bar_o_done = [&](int t) { return bar0 + 8u * (6 + 2 * kStages + t); };
    const uint32_t bar_s_free = bar0 + 8u * (8 + 2 * kStages);
    auto smem_q = [&](int t) { return base + static_cast<uint32_t>(t * kTileBytes); };
    auto smem_kv = [&](int s) { return base + static_cast<uint32_t>((T::kQTiles + s) * kTileBytes); };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cta = blockIdx.x;
    griddep_launch();
    if (tid == 0) {
        *abort_flag = 0;
        for (int t = 0; t < 2; ++t) {
            mbar_init(bar_q_full(t), 4);  // one arrival per softmax warp
            mbar_init(bar_s_full(t), 1);
            mbar_init(bar_p_full(t), 4);
            mbar_init(bar_o_done(t), 1);
        }
        mbar_init(bar_s_free, 4);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_kv_full(s), 1);
            mbar_init(bar_kv_empty(s), s < T::kKStages ? 1 : 2);  // K: the S issuer; V: both P V issuers
        }
        fence_mbar_init();
    }
    if (warp == T::kLoadWarp && lane == 0) {
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
    }
    griddep_wait();  // nothing before this touches memory
    if (tid == 0) {
        *prior_error = *reinterpret_cast<volatile int*>(a.status);
        a.cut[2 * cta + 1] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    if (*prior_error != 0) return;  // an earlier launch failed: do nothing (CTA-uniform)
    using U = AttentionUnits<BN>;
    {
        Share share;
        const Segment first = plan_start<U, T::kNThreads>(a, plan, share, cta, gridDim.x);
        if (!first.valid) return;  // no share (CTA-uniform)
        if (tid == 0) {
            plan.share = share;
            plan.seg[0] = first;
        }
    }

    if (warp == T::kMmaWarp) {
        tmem_alloc(smem_u32(tmem_slot), T::kTmemCols);
        tmem_relinquish_alloc_permit();
    }
    tcgen05_fence_before_thread_sync();
    __syncthreads();
    tcgen05_fence_after_thread_sync();
    const uint32_t tmem_base = *tmem_slot;

    // ---- what every role knows of the current segment, and how far its barriers have come
    Segment g = plan.seg[0];
    SeqView s;
    TileBlocks tb;
    int row0, rows, ntiles, hi_max, lo_min;
    uint32_t kv_done = 0;              // K/V blocks of earlier segments
    uint32_t tile1_done = 0;           // ... of those that had a second tile (the first tile takes part in all)
    uint32_t segs_done = 0, segs1_done = 0;  // segments, and those with a second tile
    auto begin_segment = [&]() {
        s = seq_view(a, g.b);
        row0 = g.tile * a.unit_rows;
        rows = tile_rows(a, s, g.tile);
        ntiles = rows > 128 ? 2 : 1;
        tb = tile_blocks<BN>(a, s, row0, rows);
        hi_max = token_hi(a, s, div_group(a, row0 + rows - 1));
        lo_min = token_lo(a, s, div_group(a, row0));
    };
    auto count_segment = [&]() {
        kv_done += g.count;
        ++segs_done;
        if (ntiles > 1) {
            tile1_done += g.count;
            ++segs1_done;
        }
    };
    // All warps but the loader's, which runs ahead into the next segments, meet; false when the CTA is through (its share is done or
    // a wait ran out).  Whether one did is decided by the barrier, the same for all: a flag read afterwards might not be.
    // The S issuer, first to be done with a segment, has left the next one in shared memory (walking the plan in every warp kept
    // so much alive across the softmax that it spilled).
    auto end_segment = [&]() {
        tcgen05_fence_before_thread_sync();
        const bool gone = bar_any(1, T::kNThreads - 32, *abort_flag != 0);
        tcgen05_fence_after_thread_sync();
        if (gone) return false;
        count_segment();
        g = plan.seg[segs_done & 1];
        return g.valid != 0;
    };

    if (warp >= T::kSoftmaxWarps) {
        // ############################################################## producer warpgroup (warps 8..11)
        setmaxnreg_dec<kProducerRegs>();
        if (warp == T::kLoadWarp) {
            // =================================================================== TMA producer: a lane per page
            const int per_block = a.page_shift >= 7 ? 1 : BN >> a.page_shift;  // pages per block (at most 16)
            const int page_rows = min(1 << a.page_shift, BN);                  // places of the block a page holds
            const Share share = plan.share;
            bool ok = true;
            do {
                begin_segment();
                auto page_id = [&](int i) {  // page of this lane in block i, num_pages (reads as zeros) if nobody sees it
                    if (lane >= per_block || i >= g.count) return a.num_pages;
                    const int j0 = tb.block(g.first + i) * BN + lane * page_rows;
                    if (j0 >= hi_max || (j0 + page_rows <= lo_min && j0 >= a.sinks)) return a.num_pages;
                    return page_of(a, g.b, j0 >> a.page_shift);  // -1: there is none
                };
                int id = page_id(0);
#pragma unroll 1
                for (int i = 0; i < g.count && ok; ++i) {
                    const bool missing = __any_sync(0xffffffffu, id < 0);
                    const int id_now = id < 0 ? a.num_pages : id;
                    id = page_id(i + 1);
                    const int in_page = (tb.block(g.first + i) * BN) & ((1 << a.page_shift) - 1) & ~(BN - 1);
                    const uint32_t n = kv_done + i;
#pragma unroll 1
                    for (int kv = 0; kv < 2; ++kv) {
                        const uint32_t nslots = kv == 0 ? T::kKStages : T::kVStages;
                        const int slot = (kv == 0 ? 0 : T::kKStages) + static_cast<int>(n % nslots);
                        const uint32_t use = n / nslots;
                        if (use > 0) {
                            ok = mbar_wait(bar_kv_empty(slot), (use - 1) & 1, abort_flag, a.status, kDevPagedLoad);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                        }
                        if (lane == 0) {
                            if (kv == 0) gap[n & 7] = missing;
                            mbar_arrive_expect_tx(bar_kv_full(slot), kTileBytes);
                        }
                        __syncwarp();
                        if (lane < per_block) {
                            const CUtensorMap* tm = kv == 0 ? &tm_k : &tm_v;
                            const uint32_t dst = smem_kv(slot) + lane * page_rows * 128;
#pragma unroll
                            for (int bx = 0; bx < kBoxes; ++bx)
                                tma_load_4d(dst + bx * kBoxBytes, tm, bar_kv_full(slot), bx * 64, in_page, g.h, id_now);
                        }
                        __syncwarp();
                    }
                }
                count_segment();
                g = plan_next<U>(a, share, g);
            } while (ok && g.valid);
        } else if (warp == T::kMmaWarp) {
            // =================================================================== UMMA issuer: S = Q K^T, both tiles
            uint32_t products = 0;  // S products issued so far; number n - 1 must have been read out before number n
            do {
                begin_segment();
                if (lane == 0) {
                    bool ok = true;
#pragma unroll 1
                    for (int i = 0; i < g.count && ok; ++i) {
                        const uint32_t n = kv_done + i;
                        const int kslot = static_cast<int>(n % T::kKStages);
                        const uint32_t kphase = (n / T::kKStages) & 1;
#pragma unroll 1
                        for (int t = 0; t < ntiles; ++t) {
                            if (i == 0) ok = mbar_wait(bar_q_full(t), (t ? segs1_done : segs_done) & 1, abort_flag, a.status, kDevPagedMmaQ);
                            if (ok && products > 0) ok = mbar_wait(bar_s_free, (products - 1) & 1, abort_flag, a.status, kDevPagedMmaS);
                            if (ok && t == 0) ok = mbar_wait(bar_kv_full(kslot), kphase, abort_flag, a.status, kDevPagedMmaKV);
                            if (!ok) break;
                            tcgen05_fence_after_thread_sync();
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk) {
                                const uint32_t off = (kk >> 2) * kBoxBytes + (kk & 3) * 32;
                                umma_ss(tmem_base + T::kTmemS, umma_desc_kmajor_sw128(smem_q(t) + off),
                                        umma_desc_kmajor_sw128(smem_kv(kslot) + off), kIdescQK, kk > 0 ? 1u : 0u);
                            }
                            umma_commit(bar_s_full(t));
                            if (t == ntiles - 1) umma_commit(bar_kv_empty(kslot));
                            ++products;
                        }
                    }
                    plan.seg[(segs_done + 1) & 1] = plan_next<U>(a, plan.share, g);
                }
                __syncwarp();
            } while (end_segment());
        } else {
            // =================================================================== UMMA issuer: O_t += P_t V, one warp per tile
            const int t = warp - (T::kMmaWarp + 1);
            do {
                begin_segment();
                bool ok = true;
#pragma unroll 1
                for (int i = 0; i < g.count && ok; ++i) {
                    const uint32_t n = kv_done + i;
                    const int vslot = T::kKStages + static_cast<int>(n % T::kVStages);
                    const uint32_t vphase = (n / T::kVStages) & 1;
                    if (lane == 0) ok = mbar_wait(bar_kv_full(vslot), vphase, abort_flag, a.status, kDevPagedMmaKV);
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    if (!ok) break;
                    if (t >= ntiles) {  // no such tile in this unit: release the slot in its name
                        if (lane == 0) mbar_arrive(bar_kv_empty(vslot));
                        continue;
                    }
                    // V rows that no row of the unit sees: zeros (both issuers may write them, the same values)
                    const int j0 = tb.block(g.first + i) * BN;
                    if (j0 + BN > hi_max || (j0 < lo_min && j0 + BN > a.sinks)) {
                        const uint32_t to = smem_kv(vslot) + (lane & 7) * 16;
                        auto clear = [&](int r, int end) {  // rows [r, end): four rows of one box at a time
#pragma unroll 1
                            for (r += lane >> 3; r < end; r += 4) {
#pragma unroll
                                for (int bx = 0; bx < kBoxes; ++bx) st_shared_v4(to + bx * kBoxBytes + r * 128, 0u, 0u, 0u, 0u);
                            }
                        };
                        clear(min(max(hi_max - j0, 0), BN), BN);
                        clear(min(max(a.sinks - j0, 0), BN), min(lo_min - j0, BN));
                        fence_proxy_async_cta();
                        __syncwarp();
                    }
                    if (lane == 0) {
                        ok = mbar_wait(bar_p_full(t), ((t ? tile1_done : kv_done) + i) & 1, abort_flag, a.status, kDevPagedMmaP);
                        if (ok) {
                            tcgen05_fence_after_thread_sync();
#pragma unroll
                            for (int kk = 0; kk < BN / 16; ++kk) {
                                umma_ts(tmem_base + T::kTmemO0 + t * D, tmem_base + T::kTmemP0 + t * T::kTmemPCols + kk * 8,
                                        umma_desc_mnmajor_sw128(smem_kv(vslot) + kk * 16 * 128, kBoxBytes), kIdescPV,
                                        (i > 0 || kk > 0) ? 1u : 0u);
                            }
                            umma_commit(bar_o_done(t));
                            umma_commit(bar_kv_empty(vslot));
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                }
            } while (end_segment());
        }
    } else {
        // ############################################################## softmax warpgroups (warps 0..7)
        setmaxnreg_inc<kSoftmaxRegs>();
        const int t = warp >> 2;
        const int quarter = warp & 3;
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t t_s = tmem_base + lane_addr + T::kTmemS;
        const uint32_t t_p = tmem_base + lane_addr + T::kTmemP0 + t * T::kTmemPCols;
        const uint32_t t_o = tmem_base + lane_addr + T::kTmemO0 + t * D;
        const float c = a.scale_log2;
        do {
            begin_segment();
            if (t < ntiles) {
                // ---- this warp's 32 query rows into the Q tile (swizzled as a TMA load would have left them)
                const int warp_row = t * 128 + quarter * 32;  // row of the unit
                {
                    constexpr int kChunks = D / 8;            // 16-byte chunks per row
                    constexpr int kRowsPer = 32 / kChunks;
                    const int ch = lane % kChunks;
                    uint4 val[32 / kRowsPer];
#pragma unroll
                    for (int u = 0; u < 32 / kRowsPer; ++u) {
                        const int r = warp_row + u * kRowsPer + lane / kChunks;
                        // the last row again instead of a row behind it: a branch around the load would take the loads one by one
                        const int at = row0 + min(r, rows - 1), tok = div_group(a, at);
                        val[u] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(s.q0 + tok) * a.q_token +
                                                                 static_cast<int64_t>(g.h * a.group + (at - tok * a.group)) * a.q_head + ch * 8);
                    }
#pragma unroll
                    for (int u = 0; u < 32 / kRowsPer; ++u) {
                        const int r = quarter * 32 + u * kRowsPer + lane / kChunks;
                        st_shared_v4(smem_q(t) + (ch >> 3) * kBoxBytes + r * 128 + (((ch & 7) ^ (r & 7)) << 4), val[u].x, val[u].y, val[u].z, val[u].w);
                    }
                    fence_proxy_async_cta();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_q_full(t));
                }
                // ---- limits of this thread's row, and of the tile (for the blocks that need no mask)
                const int row = warp_row + lane;
                const int tok = div_group(a, row0 + min(row, rows - 1));
                const int hi = token_hi(a, s, tok), lo = kWindow ? token_lo(a, s, tok) : 0;
                const int tile_first = div_group(a, row0 + t * 128), tile_last = div_group(a, row0 + min(t * 128 + 127, rows - 1));
                const int hi_min = token_hi(a, s, tile_first), lo_max = kWindow ? token_lo(a, s, tile_last) : 0;
                float m_run = -INFINITY;
                float l_run = 0.f;
                bool ok = true;
#pragma unroll 1
                for (int i = 0; i < g.count; ++i) {
                    const uint32_t n = (t ? tile1_done : kv_done) + i;
                    uint32_t sr[128];
                    float* sc = reinterpret_cast<float*>(sr);
                    ok = mbar_wait(bar_s_full(t), n & 1, abort_flag, a.status, kDevPagedSoftmaxS);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tcgen05_fence_after_thread_sync();
                    const int col0 = tb.block(g.first + i) * BN;
                    if ((kWindow && lo_max > col0 && col0 + BN > a.sinks) || gap[(kv_done + i) & 7]) {
                        hide_scores<kWindow>(a, t_s, g.b, col0, lo);
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) tmem_ld_x32(t_s + 32 * u, *reinterpret_cast<uint32_t(*)[32]>(&sr[32 * u]));
                    tmem_wait_ld();
                    tcgen05_fence_before_thread_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_s_free);

                    if (col0 + BN > hi_min) {
                        const int limit = hi - col0;
#pragma unroll
                        for (int u = 0; u < 128; ++u)
                            if (u >= limit) sc[u] = -INFINITY;
                    }

                    float mxc[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) mxc[u] = fmaxf(sc[2 * u], sc[2 * u + 1]);
#pragma unroll
                    for (int v = 16; v < 128; v += 16) {
#pragma unroll
                        for (int u = 0; u < 8; ++u) mxc[u] = fmax3(mxc[u], sc[v + 2 * u], sc[v + 2 * u + 1]);
                    }
                    const float mx = fmaxf(fmax3(mxc[0], mxc[1], mxc[2]), fmax3(fmax3(mxc[3], mxc[4], mxc[5]), mxc[6], mxc[7]));
                    float alpha = 1.f;
                    if (mx > m_run && (m_run == -INFINITY || (mx - m_run) * c > 8.f)) {  // a stale maximum is exact algebra up to 2^8
                        alpha = (m_run == -INFINITY) ? 0.f : ex2_approx((m_run - mx) * c);
                        m_run = mx;
                    }
                    const float nms = (m_run == -INFINITY) ? 0.f : -m_run * c;
                    // all on the MUFU: a quarter on the FMA pipe at head dimension 64, as in the block kernel, is not tried here; it would have
                    // to be ex2_poly2's exact form, because whole rows may be hidden and a NaN score has to stay visible
                    float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
#pragma unroll
                    for (int v = 0; v < 128; v += 4) {
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            float x0, x1;
                            ffma2(x0, x1, sc[v + u], sc[v + u + 1], c, c, nms, nms);
                            sc[v + u] = ex2_approx(x0);
                            sc[v + u + 1] = ex2_approx(x1);
                        }
                        fadd2(a0, a1, a0, a1, sc[v], sc[v + 1]);
                        fadd2(a2, a3, a2, a3, sc[v + 2], sc[v + 3]);
                    }
                    l_run = fmaf(l_run, alpha, (a0 + a1) + (a2 + a3));

                    // P_t of the block before must have been consumed before it is overwritten or O_t rescaled
                    if (i > 0) {
                        ok = mbar_wait(bar_o_done(t), (n - 1) & 1, abort_flag, a.status, kDevPagedSoftmaxO);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tcgen05_fence_after_thread_sync();
                        if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
                            for (int u = 0; u < D / 32; ++u) {
                                uint32_t orr[32];
                                tmem_ld_x32(t_o + 32 * u, orr);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) orr[e] = __float_as_uint(__uint_as_float(orr[e]) * alpha);
                                tmem_st_x32(t_o + 32 * u, orr);
                            }
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t pk[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) pk[e] = pack16<T::kIsBf16>(sc[64 * u + 2 * e], sc[64 * u + 2 * e + 1]);
                        tmem_st_x32(t_p + 32 * u, pk);
                    }
                    tmem_wait_st();
                    tcgen05_fence_before_thread_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_p_full(t));
                }

                // ---- epilogue: O / l and LSE, to the output or to a partial slot
                if (ok) {
                    ok = mbar_wait(bar_o_done(t), ((t ? tile1_done : kv_done) + g.count - 1) & 1, abort_flag, a.status, kDevPagedSoftmaxO);
                    ok = __all_sync(0xffffffffu, ok);
                    if (ok) tcgen05_fence_after_thread_sync();
                }
                if (ok) {
                    const bool have_any = l_run > 0.f || l_run != l_run;  // a NaN score stays visible in the result
                    const float w_new = have_any ? 1.f / l_run : 0.f;
                    const float lse = have_any ? (m_run == -INFINITY ? 0.f : m_run * a.scale) + logf(l_run) : -INFINITY;
                    const int slot = partial_slot(g, cta);
                    constexpr int kHalfCols = D / 2;
                    constexpr int kChunks = kHalfCols / 4;
                    constexpr int kRowsPerInst = 32 / kChunks;
                    const uint32_t stage = smem_q(t) + static_cast<uint32_t>(quarter) * (kTileBytes / 4);
#pragma unroll 1
                    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
                        for (int u = 0; u < kHalfCols / 32; ++u) {
                            uint32_t orr[32];
                            tmem_ld_x32(t_o + pass * kHalfCols + 32 * u, orr);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const int chunk = u * 8 + e;
                                st_shared_v4(stage + lane * (kChunks * 16) + ((chunk ^ (lane & (kChunks - 1))) << 4),
                                             __float_as_uint(__uint_as_float(orr[4 * e + 0]) * w_new),
                                             __float_as_uint(__uint_as_float(orr[4 * e + 1]) * w_new),
                                             __float_as_uint(__uint_as_float(orr[4 * e + 2]) * w_new),
                                             __float_as_uint(__uint_as_float(orr[4 * e + 3]) * w_new));
                            }
                        }
                        __syncwarp();
#pragma unroll 4
                        for (int rr = 0; rr < 32 / kRowsPerInst; ++rr) {
                            const int rl = rr * kRowsPerInst + lane / kChunks;
                            const int ch = lane % kChunks;
                            const float4 val = ld_shared_v4(stage + rl * (kChunks * 16) + ((ch ^ (rl & (kChunks - 1))) << 4));
                            const int r = warp_row + rl;
                            if (r < rows) {
                                const int col = pass * kHalfCols + ch * 4;
                                if (slot >= 0) {
                                    *reinterpret_cast<float4*>(a.part_o + (static_cast<int64_t>(slot) * a.unit_rows + r) * D + col) = val;
                                } else {
                                    const int at = row0 + r, tk = div_group(a, at);
                                    const int64_t to = static_cast<int64_t>(s.q0 + tk) * a.out_token +
                                                       static_cast<int64_t>(g.h * a.group + (at - tk * a.group)) * a.out_head + col;
                                    if (a.out_fp32)
                                        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + to) = val;
                                    else
                                        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + to) =
                                            make_uint2(pack16<T::kIsBf16>(val.x, val.y), pack16<T::kIsBf16>(val.z, val.w));
                                }
                            }
                        }
                        __syncwarp();
                    }
                    if (row < rows) {
                        if (slot >= 0)
                            a.part_lse[static_cast<int64_t>(slot) * a.unit_rows + row] = lse;
                        else
                            a.lse[static_cast<int64_t>(s.q0 + tok) * a.heads + g.h * a.group + (row0 + row - tok * a.group)] = lse;
                    }
                    if (slot == 2 * cta + 1 && tid == 0) note_cut(a, plan.share, g, cta, row0, rows, s.q0);
                }
            }
        } while (end_segment());
    }

    // ---- common exit: every thread arrives here, on success and on a timed-out wait alike
    tcgen05_fence_before_thread_sync();
    __syncthreads();
    if (warp == T::kMmaWarp) {
        tcgen05_fence_after_thread_sync();
        tmem_dealloc(tmem_base, T::kTmemCols);
    }
}

}  // namespace ring
