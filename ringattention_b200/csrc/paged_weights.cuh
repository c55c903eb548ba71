// Accumulated attention weights of the cached places: w_j += sum over the query rows of exp(s_rj - lse_r), the column sums of the
// probability matrix that paged attention never stores.  Two forms, chosen by the number of query rows; in both a place's
// sum is one thread's (or a fixed order of partials), so no atomics and the same bits every time.
//
// Rows form (few rows: decoding): bound by reading K once.  The few-rows attention kernel's pipeline without V; the
// places are the M side of mma.sync m16n8k16 and the query rows the N side, so 8 rows cost one instruction per 16 places.
//
// Chunk form (many rows): two 128 x 128 x D products per 128 query rows and 256 places, then 32768 exponentials and their sums: at 16 a
// clock 2048 clocks of the MUFU against 1024 of tensor time at D = 128.  A quarter of the exponentials goes to the FMA pipe, which
// leaves the MUFU 1536.  S^T = K Q^T with the places as TMEM lanes: a thread owns one place, its sum over the columns stays in a
// register, nothing crosses threads.
//
// Measured: rows form, 16 sequences of 500 to 8192 places, 8 K/V heads, group 4, D = 128, one token: 36 us, 4.1 TB/s (launch, plan and the
// last steps are a third of it).  Chunk form, 1024 tokens over 8192 places, 32 / 8 heads: 99.7 us at D = 128, 95.5 at 64 (57.7 and 55.0 with
// a window of 2048 + 4); all exponentials on the MUFU cost 3 us more, half of them on the FMA pipe 5.  No pipe is the limit (MUFU 48 %, tensor
// 32 % of the active clocks, issue slots 43 %): of the 171 thousand clocks a CTA is active, 53 blocks of about 2500 take 132, unit starts and
// the plan the rest, and the busiest CTA is active for 189.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "kernel_traits.h"
#include "paged_chunk.cuh"
#include "paged_plan.cuh"
#include "paged_rows.cuh"
#include "ptx_sm100.cuh"

namespace ring {

// The place tiles of BN that some new token of the sequence sees.
template <int BN>
__device__ __forceinline__ TileBlocks seen_tiles(const PagedArgs& a, const SeqView& s) {
    TileBlocks tb = tile_blocks<BN>(a, s, 0, s.n * a.group);
    if (token_hi(a, s, s.n - 1) == 0) tb.count = 0;
    return tb;
}

// ------------------------------------------------------------------------------------------------ rows form
template <int D_, bool kBf16_, int NT_>
struct PagedWeightsRowsTraits {
    static constexpr int D = D_;
    static constexpr bool kBf16 = kBf16_;
    static constexpr int NT = NT_;                  // tiles of 8 query rows held in registers
    static constexpr int kWarps = 4, kThreads = 128;
    static constexpr int KT = D == 128 ? 32 : 64;   // places per step of a warp: 8 KiB of K
    static constexpr int BN = kWarps * KT;          // places per block of the plan
    static constexpr int kStages = 3;
    static constexpr int kRowBytes = D * 2;
    static constexpr int kStageBytes = KT * kRowBytes;
    static constexpr int kRing = kStages * kStageBytes;
    static constexpr int kSmem = kWarps * kRing;
};

// A unit is all of a (sequence, K/V head): one tile, its blocks the place blocks that are seen.
template <int BN>
struct WeightsRowsUnits {
    static __device__ __forceinline__ int tiles(const PagedArgs& a, const SeqView& s) { return s.n > 0 && token_hi(a, s, s.n - 1) > 0; }
    static __device__ __forceinline__ int blocks(const PagedArgs& a, const SeqView& s, int) { return seen_tiles<BN>(a, s).count; }
};

template <class T>
__global__ void __launch_bounds__(T::kThreads) ring_paged_weights_rows_kernel(const PagedArgs a) {
    using namespace ptx;
    using U = WeightsRowsUnits<T::BN>;
    constexpr int D = T::D, NT = T::NT, KT = T::KT;
    constexpr int kChunks = T::kRowBytes / 16;
    constexpr int kRowsPer = 32 / kChunks;
    constexpr int NG = KT / 8;                       // groups of 8 places per step
    constexpr int kBatch = 32 / NG;                  // steps whose page ids one warp-wide load fetches
    constexpr int kAhead = T::kStages - 1;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PlanShared plan;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();    // nothing before this may touch memory
    griddep_launch();
    Share share;
    Segment g = plan_start<U, T::kThreads>(a, plan, share, blockIdx.x, gridDim.x);
    const uint32_t ring = smem_u32(smem) + warp * T::kRing;
    const int page_mask = (1 << a.page_shift) - 1;

    while (g.valid) {
        const SeqView s = seq_view(a, g.b);
        const TileBlocks tb = seen_tiles<T::BN>(a, s);
        const int rows = s.n * a.group;
        const int hi_max = token_hi(a, s, s.n - 1), hi_min = token_hi(a, s, 0);
        const int lo_min = token_lo(a, s, 0), lo_max = token_lo(a, s, s.n - 1);
        const int row_tiles = (rows + 8 * NT - 1) / (8 * NT);  // 1 unless the hint was too small
        auto place_of = [&](int i) { return tb.block(g.first + i) * T::BN + warp * KT; };
        auto load_pages = [&](int n) {
            const int i = n * kBatch + lane / NG;
            if (i >= g.count) return -1;
            return page_of(a, g.b, (place_of(i) + 8 * (lane % NG)) >> a.page_shift);
        };
        int ids = load_pages(0);

        // ---- query rows as B fragments (row = lane / 4 of each tile of 8), and of each of this lane's columns (2 (lane & 3), + 1)
        // the negated lse in base 2 and the limits
        uint32_t qf[NT][D / 16][2];
        float nl[NT][2];
        int hi[NT][2], lo[NT][2];
        auto load_rows = [&](int r0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                {
                    const int at = min(r0 + 8 * n + (lane >> 2), rows - 1), tok = div_group(a, at);
                    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(s.q0 + tok) * a.q_token +
                                         static_cast<int64_t>(g.h * a.group + (at - tok * a.group)) * a.q_head + 2 * (lane & 3);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        qf[n][kk][0] = *reinterpret_cast<const uint32_t*>(qp + 16 * kk);
                        qf[n][kk][1] = *reinterpret_cast<const uint32_t*>(qp + 16 * kk + 8);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = r0 + 8 * n + 2 * (lane & 3) + e, at = min(r, rows - 1), tok = div_group(a, at);
                    const float l = a.lse[static_cast<int64_t>(s.q0 + tok) * a.heads + g.h * a.group + (at - tok * a.group)];
                    // rows that see nothing (lse = -inf) and rows behind the last add exp2(-inf) = 0
                    nl[n][e] = (r < rows && l != -INFINITY) ? -l * 1.4426950408889634f : -INFINITY;
                    hi[n][e] = r < rows ? token_hi(a, s, tok) : 0;
                    lo[n][e] = token_lo(a, s, tok);
                }
            }
        };
        load_rows(0);

        const uint16_t* kl = static_cast<const uint16_t*>(a.k) + static_cast<int64_t>(g.h) * a.k_head + (lane % kChunks) * 8 + (lane / kChunks) * a.k_place;
        float* wrow = a.weights + static_cast<int64_t>(g.b) * a.w_batch + static_cast<int64_t>(g.h) * a.w_head;
        int ids_next = -1;
        uint32_t have = 0, seen = 0;
        float old_next[KT / 32] = {};
        bool put_next[KT / 32] = {};
#pragma unroll 1
        for (int i = -kAhead; i < g.count; ++i) {
            const int n = i + kAhead;
            if (n < g.count) {
                if (n % kBatch == 0) {
                    if (n > 0) ids = ids_next;
                    ids_next = load_pages(n / kBatch + 1);
                    have = __ballot_sync(0xffffffffu, ids >= 0);
                }
                const int j0 = place_of(n);
                seen |= ((have >> ((n % kBatch) * NG)) & ((1u << NG) - 1u)) << (kAhead * NG);
                const bool inside = j0 + KT <= hi_max && (j0 >= lo_min || j0 + KT <= a.sinks);
                const uint32_t dst = ring + (n % T::kStages) * T::kStageBytes + (lane / kChunks) * T::kRowBytes;
                __syncwarp();  // every lane is done with the stage
#pragma unroll
                for (int gr = 0; gr < NG; ++gr) {
                    const int id = __shfl_sync(0xffffffffu, ids, (n % kBatch) * NG + gr);
                    const int64_t pg = id >= 0 ? id : 0;
                    const uint16_t* kp = kl + pg * a.k_page + static_cast<int64_t>((j0 + 8 * gr) & page_mask) * a.k_place;
#pragma unroll
                    for (int u = 0; u < 8 / kRowsPer; ++u) {
                        const int r = gr * 8 + u * kRowsPer;
                        const int j = j0 + r + lane / kChunks;
                        const bool ok = id >= 0 && (inside || (j < hi_max && (j >= lo_min || j < a.sinks)));
                        cp_async16(dst + r * T::kRowBytes + (((lane % kChunks) ^ ((u * kRowsPer + lane / kChunks) & 7)) << 4), kp, ok);
                        kp += kRowsPer * a.k_place;
                    }
                }
            }
            cp_async_commit();
            // a lane's places of a step's result are 32 u + lane of it; their old weights are fetched a step ahead
            float old[KT / 32];
            bool put[KT / 32];
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) {
                old[u] = old_next[u];
                put[u] = put_next[u];
                put_next[u] = false;
                if (i + 1 >= 0 && i + 1 < g.count) {
                    const int j = place_of(i + 1) + 32 * u + lane;
                    put_next[u] = j < hi_max && (j >= lo_min || j < a.sinks) && ((seen >> (NG + 4 * u + (lane >> 3))) & 1u);
                    if (put_next[u]) old_next[u] = wrow[j];
                }
            }
            if (i < 0) {
                seen >>= NG;
                continue;
            }
            const int j0 = place_of(i);
            cp_async_wait<kAhead>();
            __syncwarp();
            const uint32_t kst = ring + (i % T::kStages) * T::kStageBytes;
            const bool edge = j0 + KT > hi_min || lo_max > j0;
            float w[KT / 16][2];
#pragma unroll
            for (int m = 0; m < KT / 16; ++m) w[m][0] = w[m][1] = 0.f;
#pragma unroll 1
            for (int rt = 0; rt < row_tiles; ++rt) {
                if (row_tiles > 1) load_rows(rt * 8 * NT);
#pragma unroll
                for (int m = 0; m < KT / 16; ++m) {
                    float sc[NT][4];
#pragma unroll
                    for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[n2][e] = 0.f;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        uint32_t kf[4];
                        const int r = 16 * m + (lane & 15), c = 2 * kk + (lane >> 4);
                        ldmatrix_x4(kf, kst + r * T::kRowBytes + ((c ^ (r & 7)) << 4));
#pragma unroll
                        for (int n2 = 0; n2 < NT; ++n2) mma_16816<T::kBf16>(sc[n2], kf, qf[n2][kk][0], qf[n2][kk][1]);
                    }
#pragma unroll
                    for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float p = ex2_approx(fmaf(sc[n2][e], a.scale_log2, nl[n2][e & 1]));
                            bool see = true;
                            if (edge) {
                                const int j = j0 + 16 * m + (lane >> 2) + 8 * (e >> 1);
                                see = j < hi[n2][e & 1] && (j >= lo[n2][e & 1] || j < a.sinks);
                            }
                            w[m][e >> 1] += see ? p : 0.f;
                        }
                }
            }
            seen >>= NG;
            // sum over the columns (the four lanes of a row), then place 16 m + 8 e + r from lane 4 r to lane (16 m + 8 e + r) % 32
#pragma unroll
            for (int m = 0; m < KT / 16; ++m)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    w[m][e] += __shfl_xor_sync(0xffffffffu, w[m][e], 1);
                    w[m][e] += __shfl_xor_sync(0xffffffffu, w[m][e], 2);
                }
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float x = __shfl_sync(0xffffffffu, w[2 * u + (k >> 1)][k & 1], (lane & 7) * 4);
                    if ((lane >> 3) == k) v = x;
                }
                if (put[u]) wrow[j0 + 32 * u + lane] = old[u] + v;
            }
        }
        cp_async_wait<0>();
        __syncwarp();
        g = plan_next<U>(a, share, g);
    }
}

// ------------------------------------------------------------------------------------------------ chunk form
template <int kHeadDim_, typename elem_type>
struct PagedWeightsTraits : public Ring_kernel_traits<kHeadDim_, 256, 128, 12, elem_type> {
    using Base = Ring_kernel_traits<kHeadDim_, 256, 128, 12, elem_type>;
    static constexpr int kHeadDim = kHeadDim_;
    static constexpr int kNThreads = 384;
    static constexpr int kPlaces = 256;       // per unit: two tiles of 128 (TMEM lanes)
    static constexpr int kQRows = 128;        // query rows per block (columns of S^T)
    // warps 0-3 / 4-7: sums of place tile 0 / 1; 8, 9: UMMA issuers of tile 0 / 1; 10: lse and limits of the query rows; 11: TMA
    static constexpr int kMmaWarp = 8, kRowWarp = 10, kLoadWarp = 11;
    static constexpr int kSumRegs = 200, kProducerRegs = 104;
    static_assert(256 * kSumRegs + 128 * kProducerRegs <= 65536, "register file");
    static constexpr int kBoxes = kHeadDim / 64;
    static constexpr int kBoxBytes = 128 * 128;
    static constexpr int kTileBytes = kBoxes * kBoxBytes;     // 128 rows
    static constexpr int kKSlots = 2;                         // the next unit's places load while this one's are used
    static constexpr int kQSlots = kHeadDim == 128 ? 2 : 4;
    static constexpr int kSmemTiles = (2 * kKSlots + kQSlots) * kTileBytes;
    static constexpr int kRowInfo = 2 * kQRows * 4 + 16;      // negated lse (base 2) of each row, the same with 0 for NaN, a bit per NaN
    static constexpr int kPolyEvery = 8;                      // of 8 columns 2 are evaluated on the FMA pipe
    static constexpr int kInfoSlots = 4;                      // a ring of its own: read until a block's sums are done, long after its tile
    static constexpr int kNumBarriers = 2 * kKSlots + 2 * kQSlots + 4 /*s_full*/ + 4 /*s_free*/ + 2 * kInfoSlots;
    static constexpr int kSmemSize = kSmemTiles + kInfoSlots * kRowInfo + 1024 /*alignment slack*/ + 256 /*barriers, TMEM slot, flags*/;
    static_assert(kNumBarriers * 8 + 16 <= 256 && kSmemSize <= 226 * 1024, "shared memory");
};

// A unit is 256 places of one K/V head that some token sees; its blocks are the tiles of `row_tokens` tokens that see any of them.
struct WeightsChunkUnits {
    static __device__ __forceinline__ int tiles(const PagedArgs& a, const SeqView& s) { return s.n > 0 ? seen_tiles<256>(a, s).count : 0; }
    static __device__ __forceinline__ void range(const PagedArgs& a, const SeqView& s, int tile, int* j0, int* first, int* count) {
        *j0 = seen_tiles<256>(a, s).block(tile) * 256;
        int t0 = 0, t1 = s.n;
        if (a.causal) t0 = max(0, *j0 - s.pos);
        if (a.window > 0 && *j0 >= a.sinks)
            t1 = static_cast<int>(min(static_cast<int64_t>(s.n), static_cast<int64_t>(*j0) + 255 + a.window - s.pos));
        *first = div_tokens(a, min(t0, s.n - 1));
        *count = max(div_tokens(a, max(t1, 0) + a.row_tokens - 1) - *first, 1);
    }
    static __device__ __forceinline__ int blocks(const PagedArgs& a, const SeqView& s, int tile) {
        int j0, first, count;
        range(a, s, tile, &j0, &first, &count);
        return count;
    }
};

// Makes the scores of the rows (columns of S^T) whose bit is set NaN where they are, in TMEM.  By a warp, for its lanes; a call, so that
// the summing loop does not carry it (as a part of that loop it cost 7 us of 99).
__device__ __noinline__ void nan_scores(uint32_t t_s, float4 rows) {
    using namespace ptx;
#pragma unroll 1
    for (int w = 0; w < 4; ++w) {
        const uint32_t bits = __float_as_uint(w == 0 ? rows.x : (w == 1 ? rows.y : (w == 2 ? rows.z : rows.w)));
        uint32_t x[32];
        tmem_ld_x32(t_s + 32 * w, x);
        tmem_wait_ld();
#pragma unroll
        for (int v = 0; v < 32; ++v)
            if ((bits >> v) & 1u) x[v] = 0x7fffffffu;
        tmem_st_x32(t_s + 32 * w, x);
    }
    tmem_wait_st();
}

template <class T>
__global__ void __launch_bounds__(T::kNThreads, 1)
ring_paged_weights_chunk_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q, const PagedArgs a) {
    using namespace ptx;
    using U = WeightsChunkUnits;
    constexpr int D = T::kHeadDim;
    constexpr uint32_t kIdesc = umma_idesc_f16(128, T::kQRows, false, false, T::kIsBf16);
    extern __shared__ uint8_t smem_raw[];
    __shared__ PlanShared plan;
    const uint32_t raw_addr = smem_u32(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw_addr);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + T::kSmemTiles + T::kInfoSlots * T::kRowInfo);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + T::kNumBarriers);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* prior_error = reinterpret_cast<volatile int*>(tmem_slot + 2);
    const uint32_t bar0 = smem_u32(bars);
    auto bar_k_full = [&](int k) { return bar0 + 8u * k; };
    auto bar_k_empty = [&](int k) { return bar0 + 8u * (T::kKSlots + k); };
    auto bar_q_full = [&](int q) { return bar0 + 8u * (2 * T::kKSlots + q); };
    auto bar_q_empty = [&](int q) { return bar0 + 8u * (2 * T::kKSlots + T::kQSlots + q); };
    auto bar_s_full = [&](int m, int buf) { return bar0 + 8u * (2 * T::kKSlots + 2 * T::kQSlots + 2 * m + buf); };
    auto bar_s_free = [&](int m, int buf) { return bar0 + 8u * (2 * T::kKSlots + 2 * T::kQSlots + 4 + 2 * m + buf); };
    auto bar_i_full = [&](int q) { return bar0 + 8u * (2 * T::kKSlots + 2 * T::kQSlots + 8 + q); };
    auto bar_i_empty = [&](int q) { return bar0 + 8u * (2 * T::kKSlots + 2 * T::kQSlots + 8 + T::kInfoSlots + q); };
    auto smem_k = [&](int k, int m) { return base + static_cast<uint32_t>((2 * k + m) * T::kTileBytes); };
    auto smem_q = [&](int q) { return base + static_cast<uint32_t>((2 * T::kKSlots + q) * T::kTileBytes); };
    auto row_info = [&](int q) { return reinterpret_cast<float*>(smem + T::kSmemTiles + q * T::kRowInfo); };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cta = blockIdx.x;
    const int used_rows = a.row_tokens * a.group;  // rows of a query tile that hold (token, head) pairs
    griddep_launch();
    if (tid == 0) {
        *abort_flag = 0;
        for (int k = 0; k < T::kKSlots; ++k) {
            mbar_init(bar_k_full(k), 1);
            mbar_init(bar_k_empty(k), 2);       // both issuers
        }
        for (int q = 0; q < T::kQSlots; ++q) {
            mbar_init(bar_q_full(q), 1);
            mbar_init(bar_q_empty(q), 2);
        }
        for (int q = 0; q < T::kInfoSlots; ++q) {
            mbar_init(bar_i_full(q), 1);        // the row warp
            mbar_init(bar_i_empty(q), 8);       // the summing warps
        }
        for (int m = 0; m < 2; ++m)
            for (int buf = 0; buf < 2; ++buf) {
                mbar_init(bar_s_full(m, buf), 1);
                mbar_init(bar_s_free(m, buf), 4);
            }
        fence_mbar_init();
    }
    // rows of the query tiles that no load ever writes: zeros, so that their scores are finite (their exponentials are exp2(-inf))
    for (int i = tid; i < T::kQSlots * T::kBoxes * (T::kQRows - used_rows) * 8; i += T::kNThreads) {
        const int chunk = i & 7, row = used_rows + (i >> 3) % (T::kQRows - used_rows), box = (i >> 3) / (T::kQRows - used_rows);
        st_shared_v4(smem_q(0) + box * T::kBoxBytes + row * 128 + chunk * 16, 0u, 0u, 0u, 0u);
    }
    fence_proxy_async_cta();
    if (warp == T::kLoadWarp && lane == 0) {
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_q);
    }
    griddep_wait();  // nothing before this touches memory
    if (tid == 0) {
        *prior_error = *reinterpret_cast<volatile int*>(a.status);
        a.cut[2 * cta + 1] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    if (*prior_error != 0) return;  // an earlier launch failed: do nothing (CTA-uniform)
    Share share;
    Segment g = plan_start<U, T::kNThreads>(a, plan, share, cta, gridDim.x);
    if (!g.valid) return;  // no share (CTA-uniform)
    if (warp == T::kMmaWarp) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish_alloc_permit();
    }
    tcgen05_fence_before_thread_sync();
    __syncthreads();
    tcgen05_fence_after_thread_sync();
    const uint32_t tmem_base = *tmem_slot;

    // Every role walks the share on its own; what it has to count is the segments (K slots) and blocks (Q slots, S buffers) so far.
    uint32_t segs = 0, blocks = 0;
    bool ok = true;
    if (warp >= T::kMmaWarp) {
        setmaxnreg_dec<T::kProducerRegs>();
        if (warp == T::kLoadWarp) {
            const int piece = min(1 << a.page_shift, 128);  // places per box
            const int pieces = T::kPlaces / piece;          // 2 .. 32: one per lane
            for (; g.valid && ok; g = plan_next<U>(a, share, g), ++segs) {
                const SeqView s = seq_view(a, g.b);
                int j0, q_first, q_count;
                U::range(a, s, g.tile, &j0, &q_first, &q_count);
                const int ks = segs % T::kKSlots;
                int id = a.num_pages, in_page = 0;
                if (lane < pieces) {
                    const int j = j0 + lane * piece;
                    const int pg = j < token_hi(a, s, s.n - 1) ? page_of(a, g.b, j >> a.page_shift) : -1;
                    if (pg >= 0) id = pg;
                    in_page = j & ((1 << a.page_shift) - 1);
                }
                if (segs >= T::kKSlots) {
                    ok = mbar_wait(bar_k_empty(ks), (segs / T::kKSlots - 1) & 1, abort_flag, a.status, kDevPagedLoad);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                if (lane == 0) mbar_arrive_expect_tx(bar_k_full(ks), 2 * T::kTileBytes);
                __syncwarp();
                if (lane < pieces) {
                    const int row = lane * piece;
                    const uint32_t dst = smem_k(ks, row >> 7) + (row & 127) * 128;
#pragma unroll
                    for (int bx = 0; bx < T::kBoxes; ++bx) tma_load_4d(dst + bx * T::kBoxBytes, &tm_k, bar_k_full(ks), bx * 64, in_page, g.h, id);
                }
                __syncwarp();
                if (lane == 0) {
#pragma unroll 1
                    for (int i = 0; i < g.count; ++i) {
                        const uint32_t n = blocks + i;
                        const int q = n % T::kQSlots;
                        if (n >= T::kQSlots) {
                            ok = mbar_wait(bar_q_empty(q), (n / T::kQSlots - 1) & 1, abort_flag, a.status, kDevPagedLoad);
                            if (!ok) break;
                        }
                        mbar_arrive_expect_tx(bar_q_full(q), T::kBoxes * used_rows * 128);
                        const int tok = s.q0 + (q_first + g.first + i) * a.row_tokens;
#pragma unroll
                        for (int bx = 0; bx < T::kBoxes; ++bx) tma_load_4d(smem_q(q) + bx * T::kBoxBytes, &tm_q, bar_q_full(q), bx * 64, 0, g.h, tok);
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                blocks += g.count;
            }
        } else if (warp == T::kRowWarp) {
            for (; g.valid && ok; g = plan_next<U>(a, share, g), ++segs) {
                const SeqView s = seq_view(a, g.b);
                int j0, q_first, q_count;
                U::range(a, s, g.tile, &j0, &q_first, &q_count);
#pragma unroll 1
                for (int i = 0; i < g.count && ok; ++i, ++blocks) {
                    const int q = blocks % T::kInfoSlots;
                    const int t0 = (q_first + g.first + i) * a.row_tokens;
                    float nl[4];
                    uint32_t nan[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {  // the loads do not wait for the slot
                        const int r = lane + 32 * u, dt = div_group(a, r);
                        nl[u] = -INFINITY;  // rows that see nothing (lse = -inf) and rows behind the last add exp2(-inf) = 0
                        if (r < used_rows && t0 + dt < s.n) {
                            const float l = a.lse[static_cast<int64_t>(s.q0 + t0 + dt) * a.heads + g.h * a.group + (r - dt * a.group)];
                            if (l != -INFINITY) nl[u] = -l * 1.4426950408889634f;
                        }
                        nan[u] = __ballot_sync(0xffffffffu, nl[u] != nl[u]);
                    }
                    if (blocks >= T::kInfoSlots) {
                        ok = mbar_wait(bar_i_empty(q), (blocks / T::kInfoSlots - 1) & 1, abort_flag, a.status, kDevPagedLoad);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                    }
                    float* info = row_info(q);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        info[lane + 32 * u] = nl[u];
                        info[T::kQRows + lane + 32 * u] = nl[u] != nl[u] ? 0.f : nl[u];
                        if (lane == 0) reinterpret_cast<uint32_t*>(info + 2 * T::kQRows)[u] = nan[u];
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_i_full(q));
                }
            }
        } else {
            const int m = warp - T::kMmaWarp;
            for (; g.valid && ok; g = plan_next<U>(a, share, g), ++segs) {
                const int ks = segs % T::kKSlots;
                if (lane == 0) {
                    ok = mbar_wait(bar_k_full(ks), (segs / T::kKSlots) & 1, abort_flag, a.status, kDevPagedMmaKV);
#pragma unroll 1
                    for (int i = 0; i < g.count && ok; ++i) {
                        const uint32_t n = blocks + i;
                        const int q = n % T::kQSlots, buf = n & 1;
                        ok = mbar_wait(bar_q_full(q), (n / T::kQSlots) & 1, abort_flag, a.status, kDevPagedMmaQ);
                        if (ok && n >= 2) ok = mbar_wait(bar_s_free(m, buf), (n / 2 - 1) & 1, abort_flag, a.status, kDevPagedMmaS);
                        if (!ok) break;
                        tcgen05_fence_after_thread_sync();
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            const uint32_t off = (kk >> 2) * T::kBoxBytes + (kk & 3) * 32;
                            umma_ss(tmem_base + (2 * m + buf) * 128, umma_desc_kmajor_sw128(smem_k(ks, m) + off),
                                    umma_desc_kmajor_sw128(smem_q(q) + off), kIdesc, kk > 0 ? 1u : 0u);
                        }
                        umma_commit(bar_s_full(m, buf));
                        umma_commit(bar_q_empty(q));
                    }
                    if (ok) umma_commit(bar_k_empty(ks));
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                blocks += g.count;
            }
        }
    } else {
        setmaxnreg_inc<T::kSumRegs>();
        const int m = warp >> 2, quarter = warp & 3;
        const uint32_t t_s = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + 2 * m * 128;
        const float c = a.scale_log2;
        for (; g.valid && ok; g = plan_next<U>(a, share, g), ++segs) {
            const SeqView s = seq_view(a, g.b);
            int j0, q_first, q_count;
            U::range(a, s, g.tile, &j0, &q_first, &q_count);
            const int jt = j0 + m * 128;                  // first place of the tile
            const int j = jt + quarter * 32 + lane;       // this thread's place
            float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
            uint32_t sr[2][32];
            // Waits for block `blocks` (+ 1)'s row information and scores and sends for the first 32 columns.
            auto acquire = [&](uint32_t ahead = 0) {
                const uint32_t n = blocks + ahead;
                bool fine = mbar_wait(bar_i_full(n % T::kInfoSlots), (n / T::kInfoSlots) & 1, abort_flag, a.status, kDevPagedSoftmaxS) &&
                            mbar_wait(bar_s_full(m, n & 1), (n / 2) & 1, abort_flag, a.status, kDevPagedSoftmaxS);
                fine = __all_sync(0xffffffffu, fine);
                if (fine) {
                    tcgen05_fence_after_thread_sync();
                    tmem_ld_x32(t_s + (n & 1) * 128, sr[0]);
                }
                return fine;
            };
#pragma unroll 1
            for (int i = 0; i < g.count; ++i, ++blocks) {
                const int q = blocks % T::kInfoSlots, buf = blocks & 1;
                if (i == 0 && !(ok = acquire())) break;
                const int t0 = (q_first + g.first + i) * a.row_tokens, t1 = min(t0 + a.row_tokens, s.n);
                const bool edge = t0 + a.row_tokens > s.n || jt + 128 > token_hi(a, s, t0) ||
                                  (token_lo(a, s, t1 - 1) > jt && jt + 128 > a.sinks);
                uint32_t info = smem_u32(row_info(q));
                if (edge) {
                    const float4 nan = ld_shared_v4(info + 2 * T::kQRows * 4);
                    if ((__float_as_uint(nan.x) | __float_as_uint(nan.y) | __float_as_uint(nan.z) | __float_as_uint(nan.w)) != 0) {
                        tmem_wait_ld();
                        nan_scores(t_s + buf * 128, nan);
                        tmem_ld_x32(t_s + buf * 128, sr[0]);
                        info += T::kQRows * 4;
                    }
                }
                // The columns whose token sees this place are one interval: behind the first token at or after the place (causal),
                // before the first whose window has left it.
                int c0 = 0, c1 = 0;
                if (edge) {
                    const int back = j - s.pos - t0;  // the place as an index into the tile's tokens
                    c1 = min(t1 - t0, a.row_tokens);
                    if (a.causal) c0 = min(max(back, 0), a.row_tokens) * a.group;
                    if (a.window > 0 && j >= a.sinks)
                        c1 = static_cast<int>(min(static_cast<int64_t>(c1), max(static_cast<int64_t>(back) + a.window, int64_t(0))));
                    c1 = j < token_hi(a, s, s.n - 1) ? c1 * a.group : 0;
                }
                // 32 columns at a time, the next ones on their way while these are summed (64 at a time: 110 us at the size below, and 114
                // with the four parts rolled into a loop of two)
#pragma unroll
                for (int part = 0; part < 4; ++part) {
                    tmem_wait_ld();
                    if (part < 3) {
                        tmem_ld_x32(t_s + buf * 128 + 32 * (part + 1), sr[(part + 1) & 1]);
                    } else {
                        tcgen05_fence_before_thread_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar_s_free(m, buf));
                        // the next block's waits and first load under this block's last exponentials
                        if (i + 1 < g.count) ok = acquire(1);
                    }
                    float* sc = reinterpret_cast<float*>(sr[part & 1]);
                    if (edge) {  // scores that do not count become -inf: exp2 of them is 0 whatever they were
#pragma unroll
                        for (int v = 0; v < 32; ++v)
                            if (32 * part + v < c0 || 32 * part + v >= c1) sc[v] = -INFINITY;
                    }
#pragma unroll
                    for (int v = 0; v < 32; v += 4) {
                        const float4 nl = ld_shared_v4(info + 4 * (32 * part + v));
                        float x0, x1, x2, x3;
                        ffma2(x0, x1, sc[v], sc[v + 1], c, c, nl.x, nl.y);
                        ffma2(x2, x3, sc[v + 2], sc[v + 3], c, c, nl.z, nl.w);
                        if (v % T::kPolyEvery == 0)
                            ex2_poly2<true>(x0, x1, x0, x1);
                        else
                            x0 = ex2_approx(x0), x1 = ex2_approx(x1);
                        fadd2(a0, a1, a0, a1, x0, x1);
                        fadd2(a2, a3, a2, a3, ex2_approx(x2), ex2_approx(x3));
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_i_empty(q));
                if (!ok) break;
            }
            if (!ok) break;
            const float w = (a0 + a1) + (a2 + a3);
            const int slot = partial_slot(g, cta);
            if (slot >= 0) {
                a.part_lse[static_cast<int64_t>(slot) * T::kPlaces + m * 128 + quarter * 32 + lane] = w;
                if (slot == 2 * cta + 1 && tid == 0) note_cut(a, share, g, cta, j0, min(T::kPlaces, token_hi(a, s, s.n - 1) - j0), 0);
            } else if (j < token_hi(a, s, s.n - 1) && page_of(a, g.b, j >> a.page_shift) >= 0) {
                a.weights[static_cast<int64_t>(g.b) * a.w_batch + static_cast<int64_t>(g.h) * a.w_head + j] += w;
            }
        }
    }

    // ---- common exit: every thread arrives here, on success and on a timed-out wait alike
    tcgen05_fence_before_thread_sync();
    __syncthreads();
    if (warp == T::kMmaWarp) {
        tcgen05_fence_after_thread_sync();
        tmem_dealloc(tmem_base, 512);
    }
}

// Adds the partial sums of the units that share boundaries have cut, in the order of the shares.
__global__ void __launch_bounds__(256) ring_paged_weights_join_kernel(const PagedArgs a) {
    ptx::griddep_wait();
    if (*reinterpret_cast<volatile int*>(a.status) != 0) return;  // a wait ran out: the partials are not whole
    const int c = blockIdx.x;
    const int parts = a.cut[2 * c + 1].x;
    if (parts <= 1) return;
    const int4 u = a.cut[2 * c];
    if (static_cast<int>(threadIdx.x) >= u.w) return;
    const int j = u.z + threadIdx.x;
    if (page_of(a, u.x, j >> a.page_shift) < 0) return;
    float* to = a.weights + static_cast<int64_t>(u.x) * a.w_batch + static_cast<int64_t>(u.y) * a.w_head + j;
    float w = 0.f;
    for (int p = 0; p < parts; ++p) w += a.part_lse[static_cast<int64_t>(p == 0 ? 2 * c + 1 : 2 * (c + p)) * 256 + threadIdx.x];
    *to += w;
}

}  // namespace ring
