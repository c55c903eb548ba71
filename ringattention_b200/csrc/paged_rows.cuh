// Paged attention for few query rows (decoding, drafted tokens): bound by reading the cache.
//
// A unit is up to 16 * MT query rows (new tokens x query heads of one K/V head) of one sequence.  Each warp walks its own
// share of the unit's places, KT at a time, through its own ring of shared-memory stages filled by cp.async (16 bytes a
// lane, places a sequence cannot see are filled with zeros and never read), so the main loop has no CTA-wide
// barrier.  S = Q K^T and O += P V are mma.sync m16n8k16: the arithmetic (4 D per row and place, rows padded to
// 16) is a small part of what the legacy tensor path does in the time the places take from HBM, and its 16-row tile
// fits these row counts where a 128-row tcgen05 tile would be mostly padding.  Running maximum, sum and O stay in registers (fp32);
// P is rounded to the inputs' type for the product (by at most 2^-8 of it for bf16, 2^-11 for fp16; the sum l takes the
// unrounded values).  The warps' partials are joined in shared memory at the end of a unit.
//
// Measured: 30 sequences of 300 to 8192 places, 8 K/V heads, group 4, D = 128, bf16, pages of 16: 93 us, 5.9 TB/s, 0.90 of the
// measured copy rate; 2 x 131072 places, 2 K/V heads, group 8: 47 us of reading (5.7 TB/s) + 8 us of joining 74 partials a unit.  Two
// CTAs of four warps an SM, three stages of 8 KiB a warp: 128 KiB on their way per SM.  Page ids
// come 32 groups of 8 places at a time, one batch ahead: loaded step by step they put a second latency before every unit's first rows.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "paged_plan.cuh"
#include "ptx_sm100.cuh"

namespace ring {

namespace ptx {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    const uint32_t n = valid ? 16u : 0u;  // 0: nothing is read, 16 zero bytes are written
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kBf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    return kBf16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}
__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace ptx

template <int D_, bool kBf16_, int MT_>
struct PagedRowsTraits {
    static constexpr int D = D_;
    static constexpr bool kBf16 = kBf16_;
    static constexpr int MT = MT_;
    static constexpr int kRows = 16 * MT;
    static constexpr int kWarps = 4, kThreads = 128;
    static constexpr int BN = 64;                    // places per block of the plan
    static constexpr int KT = D == 128 ? 16 : 32;    // places per step of a warp: 4 KiB of K and of V
    static constexpr int kSteps = BN / KT;           // steps per block
    static constexpr int kStages = 3;
    static constexpr int kRowBytes = D * 2;
    static constexpr int kHalf = KT * kRowBytes;     // K or V of a step
    static constexpr int kStageBytes = 2 * kHalf;    // 8 KiB
    static constexpr int kRing = kStages * kStageBytes;
    static constexpr int kMerge = kWarps * kRows * (D + 4) * 4 + kWarps * kRows * 8;  // joins the warps; overlays the rings
    static constexpr int kSmem = (kWarps * kRing > kMerge ? kWarps * kRing : kMerge);
};

template <class T>
__global__ void __launch_bounds__(T::kThreads) ring_paged_rows_kernel(const PagedArgs a) {
    using namespace ptx;
    using U = AttentionUnits<T::BN>;
    constexpr int D = T::D, MT = T::MT, KT = T::KT;
    constexpr int kChunks = T::kRowBytes / 16;       // 16-byte chunks per row
    constexpr int kRowsPer = 32 / kChunks;           // rows one warp-wide cp.async covers
    constexpr int kLoads = KT / kRowsPer;            // ... per K or V of a step (8)
    constexpr int NG = KT / 8;                       // groups of 8 places (a page holds whole groups)
    constexpr int kBatch = 32 / NG;                  // steps whose page ids one warp-wide load fetches
    constexpr int kAhead = T::kStages - 1;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PlanShared plan;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cta = blockIdx.x;
    griddep_wait();    // nothing before this may touch memory
    griddep_launch();  // the joining kernel may take its place; it waits for this grid's end before it reads
    Share share;
    Segment g = plan_start<U, T::kThreads>(a, plan, share, cta, gridDim.x);
    if (tid == 0) a.cut[2 * cta + 1] = make_int4(0, 0, 0, 0);

    const uint32_t ring = smem_u32(smem) + warp * T::kRing;
    const int page_mask = (1 << a.page_shift) - 1;
    // Steps of this warp: warp, warp + 4, ... of the segment's, KT places each.  D = 128: sub-block `warp` of block i; D = 64:
    // half warp & 1 of block 2 i + (warp >> 1).
    auto steps_of = [&](const Segment& sg) { return (sg.count * T::kSteps - warp + T::kWarps - 1) / T::kWarps; };
    auto place_of = [&](const Segment& sg, const TileBlocks& tb, int i) {
        const int st = warp + i * T::kWarps;
        return tb.block(sg.first + st / T::kSteps) * T::BN + (st % T::kSteps) * KT;
    };
    // Page ids of steps [kBatch * n, kBatch * (n + 1)): lane l has group l % NG of step l / NG, -1 where there is none.
    auto load_pages = [&](const Segment& sg, const TileBlocks& tb, int n) {
        const int i = n * kBatch + lane / NG;
        if (i >= steps_of(sg)) return -1;
        return page_of(a, sg.b, (place_of(sg, tb, i) + 8 * (lane % NG)) >> a.page_shift);
    };
    SeqView s;
    TileBlocks tb;
    int ids = -1;
    if (g.valid) {
        s = seq_view(a, g.b);
        tb = tile_blocks<T::BN>(a, s, g.tile * T::kRows, tile_rows(a, s, g.tile));
        ids = load_pages(g, tb, 0);
    }
    while (g.valid) {
        const int row0 = g.tile * T::kRows;
        const int rows = tile_rows(a, s, g.tile);
        const int tok_first = div_group(a, row0), tok_last = div_group(a, row0 + rows - 1);
        const int hi_max = token_hi(a, s, tok_last), hi_min = token_hi(a, s, tok_first);
        const int lo_min = token_lo(a, s, tok_first), lo_max = token_lo(a, s, tok_last);

        // ---- Q fragments and the limits of this lane's rows (lane / 4 and + 8 of each 16-row tile)
        uint32_t qf[MT][D / 16][4];
        int hi[MT][2], lo[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint16_t* qp[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 16 * m + 8 * r + (lane >> 2);
                const int at = row0 + min(row, rows - 1);
                const int tok = div_group(a, at);
                qp[r] = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(s.q0 + tok) * a.q_token +
                        static_cast<int64_t>(g.h * a.group + (at - tok * a.group)) * a.q_head + 2 * (lane & 3);
                hi[m][r] = row < rows ? token_hi(a, s, tok) : 0;
                lo[m][r] = token_lo(a, s, tok);
            }
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    qf[m][kk][r] = *reinterpret_cast<const uint32_t*>(qp[r] + 16 * kk);
                    qf[m][kk][2 + r] = *reinterpret_cast<const uint32_t*>(qp[r] + 16 * kk + 8);
                }
            }
        }

        float o[MT][D / 8][4];
        float m_run[MT][2], l_run[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][i][e] = 0.f;
            m_run[m][0] = m_run[m][1] = -INFINITY;
            l_run[m][0] = l_run[m][1] = 0.f;
        }

        const int mine = steps_of(g);
        // this lane's part of every K and V address
        const uint16_t* kl = static_cast<const uint16_t*>(a.k) + static_cast<int64_t>(g.h) * a.k_head + (lane % kChunks) * 8 + (lane / kChunks) * a.k_place;
        const uint16_t* vl = static_cast<const uint16_t*>(a.v) + static_cast<int64_t>(g.h) * a.v_head + (lane % kChunks) * 8 + (lane / kChunks) * a.v_place;
        int ids_next = -1;
        uint32_t have = 0;       // bit l: lane l's id of the current batch exists
        uint32_t seen = 0;       // NG bits per stage, the step being computed lowest: its groups' pages exist
        // The loop runs kAhead steps early to fill the ring: one copy of the code, and of its instruction fetches.
#pragma unroll 1
        for (int i = -kAhead; i < mine; ++i) {
            const int n = i + kAhead;
            if (n < mine) {
                if (n % kBatch == 0) {
                    if (n > 0) ids = ids_next;
                    ids_next = load_pages(g, tb, n / kBatch + 1);
                    have = __ballot_sync(0xffffffffu, ids >= 0);
                }
                const int j0 = place_of(g, tb, n);
                const uint32_t bits = (have >> ((n % kBatch) * NG)) & ((1u << NG) - 1u);
                seen |= bits << (kAhead * NG);
                const bool inside = j0 + KT <= hi_max && (j0 >= lo_min || j0 + KT <= a.sinks);
                const uint32_t dst = ring + (n % T::kStages) * T::kStageBytes + (lane / kChunks) * T::kRowBytes;
                __syncwarp();  // every lane is done with the stage
#pragma unroll
                for (int gr = 0; gr < NG; ++gr) {
                    const int id = __shfl_sync(0xffffffffu, ids, (n % kBatch) * NG + gr);
                    const int64_t pg = id >= 0 ? id : 0;
                    const int slot = (j0 + 8 * gr) & page_mask;
                    const uint16_t* kp = kl + pg * a.k_page + static_cast<int64_t>(slot) * a.k_place;
                    const uint16_t* vp = vl + pg * a.v_page + static_cast<int64_t>(slot) * a.v_place;
#pragma unroll
                    for (int u = 0; u < 8 / kRowsPer; ++u) {
                        const int r = gr * 8 + u * kRowsPer;  // + lane / kChunks
                        const int j = j0 + r + lane / kChunks;
                        const bool ok = id >= 0 && (inside || (j < hi_max && (j >= lo_min || j < a.sinks)));
                        const uint32_t to = dst + r * T::kRowBytes + (((lane % kChunks) ^ ((u * kRowsPer + lane / kChunks) & 7)) << 4);
                        cp_async16(to, kp, ok);
                        cp_async16(to + T::kHalf, vp, ok);
                        kp += kRowsPer * a.k_place;
                        vp += kRowsPer * a.v_place;
                    }
                }
            }
            cp_async_commit();
            if (i < 0) {
                seen >>= NG;
                continue;
            }
            cp_async_wait<kAhead>();
            __syncwarp();
            const uint32_t kst = ring + (i % T::kStages) * T::kStageBytes;
            const uint32_t vst = kst + T::kHalf;
            const int j0 = place_of(g, tb, i);

            // S = Q K^T: KT / 8 fragments of 16 rows x 8 places
            float sc[MT][NG][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[m][n][e] = 0.f;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
                for (int n = 0; n < NG; n += 2) {
                    uint32_t kf[4];  // (places 8n.., k lo), (same, k hi), (places 8(n+1).., k lo), (same, k hi)
                    const int r = 8 * n + (lane & 7) + ((lane >> 4) << 3);
                    const int ch = 2 * kk + ((lane >> 3) & 1);
                    ldmatrix_x4(kf, kst + r * T::kRowBytes + ((ch ^ (r & 7)) << 4));
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        mma_16816<T::kBf16>(sc[m][n], qf[m][kk], kf[0], kf[1]);
                        mma_16816<T::kBf16>(sc[m][n + 1], qf[m][kk], kf[2], kf[3]);
                    }
                }
            }

            const bool edge = j0 + KT > hi_min || lo_max > j0 || (seen & ((1u << NG) - 1u)) != (1u << NG) - 1u;
            if (edge) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < NG; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = j0 + 8 * n + 2 * (lane & 3) + (e & 1);
                            const bool see = j < hi[m][e >> 1] && (j >= lo[m][e >> 1] || j < a.sinks) && ((seen >> n) & 1u);
                            if (!see) sc[m][n][e] = -INFINITY;
                        }
            }
            seen >>= NG;

            uint32_t pf[MT][NG][2];  // P as A fragments
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float top[2] = {sc[m][0][0], sc[m][0][2]};
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    top[0] = fmaxf(top[0], fmaxf(sc[m][n][0], sc[m][n][1]));
                    top[1] = fmaxf(top[1], fmaxf(sc[m][n][2], sc[m][n][3]));
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                }
                const bool grow = top[0] > m_run[m][0] || top[1] > m_run[m][1];
                if (__any_sync(0xffffffffu, grow)) {
                    float alpha[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float mx = fmaxf(m_run[m][r], top[r]);
                        alpha[r] = m_run[m][r] == -INFINITY ? 0.f : ex2_approx((m_run[m][r] - mx) * a.scale_log2);
                        if (mx == m_run[m][r]) alpha[r] = 1.f;
                        m_run[m][r] = mx;
                        l_run[m][r] *= alpha[r];
                    }
#pragma unroll
                    for (int d = 0; d < D / 8; ++d) {
                        o[m][d][0] *= alpha[0];
                        o[m][d][1] *= alpha[0];
                        o[m][d][2] *= alpha[1];
                        o[m][d][3] *= alpha[1];
                    }
                }
                float nm[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) nm[r] = m_run[m][r] == -INFINITY ? 0.f : -m_run[m][r] * a.scale_log2;
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = ex2_approx(fmaf(sc[m][n][e], a.scale_log2, nm[e >> 1]));
                    l_run[m][0] += p[0] + p[1];
                    l_run[m][1] += p[2] + p[3];
                    pf[m][n][0] = pack16<T::kBf16>(p[0], p[1]);
                    pf[m][n][1] = pack16<T::kBf16>(p[2], p[3]);
                }
            }

            // O += P V
#pragma unroll
            for (int n = 0; n < NG; n += 2) {
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    uint32_t vf[4];  // (places lo, d lo), (places hi, d lo), (places lo, d hi), (places hi, d hi)
                    const int r = 8 * n + (lane & 15);
                    const int ch = 2 * d + (lane >> 4);
                    ldmatrix_x4_trans(vf, vst + r * T::kRowBytes + ((ch ^ (r & 7)) << 4));
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint32_t af[4] = {pf[m][n][0], pf[m][n][1], pf[m][n + 1][0], pf[m][n + 1][1]};
                        mma_16816<T::kBf16>(o[m][2 * d], af, vf[0], vf[1]);
                        mma_16816<T::kBf16>(o[m][2 * d + 1], af, vf[2], vf[3]);
                    }
                }
            }
        }
        // the next segment's lookups travel while this one's warps are joined
        const Segment g_next = plan_next<U>(a, share, g);
        SeqView s_next = s;
        TileBlocks tb_next = tb;
        if (g_next.valid) {
            if (g_next.b != g.b) s_next = seq_view(a, g_next.b);
            tb_next = tile_blocks<T::BN>(a, s_next, g_next.tile * T::kRows, tile_rows(a, s_next, g_next.tile));
            ids = load_pages(g_next, tb_next, 0);
        }
        cp_async_wait<0>();
        __syncthreads();  // every warp is done with its ring: the join overlays them

        // ---- join the four warps: O and (m, l) of each through shared memory
        float* jo = reinterpret_cast<float*>(smem);                     // [warp][row][D + 4]
        float* jm = jo + T::kWarps * T::kRows * (D + 4);                // [warp][row][2]
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                l_run[m][r] += __shfl_xor_sync(0xffffffffu, l_run[m][r], 1);
                l_run[m][r] += __shfl_xor_sync(0xffffffffu, l_run[m][r], 2);
                const int row = 16 * m + 8 * r + (lane >> 2);
                float* to = jo + (warp * T::kRows + row) * (D + 4) + 2 * (lane & 3);
#pragma unroll
                for (int d = 0; d < D / 8; ++d)
                    *reinterpret_cast<float2*>(to + 8 * d) = make_float2(o[m][d][2 * r], o[m][d][2 * r + 1]);
                if ((lane & 3) == 0) {
                    jm[2 * (warp * T::kRows + row)] = m_run[m][r];
                    jm[2 * (warp * T::kRows + row) + 1] = l_run[m][r];
                }
            }
        }
        __syncthreads();
        const int slot = partial_slot(g, cta);
        constexpr int kLanes = D / 4;  // threads per row, four columns each
        for (int row = tid / kLanes; row < rows; row += T::kThreads / kLanes) {
            const int col = (tid % kLanes) * 4;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < T::kWarps; ++w) mx = fmaxf(mx, jm[2 * (w * T::kRows + row)]);
            float l = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < T::kWarps; ++w) {
                const float mw = jm[2 * (w * T::kRows + row)];
                const float f = mw == mx ? 1.f : ex2_approx((mw - mx) * a.scale_log2);
                l = fmaf(jm[2 * (w * T::kRows + row) + 1], f, l);
                const float4 v = *reinterpret_cast<const float4*>(jo + (w * T::kRows + row) * (D + 4) + col);
                acc.x = fmaf(v.x, f, acc.x);
                acc.y = fmaf(v.y, f, acc.y);
                acc.z = fmaf(v.z, f, acc.z);
                acc.w = fmaf(v.w, f, acc.w);
            }
            const bool have = l > 0.f || l != l;  // a NaN score stays visible in the result
            const float inv = have ? 1.f / l : 0.f;
            const float lse = have ? mx * a.scale + logf(l) : -INFINITY;
            acc.x *= inv;
            acc.y *= inv;
            acc.z *= inv;
            acc.w *= inv;
            if (slot >= 0) {
                const int64_t at = static_cast<int64_t>(slot) * T::kRows + row;
                *reinterpret_cast<float4*>(a.part_o + at * D + col) = acc;
                if (col == 0) a.part_lse[at] = lse;
            } else {
                const int r = row0 + row, tok = div_group(a, r);
                const int64_t token = s.q0 + tok;
                const int head = g.h * a.group + (r - tok * a.group);
                const int64_t at = token * a.out_token + head * a.out_head + col;
                if (a.out_fp32) {
                    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = acc;
                } else {
                    const uint2 v = make_uint2(pack16<T::kBf16>(acc.x, acc.y), pack16<T::kBf16>(acc.z, acc.w));
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = v;
                }
                if (col == 0) a.lse[token * a.heads + head] = lse;
            }
        }
        if (slot == 2 * cta + 1 && tid == 0) note_cut(a, share, g, cta, row0, rows, s.q0);
        g = g_next;
        s = s_next;
        tb = tb_next;
        if (g.valid) __syncthreads();  // the join's memory becomes rings again
    }
}

// Joins the partials of the units that share boundaries have cut: CTA (c, y) takes rows of the unit that begins in share c.
// out = sum_p exp(lse_p - lse) out_p with lse over all partials first, so that no load waits on another one's value.
// Bound by latency, so everything that can be in flight is: units of few partials take four rows a warp with all their loads at
// once; others (long sequences: tens of shares a unit) give the partials of one row to kSplit warps.
template <int D, bool kBf16, int kSplit>
__global__ void __launch_bounds__(32 * (kSplit > 4 ? kSplit : 4)) ring_paged_join_kernel(const PagedArgs a, int unit_rows) {
    using namespace ptx;
    constexpr int kWarps = kSplit > 4 ? kSplit : 4;
    __shared__ float4 sm_o[kWarps][32];
    griddep_wait();
    const int c = blockIdx.x;
    const int4 u = a.cut[2 * c], more = a.cut[2 * c + 1];
    if (a.status && *reinterpret_cast<volatile int*>(a.status) != 0) return;  // a wait ran out: the partials are not whole
    const int parts = more.x;
    if (parts <= 1) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kLanes = D / 4;          // lanes per row
    constexpr int kSub = 32 / kLanes;      // rows, or partials of one, a warp reads at once
    const int sub = lane / kLanes, col = (lane % kLanes) * 4;
    auto at = [&](int p, int row) { return static_cast<int64_t>(p == 0 ? 2 * c + 1 : 2 * (c + p)) * unit_rows + row; };
    auto put = [&](int row, const float4& v, float lse) {
        const int r = u.z + row, tok = div_group(a, r);
        const int64_t token = more.y + tok;
        const int head = u.y * a.group + (r - tok * a.group);
        const int64_t to = token * a.out_token + head * a.out_head + col;
        if (a.out_fp32)
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + to) = v;
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + to) = make_uint2(pack16<kBf16>(v.x, v.y), pack16<kBf16>(v.z, v.w));
        if (col == 0) a.lse[token * a.heads + head] = lse;
    };
    auto add = [](float4& acc, const float4& v, float w) {
        acc.x = fmaf(v.x, w, acc.x);
        acc.y = fmaf(v.y, w, acc.y);
        acc.z = fmaf(v.z, w, acc.z);
        acc.w = fmaf(v.w, w, acc.w);
    };
    if (parts <= 4) {
        constexpr int kR = 4;  // rows of a lane
        for (int r0 = (blockIdx.y * kWarps + warp) * kR * kSub; r0 < u.w; r0 += gridDim.y * kWarps * kR * kSub) {
            float e[kR][4];
            float4 v[kR][4];
#pragma unroll
            for (int k = 0; k < kR; ++k) {
                const int row = min(r0 + k * kSub + sub, u.w - 1);
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    e[k][p] = -INFINITY;
                    v[k][p] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (p < parts) {  // the same for all threads
                        e[k][p] = a.part_lse[at(p, row)];
                        v[k][p] = *reinterpret_cast<const float4*>(a.part_o + at(p, row) * D + col);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kR; ++k) {
                const int row = r0 + k * kSub + sub;
                const float mx = fmaxf(fmaxf(e[k][0], e[k][1]), fmaxf(e[k][2], e[k][3]));
                float l = 0.f;
#pragma unroll
                for (int p = 0; p < 4; ++p) l += e[k][p] == -INFINITY ? 0.f : expf(e[k][p] - mx);
                const float lse = (l > 0.f || l != l) ? (mx == -INFINITY ? 0.f : mx) + logf(l) : -INFINITY;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int p = 0; p < 4; ++p) add(acc, v[k][p], e[k][p] == -INFINITY ? 0.f : expf(e[k][p] - lse));
                if (row < u.w) put(row, acc, lse);
            }
        }
        return;
    }
    constexpr int kRowsAtOnce = kWarps / kSplit;
    constexpr int kPieces = kSplit * kSub;
    const int piece = (warp % kSplit) * kSub + sub;
    for (int r0 = blockIdx.y * kRowsAtOnce; r0 < u.w; r0 += gridDim.y * kRowsAtOnce) {
        const int row = r0 + warp / kSplit;
        const bool live = row < u.w;
        float lse = -INFINITY;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live) {
            float mx = -INFINITY, l = 0.f;
            for (int p0 = lane; p0 < parts; p0 += 128) {
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) e[k] = p0 + 32 * k < parts ? a.part_lse[at(p0 + 32 * k, row)] : -INFINITY;
                const float m2 = fmaxf(fmaxf(fmaxf(mx, e[0]), fmaxf(e[1], e[2])), e[3]);
                l = mx == m2 ? l : l * expf(mx - m2);
#pragma unroll
                for (int k = 0; k < 4; ++k) l += e[k] == -INFINITY ? 0.f : expf(e[k] - m2);
                mx = m2;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const float m1 = __shfl_xor_sync(0xffffffffu, mx, o), l1 = __shfl_xor_sync(0xffffffffu, l, o);
                const float m2 = fmaxf(mx, m1);
                l = (mx == m2 ? l : l * expf(mx - m2)) + (m1 == m2 ? l1 : l1 * expf(m1 - m2));
                mx = m2;
            }
            if (l > 0.f || l != l) lse = (mx == -INFINITY ? 0.f : mx) + logf(l);
#pragma unroll 8
            for (int p = piece; p < parts; p += kPieces) {
                const float e = a.part_lse[at(p, row)];
                const float4 v = *reinterpret_cast<const float4*>(a.part_o + at(p, row) * D + col);
                add(acc, v, e == -INFINITY ? 0.f : expf(e - lse));
            }
        }
        if (kPieces > 1) {
            sm_o[warp][lane] = acc;
            __syncthreads();
            if (live && piece == 0) {
                for (int p = 1; p < kPieces; ++p) add(acc, sm_o[warp + p / kSub][(p % kSub) * kLanes + lane], 1.f);
            }
            __syncthreads();
        }
        if (live && piece == 0) put(row, acc, lse);
    }
}

}  // namespace ring
