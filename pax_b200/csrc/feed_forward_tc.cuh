// feed_forward_tc.cuh -- the feed-forward products on tcgen05 (sm_100a).
//
// One persistent, warp-specialised kernel template for the products whose
// bases and row pitches are multiples of 16 bytes:
//
//   FF_GLU   H = act(X.Wg) * (X.Wu)              (G and U kept on request)
//   FF_BACK  dX = dG.Wg^T + dU.Wu^T and dWg = X^T.dG, dWu = X^T.dU in one
//            launch
//   FF_I8    C = (A.B^T) * sa * sb (+ bias), 8-bit integers
//
// A CTA pair (cluster of two, cta_group::2) computes accumulator tiles of 256
// rows and 256 or 512 columns; each CTA stages 128 rows of A and 128 or 256
// columns of B per 128-byte k-block (64 fp16 or 128 int8) in a ring and holds
// its 128 rows of the accumulators in TMEM (FfCfg).
//
// The gated product needs G and U of the same element in one thread.  The
// even CTA stages 128 columns of Wg and the odd CTA the same 128 columns of
// Wu, so one 256-wide MMA gives G in accumulator columns 0-127 and U in
// 128-255: the two projections cost exactly one GEMM of 2F columns and H
// leaves the epilogue without G and U touching memory.
//
// The backward products read their operands where they lie, without a
// transposing pass: a reduction along a matrix's rows (X^T.dG over tokens)
// stages both operands MN-major, one along the columns (dG.Wg^T over F)
// K-major.  dX runs its reduction over dG, Wg and then dU, Wu into one
// accumulator.
//
// Roles (320 threads): warp 0 TMA producer, warp 1 MMA issuer (even CTA),
// warps 2-9 epilogue, two per TMEM lane quarter.  Every wait is bounded
// (sm100.cuh); a CTA that gives up lets its loads land and its MMAs finish
// before it frees TMEM.
#pragma once

#include "activation.cuh"
#include "feed_forward.h"
#include "tmap.h"

#include <atomic>
#include <type_traits>

namespace pax {

enum : int { FF_GLU = 0, FF_BACK = 1, FF_I8 = 2 };

// Tensor maps by role.  FF_GLU: X, Wg, Wu, H, G, U.  FF_BACK: dG, dU, Wg, Wu
// as rows of a product (K-major), X, dG, dU by columns (MN-major), dX, dWg,
// dWu.  FF_I8: A, B in boxes of 128, 64 and 32 rows, C.
enum : int { MG_X = 0, MG_WG, MG_WU, MG_H, MG_G, MG_U };
enum : int { MB_DGK = 0, MB_DUK, MB_WGK, MB_WUK, MB_XN, MB_DGN, MB_DUN, MB_DX, MB_DWG, MB_DWU };
enum : int { MI_A = 0, MI_B, MI_B2, MI_B4, MI_C };
struct FfMaps {
    CUtensorMap m[10];
};

struct FfParams {
    int M, N;              // rows and columns of the output (FF_GLU: N = F; FF_BACK: see below)
    int tiles_m, tiles_n;  // output tiles (FF_BACK: of dX)
    int kbs;               // k-blocks of a tile (FF_BACK: of dX, both terms)
    int group_m;           // tiles run in column-major groups of group_m tile rows
    int full, pieces;      // FF_GLU, FF_I8: tiles [0, full) whole, the others in `pieces` column pieces
    int save;              // FF_GLU: store G and U
    // FF_BACK.  dX is M x D; the weight gradients D x F each, tiles wt_n wide
    // per matrix, both matrices side by side; kbs_w k-blocks of tokens.
    int D, F, nx, nw, wt_m, wt_n, kbs_w, half_kbs, accumulate;
    int x_rem, w_extra;    // schedule: see ff_item
    // FF_I8
    void* C;
    long long ldc;
    const float *sa, *sb;
    const __half* bias;
    int c_tma, c_unit;     // stores by TMA, or by units of 2, 4 or 8 bytes that C's rows are aligned to
};

struct FfItem {
    int kind;  // 0 the product (FF_BACK: dX), 1 a weight gradient
    int mb, nb, kbs;
    int w;     // accumulator columns of one MMA
    int col;   // FF_GLU, FF_I8: first output column
};

__host__ __device__ __forceinline__ void ff_tile(int t, int tiles_m, int tiles_n, int group_m, int& mb, int& nb) {
    const int per_group = group_m * tiles_n;
    const int g = t / per_group, first = g * group_m;
    const int gm = tiles_m - first < group_m ? tiles_m - first : group_m;
    const int r = t - g * per_group;
    mb = first + r % gm;
    nb = r / gm;
}

// The idx-th tile of pair `unit` of `units`; false when there is none.
// Round-robin, so that the pairs work on neighbouring tiles at a time.
// FF_GLU and FF_I8: the tiles beyond the last full round can run in column
// pieces, so that the last round takes less than a whole tile's time.
// FF_BACK: dX's nx tiles first.  Where they do not divide by the pairs,
// x_rem pairs have one more, which is worth w_extra weight-gradient tiles;
// the other pairs start with that many rounds of those.
template <int MODE, int W>
__host__ __device__ __forceinline__ bool ff_item(const FfParams& p, int unit, int units, int idx, FfItem& it) {
    it.w = 256;
    if constexpr (MODE != FF_BACK) {
        int t = unit + idx * units, piece = 0;
        if (t >= p.full) {
            const int j = t - p.full;
            t = p.full + j / p.pieces;
            piece = j % p.pieces;
            it.w = 256 / p.pieces;
        }
        if (t >= p.tiles_m * p.tiles_n) return false;
        it.kind = 0;
        ff_tile(t, p.tiles_m, p.tiles_n, p.group_m, it.mb, it.nb);
        const int cols = MODE == FF_GLU ? it.w / 2 : it.w;  // of a piece; the wide tile has no pieces
        it.col = it.nb * (MODE == FF_GLU ? 128 : 256) * W + piece * cols;
        it.kbs = it.col < p.N ? p.kbs : 0;  // nothing of a piece beyond the last column
        return true;
    } else {
        const int q = p.nx / units, mine = q + (unit < p.x_rem ? 1 : 0);
        if (idx < mine) {
            it.kind = 0;
            it.kbs = p.kbs;
            ff_tile(unit + idx * units, p.tiles_m, p.tiles_n, p.group_m, it.mb, it.nb);
            return true;
        }
        int j = idx - mine, t;
        const int others = units - p.x_rem;
        if (unit >= p.x_rem && j < p.w_extra) {
            t = (unit - p.x_rem) + j * others;
        } else {
            if (unit >= p.x_rem) j -= p.w_extra;
            t = p.w_extra * others + unit + j * units;
        }
        if (t >= p.nw) return false;
        it.kind = 1;
        it.kbs = p.kbs_w;
        ff_tile(t, p.wt_m, 2 * p.wt_n, p.group_m, it.mb, it.nb);
        return true;
    }
}

// Tile widths.  W = 1: 256 accumulator columns a tile, two accumulators in
// TMEM, so that a tile's epilogue runs under the next one's main loop.
// W = 2: 512 columns as two MMAs per k-step that share A, one accumulator in
// all of TMEM.  It stages 48 KB for twice the MMAs instead of 2 x 32 KB, and
// shared-memory traffic is what bounds the main loop, but its epilogue is
// exposed.
//
// The 8-bit product (W = 1 only) gives one slot of its ring to tables of
// scales and bias in shared memory, one per epilogue warp: read from global
// memory in the epilogue they took longer than a main loop of K = 2048.
template <int MODE, int W>
struct FfCfg {
    static constexpr int STAGES = W == 2 ? 4 : MODE == FF_I8 ? 5 : 6;
    static constexpr uint32_t OP_BYTES = 128 * 128;         // 128 rows or columns, 128 bytes of k
    static constexpr uint32_t A_BYTES = OP_BYTES, B_BYTES = W * OP_BYTES;
    static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int ACCS = W == 2 ? 1 : 2;             // accumulators in TMEM
    static constexpr int EPI_WARPS = 8;
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr uint32_t STG_BYTES = 32 * 128;         // staging, per epilogue warp
    static constexpr uint32_t TAB_BYTES = MODE == FF_I8 ? 2 * 128 * 4 : 0;  // per epilogue warp
    static constexpr uint32_t NUM_BARS = 2 * STAGES + 6;    // full, empty, tfull[2], tempty[2], drain, report
    static constexpr size_t SMEM_BYTES = 1024 + (size_t)STAGES * STAGE_BYTES +
                                         EPI_WARPS * (STG_BYTES + TAB_BYTES) + NUM_BARS * 8 + 16;
    static_assert(MODE != FF_I8 || W == 1, "the tables need the room of a slot");
    static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

// Columns of a w-wide 8-bit item that each of the two warps of a lane quarter
// takes: half of them, or all with the first warp where half is less than a
// 128-byte row of the output.
template <typename OutT>
__device__ __forceinline__ int ff_i8_span(int w) {
    constexpr int row = 128 / (int)sizeof(OutT);
    return w / 2 >= row ? w / 2 : row;
}

// Bytes that one CTA stages per k-block of an item.
template <int W>
__device__ __forceinline__ uint32_t ff_stage_bytes(const FfItem& it) {
    return 16384u + (uint32_t)(W * (it.w / 2) * 128);
}

// Stores staged rows (128B swizzle, 128 bytes each) by a warp in UNIT-byte
// pieces, four stores in flight: `cols` columns of `rows` rows.  Bounded by the
// number of stores, so the unit is the largest that the rows are aligned to:
// 7579 x 1634 x 752 with FP16 out takes 21.9 us (28.1 by one element a store),
// 1235 x 4100 x 2064 18.0 us (20.7), and 4099 odd columns 20.0 us.
template <int UNIT, typename OutT>
__device__ __forceinline__ void ff_store_units(const uint8_t* sbuf, OutT* to, long long ld, int cols, int rows,
                                               int lane) {
    using V = typename std::conditional<UNIT == 8, uint2, typename std::conditional<UNIT == 4, uint32_t, uint16_t>::type>::type;
    constexpr int PER_ROW = 128 / UNIT, ELEMS = UNIT / (int)sizeof(OutT);
    const int bytes = cols * (int)sizeof(OutT);
#pragma unroll 1
    for (int u0 = 0; u0 < rows * PER_ROW; u0 += 4 * 32) {
        V v[4];
        OutT* at[4];
        int here[4];  // bytes of the unit that are inside
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = u0 + 32 * i + lane, r = u / PER_ROW, byte = u % PER_ROW * UNIT;
            here[i] = r < rows ? bytes - byte : 0;
            v[i] = *reinterpret_cast<const V*>(sbuf + (r & 31) * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15));
            at[i] = to + (long long)r * ld + byte / (int)sizeof(OutT);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (here[i] >= UNIT) {
                *reinterpret_cast<V*>(at[i]) = v[i];
            } else if (here[i] > 0) {  // the row ends inside the unit
                const OutT* e = reinterpret_cast<const OutT*>(&v[i]);
#pragma unroll
                for (int j = 0; j < ELEMS - 1; ++j)
                    if ((j + 1) * (int)sizeof(OutT) <= here[i]) at[i][j] = e[j];
            }
        }
    }
}
template <typename OutT>
__device__ __forceinline__ void ff_store_rows(const uint8_t* sbuf, OutT* to, long long ld, int cols, int rows, int unit,
                                              int lane) {
    if (unit == 8)
        ff_store_units<8>(sbuf, to, ld, cols, rows, lane);
    else if (unit == 4)
        ff_store_units<4>(sbuf, to, ld, cols, rows, lane);
    else if constexpr (sizeof(OutT) == 2)
        ff_store_units<2>(sbuf, to, ld, cols, rows, lane);
}

template <int MODE, int ACT, typename OutT, int W>
__global__ void __launch_bounds__(FfCfg<MODE, W>::THREADS, 1)
    ff_tc_kernel(const __grid_constant__ FfMaps maps, const __grid_constant__ FfParams p) {
    using Cfg = FfCfg<MODE, W>;
    constexpr int STAGES = Cfg::STAGES;
    constexpr int KB = MODE == FF_I8 ? 128 : 64;  // elements of a k-block
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem =
        reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + STAGES * Cfg::A_BYTES;
    uint8_t* sStg = sB + STAGES * Cfg::B_BYTES;
    float* sTab = reinterpret_cast<float*>(sStg + Cfg::EPI_WARPS * Cfg::STG_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sStg + Cfg::EPI_WARPS * (Cfg::STG_BYTES + Cfg::TAB_BYTES));
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NUM_BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile uint32_t* issued_slot = tmem_slot + 2;  // the odd CTA's k-block count

    const uint32_t full0 = smem_u32(bars);
    const uint32_t empty0 = full0 + 8u * STAGES;
    const uint32_t tfull0 = empty0 + 8u * STAGES;
    const uint32_t tempty0 = tfull0 + 16u;
    const uint32_t drain_bar = tempty0 + 16u;
    const uint32_t report_bar = drain_bar + 8u;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int unit = (int)(blockIdx.x >> 1), units = (int)(gridDim.x >> 1);
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full0 + 8u * s, 1);
            mbar_init(empty0 + 8u * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull0 + 8u * b, 1);
            mbar_init(tempty0 + 8u * b, 2 * Cfg::EPI_WARPS);  // the epilogue warps of both CTAs
        }
        mbar_init(drain_bar, 1);
        mbar_init(report_bar, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 2 && lane < (MODE == FF_BACK ? 10 : MODE == FF_I8 ? 5 : 6)) tma_prefetch_desc(&maps.m[lane]);
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(tmem_slot), 512);
        tmem_relinquish<2>();
    }
    tc_fence_before();
    cluster_sync();  // barrier initialisation visible to the peer CTA
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            pdl_wait();  // the operands may be written by the previous grid
            // Not before: what the next grid loads early (weights) is known not
            // to be written by this grid, but may be by the one before it, and
            // glu_dx_skinny relies on dG and dU being written.
            pdl_launch_dependents();
            int stage = 0, total = 0;
            uint32_t phase = 0;
            bool ok = true;
            FfItem it;
            for (int idx = 0; ok && ff_item<MODE, W>(p, unit, units, idx, it); ++idx) {
                const int row = it.mb * 256 + (int)rank * 128;
                // First column of this CTA's share of B, and from one MMA's
                // columns to the next one's.
                const int col = MODE == FF_GLU ? it.col
                                : MODE == FF_I8 ? it.col + (int)rank * (it.w / 2)
                                                : it.nb * 256 * W + (int)rank * 128;
                const uint32_t bytes = ff_stage_bytes<W>(it);
                const CUtensorMap* m_b = MODE == FF_GLU   ? &maps.m[leader ? MG_WG : MG_WU]
                                         : MODE == FF_I8 ? &maps.m[it.w == 256 ? MI_B : it.w == 128 ? MI_B2 : MI_B4]
                                                         : nullptr;
                const int boxes = it.w / 128 * W;  // FF_GLU: 64-column boxes
                constexpr int next = 256;
                for (int kb = 0; kb < it.kbs; ++kb) {
                    if (!mbar_wait(empty0 + 8u * stage, phase ^ 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = mapa_shared(full0 + 8u * stage, 0);
                    const uint32_t a = smem_u32(sA + stage * Cfg::A_BYTES), b = smem_u32(sB + stage * Cfg::B_BYTES);
                    // Both CTAs' loads complete on the even CTA's barrier.
                    if (leader) mbar_arrive_expect_tx(full0 + 8u * stage, 2 * bytes);
                    const int k = kb * KB;
                    if constexpr (MODE == FF_GLU) {
                        tma_load_3d_pair(a, &maps.m[MG_X], fb, k, row, 0);
#pragma unroll
                        for (int h = 0; h < 2 * W; ++h)
                            if (h < boxes) tma_load_3d_pair(b + h * 8192, m_b, fb, col + 64 * h, k, 0);
                    } else if constexpr (MODE == FF_I8) {
                        tma_load_3d_pair(a, &maps.m[MI_A], fb, k, row, 0);
                        tma_load_3d_pair(b, m_b, fb, k, col, 0);
                    } else if (it.kind == 0) {
                        const bool up = kb >= p.half_kbs;
                        const int kk = up ? k - p.half_kbs * KB : k;
                        tma_load_3d_pair(a, &maps.m[up ? MB_DUK : MB_DGK], fb, kk, row, 0);
#pragma unroll
                        for (int h = 0; h < W; ++h)
                            tma_load_3d_pair(b + h * Cfg::OP_BYTES, &maps.m[up ? MB_WUK : MB_WGK], fb, kk,
                                             col + next * h, 0);
                    } else {
                        const bool up = it.nb >= p.wt_n;
                        const CUtensorMap* v = &maps.m[up ? MB_DUN : MB_DGN];
                        const int c = up ? col - p.wt_n * 256 * W : col;
                        tma_load_3d_pair(a, &maps.m[MB_XN], fb, row, k, 0);
                        tma_load_3d_pair(a + 8192, &maps.m[MB_XN], fb, row + 64, k, 0);
#pragma unroll
                        for (int h = 0; h < W; ++h) {
                            tma_load_3d_pair(b + h * Cfg::OP_BYTES, v, fb, c + next * h, k, 0);
                            tma_load_3d_pair(b + h * Cfg::OP_BYTES + 8192, v, fb, c + next * h + 64, k, 0);
                        }
                    }
                    ++total;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // Every load either CTA issued must land before the pair tears
            // down; all of them complete on the even CTA's full barriers.  The
            // odd CTA reports how many k-blocks it issued, and the even CTA
            // settles the last phase of every slot: one that only one CTA
            // contributed to is completed for the other (its bytes cancelled,
            // or the phase armed for the odd CTA's bytes alone), then waited
            // for.  Both issue the same k-block sequence, gated by the same
            // slot releases, so neither is more than a ring ahead.  After a
            // normal run every phase is complete already.
            if (!leader) {
                st_shared_cluster_u32(smem_u32((const void*)issued_slot), 0, (uint32_t)total);
                mbar_arrive_cluster(report_bar, 0);
            } else {
                bool reported = mbar_wait<true>(report_bar, 0, nullptr);
                if (!reported) reported = mbar_wait<true>(report_bar, 0, nullptr);
                const int theirs = reported ? (int)*issued_slot : total;
                const int most = total > theirs ? total : theirs;
                for (int s = 0; s < STAGES && s < most; ++s) {
                    const int i = s + ((most - 1 - s) / STAGES) * STAGES;  // last k-block on slot s
                    if ((i < total) != (i < theirs)) {
                        int left = i;  // the item that k-block i belongs to
                        for (int idx = 0; ff_item<MODE, W>(p, unit, units, idx, it) && left >= it.kbs; ++idx)
                            left -= it.kbs;
                        if (i < total)
                            mbar_complete_tx(full0 + 8u * s, ff_stage_bytes<W>(it));
                        else
                            mbar_arrive_expect_tx(full0 + 8u * s, ff_stage_bytes<W>(it));
                    }
                    mbar_wait(full0 + 8u * s, (uint32_t)(i / STAGES) & 1u, nullptr);
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        if (lane == 0 && leader) {
            // The waits below count from here: for the loads of this grid, not
            // for the end of the previous one.
            pdl_wait();
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            // Descriptors of slot 0; others differ in the start address
            // (address >> 4 in the low bits).  A k-step is 32 bytes along a
            // K-major row, 16 rows of 128 bytes in an MN-major operand.
            const uint64_t aK = umma_desc_sw128(smem_u32(sA), 16, 1024), aN = umma_desc_sw128(smem_u32(sA), 8192, 1024);
            const uint64_t bK = umma_desc_sw128(smem_u32(sB), 16, 1024), bN = umma_desc_sw128(smem_u32(sB), 8192, 1024);
            FfItem it;
            for (int idx = 0; ok && ff_item<MODE, W>(p, unit, units, idx, it); ++idx) {
                const bool a_n = MODE == FF_BACK && it.kind == 1;
                const bool b_n = MODE == FF_GLU || a_n;
                const uint64_t a0 = a_n ? aN : aK, b0 = b_n ? bN : bK;
                const uint64_t a_step = a_n ? 128 : 2, b_step = b_n ? 128 : 2;
                const uint32_t id = MODE == FF_I8 ? umma_idesc_i8(256, it.w) : umma_idesc_f16(256, it.w, a_n, b_n);
                if (it.kbs == 0) continue;
                // Releases come from both CTAs' epilogues.
                if (!mbar_wait<true>(tempty0 + 8u * acc, acc_phase ^ 1u, abort_flag)) break;
                tc_fence_after();
                const uint32_t d = tmem_base + (uint32_t)(acc * 256 * W);
                for (int kb = 0; kb < it.kbs; ++kb) {
                    if (!mbar_wait(full0 + 8u * stage, phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    uint64_t ad = a0 + (uint64_t)((stage * Cfg::A_BYTES) >> 4);
                    uint64_t bd = b0 + (uint64_t)((stage * Cfg::B_BYTES) >> 4);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint32_t more = (kb | kk) != 0 ? 1u : 0u;
#pragma unroll
                        for (int h = 0; h < W; ++h) {
                            const uint64_t bh = bd + (uint64_t)(h * (Cfg::OP_BYTES >> 4));
                            if constexpr (MODE == FF_I8)
                                tc_mma_i8_pair(d + 256u * h, ad, bh, id, more);
                            else
                                tc_mma_f16_pair(d + 256u * h, ad, bh, id, more);
                        }
                        ad += a_step;
                        bd += b_step;
                    }
                    tc_commit_pair(mapa_shared(empty0 + 8u * stage, 0));
                    tc_commit_pair(mapa_shared(empty0 + 8u * stage, 1));
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                tc_commit_pair(mapa_shared(tfull0 + 8u * acc, 0));
                tc_commit_pair(mapa_shared(tfull0 + 8u * acc, 1));
                if (++acc == Cfg::ACCS) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            // No MMA may still write TMEM or read either CTA's shared memory
            // when the pair tears down.
            tc_commit_pair(mapa_shared(drain_bar, 0));
            mbar_wait(drain_bar, 0, nullptr);
        }
    } else {
        // ------------------------------------------------ epilogue warps
        pdl_wait();  // outputs and scales may belong to the previous grid
        const int q = warp & 3;          // TMEM lane quarter this warp may read
        const int wh = (warp - 2) >> 2;  // which half of the tile's columns
        uint8_t* sbuf = sStg + (warp - 2) * Cfg::STG_BYTES;
        const uint32_t srow = smem_u32(sbuf) + (uint32_t)lane * 128u;
        // One 128-byte row per lane into the staging buffer (128B swizzle:
        // 16-byte chunk j of row r lies at j ^ (r % 8)), once its last TMA
        // store has read it.
        auto stage_rows = [&](const uint32_t (&w)[32]) {
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j)
                st_shared_v4(srow + (uint32_t)((j ^ (lane & 7)) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2],
                             w[4 * j + 3]);
        };
        auto store = [&](const CUtensorMap* m, const uint32_t (&w)[32], int col, int row, bool add) {
            stage_rows(w);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (add)
                    tma_reduce_add_3d(m, smem_u32(sbuf), col, row, 0);
                else
                    tma_store_3d(m, smem_u32(sbuf), col, row, 0);
                bulk_commit();
            }
        };
        int acc = 0;
        uint32_t acc_phase = 0;
        FfItem it;
        for (int idx = 0; ff_item<MODE, W>(p, unit, units, idx, it); ++idx) {
            if (it.kbs == 0) continue;
            const int row0 = it.mb * 256 + (int)rank * 128 + q * 32;
            float* tab = sTab + (warp - 2) * 256;  // this warp's 128 scales, then its 128 bias values
            float sa = 0.f;
            if constexpr (MODE == FF_I8) {
                if (row0 + lane < p.M) sa = __ldg(p.sa + row0 + lane);
                const int span = ff_i8_span<OutT>(it.w), c0 = it.col + wh * span + lane;
#pragma unroll
                for (int i = 0; i < 128; i += 32) {
                    const int c = c0 + i;
                    const bool in = i < span && c < p.N;
                    tab[lane + i] = in ? __ldg(p.sb + c) : 0.f;
                    tab[128 + lane + i] = in && p.bias ? __half2float(p.bias[c]) : 0.f;
                }
                __syncwarp();
            }
            bool ok = mbar_wait(tfull0 + 8u * acc, acc_phase, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * 256 * W);
            auto release = [&]() {  // the accumulator is read: back to the MMA warp
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (leader)
                        mbar_arrive(tempty0 + 8u * acc);
                    else
                        mbar_arrive_cluster(tempty0 + 8u * acc, 0);
                }
            };
            if constexpr (MODE == FF_GLU) {
                // 64 columns of H per warp and MMA: G beside U
                // (half a tile: all of them with the first warp).
                const int here = p.N - it.col - wh * 64;
                const int chunks = row0 >= p.M || (it.w < 256 && wh == 1) ? 0 : min(W, max(0, (here + 127) / 128));
                if (chunks == 0) release();
#pragma unroll 1
                for (int n = 0; n < chunks; ++n) {
                    const int col = it.col + n * 128 + wh * 64;
                    const uint32_t t_gu = t_row + (uint32_t)(n * 256 + wh * 64);
                    uint32_t wH[32], wG[32], wU[32];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float g[32], u[32];
                        tmem_ld_32x32b_x32(t_gu + (uint32_t)(32 * h), g);
                        tmem_ld_32x32b_x32(t_gu + (uint32_t)(it.w / 2 + 32 * h), u);
                        tmem_wait_ld();
                        if (h == 1 && n == chunks - 1) release();
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            wG[16 * h + i] = pack_half2(g[2 * i], g[2 * i + 1]);
                            wU[16 * h + i] = pack_half2(u[2 * i], u[2 * i + 1]);
                            const float2 a = act_value2<ACT>(make_float2(g[2 * i], g[2 * i + 1]));
                            wH[16 * h + i] = pack_half2(a.x * u[2 * i], a.y * u[2 * i + 1]);
                        }
                    }
                    store(&maps.m[MG_H], wH, col, row0, false);
                    if (p.save) {
                        store(&maps.m[MG_G], wG, col, row0, false);
                        store(&maps.m[MG_U], wU, col, row0, false);
                    }
                }
            } else {
                // Half of the columns per warp (128 W of whole tiles), in chunks
                // of one 128-byte row a lane.
                const bool f16 = sizeof(OutT) == 2 || (MODE == FF_BACK && it.kind == 0);
                const bool up = MODE == FF_BACK && it.kind == 1 && it.nb >= p.wt_n;
                const int rows = MODE == FF_BACK ? (it.kind == 0 ? p.M : p.D) : p.M;
                const int cols = MODE == FF_BACK ? (it.kind == 0 ? p.D : p.F) : p.N;
                const int span = MODE == FF_I8 ? ff_i8_span<OutT>(it.w) : 128 * W;
                const int base = MODE == FF_I8 ? it.col : (up ? it.nb - p.wt_n : it.nb) * 256 * W;
                const int tcol = base + wh * span;
                const int valid = row0 < rows && wh * span < it.w * W ? min(span, cols - tcol) : 0;
                const int nsub = valid > 0 ? (valid + 31) / 32 : 0;  // 32-column parts that hold anything
                const CUtensorMap* m = MODE == FF_I8 ? &maps.m[MI_C]
                                                     : &maps.m[it.kind == 0 ? MB_DX : up ? MB_DWU : MB_DWG];
                const bool add = MODE == FF_BACK && it.kind == 1 && p.accumulate;
                if (nsub == 0) release();
                uint32_t w[32];
#pragma unroll 1
                for (int s = 0; s < nsub; ++s) {
                    float v[32];
                    tmem_ld_32x32b_x32(t_row + (uint32_t)(wh * span + 32 * s), v);
                    tmem_wait_ld();
                    if (s == nsub - 1) release();
                    const int col = tcol + 32 * s;
                    if constexpr (MODE == FF_I8) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 c = *reinterpret_cast<const float4*>(tab + 32 * s + i);
                            v[i] = (float)__float_as_int(v[i]) * sa * c.x;
                            v[i + 1] = (float)__float_as_int(v[i + 1]) * sa * c.y;
                            v[i + 2] = (float)__float_as_int(v[i + 2]) * sa * c.z;
                            v[i + 3] = (float)__float_as_int(v[i + 3]) * sa * c.w;
                        }
                        if (p.bias) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 b = *reinterpret_cast<const float4*>(tab + 128 + 32 * s + i);
                                v[i] += b.x;
                                v[i + 1] += b.y;
                                v[i + 2] += b.z;
                                v[i + 3] += b.w;
                            }
                        }
                    }
                    if (f16) {
                        // two 32-column parts make a 128-byte row
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const uint32_t h2 = pack_half2(v[2 * i], v[2 * i + 1]);
                            if (s & 1)
                                w[16 + i] = h2;
                            else
                                w[i] = h2;
                        }
                        if (!(s & 1) && s != nsub - 1) continue;
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
                    }
                    const int ccol = f16 ? tcol + 32 * (s & ~1) : col;
                    if (MODE != FF_I8 || p.c_tma) {
                        store(m, w, ccol, row0, add);
                    } else {
                        // Rows of C that TMA cannot store.
                        stage_rows(w);
                        __syncwarp();
                        OutT* to = static_cast<OutT*>(p.C) + (long long)row0 * p.ldc + ccol;
                        ff_store_rows(sbuf, to, p.ldc, min(128 / (int)sizeof(OutT), p.N - ccol), min(32, p.M - row0),
                                      p.c_unit, lane);
                        __syncwarp();
                    }
                }
            }
            if constexpr (MODE == FF_I8) __syncwarp();  // the table is read
            if (++acc == Cfg::ACCS) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        if (lane == 0) bulk_wait<0>();
        __syncwarp();
    }

    __syncwarp();
    tc_fence_before();
    cluster_sync();  // neither CTA leaves while the pair's MMAs or arrivals may touch it
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<2>(tmem_base, 512);
    }
}

// ======================================================================
// Host side
// ======================================================================

// Allow the kernel its shared memory on the current device: per device and
// context, and cheap to repeat.
template <int MODE, int ACT, typename OutT, int W>
inline bool ff_shared() {
    return cudaFuncSetAttribute(ff_tc_kernel<MODE, ACT, OutT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)FfCfg<MODE, W>::SMEM_BYTES) == cudaSuccess;
}

// CTA pairs of the kernel that device `dev` holds at once (SMs pair up
// within a GPC, so this can be below SMs / 2); asked once per device and
// kernel.
template <int MODE, int ACT, typename OutT, int W>
inline int ff_units(int dev) {
    static std::atomic<int> cache[64];  // zero; calls may come from several threads
    std::atomic<int>& v = cache[dev & 63];
    if (v == 0) {
        auto kern = ff_tc_kernel<MODE, ACT, OutT, W>;
        if (!ff_shared<MODE, ACT, OutT, W>()) return 0;
        const int sms = device_sm_count(dev);
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.blockDim = dim3(FfCfg<MODE, W>::THREADS);
        cfg.dynamicSmemBytes = FfCfg<MODE, W>::SMEM_BYTES;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(sms & ~1);
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = sms / 2;
        }
        v = n;
    }
    return v;
}

template <int MODE, int ACT, typename OutT, int W>
inline pax_status_t ff_launch(const FfMaps& maps, const FfParams& p, int units, cudaStream_t stream) {
    if (!ff_shared<MODE, ACT, OutT, W>()) return PAX_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(2 * units);
    cfg.blockDim = dim3(FfCfg<MODE, W>::THREADS);
    cfg.dynamicSmemBytes = FfCfg<MODE, W>::SMEM_BYTES;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, ff_tc_kernel<MODE, ACT, OutT, W>, maps, p) == cudaSuccess ? PAX_OK : PAX_ERR_CUDA;
}

}  // namespace pax
