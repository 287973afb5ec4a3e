// feed_forward_split.cu -- the feed-forward products with few output tiles
// and long sums, on tcgen05: each tile's K shared by a cluster.
//
// A product whose output is a handful of 256-column tiles (the input gradient
// of a narrow model, the weight gradients of a small layer over many tokens,
// a narrow projection) leaves most SMs idle on feed_forward_tc.cuh's kernel,
// while each tile works through hundreds of k-blocks.  Here a cluster of 2 S
// CTAs, S = 2 or 4 CTA pairs, computes one tile of 256 rows x 256 accumulator
// columns: pair j takes k-blocks j, j + S, ...  The partial accumulators meet
// in distributed shared memory: the rows of a tile half are dealt out among
// the S CTAs that hold them, every CTA stores its partial sums of another's
// rows straight into that CTA's (by then idle) ring, and each adds the S
// contributions of its rows in pair order, applies the epilogue and stores.
// No workspace, no atomics, the same bits every time.
//
// Operands are staged as there: Wg by the even CTA of a pair and Wu by the
// odd one for the gated product, MN-major where a sum runs down the rows.
// 320 threads: warp 0 TMA producer, warp 1 MMA issuer (even CTA of each
// pair), warps 2-9 epilogue.  Every wait is bounded (sm100.cuh).
#include "feed_forward_tc.cuh"

namespace pax {

namespace {

enum : int { SP_GLU = 0, SP_I8 = 1, SP_DX = 2, SP_DW = 3 };

// SP_GLU: X, Wg, Wu, H, G, U.  SP_I8: A, B, C.  SP_DX: dG, dU, Wg, Wu, dX.
// SP_DW: X, dG, dU, dWg, dWu.
struct SpMaps {
    CUtensorMap m[6];
};

struct SpParams {
    int M, N;              // rows and columns of the output (SP_GLU: of H; SP_DW: of one matrix)
    int tiles_m, tiles_n;  // SP_DW: of one matrix
    int kbs, half;         // k-blocks; SP_DX: of the first term
    int save, accumulate;
    void* C;               // SP_I8
    long long ldc;
    const float *sa, *sb;
    const __half* bias;
    int c_tma, c_unit;
};

struct SpCfg {
    static constexpr int STAGES = 6;
    static constexpr uint32_t OP_BYTES = 128 * 128, STAGE_BYTES = 2 * OP_BYTES;
    static constexpr int EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;
    static constexpr uint32_t STG_BYTES = 32 * 128;
    static constexpr uint32_t NUM_BARS = 2 * STAGES + 3;  // full, empty, done, drain, report
    static constexpr size_t SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + EPI_WARPS * STG_BYTES + NUM_BARS * 8 + 16;
    static_assert(SMEM_BYTES <= 232448, "shared memory budget");
    static_assert(128 * 256 * 4 <= STAGES * STAGE_BYTES, "the ring holds the contributions");
};

template <int MODE, int ACT, typename OutT>
__global__ void __launch_bounds__(SpCfg::THREADS, 1)
    ff_split_kernel(const __grid_constant__ SpMaps maps, const __grid_constant__ SpParams p) {
    using Cfg = SpCfg;
    constexpr int STAGES = Cfg::STAGES;
    constexpr int KB = MODE == SP_I8 ? 128 : 64;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem =
        reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + STAGES * Cfg::OP_BYTES;
    uint8_t* sStg = sB + STAGES * Cfg::OP_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sStg + Cfg::EPI_WARPS * Cfg::STG_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NUM_BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile uint32_t* issued_slot = tmem_slot + 2;  // the odd CTA's k-block count

    const uint32_t full0 = smem_u32(bars);
    const uint32_t empty0 = full0 + 8u * STAGES;
    const uint32_t done_bar = empty0 + 8u * STAGES;  // the pair's accumulator is complete
    const uint32_t drain_bar = done_bar + 8u;
    const uint32_t report_bar = drain_bar + 8u;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int csize;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    const uint32_t crank = cluster_ctarank(), even = crank & ~1u;
    const int S = csize >> 1, pair = (int)(crank >> 1), rank = (int)(crank & 1u);
    const bool leader = rank == 0;
    const int tile = (int)blockIdx.x / csize;
    const int mb = tile % p.tiles_m, nbt = tile / p.tiles_m;
    const bool second = MODE == SP_DW && nbt >= p.tiles_n;  // dWu
    const int nb = second ? nbt - p.tiles_n : nbt;
    const int row = mb * 256 + rank * 128;                                          // this CTA's rows of A
    const int col = MODE == SP_GLU ? nb * 128 : nb * 256 + rank * 128;              // its columns of B

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full0 + 8u * s, 1);
            mbar_init(empty0 + 8u * s, 1);
        }
        mbar_init(done_bar, 1);
        mbar_init(drain_bar, 1);
        mbar_init(report_bar, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(tmem_slot), 256);
        tmem_relinquish<2>();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            pdl_wait();  // the operands may be written by the previous grid
            pdl_launch_dependents();  // not before, as in ff_tc_kernel
            int stage = 0, total = 0;
            uint32_t phase = 0;
            for (int kb = pair; kb < p.kbs; kb += S) {
                if (!mbar_wait(empty0 + 8u * stage, phase ^ 1u, abort_flag)) break;
                const uint32_t fb = mapa_shared(full0 + 8u * stage, even);
                const uint32_t a = smem_u32(sA + stage * Cfg::OP_BYTES), b = smem_u32(sB + stage * Cfg::OP_BYTES);
                if (leader) mbar_arrive_expect_tx(full0 + 8u * stage, 2 * Cfg::STAGE_BYTES);
                const int k = kb * KB;
                if constexpr (MODE == SP_GLU) {
                    const CUtensorMap* w = &maps.m[leader ? 1 : 2];
                    tma_load_3d_pair(a, &maps.m[0], fb, k, row, 0);
                    tma_load_3d_pair(b, w, fb, col, k, 0);
                    tma_load_3d_pair(b + 8192, w, fb, col + 64, k, 0);
                } else if constexpr (MODE == SP_I8) {
                    tma_load_3d_pair(a, &maps.m[0], fb, k, row, 0);
                    tma_load_3d_pair(b, &maps.m[1], fb, k, col, 0);
                } else if constexpr (MODE == SP_DX) {
                    const bool up = kb >= p.half;
                    const int kk = up ? k - p.half * KB : k;
                    tma_load_3d_pair(a, &maps.m[up ? 1 : 0], fb, kk, row, 0);
                    tma_load_3d_pair(b, &maps.m[up ? 3 : 2], fb, kk, col, 0);
                } else {
                    const CUtensorMap* v = &maps.m[second ? 2 : 1];
                    tma_load_3d_pair(a, &maps.m[0], fb, row, k, 0);
                    tma_load_3d_pair(a + 8192, &maps.m[0], fb, row + 64, k, 0);
                    tma_load_3d_pair(b, v, fb, col, k, 0);
                    tma_load_3d_pair(b + 8192, v, fb, col + 64, k, 0);
                }
                ++total;
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            // Every load of the pair must land before the ring is reused: as
            // in ff_tc_kernel, the even CTA settles the last phase of every
            // slot, of which only one CTA may have contributed after an abort.
            if (!leader) {
                st_shared_cluster_u32(smem_u32((const void*)issued_slot), even, (uint32_t)total);
                mbar_arrive_cluster(report_bar, even);
            } else {
                bool reported = mbar_wait<true>(report_bar, 0, nullptr);
                if (!reported) reported = mbar_wait<true>(report_bar, 0, nullptr);
                const int theirs = reported ? (int)*issued_slot : total;
                const int most = total > theirs ? total : theirs;
                for (int s = 0; s < STAGES && s < most; ++s) {
                    const int i = s + ((most - 1 - s) / STAGES) * STAGES;  // last k-block on slot s
                    if (i < total && i >= theirs) mbar_complete_tx(full0 + 8u * s, Cfg::STAGE_BYTES);
                    if (i >= total && i < theirs) mbar_arrive_expect_tx(full0 + 8u * s, Cfg::STAGE_BYTES);
                    mbar_wait(full0 + 8u * s, (uint32_t)(i / STAGES) & 1u, nullptr);
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        if (lane == 0 && leader) {
            pdl_wait();  // the waits below count from the previous grid's end
            constexpr bool a_n = MODE == SP_DW, b_n = MODE == SP_GLU || MODE == SP_DW;
            const uint64_t a0 = umma_desc_sw128(smem_u32(sA), a_n ? 8192 : 16, 1024);
            const uint64_t b0 = umma_desc_sw128(smem_u32(sB), b_n ? 8192 : 16, 1024);
            constexpr uint32_t id = MODE == SP_I8 ? umma_idesc_i8(256, 256) : umma_idesc_f16(256, 256, a_n, b_n);
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = pair; kb < p.kbs; kb += S) {
                if (!mbar_wait(full0 + 8u * stage, phase, abort_flag)) break;
                tc_fence_after();
                const uint64_t ad = a0 + (uint64_t)((stage * Cfg::OP_BYTES) >> 4);
                const uint64_t bd = b0 + (uint64_t)((stage * Cfg::OP_BYTES) >> 4);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint32_t more = (kb != pair || kk != 0) ? 1u : 0u;
                    const uint64_t ak = ad + (uint64_t)(kk * (a_n ? 128 : 2)), bk = bd + (uint64_t)(kk * (b_n ? 128 : 2));
                    if constexpr (MODE == SP_I8)
                        tc_mma_i8_pair(tmem_base, ak, bk, id, more);
                    else
                        tc_mma_f16_pair(tmem_base, ak, bk, id, more);
                }
                tc_commit_pair(mapa_shared(empty0 + 8u * stage, even));
                tc_commit_pair(mapa_shared(empty0 + 8u * stage, even + 1));
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            tc_commit_pair(mapa_shared(done_bar, even));
            tc_commit_pair(mapa_shared(done_bar, even + 1));
            tc_commit_pair(mapa_shared(drain_bar, even));
            mbar_wait(drain_bar, 0, nullptr);
        }
    } else {
        pdl_wait();  // outputs and scales may belong to the previous grid
        // The pair's MMAs end within their own bounded waits; a sum of many
        // k-blocks may take longer than an abandonable wait should.
        mbar_wait<true>(done_bar, 0, nullptr);
        tc_fence_after();
    }

    // ------------------------------------------------ reduction
    __syncwarp();
    cluster_sync();  // every ring is idle: its loads and MMAs are done
    const int R = 128 / S;  // rows of this half of the tile that each CTA finishes
    if (warp >= 2) {
        // Accumulator row q * 32 + lane, columns of half wh, to the CTA that
        // finishes the row: [pair][column / 4][row of its R][column % 4], so that
        // the lanes of a warp write 512 bytes in a row.
        const int q = warp & 3, wh = (warp - 2) >> 2;
        const int r = q * 32, dest = r / R;
        const uint32_t at = (uint32_t)((pair * 64 + wh * 32) * R + r - dest * R + lane) * 16u;
        const uint32_t to = mapa_shared(smem_u32(smem) + at, (uint32_t)(2 * dest + rank));
        const uint32_t src = tmem_base + ((uint32_t)r << 16) + (uint32_t)(wh * 128);
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
            float v[32];
            tmem_ld_32x32b_x32(src + (uint32_t)c, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 4) st_shared_cluster_v4(to + (uint32_t)((c + i) / 4 * R * 16), v + i);
        }
        tc_fence_before();
    }
    __syncwarp();
    cluster_sync();  // the contributions are in; nothing remote happens after this
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<2>(tmem_base, 256);
    }
    if (warp < 2 || *abort_flag) return;

    // ------------------------------------------------ epilogue
    // Units of 32 rows x one 128-byte row of the output, one warp each.
    constexpr int EC = 128 / (int)sizeof(OutT), COLS = MODE == SP_GLU ? 128 : 256;
    uint8_t* sbuf = sStg + (warp - 2) * Cfg::STG_BYTES;
    const float4* recv = reinterpret_cast<const float4*>(smem);
    const int cols = p.N, c_base = nb * COLS;
    for (int unit = warp - 2; unit < (R / 32) * (COLS / EC); unit += Cfg::EPI_WARPS) {
        const int rg = unit / (COLS / EC), c0 = (unit - rg * (COLS / EC)) * EC;  // row group, first column in the tile
        const int row0 = mb * 256 + rank * 128 + pair * R + rg * 32;
        const int ccol = c_base + c0;
        if (row0 >= p.M || ccol >= cols) continue;
        const float4* mine = recv + rg * 32 + lane;
        // 8 accumulator columns of this lane's row, summed in pair order.
        auto sum8 = [&](int c, float (&v)[8]) {
            const float4 a = mine[c / 4 * R], b = mine[(c / 4 + 1) * R];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
#pragma unroll 1
            for (int s = 1; s < S; ++s) {
                const float4 d = mine[(s * 64 + c / 4) * R], e = mine[(s * 64 + c / 4 + 1) * R];
                const float y[8] = {d.x, d.y, d.z, d.w, e.x, e.y, e.z, e.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (MODE == SP_I8)
                        v[i] = __int_as_float(__float_as_int(v[i]) + __float_as_int(y[i]));
                    else
                        v[i] += y[i];
                }
            }
        };
        const int r = row0 + lane;
        const float sa = MODE == SP_I8 && r < p.M ? __ldg(p.sa + r) : 0.f;
        const uint32_t srow = smem_u32(sbuf) + (uint32_t)lane * 128u;
        // The code runs once, from a cold instruction cache: short loops.
        // Pass 0 the product, passes 1 and 2 the kept G and U.
        const int passes = MODE == SP_GLU && p.save ? 3 : 1;
#pragma unroll 1
        for (int pass = 0; pass < passes; ++pass) {
            if (lane == 0) bulk_wait_read<0>();  // the buffer's last store has read it
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < EC; c += 8) {
                float v[8];
                if constexpr (MODE == SP_GLU) {
                    sum8(pass == 2 ? 128 + c0 + c : c0 + c, v);
                    if (pass == 0) {
                        float u[8];
                        sum8(128 + c0 + c, u);
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            const float2 a = act_value2<ACT>(make_float2(v[i], v[i + 1]));
                            v[i] = a.x * u[i];
                            v[i + 1] = a.y * u[i + 1];
                        }
                    }
                } else {
                    sum8(c0 + c, v);
                }
                if constexpr (MODE == SP_I8) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int at = min(ccol + c + i, p.N - 1);
                        v[i] = (float)__float_as_int(v[i]) * sa * __ldg(p.sb + at);
                        if (p.bias) v[i] += __half2float(p.bias[at]);
                    }
                }
                // 128B swizzle: 16-byte chunk j of row r lies at j ^ (r % 8).
                if constexpr (sizeof(OutT) == 2) {
                    st_shared_v4(srow + (uint32_t)(((c >> 3) ^ (lane & 7)) << 4), pack_half2(v[0], v[1]),
                                 pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i += 4)
                        st_shared_v4(srow + (uint32_t)((((c + i) >> 2) ^ (lane & 7)) << 4), __float_as_uint(v[i]),
                                     __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3]));
                }
            }
            if (MODE != SP_I8 || p.c_tma) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    const CUtensorMap* m = &maps.m[MODE == SP_GLU ? 3 + pass : MODE == SP_I8 ? 2 : MODE == SP_DX ? 4 : second ? 4 : 3];
                    if (MODE == SP_DW && p.accumulate)
                        tma_reduce_add_3d(m, smem_u32(sbuf), ccol, row0, 0);
                    else
                        tma_store_3d(m, smem_u32(sbuf), ccol, row0, 0);
                    bulk_commit();
                }
            } else {
                // Rows of C that TMA cannot store.
                __syncwarp();
                OutT* to = static_cast<OutT*>(p.C) + (long long)row0 * p.ldc + ccol;
                ff_store_rows(sbuf, to, p.ldc, min(EC, p.N - ccol), min(32, p.M - row0), p.c_unit, lane);
                __syncwarp();
            }
        }
    }
    if (lane == 0) bulk_wait<0>();
}

// ------------------------------------------------------------------ host
template <int MODE, int ACT, typename OutT>
bool sp_shared() {
    return cudaFuncSetAttribute(ff_split_kernel<MODE, ACT, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)SpCfg::SMEM_BYTES) == cudaSuccess;
}

// Clusters of 2 S CTAs that a device holds at once, asked once per device.
// The kernels are alike in what that depends on (one CTA per SM).
int sp_clusters(int dev, int S) {
    static std::atomic<int> cache[64][5];  // zero
    std::atomic<int>& v = cache[dev & 63][S];
    if (v == 0) {
        if (!sp_shared<SP_DX, 0, __half>()) return 0;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2 * S;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.blockDim = dim3(SpCfg::THREADS);
        cfg.dynamicSmemBytes = SpCfg::SMEM_BYTES;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3((unsigned)(2 * S * device_sm_count(dev)));
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, ff_split_kernel<SP_DX, 0, __half>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        v = n;
    }
    return v;
}

// The better of two and four pairs a tile, and its time in k-blocks (about
// 0.36 us): a round of clusters takes its share of the k-blocks and about 26
// besides, 9 us to start up, exchange the partial sums and finish the tile,
// of which a whole tile takes some 3.  Measured, tiles of feed_forward_tc.cuh
// against this kernel: glu 512x4096x1024 26.0 and 18.0 us, 1935x3032x320 21.2
// and 16.4, 704x1544x296 12.9 and 13.6; 8-bit 1000x256x8192 25.6 and 14.7;
// backward 8192x512x512 62.6 and 50.6, 700x1024x2816 46.7 and 37.9.
constexpr double kSplitRound = 26.0;

SplitPlan plan_split(long long tiles, int kbs) {
    SplitPlan best;
    const int dev = current_device();
    for (int s = 2; s <= 4; s *= 2) {
        const int n = sp_clusters(dev, s);
        if (n <= 0 || kbs < 2 * s) continue;
        const double t = (double)((tiles + n - 1) / n) * ((kbs + s - 1) / s + kSplitRound);
        if (t < best.time) {
            best.time = t;
            best.S = s;
        }
    }
    return best;
}

int up(long long a, int b) { return (int)((a + b - 1) / b); }

template <int MODE, int ACT, typename OutT>
pax_status_t launch_split(const SpMaps& maps, const SpParams& p, long long tiles, int S, cudaStream_t stream) {
    if (!sp_shared<MODE, ACT, OutT>()) return PAX_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2 * S;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * 2 * S));
    cfg.blockDim = dim3(SpCfg::THREADS);
    cfg.dynamicSmemBytes = SpCfg::SMEM_BYTES;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, ff_split_kernel<MODE, ACT, OutT>, maps, p) == cudaSuccess ? PAX_OK : PAX_ERR_CUDA;
}

}  // namespace

SplitPlan glu_split_plan(const GluProblem& q) { return plan_split((long long)up(q.M, 256) * up(q.F, 128), up(q.D, 64)); }

pax_status_t glu_split(const GluProblem& q, int S, cudaStream_t stream) {
    SpMaps maps;
    CUtensorMap* m = maps.m;
    if (!matrix_map(&m[0], q.X, kF16, 2, q.M, q.D, q.ldx, 64, 128) || !matrix_map(&m[1], q.Wg, kF16, 2, q.D, q.F, q.ldwg, 64, 64) ||
        !matrix_map(&m[2], q.Wu, kF16, 2, q.D, q.F, q.ldwu, 64, 64) || !matrix_map(&m[3], q.H, kF16, 2, q.M, q.F, q.ldh, 64, 32))
        return PAX_ERR_CUDA;
    m[4] = m[5] = m[3];
    if (q.G && (!matrix_map(&m[4], q.G, kF16, 2, q.M, q.F, q.ldg, 64, 32) || !matrix_map(&m[5], q.U, kF16, 2, q.M, q.F, q.ldu, 64, 32)))
        return PAX_ERR_CUDA;
    SpParams p = {};
    p.M = (int)q.M, p.N = (int)q.F;
    p.tiles_m = up(q.M, 256), p.tiles_n = up(q.F, 128);
    p.kbs = up(q.D, 64);
    p.save = q.G != nullptr;
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    if (q.act == ACT_SILU) return launch_split<SP_GLU, ACT_SILU, __half>(maps, p, tiles, S, stream);
    if (q.act == ACT_GELU_TANH) return launch_split<SP_GLU, ACT_GELU_TANH, __half>(maps, p, tiles, S, stream);
    return launch_split<SP_GLU, ACT_GELU_ERF, __half>(maps, p, tiles, S, stream);
}

SplitPlan gemm_i8_split_plan(const I8Problem& q) {
    return plan_split((long long)up(q.M, 256) * up(q.N, 256), up(q.K, 128));
}

pax_status_t gemm_i8_split(const I8Problem& q, int S, cudaStream_t stream) {
    SpMaps maps;
    CUtensorMap* m = maps.m;
    const int ce = q.c_f16 ? 2 : 4;
    SpParams p = {};
    p.c_tma = out16(q.C, q.N, q.ldc, ce);
    p.c_unit = store_unit(q.C, q.ldc, ce);
    if (!matrix_map(&m[0], q.A, kU8, 1, q.M, q.K, q.lda, 128, 128) || !matrix_map(&m[1], q.B, kU8, 1, q.N, q.K, q.ldb, 128, 128))
        return PAX_ERR_CUDA;
    m[2] = m[3] = m[4] = m[5] = m[0];
    if (p.c_tma && !matrix_map(&m[2], q.C, q.c_f16 ? kF16 : kF32, ce, q.M, q.N, q.ldc, 128 / ce, 32)) return PAX_ERR_CUDA;
    p.M = (int)q.M, p.N = (int)q.N;
    p.tiles_m = up(q.M, 256), p.tiles_n = up(q.N, 256);
    p.kbs = up(q.K, 128);
    p.C = q.C, p.ldc = q.ldc;
    p.sa = q.a_scale, p.sb = q.b_scale, p.bias = q.bias;
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    return q.c_f16 ? launch_split<SP_I8, 0, __half>(maps, p, tiles, S, stream)
                   : launch_split<SP_I8, 0, float>(maps, p, tiles, S, stream);
}

SplitPlan glu_dx_split_plan(const GluGradProblem& q) {
    return plan_split((long long)up(q.M, 256) * up(q.D, 256), 2 * up(q.F, 64));
}

pax_status_t glu_dx_split(const GluGradProblem& q, int S, cudaStream_t stream) {
    SpMaps maps;
    CUtensorMap* m = maps.m;
    if (!matrix_map(&m[0], q.dG, kF16, 2, q.M, q.F, q.lddg, 64, 128) || !matrix_map(&m[1], q.dU, kF16, 2, q.M, q.F, q.lddu, 64, 128) ||
        !matrix_map(&m[2], q.Wg, kF16, 2, q.D, q.F, q.ldwg, 64, 128) || !matrix_map(&m[3], q.Wu, kF16, 2, q.D, q.F, q.ldwu, 64, 128) ||
        !matrix_map(&m[4], q.dX, kF16, 2, q.M, q.D, q.lddx, 64, 32))
        return PAX_ERR_CUDA;
    m[5] = m[4];
    SpParams p = {};
    p.M = (int)q.M, p.N = (int)q.D;
    p.tiles_m = up(q.M, 256), p.tiles_n = up(q.D, 256);
    p.half = up(q.F, 64), p.kbs = 2 * p.half;
    return launch_split<SP_DX, 0, __half>(maps, p, (long long)p.tiles_m * p.tiles_n, S, stream);
}

SplitPlan glu_dw_split_plan(const GluGradProblem& q) {
    return plan_split(2LL * up(q.D, 256) * up(q.F, 256), up(q.M, 64));
}

pax_status_t glu_dw_split(const GluGradProblem& q, int S, cudaStream_t stream) {
    SpMaps maps;
    CUtensorMap* m = maps.m;
    const int we = q.dw_f16 ? 2 : 4;
    const CUtensorMapDataType wt = q.dw_f16 ? kF16 : kF32;
    if (!matrix_map(&m[0], q.X, kF16, 2, q.M, q.D, q.ldx, 64, 64) || !matrix_map(&m[1], q.dG, kF16, 2, q.M, q.F, q.lddg, 64, 64) ||
        !matrix_map(&m[2], q.dU, kF16, 2, q.M, q.F, q.lddu, 64, 64) ||
        !matrix_map(&m[3], q.dWg, wt, we, q.D, q.F, q.lddwg, 128 / we, 32) ||
        !matrix_map(&m[4], q.dWu, wt, we, q.D, q.F, q.lddwu, 128 / we, 32))
        return PAX_ERR_CUDA;
    m[5] = m[4];
    SpParams p = {};
    p.M = (int)q.D, p.N = (int)q.F;
    p.tiles_m = up(q.D, 256), p.tiles_n = up(q.F, 256);
    p.kbs = up(q.M, 64);
    p.accumulate = q.accumulate;
    const long long tiles = 2LL * p.tiles_m * p.tiles_n;
    return q.dw_f16 ? launch_split<SP_DW, 0, __half>(maps, p, tiles, S, stream)
                    : launch_split<SP_DW, 0, float>(maps, p, tiles, S, stream);
}

int read_clear_device_error_ff_split() {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g_pax_device_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_pax_device_error, &z, sizeof(int));
    return v;
}

bool set_wait_limit_ff_split(unsigned long long ns) {
    return cudaMemcpyToSymbol(g_pax_wait_limit_ns, &ns, sizeof(ns)) == cudaSuccess;
}

}  // namespace pax
