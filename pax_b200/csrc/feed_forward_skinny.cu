// feed_forward_skinny.cu -- the gated and the 8-bit product and the input
// gradient for few tokens (decoding, short sequences), on tcgen05.
//
// With few tokens these products are bound by reading the weights once.  The
// operands are swapped: 128 weight columns are the 128 rows of the MMA and
// the tokens, padded to MP = 16, 32, 48 or 64, its columns, so that no
// tensor work is spent on absent tokens:
//   gated       64 columns of Wg and the same 64 of Wu (MN-major, as they lie)
//   8-bit       128 rows of B (K-major, as they lie)
//   input grad  128 rows of Wg, then of Wu, along F (K-major, as they lie)
// More than 64 tokens run as equal chunks (blockIdx.y), each reading the
// weights again, mostly from L2.
//
// A tile of weight columns is too coarse a unit of work for 148 SMs, so a
// cluster of S CTAs shares each tile along K: CTA r takes k-blocks r, r + S,
// and so on, which streams neighbouring rows at the same time.  The partial
// sums meet in distributed shared memory: CTA j owns the j-th part of the
// tile's columns, every CTA stores its partial sums of that part straight
// into CTA j's (by then idle) ring, and CTA j adds the S contributions in CTA
// order, applies the epilogue and stores.  No global workspace, no atomics,
// and the same bits every time.
//
// A cluster computes one tile and ends.  R = 2 or 3 CTAs are resident per SM,
// so that one streams while another starts up or reduces, and the hardware
// hands the next cluster to whichever SMs are free.
//
// 192 threads: warp 0 TMA producer, warp 1 MMA issuer, warps 2-5 epilogue
// (one TMEM lane, i.e. one weight column, per thread).  Every wait is bounded
// (sm100.cuh).
#include "activation.cuh"
#include "feed_forward.h"
#include "tmap.h"

#include <atomic>

namespace pax {

namespace {

enum : int { FS_GLU = 0, FS_I8 = 1, FS_DX = 2 };

struct FsParams {
    int M, N, kbs;  // tokens, weight columns, k-blocks
    int rows;       // tokens of a chunk
    int half;       // FS_DX: k-blocks of the first term
    int beside;     // FS_DX: see glu_dx_skinny
    int w_const;    // the weights are not written by the previous grid
    // FS_GLU; FS_DX: the gradient in H
    __half *H, *G, *U;
    long long ldh, ldg, ldu;
    int act;
    // FS_I8
    void* C;
    long long ldc;
    const float *sa, *sb;
    const __half* bias;
    int c_f16;
};

template <int MODE, int MP, int R>
struct FsCfg {
    static constexpr int KB = MODE == FS_I8 ? 128 : 64;    // k of a ring slot: 128 bytes
    static constexpr int TILE = MODE == FS_GLU ? 64 : 128;  // output columns of a tile
    static constexpr uint32_t W_BYTES = 16384, X_BYTES = MP * 128, STAGE_BYTES = W_BYTES + X_BYTES;
    // As many slots as let R CTAs share an SM.
    static constexpr uint32_t SHARE = R == 2 ? 113 * 1024 : 75 * 1024;
    static constexpr int STAGES = (int)((SHARE - 1024 - 256) / STAGE_BYTES);
    static constexpr uint32_t NUM_BARS = 2 * STAGES + 1;
    static constexpr size_t SMEM_BYTES = 1024 + (size_t)STAGES * STAGE_BYTES + NUM_BARS * 8 + 16;
    static constexpr uint32_t TMEM_COLS = MP <= 32 ? 32 : 64;
    // The reduction's buffer in the ring: S parts of at most ceil(TILE / S)
    // columns (two values each for the gated product) for MP tokens, up to
    // 128 + 2 (S - 1) values a token.
    static_assert(MP * 144 * 4 <= STAGES * STAGE_BYTES, "the ring holds the contributions");
    static_assert(SMEM_BYTES <= SHARE && STAGES >= 3, "an R-th of an SM's shared memory");
};

// First column of part j of a tile shared by S CTAs.
template <int TILE>
__device__ __forceinline__ int part_start(int j, int S) {
    return (j * TILE + S - 1) / S;
}

template <int MODE, int MP, int R>
__global__ void __launch_bounds__(192, R)
    ff_skinny_kernel(const __grid_constant__ CUtensorMap tmW0, const __grid_constant__ CUtensorMap tmW1,
                     const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmX1,
                     const __grid_constant__ FsParams p) {
    using Cfg = FsCfg<MODE, MP, R>;
    constexpr int STAGES = Cfg::STAGES, TILE = Cfg::TILE;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem =
        reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NUM_BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const uint32_t full0 = smem_u32(bars);
    const uint32_t empty0 = full0 + 8u * STAGES;
    const uint32_t done_bar = empty0 + 8u * STAGES;  // every MMA has finished

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int S;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(S));
    const int rank = (int)cluster_ctarank();
    const int tile = (int)blockIdx.x / S;
    const int m0 = (int)blockIdx.y * p.rows, M = min(p.rows, p.M - m0);  // this chunk's tokens

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full0 + 8u * s, 1);
            mbar_init(empty0 + 8u * s, 1);
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(tmem_slot), Cfg::TMEM_COLS);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    float v[MP];
    const int q = warp & 3;  // TMEM lane quarter an epilogue warp may read
    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            const int col = tile * TILE;
            int stage = 0, total = 0;
            uint32_t phase = 0;
            auto load_weights = [&](int kb) {
                const uint32_t fb = full0 + 8u * stage, w = smem_u32(smem + stage * Cfg::STAGE_BYTES);
                const int k = kb * Cfg::KB;
                if constexpr (MODE == FS_GLU) {
                    tma_load_3d(w, &tmW0, fb, col, k, 0);
                    tma_load_3d(w + 8192, &tmW1, fb, col, k, 0);
                } else {
                    const bool second = MODE == FS_DX && kb >= p.half;
                    tma_load_3d(w, second ? &tmW1 : &tmW0, fb, second ? k - p.half * Cfg::KB : k, col, 0);
                }
            };
            auto load_tokens = [&](int kb) {
                const uint32_t x = smem_u32(smem + stage * Cfg::STAGE_BYTES) + Cfg::W_BYTES;
                const bool second = MODE == FS_DX && kb >= p.half;
                tma_load_3d(x, second ? &tmX1 : &tmX, full0 + 8u * stage,
                            (second ? kb - p.half : kb) * Cfg::KB, m0, 0);
            };
            // Weights that the previous grid does not write: a ring's worth of
            // them before that grid has ended.  Their bytes are expected
            // without arriving; a slot is full once the tokens' arrival and
            // bytes have come too.
            int early = 0;
            if (MODE != FS_DX && p.w_const)
                for (int kb = rank; kb < p.kbs && early < STAGES; kb += S, ++early, ++stage) {
                    mbar_expect_tx(full0 + 8u * stage, Cfg::W_BYTES);
                    load_weights(kb);
                }
            stage = 0;
            if (MODE != FS_DX || !p.beside) {
                pdl_wait();  // the operands may be written by the previous grid
                // Not before: the next grid may load weights early, which only
                // this grid is known not to write.
                pdl_launch_dependents();
            }
            for (int kb = rank; kb < p.kbs; kb += S) {
                if (!mbar_wait(empty0 + 8u * stage, phase ^ 1u, abort_flag)) break;
                const bool have = total < early;
                mbar_arrive_expect_tx(full0 + 8u * stage, (have ? 0u : Cfg::W_BYTES) + (uint32_t)p.rows * 128u);
                if (!have) load_weights(kb);
                load_tokens(kb);
                ++total;
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            // Every load issued must land before the ring is reused.
            for (int s = 0; s < STAGES && s < total; ++s) {
                const int i = s + ((total - 1 - s) / STAGES) * STAGES;  // last k-block on slot s
                mbar_wait(full0 + 8u * s, (uint32_t)(i / STAGES) & 1u, nullptr);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        if (lane == 0) {
            // The waits below count from here: for the loads of this grid, not
            // for the end of the previous one.
            if (MODE != FS_DX || !p.beside) pdl_wait();
            int stage = 0;
            uint32_t phase = 0;
            // Weights: MN-major, two blocks of 64 columns x 64 rows, or
            // K-major, 128 rows x 128 bytes.  Tokens: MP rows x 128 bytes.
            const uint64_t w0 = MODE == FS_GLU ? umma_desc_sw128(smem_u32(smem), 8192, 1024)
                                               : umma_desc_sw128(smem_u32(smem), 16, 1024);
            const uint64_t x0 = umma_desc_sw128(smem_u32(smem) + Cfg::W_BYTES, 16, 1024);
            const uint32_t id = MODE == FS_I8 ? umma_idesc_i8(128, MP) : umma_idesc_f16(128, MP, MODE == FS_GLU, false);
            for (int kb = rank; kb < p.kbs; kb += S) {
                if (!mbar_wait(full0 + 8u * stage, phase, abort_flag)) break;
                tc_fence_after();
                const uint64_t at = (uint64_t)((stage * Cfg::STAGE_BYTES) >> 4);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint32_t more = (kb != rank || kk != 0) ? 1u : 0u;
                    const uint64_t xd = x0 + at + (uint64_t)(kk * 2);
                    const uint64_t wd = w0 + at + (uint64_t)(kk * (MODE == FS_GLU ? 128 : 2));
                    if constexpr (MODE == FS_I8)
                        tc_mma_i8(tmem_base, wd, xd, id, more);
                    else
                        tc_mma_f16(tmem_base, wd, xd, id, more);
                }
                tc_commit(empty0 + 8u * stage);
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            tc_commit(done_bar);
            mbar_wait(done_bar, 0, nullptr);
        }
    } else {
        if (MODE != FS_DX || !p.beside) pdl_wait();  // outputs and scales may belong to the previous grid
        mbar_wait(done_bar, 0, nullptr);
        __syncwarp();
        tc_fence_after();
        const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16);
#pragma unroll
        for (int c = 0; c < MP; c += 16) tmem_ld_32x32b_x16(src + (uint32_t)c, v + c);
        tmem_wait_ld();
        tc_fence_before();
    }

    // ------------------------------------------------ reduction
    __syncwarp();
    cluster_sync();  // every CTA's ring is idle: its loads and MMAs are done
    const int stride = (MODE == FS_GLU ? 2 : 1) * ((TILE + S - 1) / S);  // values a token and contribution
    if (warp >= 2) {
        const int l = q * 32 + lane;  // this thread's MMA row
        const int f = l & (TILE - 1);  // its column in the tile (gated: rows 64.. are the up projection)
        const int dest = f * S / TILE;
        const int dstart = part_start<TILE>(dest, S), dwidth = part_start<TILE>(dest + 1, S) - dstart;
        const int at = f - dstart + (MODE == FS_GLU && l >= TILE ? dwidth : 0);
        const uint32_t to = mapa_shared(smem_u32(smem) + (uint32_t)(rank * M * stride + at) * 4u, (uint32_t)dest);
#pragma unroll
        for (int m = 0; m < MP; ++m)
            if (m < M) st_shared_cluster_f32(to + (uint32_t)(m * stride * 4), v[m]);
    }
    // A thread finishes one column of this CTA's part, for every step-th token:
    // its scale and bias come while the contributions arrive.
    const int pstart = part_start<TILE>(rank, S), pwidth = part_start<TILE>(rank + 1, S) - pstart;
    int shift = 0;
    while ((1 << shift) < pwidth) ++shift;
    const int c = (int)threadIdx.x & ((1 << shift) - 1), step = 192 >> shift;
    const long long col = (long long)tile * TILE + pstart + c;
    const bool mine = (int)threadIdx.x >> shift < step && c < pwidth && col < p.N;
    float sb = 0.f, bias = 0.f;
    if (MODE == FS_I8 && mine) {
        sb = __ldg(p.sb + col);
        if (p.bias) bias = __half2float(p.bias[col]);
    }
    __syncwarp();
    cluster_sync();  // the contributions are in; nothing remote happens after this
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, Cfg::TMEM_COLS);
    }
    // What follows in the stream relies on the grid this one ran beside.
    if (MODE == FS_DX && p.beside && threadIdx.x == 0) {
        pdl_wait();
        pdl_launch_dependents();
    }
    if (*abort_flag || !mine) return;
    const float* r = reinterpret_cast<const float*>(smem);
#pragma unroll 1
    for (int m = (int)threadIdx.x >> shift; m < M; m += step) {
        const long long row = m0 + m;
        const float* x = r + m * stride + c;
        if constexpr (MODE == FS_GLU) {
            float g = 0.f, u = 0.f;
#pragma unroll 1
            for (int s = 0; s < S; ++s, x += M * stride) {
                g += x[0];
                u += x[pwidth];
            }
            p.H[row * p.ldh + col] = __float2half_rn(act_value_rt(p.act, g) * u);
            if (p.G) {
                p.G[row * p.ldg + col] = __float2half_rn(g);
                p.U[row * p.ldu + col] = __float2half_rn(u);
            }
        } else if constexpr (MODE == FS_DX) {
            float sum = 0.f;
#pragma unroll 1
            for (int s = 0; s < S; ++s, x += M * stride) sum += x[0];
            p.H[row * p.ldh + col] = __float2half_rn(sum);
        } else {
            const float sa = __ldg(p.sa + row);
            int sum = 0;
#pragma unroll 1
            for (int s = 0; s < S; ++s, x += M * stride) sum += __float_as_int(x[0]);
            float o = (float)sum * sa * sb;
            if (p.bias) o += bias;
            if (p.c_f16)
                static_cast<__half*>(p.C)[row * p.ldc + col] = __float2half_rn(o);
            else
                static_cast<float*>(p.C)[row * p.ldc + col] = o;
        }
    }
}

// ------------------------------------------------------------------ host
constexpr int kMaxSplit = 8;

// Allow the kernel its shared memory on the current device: per device and
// context, and cheap to repeat.
template <int MODE, int MP, int R>
bool fs_shared() {
    return cudaFuncSetAttribute(ff_skinny_kernel<MODE, MP, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)FsCfg<MODE, MP, R>::SMEM_BYTES) == cudaSuccess;
}

// Clusters of S CTAs that device `dev` holds at once with one CTA per SM,
// which is what the runtime answers whatever shared memory a CTA takes (a
// cluster's CTAs share a GPC, so this can be below the SMs' room); with R CTAs
// per SM it is R times that.  Asked once per device and S, of one kernel for
// all; 0: error.
int fs_clusters(int dev, int S) {
    static std::atomic<int> cache[64][kMaxSplit + 1];  // zero; calls may come from several threads
    std::atomic<int>& v = cache[dev & 63][S];
    if (v == 0) {
        if (!fs_shared<FS_GLU, 16, 2>()) return 0;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = S;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.blockDim = dim3(192);
        cfg.dynamicSmemBytes = FsCfg<FS_GLU, 16, 2>::SMEM_BYTES;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3((unsigned)(4 * device_sm_count(dev) * S));  // the answer is capped by the grid
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, ff_skinny_kernel<FS_GLU, 16, 2>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        v = n;
    }
    return v;
}

struct FsMaps {
    CUtensorMap w0, w1, x0, x1;
};

template <int MODE, int MP, int R>
pax_status_t launch_split(const FsMaps& m, const FsParams& p, long long tiles, int S, cudaStream_t stream) {
    using Cfg = FsCfg<MODE, MP, R>;
    if (!fs_shared<MODE, MP, R>()) return PAX_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = S;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * S), (unsigned)((p.M + p.rows - 1) / p.rows));
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, ff_skinny_kernel<MODE, MP, R>, m.w0, m.w1, m.x0, m.x1, p) == cudaSuccess
               ? PAX_OK
               : PAX_ERR_CUDA;
}

// Time of n resident CTAs of kb k-blocks each, in k-blocks at an SM's share of
// the memory bandwidth (44 GB/s).  SMs share the bandwidth evenly; a CTA
// alone takes in at most about one share with R = 2 (0.85 with R = 3, whose
// ring is shorter).  So first all SMs work off the CTAs that each of them
// has, then those with one more CTA finish, faster the fewer they are.
// Measured against it at D = 4096, with a fixed 2 us on top: 74 tiles unsplit,
// R = 2, 22.0 us (model 23); 176 tiles, R = 2, 35.0 (35), in pairs at R = 3,
// 31.0 (28); 350 tiles, R = 3, 57.9 (55).  Over 19 shapes of 1 to 64 tokens
// the choice is the best of 14 tried by hand, or within 6 % of it.
double fs_wave_time(long long n, double kb, int R, int sms) {
    const double cap = R == 2 ? 1.0 : 0.85;
    const long long a = n / sms, rem = n % sms;
    const double t = a > 0 ? a * kb / (a * cap < 1 ? a * cap : 1) : 0;
    if (rem == 0) return t;
    const double own = (a + 1) * cap, share = (double)sms / rem;
    return t + ((a + 1) * kb - t * (own < 1 ? own : 1)) / (own < share ? own : share);
}

// The split of a problem and its modelled time in k-blocks.
struct FsPlan {
    int S = 1, R = 2;
    double time = -1;
};

template <int MODE, int MP>
FsPlan fs_plan(const FsParams& p) {
    const int dev = current_device(), sms = device_sm_count(dev);
    constexpr int TILE = FsCfg<MODE, MP, 2>::TILE;
    const long long tiles = (long long)((p.N + TILE - 1) / TILE) * ((p.M + p.rows - 1) / p.rows);
    FsPlan best;
    // The residency and split with the shortest modelled time, among those
    // whose clusters are all resident at once (1x2048x5504 in fives at three
    // per SM, of which 78 of 86 clusters are resident: 15.7 us, in threes at
    // two per SM 10.8); or unsplit in several waves.
    for (int r = 2; r <= 3; ++r)
        for (int s = 1; s <= kMaxSplit; ++s) {
            // CTAs that share an SM with others take four k-blocks at least
            // (16x1024x2816 with two: 6.9 us, with four 5.7).
            if (s > 1 && (tiles * s > (long long)r * sms || p.kbs < (tiles * s > sms ? 4 : 2) * s)) break;
            const long long n = (long long)r * fs_clusters(dev, s);
            if (n <= 0 || (s > 1 && tiles > n)) continue;
            const long long waves = (tiles - 1) / n;  // before the last one
            const double kb = (p.kbs + s - 1) / s;
            const double t = (double)waves * r * kb + fs_wave_time((tiles - waves * n) * s, kb, r, sms) + (s > 1 ? 1 : 0);
            if (best.time < 0 || t < best.time || (t == best.time && r == best.R)) {
                best.time = t;
                best.S = s;
                best.R = r;
            }
        }
    return best;
}

template <int MODE, int MP>
pax_status_t launch_skinny(const FsMaps& m, const FsParams& p, cudaStream_t stream) {
    const FsPlan plan = fs_plan<MODE, MP>(p);
    if (plan.time < 0) return PAX_ERR_CUDA;
    constexpr int TILE = FsCfg<MODE, MP, 2>::TILE;
    const long long tiles = (p.N + TILE - 1) / TILE;
    if (tiles * plan.S > 0x7fffffffLL) return PAX_ERR_UNSUPPORTED;
    return plan.R == 2 ? launch_split<MODE, MP, 2>(m, p, tiles, plan.S, stream)
                       : launch_split<MODE, MP, 3>(m, p, tiles, plan.S, stream);
}

template <int MODE>
pax_status_t launch_tokens(const FsMaps& m, const FsParams& p, cudaStream_t stream) {
    if (p.rows <= 16) return launch_skinny<MODE, 16>(m, p, stream);
    if (p.rows <= 32) return launch_skinny<MODE, 32>(m, p, stream);
    if (p.rows <= 48) return launch_skinny<MODE, 48>(m, p, stream);
    return launch_skinny<MODE, 64>(m, p, stream);
}

template <int MODE>
double plan_time(const FsParams& p) {
    const double t = p.rows <= 16   ? fs_plan<MODE, 16>(p).time
                     : p.rows <= 32 ? fs_plan<MODE, 32>(p).time
                     : p.rows <= 48 ? fs_plan<MODE, 48>(p).time
                                    : fs_plan<MODE, 64>(p).time;
    return t < 0 ? 1e30 : t;
}

// Equal chunks of at most 64 tokens.
int chunk_rows(long long M) {
    const long long chunks = (M + 63) / 64;
    return (int)((M + chunks - 1) / chunks);
}

}  // namespace

// More tokens than this never read the weights again for another chunk.
constexpr long long kMaxChunked = 512;

// Constant weights are loaded early for one chunk at most, as w_const says:
// what a caller orders by the number of tokens does not depend on which kernel
// more of them run on.
constexpr long long kMaxEarly = 64;

bool glu_skinny_ok(const GluProblem& q) {
    return q.M <= kMaxChunked && q.D > 0 && q.D <= kMaxSum && rows16(q.X, q.ldx, 2) && rows16(q.Wg, q.ldwg, 2) && rows16(q.Wu, q.ldwu, 2);
}

static void glu_params(const GluProblem& q, FsParams& p) {
    p.M = (int)q.M;
    p.N = (int)q.F;
    p.kbs = (int)((q.D + 63) / 64);
    p.rows = chunk_rows(q.M);
}

double glu_skinny_time(const GluProblem& q) {
    FsParams p = {};
    glu_params(q, p);
    return plan_time<FS_GLU>(p);
}

pax_status_t glu_skinny(const GluProblem& q, cudaStream_t stream) {
    FsMaps m;
    FsParams p = {};
    glu_params(q, p);
    if (!matrix_map(&m.w0, q.Wg, kF16, 2, q.D, q.F, q.ldwg, 64, 64) || !matrix_map(&m.w1, q.Wu, kF16, 2, q.D, q.F, q.ldwu, 64, 64) ||
        !matrix_map(&m.x0, q.X, kF16, 2, q.M, q.D, q.ldx, 64, (uint32_t)p.rows))
        return PAX_ERR_CUDA;
    m.x1 = m.x0;
    p.w_const = q.w_const && q.M <= kMaxEarly;
    p.H = q.H, p.G = q.G, p.U = q.U;
    p.ldh = q.ldh, p.ldg = q.ldg, p.ldu = q.ldu;
    p.act = q.act;
    return launch_tokens<FS_GLU>(m, p, stream);
}

bool glu_dx_skinny_ok(const GluGradProblem& q) {
    return q.dX && q.M > 0 && q.M <= kMaxChunkedTokens && q.D > 0 && q.F > 0 && q.F <= kMaxSum && rows16(q.dG, q.lddg, 2) &&
           rows16(q.dU, q.lddu, 2) && rows16(q.Wg, q.ldwg, 2) && rows16(q.Wu, q.ldwu, 2);
}

static void dx_params(const GluGradProblem& q, FsParams& p) {
    p.M = (int)q.M;
    p.N = (int)q.D;
    p.half = (int)((q.F + 63) / 64);
    p.kbs = 2 * p.half;
    p.rows = chunk_rows(q.M);
    p.H = q.dX;
    p.ldh = q.lddx;
}

double glu_dx_skinny_time(const GluGradProblem& q) {
    FsParams p = {};
    dx_params(q, p);
    return plan_time<FS_DX>(p);
}

// beside: the previous launch in the stream is glu_back_tc's for the weight
// gradients alone, which lets this one start once dG and dU are written.
// Neither reads what the other writes, so they run side by side where the
// first leaves SMs free, and this one ends no earlier than the first.
pax_status_t glu_dx_skinny(const GluGradProblem& q, bool beside, cudaStream_t stream) {
    FsMaps m;
    FsParams p = {};
    dx_params(q, p);
    p.beside = beside;
    if (!matrix_map(&m.w0, q.Wg, kF16, 2, q.D, q.F, q.ldwg, 64, 128) || !matrix_map(&m.w1, q.Wu, kF16, 2, q.D, q.F, q.ldwu, 64, 128) ||
        !matrix_map(&m.x0, q.dG, kF16, 2, q.M, q.F, q.lddg, 64, (uint32_t)p.rows) ||
        !matrix_map(&m.x1, q.dU, kF16, 2, q.M, q.F, q.lddu, 64, (uint32_t)p.rows))
        return PAX_ERR_CUDA;
    return launch_tokens<FS_DX>(m, p, stream);
}

bool gemm_i8_skinny_ok(const I8Problem& q) {
    return q.M <= kMaxChunked && q.K > 0 && rows16(q.A, q.lda, 1) && rows16(q.B, q.ldb, 1);
}

static void i8_params(const I8Problem& q, FsParams& p) {
    p.M = (int)q.M;
    p.N = (int)q.N;
    p.kbs = (int)((q.K + 127) / 128);
    p.rows = chunk_rows(q.M);
}

double gemm_i8_skinny_time(const I8Problem& q) {
    FsParams p = {};
    i8_params(q, p);
    return plan_time<FS_I8>(p);
}

pax_status_t gemm_i8_skinny(const I8Problem& q, cudaStream_t stream) {
    FsMaps m;
    FsParams p = {};
    i8_params(q, p);
    if (!matrix_map(&m.w0, q.B, kU8, 1, q.N, q.K, q.ldb, 128, 128) ||
        !matrix_map(&m.x0, q.A, kU8, 1, q.M, q.K, q.lda, 128, (uint32_t)p.rows))
        return PAX_ERR_CUDA;
    m.w1 = m.w0;
    m.x1 = m.x0;
    p.w_const = q.b_const && q.M <= kMaxEarly;
    p.C = q.C;
    p.ldc = q.ldc;
    p.sa = q.a_scale, p.sb = q.b_scale, p.bias = q.bias;
    p.c_f16 = q.c_f16;
    return launch_tokens<FS_I8>(m, p, stream);
}

int read_clear_device_error_ff_skinny() {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g_pax_device_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_pax_device_error, &z, sizeof(int));
    return v;
}

bool set_wait_limit_ff_skinny(unsigned long long ns) {
    return cudaMemcpyToSymbol(g_pax_wait_limit_ns, &ns, sizeof(ns)) == cudaSuccess;
}

}  // namespace pax
