// feed_forward_skinny.cu -- the gated and the 8-bit product for few tokens
// (decoding), on tcgen05.
//
// With few tokens both products are bound by reading the weights once.  The
// operands are swapped: 128 weight columns are the 128 rows of the MMA and
// the tokens, padded to MP = 16, 32, 48 or 64, its columns, so that no
// tensor work is spent on absent tokens:
//   gated   64 columns of Wg and the same 64 of Wu (MN-major, as they lie)
//   8-bit   128 rows of B (K-major, as they lie)
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
// A cluster computes one tile and ends.  Two CTAs are resident per SM, so
// that one streams while the other starts up or reduces, and the hardware
// hands the next cluster to whichever SMs are free.
//
// 192 threads: warp 0 TMA producer, warp 1 MMA issuer, warps 2-5 epilogue
// (one TMEM lane, i.e. one weight column, per thread).  Every wait is bounded
// (sm100.cuh).
#include "activation.cuh"
#include "feed_forward.h"
#include "tmap.h"

namespace pax {

namespace {

enum : int { FS_GLU = 0, FS_I8 = 1 };

struct FsParams {
    int M, N, kbs;  // tokens, weight columns, k-blocks
    // FS_GLU
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

template <int MODE, int MP>
struct FsCfg {
    static constexpr int KB = MODE == FS_I8 ? 128 : 64;    // k of a ring slot: 128 bytes
    static constexpr int TILE = MODE == FS_I8 ? 128 : 64;  // output columns of a tile
    static constexpr uint32_t W_BYTES = 16384, X_BYTES = MP * 128, STAGE_BYTES = W_BYTES + X_BYTES;
    // As many slots as let two CTAs share an SM.
    static constexpr int STAGES = (int)((113 * 1024 - 1024 - 256) / STAGE_BYTES);
    static constexpr uint32_t NUM_BARS = 2 * STAGES + 1;
    static constexpr size_t SMEM_BYTES = 1024 + (size_t)STAGES * STAGE_BYTES + NUM_BARS * 8 + 16;
    static constexpr uint32_t TMEM_COLS = MP <= 32 ? 32 : 64;
    // The reduction's buffer in the ring: S parts of at most ceil(TILE / S)
    // columns (two values each for the gated product) for MP tokens, up to
    // 128 + 2 (S - 1) values a token.
    static_assert(MP * 144 * 4 <= STAGES * STAGE_BYTES, "the ring holds the contributions");
    static_assert(SMEM_BYTES <= 113 * 1024 && STAGES >= 4, "shared memory of half an SM");
};

// First column of part j of a tile shared by S CTAs.
template <int TILE>
__device__ __forceinline__ int part_start(int j, int S) {
    return (j * TILE + S - 1) / S;
}

template <int MODE, int MP>
__global__ void __launch_bounds__(192, 2)
    ff_skinny_kernel(const __grid_constant__ CUtensorMap tmW0, const __grid_constant__ CUtensorMap tmW1,
                     const __grid_constant__ CUtensorMap tmX, const __grid_constant__ FsParams p) {
    using Cfg = FsCfg<MODE, MP>;
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
    if (threadIdx.x == 0) pdl_launch_dependents();

    float v[MP];
    const int q = warp & 3;  // TMEM lane quarter an epilogue warp may read
    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            pdl_wait();  // the operands may be written by the previous grid
            const int col = tile * TILE;
            int stage = 0, total = 0;
            uint32_t phase = 0;
            for (int kb = rank; kb < p.kbs; kb += S) {
                if (!mbar_wait(empty0 + 8u * stage, phase ^ 1u, abort_flag)) break;
                const uint32_t fb = full0 + 8u * stage;
                const uint32_t w = smem_u32(smem + stage * Cfg::STAGE_BYTES);
                const int k = kb * Cfg::KB;
                mbar_arrive_expect_tx(fb, Cfg::STAGE_BYTES);
                if constexpr (MODE == FS_GLU) {
                    tma_load_3d(w, &tmW0, fb, col, k, 0);
                    tma_load_3d(w + 8192, &tmW1, fb, col, k, 0);
                } else {
                    tma_load_3d(w, &tmW0, fb, k, col, 0);
                }
                tma_load_3d(w + Cfg::W_BYTES, &tmX, fb, k, 0, 0);
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
            int stage = 0;
            uint32_t phase = 0;
            // Weights: MN-major, two blocks of 64 columns x 64 rows, or
            // K-major, 128 rows x 128 bytes.  Tokens: MP rows x 128 bytes.
            const uint64_t w0 = MODE == FS_GLU ? umma_desc_sw128(smem_u32(smem), 8192, 1024)
                                               : umma_desc_sw128(smem_u32(smem), 16, 1024);
            const uint64_t x0 = umma_desc_sw128(smem_u32(smem) + Cfg::W_BYTES, 16, 1024);
            const uint32_t id = MODE == FS_GLU ? umma_idesc_f16(128, MP, true, false) : umma_idesc_i8(128, MP);
            for (int kb = rank; kb < p.kbs; kb += S) {
                if (!mbar_wait(full0 + 8u * stage, phase, abort_flag)) break;
                tc_fence_after();
                const uint64_t at = (uint64_t)((stage * Cfg::STAGE_BYTES) >> 4);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint32_t more = (kb != rank || kk != 0) ? 1u : 0u;
                    const uint64_t xd = x0 + at + (uint64_t)(kk * 2);
                    if constexpr (MODE == FS_GLU)
                        tc_mma_f16(tmem_base, w0 + at + (uint64_t)(kk * 128), xd, id, more);
                    else
                        tc_mma_i8(tmem_base, w0 + at + (uint64_t)(kk * 2), xd, id, more);
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
        pdl_wait();  // outputs and scales may belong to the previous grid
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
        const uint32_t to = mapa_shared(smem_u32(smem) + (uint32_t)(rank * p.M * stride + at) * 4u, (uint32_t)dest);
#pragma unroll
        for (int m = 0; m < MP; ++m)
            if (m < p.M) st_shared_cluster_f32(to + (uint32_t)(m * stride * 4), v[m]);
    }
    __syncwarp();
    cluster_sync();  // the contributions are in; nothing remote happens after this
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, Cfg::TMEM_COLS);
    }
    if (*abort_flag) return;
    const float* r = reinterpret_cast<const float*>(smem);
    const int pstart = part_start<TILE>(rank, S), pwidth = part_start<TILE>(rank + 1, S) - pstart;
    for (int e = (int)threadIdx.x; e < p.M * pwidth; e += 192) {
        const int m = e / pwidth, c = e - m * pwidth;
        const long long col = (long long)tile * TILE + pstart + c;
        if (col >= p.N) continue;
        if constexpr (MODE == FS_GLU) {
            float g = 0.f, u = 0.f;
            for (int s = 0; s < S; ++s) {
                const float* x = r + (s * p.M + m) * stride + c;
                g += x[0];
                u += x[pwidth];
            }
            p.H[m * p.ldh + col] = __float2half_rn(act_value_rt(p.act, g) * u);
            if (p.G) {
                p.G[m * p.ldg + col] = __float2half_rn(g);
                p.U[m * p.ldu + col] = __float2half_rn(u);
            }
        } else {
            int sum = 0;
            for (int s = 0; s < S; ++s) sum += __float_as_int(r[(s * p.M + m) * stride + c]);
            float o = (float)sum * p.sa[m] * p.sb[col];
            if (p.bias) o += __half2float(p.bias[col]);
            if (p.c_f16)
                static_cast<__half*>(p.C)[m * p.ldc + col] = __float2half_rn(o);
            else
                static_cast<float*>(p.C)[m * p.ldc + col] = o;
        }
    }
}

// ------------------------------------------------------------------ host
bool fs_map(CUtensorMap* m, const void* base, bool i8, long long rows, long long cols, long long ld, uint32_t box_cols,
            uint32_t box_rows) {
    auto enc = tensor_map_encoder();
    if (!enc) return false;
    const uint64_t pitch = (uint64_t)ld * (i8 ? 1 : 2);
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1};
    cuuint64_t strides[2] = {pitch, (pitch * (uint64_t)rows + 15) & ~uint64_t(15)};
    cuuint32_t box[3] = {box_cols, box_rows, 1}, estr[3] = {1, 1, 1};
    return enc(m, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
               dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxSplit = 8;

template <int MODE, int MP>
bool fs_prepare(int dev) {
    static bool done[64] = {false};
    bool& d = done[dev & 63];
    if (!d)
        d = cudaFuncSetAttribute(ff_skinny_kernel<MODE, MP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)FsCfg<MODE, MP>::SMEM_BYTES) == cudaSuccess;
    return d;
}

template <int MODE, int MP>
pax_status_t launch_skinny(const CUtensorMap& w0, const CUtensorMap& w1, const CUtensorMap& x, const FsParams& p,
                           cudaStream_t stream) {
    using Cfg = FsCfg<MODE, MP>;
    const int dev = current_device(), sms = device_sm_count(dev);
    if (!fs_prepare<MODE, MP>(dev)) return PAX_ERR_CUDA;
    const long long tiles = (p.N + Cfg::TILE - 1) / Cfg::TILE;
    // As many CTAs as are resident at once, with at least four k-blocks each.
    // A CTA that has to wait for another's end costs more than the finer
    // split gains: 1x2048x5504 in 86 / 172 / 258 / 344 CTAs takes 15.4 / 13.5
    // / 13.6 / 17.7 us, 24x4096x11264 in 176 / 352 / 704 takes 35.6 / 42.9 /
    // 45.0.
    int S = 1;
    while (S < kMaxSplit && tiles * (S + 1) <= 2 * sms && p.kbs >= 4 * (S + 1)) ++S;
    if (tiles * S > 0x7fffffffLL) return PAX_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = S;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * S));
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, ff_skinny_kernel<MODE, MP>, w0, w1, x, p) == cudaSuccess ? PAX_OK : PAX_ERR_CUDA;
}

template <int MODE>
pax_status_t launch_tokens(const CUtensorMap& w0, const CUtensorMap& w1, const CUtensorMap& x, const FsParams& p,
                           cudaStream_t stream) {
    if (p.M <= 16) return launch_skinny<MODE, 16>(w0, w1, x, p, stream);
    if (p.M <= 32) return launch_skinny<MODE, 32>(w0, w1, x, p, stream);
    if (p.M <= 48) return launch_skinny<MODE, 48>(w0, w1, x, p, stream);
    return launch_skinny<MODE, 64>(w0, w1, x, p, stream);
}

bool rows16(const void* p, long long ld, int elem) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * elem) % 16 == 0;
}

uint32_t padded(long long M) { return (uint32_t)((M + 15) / 16 * 16); }

}  // namespace

bool glu_skinny_ok(const GluProblem& q) {
    return q.M <= 64 && q.D > 0 && rows16(q.X, q.ldx, 2) && rows16(q.Wg, q.ldwg, 2) && rows16(q.Wu, q.ldwu, 2);
}

pax_status_t glu_skinny(const GluProblem& q, cudaStream_t stream) {
    CUtensorMap wg, wu, x;
    if (!fs_map(&wg, q.Wg, false, q.D, q.F, q.ldwg, 64, 64) || !fs_map(&wu, q.Wu, false, q.D, q.F, q.ldwu, 64, 64) ||
        !fs_map(&x, q.X, false, q.M, q.D, q.ldx, 64, padded(q.M)))
        return PAX_ERR_CUDA;
    FsParams p = {};
    p.M = (int)q.M;
    p.N = (int)q.F;
    p.kbs = (int)((q.D + 63) / 64);
    p.H = q.H, p.G = q.G, p.U = q.U;
    p.ldh = q.ldh, p.ldg = q.ldg, p.ldu = q.ldu;
    p.act = q.act;
    return launch_tokens<FS_GLU>(wg, wu, x, p, stream);
}

bool gemm_i8_skinny_ok(const I8Problem& q) {
    return q.M <= 64 && q.K > 0 && rows16(q.A, q.lda, 1) && rows16(q.B, q.ldb, 1);
}

pax_status_t gemm_i8_skinny(const I8Problem& q, cudaStream_t stream) {
    CUtensorMap w, x;
    if (!fs_map(&w, q.B, true, q.N, q.K, q.ldb, 128, 128) || !fs_map(&x, q.A, true, q.M, q.K, q.lda, 128, padded(q.M)))
        return PAX_ERR_CUDA;
    FsParams p = {};
    p.M = (int)q.M;
    p.N = (int)q.N;
    p.kbs = (int)((q.K + 127) / 128);
    p.C = q.C;
    p.ldc = q.ldc;
    p.sa = q.a_scale, p.sb = q.b_scale, p.bias = q.bias;
    p.c_f16 = q.c_f16;
    return launch_tokens<FS_I8>(w, w, x, p, stream);
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
