// feed_forward_any.cu -- the feed-forward products for every layout.
//
// The tensor-memory-accelerator kernels need 16-byte aligned bases and row
// pitches; problems without them, and empty sums, run here.  One kernel for
// the four products
//   gated        H = act(X.Wg) * (X.Wu)          two accumulators, one A
//   input grad   dX = dG.Wg^T + dU.Wu^T          one accumulator, two terms
//   weight grad  dWg = X^T.dG, dWu = X^T.dU      blockIdx.z picks the pair
//   8-bit        C = (A.B^T) * sa * sb + b       int32 accumulators
// A block computes 128 rows x 128 accumulator columns (the gated product 64
// of each projection) with 16x16x16 warp matrix operations.  Operands come
// element by element, a warp along whichever direction is contiguous in
// memory, the next step's into registers while this one multiplies, and lie
// in shared memory the way they were read.  Bound by the number of those
// loads, 32 a thread for 32 k: glu 4096x4095x4097 takes 2.17 ms (127 TF/s), its
// backward pass 4.62 ms, the 8-bit product of that shape 1.17 ms; with few
// tokens each step waits for its loads (glu 7x1001x2001 37 us).
#include "activation.cuh"
#include "feed_forward.h"

#include <mma.h>

namespace pax {

namespace {

enum : int { ANY_GLU = 0, ANY_DX = 1, ANY_DW = 2, ANY_I8 = 3 };

struct AnyOperand {
    const void* p;
    long long ld;  // elements between rows
};

struct AnyParams {
    AnyOperand a[2], b[2];  // ANY_DX: the two terms; ANY_GLU, ANY_DW: b[1] is the up projection's
    long long M, N, R;      // output rows and columns, length of the sum
    void* out[3];
    long long ldo[3];
    int out_f16, accumulate, act;
    const float *sa, *sb;
    const __half* bias;
};

constexpr int kThreads = 256, kStep = 32;  // k of a step

// X outer positions x kStep k of one operand: in registers, then in shared
// memory as [outer][k] (RED: k is contiguous in memory) or [k][outer].  A
// fragment has to start on 32 bytes, so 8-bit k lie in two slabs of 16, 48
// bytes from row to row.
template <typename T, int X, bool RED>
struct AnyTile {
    static_assert(RED || sizeof(T) == 2, "8-bit operands have k contiguous");
    static constexpr int PER = X * kStep / kThreads;
    static constexpr int LD = sizeof(T) == 1 ? 48 : RED ? kStep + 8 : X + 8;
    static constexpr int ELEMS = sizeof(T) == 1 ? 2 * X * LD : RED ? X * LD : kStep * LD;
    // Where outer position x, k r lies.
    static __device__ __forceinline__ int at(int x, int r) {
        return sizeof(T) == 1 ? ((r >> 4) * X + x) * LD + (r & 15) : RED ? x * LD + r : r * LD + x;
    }
    T v[PER];

    __device__ __forceinline__ void load(const AnyOperand& o, long long o0, long long omax, long long r0, long long rmax) {
        const int t = (int)threadIdx.x;
        const T* p = static_cast<const T*>(o.p);
        if constexpr (RED) {
            constexpr int ROWS = kThreads / kStep;
            const long long r = r0 + t % kStep;
            const T* at = p + (o0 + t / kStep) * o.ld + r;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                v[j] = r < rmax && o0 + t / kStep + j * ROWS < omax ? *at : T(0);
                at += ROWS * o.ld;
            }
        } else {
            constexpr int ROWS = kThreads / X;
            const long long x = o0 + t % X;
            const T* at = p + (r0 + t / X) * o.ld + x;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                v[j] = x < omax && r0 + t / X + j * ROWS < rmax ? *at : T(0);
                at += ROWS * o.ld;
            }
        }
    }
    __device__ __forceinline__ void store(T* s) const {
        const int t = (int)threadIdx.x;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if constexpr (RED)
                s[at(t / kStep + j * (kThreads / kStep), t % kStep)] = v[j];
            else
                s[at(t % X, t / X + j * (kThreads / X))] = v[j];
        }
    }
};

template <int MODE>
__global__ void __launch_bounds__(kThreads) feed_forward_any_kernel(const AnyParams p) {
    using namespace nvcuda;
    using T = typename std::conditional<MODE == ANY_I8, signed char, __half>::type;
    using Acc = typename std::conditional<MODE == ANY_I8, int, float>::type;
    constexpr int NACC = MODE == ANY_GLU ? 2 : 1, BM = 128, BN = 128 / NACC;
    constexpr bool A_RED = MODE != ANY_DW, B_RED = MODE == ANY_DX || MODE == ANY_I8;
    using TileA = AnyTile<T, BM, A_RED>;
    using TileB = AnyTile<T, BN, B_RED>;
    using LayoutA = typename std::conditional<A_RED, wmma::row_major, wmma::col_major>::type;
    using LayoutB = typename std::conditional<B_RED, wmma::col_major, wmma::row_major>::type;
    __shared__ __align__(128) T sA[TileA::ELEMS];
    __shared__ __align__(128) T sB[NACC][TileB::ELEMS];
    __shared__ __align__(128) Acc sC[kThreads / 32][NACC][256];  // one fragment per warp

    const long long tiles_n = (p.N + BN - 1) / BN;
    const long long m0 = (long long)blockIdx.x / tiles_n * BM, n0 = (long long)blockIdx.x % tiles_n * BN;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int wm = (warp >> 1) * 32, wn = (warp & 1) * (BN / 2);  // this warp's 32 x BN/2 part
    constexpr int FN = BN / 32;
    const int z = MODE == ANY_DW ? (int)blockIdx.z : 0;

    wmma::fragment<wmma::accumulator, 16, 16, 16, Acc> acc[NACC][2][FN];
#pragma unroll
    for (int c = 0; c < NACC; ++c)
#pragma unroll
        for (int i = 0; i < 2 * FN; ++i) wmma::fill_fragment(acc[c][i / FN][i % FN], Acc(0));
    const long long steps = (p.R + kStep - 1) / kStep, all = MODE == ANY_DX ? 2 * steps : steps;
    TileA ta;
    TileB tb[NACC];
    auto fetch = [&](long long step) {
        const int term = MODE == ANY_DX && step >= steps ? 1 : 0;
        const long long r0 = (step - term * steps) * kStep;
        ta.load(p.a[term], m0, p.M, r0, p.R);
#pragma unroll
        for (int c = 0; c < NACC; ++c) tb[c].load(p.b[MODE == ANY_GLU ? c : term + z], n0, p.N, r0, p.R);
    };
    if (all > 0) fetch(0);
    for (long long step = 0; step < all; ++step) {
        ta.store(sA);
#pragma unroll
        for (int c = 0; c < NACC; ++c) tb[c].store(sB[c]);
        __syncthreads();
        if (step + 1 < all) fetch(step + 1);
#pragma unroll
        for (int kk = 0; kk < kStep; kk += 16) {
            wmma::fragment<wmma::matrix_a, 16, 16, 16, T, LayoutA> fa[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                wmma::load_matrix_sync(fa[i], sA + TileA::at(wm + 16 * i, kk), TileA::LD);
#pragma unroll
            for (int c = 0; c < NACC; ++c)
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    wmma::fragment<wmma::matrix_b, 16, 16, 16, T, LayoutB> fb;
                    wmma::load_matrix_sync(fb, sB[c] + TileB::at(wn + 16 * j, kk), TileB::LD);
#pragma unroll
                    for (int i = 0; i < 2; ++i) wmma::mma_sync(acc[c][i][j], fa[i], fb, acc[c][i][j]);
                }
        }
        __syncthreads();
    }
    // Epilogue, one 16 x 16 fragment at a time through the warp's buffer.
#pragma unroll
    for (int f = 0; f < 2 * FN; ++f) {
#pragma unroll
        for (int c = 0; c < NACC; ++c) wmma::store_matrix_sync(sC[warp][c], acc[c][f / FN][f % FN], 16, wmma::mem_row_major);
        __syncwarp();
        for (int e = lane; e < 256; e += 32) {
            const long long row = m0 + wm + 16 * (f / FN) + e / 16, col = n0 + wn + 16 * (f % FN) + e % 16;
            if (row >= p.M || col >= p.N) continue;
            if constexpr (MODE == ANY_GLU) {
                const float g = sC[warp][0][e], u = sC[warp][NACC - 1][e];
                static_cast<__half*>(p.out[0])[row * p.ldo[0] + col] = __float2half_rn(act_value_rt(p.act, g) * u);
                if (p.out[1]) {
                    static_cast<__half*>(p.out[1])[row * p.ldo[1] + col] = __float2half_rn(g);
                    static_cast<__half*>(p.out[2])[row * p.ldo[2] + col] = __float2half_rn(u);
                }
            } else {
                float v = (float)sC[warp][0][e];
                if constexpr (MODE == ANY_I8) {
                    v = v * p.sa[row] * p.sb[col];
                    if (p.bias) v += __half2float(p.bias[col]);
                }
                const long long at = row * p.ldo[z] + col;
                if (p.out_f16)
                    static_cast<__half*>(p.out[z])[at] = __float2half_rn(v);
                else
                    static_cast<float*>(p.out[z])[at] = p.accumulate ? static_cast<float*>(p.out[z])[at] + v : v;
            }
        }
        __syncwarp();
    }
}

template <int MODE>
pax_status_t launch_any(const AnyParams& p, cudaStream_t stream) {
    if (p.M == 0 || p.N == 0) return PAX_OK;
    const int bn = MODE == ANY_GLU ? 64 : 128;
    const long long tiles = ((p.M + 127) / 128) * ((p.N + bn - 1) / bn);
    if (tiles > 0x7fffffffLL) return PAX_ERR_UNSUPPORTED;
    feed_forward_any_kernel<MODE>
        <<<dim3((unsigned)tiles, 1, MODE == ANY_DW ? 2 : 1), kThreads, 0, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? PAX_OK : PAX_ERR_CUDA;
}

}  // namespace

pax_status_t glu_any(const GluProblem& q, cudaStream_t stream) {
    AnyParams p = {};
    p.a[0] = {q.X, q.ldx};
    p.b[0] = {q.Wg, q.ldwg};
    p.b[1] = {q.Wu, q.ldwu};
    p.M = q.M, p.N = q.F, p.R = q.D;
    p.out[0] = q.H, p.out[1] = q.G, p.out[2] = q.U;
    p.ldo[0] = q.ldh, p.ldo[1] = q.ldg, p.ldo[2] = q.ldu;
    p.act = q.act;
    return launch_any<ANY_GLU>(p, stream);
}

pax_status_t glu_dx_any(const GluGradProblem& q, cudaStream_t stream) {
    AnyParams p = {};
    p.a[0] = {q.dG, q.lddg};
    p.a[1] = {q.dU, q.lddu};
    p.b[0] = {q.Wg, q.ldwg};
    p.b[1] = {q.Wu, q.ldwu};
    p.M = q.M, p.N = q.D, p.R = q.F;
    p.out[0] = q.dX, p.ldo[0] = q.lddx;
    p.out_f16 = 1;
    return launch_any<ANY_DX>(p, stream);
}

pax_status_t glu_dw_any(const GluGradProblem& q, cudaStream_t stream) {
    AnyParams p = {};
    p.a[0] = {q.X, q.ldx};
    p.b[0] = {q.dG, q.lddg};
    p.b[1] = {q.dU, q.lddu};
    p.M = q.D, p.N = q.F, p.R = q.M;
    p.out[0] = q.dWg, p.out[1] = q.dWu;
    p.ldo[0] = q.lddwg, p.ldo[1] = q.lddwu;
    p.out_f16 = q.dw_f16, p.accumulate = q.accumulate;
    return launch_any<ANY_DW>(p, stream);
}

pax_status_t gemm_i8_any(const I8Problem& q, cudaStream_t stream) {
    AnyParams p = {};
    p.a[0] = {q.A, q.lda};
    p.b[0] = {q.B, q.ldb};
    p.M = q.M, p.N = q.N, p.R = q.K;
    p.out[0] = q.C, p.ldo[0] = q.ldc;
    p.out_f16 = q.c_f16;
    p.sa = q.a_scale, p.sb = q.b_scale, p.bias = q.bias;
    return launch_any<ANY_I8>(p, stream);
}

}  // namespace pax
