// feed_forward_any.cu -- the feed-forward products for every layout.
//
// The tensor-memory-accelerator kernels need 16-byte aligned bases and row
// pitches; problems without them, and empty sums, run here.  One kernel for
// the four products
//   gated        H = act(X.Wg) * (X.Wu)          two accumulators, one A
//   input grad   dX = dG.Wg^T + dU.Wu^T          one accumulator, two terms
//   weight grad  dWg = X^T.dG, dWu = X^T.dU      blockIdx.z picks the pair
//   8-bit        C = (A.B^T) * sa * sb + b       int32 accumulators
// with operands addressed by (row stride, reduction stride), so that one
// loader serves every orientation: elements are read one by one, coalesced
// along whichever direction is contiguous, into shared memory, and multiplied
// with 16x16x16 warp matrix operations.  Bound by those element loads.
#include "activation.cuh"
#include "feed_forward.h"

#include <mma.h>

namespace pax {

namespace {

enum : int { ANY_GLU = 0, ANY_SUM = 1, ANY_I8 = 2 };

struct AnyOperand {
    const void* p;
    long long outer, red;  // element strides along the output row / column and along the sum
};

struct AnyParams {
    AnyOperand a[2], b[2];  // ANY_SUM: sum over the terms; ANY_GLU: b[1] is the up projection
    int terms;
    int pick;               // ANY_SUM: blockIdx.z picks b and out instead of summing terms
    long long M, N, R;
    void* out[3];
    long long ldo[3];
    int out_f16, accumulate, act;
    const float *sa, *sb;
    const __half* bias;
};

constexpr int kT = 64, kR = 32, kPad = 16;  // output tile, reduction step, row padding (elements)

template <typename T>
__device__ __forceinline__ void any_load(T* s, const AnyOperand& o, long long o0, long long omax, long long r0,
                                         long long rmax) {
    const T* p = static_cast<const T*>(o.p);
    const bool along_red = o.red == 1;
    for (int i = threadIdx.x; i < kT * kR; i += 128) {
        const int x = along_red ? i / kR : i % kT, r = along_red ? i % kR : i / kT;
        const long long go = o0 + x, gr = r0 + r;
        T v = T(0);
        if (go < omax && gr < rmax) v = p[go * o.outer + gr * o.red];
        s[x * (kR + kPad) + r] = v;
    }
}

template <int MODE>
__global__ void __launch_bounds__(128) feed_forward_any_kernel(const AnyParams p) {
    using namespace nvcuda;
    using T = typename std::conditional<MODE == ANY_I8, signed char, __half>::type;
    using Acc = typename std::conditional<MODE == ANY_I8, int, float>::type;
    constexpr int NACC = MODE == ANY_GLU ? 2 : 1;
    // The operand tiles, and after the last step the accumulators.
    constexpr int kTile = kT * (kR + kPad);
    constexpr int kOps = (1 + NACC) * kTile * (int)sizeof(T), kAcc = NACC * kT * (kT + 8) * (int)sizeof(Acc);
    __shared__ __align__(128) unsigned char raw[kOps > kAcc ? kOps : kAcc];
    T* sA = reinterpret_cast<T*>(raw);
    T* sB[NACC];
#pragma unroll
    for (int c = 0; c < NACC; ++c) sB[c] = sA + (1 + c) * kTile;
    auto sC = reinterpret_cast<Acc(*)[kT][kT + 8]>(raw);
    const long long tiles_n = (p.N + kT - 1) / kT;
    const long long m0 = (long long)blockIdx.x / tiles_n * kT, n0 = (long long)blockIdx.x % tiles_n * kT;
    const int warp = threadIdx.x >> 5, wm = (warp >> 1) * 32, wn = (warp & 1) * 32;
    const int z = p.pick ? (int)blockIdx.z : 0;

    wmma::fragment<wmma::accumulator, 16, 16, 16, Acc> acc[NACC][2][2];
#pragma unroll
    for (int c = 0; c < NACC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) wmma::fill_fragment(acc[c][i >> 1][i & 1], Acc(0));
    const int terms = MODE == ANY_SUM && !p.pick ? p.terms : 1;
    for (int t = 0; t < terms; ++t) {
        for (long long r0 = 0; r0 < p.R; r0 += kR) {
            any_load<T>(sA, p.a[t], m0, p.M, r0, p.R);
#pragma unroll
            for (int c = 0; c < NACC; ++c) any_load<T>(sB[c], p.b[MODE == ANY_GLU ? c : t + z], n0, p.N, r0, p.R);
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < kR; kk += 16) {
                wmma::fragment<wmma::matrix_a, 16, 16, 16, T, wmma::row_major> fa[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    wmma::load_matrix_sync(fa[i], sA + (wm + 16 * i) * (kR + kPad) + kk, kR + kPad);
#pragma unroll
                for (int c = 0; c < NACC; ++c)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        wmma::fragment<wmma::matrix_b, 16, 16, 16, T, wmma::col_major> fb;
                        wmma::load_matrix_sync(fb, sB[c] + (wn + 16 * j) * (kR + kPad) + kk, kR + kPad);
#pragma unroll
                        for (int i = 0; i < 2; ++i) wmma::mma_sync(acc[c][i][j], fa[i], fb, acc[c][i][j]);
                    }
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int c = 0; c < NACC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            wmma::store_matrix_sync(&sC[c][wm + 16 * (i >> 1)][wn + 16 * (i & 1)], acc[c][i >> 1][i & 1], kT + 8,
                                    wmma::mem_row_major);
    __syncthreads();
    for (int i = threadIdx.x; i < kT * kT; i += 128) {
        const int r = i / kT, c = i % kT;
        const long long row = m0 + r, col = n0 + c;
        if (row >= p.M || col >= p.N) continue;
        if constexpr (MODE == ANY_GLU) {
            const float g = sC[0][r][c], u = sC[NACC - 1][r][c];
            static_cast<__half*>(p.out[0])[row * p.ldo[0] + col] = __float2half_rn(act_value_rt(p.act, g) * u);
            if (p.out[1]) {
                static_cast<__half*>(p.out[1])[row * p.ldo[1] + col] = __float2half_rn(g);
                static_cast<__half*>(p.out[2])[row * p.ldo[2] + col] = __float2half_rn(u);
            }
        } else {
            float v = (float)sC[0][r][c];
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
}

template <int MODE>
pax_status_t launch_any(const AnyParams& p, int z, cudaStream_t stream) {
    if (p.M == 0 || p.N == 0) return PAX_OK;
    const long long tiles = ((p.M + kT - 1) / kT) * ((p.N + kT - 1) / kT);
    if (tiles > 0x7fffffffLL) return PAX_ERR_UNSUPPORTED;
    feed_forward_any_kernel<MODE><<<dim3((unsigned)tiles, 1, (unsigned)z), 128, 0, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? PAX_OK : PAX_ERR_CUDA;
}

}  // namespace

pax_status_t glu_any(const GluProblem& q, cudaStream_t stream) {
    AnyParams p = {};
    p.a[0] = {q.X, q.ldx, 1};
    p.b[0] = {q.Wg, 1, q.ldwg};
    p.b[1] = {q.Wu, 1, q.ldwu};
    p.M = q.M, p.N = q.F, p.R = q.D;
    p.out[0] = q.H, p.out[1] = q.G, p.out[2] = q.U;
    p.ldo[0] = q.ldh, p.ldo[1] = q.ldg, p.ldo[2] = q.ldu;
    p.act = q.act;
    return launch_any<ANY_GLU>(p, 1, stream);
}

pax_status_t glu_dx_any(const GluGradProblem& q, cudaStream_t stream) {
    AnyParams p = {};
    p.a[0] = {q.dG, q.lddg, 1};
    p.a[1] = {q.dU, q.lddu, 1};
    p.b[0] = {q.Wg, q.ldwg, 1};
    p.b[1] = {q.Wu, q.ldwu, 1};
    p.terms = 2;
    p.M = q.M, p.N = q.D, p.R = q.F;
    p.out[0] = q.dX, p.ldo[0] = q.lddx;
    p.out_f16 = 1;
    return launch_any<ANY_SUM>(p, 1, stream);
}

pax_status_t glu_dw_any(const GluGradProblem& q, cudaStream_t stream) {
    AnyParams p = {};
    p.a[0] = {q.X, 1, q.ldx};
    p.b[0] = {q.dG, 1, q.lddg};
    p.b[1] = {q.dU, 1, q.lddu};
    p.pick = 1;
    p.M = q.D, p.N = q.F, p.R = q.M;
    p.out[0] = q.dWg, p.out[1] = q.dWu;
    p.ldo[0] = q.lddwg, p.ldo[1] = q.lddwu;
    p.out_f16 = q.dw_f16, p.accumulate = q.accumulate;
    return launch_any<ANY_SUM>(p, 2, stream);
}

pax_status_t gemm_i8_any(const I8Problem& q, cudaStream_t stream) {
    AnyParams p = {};
    p.a[0] = {q.A, q.lda, 1};
    p.b[0] = {q.B, q.ldb, 1};
    p.M = q.M, p.N = q.N, p.R = q.K;
    p.out[0] = q.C, p.ldo[0] = q.ldc;
    p.out_f16 = q.c_f16;
    p.sa = q.a_scale, p.sb = q.b_scale, p.bias = q.bias;
    return launch_any<ANY_I8>(p, 1, stream);
}

}  // namespace pax
