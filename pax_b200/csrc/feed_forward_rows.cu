// feed_forward_rows.cu -- the memory-bound parts of the feed-forward
// products: dG and dU of the gated product's backward pass, and the
// quantisation of rows to int8.
#include "activation.cuh"
#include "feed_forward.h"

namespace pax {

namespace {

__device__ __forceinline__ uint4 ld_stream_v4(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}

// ------------------------------------------------------- dG, dU
// dG = dH U act'(G), dU = dH act(G): reads three matrices and writes two, 10
// bytes an element, and is bound by that.  They are fp16 because they are the
// operands of the two matrix products: in tf32 these would read twice the bytes
// at half the rate.  That costs dX and dW a factor of 1.4 in the 2-norm of
// their error, 2.9e-4 for 2.1e-4, and narrows the gradient's range to fp16's.
//
// With 16-byte aligned rows a thread handles 8 columns at a time, two such
// vectors in flight, else one column.  Every element is read before it is
// written, by the same thread, so dG and dU may be G and U themselves.
constexpr int kGradThreads = 256;

template <int ACT>
__device__ __forceinline__ void grad8(const uint4& vh, const uint4& vg, const uint4& vu, uint4& og, uint4& ou) {
    float h[8], a[8], b[8];
    unpack_h8(vh, h);
    unpack_h8(vg, a);
    unpack_h8(vu, b);
    uint32_t g[4], u[4];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float2 v, d;
        act_value_grad2<ACT>(make_float2(a[i], a[i + 1]), v, d);
        g[i / 2] = pack_half2(h[i] * b[i] * d.x, h[i + 1] * b[i + 1] * d.y);
        u[i / 2] = pack_half2(h[i] * v.x, h[i + 1] * v.y);
    }
    og = make_uint4(g[0], g[1], g[2], g[3]);
    ou = make_uint4(u[0], u[1], u[2], u[3]);
}

// `per_row` vectors (VEC) or elements a row, n = M * per_row in all; Index is
// 32 bits wide where n allows, since a division per vector is what a wider
// one costs most.
template <int ACT, bool VEC, typename Index>
__global__ void __launch_bounds__(kGradThreads) glu_grad_kernel(const GluGradProblem p, Index per_row, Index n) {
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const Index step = (Index)gridDim.x * kGradThreads;
    for (Index i = (Index)blockIdx.x * kGradThreads + threadIdx.x; i < n; i += 2 * step) {
        if constexpr (VEC) {
            uint4 vh[2], vg[2], vu[2];
            long long at[2][2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Index j = i + k * step;
                if (k == 1 && (j >= n || j < i)) break;
                const Index row = j / per_row;
                const long long r = row, c = 8LL * (j - row * per_row);
                vh[k] = ld_stream_v4(p.dH + r * p.lddh + c);
                vg[k] = ld_stream_v4(p.G + r * p.ldg + c);
                vu[k] = ld_stream_v4(p.U + r * p.ldu + c);
                at[k][0] = r * p.lddg + c;
                at[k][1] = r * p.lddu + c;
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Index j = i + k * step;
                if (k == 1 && (j >= n || j < i)) break;
                uint4 og, ou;
                grad8<ACT>(vh[k], vg[k], vu[k], og, ou);
                *reinterpret_cast<uint4*>(p.dG + at[k][0]) = og;
                *reinterpret_cast<uint4*>(p.dU + at[k][1]) = ou;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Index j = i + k * step;
                if (k == 1 && (j >= n || j < i)) break;
                const Index row = j / per_row;
                const long long r = row, c = j - row * per_row;
                const float h = __half2float(p.dH[r * p.lddh + c]), a = __half2float(p.G[r * p.ldg + c]);
                const float b = __half2float(p.U[r * p.ldu + c]);
                float2 v, d;
                act_value_grad2<ACT>(make_float2(a, a), v, d);
                p.dG[r * p.lddg + c] = __float2half_rn(h * b * d.x);
                p.dU[r * p.lddu + c] = __float2half_rn(h * v.x);
            }
        }
    }
}

// A launch that may start while the previous kernel in the stream ends.
template <typename... Params, typename... Args>
pax_status_t launch_rows(void (*kern)(Params...), long long grid, int threads, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, Params(args)...) == cudaSuccess ? PAX_OK : PAX_ERR_CUDA;
}

template <int ACT, bool VEC>
pax_status_t launch_grad_index(const GluGradProblem& p, cudaStream_t stream) {
    const unsigned long long per_row = VEC ? p.F / 8 : p.F, n = per_row * p.M;
    const unsigned long long most = 8ull * device_sm_count(current_device());
    const unsigned long long blocks = (n + 2 * kGradThreads - 1) / (2 * kGradThreads);
    const long long grid = (long long)(blocks < most ? blocks : most);
    // 32 bits: the last index plus two steps has to fit.
    if (n < 0xf0000000ull)
        return launch_rows(glu_grad_kernel<ACT, VEC, unsigned>, grid, kGradThreads, stream, p, per_row, n);
    return launch_rows(glu_grad_kernel<ACT, VEC, unsigned long long>, grid, kGradThreads, stream, p, per_row, n);
}

template <int ACT>
pax_status_t launch_grad(const GluGradProblem& p, cudaStream_t stream) {
    const bool vec = p.F % 8 == 0 && rows16(p.dH, p.lddh, 2) && rows16(p.G, p.ldg, 2) && rows16(p.U, p.ldu, 2) &&
                     rows16(p.dG, p.lddg, 2) && rows16(p.dU, p.lddu, 2);
    return vec ? launch_grad_index<ACT, true>(p, stream) : launch_grad_index<ACT, false>(p, stream);
}

// ------------------------------------------------------- rows to int8
// The largest magnitude of a row is found on the fp16 bit patterns without
// their sign: as integers they order like the magnitudes, and infinities
// (0x7C00) and NaNs sort above every finite value.
//
// A code is round(127 x / m) of the exact quotient.  With x and m of 11
// significant bits, a quotient that is not a tie differs from one by more
// than 1 part in 254 * 2047, about 2^-19, while t = x * (127 / m) in fp32 is
// off by at most 2^-23.  So t is first rounded to 21 significant bits
// (Veltkamp's splitting: p = 9t, hi = p - (p - t)), which restores every tie
// and moves nothing across one, and then to an integer, ties to even, by
// adding 1.5 * 2^23.
__device__ __forceinline__ uint32_t code_bits(float x, float r) {
    const float t = __fmul_rn(x, r);
    const float p = __fmul_rn(t, 9.0f);
    const float hi = __fsub_rn(p, __fsub_rn(p, t));
    return __float_as_uint(__fadd_rn(hi, 12582912.0f)) & 0xffu;  // low byte = two's complement code
}

__device__ __forceinline__ uint32_t max_bits8(uint32_t m, const uint4& v) {
    m = __vmaxu2(m, v.x & 0x7fff7fffu);
    m = __vmaxu2(m, v.y & 0x7fff7fffu);
    m = __vmaxu2(m, v.z & 0x7fff7fffu);
    return __vmaxu2(m, v.w & 0x7fff7fffu);
}

__device__ __forceinline__ uint2 codes8(const uint4& v, float r) {
    float x[8];
    unpack_h8(v, x);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w[i] = code_bits(x[4 * i], r) | code_bits(x[4 * i + 1], r) << 8 | code_bits(x[4 * i + 2], r) << 16 |
               code_bits(x[4 * i + 3], r) << 24;
    return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ uint32_t max_half(uint32_t m) {  // the larger of a word's two halves
    return m >> 16 > (m & 0xffffu) ? m >> 16 : m & 0xffffu;
}

// A row's scale and 127 / max from the bits of its maximum (0 for a row of
// zeros); false for a row with an infinity or a NaN, whose codes are 0.
__device__ __forceinline__ bool row_scale(uint32_t m, float& scale, float& r) {
    const bool finite = m < 0x7C00u;
    const float amax = __half2float(__ushort_as_half((unsigned short)m));
    r = finite && m > 0 ? __fdiv_rn(127.0f, amax) : 0.0f;
    scale = finite ? __fdiv_rn(amax, 127.0f) : __int_as_float(0x7fffffff);
    return finite;
}

template <int THREADS>
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
    __shared__ uint32_t part[THREADS / 32];
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, part[threadIdx.x & (THREADS / 32 - 1)]);
}

// The row stays in registers between the two steps, NV 16-byte vectors a
// thread, so X is read once.  LANES = 32: a warp per row, 8 rows a block;
// LANES = 256: a block per row, for long rows and for few.
template <int LANES, int NV>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const __half* X, long long ldx, int8_t* Q, long long ldq, float* scale, long long M, int units) {
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const int lane = threadIdx.x & (LANES - 1);
    const long long row = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= M) return;  // whole warps
    const __half* x = X + row * ldx;
    int8_t* q = Q + row * ldq;
    uint4 v[NV];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int u = lane + i * LANES;
        v[i] = u < units ? ld_stream_v4(x + 8LL * u) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) m = max_bits8(m, v[i]);
    m = max_half(m);
    if constexpr (LANES == 32)
        m = __reduce_max_sync(0xffffffffu, m);
    else
        m = block_max<256>(m);
    float s, r;
    const bool finite = row_scale(m, s, r);
    if (lane == 0) scale[row] = s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int u = lane + i * LANES;
        if (u < units) *reinterpret_cast<uint2*>(q + 8LL * u) = finite ? codes8(v[i], r) : make_uint2(0u, 0u);
    }
}

// Rows beyond the registers of a block (VEC) and rows that are not 16-byte
// aligned: read a second time for the codes, mostly from L2.
template <bool VEC>
__global__ void __launch_bounds__(256)
    quantize_rows_twice_kernel(const __half* X, long long ldx, int8_t* Q, long long ldq, float* scale, long long K) {
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const long long row = blockIdx.x;
    const __half* x = X + row * ldx;
    int8_t* q = Q + row * ldq;
    uint32_t m = 0;
    if constexpr (VEC) {
        for (long long u = threadIdx.x; u < K / 8; u += 256) m = max_bits8(m, __ldg(reinterpret_cast<const uint4*>(x) + u));
        m = max_half(m);
    } else {
        for (long long j = threadIdx.x; j < K; j += 256) {
            const uint32_t b = __half_as_ushort(x[j]) & 0x7fffu;
            m = b > m ? b : m;
        }
    }
    float s, r;
    const bool finite = row_scale(block_max<256>(m), s, r);
    if (threadIdx.x == 0) scale[row] = s;
    if constexpr (VEC) {
        for (long long u = threadIdx.x; u < K / 8; u += 256)
            reinterpret_cast<uint2*>(q)[u] =
                finite ? codes8(__ldg(reinterpret_cast<const uint4*>(x) + u), r) : make_uint2(0u, 0u);
    } else {
        for (long long j = threadIdx.x; j < K; j += 256)
            q[j] = finite ? (int8_t)code_bits(__half2float(x[j]), r) : (int8_t)0;
    }
}

}  // namespace

pax_status_t glu_grad_rows(const GluGradProblem& p, cudaStream_t stream) {
    if (p.M == 0 || p.F == 0) return PAX_OK;
    if (p.act == ACT_SILU) return launch_grad<ACT_SILU>(p, stream);
    if (p.act == ACT_GELU_TANH) return launch_grad<ACT_GELU_TANH>(p, stream);
    return launch_grad<ACT_GELU_ERF>(p, stream);
}

pax_status_t quantize_rows(const __half* X, long long ldx, int8_t* Q, long long ldq, float* scale, long long M,
                           long long K, cudaStream_t stream) {
    if (M == 0) return PAX_OK;
    const bool vec = K % 8 == 0 && rows16(X, ldx, 2) && (reinterpret_cast<uintptr_t>(Q) & 7u) == 0 && ldq % 8 == 0;
    if (!vec) return launch_rows(quantize_rows_twice_kernel<false>, M, 256, stream, X, ldx, Q, ldq, scale, K);
    if (K > 8 * 256 * 8) return launch_rows(quantize_rows_twice_kernel<true>, M, 256, stream, X, ldx, Q, ldq, scale, K);
    const int units = (int)(K / 8);
    // A warp per row once there are rows enough to fill the SMs that way.
    if (M >= 8LL * device_sm_count(current_device()) && units <= 32 * 16) {
        auto kern = units <= 32       ? quantize_rows_kernel<32, 1>
                    : units <= 32 * 2 ? quantize_rows_kernel<32, 2>
                    : units <= 32 * 4 ? quantize_rows_kernel<32, 4>
                    : units <= 32 * 8 ? quantize_rows_kernel<32, 8>
                                      : quantize_rows_kernel<32, 16>;
        return launch_rows(kern, (M + 7) / 8, 256, stream, X, ldx, Q, ldq, scale, M, units);
    }
    auto kern = units <= 256       ? quantize_rows_kernel<256, 1>
                : units <= 256 * 2 ? quantize_rows_kernel<256, 2>
                : units <= 256 * 4 ? quantize_rows_kernel<256, 4>
                                   : quantize_rows_kernel<256, 8>;
    return launch_rows(kern, M, 256, stream, X, ldx, Q, ldq, scale, M, units);
}

}  // namespace pax
