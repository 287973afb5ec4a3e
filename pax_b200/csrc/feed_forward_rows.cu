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
// bytes an element.  A block takes kGradCols columns of one row at a time;
// with 16-byte aligned rows every thread handles 8 columns, else one by one.
// Each thread reads all its inputs before it writes, so dG and dU may be G
// and U themselves.
constexpr int kGradThreads = 256, kGradCols = kGradThreads * 8;

template <int ACT, bool VEC>
__global__ void __launch_bounds__(kGradThreads) glu_grad_kernel(const GluGradProblem p, long long chunks, long long items) {
    for (long long it = blockIdx.x; it < items; it += gridDim.x) {
        const long long row = it / chunks, c0 = (it - row * chunks) * kGradCols;
        const __half* dh = p.dH + row * p.lddh;
        const __half* g = p.G + row * p.ldg;
        const __half* u = p.U + row * p.ldu;
        __half* dg = p.dG + row * p.lddg;
        __half* du = p.dU + row * p.lddu;
        if constexpr (VEC) {
            const long long c = c0 + threadIdx.x * 8;
            if (c >= p.F) continue;
            float h[8], a[8], b[8];
            const uint4 vh = ld_stream_v4(dh + c), vg = ld_stream_v4(g + c), vu = ld_stream_v4(u + c);
            unpack_h8(vh, h);
            unpack_h8(vg, a);
            unpack_h8(vu, b);
            uint32_t og[4], ou[4];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                float v0, d0, v1, d1;
                act_value_grad<ACT>(a[i], v0, d0);
                act_value_grad<ACT>(a[i + 1], v1, d1);
                og[i / 2] = pack_half2(h[i] * b[i] * d0, h[i + 1] * b[i + 1] * d1);
                ou[i / 2] = pack_half2(h[i] * v0, h[i + 1] * v1);
            }
            *reinterpret_cast<uint4*>(dg + c) = make_uint4(og[0], og[1], og[2], og[3]);
            *reinterpret_cast<uint4*>(du + c) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
        } else {
            for (int i = 0; i < 8; ++i) {
                const long long c = c0 + i * kGradThreads + threadIdx.x;
                if (c >= p.F) break;
                const float h = __half2float(dh[c]), a = __half2float(g[c]), b = __half2float(u[c]);
                float v, d;
                act_value_grad<ACT>(a, v, d);
                dg[c] = __float2half_rn(h * b * d);
                du[c] = __float2half_rn(h * v);
            }
        }
    }
}

bool row16(const void* p, long long ld, int elem) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * elem) % 16 == 0;
}

template <int ACT>
pax_status_t launch_grad(const GluGradProblem& p, cudaStream_t stream) {
    const long long chunks = (p.F + kGradCols - 1) / kGradCols, items = chunks * p.M;
    const int dev = current_device();
    const long long most = 8LL * device_sm_count(dev);
    const unsigned grid = (unsigned)(items < most ? items : most);
    const bool vec = p.F % 8 == 0 && row16(p.dH, p.lddh, 2) && row16(p.G, p.ldg, 2) && row16(p.U, p.ldu, 2) &&
                     row16(p.dG, p.lddg, 2) && row16(p.dU, p.lddu, 2);
    if (vec)
        glu_grad_kernel<ACT, true><<<grid, kGradThreads, 0, stream>>>(p, chunks, items);
    else
        glu_grad_kernel<ACT, false><<<grid, kGradThreads, 0, stream>>>(p, chunks, items);
    return cudaGetLastError() == cudaSuccess ? PAX_OK : PAX_ERR_CUDA;
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

// Row maximum over the block, the row's scale, and 127 / max (0 for a row of
// zeros and for one with an infinity or a NaN, whose codes are then masked).
template <int THREADS>
__device__ __forceinline__ bool row_scale(uint32_t m, float* scale, float& r) {
    __shared__ uint32_t part[THREADS / 32];
    m = m >> 16 > (m & 0xffffu) ? m >> 16 : m & 0xffffu;
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (THREADS > 32) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
        __syncthreads();
        m = part[threadIdx.x & (THREADS / 32 - 1)];
        m = __reduce_max_sync(0xffffffffu, m);
    }
    const bool finite = m < 0x7C00u;
    const float amax = __half2float(__ushort_as_half((unsigned short)m));
    r = finite && m > 0 ? __fdiv_rn(127.0f, amax) : 0.0f;
    if (threadIdx.x == 0) *scale = finite ? __fdiv_rn(amax, 127.0f) : __int_as_float(0x7fffffff);
    return finite;
}

// One block per row.  NV > 0: the row stays in registers, NV 16-byte vectors
// a thread, so X is read once.  NV = 0: longer rows and unaligned ones, read
// a second time for the codes (from L2 mostly).
template <int THREADS, int NV>
__global__ void __launch_bounds__(THREADS)
    quantize_rows_kernel(const __half* X, long long ldx, int8_t* Q, long long ldq, float* scale, long long K) {
    const long long row = blockIdx.x;
    const __half* x = X + row * ldx;
    int8_t* q = Q + row * ldq;
    float r;
    if constexpr (NV > 0) {
        const int units = (int)(K / 8);
        uint4 v[NV];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int u = threadIdx.x + i * THREADS;
            v[i] = u < units ? ld_stream_v4(x + 8 * u) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) m = max_bits8(m, v[i]);
        const bool finite = row_scale<THREADS>(m, scale + row, r);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int u = threadIdx.x + i * THREADS;
            if (u < units) *reinterpret_cast<uint2*>(q + 8 * u) = finite ? codes8(v[i], r) : make_uint2(0u, 0u);
        }
    } else {
        uint32_t m = 0;
        for (long long j = threadIdx.x; j < K; j += THREADS) {
            const uint32_t b = __half_as_ushort(x[j]) & 0x7fffu;
            m = b > m ? b : m;
        }
        const bool finite = row_scale<THREADS>(m, scale + row, r);
        for (long long j = threadIdx.x; j < K; j += THREADS)
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
    const unsigned grid = (unsigned)M;
    const bool vec = K % 8 == 0 && row16(X, ldx, 2) && (reinterpret_cast<uintptr_t>(Q) & 7u) == 0 && ldq % 8 == 0;
    if (vec && K <= 8 * 256)
        quantize_rows_kernel<256, 1><<<grid, 256, 0, stream>>>(X, ldx, Q, ldq, scale, K);
    else if (vec && K <= 8 * 256 * 4)
        quantize_rows_kernel<256, 4><<<grid, 256, 0, stream>>>(X, ldx, Q, ldq, scale, K);
    else
        quantize_rows_kernel<256, 0><<<grid, 256, 0, stream>>>(X, ldx, Q, ldq, scale, K);
    return cudaGetLastError() == cudaSuccess ? PAX_OK : PAX_ERR_CUDA;
}

}  // namespace pax
