// feed_forward.h -- host-side interface of the feed-forward products: the
// validated problems that feed_forward.cpp hands to the kernel translation
// units.  Not part of the public ABI.
#pragma once

#include "internal.h"

namespace pax {

// H = act(X.Wg) * (X.Wu); G and U may be null.
struct GluProblem {
    const __half *X, *Wg, *Wu;
    __half *H, *G, *U;
    long long M, D, F;
    long long ldx, ldwg, ldwu, ldh, ldg, ldu;
    int act;
    bool w_const;
};

struct GluGradProblem {
    const __half *dH, *X, *Wg, *Wu, *G, *U;
    __half *dG, *dU, *dX;  // dX may be null
    void *dWg, *dWu;       // may be null
    long long M, D, F;
    long long lddh, ldx, ldwg, ldwu, ldg, ldu, lddg, lddu, lddx, lddwg, lddwu;
    bool dw_f16, accumulate;
    int act;
};

struct I8Problem {
    const int8_t *A, *B;
    void* C;
    const float *a_scale, *b_scale;
    const __half* bias;  // may be null
    long long M, N, K;
    long long lda, ldb, ldc;
    bool c_f16, b_const;
};

// Rows that TMA can read: base and pitch of whole 16-byte units.
inline bool rows16(const void* p, long long ld, int elem) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * elem) % 16 == 0;
}
// Output rows that it may write: a store covers whole 16-byte units, so that a
// width that ends inside one would write beyond it.
inline bool out16(const void* p, long long cols, long long ld, int elem) {
    return rows16(p, ld, elem) && (cols * elem) % 16 == 0;
}

// The longest sum the kernels with bounded waits take: a tile's k-blocks, 2^20
// of 64 (two terms: 2^21), end in about 0.8 s (1.3 s in wide tiles), below the
// waits' limit of 2 s.  Longer ones run on the any-layout kernel, which waits
// for nothing.
constexpr long long kMaxSum = 1LL << 26;

// The most tokens that the few-token kernel's chunks of 64 cover: a grid has
// 65535 of them.
constexpr long long kMaxChunkedTokens = 64LL * 65535;

// The largest of 8, 4 and 2 bytes that all rows start on.
inline int store_unit(const void* p, long long ld, int elem) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * elem);
    return bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

// feed_forward_any.cu: any layout, any alignment, empty sums.
pax_status_t glu_any(const GluProblem& p, cudaStream_t stream);
pax_status_t glu_dx_any(const GluGradProblem& p, cudaStream_t stream);
pax_status_t glu_dw_any(const GluGradProblem& p, cudaStream_t stream);
pax_status_t gemm_i8_any(const I8Problem& p, cudaStream_t stream);

// feed_forward_tc.cu: tcgen05 kernels; *_ok says whether the problem's
// layout lets them, *_time how long they are expected to take, in k-blocks of
// about 0.36 us.  glu_back_tc takes dG and dU as glu_grad_rows left them.
bool glu_tc_ok(const GluProblem& p);
double glu_tc_time(const GluProblem& p);
pax_status_t glu_tc(const GluProblem& p, cudaStream_t stream);
bool glu_back_tc_ok(const GluGradProblem& p);
double glu_back_tc_time(const GluGradProblem& p);
pax_status_t glu_back_tc(const GluGradProblem& p, cudaStream_t stream);
bool gemm_i8_tc_ok(const I8Problem& p);
double gemm_i8_tc_time(const I8Problem& p);
pax_status_t gemm_i8_tc(const I8Problem& p, cudaStream_t stream);
int read_clear_device_error_ff_tc();
bool set_wait_limit_ff_tc(unsigned long long ns);

// feed_forward_split.cu: few tiles with long sums, S CTA pairs to a tile; for
// problems that the tiles of feed_forward_tc.cu take.  A plan's time is in the
// same k-blocks.
struct SplitPlan {
    int S = 0;
    double time = 1e30;
};
SplitPlan glu_split_plan(const GluProblem& p);
pax_status_t glu_split(const GluProblem& p, int S, cudaStream_t stream);
SplitPlan gemm_i8_split_plan(const I8Problem& p);
pax_status_t gemm_i8_split(const I8Problem& p, int S, cudaStream_t stream);
SplitPlan glu_dx_split_plan(const GluGradProblem& p);
pax_status_t glu_dx_split(const GluGradProblem& p, int S, cudaStream_t stream);
SplitPlan glu_dw_split_plan(const GluGradProblem& p);
pax_status_t glu_dw_split(const GluGradProblem& p, int S, cudaStream_t stream);
int read_clear_device_error_ff_split();
bool set_wait_limit_ff_split(unsigned long long ns);

// feed_forward_skinny.cu: few tokens, in chunks of at most 64 (the gated and
// the 8-bit product up to 512), with the same kind of expectation.
bool glu_dx_skinny_ok(const GluGradProblem& p);
double glu_dx_skinny_time(const GluGradProblem& p);
pax_status_t glu_dx_skinny(const GluGradProblem& p, bool beside, cudaStream_t stream);
bool glu_skinny_ok(const GluProblem& p);
double glu_skinny_time(const GluProblem& p);
pax_status_t glu_skinny(const GluProblem& p, cudaStream_t stream);
bool gemm_i8_skinny_ok(const I8Problem& p);
double gemm_i8_skinny_time(const I8Problem& p);
pax_status_t gemm_i8_skinny(const I8Problem& p, cudaStream_t stream);
int read_clear_device_error_ff_skinny();
bool set_wait_limit_ff_skinny(unsigned long long ns);

// feed_forward_rows.cu: the elementwise part of the backward pass, and the
// quantisation of rows.
pax_status_t glu_grad_rows(const GluGradProblem& p, cudaStream_t stream);
pax_status_t quantize_rows(const __half* X, long long ldx, int8_t* Q, long long ldq, float* scale, long long M,
                           long long K, cudaStream_t stream);

}  // namespace pax
