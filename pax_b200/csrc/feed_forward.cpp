// feed_forward.cpp -- C entries of the feed-forward products: argument
// checks, and the choice between the tcgen05 kernels and the any-layout
// kernel.  No entry allocates, synchronises or throws.
#include "feed_forward.h"

#include <stdarg.h>
#include <stdio.h>

namespace pax {

namespace {

pax_status_t refuse(pax_status_t s, const char* fmt, ...) {
    char msg[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    return report_status(s, msg);
}

// Room for the kernels' rounded-up tile coordinates in 32 bits.
constexpr long long kMaxDim = 0x7fffffffLL - 1024;

bool dim_ok(long long v) { return v >= 0 && v <= kMaxDim; }

// A matrix operand of T: rows x cols with its leading dimension (0: cols).
// False when it has elements but no base, a base that is not aligned to its
// elements, or overlapping rows.  A single row has no pitch; it gets one that
// any kernel takes, so that its length alone keeps no product off the
// tensor-core kernels (one token of 1001 features beside padded weights).
bool matrix_ok_sized(const void* base, size_t elem, long long rows, long long cols, long long* ld) {
    if (*ld == 0) *ld = cols;
    if (rows == 0 || cols == 0) return true;
    if (base == nullptr || reinterpret_cast<uintptr_t>(base) % elem != 0 || *ld < cols || *ld >= (1LL << 38))
        return false;
    if (rows == 1) *ld = (cols + 15) / 16 * 16;
    return true;
}
template <typename T>
bool matrix_ok(const T* base, long long rows, long long cols, long long* ld) {
    return matrix_ok_sized(base, sizeof(T), rows, cols, ld);
}

pax_status_t device_ok(const char* who) {
    const int dev = current_device();
    int major = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10) {
        cudaGetLastError();
        return refuse(PAX_ERR_NO_DEVICE, "%s: device %d is not sm_100", who, dev);
    }
    return PAX_OK;
}

// Beyond 64 tokens: whether chunks of 64 on the few-token kernel, which
// splits K, end sooner than tiles of 256 rows.  Both times come in k-blocks of
// 0.36 us; a chunk's k-block also carries 64 tokens (0.47 us) and the kernel
// about 5 us besides.  8-bit 128x4096x4096 takes 12.7 us in chunks and 15.3
// in tiles, 256x1024x4096 10.8 and 14.2, but 128x11264x4096 24.0 and 17.5.
bool chunks_pay(double chunks, double tiles) { return 1.15 * (0.47 * chunks + 5.0) < 0.36 * tiles + 1.0; }

// dX and the weight gradients, from dG and dU.  Both in one launch of tiles,
// where dX's few and long tiles do not keep it waiting; else dX apart, split
// along F by clusters of pairs or, for few tokens, on the few-token kernel, and
// the weight gradients in tiles or split along the tokens.  A second launch
// counts as 6 k-blocks, about 2 us; a k-block of the few-token kernel, with 64
// tokens beside it, as 1.3.  The choice goes by the shape, not by which
// gradients are asked for, so that they have the same bits either way.
pax_status_t back_products(const GluGradProblem& p, cudaStream_t stream) {
    if (p.M == 0 || p.D == 0 || p.F == 0) {
        const pax_status_t st = p.dX ? glu_dx_any(p, stream) : PAX_OK;
        return st == PAX_OK && p.dWg ? glu_dw_any(p, stream) : st;
    }
    GluGradProblem x = p, w = p, both = p;
    // What both together, dX alone and the weight gradients alone would take;
    // the pointers stand for "asked for" and are not read.
    both.dX = x.dX = p.dX ? p.dX : p.dG;
    both.dWg = both.dWu = w.dWg = w.dWu = p.dWg ? p.dWg : static_cast<void*>(p.dG);
    x.dWg = x.dWu = nullptr;
    w.dX = nullptr;
    const SplitPlan xs = glu_dx_split_plan(p), ws = glu_dw_split_plan(p);
    // A kernel that cannot run dX's shape has no time: dX apart is then left to
    // the tiles (8388608x64x64: too many chunks, too few k-blocks to split).
    const bool chunked = p.M <= kMaxChunkedTokens, split = xs.S > 0;
    const double few = chunked ? 1.3 * glu_dx_skinny_time(p) + 8.0 : 1e30, wt = glu_back_tc_time(w);
    const double x_time = !chunked && !split ? glu_back_tc_time(x) : few < xs.time ? few : xs.time;
    const double w_time = wt < ws.time ? wt : ws.time;
    const bool apart = x_time + w_time + 6.0 < glu_back_tc_time(both);

    GluGradProblem px = p, pw = p;  // each part as asked for
    px.dWg = px.dWu = nullptr;
    pw.dX = nullptr;
    pax_status_t st = PAX_OK;
    if (!apart && glu_back_tc_ok(p)) return glu_back_tc(p, stream);
    // The weight gradients first: dX's few-token kernel can run beside them.
    bool beside = false;
    if (p.dWg) {
        if (!glu_back_tc_ok(pw)) {
            st = glu_dw_any(pw, stream);
        } else {
            beside = true;
            st = apart && ws.time < wt ? glu_dw_split(pw, ws.S, stream) : glu_back_tc(pw, stream);
        }
    }
    if (st != PAX_OK || !p.dX) return st;
    const bool tiles_ok = glu_back_tc_ok(px);
    if (glu_dx_skinny_ok(p) && (!tiles_ok || (apart && few < xs.time))) return glu_dx_skinny(p, beside, stream);
    if (!tiles_ok) return glu_dx_any(px, stream);
    return apart && split ? glu_dx_split(px, xs.S, stream) : glu_back_tc(px, stream);
}

pax_status_t done(pax_status_t st, const char* who) {
    if (st == PAX_OK) return report_status(PAX_OK, "");
    return refuse(st, "%s: launch failed (%s)", who, pax_status_string(st));
}

pax_status_t check_glu(const pax_glu_desc_t* d, GluProblem* p) {
    static const char* who = "pax_glu_ex";
    if (!d) return refuse(PAX_ERR_INVALID, "%s: NULL descriptor", who);
    if (!dim_ok(d->M) || !dim_ok(d->D) || !dim_ok(d->F))
        return refuse(PAX_ERR_INVALID, "%s: bad shape m=%lld d=%lld f=%lld", who, (long long)d->M, (long long)d->D,
                      (long long)d->F);
    if (d->act < PAX_ACT_SILU || d->act > PAX_ACT_GELU_ERF)
        return refuse(PAX_ERR_INVALID, "%s: bad activation %d", who, (int)d->act);
    p->X = static_cast<const __half*>(d->X);
    p->Wg = static_cast<const __half*>(d->Wg);
    p->Wu = static_cast<const __half*>(d->Wu);
    p->H = static_cast<__half*>(d->H);
    p->G = static_cast<__half*>(d->G);
    p->U = static_cast<__half*>(d->U);
    p->M = d->M, p->D = d->D, p->F = d->F;
    p->ldx = d->ldx, p->ldwg = d->ldwg, p->ldwu = d->ldwu, p->ldh = d->ldh, p->ldg = d->ldg, p->ldu = d->ldu;
    p->act = (int)d->act;
    p->w_const = d->w_const != 0;
    if (p->M == 0 || p->F == 0) return PAX_OK;
    if ((p->G != nullptr) != (p->U != nullptr)) return refuse(PAX_ERR_INVALID, "%s: G and U go together", who);
    if (!matrix_ok(p->X, p->M, p->D, &p->ldx) || !matrix_ok(p->Wg, p->D, p->F, &p->ldwg) ||
        !matrix_ok(p->Wu, p->D, p->F, &p->ldwu) || !matrix_ok(p->H, p->M, p->F, &p->ldh) ||
        (p->G && (!matrix_ok(p->G, p->M, p->F, &p->ldg) || !matrix_ok(p->U, p->M, p->F, &p->ldu))))
        return refuse(PAX_ERR_INVALID, "%s: NULL or misaligned operand, or leading dimension smaller than the row length", who);
    return PAX_OK;
}

pax_status_t check_grad(const pax_glu_grad_desc_t* d, GluGradProblem* p) {
    static const char* who = "pax_glu_backward_ex";
    if (!d) return refuse(PAX_ERR_INVALID, "%s: NULL descriptor", who);
    if (!dim_ok(d->M) || !dim_ok(d->D) || !dim_ok(d->F))
        return refuse(PAX_ERR_INVALID, "%s: bad shape m=%lld d=%lld f=%lld", who, (long long)d->M, (long long)d->D,
                      (long long)d->F);
    if (d->act < PAX_ACT_SILU || d->act > PAX_ACT_GELU_ERF)
        return refuse(PAX_ERR_INVALID, "%s: bad activation %d", who, (int)d->act);
    if (d->dw_dtype != PAX_DT_F32 && d->dw_dtype != PAX_DT_F16)
        return refuse(PAX_ERR_INVALID, "%s: bad weight gradient dtype %d", who, (int)d->dw_dtype);
    if (d->accumulate && d->dw_dtype != PAX_DT_F32)
        return refuse(PAX_ERR_INVALID, "%s: accumulation needs fp32 weight gradients", who);
    p->dH = static_cast<const __half*>(d->dH);
    p->X = static_cast<const __half*>(d->X);
    p->Wg = static_cast<const __half*>(d->Wg);
    p->Wu = static_cast<const __half*>(d->Wu);
    p->G = static_cast<const __half*>(d->G);
    p->U = static_cast<const __half*>(d->U);
    p->dG = static_cast<__half*>(d->dG);
    p->dU = static_cast<__half*>(d->dU);
    p->dX = static_cast<__half*>(d->dX);
    p->dWg = d->dWg;
    p->dWu = d->dWu;
    p->M = d->M, p->D = d->D, p->F = d->F;
    p->lddh = d->lddh, p->ldx = d->ldx, p->ldwg = d->ldwg, p->ldwu = d->ldwu, p->ldg = d->ldg, p->ldu = d->ldu;
    p->lddg = d->lddg, p->lddu = d->lddu, p->lddx = d->lddx, p->lddwg = d->lddwg, p->lddwu = d->lddwu;
    p->dw_f16 = d->dw_dtype == PAX_DT_F16;
    p->accumulate = d->accumulate != 0;
    p->act = (int)d->act;
    // Empty matrices have no address in some callers: what they would feed is
    // decided by the shapes.
    if (p->D > 0 && p->F > 0 && (p->dWg != nullptr) != (p->dWu != nullptr))
        return refuse(PAX_ERR_INVALID, "%s: dWg and dWu go together", who);
    const bool dx = p->dX != nullptr, dw = p->dWg != nullptr;
    if (!matrix_ok(p->dH, p->M, p->F, &p->lddh) || !matrix_ok(p->G, p->M, p->F, &p->ldg) ||
        !matrix_ok(p->U, p->M, p->F, &p->ldu) || !matrix_ok(p->dG, p->M, p->F, &p->lddg) ||
        !matrix_ok(p->dU, p->M, p->F, &p->lddu) || (dw && !matrix_ok(p->X, p->M, p->D, &p->ldx)) ||
        (dx && (!matrix_ok(p->Wg, p->D, p->F, &p->ldwg) || !matrix_ok(p->Wu, p->D, p->F, &p->ldwu) ||
                !matrix_ok(p->dX, p->M, p->D, &p->lddx))) ||
        (dw && (!matrix_ok_sized(p->dWg, p->dw_f16 ? 2 : 4, p->D, p->F, &p->lddwg) ||
                !matrix_ok_sized(p->dWu, p->dw_f16 ? 2 : 4, p->D, p->F, &p->lddwu))))
        return refuse(PAX_ERR_INVALID, "%s: NULL or misaligned operand, or leading dimension smaller than the row length", who);
    // In place means element by element: one buffer, one pitch.
    const struct {
        const __half* base;
        long long ld;
    } outs[2] = {{p->dG, p->lddg}, {p->dU, p->lddu}}, ins[3] = {{p->dH, p->lddh}, {p->G, p->ldg}, {p->U, p->ldu}};
    for (const auto& o : outs)
        for (const auto& i : ins)
            if (p->M > 1 && p->F > 0 && o.base == i.base && o.ld != i.ld)
                return refuse(PAX_ERR_INVALID, "%s: dG or dU in place of an input needs its leading dimension", who);
    if (p->M > 0 && p->F > 0 && p->dG == p->dU)
        return refuse(PAX_ERR_INVALID, "%s: dG and dU are one buffer", who);
    return PAX_OK;
}

pax_status_t check_i8(const pax_gemm_i8_desc_t* d, I8Problem* p) {
    static const char* who = "pax_gemm_i8_ex";
    if (!d) return refuse(PAX_ERR_INVALID, "%s: NULL descriptor", who);
    if (!dim_ok(d->M) || !dim_ok(d->N) || !dim_ok(d->K))
        return refuse(PAX_ERR_INVALID, "%s: bad shape m=%lld n=%lld k=%lld", who, (long long)d->M, (long long)d->N,
                      (long long)d->K);
    // 131071 products of two codes of -128 sum to less than 2^31.
    if (d->K > 131071)
        return refuse(PAX_ERR_INVALID, "%s: k=%lld above 131071, the sum could leave int32", who, (long long)d->K);
    if (d->c_dtype != PAX_DT_F32 && d->c_dtype != PAX_DT_F16)
        return refuse(PAX_ERR_INVALID, "%s: bad output dtype %d", who, (int)d->c_dtype);
    p->A = static_cast<const int8_t*>(d->A);
    p->B = static_cast<const int8_t*>(d->B);
    p->C = d->C;
    p->a_scale = d->a_scale;
    p->b_scale = d->b_scale;
    p->bias = static_cast<const __half*>(d->bias);
    p->M = d->M, p->N = d->N, p->K = d->K;
    p->lda = d->lda, p->ldb = d->ldb, p->ldc = d->ldc;
    p->c_f16 = d->c_dtype == PAX_DT_F16;
    p->b_const = d->b_const != 0;
    if (p->M == 0 || p->N == 0) return PAX_OK;
    if (!matrix_ok(p->A, p->M, p->K, &p->lda) || !matrix_ok(p->B, p->N, p->K, &p->ldb) ||
        !matrix_ok_sized(p->C, p->c_f16 ? 2 : 4, p->M, p->N, &p->ldc))
        return refuse(PAX_ERR_INVALID, "%s: NULL or misaligned operand, or leading dimension smaller than the row length", who);
    if (!p->a_scale || !p->b_scale) return refuse(PAX_ERR_INVALID, "%s: NULL scales", who);
    if (((reinterpret_cast<uintptr_t>(p->a_scale) | reinterpret_cast<uintptr_t>(p->b_scale)) & 3u) ||
        (reinterpret_cast<uintptr_t>(p->bias) & 1u))
        return refuse(PAX_ERR_INVALID, "%s: scales or bias not aligned to their elements", who);
    return PAX_OK;
}

}  // namespace

}  // namespace pax

using namespace pax;

extern "C" {

pax_status_t pax_glu_ex(const pax_glu_desc_t* desc, cudaStream_t stream) {
    GluProblem p;
    pax_status_t st = check_glu(desc, &p);
    if (st != PAX_OK) return st;
    if (p.M == 0 || p.F == 0) return report_status(PAX_OK, "");
    if ((st = device_ok("pax_glu_ex")) != PAX_OK) return st;
    if (glu_skinny_ok(p) && p.M <= 64) return done(glu_skinny(p, stream), "pax_glu_ex");
    if (glu_tc_ok(p)) {
        const double tiles = glu_tc_time(p);
        const SplitPlan split = glu_split_plan(p);
        if (glu_skinny_ok(p) && chunks_pay(glu_skinny_time(p), tiles < split.time ? tiles : split.time))
            st = glu_skinny(p, stream);
        else
            st = split.time < tiles ? glu_split(p, split.S, stream) : glu_tc(p, stream);
    } else {
        st = glu_skinny_ok(p) ? glu_skinny(p, stream) : glu_any(p, stream);
    }
    return done(st, "pax_glu_ex");
}

pax_status_t pax_glu_backward_ex(const pax_glu_grad_desc_t* desc, cudaStream_t stream) {
    GluGradProblem p;
    pax_status_t st = check_grad(desc, &p);
    if (st != PAX_OK) return st;
    if (p.M == 0 && (p.D == 0 || p.F == 0 || !p.dWg)) return report_status(PAX_OK, "");
    if ((st = device_ok("pax_glu_backward_ex")) != PAX_OK) return st;
    st = glu_grad_rows(p, stream);
    if (st == PAX_OK && (p.dX || p.dWg)) {
        st = back_products(p, stream);
    }
    return done(st, "pax_glu_backward_ex");
}

pax_status_t pax_quantize_rows(const void* X, int64_t ldx, void* Q, int64_t ldq, float* scale, int64_t M, int64_t K,
                               cudaStream_t stream) {
    static const char* who = "pax_quantize_rows";
    if (!dim_ok(M) || !dim_ok(K))
        return refuse(PAX_ERR_INVALID, "%s: bad shape m=%lld k=%lld", who, (long long)M, (long long)K);
    if (M == 0) return report_status(PAX_OK, "");
    long long lx = ldx, lq = ldq;
    if (!scale || (reinterpret_cast<uintptr_t>(scale) & 3u) || !matrix_ok_sized(X, 2, M, K, &lx) ||
        !matrix_ok_sized(Q, 1, M, K, &lq))
        return refuse(PAX_ERR_INVALID, "%s: NULL or misaligned operand, or leading dimension smaller than the row length", who);
    pax_status_t st = device_ok(who);
    if (st != PAX_OK) return st;
    return done(quantize_rows(static_cast<const __half*>(X), lx, static_cast<int8_t*>(Q), lq, scale, M, K, stream),
                who);
}

pax_status_t pax_gemm_i8_ex(const pax_gemm_i8_desc_t* desc, cudaStream_t stream) {
    I8Problem p;
    pax_status_t st = check_i8(desc, &p);
    if (st != PAX_OK) return st;
    if (p.M == 0 || p.N == 0) return report_status(PAX_OK, "");
    if ((st = device_ok("pax_gemm_i8_ex")) != PAX_OK) return st;
    if (gemm_i8_skinny_ok(p) && p.M <= 64) return done(gemm_i8_skinny(p, stream), "pax_gemm_i8_ex");
    if (gemm_i8_tc_ok(p)) {
        const double tiles = gemm_i8_tc_time(p);
        const SplitPlan split = gemm_i8_split_plan(p);
        if (gemm_i8_skinny_ok(p) && chunks_pay(gemm_i8_skinny_time(p), tiles < split.time ? tiles : split.time))
            st = gemm_i8_skinny(p, stream);
        else
            st = split.time < tiles ? gemm_i8_split(p, split.S, stream) : gemm_i8_tc(p, stream);
    } else {
        st = gemm_i8_skinny_ok(p) ? gemm_i8_skinny(p, stream) : gemm_i8_any(p, stream);
    }
    return done(st, "pax_gemm_i8_ex");
}

size_t pax_sizeof_feed_forward_desc(int which) {
    return which == 0   ? sizeof(pax_glu_desc_t)
           : which == 1 ? sizeof(pax_glu_grad_desc_t)
           : which == 2 ? sizeof(pax_gemm_i8_desc_t)
                        : 0;
}

}  // extern "C"
