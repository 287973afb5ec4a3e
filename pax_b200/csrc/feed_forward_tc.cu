// feed_forward_tc.cu -- launches of the tcgen05 feed-forward kernel
// (feed_forward_tc.cuh).
#include "feed_forward_tc.cuh"

namespace pax {

namespace {

int up(long long a, int b) { return (int)((a + b - 1) / b); }

// Tiles run in column-major groups of this many tile rows (as in
// gemm_tc.cuh, where 16 measured best at every shape).
constexpr int kGroupM = 16;

// Which tile width: the time in k-blocks of the narrow tile, about 0.36 us
// each.  A k-block of the wide tile takes 1.62 of them for twice the work;
// its epilogue, not overlapped, about 12 (measured over K = 64 to 2048 on
// 777 x 4104 .. 9472; the last epilogue of a narrow tile about 8).
// 4096x4096x11264 takes 608-628 us with the wide tile and 646 with the
// narrow one, 777x1024x4736 (148 narrow tiles) 27.2 and 17.3 us.
constexpr double kWideBlock = 1.62, kWideEpilogue = 12.0, kLastEpilogue = 8.0;

double tile_cost(int w, int kbs) { return w == 2 ? kbs * kWideBlock + kWideEpilogue : kbs; }

int rounds(long long tiles, int units) { return (int)((tiles + units - 1) / units); }

// What a piece of a narrow tile costs: half and quarter widths stage and
// multiply less per k-block, but A in full, and have a shorter epilogue.
double piece_cost(int pieces, int kbs) {
    return pieces == 4 ? 0.6 * kbs + 3.0 : pieces == 2 ? 0.75 * kbs + 5.0 : kbs + kLastEpilogue;
}

// Whole rounds of narrow tiles, and the rest in the number of column pieces
// that ends soonest; returns the time.  1235x4099x2064 has 85 tiles on 74
// pairs: 11 left over.
double plan_pieces(FfParams& p, int tiles, int units, int most) {
    const int rest = tiles % units;
    p.full = tiles - rest;
    p.pieces = 1;
    const double whole = (double)(p.full / units) * p.kbs;
    double best = rest == 0 ? kLastEpilogue : piece_cost(1, p.kbs);
    for (int n = 2; n <= most && rest > 0; n *= 2) {
        const double t = rounds((long long)rest * n, units) * piece_cost(n, p.kbs);
        if (t < best) {
            best = t;
            p.pieces = n;
        }
    }
    return whole + best;
}

int ff_grid(const FfParams& p, int tiles, int units) {
    const int items = p.full + (tiles - p.full) * p.pieces;
    return items < units ? items : units;
}

// The tile width of the gated product, 1 or 2, and its tiles for that many
// CTA pairs of each width; the grid in pairs.
int plan_glu(FfParams& p, int units, int units2, int& grid) {
    p.tiles_n = up(p.N, 128);
    const int tiles = p.tiles_m * p.tiles_n, tiles2 = p.tiles_m * up(p.N, 256);
    if (rounds(tiles2, units2) * tile_cost(2, p.kbs) < plan_pieces(p, tiles, units, 2)) {
        p.tiles_n = up(p.N, 256);
        p.full = tiles2;
        p.pieces = 1;
        grid = tiles2 < units2 ? tiles2 : units2;
        return 2;
    }
    grid = ff_grid(p, tiles, units);
    return 1;
}

template <int ACT>
pax_status_t launch_glu(const FfMaps& maps, FfParams& p, cudaStream_t stream) {
    const int units = ff_units<FF_GLU, ACT, __half, 1>(current_device());
    const int units2 = ff_units<FF_GLU, ACT, __half, 2>(current_device());
    if (units <= 0 || units2 <= 0) return PAX_ERR_CUDA;
    int grid;
    return plan_glu(p, units, units2, grid) == 2 ? ff_launch<FF_GLU, ACT, __half, 2>(maps, p, grid, stream)
                                                 : ff_launch<FF_GLU, ACT, __half, 1>(maps, p, grid, stream);
}

// The gradients' tiles of width w and their schedule on at most `most` CTA
// pairs; the grid in pairs.
int plan_back(FfParams& p, int w, int most) {
    p.tiles_n = up(p.D, 256 * w);
    p.wt_n = up(p.F, 256 * w);
    p.nx = p.nx ? p.tiles_m * p.tiles_n : 0;
    p.nw = p.nw ? p.wt_m * 2 * p.wt_n : 0;
    const long long items = (long long)p.nx + p.nw;
    const int units = (int)(items < most ? items : most);
    p.x_rem = p.nx % units;
    p.w_extra = 0;
    if (p.x_rem > 0 && p.nw > 0) p.w_extra = (p.kbs + p.kbs_w / 2) / p.kbs_w;
    return units;
}

template <typename OutT, int W>
pax_status_t launch_back_w(const FfMaps& maps, FfParams& p, cudaStream_t stream) {
    const int most = ff_units<FF_BACK, 0, OutT, W>(current_device());
    if (most <= 0) return PAX_ERR_CUDA;
    const int units = plan_back(p, W, most);
    return ff_launch<FF_BACK, 0, OutT, W>(maps, p, units, stream);
}
// The time of both gradients in one launch with tiles of width w.  The weight
// gradients fill up what dX's tiles leave uneven; a launch ends no earlier
// than its longest tile.
double back_time(const FfParams& p, int w, int units) {
    const double x = p.nx ? tile_cost(w, p.kbs) : 0, y = p.nw ? tile_cost(w, p.kbs_w) : 0;
    const long long nx = p.nx ? (long long)p.tiles_m * up(p.D, 256 * w) : 0;
    const long long nw = p.nw ? 2LL * p.wt_m * up(p.F, 256 * w) : 0;
    double t = p.nx && p.nw ? (nx * x + nw * y) / units + 0.5 * y : rounds(nx, units) * x + rounds(nw, units) * y;
    if (t < x) t = x;
    if (t < y) t = y;
    return t + (w == 1 ? kLastEpilogue : 0);
}

int back_width(const FfParams& p, int units) { return back_time(p, 2, units) < back_time(p, 1, units) ? 2 : 1; }

template <typename OutT>
pax_status_t launch_back(const FfMaps& maps, FfParams& p, cudaStream_t stream) {
    const int units = ff_units<FF_BACK, 0, OutT, 1>(current_device());
    if (units <= 0) return PAX_ERR_CUDA;
    return back_width(p, units) == 2 ? launch_back_w<OutT, 2>(maps, p, stream) : launch_back_w<OutT, 1>(maps, p, stream);
}

template <typename OutT>
pax_status_t launch_i8(const FfMaps& maps, FfParams& p, cudaStream_t stream) {
    const int units = ff_units<FF_I8, 0, OutT, 1>(current_device());
    if (units <= 0) return PAX_ERR_CUDA;
    p.tiles_n = up(p.N, 256);
    const int tiles = p.tiles_m * p.tiles_n;
    plan_pieces(p, tiles, units, 4);
    return ff_launch<FF_I8, 0, OutT, 1>(maps, p, ff_grid(p, tiles, units), stream);
}

bool tiles_ok(long long a, long long b) { return a * b <= 0x3fffffffLL; }

}  // namespace

bool glu_tc_ok(const GluProblem& q) {
    return q.D > 0 && q.D <= kMaxSum && rows16(q.X, q.ldx, 2) && rows16(q.Wg, q.ldwg, 2) && rows16(q.Wu, q.ldwu, 2) &&
           out16(q.H, q.F, q.ldh, 2) && (!q.G || (out16(q.G, q.F, q.ldg, 2) && out16(q.U, q.F, q.ldu, 2))) &&
           tiles_ok(up(q.M, 256), up(q.F, 128));
}

// Few tiles read their operands from DRAM at the pace of the ring's depth, a
// k-block in 0.36 us however narrow its piece.
static double cold_tiles(double time, int kbs) { return time < kbs + kLastEpilogue ? kbs + kLastEpilogue : time; }

double glu_tc_time(const GluProblem& q) {
    FfParams p = {};
    p.kbs = up(q.D, 64);
    const int units = device_sm_count(current_device()) / 2, tm = up(q.M, 256);
    const double wide = rounds((long long)tm * up(q.F, 256), units) * tile_cost(2, p.kbs);
    const double narrow = cold_tiles(plan_pieces(p, tm * up(q.F, 128), units, 2), p.kbs);
    return wide < narrow ? wide : narrow;
}

static void glu_params(const GluProblem& q, FfParams& p) {
    p.M = (int)q.M;
    p.N = (int)q.F;
    p.tiles_m = up(q.M, 256);
    p.kbs = up(q.D, 64);
    p.group_m = kGroupM;
}

pax_status_t glu_tc(const GluProblem& q, cudaStream_t stream) {
    FfMaps maps;
    FfParams p = {};
    CUtensorMap* m = maps.m;
    bool ok = matrix_map(&m[MG_X], q.X, kF16, 2, q.M, q.D, q.ldx, 64, 128) &&
              matrix_map(&m[MG_WG], q.Wg, kF16, 2, q.D, q.F, q.ldwg, 64, 64) &&
              matrix_map(&m[MG_WU], q.Wu, kF16, 2, q.D, q.F, q.ldwu, 64, 64) &&
              matrix_map(&m[MG_H], q.H, kF16, 2, q.M, q.F, q.ldh, 64, 32);
    if (ok && q.G)
        ok = matrix_map(&m[MG_G], q.G, kF16, 2, q.M, q.F, q.ldg, 64, 32) &&
             matrix_map(&m[MG_U], q.U, kF16, 2, q.M, q.F, q.ldu, 64, 32);
    if (!ok) return PAX_ERR_CUDA;
    for (int i = q.G ? MG_U + 1 : MG_H + 1; i < 10; ++i) m[i] = m[MG_X];
    glu_params(q, p);
    p.save = q.G != nullptr;
    if (q.act == ACT_SILU) return launch_glu<ACT_SILU>(maps, p, stream);
    if (q.act == ACT_GELU_TANH) return launch_glu<ACT_GELU_TANH>(maps, p, stream);
    return launch_glu<ACT_GELU_ERF>(maps, p, stream);
}

bool glu_back_tc_ok(const GluGradProblem& q) {
    const int w = q.dw_f16 ? 2 : 4;
    return q.M > 0 && q.D > 0 && q.F > 0 && rows16(q.dG, q.lddg, 2) && rows16(q.dU, q.lddu, 2) &&
           (!q.dX || (q.F <= kMaxSum && rows16(q.Wg, q.ldwg, 2) && rows16(q.Wu, q.ldwu, 2) && out16(q.dX, q.D, q.lddx, 2))) &&
           (!q.dWg || (q.M <= kMaxSum && rows16(q.X, q.ldx, 2) && out16(q.dWg, q.F, q.lddwg, w) && out16(q.dWu, q.F, q.lddwu, w))) &&
           tiles_ok(up(q.M, 256), up(q.D, 256)) && tiles_ok(up(q.D, 256), 2LL * up(q.F, 256));
}

static void back_params(const GluGradProblem& q, FfParams& p) {
    p.M = (int)q.M;
    p.D = (int)q.D;
    p.F = (int)q.F;
    p.N = p.D;
    p.tiles_m = up(q.M, 256);
    p.half_kbs = up(q.F, 64);
    p.kbs = 2 * p.half_kbs;
    p.group_m = kGroupM;
    p.wt_m = up(q.D, 256);
    p.kbs_w = up(q.M, 64);
    p.nx = q.dX != nullptr;  // counted once the tile width is chosen
    p.nw = q.dWg != nullptr;
    p.accumulate = q.accumulate;
}

double glu_back_tc_time(const GluGradProblem& q) {
    FfParams p = {};
    back_params(q, p);
    const int units = device_sm_count(current_device()) / 2;
    const double a = back_time(p, 1, units), b = back_time(p, 2, units);
    return a < b ? a : b;
}

pax_status_t glu_back_tc(const GluGradProblem& q, cudaStream_t stream) {
    FfMaps maps;
    FfParams p = {};
    CUtensorMap* m = maps.m;
    const CUtensorMapDataType wt = q.dw_f16 ? kF16 : kF32;
    const int we = q.dw_f16 ? 2 : 4;
    bool ok = true;
    if (q.dX)
        ok = matrix_map(&m[MB_DGK], q.dG, kF16, 2, q.M, q.F, q.lddg, 64, 128) &&
             matrix_map(&m[MB_DUK], q.dU, kF16, 2, q.M, q.F, q.lddu, 64, 128) &&
             matrix_map(&m[MB_WGK], q.Wg, kF16, 2, q.D, q.F, q.ldwg, 64, 128) &&
             matrix_map(&m[MB_WUK], q.Wu, kF16, 2, q.D, q.F, q.ldwu, 64, 128) &&
             matrix_map(&m[MB_DX], q.dX, kF16, 2, q.M, q.D, q.lddx, 64, 32);
    if (ok && q.dWg)
        ok = matrix_map(&m[MB_DGN], q.dG, kF16, 2, q.M, q.F, q.lddg, 64, 64) &&
             matrix_map(&m[MB_DUN], q.dU, kF16, 2, q.M, q.F, q.lddu, 64, 64) &&
             matrix_map(&m[MB_XN], q.X, kF16, 2, q.M, q.D, q.ldx, 64, 64) &&
             matrix_map(&m[MB_DWG], q.dWg, wt, we, q.D, q.F, q.lddwg, 128 / we, 32) &&
             matrix_map(&m[MB_DWU], q.dWu, wt, we, q.D, q.F, q.lddwu, 128 / we, 32);
    if (!ok) return PAX_ERR_CUDA;
    // Maps of what is not computed are never used.
    if (!q.dX) m[MB_DGK] = m[MB_DUK] = m[MB_WGK] = m[MB_WUK] = m[MB_DX] = m[MB_XN];
    if (!q.dWg) m[MB_DGN] = m[MB_DUN] = m[MB_XN] = m[MB_DWG] = m[MB_DWU] = m[MB_DX];
    back_params(q, p);
    return q.dw_f16 ? launch_back<__half>(maps, p, stream) : launch_back<float>(maps, p, stream);
}

// The items that the kernel's pairs run, as ff_item deals them out.
template <int MODE, int W>
static int list_items(const FfParams& p, int units, int* out, int max_items) {
    int n = 0;
    FfItem it;
    for (int u = 0; u < units; ++u)
        for (int idx = 0; ff_item<MODE, W>(p, u, units, idx, it); ++idx, ++n) {
            if (n >= max_items) return -1;
            int* o = out + 5 * n;
            o[0] = u;
            o[1] = it.kind;
            o[2] = it.mb;
            o[3] = MODE == FF_BACK ? it.nb * 256 * W : it.col;
            o[4] = (MODE == FF_GLU ? it.w / 2 : it.w) * W;
        }
    return n;
}

int feed_forward_items(int which, long long M, long long D, long long F, int units, int* width, int* items,
                       int max_items) {
    FfParams p = {};
    int w = 1, grid;
    if (which == 0) {
        GluProblem q = {};
        q.M = M, q.D = D, q.F = F;
        glu_params(q, p);
        w = plan_glu(p, units, units, grid);
    } else {
        GluGradProblem q = {};
        __half there;
        q.M = M, q.D = D, q.F = F;
        q.dX = &there, q.dWg = q.dWu = &there;
        back_params(q, p);
        w = back_width(p, units);
        grid = plan_back(p, w, units);
    }
    *width = w;
    if (which == 0) return w == 2 ? list_items<FF_GLU, 2>(p, grid, items, max_items) : list_items<FF_GLU, 1>(p, grid, items, max_items);
    return w == 2 ? list_items<FF_BACK, 2>(p, grid, items, max_items) : list_items<FF_BACK, 1>(p, grid, items, max_items);
}

bool gemm_i8_tc_ok(const I8Problem& q) {
    return q.K > 0 && rows16(q.A, q.lda, 1) && rows16(q.B, q.ldb, 1) && tiles_ok(up(q.M, 256), up(q.N, 256));
}

double gemm_i8_tc_time(const I8Problem& q) {
    FfParams p = {};
    p.kbs = up(q.K, 128);
    return cold_tiles(plan_pieces(p, up(q.M, 256) * up(q.N, 256), device_sm_count(current_device()) / 2, 4), p.kbs);
}

pax_status_t gemm_i8_tc(const I8Problem& q, cudaStream_t stream) {
    FfMaps maps;
    FfParams p = {};
    CUtensorMap* m = maps.m;
    const int ce = q.c_f16 ? 2 : 4;
    bool ok = matrix_map(&m[MI_A], q.A, kU8, 1, q.M, q.K, q.lda, 128, 128) &&
              matrix_map(&m[MI_B], q.B, kU8, 1, q.N, q.K, q.ldb, 128, 128) &&
              matrix_map(&m[MI_B2], q.B, kU8, 1, q.N, q.K, q.ldb, 128, 64) &&
              matrix_map(&m[MI_B4], q.B, kU8, 1, q.N, q.K, q.ldb, 128, 32);
    p.c_tma = out16(q.C, q.N, q.ldc, ce);
    p.c_unit = store_unit(q.C, q.ldc, ce);
    m[MI_C] = m[MI_A];
    if (ok && p.c_tma) ok = matrix_map(&m[MI_C], q.C, q.c_f16 ? kF16 : kF32, ce, q.M, q.N, q.ldc, 128 / ce, 32);
    if (!ok) return PAX_ERR_CUDA;
    for (int i = MI_C + 1; i < 10; ++i) m[i] = m[MI_A];
    p.M = (int)q.M;
    p.N = (int)q.N;
    p.tiles_m = up(q.M, 256);
    p.kbs = up(q.K, 128);
    p.group_m = kGroupM;
    p.C = q.C;
    p.ldc = q.ldc;
    p.sa = q.a_scale;
    p.sb = q.b_scale;
    p.bias = q.bias;
    return q.c_f16 ? launch_i8<__half>(maps, p, stream) : launch_i8<float>(maps, p, stream);
}

int read_clear_device_error_ff_tc() {
    int v = 0, z = 0;
    if (cudaMemcpyFromSymbol(&v, g_pax_device_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_pax_device_error, &z, sizeof(int));
    return v;
}

bool set_wait_limit_ff_tc(unsigned long long ns) {
    return cudaMemcpyToSymbol(g_pax_wait_limit_ns, &ns, sizeof(ns)) == cudaSuccess;
}

}  // namespace pax

extern "C" int pax_selftest_feed_forward_items(int which, long long M, long long D, long long F, int units, int* width,
                                               int* items, int max_items) {
    if ((which != 0 && which != 1) || M <= 0 || D <= 0 || F <= 0 || M > (1 << 24) || D > (1 << 24) || F > (1 << 24) ||
        units < 1 || !width || !items || max_items < 0)
        return -1;
    return pax::feed_forward_items(which, M, D, F, units, width, items, max_items);
}
