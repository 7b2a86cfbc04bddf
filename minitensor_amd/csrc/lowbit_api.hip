// lowbit_api.hip -- the C ABI of include/mtlowbit.h: argument checking, the
// choice of kernel and split, launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "lowbit_back_kernel.hpp"
#include "lowbit_q4_kernel.hpp"
#include "lowbit_rows_kernel.hpp"
#include "mtlowbit.h"

using namespace mtk;

namespace {

// Extents are 32-bit inside the kernels, and blocks past an end stay below 2^31.
constexpr int64_t kMaxDim = ((int64_t)1 << 31) - (1 << 16);
constexpr int64_t kMaxOut = (int64_t)1 << 26;   // rows of a 4-bit weight (32 threads each in a grid)
constexpr int64_t kMaxScaleStride = (int64_t)1 << 22;   // a tile's 256 rows of scales within 32 bits of bytes
constexpr int kCus = 256;                       // what plans fill (MI355X)
constexpr int64_t kMaxTiles = (int64_t)1 << 23; // of 512 threads: a grid's threads are a 32-bit number

int launched() {
    // (as mt_gemm_f32: a launch recorded by a stream capture reports this)
    const hipError_t e = hipGetLastError();
    return e == hipSuccess || e == hipErrorStreamCaptureUnsupported ? MT_OK : MT_ERR_HIP;
}

// A 2-D fp32 view; written: no two elements on one address.
bool valid(const mt_mat_f32* X, bool written) {
    if (!X || X->batch != 1 || X->rows < 0 || X->cols < 0 || X->row_stride < 0 ||
        X->col_stride < 0 || X->offset < 0 || X->rows >= kMaxDim || X->cols >= kMaxDim)
        return false;
    if (X->rows == 0 || X->cols == 0) return true;
    if (!X->base) return false;
    return !written || ((X->rows <= 1 || X->row_stride > 0) && (X->cols <= 1 || X->col_stride > 0));
}
bool same_shape(const mt_mat_f32* A, const mt_mat_f32* B) {
    return A->rows == B->rows && A->cols == B->cols;
}
bool valid(const mt_rows_q8* Q) {
    if (!Q || Q->rows < 0 || Q->cols < 0 || Q->rows >= kMaxDim || Q->cols >= kMaxDim ||
        Q->row_stride < 0 || (Q->rows > 1 && Q->row_stride < Q->cols))
        return false;
    return Q->rows == 0 || (Q->scale && (Q->cols == 0 || Q->q));
}
bool valid(const mt_weight_q4* W) {
    if (!W || W->n < 0 || W->k < 0 || W->n >= kMaxOut || W->k >= kMaxDim ||
        (W->group != 32 && W->group != 64 && W->group != 128) || W->row_stride < 0 ||
        W->scale_stride < 0)
        return false;
    if (W->n == 0 || W->k == 0) return true;
    if (!W->packed || !W->scale || ((uintptr_t)W->packed & 15) || (W->row_stride & 15)) return false;
    return W->n == 1 || (W->scale_stride < kMaxScaleStride && W->row_stride >= (W->k + 31) / 32 * 16 &&
                         W->scale_stride >= (W->k + W->group - 1) / W->group);
}

RowView view(const mt_mat_f32* X) {
    if (!X) return {nullptr, 0, 0};
    return {const_cast<float*>(X->base) + X->offset, X->row_stride, X->col_stride};
}
// Rows whose elements are neighbours (or absent).
bool unit(const RowView& v) { return !v.p || v.cs == 1; }

// Threads of a row: 16 values each (lowbit_rows_kernel.hpp).
int row_threads(int64_t cols) { return cols <= 1024 ? 64 : cols <= 4096 ? 256 : 1024; }
bool row_resident(int64_t cols) { return cols <= 16384; }
// (workgroups beyond these take a second row: a grid's threads are a 32-bit number)
unsigned row_blocks(int64_t rows, int nt) {
    return (unsigned)std::min<int64_t>(nt == 64 ? (rows + 3) / 4 : rows, 1 << 20);
}

// The scales and rstd of rows without columns (nullptr: not wanted).
int empty_rows(int64_t rows, const mt_rows_q8* Q, float* rstd, float eps, void* stream) {
    int rc = MT_OK;
    if (Q) rc = mt_fill_f32(Q->scale, rows, kScaleMin, stream);
    if (rc == MT_OK && rstd) rc = mt_fill_f32(rstd, rows, 1.f / std::sqrt(eps), stream);
    return rc;
}

// Calls go(NT, MODE, RES) as constants: see lowbit_rows_kernel.hpp.
template <class Go>
void row_kernel(int64_t cols, bool units, Go go) {
    using std::integral_constant;
    using Res = std::true_type;
    using Again = std::false_type;
    if (!units) return go(integral_constant<int, 1024>{}, integral_constant<int, R_STRIDED>{}, Again{});
    auto pick = [&](auto mode) {
        if (!row_resident(cols)) go(integral_constant<int, 1024>{}, mode, Again{});
        else if (row_threads(cols) == 64) go(integral_constant<int, 64>{}, mode, Res{});
        else if (row_threads(cols) == 256) go(integral_constant<int, 256>{}, mode, Res{});
        else go(integral_constant<int, 1024>{}, mode, Res{});
    };
    if (cols & 3) pick(integral_constant<int, R_TAIL>{});
    else pick(integral_constant<int, R_VEC>{});
}

template <bool NORM>
void launch_rows(const RowParams& p, bool units, hipStream_t s) {
    row_kernel(p.cols, units, [&](auto nt, auto mode, auto res) {
        hipLaunchKernelGGL((rows_forward<nt(), mode(), res(), NORM>), dim3(row_blocks(p.rows, nt())),
                           dim3(std::max<int>(nt(), 256)), 0, s, p);
    });
}

// Row groups of the backward kernel, each of which keeps a part of dweight: enough to keep
// the loads in flight, few enough that the parts weigh little (2048 x 4096, 256 to 2048
// groups: 31, 29, 32, 41 us; 8192 x 2048: 67, 48, 46, 53; 1024 x 8192: 29, 35, 45, 45;
// 8192 x 512: 51, 30, 20, 20).  A multiple of four, whether a workgroup holds four groups or one.
int64_t row_groups(int64_t rows, int64_t cols) {
    const int nt = row_threads(cols);
    const int64_t most = nt == 64 ? 2048 : nt == 256 ? 768 : 256;
    return (std::min(rows, most) + 3) / 4 * 4;
}

// Workgroups of the parts' sum, 16 columns each at a time (a grid's threads are a 32-bit
// number: 64 a column, one column in each, were 2^32 of them from 2^26 columns on).
unsigned dweight_blocks(int64_t cols) { return (unsigned)std::min<int64_t>((cols + 15) / 16, 1 << 20); }

// Tiles and splits of a product over chunks of 32 k, from measured times in us: of a chunk,
// by workgroups on a CU, where each holds as many as its LDS and registers allow, and of a
// round's beginning and end.  The tile and the number of splits that come out fastest,
// workgroups going in rounds over the CUs, with a launch and the partials' sum.  (4096 ->
// 4096: 1024 fp32 rows, 128x256 tiles in 2 splits 100 us, 64x128 unsplit 118; 1024 8-bit
// rows 53 and 46, 2048 of them unsplit 63 and 84, 256 of them, 64x128 in 2 splits 28,
// unsplit 31.)
struct Tiling {
    int bm;                           // of bm x 2·bm
    int per_cu;
    double alone, more;               // a chunk's time: one workgroup on the CU, each further one
};
struct Tiled {
    int bm, splits, k_per_split;
    int64_t tiles;                    // the splits' among them
    size_t partials;                  // floats, 0 without splits
};
Tiled plan_tiles(int64_t M, int64_t N, int64_t K, const Tiling* t, int n) {
    Tiled best{};
    double least = 0;
    const int64_t blocks = std::max<int64_t>(1, (K + 127) / 128);
    for (int i = 0; i < n; ++i) {
        const int64_t tiles = ((M + t[i].bm - 1) / t[i].bm) * ((N + 2 * t[i].bm - 1) / (2 * t[i].bm));
        for (int64_t s = 1; s <= std::min<int64_t>(blocks, 32); ++s) {
            const int64_t per = (blocks + s - 1) / s;
            if ((blocks + per - 1) / per != s) continue;
            const int64_t wgs = tiles * s, slots = (int64_t)kCus * t[i].per_cu;
            const double chunks = (double)std::min<int64_t>(4 * per, (K + 31) / 32);
            auto round = [&](int64_t n) {             // with n workgroups on a CU
                return chunks * (t[i].alone + (double)(n - 1) * t[i].more) + 5 +
                       (double)(n * t[i].bm / 32);
            };
            double us = (double)(wgs / slots) * round(t[i].per_cu);
            if (wgs % slots) us += round((wgs % slots + kCus - 1) / kCus);
            if (s > 1) us += 4 + (double)(s + 1) * (double)M * (double)N * 1.2e-6;
            if (least == 0 || us < least) {
                least = us;
                best = {t[i].bm, (int)s, (int)(per * 128), wgs, s > 1 ? (size_t)(s * M * N) : 0};
            }
            if (wgs >= 4 * slots) break;
        }
    }
    return best;
}

struct Q4Plan {
    bool few;
    Tiled tiled;
};
Q4Plan q4_plan(int64_t M, int64_t N, int64_t K, int group, bool q8) {
    if (M * (q8 ? 1 : 3) <= 48) return {true, {}};
    // (groups of 32: the wide tile's scales do not fit the registers)
    static const Tiling f32[] = {{64, 2, 0.5, 0.42}, {128, 1, 1.2, 0}};
    static const Tiling int8_32[] = {{64, 4, 0.3, 0.13}};
    static const Tiling int8_64[] = {{64, 4, 0.25, 0.1}, {128, 1, 0.53, 0}};
    static const Tiling int8_128[] = {{64, 4, 0.18, 0.117}, {128, 1, 0.38, 0}};
    const Tiling* const t = !q8 ? f32 : group == 32 ? int8_32 : group == 64 ? int8_64 : int8_128;
    return {false, plan_tiles(M, N, K, t, group == 32 ? 1 : 2)};
}

// Column blocks of a workgroup for few rows (of parts), where that leaves one for every CU
// (four of them, and 48 rows, do not fit the registers).
int few_columns(int rows, int64_t N) {
    const int64_t cols = (N + 15) / 16;
    return rows <= 6 ? 1 : cols >= 4 * kCus && rows <= 32 ? 4 : cols >= 2 * kCus ? 2 : 1;
}

template <bool Q8, int G>
void launch_few(const Q4Params& p, hipStream_t s) {
    const int rows = p.M * (Q8 ? 1 : 3), cols = (p.N + 15) / 16, nc = few_columns(rows, p.N);
    const dim3 grid((unsigned)((cols + nc - 1) / nc)), block(512);
    auto go = [&](auto cap, auto u) {
        if constexpr (cap() <= 32)
            if (nc == 4) {
                hipLaunchKernelGGL((q4_few<cap(), 1, 4, G, Q8, 8>), grid, block, 0, s, p);
                return;
            }
        if (nc == 2) hipLaunchKernelGGL((q4_few<cap(), 1, 2, G, Q8, 8>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((q4_few<cap(), u(), 1, G, Q8, 8>), grid, block, 0, s, p);
    };
    using std::integral_constant;
    if (rows <= 3)
        hipLaunchKernelGGL((q4_few<3, 4, 1, G, Q8, 8>), grid, block, 0, s, p);
    else if (rows <= 6)
        hipLaunchKernelGGL((q4_few<6, 4, 1, G, Q8, 8>), grid, block, 0, s, p);
    else if (rows <= 16)
        go(integral_constant<int, Q8 ? 16 : 15>{}, integral_constant<int, 2>{});
    else if (rows <= 32)
        go(integral_constant<int, Q8 ? 32 : 30>{}, integral_constant<int, 1>{});
    else
        go(integral_constant<int, 48>{}, integral_constant<int, 1>{});
}
template <bool Q8, int G>
void launch_gemm(const Q4Params& p, const Tiled& plan, hipStream_t s) {
    const dim3 grid((unsigned)plan.tiles);
    if constexpr (Q8) {
        if (plan.bm == 64)
            hipLaunchKernelGGL((q4_gemm_q8<64, 128, 32, 64, G>), grid, dim3(256), 0, s, p);
        else if constexpr (G > 32)
            hipLaunchKernelGGL((q4_gemm_q8<128, 256, 64, 64, G>), grid, dim3(512), 0, s, p);
    } else if (plan.bm == 64)
        hipLaunchKernelGGL((q4_gemm<64, 128, 32, 64, G>), grid, dim3(256), 0, s, p);
    else if constexpr (G > 32)
        hipLaunchKernelGGL((q4_gemm<128, 256, 32, 128, G>), grid, dim3(512), 0, s, p);
}

template <bool Q8>
int run_q4(Q4Params p, int64_t M, const mt_weight_q4* W, const float* bias, int64_t bias_stride,
           const mt_mat_f32* Y, void* workspace, size_t ws_bytes, hipStream_t s) {
    if (M == 0 || W->n == 0) return MT_OK;
    const RowView y = view(Y);
    p.w = W->packed;
    p.w_n = W->row_stride;
    p.s = W->scale;
    p.s_n = W->scale_stride;
    p.bias = bias;
    p.bias_stride = bias_stride;
    p.y = y.p;
    p.y_m = y.rs;
    p.y_n = y.cs;
    p.M = (int)M;
    p.N = (int)W->n;
    p.K = (int)W->k;
    const Q4Plan plan = q4_plan(M, W->n, W->k, W->group, Q8);
    if (W->k == 0) {                                  // no inputs: the bias alone
        const unsigned blocks = (unsigned)std::min<int64_t>((M * W->n + 255) / 256, 4096);
        hipLaunchKernelGGL(lb_sum, dim3(blocks), dim3(256), 0, s,
                           LbSum{nullptr, 0, p.M, p.N, bias, bias_stride, p.y, p.y_m, p.y_n});
        return launched();
    }
    const size_t need = plan.tiled.partials * 4;
    if (plan.tiled.tiles >= kMaxTiles) return MT_ERR_INVALID;
    if (need > 0 && (!workspace || ws_bytes < need)) return MT_ERR_WORKSPACE;
    p.splits = plan.few ? 1 : plan.tiled.splits;
    p.k_per_split = plan.tiled.k_per_split;
    p.part = static_cast<float*>(workspace);
    auto go = [&](auto g) {
        constexpr int G = decltype(g)::value;
        if (plan.few) launch_few<Q8, G>(p, s);
        else launch_gemm<Q8, G>(p, plan.tiled, s);
    };
    if (W->group == 32) go(std::integral_constant<int, 32>{});
    else if (W->group == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
    if (p.splits > 1) {
        const unsigned blocks = (unsigned)std::min<int64_t>((M * W->n + 255) / 256, 8192);
        hipLaunchKernelGGL(lb_sum, dim3(blocks), dim3(256), 0, s,
                           LbSum{p.part, p.splits, p.M, p.N, bias, bias_stride, p.y, p.y_m, p.y_n});
    }
    return launched();
}

// The weight gradient [O][C] over R rows, and the floats of its workspace: the splits'
// partial products and row sums.
Tiled back_plan(int64_t R, int64_t O, int64_t C) {
    static const Tiling tiles[] = {{64, 2, 0.8, 0.2}, {128, 1, 1.35, 0}};
    Tiled t = plan_tiles(O, C, R, tiles, 2);
    if (t.partials) t.partials += (size_t)t.splits * O;
    return t;
}

}  // namespace

extern "C" {

int mt_rms_norm_f32(const mt_mat_f32* X, const mt_mat_f32* R, const float* weight,
                    int64_t weight_stride, float eps, const mt_mat_f32* H, const mt_mat_f32* Y,
                    const mt_rows_q8* Q, float* rstd, void* stream) {
    if (!valid(X, false) || (R && (!valid(R, false) || !same_shape(X, R))) ||
        (H && (!valid(H, true) || !same_shape(X, H))) ||
        (Y && (!valid(Y, true) || !same_shape(X, Y))) ||
        (Q && (!valid(Q) || Q->rows != X->rows || Q->cols != X->cols)) || weight_stride < 0 ||
        !(eps >= 0.f))
        return MT_ERR_INVALID;
    if (X->rows == 0) return MT_OK;
    if (X->cols == 0) return empty_rows(X->rows, Q, rstd, eps, stream);
    RowParams p{};
    p.x = view(X);
    p.r = view(R);
    p.h = view(H);
    p.y = view(Y);
    p.w = weight;
    p.ws = weight_stride;
    if (Q) {
        p.q = Q->q;
        p.qs = Q->row_stride;
        p.scale = Q->scale;
    }
    p.rstd = rstd;
    p.eps = eps;
    p.rows = X->rows;
    p.cols = (int)X->cols;
    const bool units = unit(p.x) && unit(p.r) && unit(p.h) && unit(p.y) &&
                       (!weight || weight_stride == 1);
    launch_rows<true>(p, units, static_cast<hipStream_t>(stream));
    return launched();
}

size_t mt_rms_norm_backward_workspace_f32(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || rows >= kMaxDim || cols >= kMaxDim) return 0;
    return (size_t)(row_groups(rows, cols) * cols) * 4;
}

int mt_rms_norm_backward_f32(const mt_mat_f32* dY, const mt_mat_f32* H, const float* weight,
                             int64_t weight_stride, const float* rstd, const mt_mat_f32* dH0,
                             const mt_mat_f32* dH, float* dweight, int64_t dweight_stride,
                             float beta, void* workspace, size_t ws_bytes, void* stream) {
    if (!valid(dY, false) || !valid(H, false) || !same_shape(dY, H) ||
        (dH0 && (!valid(dH0, false) || !same_shape(dY, dH0))) ||
        (dH && (!valid(dH, true) || !same_shape(dY, dH))) || weight_stride < 0 ||
        (dweight && (dweight_stride < 0 || (dY->cols > 1 && dweight_stride == 0))) ||
        (dY->rows > 0 && !rstd))
        return MT_ERR_INVALID;
    if (dY->cols == 0 || (!dH && !dweight)) return MT_OK;
    const size_t need = dweight ? mt_rms_norm_backward_workspace_f32(dY->rows, dY->cols) : 0;
    if (need > 0 && (!workspace || ws_bytes < need)) return MT_ERR_WORKSPACE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    RowBwdParams p{};
    p.dy = view(dY);
    p.h = view(H);
    p.dh0 = view(dH0);
    p.dh = view(dH);
    p.w = weight;
    p.ws = weight_stride;
    p.rstd = rstd;
    p.part = dweight ? static_cast<float*>(workspace) : nullptr;
    p.rows = dY->rows;
    p.cols = (int)dY->cols;
    const int64_t groups = row_groups(p.rows, p.cols);
    if (p.rows > 0) {
        p.row_step = (int)groups;
        const bool units = unit(p.dy) && unit(p.h) && unit(p.dh0) && unit(p.dh) &&
                           (!weight || weight_stride == 1);
        row_kernel(p.cols, units, [&](auto nt, auto mode, auto res) {
            hipLaunchKernelGGL((rms_backward<nt(), mode(), res()>),
                               dim3((unsigned)(nt() == 64 ? groups / 4 : groups)),
                               dim3(std::max<int>(nt(), 256)), 0, s, p);
        });
    }
    if (dweight)
        hipLaunchKernelGGL(rms_dweight_sum, dim3(dweight_blocks(p.cols)), dim3(1024), 0, s, p.part,
                           p.rows > 0 ? (int)groups : 0, p.cols, dweight, dweight_stride, beta);
    return launched();
}

int mt_quantize_q8_f32(const mt_mat_f32* X, const mt_rows_q8* Q, void* stream) {
    if (!valid(X, false) || !valid(Q) || Q->rows != X->rows || Q->cols != X->cols)
        return MT_ERR_INVALID;
    if (X->rows == 0) return MT_OK;
    if (X->cols == 0) return empty_rows(X->rows, Q, nullptr, 0.f, stream);
    RowParams p{};
    p.x = view(X);
    p.q = Q->q;
    p.qs = Q->row_stride;
    p.scale = Q->scale;
    p.rows = X->rows;
    p.cols = (int)X->cols;
    launch_rows<false>(p, unit(p.x), static_cast<hipStream_t>(stream));
    return launched();
}

int mt_dequantize_q8_f32(const mt_rows_q8* Q, const mt_mat_f32* Y, void* stream) {
    if (!valid(Q) || !valid(Y, true) || Q->rows != Y->rows || Q->cols != Y->cols)
        return MT_ERR_INVALID;
    if (Y->rows == 0 || Y->cols == 0) return MT_OK;
    const RowView y = view(Y);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t waves = Y->rows * ((Y->cols + 1023) / 1024), n = Y->rows * Y->cols;
    if (y.cs == 1)
        hipLaunchKernelGGL(dequantize_q8<true>,
                           dim3((unsigned)std::min<int64_t>((waves + 3) / 4, 1 << 20)), dim3(256), 0,
                           s, Q->q, Q->row_stride, Q->scale, y, Y->rows, (int)Y->cols);
    else
        hipLaunchKernelGGL(dequantize_q8<false>,
                           dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 16)), dim3(256), 0,
                           s, Q->q, Q->row_stride, Q->scale, y, Y->rows, (int)Y->cols);
    return launched();
}

size_t mt_linear_backward_q8_workspace_f32(int64_t rows, int64_t in_f, int64_t out_f) {
    if (rows < 0 || in_f < 0 || out_f < 0 || rows >= kMaxDim || in_f >= kMaxDim || out_f >= kMaxDim)
        return 0;
    return std::max(mt_linear_workspace_f32(rows, in_f, out_f), back_plan(rows, out_f, in_f).partials * 4);
}

int mt_linear_backward_q8_f32(const mt_mat_f32* dY, const mt_rows_q8* X, const mt_mat_f32* W,
                              const mt_mat_f32* dX, const mt_mat_f32* dW, float beta_w, float* db,
                              int64_t db_stride, float beta_b, void* workspace, size_t ws_bytes,
                              void* stream) {
    if (!valid(dY, false) || !valid(X) || dY->rows != X->rows) return MT_ERR_INVALID;
    if (dX && (!W || !valid(W, false) || W->rows != dY->cols || W->cols != X->cols ||
               !valid(dX, true) || dX->rows != X->rows || dX->cols != X->cols))
        return MT_ERR_INVALID;
    if (dW && (!valid(dW, true) || dW->rows != dY->cols || dW->cols != X->cols))
        return MT_ERR_INVALID;
    if (db && (db_stride < 0 || (dY->cols > 1 && db_stride == 0))) return MT_ERR_INVALID;
    const Tiled plan = back_plan(X->rows, dY->cols, X->cols);
    if (dW && plan.tiles >= kMaxTiles) return MT_ERR_INVALID;
    if (dW && plan.partials > 0 && (!workspace || ws_bytes < plan.partials * 4))
        return MT_ERR_WORKSPACE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dX) {
        const int rc = mt_gemm_f32(dY, W, dX, nullptr, workspace, ws_bytes, stream);
        if (rc != MT_OK) return rc;
    }
    if (dW && dW->rows > 0 && dW->cols > 0) {
        BackParams p{};
        const RowView dy = view(dY), dw = view(dW);
        p.dy = dy.p;
        p.dy_r = dy.rs;
        p.dy_o = dy.cs;
        p.q = X->q;
        p.q_r = X->row_stride;
        p.scale = X->scale;
        p.dw = dw.p;
        p.dw_o = dw.rs;
        p.dw_c = dw.cs;
        p.beta = beta_w;
        p.part = static_cast<float*>(workspace);
        p.R = (int)X->rows;
        p.O = (int)dY->cols;
        p.C = (int)X->cols;
        p.splits = plan.splits;
        p.r_per_split = plan.k_per_split;
        if (db) {
            p.db = db;
            p.db_stride = db_stride;
            p.beta_b = beta_b;
            p.part_b = p.part + (int64_t)p.splits * p.O * p.C;
        }
        const LbSum sum{p.part, p.R > 0 ? p.splits : 0, p.O, p.C, nullptr, 0, p.dw, p.dw_o, p.dw_c,
                        beta_w, p.part_b, db, db_stride, beta_b, p.O};
        if (p.R > 0) {
            const dim3 grid((unsigned)plan.tiles);
            if (plan.bm == 64)
                hipLaunchKernelGGL((back_dw<64, 128, 32, 64>), grid, dim3(256), 0, s, p);
            else
                hipLaunchKernelGGL((back_dw<128, 256, 32, 128>), grid, dim3(512), 0, s, p);
        }
        if (p.R == 0 || p.splits > 1) {               // (no rows: beta·dW, beta·db)
            const int64_t n = (int64_t)p.O * p.C + p.O;
            hipLaunchKernelGGL(lb_sum, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 8192)),
                               dim3(256), 0, s, sum);
        }
        return launched();
    }
    if (db) return mt_colsum_f32(dY, db, db_stride, beta_b, stream);
    return MT_OK;
}

int mt_quantize_q4_f32(const mt_mat_f32* W, const mt_weight_q4* Q, void* stream) {
    if (!valid(W, false) || !valid(Q) || W->rows != Q->n || W->cols != Q->k) return MT_ERR_INVALID;
    if (Q->n == 0 || Q->k == 0) return MT_OK;
    const RowView w = view(W);
    const int64_t groups = (Q->k + Q->group - 1) / Q->group;
    const int64_t n = Q->n * groups * (Q->group / 8);
    const unsigned blocks = (unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto g) {
        hipLaunchKernelGGL(quantize_q4<g()>, dim3(blocks), dim3(256), 0, s, w.p, w.rs, w.cs, Q->packed, Q->row_stride, Q->scale,
                           Q->scale_stride, (int)Q->n, (int)Q->k);
    };
    if (Q->group == 32) go(std::integral_constant<int, 32>{});
    else if (Q->group == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
    return launched();
}

int mt_dequantize_q4_f32(const mt_weight_q4* Q, const mt_mat_f32* W, void* stream) {
    if (!valid(Q) || !valid(W, true) || W->rows != Q->n || W->cols != Q->k) return MT_ERR_INVALID;
    if (Q->n == 0 || Q->k == 0) return MT_OK;
    const RowView w = view(W);
    const int64_t n = Q->n * ((Q->k + 7) / 8);
    const unsigned blocks = (unsigned)std::min<int64_t>((n + 255) / 256, 1 << 16);
    hipLaunchKernelGGL(dequantize_q4, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream),
                       Q->packed, Q->row_stride, Q->scale, Q->scale_stride, (int)Q->group, w.p, w.rs,
                       w.cs, (int)Q->n, (int)Q->k);
    return launched();
}

size_t mt_linear_q4_workspace(int64_t rows, int64_t in_f, int64_t out_f) {
    if (rows <= 0 || in_f <= 0 || out_f <= 0 || rows >= kMaxDim || in_f >= kMaxDim ||
        out_f >= kMaxDim)
        return 0;
    size_t n = 0;
    for (const int group : {32, 64, 128})
        for (const bool q8 : {false, true})
            n = std::max(n, q4_plan(rows, out_f, in_f, group, q8).tiled.partials);
    return n * 4;
}

int mt_linear_q4_plan(int64_t rows, int64_t in_f, int64_t out_f, int group, int x_in_8_bits,
                      mt_lowbit_plan* plan) {
    if (rows <= 0 || in_f <= 0 || out_f <= 0 || rows >= kMaxDim || in_f >= kMaxDim ||
        out_f >= kMaxOut || (group != 32 && group != 64 && group != 128) || !plan)
        return MT_ERR_INVALID;
    const Q4Plan p = q4_plan(rows, out_f, in_f, group, x_in_8_bits != 0);
    if (p.few) *plan = {0, 1, few_columns((int)rows * (x_in_8_bits ? 1 : 3), out_f)};
    else *plan = {p.tiled.bm, p.tiled.splits, 0};
    return MT_OK;
}

int mt_linear_backward_q8_plan(int64_t rows, int64_t in_f, int64_t out_f, mt_lowbit_plan* plan) {
    if (rows <= 0 || in_f <= 0 || out_f <= 0 || rows >= kMaxDim || in_f >= kMaxDim ||
        out_f >= kMaxDim || !plan)
        return MT_ERR_INVALID;
    const Tiled t = back_plan(rows, out_f, in_f);
    *plan = {t.bm, t.splits, 0};
    return MT_OK;
}

int mt_linear_q4_f32(const mt_mat_f32* X, const mt_weight_q4* W, const float* bias,
                     int64_t bias_stride, const mt_mat_f32* Y, void* workspace, size_t ws_bytes,
                     void* stream) {
    if (!valid(X, false) || !valid(W) || !valid(Y, true) || X->cols != W->k || Y->rows != X->rows ||
        Y->cols != W->n || (bias && bias_stride < 0))
        return MT_ERR_INVALID;
    Q4Params p{};
    const RowView x = view(X);
    p.x = x.p;
    p.x_m = x.rs;
    p.x_k = x.cs;
    return run_q4<false>(p, X->rows, W, bias, bias_stride, Y, workspace, ws_bytes,
                         static_cast<hipStream_t>(stream));
}

int mt_linear_q4_q8(const mt_rows_q8* X, const mt_weight_q4* W, const float* bias,
                    int64_t bias_stride, const mt_mat_f32* Y, void* workspace, size_t ws_bytes,
                    void* stream) {
    if (!valid(X) || !valid(W) || !valid(Y, true) || X->cols != W->k || Y->rows != X->rows ||
        Y->cols != W->n || (bias && bias_stride < 0))
        return MT_ERR_INVALID;
    Q4Params p{};
    p.q = X->q;
    p.q_m = X->row_stride;
    p.q_scale = X->scale;
    return run_q4<true>(p, X->rows, W, bias, bias_stride, Y, workspace, ws_bytes,
                        static_cast<hipStream_t>(stream));
}

}  // extern "C"
