// q8_api.hip -- products of 8-bit rows and 8-bit weights: mt_linear_q8 of
// include/mtlowbit.h, and the gated form of include/mtffn.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "api_checks.hpp"
#include "mtffn.h"
#include "mtlowbit.h"
#include "q8_kernel.hpp"

using namespace mtk;

namespace {

// A product's sums are 32-bit below this many terms: a split holds no more.
constexpr int64_t kMaxTerms = ((int64_t)1 << 17) - 128;

struct Q8Plan {
    bool few;
    int bm, bn;
    int splits, k_per_split;
    int64_t tiles;                    // the splits' among them
    int64_t part_n;
    size_t partials;                  // of 4 bytes, 0 without splits
};

struct Q8Tile {
    int bm, bn, per_cu;
    double alone, more;               // us a chunk of 128 inputs: one workgroup on the CU, each further one
};
constexpr Q8Tile kTiles[] = {{64, 128, 3, 0.30, 0.14}, {128, 128, 2, 0.36, 0.22}, {256, 256, 1, 1.0, 0}};

// cols: columns of the launch (gated: whole blocks of 32 features, twice).
Q8Plan q8_plan(int64_t M, int64_t cols, int64_t K) {
    if (M <= 32 && K < ((int64_t)1 << 19)) return {true, 0, 0, 1, 0, 0, 0, 0};
    Q8Plan best{};
    double least = 0;
    const int64_t chunks = std::max<int64_t>(1, (K + 127) / 128);
    const int64_t fewest = (K + kMaxTerms - 1) / kMaxTerms;
    for (const Q8Tile& t : kTiles) {
        const int64_t tm = (M + t.bm - 1) / t.bm, tn = (cols + t.bn - 1) / t.bn;
        for (int64_t s = std::max<int64_t>(1, fewest); s <= std::max<int64_t>(fewest, std::min<int64_t>(chunks, 32)); ++s) {
            const int64_t per = (chunks + s - 1) / s;
            if ((chunks + per - 1) / per != s && s != fewest) continue;
            const int64_t splits = (chunks + per - 1) / per, wgs = tm * tn * splits;
            const int64_t slots = (int64_t)kCus * t.per_cu;
            auto round = [&](int64_t n) {
                return (double)per * (t.alone + (double)(n - 1) * t.more) + 3 +
                       (double)n * t.bm * t.bn * 1.5e-4;
            };
            double us = (double)(wgs / slots) * round(t.per_cu);
            if (wgs % slots) us += round((wgs % slots + kCus - 1) / kCus);
            if (splits > 1) us += 4 + (double)(splits + 1) * (double)M * (double)cols * 1.2e-6;
            if (least == 0 || us < least) {
                least = us;
                best = {false, t.bm, t.bn, (int)splits, (int)(per * 128), wgs, tn * t.bn,
                        splits > 1 ? (size_t)(splits * M) * (size_t)(tn * t.bn) : 0};
            }
            if (wgs >= 4 * slots) break;
        }
    }
    return best;
}
int64_t launch_cols(int64_t n, bool gated) { return gated ? (n + 31) / 32 * 64 : n; }

// Rows on multiples of 16 bytes.
bool aligned16(const int8_t* p, int64_t stride, int64_t rows) {
    return ((uintptr_t)p & 15) == 0 && (rows <= 1 || (stride & 15) == 0);
}

template <bool GATED>
void launch_few(const Q8Params& p, hipStream_t s) {
    using std::integral_constant;
    auto go = [&](auto mb, auto nc) {
        constexpr int F = GATED ? 8 * nc() : 16 * nc();
        hipLaunchKernelGGL((q8_few<mb(), nc(), GATED>), dim3((unsigned)((p.N + F - 1) / F)), dim3(512),
                           0, s, p);
    };
    if constexpr (GATED) {
        if (p.M <= 16) go(integral_constant<int, 1>{}, integral_constant<int, 2>{});
        else go(integral_constant<int, 2>{}, integral_constant<int, 2>{});
    } else {
        if (p.M <= 16) go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
        else go(integral_constant<int, 2>{}, integral_constant<int, 1>{});
    }
}
template <bool GATED, bool DMA>
void launch_tiles(const Q8Params& p, const Q8Plan& plan, hipStream_t s) {
    const dim3 grid((unsigned)plan.tiles);
    if (plan.bm == 64)
        hipLaunchKernelGGL((q8_gemm<64, 128, 32, 128, 2, DMA, GATED>), grid, dim3(256), 0, s, p);
    else if (plan.bm == 128)
        hipLaunchKernelGGL((q8_gemm<128, 128, 64, 128, 2, DMA, GATED>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((q8_gemm<256, 256, 128, 128, 2, DMA, GATED>), grid, dim3(512), 0, s, p);
}

template <bool GATED>
int run_q8(Q8Params& p, void* workspace, size_t ws_bytes, hipStream_t s) {
    const Q8Plan plan = q8_plan(p.M, launch_cols(p.N, GATED), p.K);
    if (plan.few) {
        p.splits = 1;
        launch_few<GATED>(p, s);
        return launched();
    }
    if (plan.tiles >= kMaxTiles) return MT_ERR_INVALID;
    const size_t need = plan.partials * 4;
    if (need > 0 && (!workspace || ws_bytes < need || ((uintptr_t)workspace & 3)))
        return MT_ERR_WORKSPACE;
    p.splits = plan.splits;
    p.k_per_split = plan.k_per_split;
    p.part = static_cast<int32_t*>(workspace);
    p.part_n = plan.part_n;
    if (aligned16(p.x, p.x_m, p.M) && aligned16(p.w, p.w_n, GATED ? 2 * (int64_t)p.N : p.N))
        launch_tiles<GATED, true>(p, plan, s);
    else
        launch_tiles<GATED, false>(p, plan, s);
    if (plan.splits > 1) {
        const int64_t n = (int64_t)p.M * ((p.N + 3) / 4);
        hipLaunchKernelGGL(q8_sum<GATED>, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 8192)),
                           dim3(256), 0, s, p);
    }
    return launched();
}

Q8Params q8_params(const mt_rows_q8* X, const mt_rows_q8* W, const float* bias, int64_t bias_stride,
                   const mt_mat_f32* Y) {
    Q8Params p{};
    p.x = X->q;
    p.x_m = X->row_stride;
    p.xs = X->scale;
    p.w = W->q;
    p.w_n = W->row_stride;
    p.ws = W->scale;
    p.bias = bias;
    p.bias_stride = bias_stride;
    p.y = view(Y);
    p.M = (int)X->rows;
    p.N = (int)Y->cols;
    p.K = (int)X->cols;
    return p;
}
size_t workspace_of(int64_t rows, int64_t in_f, int64_t out_f, bool gated) {
    if (rows <= 0 || in_f <= 0 || out_f <= 0 || rows >= kMaxDim || in_f >= kMaxDim ||
        out_f >= (gated ? kMaxDim / 2 : kMaxDim))
        return 0;
    return q8_plan(rows, launch_cols(out_f, gated), in_f).partials * 4;
}
int plan_of(int64_t rows, int64_t in_f, int64_t out_f, bool gated, mt_lowbit_plan* plan) {
    if (rows <= 0 || in_f <= 0 || out_f <= 0 || rows >= kMaxDim || in_f >= kMaxDim ||
        out_f >= (gated ? kMaxDim / 2 : kMaxDim) || !plan)
        return MT_ERR_INVALID;
    const Q8Plan p = q8_plan(rows, launch_cols(out_f, gated), in_f);
    *plan = {p.bm, p.splits, p.few ? 1 : 0};
    return MT_OK;
}

}  // namespace

extern "C" {

int mt_linear_q8(const mt_rows_q8* X, const mt_rows_q8* W, const float* bias, int64_t bias_stride,
                 const mt_mat_f32* Y, void* workspace, size_t ws_bytes, void* stream) {
    if (!valid(X) || !valid(W) || !valid(Y, true) || X->cols != W->cols || Y->rows != X->rows ||
        Y->cols != W->rows || (bias && bias_stride < 0))
        return MT_ERR_INVALID;
    if (Y->rows == 0 || Y->cols == 0) return MT_OK;
    Q8Params p = q8_params(X, W, bias, bias_stride, Y);
    return run_q8<false>(p, workspace, ws_bytes, static_cast<hipStream_t>(stream));
}

size_t mt_linear_q8_workspace(int64_t rows, int64_t in_f, int64_t out_f) {
    return workspace_of(rows, in_f, out_f, false);
}
int mt_linear_q8_plan(int64_t rows, int64_t in_f, int64_t out_f, mt_lowbit_plan* plan) {
    return plan_of(rows, in_f, out_f, false, plan);
}

int mt_gated_linear_q8(const mt_rows_q8* X, const mt_rows_q8* W, const float* bias,
                       int64_t bias_stride, int act, const mt_mat_f32* H, const mt_mat_f32* GU,
                       void* workspace, size_t ws_bytes, void* stream) {
    if (!valid(X) || !valid(W) || !valid(H, true) || X->cols != W->cols || H->rows != X->rows ||
        W->rows % 2 != 0 || H->cols != W->rows / 2 || (bias && bias_stride < 0) || act < 0 ||
        act >= kActs ||
        (GU && (!valid(GU, true) || GU->rows != H->rows || GU->cols != W->rows)))
        return MT_ERR_INVALID;
    if (H->rows == 0 || H->cols == 0) return MT_OK;
    Q8Params p = q8_params(X, W, bias, bias_stride, H);
    p.gu = view(GU);
    p.act = act;
    return run_q8<true>(p, workspace, ws_bytes, static_cast<hipStream_t>(stream));
}

size_t mt_gated_linear_q8_workspace(int64_t rows, int64_t in_f, int64_t features) {
    return workspace_of(rows, in_f, features, true);
}
int mt_gated_linear_q8_plan(int64_t rows, int64_t in_f, int64_t features, mt_lowbit_plan* plan) {
    return plan_of(rows, in_f, features, true, plan);
}

}  // extern "C"
