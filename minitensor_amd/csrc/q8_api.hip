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
// Bytes between a tile's rows: their offsets, 255 of them and a chunk, are 32-bit.
constexpr int64_t kMaxRow = ((int64_t)1 << 24) - 256;
// Times in us by workgroups on a CU, of a chunk of 128 inputs and of a workgroup's beginning
// and end, from products of 64-4096 rows, 1000-16384 columns, 512 and 4096 inputs; workgroups
// go in rounds over the CUs.  (2048 x 4096 -> 8192: 256x256 tiles 66-69 us, 128x256 73-78,
// 128x128 90-100, 64x128 117-124; 1024 x 4096 -> 4096: 49, 33, 26, 33; 256 x 4096 -> 4096:
// 46, 28, 21, 15.)
struct Q8Tile {
    int bm, bn, per_cu;
    double alone, more, fixed;        // one workgroup on the CU, each further one; a workgroup
};
constexpr Q8Tile kTiles[] = {{64, 128, 2, 0.34, 0.45, 2.2},
                             {128, 128, 2, 0.56, 0.70, 4},
                             {128, 256, 1, 0.88, 0, 6.5},
                             {256, 256, 1, 1.6, 0, 10}};

// Variants of the kernel that reads both operands straight from memory (q8_few): blocks of 16
// rows and of 16 columns (gated ones counted twice) of a workgroup, and us of a launch, of each
// round of workgroups over the CUs, of 2048 inputs in it; 2.5 us a million outputs, which go to
// memory one by one.  From 80-4096 rows, 64-4096 columns, 64-4096 inputs.  (256 x 2048 -> 512:
// 5.8, 4.9, 4.9, 5.9, 8.2 and 8.0 us by these, 9.1 in tiles; 80 x 2048 -> 4096 11.2, 9.6, 10.2, 8.7,
// 8.3, 8.2 and 9.3; 512 x 512 -> 512 4.1, 3.8, 3.9, 3.5, 4.4, 4.3 and 5.7; 1024 x 4096 -> 512 30.7,
// 23.9, 23.9, 17.2, 14.4, 14.0 and 14.4.  Of few rows a weight that is read twice costs more: 33 x
// 2048 -> 8192 7.6 by the fifth, 9.4 by the last; 20 x 4096 -> 4096 6.8 by the second, 9.4 by the
// third.  Of rows on multiples of four bytes: at odd addresses a launch takes longer, one row
// 4095 -> 4096 7.6 us for 5.0, 256 x 2047 -> 512 6.8 for 5.2, and so does a copy before the tiles,
// neither of which is priced.)
struct Q8Few {
    int mb, nc;
    double fixed, round, inputs;
};
constexpr Q8Few kFew[] = {{1, 1, 1.8, 0.38, 1.6}, {2, 1, 2.0, 0.3, 2.45}, {1, 2, 2.0, 0.3, 2.45},
                          {2, 2, 2.2, 0.3, 3.35}, {4, 2, 2.5, 0.3, 4.9},  {2, 4, 2.6, 0.3, 5.1}};
// The best of them, or nullptr: beyond 64 rows up to 2048 workgroups are measured.
const Q8Few* few_variant(int64_t M, int64_t cols, int64_t K, bool gated, double* us) {
    const Q8Few* best = nullptr;
    if (K >= kQ8Segment) return best;
    for (const Q8Few& f : kFew) {
        if (gated && f.nc == 1) continue;
        const int64_t wgs = (M + 16 * f.mb - 1) / (16 * f.mb) * ((cols + 16 * f.nc - 1) / (16 * f.nc));
        if (wgs > (M <= 64 ? kMaxTiles - 1 : 8 * kCus)) continue;
        const double t = f.fixed + 2.5e-6 * (double)M * (double)cols +
                         (double)((wgs + kCus - 1) / kCus) * (f.round + f.inputs * (double)K / 2048);
        if (best && t >= *us) continue;
        best = &f;
        *us = t;
    }
    return best;
}

enum Kind { FEW, LONG, TILES };
struct Q8Plan {
    Kind kind;
    int bm, bn;
    int splits, k_per_split;
    int64_t tiles;                    // the splits' among them
    int64_t part_n;
    size_t partials;                  // bytes, 0 without splits
    const Q8Few* few;
};

// cols: columns of the launch (gated: whole blocks of 32 features, twice).
Q8Plan q8_plan(int64_t M, int64_t cols, int64_t K, bool gated) {
    if (K > kMaxRow) return {LONG, 0, 0, 1, 0, 0, 0, 0, nullptr};
    double few_us = 0;
    const Q8Few* const few = few_variant(M, cols, K, gated, &few_us);
    const Q8Plan direct{FEW, 0, 0, 1, 0, 0, 0, 0, few};
    // (No tiles take less; of 16 rows and fewer they waste three quarters and more.  But their
    // splits are not to be had so, and of a long K into few columns a few workgroups walk all of
    // it: 16 x 65536 -> 16 56 us, where 17 rows go in 32 splits of tiles and take 13.)
    if (few && (few_us < 4.5 || M <= 16)) return direct;
    Q8Plan best{};
    double least = 0;
    const int64_t chunks = std::max<int64_t>(1, (K + 127) / 128);
    const int64_t fewest = std::max<int64_t>(1, (K + kMaxTerms - 1) / kMaxTerms);
    for (const Q8Tile& t : kTiles) {
        const int64_t tm = (M + t.bm - 1) / t.bm, tn = (cols + t.bn - 1) / t.bn;
        for (int64_t s = fewest; s <= std::max(fewest, std::min<int64_t>(chunks, 32)); ++s) {
            const int64_t per = (chunks + s - 1) / s, splits = (chunks + per - 1) / per;
            if (splits != s && s != fewest) continue;
            const int64_t wgs = tm * tn * splits, slots = (int64_t)kCus * t.per_cu;
            auto round = [&](int64_t n) {
                return (double)per * (t.alone + (double)(n - 1) * t.more) + t.fixed * (0.4 + 0.6 * (double)n);
            };
            double us = (double)(wgs / slots) * round(t.per_cu);
            if (wgs % slots) us += round((wgs % slots + kCus - 1) / kCus);
            if (splits > 1) us += 4 + (double)(splits + 1) * (double)M * (double)cols * 0.9e-6;
            if (least == 0 || us < least) {
                least = us;
                best = {TILES, t.bm, t.bn, (int)splits, (int)(per * 128), wgs, tn * t.bn,
                        splits > 1 ? (size_t)(splits * M) * (size_t)(tn * t.bn) * 4 : 0, nullptr};
            }
            if (wgs >= 4 * slots) break;
        }
    }
    // (the tiles' times are without a launch, 2 us)
    if (few && few_us < least + 2) return direct;
    return best;
}
int64_t launch_cols(int64_t n, bool gated) { return gated ? (n + 31) / 32 * 64 : n; }

// Rows on multiples of `bytes`.
bool on(int bytes, const mt_rows_q8* r) {
    return r->cols == 0 || (((uintptr_t)r->q % bytes) == 0 && (r->rows <= 1 || r->row_stride % bytes == 0));
}
// Whether the tiles take the rows as they lie.
// (of no inputs nothing is read)
bool in_place(const mt_rows_q8* r) {
    return r->cols == 0 || (on(16, r) && (r->rows <= 1 || r->row_stride <= kMaxRow));
}
size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// The workspace: the splits' sums, then rows of x and of the weight that do not lie as the
// tiles take them, `row` bytes each: whole chunks of the tiles' k, zeros at the end.  (A chunk
// of a row is then one or two cache lines: 1024 rows 2048 -> 4096 in place, rows 2048 bytes
// apart 19.2 us, 2064 25.3.  And where both operands are copied no chunk is short: 1027 rows
// 2047 -> 4095 33.7 us, padded to 16 bytes 37.5.)
struct Q8Space {
    size_t x, w, all;
    int64_t row;
};
Q8Space q8_space(const Q8Plan& plan, const mt_rows_q8* X, const mt_rows_q8* W) {
    Q8Space s{};
    if (plan.kind != TILES) return s;
    const int64_t to = plan.bn == 256 ? 128 : 64;
    s.row = (X->cols + to - 1) / to * to;
    s.x = round16(plan.partials);
    s.w = s.x + (in_place(X) ? 0 : (size_t)(X->rows * s.row));
    s.all = s.w + (in_place(W) ? 0 : (size_t)(W->rows * s.row));
    if (s.all) s.all += 15;           // (from any address)
    return s;
}

template <bool GATED>
void launch_few(const Q8Params& p, const Q8Few& f, bool words, hipStream_t s) {
    using std::integral_constant;
    auto go = [&](auto mb, auto nc, auto kind) {
        constexpr int F = 16 * nc() / (GATED ? 2 : 1);
        const int64_t wgs = (((int64_t)p.N + F - 1) / F) * (((int64_t)p.M + 16 * mb() - 1) / (16 * mb()));
        hipLaunchKernelGGL((q8_few<mb(), nc(), GATED, kind()>), dim3((unsigned)wgs), dim3(512), 0, s, p);
    };
    auto blocks = [&](auto kind) {
        constexpr integral_constant<int, 1> one{};
        constexpr integral_constant<int, 2> two{};
        if constexpr (!GATED) {
            if (f.nc == 1) return f.mb == 1 ? go(one, one, kind) : go(two, one, kind);
        }
        if (f.nc == 4) go(two, integral_constant<int, 4>{}, kind);
        else if (f.mb == 4) go(integral_constant<int, 4>{}, two, kind);
        else if (f.mb == 2) go(two, two, kind);
        else go(one, two, kind);
    };
    if (words) blocks(integral_constant<int, Q8_WORDS>{});
    else blocks(integral_constant<int, Q8_BYTES>{});
}
template <bool GATED>
void launch_tiles(const Q8Params& p, const Q8Plan& plan, hipStream_t s) {
    const dim3 grid((unsigned)plan.tiles);
    if (plan.bm == 64)
        hipLaunchKernelGGL((q8_gemm<64, 128, 32, 64, 64, 5, GATED>), grid, dim3(256), 0, s, p);
    else if (plan.bm == 128 && plan.bn == 128)
        hipLaunchKernelGGL((q8_gemm<128, 128, 64, 64, 64, 5, GATED>), grid, dim3(256), 0, s, p);
    else if (plan.bm == 128)
        hipLaunchKernelGGL((q8_gemm<128, 256, 64, 64, 128, 2, GATED>), grid, dim3(512), 0, s, p);
    else
        hipLaunchKernelGGL((q8_gemm<256, 256, 64, 128, 128, 2, GATED>), grid, dim3(512), 0, s, p);
}

template <bool GATED>
int run_q8(Q8Params& p, const mt_rows_q8* X, const mt_rows_q8* W, void* workspace, size_t ws_bytes,
           hipStream_t s) {
    const Q8Plan plan = q8_plan(p.M, launch_cols(p.N, GATED), p.K, GATED);
    p.splits = 1;
    if (plan.kind == FEW) {
        launch_few<GATED>(p, *plan.few, on(4, X) && on(4, W), s);
        return launched();
    }
    if (plan.kind == LONG) {
        const int64_t blocks = ((int64_t)p.M + 15) / 16 * (((int64_t)p.N + 15) / 16);
        if (blocks >= kMaxTiles) return MT_ERR_INVALID;
        hipLaunchKernelGGL((q8_few<1, GATED ? 2 : 1, GATED, Q8_LONG>), dim3((unsigned)blocks), dim3(512),
                           0, s, p);
        return launched();
    }
    if (plan.tiles >= kMaxTiles) return MT_ERR_INVALID;
    const Q8Space space = q8_space(plan, X, W);
    if (space.all > 0 && (!workspace || ws_bytes < space.all)) return MT_ERR_WORKSPACE;
    char* const ws = reinterpret_cast<char*>(round16((uintptr_t)workspace));
    Q8Align a{};
    a.ld_dst = space.row;
    a.K = p.K;
    auto align = [&](int i, const mt_rows_q8* r, size_t at, const int8_t*& q, int64_t& ld) {
        if (in_place(r)) return;
        a.src[i] = r->q;
        a.ld[i] = r->row_stride;
        a.rows[i] = r->rows;
        a.dst[i] = reinterpret_cast<int8_t*>(ws + at);
        q = a.dst[i];
        ld = space.row;
    };
    align(0, X, space.x, p.x, p.x_m);
    align(1, W, space.w, p.w, p.w_n);
    if (const int64_t n = a.rows[0] + a.rows[1]; n > 0) {
        a.wave_blocks = p.K >= 16 ? (int)std::min<int64_t>((n + 3) / 4, 1 << 16) : 0;
        const int64_t parts = p.K < space.row ? std::min<int64_t>((n + 255) / 256, 1 << 12) : 0;
        hipLaunchKernelGGL(q8_align_rows<>, dim3((unsigned)(a.wave_blocks + parts)), dim3(256), 0, s, a);
        if (a.rows[0] > 0 && a.rows[1] > 0) p.K = (int)space.row;
    }
    p.splits = plan.splits;
    p.k_per_split = plan.k_per_split;
    p.part = reinterpret_cast<int32_t*>(ws);
    p.part_n = plan.part_n;
    launch_tiles<GATED>(p, plan, s);
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
size_t workspace_of(const mt_rows_q8* X, const mt_rows_q8* W, bool gated) {
    if (!valid(X) || !valid(W) || X->cols != W->cols || X->rows == 0 || W->rows < (gated ? 2 : 1))
        return 0;
    const Q8Plan plan = q8_plan(X->rows, launch_cols(gated ? W->rows / 2 : W->rows, gated), X->cols,
                                gated);
    return q8_space(plan, X, W).all;
}
int plan_of(int64_t rows, int64_t in_f, int64_t out_f, bool gated, mt_q8_plan* plan) {
    if (rows <= 0 || in_f <= 0 || out_f <= 0 || rows >= kMaxDim || in_f >= kMaxDim ||
        out_f >= (gated ? kMaxDim / 2 : kMaxDim) || !plan)
        return MT_ERR_INVALID;
    const Q8Plan p = q8_plan(rows, launch_cols(out_f, gated), in_f, gated);
    *plan = {p.bm, p.bn, p.splits, 0, 0};
    if (p.kind == FEW) {
        plan->row_blocks = p.few->mb;
        plan->column_blocks = p.few->nc;
    } else if (p.kind == LONG) {
        plan->row_blocks = 1;
        plan->column_blocks = gated ? 2 : 1;
    }
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
    return run_q8<false>(p, X, W, workspace, ws_bytes, static_cast<hipStream_t>(stream));
}

size_t mt_linear_q8_workspace(const mt_rows_q8* X, const mt_rows_q8* W) {
    return workspace_of(X, W, false);
}
int mt_linear_q8_plan(int64_t rows, int64_t in_f, int64_t out_f, mt_q8_plan* plan) {
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
    return run_q8<true>(p, X, W, workspace, ws_bytes, static_cast<hipStream_t>(stream));
}

size_t mt_gated_linear_q8_workspace(const mt_rows_q8* X, const mt_rows_q8* W) {
    return workspace_of(X, W, true);
}
int mt_gated_linear_q8_plan(int64_t rows, int64_t in_f, int64_t features, mt_q8_plan* plan) {
    return plan_of(rows, in_f, features, true, plan);
}

}  // extern "C"
