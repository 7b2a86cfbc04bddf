// ffn_api.hip -- the C ABI of include/mtffn.h but for its 8-bit products: gated feed-forward
// blocks in fp32, their elementwise passes, and the norm and clipping of gradients.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <functional>
#include <new>
#include <vector>

#include "api_checks.hpp"
#include "clip_kernel.hpp"
#include "gate_f32_kernel.hpp"
#include "gate_kernel.hpp"
#include "gemm_configs.hpp"
#include "mtffn.h"

using namespace mtk;

namespace {

bool valid_act(int act) { return act >= 0 && act < kActs; }

template <bool BACK>
int run_gate(const mt_mat_f32* GU, const mt_mat_f32* dH, const mt_mat_f32* out, int64_t features,
             int act, void* stream) {
    if (GU->rows == 0 || features == 0) return MT_OK;
    GateParams p{view(GU), view(dH), view(out), GU->rows, (int)features, act};
    const bool units = unit(p.gu) && unit(p.dh) && unit(p.out);
    const int64_t n = p.M * (units ? (features + 3) / 4 : features);
    const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (units) hipLaunchKernelGGL((gate_rows<true, BACK>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((gate_rows<false, BACK>), grid, dim3(256), 0, s, p);
    return launched();
}

// The gradients with their sums over the rows: runs of rows, 8 at least (two a wave, loaded
// together), for eight workgroups on a CU.  (With sums in fp32, 509 x 2 x 2570: 10.4 us; 16 at
// least 14.0, 4 9.5, but 1024 x 2 x 2048 10.9, 10.9 and 12.7.)
int64_t bias_run(int64_t rows, int64_t strips) {
    const int64_t runs = std::min((rows + 7) / 8, std::max<int64_t>(8 * kCus / strips, 1));
    return ((rows + runs - 1) / runs + 3) / 4 * 4;
}
int64_t bias_runs(int64_t rows, int64_t strips) {
    const int64_t run = bias_run(rows, strips);
    return (rows + run - 1) / run;
}
int run_gate_bias(const mt_mat_f32* dH, const mt_mat_f32* GU, int act, const mt_mat_f32* dGU,
                  const GateBias& b, void* workspace, size_t ws_bytes, hipStream_t s) {
    const int64_t M = GU->rows, F = dH->cols;
    if (F == 0) return MT_OK;
    GateParams p{view(GU), view(dH), view(dGU), M, (int)F, act};
    const bool units = unit(p.gu) && unit(p.dh) && unit(p.out);
    const int64_t strips = (F + (units ? 255 : 63)) / (units ? 256 : 64);
    if (strips >= kMaxTiles) return MT_ERR_INVALID;
    const int64_t run = M ? bias_run(M, strips) : 4, runs = M ? bias_runs(M, strips) : 1;
    if (run >= kMaxDim) return MT_ERR_INVALID;
    float* const part = static_cast<float*>(workspace);
    if (runs > 1 && (!workspace || ws_bytes < (size_t)(runs * 2 * F) * 4)) return MT_ERR_WORKSPACE;
    const dim3 grid((unsigned)strips, (unsigned)runs);
    if (units) hipLaunchKernelGGL(gate_rows_sums<true>, grid, dim3(256), 0, s, p, b, part, (int)run);
    else hipLaunchKernelGGL(gate_rows_sums<false>, grid, dim3(256), 0, s, p, b, part, (int)run);
    if (runs > 1)
        hipLaunchKernelGGL(gate_bias_sum<>, dim3((unsigned)((2 * F + 63) / 64)), dim3(512), 0, s, part,
                           (int)runs, 2 * F, b);
    return launched();
}

// ---- gated projections in fp32 ---------------------------------------------------------

// How a call goes: straight from memory (few rows on the vector units; few rows and small
// products on the fp32 matrix units), tiles of gemm_f32_sp with the gate in their epilogue, or
// (operands with no neighbouring elements either way, or too far apart for the tiles' 32-bit
// offsets) the product to memory first.
enum GateKind { GATE_GEMV, GATE_FEW, GATE_TILES, GATE_APART };
constexpr int64_t kFewRows = 48;

// Times in us by workgroups on a CU, of a chunk of 16 inputs -- one workgroup on every fourth
// CU or fewer, on every CU, each further one there -- and of a workgroup's beginning and end.
// From products of 64-4096 rows, 512-4096 features, 256 and 2048 inputs.  (4096 x 2048 ->
// 2 x 4096: 128x256 687 us, 128x128 748, 64x128 1072; 1024 x 2048 -> 2 x 2048: 135, 104, 125;
// 256 x 2048 -> 2 x 2048: 114, 78, 67.)
struct GateTile {
    int bm, bn, per_cu;
    double sparse, full, more, fixed;
    GemmLaunchFn (*launcher)(int, int);
};
template <int C>
constexpr GateTile gate_tile(int per_cu, double sparse, double full, double more, double fixed,
                             GemmLaunchFn (*fn)(int, int)) {
    return {GateCfg<C>::BM, GateCfg<C>::BN, per_cu, sparse, full, more, fixed, fn};
}
constexpr GateTile kGateTiles[kNumGateCfg] = {
    gate_tile<0>(3, 0.45, 0.515, 0.40, 4, gate_launcher_cfg0),
    gate_tile<1>(2, 0.52, 0.73, 0.65, 6.5, gate_launcher_cfg1),
    gate_tile<2>(1, 0.79, 1.27, 0, 8, gate_launcher_cfg2)};

struct GatePlan {
    GateKind kind;
    int tile;                         // or (GATE_FEW) blocks of rows
    int tiles_m, tiles_n, splits, k_per_split;
    size_t partials;                  // bytes, 0 without splits
};
GatePlan gate_tiles_plan(int64_t M, int64_t F, int64_t K, double* time) {
    GatePlan best{};
    double& least = *time;
    const int64_t cols = (F + 31) / 32 * 64, chunks = (K + 15) / 16;
    for (int i = 0; i < kNumGateCfg; ++i) {
        const GateTile& t = kGateTiles[i];
        const int64_t tm = (M + t.bm - 1) / t.bm, tn = (cols + t.bn - 1) / t.bn;
        for (int64_t s = 1; s <= std::min<int64_t>(std::max<int64_t>(chunks / 4, 1), 32); ++s) {
            const int64_t per = (chunks + s - 1) / s;
            if ((chunks + per - 1) / per != s) continue;
            const int64_t wgs = tm * tn * s, slots = (int64_t)kCus * t.per_cu;
            const double fill = std::min(1.0, (double)wgs / kCus);
            auto round = [&](int64_t n) {
                const double one = t.sparse + (t.full - t.sparse) * std::max(0.0, (fill - 0.25) / 0.75);
                return (double)per * (one + (double)(n - 1) * t.more) + t.fixed;
            };
            double us = (double)(wgs / slots) * round(t.per_cu);
            if (wgs % slots) us += round((wgs % slots + kCus - 1) / kCus);
            if (s > 1) us += 4 + (double)(s + 1) * (double)M * (double)cols * 0.9e-6;
            if (least == 0 || us < least) {
                least = us;
                best = {GATE_TILES, i, (int)tm, (int)tn, (int)s, (int)(per * 16),
                        s > 1 ? (size_t)(s * M * cols) * 4 : 0};
            }
            if (wgs >= 4 * slots) break;
        }
    }
    return best;
}
// The layout in which the tiles read an operand (rows of a tile at most `rows`, the last of
// them `span` rows from the first), or -1.
int gate_layout(const RowView& v, int64_t K, int64_t span, bool weight) {
    if ((v.cs == 1 || K == 1) && span * v.rs < ((int64_t)1 << 30) - 16) return weight ? L_GKV : L_KV;
    if (v.rs == 1 && span < ((int64_t)1 << 30)) return weight ? L_GMV : L_MV;
    return -1;
}
// Rows that the vector units' kernel takes: more than four where the matrix units' blocks of 16
// features are few workgroups, each of which walks a long K.  (Against those and the tiles, us:
// 8 rows 2048 -> 2 x 512 4.5 and 11.3, 1024 -> 2 x 1024 4.8 and 6.8, 5632 -> 2 x 2048 18.8 and 28,
// but 512 -> 2 x 2048 6.1 and 4.8, 1285 -> 2 x 2570 13.2 and 7.6; 16 rows 4096 -> 2 x 1024 13.6 and
// 23.4, 8192 -> 2 x 512 12.2 and 18.1, but 1024 -> 2 x 1024 8.1 and 7.6, 5632 -> 2 x 2048 30.1 and
// 31.3.)
// (Its grid holds 4 features a workgroup.)
int64_t gemv_rows(int64_t F, int64_t K) {
    if (F > 4 * (kMaxTiles - 1)) return 0;
    if (F <= 1024) return K >= 2 * F ? 16 : 8;
    return F <= 2048 && K >= 2 * F ? 8 : 4;
}
// Rows that a kernel of the vector units is made for.
int gemv_made_for(int64_t M) { return M <= 2 ? (int)M : M <= 4 ? 4 : M <= 8 ? 8 : 16; }
// The fp32 matrix units' kernel (gate_few), whose waves walk all of K and read x for 16 features
// each: us by blocks of 16 rows of a workgroup, its beginning and end and 512 inputs of each
// round over the CUs.  (64 x 512 -> 2 x 2048: 7.9, 6.4 and 7.7 by one, two and three blocks, in
// tiles 13.3; 64 x 64 -> 2 x 32: 2.7, 3.5, 4.3, 6.6; 512 x 1024 -> 2 x 512: 23.3, 17.1, 21.3, 19.0; 128 x
// 2048 -> 2 x 256: 12.9, 16.5, 21.6, 14.7; 64 x 4000 -> 2 x 512: 23, 31, 40, 17.)  From up to
// 4096 rows, 2048 features and 1024 workgroups, which it is kept to beyond 48 rows.
struct GateFew {
    double fixed, round;
};
constexpr GateFew kGateFew[] = {{2.4, 2.55}, {2.9, 3.6}, {3.6, 4.75}};
// Blocks of rows, and the time; 0: none.
int few_blocks(int64_t M, int64_t F, int64_t K, double* us) {
    int best = 0;
    for (int mb = 1; mb <= 3; ++mb) {
        const int64_t wgs = (M + 16 * mb - 1) / (16 * mb) * ((F + 15) / 16);
        if (wgs > (M <= kFewRows ? kMaxTiles - 1 : 4 * kCus)) continue;
        const GateFew& c = kGateFew[mb - 1];
        const int64_t rounds = (wgs + kCus - 1) / kCus;
        // (more than two: 280 x 576 -> 2 x 1379, four rounds of the second, 21.8 us; in tiles 19.7)
        const double t = c.fixed + c.round * (double)K / 512 * (double)rounds * (rounds > 2 ? 1.12 : 1.0);
        if (best && t >= *us) continue;
        best = mb;
        *us = t;
    }
    return best;
}
GatePlan gate_plan(const mt_mat_f32* X, const mt_mat_f32* W, int* la, int* lb) {
    const int64_t M = X->rows, F = W->rows / 2, K = X->cols;
    const RowView x = view(X), w = view(W);
    const bool rows = K > 0 && (x.cs == 1 || K == 1) && (w.cs == 1 || K == 1);
    // (The product and the gate after it are not priced against the kernels here, although they are
    // less of some few rows into wide layers: 32 x 4096 -> 2 x 8192 61 us, in blocks of 32 rows 66.)
    if (rows && M <= gemv_rows(F, K)) return {GATE_GEMV};
    double few = 0;
    const int blocks = rows ? few_blocks(M, F, K, &few) : 0;
    if (blocks && few < 5) return {GATE_FEW, blocks};   // (tiles take 6.6 at least)
    // (a tile's rows; of the weight those of 128 features, and their up rows)
    *la = gate_layout(x, K, std::min<int64_t>(M, 256), false);
    *lb = gate_layout(w, K, F + std::min<int64_t>(F, 128), true);
    if (K == 0) return {GATE_APART};
    double us = 0;
    const GatePlan p = gate_tiles_plan(M, F, K, &us);
    if (blocks && (few < us || *la < 0 || *lb < 0)) return {GATE_FEW, blocks};
    if (*la < 0 || *lb < 0) return {GATE_APART};
    if ((int64_t)p.tiles_m * p.tiles_n * p.splits >= kMaxTiles) return {GATE_APART};
    return p;
}
size_t apart_bytes(const mt_mat_f32* X, const mt_mat_f32* W) {
    return (size_t)X->rows * (size_t)W->rows * 4;
}

int run_gated(const mt_mat_f32* X, const mt_mat_f32* W, const float* bias, int64_t bias_stride,
              int act, const mt_mat_f32* H, const mt_mat_f32* GU, void* workspace, size_t ws_bytes,
              hipStream_t s) {
    int la = -1, lb = -1;
    const GatePlan plan = gate_plan(X, W, &la, &lb);
    const RowView x = view(X), w = view(W), h = view(H), gu = view(GU);
    const int M = (int)X->rows, F = (int)H->cols, K = (int)X->cols;
    if (plan.kind == GATE_GEMV || plan.kind == GATE_FEW) {
        const GateGemv p{x.p, x.rs, w.p, w.rs, bias, bias_stride, h, gu, M, F, K, act};
        auto go = [&](auto kernel, int features, int rows) {
            const dim3 grid((unsigned)((F + features - 1) / features), (unsigned)((M + rows - 1) / rows));
            hipLaunchKernelGGL(kernel, grid, dim3(512), 0, s, p);
        };
        if (plan.kind == GATE_FEW) {
            if (plan.tile == 1) go(gate_few<1>, 16, 16);
            else if (plan.tile == 2) go(gate_few<2>, 16, 32);
            else go(gate_few<3>, 16, 48);
        } else {
            switch (gemv_made_for(M)) {
                case 1: go(gate_gemv<1, 4>, 4, 1); break;
                case 2: go(gate_gemv<2, 4>, 4, 2); break;
                case 4: go(gate_gemv<4, 4>, 4, 4); break;
                case 8: go(gate_gemv<8, 2>, 2, 8); break;
                default: go(gate_gemv<16, 2>, 2, 16);
            }
        }
        return launched();
    }
    if (plan.kind == GATE_APART) {
        mt_mat_f32 to;
        char* ws = static_cast<char*>(workspace);
        if (GU) {
            to = *GU;
        } else {
            const size_t own = apart_bytes(X, W);
            if (!ws || ws_bytes < own) return MT_ERR_WORKSPACE;
            to = mt_mat_f32{reinterpret_cast<float*>(ws), 0, X->rows, W->rows, W->rows, 1, 1, 0};
            ws += own;
            ws_bytes -= own;
        }
        const int rc = mt_linear_forward_f32(X, W, bias, bias_stride, &to, ws, ws_bytes, s);
        return rc == MT_OK ? mt_gate_f32(&to, act, H, s) : rc;
    }
    if (plan.partials > 0 && (!workspace || ws_bytes < plan.partials)) return MT_ERR_WORKSPACE;
    GemmParams p{};
    p.A = x.p;
    p.a_mn = x.rs;
    p.a_k = x.cs;
    p.B = w.p;
    p.b_mn = w.rs;
    p.b_k = w.cs;
    p.M = M;
    p.N = (F + 31) / 32 * 64;
    p.K = K;
    p.batch = 1;
    p.c_n_inner = p.N;
    p.bias = bias;
    p.bias_stride = bias_stride;
    p.splits = plan.splits;
    p.k_per_split = plan.k_per_split;
    p.ws = static_cast<float*>(workspace);
    p.ws_vec = ((uintptr_t)workspace & 15) == 0;
    p.tiles_m = plan.tiles_m;
    p.tiles_n = plan.tiles_n;
    p.group_m = 4;
    p.gate = {h.p, h.rs, h.cs, gu.p, gu.rs, gu.cs, F, act};
    const GemmLaunchFn fn = kGateTiles[plan.tile].launcher(la, lb);
    hipError_t e = fn(p, (unsigned)(plan.tiles_m * plan.tiles_n * plan.splits), s);
    if (e != hipSuccess && e != hipErrorStreamCaptureUnsupported) return MT_ERR_HIP;
    if (plan.splits > 1) {
        const int64_t n = (int64_t)M * ((F + 3) / 4);
        hipLaunchKernelGGL(gate_sum<>, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 8192)), dim3(256),
                           0, s, GateSum{p.ws, p.N, p.splits, bias, bias_stride, h, gu, M, F, act});
    }
    return launched();
}

// ---- clipping --------------------------------------------------------------------

constexpr int64_t kMaxTensors = (int64_t)1 << 20;
constexpr int64_t kMaxElements = (int64_t)1 << 42;   // of a tensor: its chunks are counted in 32 bits
constexpr int kStridedBlocks = 256;

// A tensor of up to three axes, as few as it takes, and whether it is one run.
struct Tensor {
    const float* src;
    float* dst;
    int64_t n;
    bool dense;
    ClipStrided strided;
};
bool tensor_of(const mt_mat_f32* g, const mt_mat_f32* o, bool written, Tensor* t) {
    for (const mt_mat_f32* m : {g, o})
        if (m->rows < 0 || m->cols < 0 || m->batch < 0 || m->row_stride < 0 || m->col_stride < 0 ||
            m->batch_stride < 0 || m->offset < 0)
            return false;
    if (o->rows != g->rows || o->cols != g->cols || o->batch != g->batch) return false;
    const int64_t size[3] = {g->batch, g->rows, g->cols};
    const int64_t a[3] = {g->batch_stride, g->row_stride, g->col_stride};
    const int64_t b[3] = {o->batch_stride, o->row_stride, o->col_stride};
    t->n = size[0] && size[1] && size[2] ? 1 : 0;
    if (t->n == 0) return true;
    for (int64_t s : size) {
        if (t->n > kMaxElements / s) return false;
        t->n *= s;
    }
    if (!g->base || !o->base) return false;
    t->src = g->base + g->offset;
    t->dst = const_cast<float*>(o->base) + o->offset;
    t->dense = true;
    int64_t run = 1;
    for (int i = 2; i >= 0; --i) {
        if (size[i] > 1) {
            if (written && b[i] == 0) return false;    // two elements of an output on one address
            t->dense = t->dense && a[i] == run && b[i] == run;
        }
        run *= size[i];
        t->strided.size[i] = size[i];
        t->strided.src_stride[i] = a[i];
        t->strided.dst_stride[i] = b[i];
    }
    t->strided.src = t->src;
    t->strided.dst = t->dst;
    return true;
}

// What tensors' elements lie in, of a strided one its first element: views may lie between
// each other's elements.
struct Extent {
    const float *begin, *end;
    bool operator<(const Extent& o) const { return std::less<const float*>()(begin, o.begin); }
};
struct Extents {
    std::vector<Extent> written, read;
    // false where t's output is over itself in another order
    bool add(const Tensor& t) {
        const int64_t n = t.dense ? t.n : 1;
        written.push_back({t.dst, t.dst + n});
        if (t.src != t.dst) {
            read.push_back({t.src, t.src + n});
            return true;
        }
        for (int i = 0; i < 3 && !t.dense; ++i)
            if (t.strided.size[i] > 1 && t.strided.src_stride[i] != t.strided.dst_stride[i]) return false;
        return true;
    }
    // whether something written lies over another tensor
    bool overlap() {
        for (auto* v : {&written, &read})              // (out of one buffer they are in order)
            if (!std::is_sorted(v->begin(), v->end())) std::sort(v->begin(), v->end());
        for (size_t i = 1; i < written.size(); ++i)
            if (written[i].begin < written[i - 1].end) return true;
        size_t i = 0;
        for (const Extent& r : read) {
            while (i < written.size() && written[i].end <= r.begin) ++i;
            if (i < written.size() && written[i].begin < r.end) return true;
        }
        return false;
    }
};

int run_clip(const mt_mat_f32* grads, const mt_mat_f32* out, int64_t count, bool scale,
             float most, float eps, float* norm, void* workspace, size_t ws_bytes, hipStream_t s) {
    if (count < 0 || count > kMaxTensors || (count > 0 && !grads) || !norm) return MT_ERR_INVALID;
    if (scale && (!(most >= 0.f) || !(eps >= 0.f))) return MT_ERR_INVALID;
    const mt_mat_f32* const to = out ? out : grads;
    Tensor d{};
    Extents extents;
    int64_t all = 0, pieces = 0;
    bool dense = true;
    for (int64_t i = 0; i < count; ++i) {
        if (!tensor_of(&grads[i], &to[i], scale, &d)) return MT_ERR_INVALID;
        all += d.n;
        if (d.n == 0) continue;
        pieces += (d.n + kClipOneChunk - 1) / kClipOneChunk;
        dense = dense && d.dense;
        if (scale && !extents.add(d)) return MT_ERR_INVALID;
    }
    if (extents.overlap()) return MT_ERR_INVALID;
    const size_t need = mt_grad_norm_workspace_f32(count);
    if (!workspace || ws_bytes < need || ((uintptr_t)workspace & 7)) return MT_ERR_WORKSPACE;
    double* const part = static_cast<double*>(workspace);

    // Launches: the dense tensors' by the table, the others' one by one.
    auto launches = [&](bool apart, int chunk, auto table, auto single) {
        ClipTable t;
        auto clear = [&] {
            t.count = 0;
            t.chunks = 0;
            std::fill(t.first, t.first + kClipTensors, ~0u);
        };
        auto flush = [&] {
            if (t.count > 0) table(t, std::min<uint32_t>(t.chunks, kClipBlocks));
            clear();
        };
        clear();
        t.to = apart ? kClipTensors / 2 : 0;
        const int most = kClipTensors - t.to;
        for (int64_t i = 0; i < count; ++i) {
            tensor_of(&grads[i], &to[i], scale, &d);
            if (d.n == 0) continue;
            if (!d.dense) {
                single(d.strided, (unsigned)std::min<int64_t>((d.n + 255) / 256, kStridedBlocks));
                continue;
            }
            const int64_t chunks = (d.n + chunk - 1) / chunk;
            if (t.count == most || t.chunks + chunks > (int64_t)1 << 31) flush();
            t.at[t.count] = const_cast<float*>(d.src);
            if (apart) t.at[t.count + t.to] = d.dst;
            t.last[t.count] = (uint16_t)((d.n - 1) % chunk);
            t.first[t.count++] = t.chunks;
            t.chunks += (uint32_t)chunks;
        }
        flush();
    };
    if (dense && pieces > 0 && pieces <= kClipOneWaves * kClipOnePieces) {
        launches(
            out != nullptr, kClipOneChunk,
            [&](const ClipTable& t, unsigned) {
                hipLaunchKernelGGL(clip_one<>, dim3(1), dim3(64 * kClipOneWaves), 0, s, t,
                                   ClipNorm{part, 0, norm, most, eps}, (int)scale);
            },
            [](const ClipStrided&, unsigned) {});
        return launched();
    }
    int parts = 0;
    launches(
        false, kClipChunk,
        [&](const ClipTable& t, unsigned blocks) {
            hipLaunchKernelGGL(clip_squares, dim3(blocks), dim3(kClipThreads), 0, s, t, part + parts);
            parts += (int)blocks;
        },
        [&](const ClipStrided& t, unsigned blocks) {
            hipLaunchKernelGGL(clip_squares_strided, dim3(blocks), dim3(256), 0, s, t, part + parts);
            parts += (int)blocks;
        });
    const bool past = out != nullptr && all * 4 > kClipStream;
    ClipNorm c{part, parts, norm, most, eps};
    if (!scale || parts == 0) {
        hipLaunchKernelGGL(clip_norm, dim3(1), dim3(kClipThreads), 0, s, c);
        return launched();
    }
    if (parts > kClipMostParts) {
        c.norm = nullptr;
        hipLaunchKernelGGL(clip_norm, dim3(1), dim3(kClipThreads), 0, s, c);
        c = {part + parts, 1, norm, most, eps};
    }
    launches(
        out != nullptr, kClipChunk,
        [&](const ClipTable& t, unsigned blocks) {
            if (past) hipLaunchKernelGGL(clip_scale<true>, dim3(blocks), dim3(kClipThreads), 0, s, t, c);
            else hipLaunchKernelGGL(clip_scale<false>, dim3(blocks), dim3(kClipThreads), 0, s, t, c);
        },
        [&](const ClipStrided& t, unsigned blocks) {
            hipLaunchKernelGGL(clip_scale_strided, dim3(blocks), dim3(256), 0, s, t, c);
        });
    return launched();
}

}  // namespace

extern "C" {

int mt_gate_f32(const mt_mat_f32* GU, int act, const mt_mat_f32* H, void* stream) {
    if (!valid(GU, false) || !valid(H, true) || !valid_act(act) || GU->rows != H->rows ||
        GU->cols != 2 * H->cols)
        return MT_ERR_INVALID;
    return run_gate<false>(GU, nullptr, H, H->cols, act, stream);
}

int mt_gate_backward_f32(const mt_mat_f32* dH, const mt_mat_f32* GU, int act, const mt_mat_f32* dGU,
                         void* stream) {
    if (!valid(dH, false) || !valid(GU, false) || !valid(dGU, true) || !valid_act(act) ||
        GU->rows != dH->rows || GU->cols != 2 * dH->cols || !same_shape(GU, dGU))
        return MT_ERR_INVALID;
    return run_gate<true>(GU, dH, dGU, dH->cols, act, stream);
}

size_t mt_gate_backward_bias_workspace_f32(int64_t rows, int64_t features) {
    if (rows <= 0 || features <= 0 || rows >= kMaxDim || features >= kMaxDim / 2) return 0;
    // (of rows with neighbouring elements: of others the runs are fewer)
    const int64_t runs = bias_runs(rows, (features + 255) / 256);
    return runs > 1 ? (size_t)(runs * 2 * features) * 4 : 0;
}

int mt_gate_backward_bias_f32(const mt_mat_f32* dH, const mt_mat_f32* GU, int act,
                              const mt_mat_f32* dGU, float* db, int64_t db_stride, float beta,
                              void* workspace, size_t ws_bytes, void* stream) {
    if (!valid(dH, false) || !valid(GU, false) || !valid(dGU, true) || !valid_act(act) ||
        GU->rows != dH->rows || GU->cols != 2 * dH->cols || !same_shape(GU, dGU) ||
        (dH->cols > 0 && (!db || db_stride <= 0)) || ((uintptr_t)workspace & 3) != 0)
        return MT_ERR_INVALID;
    return run_gate_bias(dH, GU, act, dGU, {db, db_stride, beta}, workspace, ws_bytes,
                         static_cast<hipStream_t>(stream));
}

size_t mt_gated_linear_workspace_f32(const mt_mat_f32* X, const mt_mat_f32* W) {
    if (!valid(X, false) || !valid(W, false) || X->cols != W->cols || X->rows == 0 || W->rows < 2)
        return 0;
    int la, lb;
    const GatePlan p = gate_plan(X, W, &la, &lb);
    if (p.kind != GATE_APART) return p.partials;
    return apart_bytes(X, W) + mt_linear_workspace_f32(X->rows, X->cols, W->rows);
}

int mt_gated_linear_plan_f32(const mt_mat_f32* X, const mt_mat_f32* W, mt_gate_plan* plan) {
    if (!valid(X, false) || !valid(W, false) || X->cols != W->cols || X->rows == 0 || W->rows < 2 ||
        !plan)
        return MT_ERR_INVALID;
    int la, lb;
    const GatePlan p = gate_plan(X, W, &la, &lb);
    *plan = {p.kind == GATE_TILES ? 1 : p.kind == GATE_APART ? 2 : 0, 0, 0,
             p.kind == GATE_TILES ? p.splits : 1, p.kind == GATE_GEMV ? gemv_made_for(X->rows) : 0};
    if (p.kind == GATE_FEW) plan->tile_rows = 16 * p.tile;
    if (p.kind == GATE_TILES) {
        plan->tile_rows = kGateTiles[p.tile].bm;
        plan->tile_cols = kGateTiles[p.tile].bn;
    }
    return MT_OK;
}

int mt_gated_linear_f32(const mt_mat_f32* X, const mt_mat_f32* W, const float* bias,
                        int64_t bias_stride, int act, const mt_mat_f32* H, const mt_mat_f32* GU,
                        void* workspace, size_t ws_bytes, void* stream) {
    if (!valid(X, false) || !valid(W, false) || !valid(H, true) || !valid_act(act) ||
        X->cols != W->cols || W->rows % 2 != 0 || H->rows != X->rows || H->cols != W->rows / 2 ||
        (bias && bias_stride < 0) || ((uintptr_t)workspace & 3) != 0 ||
        (GU && (!valid(GU, true) || GU->rows != X->rows || GU->cols != W->rows)))
        return MT_ERR_INVALID;
    if (H->rows == 0 || H->cols == 0) return MT_OK;
    return run_gated(X, W, bias, bias_stride, act, H, GU, workspace, ws_bytes,
                     static_cast<hipStream_t>(stream));
}

size_t mt_grad_norm_workspace_f32(int64_t count) {
    if (count < 0 || count > kMaxTensors) return 0;
    const size_t tables = (size_t)((count + kClipTensors - 1) / kClipTensors);
    return (tables * kClipBlocks + (size_t)count * kStridedBlocks + 1) * 8;
}

int mt_grad_norm_f32(const mt_mat_f32* grads, int64_t count, float* norm, void* workspace,
                     size_t ws_bytes, void* stream) {
    try {
        return run_clip(grads, nullptr, count, false, 0.f, 0.f, norm, workspace, ws_bytes,
                        static_cast<hipStream_t>(stream));
    } catch (const std::bad_alloc&) {
        return MT_ERR_HIP;
    }
}

int mt_clip_grad_norm_f32(const mt_mat_f32* grads, const mt_mat_f32* out, int64_t count,
                          float max_norm, float eps, float* norm, void* workspace, size_t ws_bytes,
                          void* stream) {
    try {
        return run_clip(grads, out, count, true, max_norm, eps, norm, workspace, ws_bytes,
                        static_cast<hipStream_t>(stream));
    } catch (const std::bad_alloc&) {
        return MT_ERR_HIP;
    }
}

}  // extern "C"
