// ffn_api.hip -- the C ABI of include/mtffn.h but for its 8-bit products: gated feed-forward
// blocks in fp32, their elementwise passes, and the norm and clipping of gradients.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <new>
#include <vector>

#include "api_checks.hpp"
#include "clip_kernel.hpp"
#include "gate_kernel.hpp"
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

int run_clip(const mt_mat_f32* grads, const mt_mat_f32* out, int64_t count, bool scale,
             float most, float eps, float* norm, void* workspace, size_t ws_bytes, hipStream_t s) {
    if (count < 0 || count > kMaxTensors || (count > 0 && !grads) || !norm) return MT_ERR_INVALID;
    if (scale && (!(most >= 0.f) || !(eps >= 0.f))) return MT_ERR_INVALID;
    const mt_mat_f32* const to = out ? out : grads;
    Tensor d{};
    std::vector<const float*> at;
    for (int64_t i = 0; i < count; ++i) {
        if (!tensor_of(&grads[i], &to[i], scale, &d)) return MT_ERR_INVALID;
        if (scale && d.n > 0) at.push_back(d.dst);
    }
    std::sort(at.begin(), at.end());                   // no output twice
    if (std::adjacent_find(at.begin(), at.end()) != at.end()) return MT_ERR_INVALID;
    const size_t need = mt_grad_norm_workspace_f32(count);
    if (!workspace || ws_bytes < need || ((uintptr_t)workspace & 7)) return MT_ERR_WORKSPACE;
    double* const part = static_cast<double*>(workspace);

    // Launches: the dense tensors' by the table, the others' one by one.
    auto launches = [&](auto table, auto single) {
        ClipTable t;
        t.count = 0;
        t.chunks = 0;
        auto flush = [&] {
            if (t.count > 0) table(t, std::min<uint32_t>(t.chunks, kClipBlocks));
            t.count = 0;
            t.chunks = 0;
        };
        for (int64_t i = 0; i < count; ++i) {
            tensor_of(&grads[i], &to[i], scale, &d);
            if (d.n == 0) continue;
            if (!d.dense) {
                single(d.strided, (unsigned)std::min<int64_t>((d.n + 255) / 256, kStridedBlocks));
                continue;
            }
            const int64_t chunks = (d.n + kClipChunk - 1) / kClipChunk;
            if (t.count == kClipTensors || t.chunks + chunks > (int64_t)1 << 31) flush();
            t.src[t.count] = d.src;
            t.dst[t.count] = d.dst;
            t.n[t.count] = d.n;
            t.first[t.count++] = t.chunks;
            t.chunks += (uint32_t)chunks;
        }
        flush();
    };
    int parts = 0;
    launches(
        [&](const ClipTable& t, unsigned blocks) {
            hipLaunchKernelGGL(clip_squares, dim3(blocks), dim3(256), 0, s, t, part + parts);
            parts += (int)blocks;
        },
        [&](const ClipStrided& t, unsigned blocks) {
            hipLaunchKernelGGL(clip_squares_strided, dim3(blocks), dim3(256), 0, s, t, part + parts);
            parts += (int)blocks;
        });
    const ClipNorm c{part, parts, norm, most, eps};
    if (!scale || parts == 0) {
        hipLaunchKernelGGL(clip_norm, dim3(1), dim3(256), 0, s, c);
        return launched();
    }
    launches(
        [&](const ClipTable& t, unsigned blocks) {
            hipLaunchKernelGGL(clip_scale, dim3(blocks), dim3(256), 0, s, t, c);
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

size_t mt_gated_linear_workspace_f32(int64_t rows, int64_t in_f, int64_t features) {
    if (rows <= 0 || in_f < 0 || features <= 0 || rows >= kMaxDim || in_f >= kMaxDim ||
        features >= kMaxDim / 2)
        return 0;
    return (size_t)rows * (size_t)features * 8 + mt_linear_workspace_f32(rows, in_f, 2 * features);
}

int mt_gated_linear_f32(const mt_mat_f32* X, const mt_mat_f32* W, const float* bias,
                        int64_t bias_stride, int act, const mt_mat_f32* H, const mt_mat_f32* GU,
                        void* workspace, size_t ws_bytes, void* stream) {
    if (!valid(X, false) || !valid(W, false) || !valid(H, true) || !valid_act(act) ||
        X->cols != W->cols || W->rows % 2 != 0 || H->rows != X->rows || H->cols != W->rows / 2 ||
        (bias && bias_stride < 0) ||
        (GU && (!valid(GU, true) || GU->rows != X->rows || GU->cols != W->rows)))
        return MT_ERR_INVALID;
    if (H->rows == 0 || H->cols == 0) return MT_OK;
    mt_mat_f32 gu;
    char* ws = static_cast<char*>(workspace);
    if (GU) {
        gu = *GU;
    } else {
        const size_t own = (size_t)H->rows * (size_t)W->rows * 4;
        if (!ws || ws_bytes < own) return MT_ERR_WORKSPACE;
        gu = mt_mat_f32{reinterpret_cast<float*>(ws), 0, H->rows, W->rows, W->rows, 1, 1, 0};
        ws += own;
        ws_bytes -= own;
    }
    const int rc = mt_linear_forward_f32(X, W, bias, bias_stride, &gu, ws, ws_bytes, stream);
    return rc == MT_OK ? mt_gate_f32(&gu, act, H, stream) : rc;
}

size_t mt_grad_norm_workspace_f32(int64_t count) {
    if (count < 0 || count > kMaxTensors) return 0;
    return ((size_t)((count + kClipTensors - 1) / kClipTensors) * kClipBlocks + (size_t)count * kStridedBlocks + 1) * 8;
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
