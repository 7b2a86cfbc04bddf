// gate_kernel.hpp -- activations of a gated feed-forward block and its elementwise passes
// (include/mtffn.h): h = act(g) * u, and its gradients.
//
// The passes are bound by memory: 12 and 20 bytes per element of h (backward, 4096 x 2 x 4096:
// 52 us, 6.4 TB/s, part of it from the 256 MB cache; 509 x 2 x 2570: 6.6 us, a launch and a load).  exp and erfc are the
// device library's; a quotient by 1 + e, 1 <= 1 + e <= 2, is a product with v_rcp_f32 (1 ulp).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "row_access.hpp"

namespace mtk {

enum : int { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2, ACT_RELU = 3, ACT_SIGMOID = 4, kActs = 5 };

// 1/(1 + exp(-a)) and, in rest, 1/(1 + exp(a)), neither by a difference.
__device__ __forceinline__ float logistic(float a, float& rest) {
    const float e = expf(-__builtin_fabsf(a)), r = __builtin_amdgcn_rcpf(1.f + e), s = e * r;
    rest = a < 0.f ? r : s;
    return a < 0.f ? s : r;
}

constexpr float kGeluC = 0.7978845608028654f;        // sqrt(2/pi)
constexpr float kGeluA = 0.044715f;
constexpr float kHalfRoot = 0.7071067811865476f;     // sqrt(1/2)
constexpr float kNormalPeak = 0.3989422804014327f;   // 1/sqrt(2 pi)

// act(a) and, with SLOPE, its derivative in d.
template <int ACT, bool SLOPE>
__device__ __forceinline__ float act_at(float a, float& d) {
    float q;
    if constexpr (ACT == ACT_SILU || ACT == ACT_SIGMOID) {
        const float t = logistic(a, q);
        // (where t*q is zero, a may be infinite)
        const float p = t * q;
        if constexpr (SLOPE) d = ACT == ACT_SIGMOID ? p : p == 0.f ? t : __builtin_fmaf(a, p, t);
        return ACT == ACT_SIGMOID ? t : a * t;
    } else if constexpr (ACT == ACT_GELU) {
        const float t = 0.5f * erfcf(-kHalfRoot * a);
        if constexpr (SLOPE) {
            const float p = kNormalPeak * expf(-0.5f * a * a);
            d = p == 0.f ? t : __builtin_fmaf(a, p, t);
        }
        return a * t;
    } else if constexpr (ACT == ACT_GELU_TANH) {
        // (1 + tanh z)/2 = 1/(1 + exp(-2z))
        const float a2 = a * a;
        const float t = logistic(2.f * kGeluC * a * __builtin_fmaf(kGeluA, a2, 1.f), q);
        if constexpr (SLOPE) {
            const float p = t * q;
            d = p == 0.f ? t
                         : __builtin_fmaf(2.f * kGeluC * a * p, __builtin_fmaf(3.f * kGeluA, a2, 1.f), t);
        }
        return a * t;
    } else {
        if constexpr (SLOPE) d = a > 0.f ? 1.f : 0.f;
        return a <= 0.f ? 0.f : a;                   // (a NaN stays)
    }
}

// Calls f(constant) for a run-time activation (the same throughout a launch).
template <class F>
__device__ __forceinline__ void with_act(int act, F f) {
    using std::integral_constant;
    switch (act) {
        case ACT_SILU: return f(integral_constant<int, ACT_SILU>{});
        case ACT_GELU: return f(integral_constant<int, ACT_GELU>{});
        case ACT_GELU_TANH: return f(integral_constant<int, ACT_GELU_TANH>{});
        case ACT_RELU: return f(integral_constant<int, ACT_RELU>{});
        default: return f(integral_constant<int, ACT_SIGMOID>{});
    }
}

// h = act(g)*u of four elements.
__device__ __forceinline__ rowf4 gate4(int act, const rowf4& g, const rowf4& u) {
    rowf4 h;
    with_act(act, [&](auto a) {
        float d;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = act_at<a(), false>(g[e], d) * u[e];
    });
    return h;
}

// dh·u·d of a slope d, |d| < 1.2.  Where dh·u overflows the larger of them meets d first: the
// whole may fit, or be zero (a relu's), and does not get lost on the way either.
__device__ __forceinline__ float gate_slope(float dh, float u, float d) {
    const float t = dh * u;
    if (__builtin_expect(__builtin_isinf(t), 0)) {
        const bool up = __builtin_fabsf(u) >= __builtin_fabsf(dh);
        return (up ? u : dh) * d * (up ? dh : u);
    }
    return t * d;
}

// Projections g, u, and the gradient dh at act(g)*u, to the gradients at them.
__device__ __forceinline__ void gate_slopes(int act, float dh, float& g, float& u) {
    with_act(act, [&](auto a) {
        float d;
        const float v = act_at<a(), true>(g, d);
        g = gate_slope(dh, u, d);
        u = dh * v;
    });
}
__device__ __forceinline__ void gate_slopes(int act, const rowf4& dh, rowf4& g, rowf4& u) {
    with_act(act, [&](auto a) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float d;
            const float v = act_at<a(), true>(g[e], d);
            g[e] = gate_slope(dh[e], u[e], d);
            u[e] = dh[e] * v;
        }
    });
}

struct GateParams {
    RowView gu;                       // [M][2F], the gates first
    RowView dh;                       // backward
    RowView out;                      // h [M][F], or the gradients [M][2F] (gu itself, if need be)
    int64_t M;
    int F, act;
};

// VEC: elements of a row are neighbours in every operand: a thread takes four of them, the
// last of a row one by one.
template <bool VEC, bool BACK>
__global__ void __launch_bounds__(256) gate_rows(GateParams p) {
    const int per = VEC ? (p.F + 3) / 4 : p.F;
    const int64_t total = p.M * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / per;
        const int f = (int)(i - m * per) * (VEC ? 4 : 1);
        constexpr int MODE = VEC ? R_TAIL : R_STRIDED;
        // (the up columns as rows of their own, so that a row's end is theirs)
        const RowView up{p.gu.p + (int64_t)p.F * p.gu.cs, p.gu.rs, p.gu.cs};
        const auto g = row_load<MODE>(p.gu, m, f, p.F), u = row_load<MODE>(up, m, f, p.F);
        if constexpr (!BACK) {
            auto h = g;
            with_act(p.act, [&](auto a) {
                float d;
                if constexpr (VEC) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) h[e] = act_at<a(), false>(g[e], d) * u[e];
                } else {
                    h = act_at<a(), false>(g, d) * u;
                }
            });
            row_store<MODE>(p.out, m, f, p.F, h);
        } else {
            const auto dh = row_load<MODE>(p.dh, m, f, p.F);
            auto dg = g, du = u;
            gate_slopes(p.act, dh, dg, du);
            const RowView dup{p.out.p + (int64_t)p.F * p.out.cs, p.out.rs, p.out.cs};
            row_store<MODE>(p.out, m, f, p.F, dg);
            row_store<MODE>(dup, m, f, p.F, du);
        }
    }
}

// The gradients as gate_rows gives them, and their sums over the rows (a bias's gradient) from
// the same pass.  A workgroup owns a strip of features -- 64 lanes of four, or one -- and a run
// of rows, which its four waves take in turn; the runs' sums go to `part` [runs][2F], or, of one
// run, to the bias gradient.  A wave adds up eight rows in fp32 and those sums in fp64, for a run
// has as many rows as it takes (in fp32 throughout 3e-6 of a sum of 70000 rows of one sign was
// lost).  (4096 x 2 x 4096, with the runs' sums together: 67 us, 55 without sums; 509 x 2 x 2570:
// 10.7, 5.7.  Every row in fp64: 69 and 10.8.  Strips four times as wide: 71, and 24.)
struct GateBias {
    float* db;
    int64_t stride;
    float beta;                       // 0: what was there is not read
};
__device__ __forceinline__ void bias_put(const GateBias& b, int64_t c, double sum) {
    float* const d = b.db + c * b.stride;
    *d = (float)(b.beta == 0.f ? sum : sum + (double)b.beta * *d);
}
template <bool VEC>
__global__ void __launch_bounds__(256) gate_rows_sums(GateParams p, GateBias b, float* part, int run) {
    constexpr int E = VEC ? 4 : 1, STRIP = 64 * E, MODE = VEC ? R_TAIL : R_STRIDED;
    __shared__ float red[2][4][STRIP];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int f0 = blockIdx.x * STRIP, f = f0 + lane * E;
    const int64_t first = (int64_t)blockIdx.y * run, end = min(first + run, p.M);
    const RowView up{p.gu.p + (int64_t)p.F * p.gu.cs, p.gu.rs, p.gu.cs};
    const RowView dup{p.out.p + (int64_t)p.F * p.out.cs, p.out.rs, p.out.cs};
    using V = std::conditional_t<VEC, rowf4, float>;
    double sg[E] = {}, su[E] = {};
    auto add = [](double (&s)[E], const V& x) {
        if constexpr (VEC) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += (double)x[e];
        } else {
            s[0] += (double)x;
        }
    };
    for (int64_t b0 = first; b0 < end && f < p.F; b0 += 32) {
        const int64_t b1 = min(b0 + 32, end);
        V pg{}, pu{};
#pragma unroll 2
        for (int64_t m = b0 + wave; m < b1; m += 4) {
            V g = row_load<MODE>(p.gu, m, f, p.F), u = row_load<MODE>(up, m, f, p.F);
            const V dh = row_load<MODE>(p.dh, m, f, p.F);
            gate_slopes(p.act, dh, g, u);
            row_store<MODE>(p.out, m, f, p.F, g);
            row_store<MODE>(dup, m, f, p.F, u);
            pg += g;
            pu += u;
        }
        add(sg, pg);
        add(su, pu);
    }
    auto put = [&](float* d, const double (&x)[E]) {
        V v;
        if constexpr (VEC) v = rowf4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
        else v = (float)x[0];
        *reinterpret_cast<V*>(d) = v;
    };
    put(&red[0][wave][lane * E], sg);
    put(&red[1][wave][lane * E], su);
    __syncthreads();
    for (int i = t; i < 2 * STRIP; i += 256) {
        const int h = i / STRIP, c = i % STRIP;
        if (f0 + c >= p.F) continue;
        double s = red[h][0][c];
#pragma unroll
        for (int w = 1; w < 4; ++w) s += red[h][w][c];
        const int64_t col = (int64_t)h * p.F + f0 + c;
        if (gridDim.y == 1) bias_put(b, col, s);
        else part[blockIdx.y * 2 * (int64_t)p.F + col] = (float)s;
    }
}
// The runs' sums together, in fp64: 64 columns a workgroup, whose waves take the runs in turn.
template <int W = 8>
__global__ void __launch_bounds__(64 * W) gate_bias_sum(const float* part, int runs, int64_t cols, GateBias b) {
    __shared__ double red[W][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    double s = 0;
    if (c < cols) {
#pragma unroll 8
        for (int r = wave; r < runs; r += W) s += part[r * cols + c];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave > 0 || c >= cols) return;
    s = red[0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s += red[w][lane];
    bias_put(b, c, s);
}

}  // namespace mtk
