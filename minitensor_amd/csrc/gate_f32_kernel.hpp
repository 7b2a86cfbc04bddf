// gate_f32_kernel.hpp -- a gated block's projections in fp32 beside the tiles of gemm_f32_sp
// (GateOut, gemm_kernel.hpp): few rows on the vector units, few rows and small products on the
// fp32 matrix units, and the sum of a split product.
#pragma once

#include "gate_kernel.hpp"

namespace mtk {

struct GateGemv {
    const float* x;                   // neighbouring inputs, rows x_m apart
    int64_t x_m;
    const float* w;                   // [2F], the gates first, neighbouring inputs
    int64_t w_n;
    const float* bias;                // nullptr: none
    int64_t bias_stride;
    RowView h, gu;                    // gu.p nullptr: not wanted
    int M, F, K, act;
};

// h and the projections of row m, feature f.
__device__ __forceinline__ void gate_put(const GateGemv& p, int m, int f, float g, float u) {
    if (p.bias) {
        g += p.bias[(int64_t)f * p.bias_stride];
        u += p.bias[((int64_t)p.F + f) * p.bias_stride];
    }
    if (p.gu.p) {
        p.gu.p[m * p.gu.rs + f * p.gu.cs] = g;
        p.gu.p[m * p.gu.rs + ((int64_t)p.F + f) * p.gu.cs] = u;
    }
    float h = 0.f;
    with_act(p.act, [&](auto a) {
        float d;
        h = act_at<a(), false>(g, d) * u;
    });
    p.h.p[m * p.h.rs + f * p.h.cs] = h;
}

// The sum over a wave of each of v[0..V): after it lane l holds that of v[l / (64/V)].  Half
// of the values change lanes in each step while there are two or more: V + 5 - log2 V
// exchanges in place of 6 V.
template <int V, int O = 32>
__device__ __forceinline__ float wave_sums(const float (&v)[V], int lane) {
    if constexpr (V > 1) {
        const bool up = lane & O;
        float x[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            x[i] = (up ? v[i + V / 2] : v[i]) + __shfl_xor(up ? v[i] : v[i + V / 2], O);
        return wave_sums<V / 2, O / 2>(x, lane);
    } else {
        float s = v[0];
#pragma unroll
        for (int o = O; o >= 1; o >>= 1) s += __shfl_xor(s, o);
        return s;
    }
}

// Few rows (M <= MR), bound by the weight's bytes.  A workgroup of eight waves owns NF
// features; the waves take runs of 256 inputs in turn, a lane four neighbouring ones of each
// of the 2·NF weight rows and of x, and their sums meet in LDS in wave order.  (One row 2048 ->
// 2 x 4096, 67 MB of weight: 9.6 us where it is in the 256 MB cache, 7 TB/s.)
template <int MR, int NF>
__global__ void __launch_bounds__(512) gate_gemv(GateGemv p) {
    constexpr int W = 8, V = 2 * NF * MR;
    static_assert((V & (V - 1)) == 0 && V <= 64, "values of a lane change places by halves");
    __shared__ float red[W][V];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int f0 = blockIdx.x * NF;
    const float* w[2 * NF];
    const float* x[MR];
#pragma unroll
    for (int j = 0; j < 2 * NF; ++j) {                // (past the end: the last, not stored)
        const int f = min(f0 + j % NF, p.F - 1);
        w[j] = p.w + (j >= NF ? (int64_t)p.F + f : (int64_t)f) * p.w_n + 4 * lane;
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) x[m] = p.x + min(m, p.M - 1) * p.x_m + 4 * lane;
    float sum[V];                                     // [row][feature]
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    auto add = [&](const rowf4 (&a)[MR], const rowf4 (&b)[2 * NF]) {
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int j = 0; j < 2 * NF; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sum[m * 2 * NF + j] = __builtin_fmaf(a[m][e], b[j][e], sum[m * 2 * NF + j]);
    };
    const int whole = p.K >> 8;
#pragma unroll 2
    for (int c = wave; c < whole; c += W) {
        rowf4 a[MR], b[2 * NF];
#pragma unroll
        for (int j = 0; j < 2 * NF; ++j) b[j] = *reinterpret_cast<const rowf4_u*>(w[j] + 256 * c);
#pragma unroll
        for (int m = 0; m < MR; ++m) a[m] = *reinterpret_cast<const rowf4_u*>(x[m] + 256 * c);
        add(a, b);
    }
    if (whole % W == wave && 256 * whole + 4 * lane < p.K) {
        const int n = p.K - 256 * whole - 4 * lane;   // inputs of this lane's last four
        auto some = [&](const float* q) {
            rowf4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) v[e] = q[256 * whole + e];
            return v;
        };
        rowf4 a[MR], b[2 * NF];
#pragma unroll
        for (int j = 0; j < 2 * NF; ++j) b[j] = some(w[j]);
#pragma unroll
        for (int m = 0; m < MR; ++m) a[m] = some(x[m]);
        add(a, b);
    }
    const float s = wave_sums<V>(sum, lane);
    if (lane % (64 / V) == 0) red[wave][lane / (64 / V)] = s;
    __syncthreads();
    for (int i = t; i < MR * NF; i += 512) {
        const int m = i / NF, f = f0 + i % NF;
        if (m >= p.M || f >= p.F) continue;
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            g += red[k][m * 2 * NF + i % NF];
            u += red[k][m * 2 * NF + NF + i % NF];
        }
        gate_put(p, m, f, g, u);
    }
}

// Few or small: fp32 products of 16x16x4 straight from memory.  A workgroup of eight waves
// owns 16·MB rows and 16 features' gate and up rows; the waves take runs
// of 64 inputs in turn.  Lane l of a product holds row (of x or of the weight) l % 16 and one
// input; it loads four neighbouring ones, of 16 that the four lanes of a row hold, and takes
// them in turn, x and weight alike.  (16 rows 2048 -> 2 x 4096: 13 us, 5 TB/s of weight; 64 rows
// 64 -> 2 x 32: 2.7 us, in tiles, whose chunks come one after another, 6.6; 512 rows 512 -> 2 x
// 512 10.9 us, 49 of the fp32 units' 157 TFLOP/s: each row of x is read again for every 16
// features and each feature for every 32 rows, 67 MB of operands in 512 workgroups, two a CU in
// turn, for 3 MB of them.)
template <int MB>
__global__ void __launch_bounds__(512) gate_few(GateGemv p) {
    constexpr int W = 8, U = 4;                       // products of 16 inputs in flight
    __shared__ float red[W][16 * MB][32];
    const int t = threadIdx.x, lane = t & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int f0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MB;
    const float* w[2];
    const float* x[MB];
#pragma unroll
    for (int q = 0; q < 2; ++q)                       // (past the end: the last, not stored)
        w[q] = p.w + ((int64_t)q * p.F + min(f0 + col, p.F - 1)) * p.w_n + 4 * j;
#pragma unroll
    for (int b = 0; b < MB; ++b) x[b] = p.x + min(m0 + 16 * b + col, p.M - 1) * p.x_m + 4 * j;
    typedef float acc4 __attribute__((ext_vector_type(4)));
    acc4 acc[MB][2];
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int q = 0; q < 2; ++q) acc[b][q] = acc4{0.f, 0.f, 0.f, 0.f};
    auto add = [&](const rowf4 (&a)[MB], const rowf4 (&b)[2]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    acc[m][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m][e], b[q][e], acc[m][q], 0, 0, 0);
    };
    const int whole = p.K >> 6;
#pragma unroll 1
    for (int c = wave; c < whole; c += W) {
        rowf4 a[U][MB], b[U][2];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int k = 64 * c + 16 * i;
#pragma unroll
            for (int q = 0; q < 2; ++q) b[i][q] = *reinterpret_cast<const rowf4_u*>(w[q] + k);
#pragma unroll
            for (int m = 0; m < MB; ++m) a[i][m] = *reinterpret_cast<const rowf4_u*>(x[m] + k);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) add(a[i], b[i]);
    }
    // the rest, 16 inputs a wave
    const int k = 64 * whole + 16 * wave;
    if (wave < 4 && k < p.K) {
        const int n = p.K - k - 4 * j;                // inputs of this lane's four
        auto some = [&](const float* q) {
            rowf4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) v[e] = q[k + e];
            return v;
        };
        rowf4 a[MB], b[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) b[q] = some(w[q]);
#pragma unroll
        for (int m = 0; m < MB; ++m) a[m] = some(x[m]);
        add(a, b);
    }
    // (lane l, register r of a product: row 4·(l/16) + r, column l % 16)
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[wave][16 * m + 4 * j + r][16 * q + col] = acc[m][q][r];
    __syncthreads();
    const int rows = min(16 * MB, p.M - m0);
    for (int i = t; i < rows * 16; i += 512) {
        const int m = i >> 4, c = i & 15, f = f0 + c;
        if (f >= p.F) continue;
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int v = 0; v < W; ++v) {
            g += red[v][m][c];
            u += red[v][m][16 + c];
        }
        gate_put(p, m0 + m, f, g, u);
    }
}

// The splits' partials [splits][M][N] (32 gates and their 32 up columns in turn) together in
// order, and on: a thread takes four features.
struct GateSum {
    const float* part;
    int64_t N;
    int splits;
    const float* bias;
    int64_t bias_stride;
    RowView h, gu;
    int M, F, act;
};
template <int = 0>
__global__ void __launch_bounds__(256) gate_sum(GateSum p) {
    const int per = (p.F + 3) / 4;
    const int64_t total = (int64_t)p.M * per, step = (int64_t)p.M * p.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int m = (int)(i / per), f = (int)(i - (int64_t)m * per) * 4;
        const float* const q = p.part + m * p.N + (f >> 5) * 64 + (f & 31);
        rowf4 g = {0.f, 0.f, 0.f, 0.f}, u = g;
#pragma unroll 4
        for (int k = 0; k < p.splits; ++k) {
            g += *reinterpret_cast<const rowf4_u*>(q + k * step);
            u += *reinterpret_cast<const rowf4_u*>(q + k * step + 32);
        }
        if (p.bias)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t c = min(f + e, p.F - 1);
                g[e] += p.bias[c * p.bias_stride];
                u[e] += p.bias[(p.F + c) * p.bias_stride];
            }
        if (p.gu.p) {
            put4(p.gu, m, f, p.F, g);
            put4(p.gu, m, (int64_t)p.F + f, 2 * (int64_t)p.F, u);
        }
        put4(p.h, m, f, p.F, gate4(p.act, g, u));
    }
}

}  // namespace mtk
