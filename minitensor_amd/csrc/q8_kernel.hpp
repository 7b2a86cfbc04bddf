// q8_kernel.hpp -- products of 8-bit rows and 8-bit weights (include/mtlowbit.h,
// include/mtffn.h): S[m][n] = sum_k q[m][k] wq[n][k] on the integer matrix unit, whole
// numbers throughout, y = S·s[m]·ws[n] + bias[n], and the gated form
// h[m][f] = act(y[m][f]) * y[m][F + f].
//
// S is exact while a sum has fewer than 2^17 terms (|q|, |wq| <= 128), which k_per_split
// sees to; the splits' sums are added up in 64 bits.  So the result does not depend on the
// tile or the splits: one rounding to fp32, and one for each factor.
//
// Gated: a tile of BN columns has BN/2 features, in blocks of 32 gate columns and the same
// features' 32 up columns, so that a wave's two neighbouring blocks meet in its epilogue.
#pragma once

#include "gate_kernel.hpp"
#include "gemm_split.hpp"
#include "tile_helpers.hpp"

namespace mtk {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef u32x4 u32x4_u __attribute__((aligned(1)));

struct Q8Params {
    const int8_t* x;                  // rows: bytes between them, a scale each
    int64_t x_m;
    const float* xs;
    const int8_t* w;                  // output channels, the same; gated: [2F], the gates first
    int64_t w_n;
    const float* ws;
    const float* bias;                // nullptr: none
    int64_t bias_stride;
    RowView y;                        // y [M][N], gated h [M][F]
    RowView gu;                       // gated: y [M][2F] too (nullptr: not wanted)
    int32_t* part;                    // [splits][M][part_n] sums, where splits > 1
    int64_t part_n;                   // whole tiles of columns
    int M, N, K;                      // N: columns of y, gated F
    int splits, k_per_split;          // a multiple of 128, below 2^17
    int act;
};

// The weight's row of column c (of a launch's, gated ones in pairs of blocks).
template <bool GATED>
__device__ __forceinline__ int64_t q8_channel(const Q8Params& p, int c) {
    if constexpr (!GATED) return min(c, p.N - 1);
    const int f = min((c >> 6) * 32 + (c & 31), p.N - 1);
    return (c & 32) ? (int64_t)p.N + f : f;
}

// Four sums of neighbouring columns n.. of row m (gated: and of their up columns) to y.
__device__ __forceinline__ rowf4 q8_scaled(const Q8Params& p, float s, int64_t n, int64_t last,
                                           const rowf4& sum) {
    rowf4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t c = min(n + e, last);
        v[e] = sum[e] * (s * p.ws[c]);
        if (p.bias) v[e] += p.bias[c * p.bias_stride];
    }
    return v;
}
__device__ __forceinline__ void q8_put4(const RowView& v, int64_t m, int64_t n, int64_t end,
                                        const rowf4& x) {
    float* const d = v.p + m * v.rs + n * v.cs;
    if (v.cs == 1 && n + 4 <= end) {
        *reinterpret_cast<rowf4_u*>(d) = x;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < end) d[e * v.cs] = x[e];
    }
}
template <bool GATED>
__device__ __forceinline__ void q8_finish4(const Q8Params& p, int m, int n, const rowf4& a,
                                           const rowf4& b) {
    const float s = p.xs[m];
    if constexpr (!GATED) {
        q8_put4(p.y, m, n, p.N, q8_scaled(p, s, n, p.N - 1, a));
    } else {
        const rowf4 g = q8_scaled(p, s, n, p.N - 1, a);
        const rowf4 u = q8_scaled(p, s, (int64_t)p.N + n, 2 * (int64_t)p.N - 1, b);
        if (p.gu.p) {
            q8_put4(p.gu, m, n, p.N, g);
            q8_put4(p.gu, m, (int64_t)p.N + n, 2 * (int64_t)p.N, u);
        }
        q8_put4(p.y, m, n, p.N, gate4(p.act, g, u));
    }
}

// Sixteen bytes of a row from k on, zero from `end` on.
__device__ __forceinline__ u32x4 q8_bytes(const int8_t* row, int k, int end) {
    if (k + 16 <= end) return *reinterpret_cast<const u32x4_u*>(row + k);
    u32x4 r = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + 4 * d + e < end) r[d] |= (uint32_t)(uint8_t)row[k + 4 * d + e] << (8 * e);
    return r;
}

// Tiles of BM x BN over chunks of BK bytes of k, in S LDS buffers.  A buffer holds the
// tile's rows, then its columns, BK bytes each; a row's 16-byte units change places by its
// number, so that the 16 rows that a fragment read takes at a time lie on different banks.
// DMA: the units go straight from memory to LDS, 1 KB a wave instruction, S-1 chunks ahead
// (rows on multiples of 16 bytes); otherwise through registers, a chunk ahead, from any
// address.  A chunk that the range of k ends in goes through registers with its bounds
// checked.
template <int BM, int BN, int WM, int BK, int S, bool DMA, bool GATED>
__global__ void __launch_bounds__(BM / WM * (BN / 64) * 64) q8_gemm(Q8Params p) {
    constexpr int WN = 64, WAVES_N = BN / WN, NW = BM / WM * WAVES_N, NT = 64 * NW;
    constexpr int MB = WM / 32, NB = 2;
    constexpr int UNITS = BK / 16, ROWS = BM + BN;
    constexpr int BUF = ROWS * BK;
    constexpr int NI = ROWS * UNITS / NT;              // units of a thread, a chunk
    static_assert(NI * NT == ROWS * UNITS && BM * UNITS % 64 == 0, "whole instructions");
    static_assert(BK == 64 || BK == 128, "four or eight units a row");
    static_assert(S * BUF >= NW * 32 * 64 * 4, "the epilogue's staging");
    __shared__ __attribute__((aligned(1024))) char smem[S * BUF];
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5, lrow = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int ra = wave / WAVES_N * WM, rb = wave % WAVES_N * WN;
    const int cols = GATED ? (p.N + 31) / 32 * 64 : p.N;
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (cols + BN - 1) / BN;
    const int split = blockIdx.x / (tiles_m * tiles_n);
    int im, in;
    lb_tile(blockIdx.x - split * tiles_m * tiles_n, tiles_m, tiles_n, im, in);
    const int m0 = im * BM, n0 = in * BN;
    const int kb = split * p.k_per_split, ke = min(p.K, kb + p.k_per_split);

    // unit i of this thread: row and place of i*NT + t, holding the row's unit there
    auto swz = [](int row) { return BK == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
    const int8_t* src[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int e = i * NT + t, r = e / UNITS, unit = (e % UNITS) ^ swz(r);
        src[i] = (r < BM ? p.x + min(m0 + r, p.M - 1) * p.x_m
                         : p.w + q8_channel<GATED>(p, n0 + r - BM) * p.w_n) +
                 kb + 16 * unit;
    }
    auto dma = [&](int slot, int c) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            __builtin_amdgcn_global_load_lds(
                (const void __attribute__((address_space(1)))*)(src[i] + (int64_t)c * BK),
                (void __attribute__((address_space(3)))*)(smem + slot * BUF + (i * NT + wave * 64) * 16),
                16, 0, 0);
    };
    u32x4 raw[DMA ? 1 : NI];
    auto load = [&](int c) {
        if constexpr (!DMA)
#pragma unroll
            for (int i = 0; i < NI; ++i)
                raw[i] = *reinterpret_cast<const u32x4_u*>(src[i] + (int64_t)c * BK);
    };
    auto put = [&](int slot) {
        if constexpr (!DMA)
#pragma unroll
            for (int i = 0; i < NI; ++i)
                *reinterpret_cast<u32x4*>(smem + slot * BUF + (i * NT + t) * 16) = raw[i];
    };
    auto put_checked = [&](int slot, int c) {
#pragma unroll 1
        for (int e = t; e < ROWS * UNITS; e += NT) {
            const int r = e / UNITS, unit = (e % UNITS) ^ swz(r);
            const int8_t* const row = r < BM ? p.x + min(m0 + r, p.M - 1) * p.x_m
                                             : p.w + q8_channel<GATED>(p, n0 + r - BM) * p.w_n;
            *reinterpret_cast<u32x4*>(smem + slot * BUF + e * 16) =
                q8_bytes(row, kb + c * BK + 16 * unit, ke);
        }
    };

    i32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int sw = swz(lrow);
    auto multiply = [&](int slot) {
        const char* const buf = smem + slot * BUF;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            const int unit = ((2 * kk + half) ^ sw) * 16;
            i32x4 a[MB], b[NB];
#pragma unroll
            for (int i = 0; i < MB; ++i)
                a[i] = *reinterpret_cast<const i32x4*>(buf + (ra + 32 * i + lrow) * BK + unit);
#pragma unroll
            for (int j = 0; j < NB; ++j)
                b[j] = *reinterpret_cast<const i32x4*>(buf + (BM + rb + 32 * j + lrow) * BK + unit);
            // (the transposed block: a lane has four neighbouring columns of a row)
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[j], a[i], acc[i][j], 0, 0, 0);
        }
    };

    const int whole = (ke - kb) / BK, part_k = (ke - kb) % BK;
    if (part_k) {                                      // first, in the last buffer
        put_checked(S - 1, whole);
        lb_barrier();
        multiply(S - 1);
    }
    if constexpr (DMA) {
        // buffers 0 .. S-2 first: the last is being read until the loop's first barrier
        for (int c = 0; c < S - 1; ++c)
            if (c < whole) dma(c, c);
        for (int c = 0; c < whole; ++c) {
            // this wave's part of chunk c is in LDS, then everyone's
            if (c + S - 1 <= whole)
                __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(NI * (S - 2)));
            else
                __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));
            __builtin_amdgcn_s_barrier();
            if (c + S - 1 < whole) dma((c + S - 1) % S, c + S - 1);
            multiply(c % S);
        }
    } else {
        static_assert(DMA || S == 2, "two buffers");
        if (whole > 0) {
            load(0);
            put(0);
        }
        for (int c = 0; c < whole; ++c) {
            lb_barrier();
            if (c + 1 < whole) load(c + 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(c & 1);
            if (c + 1 < whole) put((c + 1) & 1);
        }
    }

    // Each wave turns its block rows round in a part of LDS of its own: 16 lanes then write
    // a row's 64 columns (gated: eight lanes its 32 features).
    __syncthreads();
    i32x4* const stage = reinterpret_cast<i32x4*>(smem) + wave * 32 * 16;
    const bool part = p.splits > 1;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                stage[lrow * 16 + ((8 * j + 2 * q + half) ^ (lrow & 15))] =
                    i32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                          acc[i][j][4 * q + 3]};
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        constexpr int GROUPS = GATED ? 8 : 16;
        const int g = lane % GROUPS;
        if (part) {
#pragma unroll 1
            for (int r = lane >> 4; r < 32; r += 4) {
                const int m = m0 + ra + 32 * i + r;
                if (m < p.M)
                    *reinterpret_cast<i32x4*>(p.part + ((int64_t)split * p.M + m) * p.part_n + n0 +
                                              rb + 4 * (lane & 15)) =
                        stage[r * 16 + ((lane & 15) ^ (r & 15))];
            }
        } else {
            const int n = (GATED ? (n0 + rb) / 2 : n0 + rb) + 4 * g;
#pragma unroll 1
            for (int r = lane / GROUPS; r < 32; r += 64 / GROUPS) {
                const int m = m0 + ra + 32 * i + r;
                if (m >= p.M || n >= p.N) continue;
                const i32x4 a = stage[r * 16 + (g ^ (r & 15))];
                i32x4 b = a;
                if constexpr (GATED) b = stage[r * 16 + ((g + 8) ^ (r & 15))];
                q8_finish4<GATED>(p, m, n, __builtin_convertvector(a, rowf4),
                                  __builtin_convertvector(b, rowf4));
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// The splits' sums together, and to y: a thread takes four columns (features).
template <bool GATED>
__global__ void __launch_bounds__(256) q8_sum(Q8Params p) {
    const int per = (p.N + 3) / 4;
    const int64_t total = (int64_t)p.M * per, step = (int64_t)p.M * p.part_n;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * 256) {
        const int m = (int)(i / per), n = (int)(i - (int64_t)m * per) * 4;
        const int c = GATED ? (n >> 5) * 64 + (n & 31) : n;
        auto sum = [&](int col) {
            const int32_t* const q = p.part + (int64_t)m * p.part_n + col;
            int64_t s[4] = {0, 0, 0, 0};
#pragma unroll 4
            for (int k = 0; k < p.splits; ++k) {
                const i32x4 v = *reinterpret_cast<const i32x4*>(q + k * step);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += v[e];
            }
            return rowf4{(float)s[0], (float)s[1], (float)s[2], (float)s[3]};
        };
        const rowf4 a = sum(c);
        q8_finish4<GATED>(p, m, n, a, GATED ? sum(c + 32) : a);
    }
}

// Few rows, bound by the weight's bytes.  A workgroup owns NC blocks of 16 columns (gated:
// NC/2 of gates and the same features' up columns) and all of K; its waves take chunks of
// 256 inputs in turn, straight from memory to the operands of 16x16x64 products (lane l: row
// or column l % 16, 16 bytes from 16·(l/16) on), and their sums meet in LDS.
// MB: blocks of 16 rows.
template <int MB, int NC, bool GATED>
__global__ void __launch_bounds__(512) q8_few(Q8Params p) {
    constexpr int W = 8, C = 16 * NC;
    static_assert(!GATED || NC % 2 == 0, "gates and up columns");
    __shared__ int red[W][16 * MB][C];
    const int t = threadIdx.x, lane = t & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // features of a workgroup: half its columns where they are gated
    const int n0 = blockIdx.x * (GATED ? C / 2 : C);
    const int8_t* wr[NC];
#pragma unroll
    for (int q = 0; q < NC; ++q) {                    // (past the end: the last, not stored)
        const int f = min(n0 + 16 * (GATED ? q % (NC / 2) : q) + col, p.N - 1);
        wr[q] = p.w + (GATED && q >= NC / 2 ? (int64_t)p.N + f : (int64_t)f) * p.w_n + 16 * j;
    }
    const int8_t* xr[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) xr[b] = p.x + (int64_t)min(16 * b + col, p.M - 1) * p.x_m + 16 * j;
    i32x4 acc[MB][NC];
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int q = 0; q < NC; ++q) acc[b][q] = i32x4{0, 0, 0, 0};
    const int whole = p.K >> 8;
    for (int c = wave; c < whole; c += W) {
        i32x4 x[4][MB], w[4][NC];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = 256 * c + 64 * i;
#pragma unroll
            for (int q = 0; q < NC; ++q)
                w[i][q] = __builtin_bit_cast(i32x4, *reinterpret_cast<const u32x4_u*>(wr[q] + k));
#pragma unroll
            for (int b = 0; b < MB; ++b)
                x[i][b] = __builtin_bit_cast(i32x4, *reinterpret_cast<const u32x4_u*>(xr[b] + k));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int q = 0; q < NC; ++q)
                    acc[b][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[i][b], w[i][q], acc[b][q], 0, 0, 0);
    }
    if (whole % W == wave) {                          // the rest of K, 64 inputs at a time
#pragma unroll 1
        for (int k = 256 * whole; k < p.K; k += 64) {
            i32x4 x[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b)
                x[b] = __builtin_bit_cast(i32x4, q8_bytes(xr[b] - 16 * j, k + 16 * j, p.K));
#pragma unroll
            for (int q = 0; q < NC; ++q) {
                const i32x4 w = __builtin_bit_cast(i32x4, q8_bytes(wr[q] - 16 * j, k + 16 * j, p.K));
#pragma unroll
                for (int b = 0; b < MB; ++b)
                    acc[b][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[b], w, acc[b][q], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int q = 0; q < NC; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[wave][16 * b + 4 * j + r][16 * q + col] = acc[b][q][r];
    __syncthreads();
    constexpr int F = GATED ? C / 2 : C;
    for (int e = t; e < p.M * F; e += 64 * W) {
        const int m = e / F, c = e % F, n = n0 + c;
        if (n >= p.N) continue;
        auto value = [&](int at, int64_t ch) {
            int64_t s = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) s += red[w][m][at];
            float v = (float)s * (p.xs[m] * p.ws[ch]);
            if (p.bias) v += p.bias[ch * p.bias_stride];
            return v;
        };
        const float g = value(c, n);
        if constexpr (!GATED) {
            p.y.p[m * p.y.rs + n * p.y.cs] = g;
        } else {
            const float u = value(F + c, (int64_t)p.N + n);
            if (p.gu.p) {
                p.gu.p[m * p.gu.rs + n * p.gu.cs] = g;
                p.gu.p[m * p.gu.rs + ((int64_t)p.N + n) * p.gu.cs] = u;
            }
            float h = 0.f;
            with_act(p.act, [&](auto a) {
                float d;
                h = act_at<a(), false>(g, d) * u;
            });
            p.y.p[m * p.y.rs + n * p.y.cs] = h;
        }
    }
}

}  // namespace mtk
