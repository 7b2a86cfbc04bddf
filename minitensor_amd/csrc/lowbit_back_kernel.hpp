// lowbit_back_kernel.hpp -- a Linear layer's weight gradient from an input kept
// in 8 bits: dW[o][c] = sum_r (dY[r][o]·scale[r]) q[r][c].
//
// The row's scale goes to dY (one fp32 rounding), and q is exact in bf16: three
// bf16 products on the matrix units in fp32's precision, as lowbit_q4_kernel.hpp,
// where a product of two fp32 operands takes six.  The sums of 128 rows are
// taken on the matrix unit from zero and added up in fp32: the unit does not
// round to nearest, and over 10^5 rows that would show.
#pragma once

#include "lowbit_q4_kernel.hpp"

namespace mtk {

struct BackParams {
    const float* dy;                  // [R][O] at any strides
    int64_t dy_r, dy_o;
    const int8_t* q;                  // [R][C]
    int64_t q_r;
    const float* scale;               // [R]
    float* dw;                        // [O][C]
    int64_t dw_o, dw_c;
    float beta;
    float* part;                      // [splits][O][C] where splits > 1
    int R, O, C;
    int splits, r_per_split;          // a multiple of 128
    int q_vec;                        // q's rows are 4-byte aligned
};

// Tiles of BM outputs x BN inputs.  Both operands lie across k (= r): a thread
// takes eight rows of one output (loads of consecutive outputs on consecutive
// lanes), and four rows of four inputs, which change places in registers.  The
// entries of four neighbouring inputs lie in four runs, so that consecutive
// lanes write consecutive entries; the runs start 32 bytes apart modulo 128, so
// that a fragment's rows fall on different banks.
template <int BN>
constexpr int back_run() { return BN / 4 + 2; }
template <int BN>
constexpr int back_group() { return 4 * back_run<BN>() * 16; }

template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64, 2) back_dw(BackParams p) {
    constexpr int WAVES_N = BN / WN, NT = BM / WM * WAVES_N * 64;
    constexpr int MB = WM / 32, NB = WN / 32;
    constexpr int NA = BM * 4 / NT, NQ = (BN * 2 + NT - 1) / NT;
    static_assert(NA * NT == BM * 4, "whole items per thread");
    constexpr int APL = lb_plane<BM>(), BUF = 3 * APL + 4 * back_group<BN>();
    __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int ra = wave / WAVES_N * WM, rb = wave % WAVES_N * WN;
    const int tiles_m = (p.O + BM - 1) / BM, tiles_n = (p.C + BN - 1) / BN;
    const int split = blockIdx.x / (tiles_m * tiles_n);
    int im, in;
    lb_tile(blockIdx.x - split * tiles_m * tiles_n, tiles_m, tiles_n, im, in);
    const int m0 = im * BM, n0 = in * BN;
    const int rbeg = split * p.r_per_split, rend = min(p.R, rbeg + p.r_per_split);
    const int nk = (rend - rbeg + 31) >> 5;

    struct Items {
        float a[NA][8];
        uint32_t q[NQ][4];            // four inputs of each of four rows
    };
    auto load = [&](Items& x, int r0) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int v = i * NT + t, o = min(m0 + v % BM, p.O - 1);
            const int r = r0 + 8 * __builtin_amdgcn_readfirstlane(v / BM);
#pragma unroll
            for (int e = 0; e < 8; ++e)                    // (r is the same in a wave)
                x.a[i][e] = r + e < p.R ? p.dy[(int64_t)(r + e) * p.dy_r + (int64_t)o * p.dy_o] *
                                              p.scale[r + e]
                                        : 0.f;
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int v = i * NT + t, c = n0 + v % (BN / 4) * 4, r = r0 + 4 * (v / (BN / 4));
            if (NQ * NT > BN * 2 && v >= BN * 2) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x.q[i][e] = 0;
                if (r + e >= p.R) continue;
                const int8_t* const src = p.q + (int64_t)(r + e) * p.q_r + c;
                if (p.q_vec && c + 4 <= p.C) {
                    x.q[i][e] = *reinterpret_cast<const uint32_t*>(src);
                } else {
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (c + b < p.C) x.q[i][e] |= (uint32_t)(uint8_t)src[b] << (8 * b);
                }
            }
        }
    };
    auto store = [&](const Items& x, char* buf) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int v = i * NT + t;
            const float* const a = x.a[i];
            u32x4 h, m, l;
            cut8(rowf4{a[0], a[1], a[2], a[3]}, rowf4{a[4], a[5], a[6], a[7]}, h, m, l);
            char* const d = buf + v / BM * lb_group<BM>() + v % BM * 16;
            *reinterpret_cast<u32x4*>(d) = h;
            *reinterpret_cast<u32x4*>(d + APL) = m;
            *reinterpret_cast<u32x4*>(d + 2 * APL) = l;
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int v = i * NT + t, c4 = v % (BN / 4), kq = v / (BN / 4);
            if (NQ * NT > BN * 2 && v >= BN * 2) continue;
            char* const d = buf + 3 * APL + (kq >> 1) * back_group<BN>() + c4 * 16 + (kq & 1) * 8;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(x.q[i][e] >> (8 * b));
                u32x2 w;
                w[0] = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302);
                w[1] = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302);
                *reinterpret_cast<u32x2*>(d + b * back_run<BN>() * 16) = w;
            }
        }
    };

    f32x16 sum[MB][NB], acc[MB][NB];
    zero_blocks<MB, NB>(sum);
    zero_blocks<MB, NB>(acc);
    const int half = lane >> 5, row = lane & 31;
    auto multiply = [&](const char* buf) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 a[3][MB], b[NB];
#pragma unroll
            for (int jn = 0; jn < NB; ++jn) {
                const int c = rb + 32 * jn + row;
                b[jn] = *reinterpret_cast<const u32x4*>(buf + 3 * APL + (2 * s + half) * back_group<BN>() +
                                                        ((c & 3) * back_run<BN>() + (c >> 2)) * 16);
            }
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int i = 0; i < MB; ++i)
                    a[q][i] = *reinterpret_cast<const u32x4*>(
                        buf + q * APL + (2 * s + half) * lb_group<BM>() + (ra + 32 * i + row) * 16);
#pragma unroll
            for (int q = 2; q >= 0; --q)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int jn = 0; jn < NB; ++jn)
                        acc[i][jn] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            __builtin_bit_cast(bf16x8, a[q][i]), __builtin_bit_cast(bf16x8, b[jn]),
                            acc[i][jn], 0, 0, 0);
        }
    };
    Items x;
    load(x, rbeg);
    store(x, smem);
    for (int c = 0; c < nk; ++c) {
        __syncthreads();
        const bool more = c + 1 < nk;
        if (more) load(x, rbeg + 32 * (c + 1));
        multiply(smem + (c & 1) * BUF);
        if (more) store(x, smem + ((c + 1) & 1) * BUF);
        if ((c & 3) == 3 || !more) {
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int jn = 0; jn < NB; ++jn)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        sum[i][jn][r] += acc[i][jn][r];
                        acc[i][jn][r] = 0.f;
                    }
        }
    }
    const bool part = p.splits > 1;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int jn = 0; jn < NB; ++jn) {
            const int n = n0 + rb + 32 * jn + (lane & 31);
            if (n >= p.C) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + ra + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (m >= p.O) continue;
                const float v = sum[i][jn][r];
                if (part) {
                    p.part[((int64_t)split * p.O + m) * p.C + n] = v;
                } else {
                    float* const d = p.dw + (int64_t)m * p.dw_o + (int64_t)n * p.dw_c;
                    *d = p.beta != 0.f ? p.beta * *d + v : v;
                }
            }
        }
}

}  // namespace mtk
