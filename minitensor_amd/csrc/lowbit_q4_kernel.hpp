// lowbit_q4_kernel.hpp -- products with 4-bit weights and group scales
// (include/mtlowbit.h): y[m][n] = bias[n] + sum_g s[n][g] sum_{k in g} x[m][k] c[n][k].
//
// A 4-bit code is exact in bf16, and an fp32 x is the sum of three bf16 values
// h + m + l (gemm_split.hpp): the product is three bf16 products on the matrix
// units, each exact, with fp32's precision (six for two fp32 operands); an
// 8-bit x is exact in bf16 by itself, one product, and its sums within a group
// are whole numbers below 2^24, exact too.  The sums of a group are taken on
// the matrix unit from zero and added to the fp32 result with one fused
// multiply-add by the group's scale.
//
// q4_few: few rows of x, bound by the weight's bytes.  q4_gemm: the rest.
#pragma once

#include "gemm_split.hpp"
#include "lowbit_rows_kernel.hpp"

namespace mtk {

struct Q4Params {
    const float* x;                   // fp32 x: strides of rows and inputs
    int64_t x_m, x_k;
    const int8_t* q;                  // or 8-bit rows with a scale each
    int64_t q_m;
    const float* q_scale;
    const uint8_t* w;                 // packed codes
    int64_t w_n;                      // bytes
    const float* s;                   // group scales
    int64_t s_n;
    const float* bias;                // nullptr: none
    int64_t bias_stride;
    float* y;
    int64_t y_m, y_n;
    float* part;                      // [splits][M][N] partial sums, where splits > 1
    int M, N, K;
    int splits, k_per_split;          // a multiple of 128
    int x_vec;                        // rows of x are 16-byte aligned (8-bit ones 8-byte) runs
};

// The eight codes of a dword, over 16, as bf16 (exact): v_cvt_off_f32_i4 gives
// a code over 16, whose low half as fp32 is zero.  19 instructions.
__device__ __forceinline__ u32x4 q4_unpack(uint32_t w) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4(w >> (8 * i)));
        const uint32_t b = __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4(w >> (8 * i + 4)));
        r[i] = __builtin_amdgcn_perm(b, a, 0x07060302);
    }
    return r;
}
constexpr float kQ4Unit = 16.f;

// The parts of eight values.  What is left of an infinity or a NaN (a NaN) is
// made zero, so that its products are those of fp32: the middle of (r, r, 0)
// is r, and 0 where r is a NaN.
__device__ __forceinline__ void cut8(const rowf4& a, const rowf4& b, u32x4& h, u32x4& m, u32x4& l) {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = bf16_pair(x[2 * i], x[2 * i + 1]);
        float r0 = x[2 * i] - bf16_lo(h[i]), r1 = x[2 * i + 1] - bf16_hi(h[i]);
        r0 = __builtin_amdgcn_fmed3f(r0, r0, 0.f);
        r1 = __builtin_amdgcn_fmed3f(r1, r1, 0.f);
        m[i] = bf16_pair(r0, r1);
        l[i] = bf16_pair(r0 - bf16_lo(m[i]), r1 - bf16_hi(m[i]));
    }
}

// Eight int8 values as bf16.
__device__ __forceinline__ u32x4 q8_bf16(uint32_t lo, uint32_t hi) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? lo : hi;
        const float a = (float)(int8_t)(w >> (16 * (i & 1)));
        const float b = (float)(int8_t)(w >> (16 * (i & 1) + 8));
        r[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
    }
    return r;
}

// Eight consecutive inputs k..k+7 of row m, zero from K on.
__device__ __forceinline__ void q4_x8(const Q4Params& p, int m, int k, rowf4& a, rowf4& b) {
    const float* const src = p.x + (int64_t)m * p.x_m + (int64_t)k * p.x_k;
    if (p.x_vec && k + 8 <= p.K) {
        a = *reinterpret_cast<const rowf4*>(src);
        b = *reinterpret_cast<const rowf4*>(src + 4);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a[e] = k + e < p.K ? src[e * p.x_k] : 0.f;
        b[e] = k + 4 + e < p.K ? src[(4 + e) * p.x_k] : 0.f;
    }
}
__device__ __forceinline__ void q4_q8(const Q4Params& p, int m, int k, uint32_t& lo, uint32_t& hi) {
    const int8_t* const src = p.q + (int64_t)m * p.q_m + k;
    if (p.x_vec && k + 8 <= p.K) {
        const uint2 v = *reinterpret_cast<const uint2*>(src);
        lo = v.x;
        hi = v.y;
        return;
    }
    lo = hi = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        lo |= (k + e < p.K ? (uint32_t)(uint8_t)src[e] : 0u) << (8 * e);
        hi |= (k + 4 + e < p.K ? (uint32_t)(uint8_t)src[4 + e] : 0u) << (8 * e);
    }
}

__device__ __forceinline__ f32x4 mfma_16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Few rows.  A workgroup owns 16 columns n and all of K, in blocks of 128: wave
// w takes the blocks w, w + W, ...; the waves' sums meet in LDS in wave order.
// The parts of x are rows of their own (row 3m + part; row m for 8-bit x): one
// MFMA of 16x16x32 covers five rows of fp32 x.  Each wave stages its block of x in an LDS region
// of its own, so that nothing waits for another wave until the end.
//
// Lane (n = lane % 16, j = lane / 16) reads its weights as they lie: with
// groups of 128 the 16 bytes of k = 32j..32j+31 (four MFMAs), with smaller ones
// 8 or 4 bytes of each group, so that the 32 inputs of an MFMA are of one group.
template <int MB, int G, bool Q8, int W>
__global__ void __launch_bounds__(64 * W) q4_few(Q4Params p) {
    constexpr int P = Q8 ? 1 : 3;
    constexpr int LW = G / 32;                        // dwords per load, MFMAs per group
    constexpr int NL = 4 / LW;                        // loads (groups) per block
    constexpr int RS = 256 + 16;                      // bytes of a row of a staged block
    constexpr int XB = 16 * MB * RS;
    constexpr int RED = W * 16 * MB * 16 * 4;
    __shared__ __attribute__((aligned(16))) char smem[W * XB > RED ? W * XB : RED];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int col = lane & 15, j = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int n = min(n0 + col, p.N - 1);             // (columns past N are not stored)
    const uint8_t* const wr = p.w + (int64_t)n * p.w_n;
    const float* const sr = p.s + (int64_t)n * p.s_n;
    const int kp = (p.K + 31) & ~31;                  // inputs that the packed row holds
    const int groups = (p.K + G - 1) / G;
    const int blocks = (p.K + 127) >> 7;
    char* const xs = smem + wave * XB;

    f32x4 sum[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) sum[b] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int kb = wave; kb < blocks; kb += W) {
        const int k0 = kb * 128;
        uint32_t cw[4];
        float sc[NL];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int k = k0 + G * i + 8 * LW * j;    // of the load's first dword
            const uint32_t* const src = reinterpret_cast<const uint32_t*>(wr + (k >> 1));
#pragma unroll
            for (int d = 0; d < LW; ++d) cw[LW * i + d] = 0;
            if (k < kp) {
                if constexpr (LW == 4) {
                    const u32x4 v = *reinterpret_cast<const u32x4*>(src);
#pragma unroll
                    for (int d = 0; d < 4; ++d) cw[d] = v[d];
                } else if constexpr (LW == 2) {
                    const u32x2 v = *reinterpret_cast<const u32x2*>(src);
                    cw[2 * i] = v[0];
                    cw[2 * i + 1] = v[1];
                } else {
                    cw[i] = *src;
                }
            }
            const int g = kb * NL + i;
            sc[i] = g < groups ? sr[g] * kQ4Unit : 0.f;
        }
        // the block of x: 16 pieces of eight inputs per row
        for (int e = lane; e < p.M * 16; e += 64) {
            const int m = e >> 4, piece = e & 15;
            char* const d = xs + P * m * RS + piece * 16;
            if constexpr (Q8) {
                uint32_t lo, hi;
                q4_q8(p, m, k0 + 8 * piece, lo, hi);
                *reinterpret_cast<u32x4*>(d) = q8_bf16(lo, hi);
            } else {
                rowf4 a, b;
                u32x4 h, mm, l;
                q4_x8(p, m, k0 + 8 * piece, a, b);
                cut8(a, b, h, mm, l);
                *reinterpret_cast<u32x4*>(d) = h;
                *reinterpret_cast<u32x4*>(d + RS) = mm;
                *reinterpret_cast<u32x4*>(d + 2 * RS) = l;
            }
        }
        // (the wave's own region: its LDS accesses are in order)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        f32x4 acc[MB];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
#pragma unroll
            for (int d = 0; d < LW; ++d) {
                const u32x4 b = q4_unpack(cw[LW * i + d]);
                const int piece = (G * i + 8 * LW * j + 8 * d) >> 3;
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) {
                    // (rows past the last one hold what they hold: their sums are not used)
                    const u32x4 a = *reinterpret_cast<const u32x4*>(xs + (16 * mb + col) * RS +
                                                                    piece * 16);
                    acc[mb] = mfma_16(a, b, d == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[mb]);
                }
            }
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) sum[mb] += acc[mb] * sc[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    __syncthreads();
    // [wave][row][column]
    float* const red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            red[(wave * 16 * MB + 16 * mb + 4 * j + r) * 16 + col] = sum[mb][r];
    __syncthreads();
    for (int e = t; e < p.M * 16; e += 64 * W) {
        const int m = e >> 4, c = e & 15;
        if (n0 + c >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int q = P - 1; q >= 0; --q) v += red[(w * 16 * MB + P * m + q) * 16 + c];
        if constexpr (Q8) v *= p.q_scale[m];
        if (p.bias) v += p.bias[(int64_t)(n0 + c) * p.bias_stride];
        p.y[(int64_t)m * p.y_m + (int64_t)(n0 + c) * p.y_n] = v;
    }
}

// LDS of a chunk of 32 k: per part four groups of eight k, each a column of
// 16-byte entries, one per row, and two entries more (the groups of a row then
// start 32 bytes apart modulo the banks' 128).
template <int ROWS>
constexpr int lb_group() { return (ROWS + 2) * 16; }
template <int ROWS>
constexpr int lb_plane() { return 4 * lb_group<ROWS>(); }

// One chunk of 32 k for a wave's MB x NB blocks of 32x32: P parts of A times B,
// the small parts first.
template <int P, int MB, int NB, int BM, int BN>
__device__ __forceinline__ void lb_multiply(const char* lds, int ra, int rb, int lane,
                                            f32x16 (&acc)[MB][NB]) {
    const int half = lane >> 5, row = lane & 31;
    const char* const lb = lds + P * lb_plane<BM>();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        u32x4 a[P][MB], b[NB];
#pragma unroll
        for (int jn = 0; jn < NB; ++jn)
            b[jn] = *reinterpret_cast<const u32x4*>(lb + (2 * s + half) * lb_group<BN>() +
                                                    (rb + 32 * jn + row) * 16);
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
            for (int i = 0; i < MB; ++i)
                a[q][i] = *reinterpret_cast<const u32x4*>(lds + q * lb_plane<BM>() +
                                                          (2 * s + half) * lb_group<BM>() +
                                                          (ra + 32 * i + row) * 16);
#pragma unroll
        for (int q = P - 1; q >= 0; --q)
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int jn = 0; jn < NB; ++jn)
                    acc[i][jn] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        __builtin_bit_cast(bf16x8, a[q][i]), __builtin_bit_cast(bf16x8, b[jn]),
                        acc[i][jn], 0, 0, 0);
    }
}

// The tile of a workgroup: eight XCDs take consecutive workgroups in turn; each
// gets a run of tiles, walked down eight rows of tiles at a time, so that the
// tiles in flight on one L2 share their operands.
__device__ __forceinline__ void lb_tile(int b, int tm, int tn, int& im, int& in) {
    const int n = tm * tn;
    const int xcd = b & 7, q = n >> 3, rem = n & 7;
    b = xcd * q + min(xcd, rem) + (b >> 3);
    const int band = 8 * tn, first = b / band * 8, h = min(8, tm - first);
    const int w = b % band;
    im = first + w % h;
    in = w / h;
}

// Many rows: tiles of BM x BN, waves of 64x64 (or 32x64).
template <int BM, int BN, int WM, int WN, int G, bool Q8>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64, 2) q4_gemm(Q4Params p) {
    constexpr int P = Q8 ? 1 : 3;
    constexpr int WAVES_N = BN / WN, NT = BM / WM * WAVES_N * 64;
    constexpr int MB = WM / 32, NB = WN / 32;
    constexpr int NA = BM * 4 / NT, NBI = BN * 4 / NT;     // items of eight k per thread
    static_assert(NA * NT == BM * 4 && NBI * NT == BN * 4, "whole items per thread");
    constexpr int BUF = P * lb_plane<BM>() + lb_plane<BN>();
    __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int ra = wave / WAVES_N * WM, rb = wave % WAVES_N * WN;
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    const int split = blockIdx.x / (tiles_m * tiles_n);
    int im, in;
    lb_tile(blockIdx.x - split * tiles_m * tiles_n, tiles_m, tiles_n, im, in);
    const int m0 = im * BM, n0 = in * BN;
    const int kb = split * p.k_per_split, ke = min(p.K, kb + p.k_per_split);
    const int nk = (ke - kb + 31) >> 5;
    const int kp = (p.K + 31) & ~31;

    // (rows past M or N: the last row's values, not stored)
    struct Items {
        rowf4 a[Q8 ? 1 : NA][2];
        uint32_t q[Q8 ? NA : 1][2];
        uint32_t w[NBI];
    };
    auto load = [&](Items& x, int k0) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int v = i * NT + t, m = min(m0 + (v >> 2), p.M - 1), k = k0 + 8 * (v & 3);
            if constexpr (Q8) q4_q8(p, m, k, x.q[i][0], x.q[i][1]);
            else q4_x8(p, m, k, x.a[i][0], x.a[i][1]);
        }
#pragma unroll
        for (int i = 0; i < NBI; ++i) {
            const int v = i * NT + t, n = min(n0 + (v >> 2), p.N - 1), k = k0 + 8 * (v & 3);
            x.w[i] = k < kp ? *reinterpret_cast<const uint32_t*>(p.w + (int64_t)n * p.w_n + (k >> 1))
                            : 0u;
        }
    };
    auto store = [&](const Items& x, char* buf) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int v = i * NT + t;
            char* const d = buf + (v & 3) * lb_group<BM>() + (v >> 2) * 16;
            if constexpr (Q8) {
                *reinterpret_cast<u32x4*>(d) = q8_bf16(x.q[i][0], x.q[i][1]);
            } else {
                u32x4 h, m, l;
                cut8(x.a[i][0], x.a[i][1], h, m, l);
                *reinterpret_cast<u32x4*>(d) = h;
                *reinterpret_cast<u32x4*>(d + lb_plane<BM>()) = m;
                *reinterpret_cast<u32x4*>(d + 2 * lb_plane<BM>()) = l;
            }
        }
#pragma unroll
        for (int i = 0; i < NBI; ++i) {
            const int v = i * NT + t;
            *reinterpret_cast<u32x4*>(buf + P * lb_plane<BM>() + (v & 3) * lb_group<BN>() +
                                      (v >> 2) * 16) = q4_unpack(x.w[i]);
        }
    };

    f32x16 sum[MB][NB], acc[MB][NB];
    zero_blocks<MB, NB>(sum);
    zero_blocks<MB, NB>(acc);
    constexpr int GC = G / 32;                             // chunks per group
    const float* sr[NB];
#pragma unroll
    for (int jn = 0; jn < NB; ++jn)
        sr[jn] = p.s + (int64_t)min(n0 + rb + 32 * jn + (lane & 31), p.N - 1) * p.s_n;
    Items x;
    load(x, kb);
    store(x, smem);
    for (int c = 0; c < nk; ++c) {
        __syncthreads();
        const bool more = c + 1 < nk;
        if (more) load(x, kb + 32 * (c + 1));
        lb_multiply<P, MB, NB, BM, BN>(smem + (c & 1) * BUF, ra, rb, lane, acc);
        if (more) store(x, smem + ((c + 1) & 1) * BUF);
        if ((c + 1) % GC == 0 || !more) {
            const int g = (kb + 32 * c) / G;
#pragma unroll
            for (int jn = 0; jn < NB; ++jn) {
                const float s = sr[jn][g] * kQ4Unit;
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        sum[i][jn][r] = __builtin_fmaf(acc[i][jn][r], s, sum[i][jn][r]);
                        acc[i][jn][r] = 0.f;
                    }
            }
        }
    }
    // block element r of a lane: row 8*(r/4) + 4*(lane/32) + r%4, column lane%32
    const bool part = p.splits > 1;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int jn = 0; jn < NB; ++jn) {
            const int n = n0 + rb + 32 * jn + (lane & 31);
            if (n >= p.N) continue;
            const float b = !part && p.bias ? p.bias[(int64_t)n * p.bias_stride] : 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + ra + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (m >= p.M) continue;
                float v = sum[i][jn][r];
                if constexpr (Q8) v *= p.q_scale[m];
                if (part) p.part[((int64_t)split * p.M + m) * p.N + n] = v;
                else p.y[(int64_t)m * p.y_m + (int64_t)n * p.y_n] = v + b;
            }
        }
}

// y[m][n] = beta*y + bias[n] + the splits' partials [splits][M][N] in order (no
// splits: part is not read).
__global__ void __launch_bounds__(256)
lb_sum(const float* part, int splits, int M, int N, const float* bias, int64_t bias_stride, float* y,
       int64_t y_m, int64_t y_n, float beta) {
    const int64_t n = (int64_t)M * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int m = (int)(i / N), c = (int)(i - (int64_t)m * N);
        float v = 0.f;
        for (int s = 0; s < splits; ++s) v += part[s * n + i];
        if (bias) v += bias[(int64_t)c * bias_stride];
        float* const d = y + (int64_t)m * y_m + (int64_t)c * y_n;
        *d = beta != 0.f ? beta * *d + v : v;
    }
}

// Codes and scales of a weight: a thread takes eight inputs (a dword of codes),
// G/8 neighbouring threads a group.
template <int G>
__global__ void __launch_bounds__(256)
quantize_q4(const float* w, int64_t w_n, int64_t w_k, uint8_t* out, int64_t o_n, float* s,
            int64_t s_n, int N, int K) {
    constexpr int T = G / 8;
    const int kp = (K + 31) & ~31, groups = (K + G - 1) / G;
    const int64_t per = (int64_t)groups * T, total = per * N;
    for (int64_t i0 = (int64_t)blockIdx.x * 256; i0 < total; i0 += (int64_t)gridDim.x * 256) {
        const int64_t i = i0 + threadIdx.x;
        const bool live = i < total;                       // (whole groups)
        const int64_t n = live ? i / per : 0;
        const int k0 = live ? (int)(i - n * per) * 8 : 0;
        float v[8];
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = live && k0 + e < K ? w[n * w_n + (int64_t)(k0 + e) * w_k] : 0.f;
            m = max(m, magnitude(v[e]));
        }
#pragma unroll
        for (int o = T / 2; o >= 1; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
        float sc = __uint_as_float(m) * (1.f / 7.f);
        sc = sc < kScaleMin ? kScaleMin : sc;
        const float inv = 1.f / sc;
        uint32_t b = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) b |= ((uint32_t)q8_code(v[e], inv) & 15u) << (4 * e);
        if (!live) continue;
        if (k0 < kp) *reinterpret_cast<uint32_t*>(out + n * o_n + (k0 >> 1)) = b;
        if (k0 % G == 0) s[n * s_n + k0 / G] = sc;
    }
}

__global__ void __launch_bounds__(256)
dequantize_q4(const uint8_t* w, int64_t w_n, const float* s, int64_t s_n, int group, float* y,
              int64_t y_n, int64_t y_k, int N, int K) {
    const int64_t per = (K + 7) / 8, total = per * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * 256) {
        const int64_t n = i / per;
        const int k0 = (int)(i - n * per) * 8;
        const uint32_t b = *reinterpret_cast<const uint32_t*>(w + n * w_n + (k0 >> 1));
        const float sc = s[n * s_n + k0 / group];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k0 + e < K)
                y[n * y_n + (int64_t)(k0 + e) * y_k] =
                    (float)((int32_t)(b << (28 - 4 * e)) >> 28) * sc;
    }
}

}  // namespace mtk
