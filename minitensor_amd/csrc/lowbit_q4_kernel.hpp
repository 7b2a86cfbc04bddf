// lowbit_q4_kernel.hpp -- products with 4-bit weights and group scales
// (include/mtlowbit.h): y[m][n] = bias[n] + sum_g s[n][g] sum_{k in g} x[m][k] c[n][k].
//
// A 4-bit code is exact in bf16, and an fp32 x is the sum of three bf16 values
// h + m + l (lowbit_gemm.hpp): the product is three bf16 products on the matrix
// units, each exact, with fp32's precision (six for two fp32 operands); an
// 8-bit x takes one product, whose sums within a group are whole numbers below
// 2^24, exact too.  The sums of a group are taken on the matrix unit from zero
// and added to the fp32 result with one fused multiply-add by the group's
// scale.
//
// q4_few: few rows of x, bound by the weight's bytes.  The rest: q4_gemm, fp32
// rows, and q4_gemm_q8, 8-bit ones.
#pragma once

#include "lowbit_gemm.hpp"

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
};

// The eight codes of a dword, over 16, as bf16 (exact): v_cvt_off_f32_i4 gives
// a code over 16, whose low half as fp32 is zero.  13 instructions.  The factor comes back at
// a sum's end: times 16 a group's scale may leave fp32's range.
__device__ __forceinline__ u32x4 q4_unpack(uint32_t w) {
    const uint32_t odd = w >> 4;
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = bf16_cut(__builtin_amdgcn_cvt_off_f32_i4((w >> (8 * i)) & 0xff),
                          __builtin_amdgcn_cvt_off_f32_i4((odd >> (8 * i)) & 0xff));
    return r;
}
constexpr float kQ4Unit = 16.f;

typedef u32x2 u32x2_u __attribute__((aligned(1)));

// Eight consecutive inputs k..k+7 of row m, zero from K on.
__device__ __forceinline__ void q4_x8(const Q4Params& p, const float* row, int k, float (&x)[8]) {
    if (p.x_k == 1 && k + 8 <= p.K) {
        const rowf4 a = *reinterpret_cast<const rowf4_u*>(row + k);
        const rowf4 b = *reinterpret_cast<const rowf4_u*>(row + k + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = a[e];
            x[4 + e] = b[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = k + e < p.K ? row[(k + e) * p.x_k] : 0.f;
    }
}
__device__ __forceinline__ u32x2 q4_x8(const Q4Params& p, const int8_t* row, int k) {
    if (k + 8 <= p.K) return *reinterpret_cast<const u32x2_u*>(row + k);
    u32x2 r = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < p.K) r[e >> 2] |= (uint32_t)(uint8_t)row[k + e] << (8 * (e & 3));
    return r;
}

__device__ __forceinline__ f32x4 mfma_16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Few rows.  A workgroup owns NC blocks of 16 columns n and all of K, in blocks of 128, of
// which each wave takes up to four neighbouring ones at a time; the waves' sums meet in LDS
// in wave order.  The parts of x are rows of their own (row 3m + part; row m for 8-bit x), so
// that one MFMA of 16x16x32 covers five rows of fp32 x.  Each wave stages U blocks of x at a
// time in an LDS region of its own, so that nothing waits for another wave until the end.
// CAP: rows that a block there has room for; the MFMAs' rows past it are its last one again,
// their sums not used.
//
// NC = 1: the loads of all four blocks are in flight at once (one row, 4096 -> 4096: 6.7 us
// block by block, 5.5 so).  NC > 1: a block of all NC at a time, the next one on its way; x
// is cut once for 16·NC columns, which is what many rows cost most.
//
// Lane (n = lane % 16, j = lane / 16) reads 16 bytes of a block's 64, and the 32 inputs of an
// MFMA have to be of one group: with smaller groups than 128 the four lanes of a column
// exchange dwords (loads of 4 bytes, each lane's in place, took 34 us where these take 16).
template <int G>
struct Q4Lanes {
    static constexpr int LW = G / 32, NL = 4 / LW;    // dwords per group and lane, groups
    // dword i·LW + d of lane j: piece (of eight inputs) of the block
    __device__ __forceinline__ static int piece(int i, int d, int j) {
        return G == 128 ? 4 * j + d : G == 64 ? 8 * i + 4 * (j & 1) + 2 * (j >> 1) + d : 4 * i + j;
    }
    // from dword 4j + r in register r of lane j
    __device__ __forceinline__ static void exchange(uint32_t (&w)[4]) {
        if constexpr (G < 128) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const auto x = __builtin_amdgcn_permlane32_swap(w[r], w[r + 2], false, false);
                w[r] = x[0];
                w[r + 2] = x[1];
            }
        }
        if constexpr (G < 64) {
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const auto x = __builtin_amdgcn_permlane16_swap(w[r], w[r + 1], false, false);
                w[r] = x[0];
                w[r + 1] = x[1];
            }
        }
    }
};

template <int CAP, int U, int NC, int G, bool Q8, int W>
__global__ void __launch_bounds__(64 * W, CAP <= 4 && G > 32 ? 8 : 2) q4_few(Q4Params p) {
    using Lanes = Q4Lanes<G>;
    constexpr int P = Q8 ? 1 : 3, MB = (CAP + 15) / 16;
    constexpr int LW = Lanes::LW, NL = Lanes::NL;
    constexpr int RS = 256 + 16;                      // bytes of a row of a staged block
    constexpr int XB = U * CAP * RS;
    constexpr int RED = W * 16 * MB * 16 * NC * 4;
    constexpr int AHEAD = NC == 1 ? 4 : 2;            // blocks of weights in registers
    static_assert(NC == 1 || U == 1, "several columns go block by block");
    __shared__ __attribute__((aligned(16))) char smem[W * XB > RED ? W * XB : RED];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int col = lane & 15, j = lane >> 4;
    const int n0 = blockIdx.x * (16 * NC);
    const uint8_t* wr[NC];
    const float* sr[NC];
#pragma unroll
    for (int q = 0; q < NC; ++q) {                    // (columns past N: the last, not stored)
        const int64_t n = min(n0 + 16 * q + col, p.N - 1);
        wr[q] = p.w + n * p.w_n;
        sr[q] = p.s + n * p.s_n;
    }
    const int kp = (p.K + 31) & ~31;                  // inputs that the packed row holds
    const int groups = (p.K + G - 1) / G;
    const int blocks = (p.K + 127) >> 7;
    const int per = min(4, (blocks + W - 1) / W);     // a wave's neighbouring blocks
    char* const xs = smem + wave * XB;

    f32x4 sum[NC][MB];
#pragma unroll
    for (int q = 0; q < NC; ++q)
#pragma unroll
        for (int b = 0; b < MB; ++b) sum[q][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Pieces of eight inputs of x: 16 per row and block.  A lane takes the pieces lane, lane +
    // 64, ... of U blocks, MAXP of them at most.
    constexpr int MAXP = (CAP / P * 16 * U + 63) / 64;
    using Piece = std::conditional_t<Q8, u32x2, float[8]>;
    typedef float Scales __attribute__((ext_vector_type(NL), aligned(4)));
    for (int kb0 = wave * per; kb0 < blocks; kb0 += per * W) {
        const int end = min(kb0 + per, blocks);
        Piece x[MAXP];
        auto load_x = [&](int kb) {                   // U blocks from kb on (zeros past K)
#pragma unroll
            for (int i = 0; i < MAXP; ++i) {
                const int e = lane + 64 * i, m = e / (16 * U);
                if (m >= p.M) break;
                const int k = 128 * (kb + (e >> 4) % U) + 8 * (e & 15);
                if constexpr (Q8) x[i] = q4_x8(p, p.q + (int64_t)m * p.q_m, k);
                else q4_x8(p, p.x + (int64_t)m * p.x_m, k, x[i]);
            }
        };
        uint32_t cw[AHEAD][NC][4];
        float sc[AHEAD][NC][NL];
        auto load_w = [&](int kb, uint32_t (&w)[NC][4], float (&s)[NC][NL]) {
#pragma unroll
            for (int q = 0; q < NC; ++q) {
                const int k = 128 * kb + 32 * j;
                u32x4 v = {0u, 0u, 0u, 0u};
                if (k < kp) v = *reinterpret_cast<const u32x4*>(wr[q] + (k >> 1));
#pragma unroll
                for (int d = 0; d < 4; ++d) w[q][d] = v[d];
                const int g = kb * NL;
                if (g + NL <= groups) {
                    const Scales f = *reinterpret_cast<const Scales*>(sr[q] + g);
#pragma unroll
                    for (int i = 0; i < NL; ++i) s[q][i] = f[i];
                } else {
#pragma unroll
                    for (int i = 0; i < NL; ++i) s[q][i] = g + i < groups ? sr[q][g + i] : 0.f;
                }
            }
        };
        load_x(kb0);
#pragma unroll
        for (int u = 0; u < (NC == 1 ? 4 : 1); ++u)
            if (u == 0 || kb0 + u < end) load_w(kb0 + u, cw[u], sc[u]);
#pragma unroll
        for (int h = 0; h < 4; h += U) {
            if (kb0 + h >= end) break;                // (uniform)
#pragma unroll
            for (int i = 0; i < MAXP; ++i) {
                const int e = lane + 64 * i, m = e / (16 * U);
                if (m >= p.M) break;
                char* const d = xs + ((e >> 4) % U * CAP + P * m) * RS + (e & 15) * 16;
                if constexpr (Q8) {
                    *reinterpret_cast<u32x4*>(d) = q8_bf16(x[i]);
                } else {
                    u32x4 hi, mi, lo;
                    cut8<false>(x[i], hi, mi, lo);
                    *reinterpret_cast<u32x4*>(d) = hi;
                    *reinterpret_cast<u32x4*>(d + RS) = mi;
                    *reinterpret_cast<u32x4*>(d + 2 * RS) = lo;
                }
            }
            if (kb0 + h + U < end) {
                load_x(kb0 + h + U);
                if constexpr (NC > 1) load_w(kb0 + h + 1, cw[(h + 1) & 1], sc[(h + 1) & 1]);
            }
            // (the wave's own region: its LDS accesses are in order)
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u > 0 && kb0 + h + u >= end) break;
                auto& w = cw[NC == 1 ? h + u : h & 1];
                auto& s = sc[NC == 1 ? h + u : h & 1];
#pragma unroll
                for (int q = 0; q < NC; ++q) Lanes::exchange(w[q]);
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    f32x4 acc[NC][MB];
#pragma unroll
                    for (int d = 0; d < LW; ++d) {
                        u32x4 b[NC];
#pragma unroll
                        for (int q = 0; q < NC; ++q) b[q] = q4_unpack(w[q][LW * i + d]);
#pragma unroll
                        for (int mb = 0; mb < MB; ++mb) {
                            const u32x4 a = *reinterpret_cast<const u32x4*>(
                                xs + (u * CAP + min(16 * mb + col, CAP - 1)) * RS +
                                Lanes::piece(i, d, j) * 16);
#pragma unroll
                            for (int q = 0; q < NC; ++q)
                                acc[q][mb] = mfma_16(a, b[q], d == 0 ? f32x4{0.f, 0.f, 0.f, 0.f}
                                                                     : acc[q][mb]);
                        }
                    }
#pragma unroll
                    for (int q = 0; q < NC; ++q)
#pragma unroll
                        for (int mb = 0; mb < MB; ++mb)
                            sum[q][mb] += acc[q][mb] * s[q][i];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }
    __syncthreads();
    // [wave][row][column]
    constexpr int C = 16 * NC;
    float* const red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int q = 0; q < NC; ++q)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                red[(wave * 16 * MB + 16 * mb + 4 * j + r) * C + 16 * q + col] = sum[q][mb][r];
    __syncthreads();
    for (int e = t; e < p.M * C; e += 64 * W) {
        const int m = e / C, c = e % C;
        if (n0 + c >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int q = P - 1; q >= 0; --q) v += red[(w * 16 * MB + P * m + q) * C + c];
        v *= kQ4Unit;
        if constexpr (Q8) v *= p.q_scale[m];
        if (p.bias) v += p.bias[(int64_t)(n0 + c) * p.bias_stride];
        p.y[(int64_t)m * p.y_m + (int64_t)(n0 + c) * p.y_n] = v;
    }
}

// Many rows of fp32: x as A; a thread takes eight inputs of a row.
template <int BM, int NT>
struct Q4X {
    static constexpr int N = BM * 4 / NT, kGroup = lb_group<BM>(), kBytes = lb_plane<BM>();
    static_assert(N * NT == BM * 4, "whole items");
    static constexpr int kWork = N * 56;
    static constexpr bool kLate = false;
    struct Raw {
        float a[N][8];
    };
    const Q4Params& p;
    const float* base;                // row m0
    uint32_t off[N];                  // of the item, in bytes
    int64_t ld;
    int t, last;
    bool fast;                        // a row's inputs are neighbours, the tile within 32 bits of bytes
    __device__ __forceinline__ static int entry(int row) { return row; }
    __device__ __forceinline__ Q4X(const Q4Params& p_, int m0, int t_)
        : p(p_), base(p_.x + m0 * p_.x_m), ld(p_.x_m), t(t_), last(p_.M - 1 - m0),
          fast(p_.x_k == 1 && p_.x_m < (1 << 22)) {
#pragma unroll
        for (int i = 0; i < N; ++i)                        // (rows past M: the last, not stored)
            off[i] = ((uint32_t)min((i * NT + t) >> 2, last) * (uint32_t)ld + 8 * (t & 3)) * 4u;
    }
    __device__ __forceinline__ void load_fast(Raw& r, int k0) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float* const x = at_bytes(base + k0, off[i]);
            const rowf4 a = *reinterpret_cast<const rowf4_u*>(x);
            const rowf4 b = *reinterpret_cast<const rowf4_u*>(x + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r.a[i][e] = a[e];
                r.a[i][4 + e] = b[e];
            }
        }
    }
    __device__ __forceinline__ void load(Raw& r, int k0) const {
        if (fast && k0 + 32 <= p.K) return load_fast(r, k0);
        const int v = anew(t);
#pragma unroll
        for (int i = 0; i < N; ++i)
            q4_x8(p, base + min((i * NT + v) >> 2, last) * ld, k0 + 8 * (v & 3), r.a[i]);
    }
    __device__ __forceinline__ void store(const Raw& r, char* buf, bool) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            char* const d = buf + (t & 3) * kGroup + ((i * NT + t) >> 2) * 16;
            u32x4 h, m, l;
            cut8<(BM > 64)>(r.a[i], h, m, l);
            *reinterpret_cast<u32x4*>(d) = h;
            *reinterpret_cast<u32x4*>(d + kBytes) = m;
            *reinterpret_cast<u32x4*>(d + 2 * kBytes) = l;
        }
    }
};

// The weight as B: a thread converts eight inputs (a dword of codes) of a column per chunk.
// BLOCK: blocks of 128 inputs of a column, 64 bytes, go to LDS as they lie in memory and are
// converted from there: loaded chunk by chunk, each 64 bytes are asked for four times, and
// the lines of a narrow tile, of which a CU holds several, do not stay in L1 meanwhile.
// The 16-byte pieces of a column change places by its number, so that the dwords of 16
// columns fall on different banks.  (The wide tile has no registers left for it.)
template <int BN, int NT, bool BLOCK>
struct Q4W {
    static constexpr int N = BN * 4 / NT, kGroup = lb_group<BN>(), kBytes = lb_plane<BN>();
    static_assert(N * NT == BN * 4, "whole items");
    static constexpr bool kBlock = BLOCK;
    static constexpr int kWork = N * 14, kReads = BLOCK ? N : 0, kRaw = BLOCK ? BN * 64 : 0;
    struct Codes {
        uint32_t w[N];
    };
    struct Block {
        u32x4 w[N];
    };
    using Raw = std::conditional_t<BLOCK, Block, Codes>;
    const uint8_t* base;              // column n0
    uint32_t off[N];                  // of the item's column, in bytes
    int64_t ld;
    int t, last, end;                 // bytes of a row
    bool fast;                        // the tile within 32 bits of bytes
    static constexpr int kStep = NT / 4;   // columns between a thread's items, a multiple of 16
    __device__ __forceinline__ static int entry(int c) { return c; }
    __device__ __forceinline__ static int slot(int c, int piece) {
        return c * 64 + ((piece ^ (c >> 2)) & 3) * 16;
    }
    __device__ __forceinline__ Q4W(const Q4Params& p, int n0, int t_)
        : base(p.w + n0 * p.w_n), ld(p.w_n), t(t_), last(p.N - 1 - n0),
          end(((p.K + 31) & ~31) >> 1), fast(p.w_n < (1 << 23)) {
#pragma unroll
        for (int i = 0; i < N; ++i)                        // (columns past N: the last, not stored)
            off[i] = (uint32_t)min((i * NT + t) >> 2, last) * (uint32_t)ld;
    }
    // The thread's place in a row from input k0 on: a dword of a chunk (whole in a row), or a
    // piece of a block (past the end of the row its last piece again: x is zero there).
    __device__ __forceinline__ int place(int k0) const {
        if constexpr (BLOCK) return min((k0 >> 1) + 16 * (t & 3), end - 16);
        else return (k0 >> 1) + 4 * (t & 3);
    }
    using Item = std::conditional_t<BLOCK, u32x4, uint32_t>;
    __device__ __forceinline__ void load_fast(Raw& r, int k0) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            r.w[i] = *reinterpret_cast<const Item*>(base + (off[i] + (uint32_t)place(k0)));
    }
    __device__ __forceinline__ void load(Raw& r, int k0) const {
        if (fast) return load_fast(r, k0);
        const int v = anew(t);
#pragma unroll
        for (int i = 0; i < N; ++i)
            r.w[i] = *reinterpret_cast<const Item*>(base + min((i * NT + v) >> 2, last) * ld +
                                                    place(k0));
    }
    __device__ __forceinline__ void stage(const Block& r, char* raw) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            *reinterpret_cast<u32x4*>(raw + slot(t >> 2, t & 3) + i * kStep * 64) = r.w[i];
    }
    __device__ __forceinline__ void peek(Codes& x, const char* raw, int s) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            x.w[i] = *reinterpret_cast<const uint32_t*>(
                raw + ((slot(t >> 2, 0) + 4 * (t & 3)) ^ (16 * s)) + i * kStep * 64);
    }
    __device__ __forceinline__ void store(const Codes& x, char* buf) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            *reinterpret_cast<u32x4*>(buf + (t & 3) * kGroup + (t >> 2) * 16 + i * kStep * 16) =
                q4_unpack(x.w[i]);
    }
};

// The scales of a lane's NB columns, NG groups at a time: those that are being summed, and
// the next ones, on their way.
template <int NB, int G, int NG>
struct Q4Scales {
    typedef float Vec __attribute__((ext_vector_type(NG), aligned(4)));
    const float* s0;                  // column n0
    uint32_t off[NB];                 // in bytes (the host limits s_n)
    int groups;
    float cur[NB][NG], next[NB][NG];
    __device__ __forceinline__ Q4Scales(const Q4Params& p, int n0, int col, int k0)
        : s0(p.s + (int64_t)n0 * p.s_n), groups((p.K + G - 1) / G) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
            off[j] = (uint32_t)min(col + 32 * j, p.N - 1 - n0) * (uint32_t)p.s_n * 4u;
        load(cur, k0 / G);
        load(next, k0 / G + NG);
    }
    // Groups g0.. of every column; those past the last are never used.  One load per column,
    // which starts early enough to end with the row.
    __device__ __forceinline__ void load(float (&x)[NB][NG], int g0) const {
        const int g = max(min(g0, groups - NG), 0), late = g0 - g;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const float* const q = at_bytes(s0 + g, off[j]);
            if (NG == 1 || groups >= NG) {
                const Vec v = *reinterpret_cast<const Vec*>(q);
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    x[j][i] = v[i];
#pragma unroll
                    for (int d = 1; i + d < NG; ++d) x[j][i] = late == d ? v[i + d] : x[j][i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < NG; ++i) x[j][i] = q[min(i, groups - 1)];
            }
        }
    }
    __device__ __forceinline__ void advance(int g0) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int i = 0; i < NG; ++i) cur[j][i] = next[j][i];
        load(next, g0);
    }
};

// 2048 rows, 4096 -> 8192, groups of 128: 342 us, the matrix unit's power (three bf16
// products at a library's rate: 325).  (Groups of 32: registers for two workgroups a CU.)
template <int BM, int BN, int WM, int WN, int G>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64, BM > 64 || G == 32 ? 2 : 3)
q4_gemm(Q4Params p) {
    constexpr int P = 3;
    constexpr int WAVES_N = BN / WN, NT = BM / WM * WAVES_N * 64;
    constexpr int MB = WM / 32, NB = WN / 32;
    using LA = Q4X<BM, NT>;
    using LB = Q4W<BN, NT, BN == 128>;
    __shared__ __attribute__((aligned(16))) char smem[2 * (P * LA::kBytes + LB::kBytes) +
                                                         2 * LB::kRaw];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int ra = wave / WAVES_N * WM, rb = wave % WAVES_N * WN;
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    const int split = blockIdx.x / (tiles_m * tiles_n);
    int im, in;
    lb_tile(blockIdx.x - split * tiles_m * tiles_n, tiles_m, tiles_n, im, in);
    const int m0 = im * BM, n0 = in * BN;
    const int kb = split * p.k_per_split, ke = min(p.K, kb + p.k_per_split);
    LA la(p, m0, t);
    LB lb(p, n0, t);
    f32x16 sum[MB][NB], acc[MB][NB];
    zero_blocks<MB, NB>(sum);
    // (one load for all groups of 128 inputs where there are registers for them)
    constexpr int GB = 128 / G, NG = BN == 128 ? GB : 1;
    Q4Scales<NB, G, NG> sc(p, n0, rb + (lane & 31), kb);
    lb_product<P, G / 32, BM == 64 ? 4 : 2, MB, NB>(
        la, lb, smem, kb, ke, ra, rb, lane, acc, [&](auto i, int block) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const float s = sc.cur[j][i % NG];
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sum[m][j][r] = __builtin_fmaf(acc[m][j][r], s, sum[m][j][r]);
            // here, and not four groups' together at the end of the loop, as the compiler
            // had it: their sums do not fit the registers
            if constexpr (G < 128)
#pragma unroll
                for (int m = 0; m < MB; ++m) asm volatile("" : "+v"(sum[m][j]));
        }
        if constexpr (i % NG == NG - 1) sc.advance(kb / G + block * GB + i + 1 + NG);
    });
    const bool part = p.splits > 1;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int n = n0 + rb + 32 * j + (lane & 31);
            if (n >= p.N) continue;
            const float b = !part && p.bias ? p.bias[(int64_t)n * p.bias_stride] : 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + ra + 32 * i + lb_row(lane, r);
                if (m >= p.M) continue;
                const float v = sum[i][j][r] * kQ4Unit;
                if (part) p.part[((int64_t)split * p.M + m) * p.N + n] = v;
                else p.y[(int64_t)m * p.y_m + (int64_t)n * p.y_n] = v + b;
            }
        }
}

// Many 8-bit rows: both operands in int8 on the integer matrix unit, at twice bf16's rate and
// half its bytes in LDS; the sums of a group are whole numbers below 2^21.  A code goes in as
// 16 times itself, the high half of a byte: two masks and a shift for the eight of a dword,
// four even inputs and four odd ones, in which order x is put to LDS too.  The codes stay
// packed there, and each wave unpacks the columns that it multiplies.
//
// Chunks of 64 k in two LDS buffers, as lb_product, and two on their way.  What bounds it is
// the vector unit, which turns each sum into fp32 and adds it, in groups of 32 three
// instructions of four (1536 rows, 4096 -> 4096: 91% of its cycles), so four workgroups of
// the narrow tile share a CU.  2048 rows, 4096 -> 8192, groups of 128, 64 and
// 32: 124, 158 and 201 us, where the unit's rate would take 54 (on the bf16 units, x and codes converted: 211, 219 and, of 32,
// 1027 rows, 2047 -> 4096, 64 where this takes 48).  Sums added beside the next group's
// MFMAs, from accumulators of their own, took as long.
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_u __attribute__((aligned(1)));

template <int BM, int BN, int WM, int WN, int G>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64, BM > 64 ? 2 : 4) q4_gemm_q8(Q4Params p) {
    constexpr int WAVES_N = BN / WN, NT = BM / WM * WAVES_N * 64;
    constexpr int MB = WM / 32, NB = WN / 32;
    static_assert(BM * 4 == NT && BN * 2 == NT, "16 bytes of x and of the weight per thread");
    constexpr int XG = lb_group<BM>(), WG = lb_group<BN>(), BUF = 4 * XG + 2 * WG;
    __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int ra = wave / WAVES_N * WM, rb = wave % WAVES_N * WN;
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    const int split = blockIdx.x / (tiles_m * tiles_n);
    int im, in;
    lb_tile(blockIdx.x - split * tiles_m * tiles_n, tiles_m, tiles_n, im, in);
    const int m0 = im * BM, n0 = in * BN;
    const int kb = split * p.k_per_split, ke = min(p.K, kb + p.k_per_split);

    // (rows and columns past the end: the last, not stored)
    const int row = min(t >> 2, p.M - 1 - m0), col = min(t >> 1, p.N - 1 - n0);
    const int8_t* const xt = p.q + m0 * p.q_m;
    const uint8_t* const wt = p.w + n0 * p.w_n;
    const bool fast = p.q_m < (1 << 22) && p.w_n < (1 << 23);   // the tile within 32 bits of bytes
    const uint32_t xo = (uint32_t)row * (uint32_t)p.q_m + 16 * (t & 3);
    const uint32_t wo = (uint32_t)col * (uint32_t)p.w_n + 16 * (t & 1);
    const int w_end = ((p.K + 31) & ~31) >> 1;                  // bytes of a row of codes
    u32x4 xr[2], wr[2];                                         // chunk c in [c % 2]
    auto load_fast = [&](int slot, int c) {
        const int k0 = kb + 64 * c;
        xr[slot] = *reinterpret_cast<const u32x4_u*>(at_bytes(xt + k0, xo));
        wr[slot] = *reinterpret_cast<const u32x4*>(at_bytes(wt + (k0 >> 1), wo));
    };
    auto load = [&](int slot, int c) {                          // x zero past K, so that codes do not matter
        const int k0 = kb + 64 * c;
        if (fast && k0 + 64 <= p.K) return load_fast(slot, c);
        const int v = anew(t), k = k0 + 16 * (v & 3);
        const int8_t* const x = xt + min(v >> 2, p.M - 1 - m0) * p.q_m + k;
        if (k + 16 <= p.K) {
            xr[slot] = *reinterpret_cast<const u32x4_u*>(x);
        } else {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint32_t b = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k + 4 * d + e < p.K) b |= (uint32_t)(uint8_t)x[4 * d + e] << (8 * e);
                xr[slot][d] = b;
            }
        }
        wr[slot] = *reinterpret_cast<const u32x4*>(wt + min(v >> 1, p.N - 1 - n0) * p.w_n +
                                                   min((k0 >> 1) + 16 * (v & 1), w_end - 16));
    };
    auto put = [&](int slot, int b) {
        char* const buf = smem + b * BUF;
        const u32x4 x = xr[slot];
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            o[i] = __builtin_amdgcn_perm(x[i + 1], x[i], 0x06040200);
            o[i + 1] = __builtin_amdgcn_perm(x[i + 1], x[i], 0x07050301);
        }
        *reinterpret_cast<u32x4*>(buf + (t & 3) * XG + (t >> 2) * 16) = o;
        *reinterpret_cast<u32x4*>(buf + 4 * XG + (t & 1) * WG + (t >> 1) * 16) = wr[slot];
    };

    f32x16 sum[MB][NB];
    i32x16 acc[MB][NB];
    zero_blocks<MB, NB>(sum);
    constexpr int GB = 128 / G;
    Q4Scales<NB, G, GB> sc(p, n0, rb + (lane & 31), kb);
    // group i of a block of 128 inputs has its sums
    auto flush = [&](auto i, int block) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const float s = sc.cur[j][i] * (1.f / 16);
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sum[m][j][r] = __builtin_fmaf((float)acc[m][j][r], s, sum[m][j][r]);
#pragma unroll
            for (int m = 0; m < MB; ++m) asm volatile("" : "+v"(sum[m][j]));   // (as q4_gemm)
        }
        if constexpr (i == GB - 1) sc.advance(kb / G + (block + 2) * GB);
    };
    using std::integral_constant;
    // chunk c, c % 2 = s
    auto multiply = [&](int c, auto s) {
        const char* const buf = smem + s() * BUF;
        u32x4 a[2][MB];
        u32x2 w[2][NB];
#pragma unroll
        for (int h = 0; h < 2; ++h) {                           // 32 k each
#pragma unroll
            for (int i = 0; i < MB; ++i)
                a[h][i] = *reinterpret_cast<const u32x4*>(buf + (2 * h + half) * XG +
                                                          (ra + 32 * i + (lane & 31)) * 16);
#pragma unroll
            for (int j = 0; j < NB; ++j)
                w[h][j] = *reinterpret_cast<const u32x2*>(
                    buf + 4 * XG + h * WG + (rb + 32 * j + (lane & 31)) * 16 + 8 * half);
        }
        auto part = [&](auto h) {
            constexpr int group = (2 * s() + h()) * 32 / G;
            constexpr bool first = (2 * s() + h()) * 32 % G == 0;
            constexpr bool whole = (2 * s() + h() + 1) * 32 % G == 0;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                u32x4 b;
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    b[2 * d] = (w[h()][j][d] << 4) & 0xf0f0f0f0u;
                    b[2 * d + 1] = w[h()][j][d] & 0xf0f0f0f0u;
                }
#pragma unroll
                for (int i = 0; i < MB; ++i) {
                    i32x16 o = acc[i][j];
                    if constexpr (first)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[r] = 0;
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
                        __builtin_bit_cast(i32x4, a[h()][i]), __builtin_bit_cast(i32x4, b), o, 0, 0, 0);
                }
            }
            if constexpr (whole) flush(integral_constant<int, group>{}, c >> 1);
        };
        part(integral_constant<int, 0>{});
        part(integral_constant<int, 1>{});
    };
    const int nk = (ke - kb + 127) >> 7 << 1;                   // (an odd one's last chunk: zeros)
    const int whole = fast ? (ke - kb) >> 6 : 0;
    load(0, 0);
    load(1, 1);
    put(0, 0);
    auto step = [&](int c, auto s) {
        lb_barrier();
        load_fast(s(), min(c + 2, nk - 1));                     // (past the last chunk: that again)
        __builtin_amdgcn_sched_barrier(0);
        multiply(c, s);
        put(~s() & 1, ~s() & 1);
    };
    int c = 0;
    for (; c + 4 <= whole || (c < whole && whole == nk); c += 2) {
        step(c, integral_constant<int, 0>{});
        step(c + 1, integral_constant<int, 1>{});
    }
    for (; c < nk; c += 2) {
        lb_barrier();
        if (c + 2 < nk) load(0, c + 2);
        multiply(c, integral_constant<int, 0>{});
        put(1, 1);
        lb_barrier();
        if (c + 3 < nk) load(1, c + 3);
        multiply(c + 1, integral_constant<int, 1>{});
        if (c + 2 < nk) put(0, 0);
    }
    const bool part = p.splits > 1;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int n = n0 + rb + 32 * j + (lane & 31);
            if (n >= p.N) continue;
            const float b = !part && p.bias ? p.bias[(int64_t)n * p.bias_stride] : 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + ra + 32 * i + lb_row(lane, r);
                if (m >= p.M) continue;
                const float v = sum[i][j][r] * p.q_scale[m];
                if (part) p.part[((int64_t)split * p.M + m) * p.N + n] = v;
                else p.y[(int64_t)m * p.y_m + (int64_t)n * p.y_n] = v + b;
            }
        }
}

// Codes and scales of a weight: a thread takes eight inputs (a dword of codes),
// G/8 neighbouring threads a group.  4096 x 16384: 119 us for 302 MB (a copy's rate: 58),
// bound by its single loads, 32 bytes apart between lanes.
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

// w = code·scale, a thread a dword of codes.  4096 x 16384: 166 us for 302 MB, bound by its
// single stores, 32 bytes apart between lanes.
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
