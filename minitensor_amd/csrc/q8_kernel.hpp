// q8_kernel.hpp -- products of 8-bit rows and 8-bit weights (include/mtlowbit.h,
// include/mtffn.h): S[m][n] = sum_k q[m][k] wq[n][k] on the integer matrix unit, whole
// numbers throughout, y = S·s[m]·ws[n] + bias[n], and the gated form
// h[m][f] = act(y[m][f]) * y[m][F + f].
//
// S is exact while a sum has fewer than 2^17 terms (|q|, |wq| <= 128), which k_per_split
// sees to; the splits' sums are added up in 64 bits.  So the result does not depend on the
// tile or the splits: one rounding to fp32, and one for each factor.  The scales are not
// multiplied by each other, whose product may leave fp32's range where y does not: the sum, zero
// or at least one, takes the row's scale first, or, where that is so large that it might
// overflow, the column's.
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
typedef u32x4 u32x4_w __attribute__((aligned(4)));
typedef i32x4 i32x4_w __attribute__((aligned(4)));

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

// A sum to y, the same wherever it is taken.  LARGE: the row's scale may be (a sum is below 2^38).
__device__ __forceinline__ bool q8_large(float s) { return __builtin_fabsf(s) > 0x1p64f; }
template <bool LARGE = true>
__device__ __forceinline__ float q8_value(float sum, float s, float ws, float bias) {
    const bool l = LARGE && q8_large(s);
    return __builtin_fmaf(sum * (l ? ws : s), l ? s : ws, bias);
}
template <bool LARGE = true>
__device__ __forceinline__ rowf4 q8_value(const rowf4& sum, float s, const rowf4& ws,
                                          const rowf4& bias) {
    rowf4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = q8_value<LARGE>(sum[e], s, ws[e], bias[e]);
    return v;
}
// The scales and biases of four neighbouring columns n.., and of their up columns.
template <bool GATED>
struct Q8Cols {
    rowf4 s[1 + GATED], b[1 + GATED];
    __device__ __forceinline__ Q8Cols(const Q8Params& p, int n) {
#pragma unroll
        for (int h = 0; h < 1 + GATED; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t c = (int64_t)h * p.N + min(n + e, p.N - 1);
                s[h][e] = p.ws[c];
                b[h][e] = p.bias ? p.bias[c * p.bias_stride] : 0.f;
            }
    }
};
// Four sums of row m, of scale s, to y; gated: a of the gates, b of the up columns.
template <bool GATED, bool LARGE = true>
__device__ __forceinline__ void q8_finish4(const Q8Params& p, int m, int n, float s,
                                           const Q8Cols<GATED>& c, const rowf4& a, const rowf4& b) {
    const rowf4 g = q8_value<LARGE>(a, s, c.s[0], c.b[0]);
    if constexpr (!GATED) {
        put4(p.y, m, n, p.N, g);
    } else {
        const rowf4 u = q8_value<LARGE>(b, s, c.s[1], c.b[1]);
        if (p.gu.p) {
            put4(p.gu, m, n, p.N, g);
            put4(p.gu, m, (int64_t)p.N + n, 2 * (int64_t)p.N, u);
        }
        put4(p.y, m, n, p.N, gate4(p.act, g, u));
    }
}

// Sixteen bytes from any address, by dwords on multiples of four bytes (a load off those
// comes apart: tiles of 1027 x 2047 -> 4095 loaded so took 48 us, so 39, copied to aligned
// rows first 33).  A dword is read only where it holds a byte that is asked for.
struct Q8Unit {
    u32x4 d;
    uint32_t last;
};
__device__ __forceinline__ u32x4 q8_align(const Q8Unit& u, uint32_t shift) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = __builtin_amdgcn_alignbyte(i < 3 ? u.d[i + 1] : u.last, u.d[i], shift);
    return r;
}

__device__ __forceinline__ Q8Unit q8_load(const int8_t* p) {
    const uint32_t shift = (uint32_t)(uintptr_t)p & 3;
    const char* const q = reinterpret_cast<const char*>(p) - shift;
    return {*reinterpret_cast<const u32x4_w*>(q),
            *reinterpret_cast<const uint32_t*>(q + (shift ? 16 : 12))};
}
__device__ __forceinline__ i32x4 q8_any(const int8_t* p) {
    return __builtin_bit_cast(i32x4, q8_align(q8_load(p), (uint32_t)(uintptr_t)p & 3));
}
// ... of a row from k on, zero from `end` (>= 1) on.
__device__ __forceinline__ u32x4 q8_bytes(const int8_t* row, int k, int end) {
    const int n = min(end - k, 16);                    // that there are
    const int8_t* const p = n > 0 ? row + k : row;
    const uint32_t shift = (uint32_t)(uintptr_t)p & 3;
    const uint32_t* const q = reinterpret_cast<const uint32_t*>(p - shift);
    const int most = ((int)shift + max(n, 1) - 1) >> 2;
    Q8Unit u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.d[i] = q[min(i, most)];
    u.last = q[most];
    u32x4 r = q8_align(u, shift);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = n - 4 * i;                    // bytes of this dword
        r[i] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1;
    }
    return r;
}

// Tiles of BM x BN over chunks of BK bytes of k, in S LDS buffers.  A buffer holds the
// tile's rows, then its columns, BK bytes each; a row's 16-byte units change places by its
// number, so that the 16 rows that a fragment read takes at a time lie on different banks.
// The units go straight from memory to LDS, 1 KB a wave instruction, up to S chunks ahead
// (rows on multiples of 16 bytes, 2^24 apart at most: q8_align_rows).  The fragments of the next
// 32 k are read beside these ones' MFMAs, the next chunk's first ones too: a chunk's one
// barrier stands before its last MFMAs, when all of it is in registers and the next one in
// LDS, and its buffer is filled again from there on.  (2048 x 4096 -> 8192 with 256 x 256 tiles:
// 67 us, 2.05 POP/s, gated -> 2 x 8192 137 us, 2.0: the matrix units at the power limit, a library's
// product 2.1.)  A chunk that the range of k ends in goes
// first, with its bounds checked, all its units at once (1024 x 2064 -> 4096, rows
// 2176 bytes apart: 20.8 us, 2048 of those inputs 19.1).
template <int BM, int BN, int WM, int WN, int BK, int S, bool GATED>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64) q8_gemm(Q8Params p) {
    constexpr int WAVES_N = BN / WN, NW = BM / WM * WAVES_N, NT = 64 * NW;
    constexpr int MB = WM / 32, NB = WN / 32, KK = BK / 32;
    constexpr int UNITS = BK / 16, ROWS = BM + BN;
    constexpr int BUF = ROWS * BK;
    constexpr int NI = ROWS * UNITS / NT;              // units of a thread, a chunk
    constexpr int NA = BM * UNITS / NT;                // of rows; the rest are columns'
    static_assert(NI * NT == ROWS * UNITS && NA * NT == BM * UNITS, "whole instructions");
    static_assert(BK == 64 || BK == 128, "four or eight units a row");
    static_assert(S * BUF >= NW * 32 * 64 * 4 + BM * 4, "the epilogue's staging");
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
    const int whole = (ke - kb) / BK, part_k = (ke - kb) % BK;

    // unit i of this thread: row and place of i*NT + t, holding the row's unit there
    auto swz = [](int row) { return BK == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
    auto row_of = [&](int r) {
        return r < BM ? p.x + min(m0 + r, p.M - 1) * p.x_m
                      : p.w + q8_channel<GATED>(p, n0 + r - BM) * p.w_n;
    };
    // (eight or sixteen rows an instruction: all of them x's, gates or up columns)
    const int8_t* const xb = p.x + m0 * p.x_m + kb;
    const int8_t* const wb = p.w + (int64_t)(GATED ? n0 / 2 : n0) * p.w_n + kb;
    const int8_t* const ub = wb + (int64_t)p.N * p.w_n;
    auto base = [&](int i) {
        if (i < NA) return xb;
        if constexpr (!GATED) return wb;
        return ((i * NT + wave * 64) / UNITS - BM) & 32 ? ub : wb;
    };
    uint32_t src[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int e = i * NT + t, r = e / UNITS, unit = (e % UNITS) ^ swz(r);
        src[i] = (uint32_t)(row_of(r) + kb + 16 * unit - base(i));
    }
    auto dma = [&](int slot, int c) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            __builtin_amdgcn_global_load_lds(
                (const void __attribute__((address_space(1)))*)(base(i) + (int64_t)c * BK + src[i]),
                (void __attribute__((address_space(3)))*)(smem + slot * BUF + (i * NT + wave * 64) * 16),
                16, 0, 0);
    };

    i32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int sw = swz(lrow);
    struct Frags {
        i32x4 a[MB], b[NB];
    };
    auto read = [&](Frags& f, int slot, int kk) {
        const char* const buf = smem + slot * BUF + lrow * BK + ((2 * kk + half) ^ sw) * 16;
#pragma unroll
        for (int i = 0; i < MB; ++i)
            f.a[i] = *reinterpret_cast<const i32x4*>(buf + (ra + 32 * i) * BK);
#pragma unroll
        for (int j = 0; j < NB; ++j)
            f.b[j] = *reinterpret_cast<const i32x4*>(buf + (BM + rb + 32 * j) * BK);
    };
    // (the transposed block: a lane has four neighbouring columns of a row)
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.b[j], f.a[i], acc[i][j], 0, 0, 0);
    };

    const int last = whole - 1;
    if (whole > 0)
        for (int c = 0; c < S - 1; ++c) dma(c, min(c, last));
    if (part_k) {                                      // in the last buffer
        char* const buf = smem + (S - 1) * BUF;
        u32x4 v[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int e = i * NT + t, unit = (e % UNITS) ^ swz(e / UNITS);
            v[i] = u32x4{0, 0, 0, 0};
            if (16 * unit + 16 <= part_k)
                v[i] = *reinterpret_cast<const u32x4*>(base(i) + (int64_t)whole * BK + src[i]);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) *reinterpret_cast<u32x4*>(buf + (i * NT + t) * 16) = v[i];
        if (part_k % 16) {                             // a unit that the range ends in
            lb_barrier();
            const int unit = part_k / 16;
            for (int r = t; r < ROWS; r += NT)
                *reinterpret_cast<u32x4*>(buf + (r * UNITS + (unit ^ swz(r))) * 16) =
                    q8_bytes(row_of(r), kb + whole * BK + 16 * unit, ke);
        }
        lb_barrier();
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            Frags f;
            read(f, S - 1, kk);
            multiply(f);
        }
        lb_barrier();
    }
    if (whole > 0) {
        dma(S - 1, min(S - 1, last));
        __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(NI * (S - 1)));
        __builtin_amdgcn_s_barrier();
        Frags f[2];
        read(f[0], 0, 0);
        int slot = 0;
#pragma unroll 1
        for (int c = 0; c < whole; ++c) {
            const int next = slot + 1 == S ? 0 : slot + 1;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                if (kk == KK - 1) {
                    // chunk c is in registers, the next one in LDS
                    // (past the last chunk: that again, where nobody reads it)
                    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(NI * (S - 2)));
                    __builtin_amdgcn_s_barrier();
                    dma(slot, min(c + S, last));
                    read(f[(kk + 1) & 1], next, 0);
                } else {
                    read(f[(kk + 1) & 1], slot, kk + 1);
                }
                multiply(f[kk & 1]);
                // a read (and a load) beside each MFMA
#pragma unroll
                for (int i = 0; i < MB * NB; ++i) {
                    if (i < MB + NB) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (kk == KK - 1)
                        __builtin_amdgcn_sched_group_barrier(0x020, (NI + MB * NB - 1) / (MB * NB), 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            slot = next;
        }
    }
    // (what was fetched again has landed before the buffers are used anew)
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));

    // Each wave turns its blocks round in a part of LDS of its own, two neighbouring ones at a
    // time (gated: of gates and up columns), so that sixteen lanes write a row's 64 columns
    // (eight its 32 features).  No load from memory stands between two stores: it would wait
    // for the first.  (Two rows of 32 columns a store straight from the registers saved 3 us
    // of 16 where few tiles are stored and nothing where many are, and cost 5 at an edge,
    // whose unrolled code a tile runs once.)
    const bool part = p.splits > 1;
    __syncthreads();
    i32x4* const stage = reinterpret_cast<i32x4*>(smem) + wave * 32 * 16;
    float* const scales = reinterpret_cast<float*>(smem + NW * 32 * 64 * 4);
    bool large = false;                                // among the wave's rows
    if (!part) {
        for (int r = t; r < BM; r += NT) scales[r] = p.xs[min(m0 + r, p.M - 1)];
        __syncthreads();
        if constexpr (!GATED) large = __ballot(q8_large(scales[ra + lane % WM])) != 0;
    }
    constexpr int GROUPS = GATED ? 8 : 16, STEP = 64 / GROUPS, PASS = 32 / STEP;
    const int g = lane % GROUPS, r0 = lane / GROUPS;
#pragma unroll
    for (int jj = 0; jj < NB; jj += 2) {
        const int c0 = n0 + rb + 32 * jj, n = (GATED ? c0 / 2 : c0) + 4 * g;
        const Q8Cols<GATED> cols4(p, min(n, p.N - 1));
#pragma unroll
        for (int i = 0; i < MB; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    stage[lrow * 16 + ((8 * j + 2 * q + half) ^ (lrow & 15))] =
                        i32x4{acc[i][jj + j][4 * q], acc[i][jj + j][4 * q + 1],
                              acc[i][jj + j][4 * q + 2], acc[i][jj + j][4 * q + 3]};
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const int m1 = m0 + ra + 32 * i;
            if (part) {
                i32x4 a[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int r = (lane >> 4) + 4 * k;
                    a[k] = stage[r * 16 + ((lane & 15) ^ (r & 15))];
                }
                int32_t* const d = p.part + ((int64_t)split * p.M + m1 + (lane >> 4)) * p.part_n + c0 +
                                   4 * (lane & 15);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (m1 + (lane >> 4) + 4 * k < p.M)
                        *reinterpret_cast<i32x4_w*>(d + 4 * k * p.part_n) = a[k];
            } else if (!GATED && __builtin_expect(large, 0)) {   // (rolled up, and out of the way)
#pragma unroll 1
                for (int r = r0; r < 32; r += STEP) {
                    const int m = m1 + r;
                    if (m >= p.M || n >= p.N) continue;
                    const rowf4 x = __builtin_convertvector(stage[r * 16 + (g ^ (r & 15))], rowf4);
                    q8_finish4<GATED>(p, m, n, scales[ra + 32 * i + r], cols4, x, x);
                }
            } else {
                i32x4 a[PASS], b[GATED ? PASS : 1];
                float s[PASS];
#pragma unroll
                for (int k = 0; k < PASS; ++k) {
                    const int r = r0 + STEP * k;
                    a[k] = stage[r * 16 + (g ^ (r & 15))];
                    if constexpr (GATED) b[k] = stage[r * 16 + ((g + 8) ^ (r & 15))];
                    s[k] = scales[ra + 32 * i + r];
                }
                // (whole groups of four neighbouring columns)
                const bool vec = p.y.cs == 1 && n + 4 <= p.N;
                float* const d = p.y.p + (int64_t)(m1 + r0) * p.y.rs + n;
#pragma unroll
                for (int k = 0; k < PASS; ++k) {
                    const int m = m1 + r0 + STEP * k;
                    if (m >= p.M || n >= p.N) continue;
                    const rowf4 x = __builtin_convertvector(a[k], rowf4);
                    if constexpr (GATED) {
                        q8_finish4<GATED>(p, m, n, s[k], cols4, x, __builtin_convertvector(b[k], rowf4));
                    } else {
                        const rowf4 y = q8_value<false>(x, s[k], cols4.s[0], cols4.b[0]);
                        if (vec) *reinterpret_cast<rowf4_u*>(d + STEP * k * p.y.rs) = y;
                        else put4(p.y, m, n, p.N, y);
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
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
        q8_finish4<GATED>(p, m, n, p.xs[m], Q8Cols<GATED>(p, n), a, GATED ? sum(c + 32) : a);
    }
}

// Rows to a workspace where each starts on a multiple of 16 bytes and is zero to its end
// there, of one operand or of both: a wave to a row's whole units, and, in workgroups of
// their own, a thread to each row's last part.  (1027 and 4095 rows of 2047: 9 us.)
struct Q8Align {
    const int8_t* src[2];
    int64_t ld[2], rows[2];           // no rows: the operand stays where it is
    int8_t* dst[2];
    int64_t ld_dst;
    int K;
    int wave_blocks;                  // workgroups of the whole units
};
template <int = 0>
__global__ void __launch_bounds__(256) q8_align_rows(Q8Align p) {
    const int64_t total = p.rows[0] + p.rows[1];
    const int whole = p.K >> 4, t = threadIdx.x, lane = t & 63;
    auto at = [&](int64_t i, const int8_t*& src, char*& dst) {
        const int o = i >= p.rows[0];
        const int64_t r = o ? i - p.rows[0] : i;
        src = p.src[o] + r * p.ld[o];
        dst = reinterpret_cast<char*>(p.dst[o]) + r * p.ld_dst;
    };
    const int8_t* src;
    char* dst;
    if ((int)blockIdx.x < p.wave_blocks) {
        for (int64_t i = (int64_t)blockIdx.x * 4 + (t >> 6); i < total; i += (int64_t)p.wave_blocks * 4) {
            at(i, src, dst);
            const uint32_t shift = (uint32_t)(uintptr_t)src & 3;
            constexpr int U = 2;
            for (int u0 = lane; u0 < whole; u0 += 64 * U) {
                Q8Unit x[U];
#pragma unroll
                for (int i = 0; i < U; ++i) x[i] = q8_load(src + 16 * min(u0 + 64 * i, whole - 1));
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (u0 + 64 * i < whole)
                        *reinterpret_cast<u32x4*>(dst + 16 * (u0 + 64 * i)) = q8_align(x[i], shift);
            }
        }
    } else {
        const int64_t step = (int64_t)(gridDim.x - p.wave_blocks) * 256;
        for (int64_t i = (int64_t)(blockIdx.x - p.wave_blocks) * 256 + t; i < total; i += step) {
            at(i, src, dst);
            if (p.K % 16) *reinterpret_cast<u32x4*>(dst + 16 * whole) = q8_bytes(src, 16 * whole, p.K);
            for (int64_t k = (p.K + 15) / 16 * 16; k < p.ld_dst; k += 16)
                *reinterpret_cast<u32x4*>(dst + k) = u32x4{0, 0, 0, 0};
        }
    }
}

// Few rows, bound by the weight's bytes, and small products.  A workgroup owns MB blocks of 16
// rows and NC blocks of 16 columns (gated:
// NC/2 of gates and the same features' up columns) and all of K; its waves take chunks of
// 256 inputs in turn, straight from memory to the operands of 16x16x64 products (lane l: row
// or column l % 16, 16 bytes from 16·(l/16) on), and their sums meet in LDS.  (One row 4096 ->
// 4096: 5.0 us, a launch and one trip to memory; gated 4096 -> 2 x 8192, 67 MB: 10.8 us where the
// weight is in the 256 MB cache, 6.2 TB/s.)
// KIND: rows on multiples of 4 bytes, at any address, or (Q8_LONG) at any address and any number
// of inputs: the waves' sums, 2^16 inputs' each, added up in 64 bits.  (For what the tiles do not take: rows of
// 2^24 inputs and more.)
enum { Q8_WORDS = 0, Q8_BYTES = 1, Q8_LONG = 2 };
constexpr int kQ8Segment = 1 << 19;   // inputs of eight waves' 32-bit sums

template <int MB, int NC, bool GATED, int KIND>
__global__ void __launch_bounds__(512) q8_few(Q8Params p) {
    constexpr int W = 8, C = 16 * NC;
    static_assert(!GATED || NC % 2 == 0, "gates and up columns");
    using Sum = std::conditional_t<KIND == Q8_LONG, int64_t, int>;
    __shared__ Sum red[W][16 * MB][C];
    const int t = threadIdx.x, lane = t & 63, col = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // features of a workgroup: half its columns where they are gated
    constexpr int F = GATED ? C / 2 : C;
    // (blocks of rows of the same columns side by side, so that these come from memory once)
    const int blocks = (p.M + 16 * MB - 1) / (16 * MB);
    const int n0 = blockIdx.x / blocks * F, m0 = blockIdx.x % blocks * (16 * MB);
    const int8_t* wr[NC];
#pragma unroll
    for (int q = 0; q < NC; ++q) {                    // (past the end: the last, not stored)
        const int f = min(n0 + 16 * (GATED ? q % (NC / 2) : q) + col, p.N - 1);
        wr[q] = p.w + (GATED && q >= NC / 2 ? (int64_t)p.N + f : (int64_t)f) * p.w_n;
    }
    const int8_t* xr[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) xr[b] = p.x + (int64_t)min(m0 + 16 * b + col, p.M - 1) * p.x_m;
    auto get = [&](const int8_t* row, int k) {
        if constexpr (KIND == Q8_WORDS) return *reinterpret_cast<const i32x4_w*>(row + k + 16 * j);
        else return q8_any(row + k + 16 * j);
    };
    i32x4 acc[MB][NC];
    auto clear = [&] {
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int q = 0; q < NC; ++q) acc[b][q] = i32x4{0, 0, 0, 0};
    };
    // inputs from kb on, whole chunks of 256 of them
    auto run = [&](int kb, int whole) {
#pragma unroll 1
        for (int c = wave; c < whole; c += W) {
            i32x4 x[4][MB], w[4][NC];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = kb + 256 * c + 64 * i;
#pragma unroll
                for (int q = 0; q < NC; ++q) w[i][q] = get(wr[q], k);
#pragma unroll
                for (int b = 0; b < MB; ++b) x[i][b] = get(xr[b], k);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int q = 0; q < NC; ++q)
                        acc[b][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[i][b], w[i][q], acc[b][q], 0, 0, 0);
        }
    };
    // fewer than 256 inputs from kb on, 64 a wave
    auto rest = [&](int kb) {
        const int k = kb + 64 * wave;
        if (wave >= 4 || k >= p.K) return;
        i32x4 x[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) x[b] = __builtin_bit_cast(i32x4, q8_bytes(xr[b], k + 16 * j, p.K));
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            const i32x4 w = __builtin_bit_cast(i32x4, q8_bytes(wr[q], k + 16 * j, p.K));
#pragma unroll
            for (int b = 0; b < MB; ++b)
                acc[b][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[b], w, acc[b][q], 0, 0, 0);
        }
    };
    auto put = [&](bool add) {
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int q = 0; q < NC; ++q)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    Sum& d = red[wave][16 * b + 4 * j + r][16 * q + col];
                    d = add ? d + acc[b][q][r] : acc[b][q][r];
                }
    };
    const int whole = p.K >> 8;
    clear();
    if constexpr (KIND == Q8_LONG) {
        int kb = 0;
        for (; p.K - kb > kQ8Segment; kb += kQ8Segment) {
            run(kb, kQ8Segment >> 8);
            put(kb > 0);
            clear();
        }
        const int left = (p.K - kb) >> 8;
        run(kb, left);
        rest(kb + 256 * left);
        put(kb > 0);
    } else {
        run(0, whole);
        rest(256 * whole);
        put(false);
    }
    __syncthreads();
    const int rows = min(16 * MB, p.M - m0);
    for (int e = t; e < rows * F; e += 64 * W) {
        const int r = e / F, c = e % F, n = n0 + c, m = m0 + r;
        if (n >= p.N) continue;
        auto value = [&](int at, int64_t ch) {
            int64_t s = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) s += red[w][r][at];
            return q8_value((float)s, p.xs[m], p.ws[ch], p.bias ? p.bias[ch * p.bias_stride] : 0.f);
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
