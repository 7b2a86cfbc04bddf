// lowbit_gemm.hpp -- the product that the operators of include/mtlowbit.h share: an
// operand A in fp32, cut into three bf16 values, times an operand B in 8 or 4 bits
// (exact in bf16), on the bf16 matrix units.
//
// Tiles of BM x BN over chunks of 32 k, in two LDS buffers: while chunk c is multiplied,
// chunk c+1, loaded into registers before, is converted to bf16 and written to the other
// buffer, and the chunks up to c+D are on their way from memory.  One barrier per chunk; it
// waits for LDS alone, so that the loads stay in flight across it.  (A third buffer, from
// which the next chunk's first fragments came before the barrier, cost more in addresses
// than it saved in waiting: the 2048-row prompt 4096 -> 8192 took 435 us against 402.)
//
// Each wave multiplies WM x WN in blocks of 32x32.  A's parts make a row three times
// as dear as a column in LDS reads (three fragments, one for B) and four to five times
// as dear in conversions, so tiles and waves are wider than high: 128x256 in waves of 32x128
// reads 7 fragments per 12 MFMAs, 64x64 ones 8.
//
// The sums of a group of k are taken on the matrix unit from zero and then added to
// the result in fp32, by the group's scale where there is one: the unit does not
// round to nearest, and over 10^5 terms that would show.
#pragma once

#include "gemm_split.hpp"
#include "lowbit_rows_kernel.hpp"
#include "tile_helpers.hpp"

namespace mtk {

// Two floats' upper halves: themselves where they are exact in bf16, else cut off.
__device__ __forceinline__ uint32_t bf16_cut(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
}

// The parts of eight values, h + m + l = x (6.5 instructions each): eight of its 24 bits each,
// cut off and not rounded; with h rounded the values above bf16's largest, 3.39e38, would
// become infinite.  Only l is, to the nearest: below 2^-110 it may reach past bf16's last
// place, 2^-133.  What is left of an infinity or a NaN (a NaN) is made zero, so that its
// products are those of fp32: the middle of (r, r, 0) is r, and 0 where r is a NaN.  (A NaN
// whose set bits are all in the lower half, a signalling one, would count as an infinity; no
// operation gives such a one.)
// WIDE: the cut values are kept for the subtractions and converted, rather than packed by
// v_perm and taken apart again: as many instructions and two registers more (the weight
// gradient's 128x256 tile, 8192 rows, 4096 -> 4096: 672 us against 683; its 64x128 tile, 256
// rows, 2048 -> 1000 with dX: 41.1 against 40.6).
template <bool WIDE>
__device__ __forceinline__ void cut8(const float (&x)[8], u32x4& h, u32x4& m, u32x4& l) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x0 = x[2 * i], x1 = x[2 * i + 1];
        float h0, h1, m0, m1;
        if constexpr (WIDE) {
            h0 = bf16_hi(__float_as_uint(x0));
            h1 = bf16_hi(__float_as_uint(x1));
            h[i] = bf16_pair(h0, h1);
        } else {
            h[i] = opaque(bf16_cut(x0, x1));
            h0 = bf16_lo(h[i]);
            h1 = bf16_hi(h[i]);
        }
        float r0 = x0 - h0, r1 = x1 - h1;
        r0 = __builtin_amdgcn_fmed3f(r0, r0, 0.f);
        r1 = __builtin_amdgcn_fmed3f(r1, r1, 0.f);
        if constexpr (WIDE) {
            m0 = bf16_hi(__float_as_uint(r0));
            m1 = bf16_hi(__float_as_uint(r1));
            m[i] = bf16_pair(m0, m1);
            l[i] = bf16_pair(r0 - m0, r1 - m1);
        } else {
            m[i] = opaque(bf16_cut(r0, r1));
            m0 = bf16_lo(m[i]);
            m1 = bf16_hi(m[i]);
            l[i] = bf16_pair(r0 - m0, r1 - m1);
        }
    }
}

// Eight int8 values as bf16.
__device__ __forceinline__ u32x4 q8_bf16(const u32x2& q) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = q[i >> 1] >> (16 * (i & 1));
        r[i] = bf16_cut((float)(int8_t)w, (float)(int8_t)(w >> 8));
    }
    return r;
}

// LDS of a chunk: per part four groups of eight k, each a column of 16-byte entries, one
// per row, and two entries more, so that the groups of a row start 32 bytes apart modulo
// the banks' 128.
template <int ROWS>
constexpr int lb_group() { return (ROWS + 2) * 16; }
template <int ROWS>
constexpr int lb_plane() { return 4 * lb_group<ROWS>(); }

// The loop.  LA: loader with
//   Raw                          what a thread holds of a chunk
//   fast                         whether load_fast may be called at all
//   load_fast(Raw&, int k0)      chunk of 32 k from k0 on, all of them below k_end
//   load(Raw&, int k0)           any chunk, zero past the end
//   store(const Raw&, char*, live)   converted, to its part of the buffer (live: not a
//                                chunk that is there only again)
//   kBytes, kGroup, entry(row)   LDS size of a part and of a group of eight k, and the
//                                entry of a row in a group: entry(32a + b) = entry(32a)
//                                + entry(b)
//   kWork                        vector instructions of store
// LB: the same, or (kBlock) with its values brought to LDS as they are, in blocks of four
// chunks, from which each chunk is converted:
//   load(Raw&, int k0)           block from k0 on; past the end anything
//   stage(const Raw&, char*)     to LDS, kRaw bytes
//   Codes, peek(Codes&, const char*, int s)   chunk s of the block there
//   store(const Codes&, char*)
// smem: two buffers of a chunk, and two of kRaw.
// P: parts of A.  D: chunks ahead (2 or 4).  GC: chunks (1, 2 or 4) whose sums are taken on the matrix unit;
// flush(i, block) adds those of group i of a block (from k_begin on) to the result; called
// in order, with kLate a step late, beside the next group's first MFMAs.
template <int P, int GC, int D, int MB, int NB, class LA, class LB, class Flush>
__device__ __forceinline__ void lb_product(LA& la, LB& lb, char* smem, int k_begin, int k_end, int ra,
                                           int rb, int lane, f32x16 (&acc)[MB][NB], Flush flush) {
    using std::integral_constant;
    constexpr int BUF = P * LA::kBytes + LB::kBytes;
    constexpr int NH = P * MB * NB, NR = P * MB + NB;         // MFMAs and reads of half a chunk
    constexpr bool kLate = GC == 4 && (MB * NB < 4 || LA::kLate);
    const int nk = (k_end - k_begin + 31) >> 5, nb = (nk + 3) >> 2;
    // chunks that load_fast takes: all but a partial one
    const int whole = la.fast && lb.fast ? (k_end - k_begin) >> 5 : 0;
    const int half = lane >> 5, row = lane & 31;
    char* const raw = smem + 2 * BUF;
    typename LA::Raw xa[D];               // chunk c in xa[c % D]
    typename LB::Raw xb[LB::kBlock ? 1 : D];   // (kBlock: the next block)
    auto fetch = [&](int c, int slot) {
        if (c >= nk) return;
        la.load(xa[slot], k_begin + 32 * c);
        if constexpr (!LB::kBlock) lb.load(xb[slot], k_begin + 32 * c);
    };
    // (what is read from LDS is read before anything is written there: the compiler
    // keeps the order of the two)
    typename LB::Codes codes;
    auto peek = [&](int c) {
        if constexpr (LB::kBlock) lb.peek(codes, raw + (c >> 2 & 1) * LB::kRaw, c & 3);
    };
    auto put = [&](int c, int slot) {
        char* const buf = smem + (c & 1) * BUF;
        la.store(xa[slot], buf, c < nk);
        if constexpr (LB::kBlock) lb.store(codes, buf + P * LA::kBytes);
        else lb.store(xb[slot], buf + P * LA::kBytes);
    };
    // the fragments of half h of the chunk in buf, and its MFMAs
    struct Frags {
        u32x4 a[P][MB], b[NB];
    };
    auto read = [&](Frags& f, const char* buf, int h) {
        const int g = 2 * h + half;
#pragma unroll
        for (int q = P - 1; q >= 0; --q)
#pragma unroll
            for (int i = 0; i < MB; ++i)
                f.a[q][i] = *reinterpret_cast<const u32x4*>(
                    buf + q * LA::kBytes + g * LA::kGroup +
                    (LA::entry(row) + LA::entry(ra) + LA::entry(32 * i)) * 16);
#pragma unroll
        for (int j = 0; j < NB; ++j)
            f.b[j] = *reinterpret_cast<const u32x4*>(
                buf + P * LA::kBytes + g * LB::kGroup +
                (LB::entry(row) + LB::entry(rb) + LB::entry(32 * j)) * 16);
    };
    auto multiply = [&](const Frags& f, bool first) {
#pragma unroll
        for (int q = P - 1; q >= 0; --q)
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    f32x16 c = acc[i][j];
                    if (first && q == P - 1)
#pragma unroll
                        for (int r = 0; r < 16; ++r) c[r] = 0.f;
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        __builtin_bit_cast(bf16x8, f.a[q][i]), __builtin_bit_cast(bf16x8, f.b[j]), c,
                        0, 0, 0);
                }
    };
    // Chunk c = 4n + s, all of whose neighbours are whole: no branch, so that the
    // conversions can go beside the MFMAs (after them, as the compiler had it, the
    // matrix unit stood still meanwhile).
    auto step = [&](int n, auto sc) {
        constexpr int s = sc;
        const int c = 4 * n + s;
        lb_barrier();
        // (past the last chunk: that again)
        const int k = k_begin + 32 * min(c + D, nk - 1);
        la.load_fast(xa[s % D], k);
        if constexpr (!LB::kBlock) lb.load_fast(xb[s % D], k);
        if constexpr (LB::kBlock)
            if constexpr (s == 3) lb.load_fast(xb[0], k_begin + 128 * min(n + 2, nb - 1));
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kLate && s == 0)
            if (n > 0) flush(integral_constant<int, 0>{}, n - 1);
        const char* const buf = smem + (s & 1) * BUF;
        Frags f, g;
        peek(c + 1);
        read(f, buf, 0);
        read(g, buf, 1);
        multiply(f, s % GC == 0);
        multiply(g, false);
        if constexpr (LB::kBlock)
            if constexpr (s == 2) lb.stage(xb[0], raw + (n + 1 & 1) * LB::kRaw);
        put(c + 1, (s + 1) % D);
        constexpr int NV = (LA::kWork + LB::kWork + 2 * NH - 1) / (2 * NH) + 1;
        // (the second half's fragments as late as they may come: registers)
        constexpr int R0 = NH > NR + 2 ? NH - NR - 2 : 0;
        __builtin_amdgcn_sched_group_barrier(0x100, LB::kReads + NR, 0);
#pragma unroll
        for (int i = 0; i < 2 * NH; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (i >= R0 && i < R0 + NR) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, NV, 0);
        }
        if constexpr (!kLate && s % GC == GC - 1) {
            __builtin_amdgcn_sched_barrier(0);
            flush(integral_constant<int, s / GC>{}, n);
        }
    };
    if (nk <= 0) return;
#pragma unroll
    for (int c = 0; c < D; ++c) fetch(c, c);
    if constexpr (LB::kBlock) {
        lb.load(xb[0], k_begin);
        lb.stage(xb[0], raw);
        if (nb > 1) lb.load(xb[0], k_begin + 128);
        lb_barrier();
    }
    peek(0);
    put(0, 0);
    int n = 0;
    for (; 4 * n + 4 <= whole && (4 * n + 4 + D <= whole || whole == nk); ++n) {
        step(n, integral_constant<int, 0>{});
        step(n, integral_constant<int, 1>{});
        step(n, integral_constant<int, 2>{});
        step(n, integral_constant<int, 3>{});
    }
    // the rest, in one rolled step; the chunks move up in their places instead
    for (int c = 4 * n; c < nk; ++c) {
        lb_barrier();
#pragma unroll
        for (int i = 0; i + 1 < D; ++i) {
            xa[i] = xa[i + 1];
            if constexpr (!LB::kBlock) xb[i] = xb[i + 1];
        }
        fetch(c + D, D - 1);
        if (c % GC == 0) {
            if (kLate && c > 0) flush(integral_constant<int, 0>{}, (c >> 2) - 1);
            zero_blocks<MB, NB>(acc);
        }
        if (c + 1 < nk) peek(c + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Frags f;
            read(f, smem + (c & 1) * BUF, h);
            multiply(f, false);
        }
        if constexpr (LB::kBlock) {
            if ((c & 3) == 2 && (c >> 2) + 1 < nb)
                lb.stage(xb[0], raw + ((c >> 2) + 1 & 1) * LB::kRaw);
            if ((c & 3) == 3 && (c >> 2) + 2 < nb) lb.load(xb[0], k_begin + 32 * (c + 5));
        }
        if (c + 1 < nk) put(c + 1, 0);
        if (!kLate && ((c + 1) % GC == 0 || c + 1 == nk)) {
            const int i = (c & 3) / GC;
            if (i == 0) flush(integral_constant<int, 0>{}, c >> 2);
            if constexpr (GC < 4)
                if (i == 1) flush(integral_constant<int, 1>{}, c >> 2);
            if constexpr (GC < 2) {
                if (i == 2) flush(integral_constant<int, 2>{}, c >> 2);
                if (i == 3) flush(integral_constant<int, 3>{}, c >> 2);
            }
        }
    }
    if (kLate) flush(integral_constant<int, 0>{}, nb - 1);
}

// Block element r of a lane: row 8*(r/4) + 4*(lane/32) + r%4, column lane%32.
__device__ __forceinline__ int lb_row(int lane, int r) {
    return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}

// y[m][n] = beta*y + bias[n] + the splits' partials [splits][M][N] in order, and
// v[i] = beta_v*v + those of part_v [splits][L] (no splits: nothing is read).
struct LbSum {
    const float* part;
    int splits, M, N;
    const float* bias;                // nullptr: none
    int64_t bias_stride;
    float* y;
    int64_t y_m, y_n;
    float beta;
    const float* part_v;
    float* v;                         // nullptr: none
    int64_t v_stride;
    float beta_v;
    int L;
};
__global__ void __launch_bounds__(256) lb_sum(LbSum p) {
    const int64_t n = (int64_t)p.M * p.N, all = n + (p.v ? p.L : 0);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all;
         i += (int64_t)gridDim.x * 256) {
        const bool vec = i >= n;
        const float* const part = vec ? p.part_v + (i - n) : p.part + i;
        const int64_t stride = vec ? p.L : n;
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < p.splits; ++k) s += part[k * stride];
        const int m = (int)(i / p.N), c = (int)(i - (int64_t)m * p.N);
        if (p.bias && !vec) s += p.bias[(int64_t)c * p.bias_stride];
        float* const d = vec ? p.v + (i - n) * p.v_stride : p.y + (int64_t)m * p.y_m + (int64_t)c * p.y_n;
        const float beta = vec ? p.beta_v : p.beta;
        *d = beta != 0.f ? beta * *d + s : s;
    }
}

}  // namespace mtk
