// lowbit_back_kernel.hpp -- a Linear layer's weight gradient from an input kept
// in 8 bits: dW[o][c] = sum_r (dY[r][o]·scale[r]) q[r][c].
//
// The row's scale goes to dY (one fp32 rounding), and q is exact in bf16: three
// bf16 products in fp32's precision (lowbit_gemm.hpp), where a product of two fp32
// operands takes six.  The matrix unit bounds it, at the clock that its power
// allows: 8192 rows, 4096 -> 4096, 661-718 us (a bf16 product of that size and
// three parts at a library's rate: 650); dY is read down its columns, 8 rows of an
// output per thread, and cut there, which costs four to five times what q does, so
// the tiles are wider in inputs than in outputs.
#pragma once

#include "lowbit_gemm.hpp"

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
    float* db;                        // [O], nullptr: not wanted
    int64_t db_stride;
    float beta_b;
    float* part_b;                    // [splits][O]
    int R, O, C;
    int splits, r_per_split;          // a multiple of 128
};

// A load of an address that is the same across the wave.
__device__ __forceinline__ float uniform_load(const float* p) {
    return *(const float __attribute__((address_space(4)))*)p;
}

// Both operands lie across k (= r).  dY: a thread takes eight rows of one output,
// consecutive outputs on consecutive lanes.  SUM: the rows of each output added up as they
// pass (the bias gradient; dY is read once for both), and what each addition's rounding lost
// beside it: a thread adds R / 32 times (8192 rows of normal values, 2-norm error 2.9e-7
// without).
template <int BM, int NT, bool SUM>
struct BackDy {
    static constexpr int N = BM * 4 / NT, kGroup = lb_group<BM>(), kBytes = lb_plane<BM>();
    static_assert(N * NT == BM * 4 && BM % 64 == 0, "whole items, rows the same across a wave");
    static constexpr int kWork = N * 8 * 8;
    static constexpr bool kLate = true;
    struct Raw {
        float a[N][8], s[N][8];
    };
    const float* base;                // output m0, row 0
    uint32_t off[N];                  // of the item's output, in bytes
    const float* scale;
    int64_t ld, so;
    int R, t, last, g[N];
    float sum[N], lost[N];
    bool fast;                        // the tile's outputs within 32 bits of bytes
    __device__ __forceinline__ static int entry(int row) { return row; }
    __device__ __forceinline__ BackDy(const BackParams& p, int m0, int t_)
        : base(p.dy + m0 * p.dy_o), scale(p.scale), ld(p.dy_r), so(p.dy_o), R(p.R), t(t_),
          last(p.O - 1 - m0), fast(p.dy_o < (1 << 22)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {                      // (outputs past O: the last, not stored)
            g[i] = __builtin_amdgcn_readfirstlane((i * NT + t) / BM);
            off[i] = (uint32_t)min((i * NT + t) % BM, last) * (uint32_t)so * 4u;
            sum[i] = lost[i] = 0.f;
        }
    }
    __device__ __forceinline__ void load_fast(Raw& x, int k0) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = k0 + 8 * g[i];
            const float* q = base + r * ld;
#pragma unroll
            for (int e = 0; e < 8; ++e, q += ld) {
                x.a[i][e] = *at_bytes(q, off[i]);
                x.s[i][e] = uniform_load(scale + r + e);
            }
        }
    }
    __device__ __forceinline__ void load(Raw& x, int k0) const {
        if (fast && k0 + 32 <= R) return load_fast(x, k0);
        const int u = anew(t);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = k0 + 8 * g[i];
            const float* const q = base + min((i * NT + u) % BM, last) * so;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x.a[i][e] = r + e < R ? q[(r + e) * ld] : 0.f;
                x.s[i][e] = r + e < R ? uniform_load(scale + r + e) : 0.f;
            }
        }
    }
    // (an infinite sum has lost what is no number)
    __device__ __forceinline__ float total(int i) const {
        return sum[i] + (lost[i] - lost[i] == 0.f ? lost[i] : 0.f);
    }
    __device__ __forceinline__ void store(const Raw& x, char* buf, bool live) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (SUM) {
                const float* const a = x.a[i];
                const float v = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
                const float u = live ? v : 0.f, s = sum[i] + u;
                lost[i] += u - (s - sum[i]);
                sum[i] = s;
            }
            float a[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = x.a[i][e] * x.s[i][e];
            u32x4 h, m, l;
            cut8<(BM > 64)>(a, h, m, l);
            char* const d = buf + g[i] * kGroup + (i * NT + t) % BM * 16;
            *reinterpret_cast<u32x4*>(d) = h;
            *reinterpret_cast<u32x4*>(d + kBytes) = m;
            *reinterpret_cast<u32x4*>(d + 2 * kBytes) = l;
        }
    }
};

// q: a thread takes four rows of four inputs (a dword each, at any byte's address),
// which change places in registers.  The entries of four neighbouring inputs lie
// in four runs, so that consecutive lanes write consecutive entries; the runs start 32
// bytes apart modulo 128, so that a fragment's rows fall on different banks.
// EDGE: a tile that reaches past the last input (four inputs or more in all).  Items there
// start early enough to end with the row, and are shifted back into place.
template <int BN, int NT, bool EDGE>
struct BackQ {
    static constexpr int N = BN * 2 / NT, kRun = BN / 4 + 2, kGroup = 4 * kRun * 16,
                         kBytes = 4 * kGroup;
    static_assert(N * NT == BN * 2, "whole items");
    static constexpr int kWork = N * 16 * 2, kReads = 0, kRaw = 0;
    static constexpr bool kBlock = false;
    struct Codes {};
    struct Raw {
        uint32_t q[N][4];
    };
    const int8_t* base;               // input n0, row 0
    uint32_t off[N];                  // of the item from its wave's first row on
    int64_t ld;
    int R, t, left, row[N];           // inputs from n0 on; the wave's first row in a chunk
    int shift[EDGE ? N : 1];          // of an edge item, in bits
    bool fast;                        // rows within 32 bits of bytes, and four inputs or more
    __device__ __forceinline__ static int entry(int c) { return (c & 3) * kRun + (c >> 2); }
    __device__ __forceinline__ BackQ(const BackParams& p, int n0, int t_)
        : base(p.q + n0), ld(p.q_r), R(p.R), t(t_), left(p.C - n0),
          fast(p.C >= 4 && p.q_r < (1 << 28)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = 4 * ((i * NT + t) / (BN / 4));
            row[i] = __builtin_amdgcn_readfirstlane(r);
            int c = (i * NT + t) % (BN / 4) * 4;
            if constexpr (EDGE) {                          // (inputs past C: anything, not stored)
                const int early = min(c, left - 4);
                shift[i] = 8 * (c - early) & 31;
                c = early;
            }
            off[i] = (uint32_t)c + (uint32_t)(r - row[i]) * (uint32_t)ld;
        }
    }
    __device__ __forceinline__ void load_fast(Raw& x, int k0) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int8_t* q = base + (k0 + row[i]) * ld;
#pragma unroll
            for (int e = 0; e < 4; ++e, q += ld) {
                if constexpr (EDGE)                        // (off may be negative)
                    x.q[i][e] = *reinterpret_cast<const row_codes*>(q + (int32_t)off[i]);
                else
                    x.q[i][e] = *reinterpret_cast<const row_codes*>(at_bytes(q, off[i]));
            }
        }
    }
    __device__ __forceinline__ void load(Raw& x, int k0) const {
        if (k0 + 32 <= R && fast) return load_fast(x, k0);
        const int u = anew(t);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = k0 + 4 * ((i * NT + u) / (BN / 4)), c = (i * NT + u) % (BN / 4) * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int8_t* const q = base + (r + e) * ld + c;
                uint32_t v = 0;
                if (r + e < R && c + 4 <= left) {
                    v = *reinterpret_cast<const row_codes*>(q);
                } else {
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (r + e < R && c + b < left) v |= (uint32_t)(uint8_t)q[b] << (8 * b);
                }
                x.q[i][e] = EDGE ? v << shift[i] : v;
            }
        }
    }
    __device__ __forceinline__ void store(const Raw& x, char* buf) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int v = i * NT + t, c4 = v % (BN / 4), kq = v / (BN / 4);
            char* const d = buf + (kq >> 1) * kGroup + c4 * 16 + (kq & 1) * 8;
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = EDGE ? x.q[i][e] >> shift[i] : x.q[i][e];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(w[e] >> (8 * b));
                *reinterpret_cast<u32x2*>(d + b * kRun * 16) =
                    u32x2{bf16_cut(f[0], f[1]), bf16_cut(f[2], f[3])};
            }
        }
    }
};

template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64, 2) back_dw(BackParams p) {
    constexpr int WAVES_N = BN / WN, NT = BM / WM * WAVES_N * 64;
    constexpr int MB = WM / 32, NB = WN / 32;
    using LA = BackDy<BM, NT, true>;
    using LB = BackQ<BN, NT, false>;
    __shared__ __attribute__((aligned(16))) char smem[2 * (3 * LA::kBytes + LB::kBytes)];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int ra = wave / WAVES_N * WM, rb = wave % WAVES_N * WN;
    const int tiles_m = (p.O + BM - 1) / BM, tiles_n = (p.C + BN - 1) / BN;
    const int split = blockIdx.x / (tiles_m * tiles_n);
    int im, in;
    lb_tile(blockIdx.x - split * tiles_m * tiles_n, tiles_m, tiles_n, im, in);
    const int m0 = im * BM, n0 = in * BN;
    const int rbeg = split * p.r_per_split, rend = min(p.R, rbeg + p.r_per_split);
    const bool part = p.splits > 1;
    f32x16 sum[MB][NB], acc[MB][NB];
    zero_blocks<MB, NB>(sum);
    auto multiply = [&](auto& la, auto lb) {
        lb_product<3, 4, BM == 64 ? 4 : 2, MB, NB>(
            la, lb, smem, rbeg, rend, ra, rb, lane, acc, [&](auto, int) {
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j)
#pragma unroll
                        for (int r = 0; r < 16; ++r) sum[i][j][r] += acc[i][j][r];
            });
    };
    auto product = [&](auto& la) {
        if (n0 + BN <= p.C) multiply(la, LB(p, n0, t));
        else multiply(la, BackQ<BN, NT, true>(p, n0, t));
    };
    if (p.db && in == 0) {
        LA la(p, m0, t);
        product(la);
        // the four groups of rows of each output
        float* const red = reinterpret_cast<float*>(smem);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LA::N; ++i) red[i * NT + t] = la.total(i);
        __syncthreads();
        if (t < BM && m0 + t < p.O) {
            const float v = (red[t] + red[BM + t]) + (red[2 * BM + t] + red[3 * BM + t]);
            if (part) {
                p.part_b[(int64_t)split * p.O + m0 + t] = v;
            } else {
                float* const d = p.db + (int64_t)(m0 + t) * p.db_stride;
                *d = p.beta_b != 0.f ? p.beta_b * *d + v : v;
            }
        }
    } else {
        BackDy<BM, NT, false> la(p, m0, t);
        product(la);
    }
    auto each = [&](auto put) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int n = n0 + rb + 32 * j + (lane & 31);
                if (n >= p.C) continue;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int m = m0 + ra + 32 * i + lb_row(lane, r);
                    float v = sum[i][j][r], old = acc[i][j][r];
                    if (m < p.O) put(m, n, v, old);
                    sum[i][j][r] = v;
                    acc[i][j][r] = old;
                }
            }
    };
    float* const out = part ? p.part + (int64_t)split * p.O * p.C : p.dw;
    const int64_t om = part ? p.C : p.dw_o, on = part ? 1 : p.dw_c;
    // (the old values first, all on their way at once: with loads and stores in turn 256 rows,
    // 2048 -> 1000, took 14.8 us, so 13.4)
    const float beta = part ? 0.f : p.beta;
    if (beta != 0.f) {
        each([&](int m, int n, float& v, float& old) { old = out[m * om + n * on]; });
        each([&](int m, int n, float& v, float& old) { v = beta * old + v; });
    }
    each([&](int m, int n, float& v, float&) { out[m * om + n * on] = v; });
}

}  // namespace mtk
