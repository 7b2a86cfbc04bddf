// lowbit_rows_kernel.hpp -- kernels that take rows one at a time: RMS norm with
// the residual's addition and rows in 8 bits, its gradients, rows put away in 8
// bits and read back (include/mtlowbit.h).
//
// All are bound by memory: 9 to 17 bytes per element against some ten flops.
// A row is held in registers between the passes that it needs (sum of squares,
// largest magnitude, outputs), so that each operand is read once: NT threads
// per row, 16 values each; 64 threads (four rows per workgroup) up to 1024
// columns, 256 up to 4096, 1024 up to 16384.  Longer rows are read again for
// each pass (RES = false), from L2.
//
// MODE: R_VEC, rows whose elements are neighbours, four at a time with 16-byte
// accesses at any element's address (8-bit rows 4 bytes at any byte's), the
// width a multiple of four; R_TAIL, the same at any width, the last elements one
// by one; R_STRIDED, single elements at any strides (read again for each pass,
// since sixteen 64-bit offsets per operand would not stay in registers).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace mtk {

constexpr int kRowVals = 16;          // values of a row per thread
constexpr float kQ8Inv = 1.f / 127.f;
constexpr float kScaleMin = 0x1p-126f;

typedef float rowf4 __attribute__((ext_vector_type(4)));

struct RowView {                      // fp32 rows (base nullptr: none)
    float* p;
    int64_t rs, cs;
};

struct RowParams {
    RowView x, r, h, y;               // forward: inputs x, r; outputs h, y
    const float* w;                   // nullptr: ones
    int64_t ws;
    int8_t* q;                        // nullptr: none
    int64_t qs;
    float* scale;
    float* rstd;                      // nullptr: none
    float eps;
    int64_t rows;
    int cols;
};

struct RowBwdParams {
    RowView dy, h, dh0, dh;
    const float* w;
    int64_t ws;
    const float* rstd;
    float* part;                      // [workgroup][row group][cols] of dweight, or nullptr
    int64_t rows;
    int cols;
    int row_step;                     // rows between a row group's consecutive rows
};

enum { R_STRIDED = 0, R_TAIL = 1, R_VEC = 2 };

typedef rowf4 rowf4_u __attribute__((aligned(4)));
typedef uint32_t row_codes __attribute__((aligned(1)));

// What a thread takes at a time: four elements of row r from column c, or one.
template <int MODE>
using RowV = std::conditional_t<MODE == R_STRIDED, float, rowf4>;

template <int MODE>
__device__ __forceinline__ RowV<MODE> run_load(const float* p, int64_t cs, int c, int cols) {
    if constexpr (MODE == R_STRIDED) return p[(int64_t)c * cs];
    else if (MODE == R_VEC || c + 4 <= cols) return *reinterpret_cast<const rowf4_u*>(p + c);
    else {
        rowf4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (c + e < cols) x[e] = p[c + e];
        return x;
    }
}
template <int MODE>
__device__ __forceinline__ RowV<MODE> row_load(const RowView& v, int64_t r, int c, int cols) {
    return run_load<MODE>(v.p + r * v.rs, v.cs, c, cols);
}
template <int MODE>
__device__ __forceinline__ void row_store(const RowView& v, int64_t r, int c, int cols,
                                          const RowV<MODE>& x) {
    float* const p = v.p + r * v.rs;
    if constexpr (MODE == R_STRIDED) p[(int64_t)c * v.cs] = x;
    else if (MODE == R_VEC || c + 4 <= cols) *reinterpret_cast<rowf4_u*>(p + c) = x;
    else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (c + e < cols) p[c + e] = x[e];
    }
}
template <int MODE>
__device__ __forceinline__ RowV<MODE> weight_load(const float* w, int64_t ws, int c, int cols) {
    if (w) return run_load<MODE>(w, ws, c, cols);
    if constexpr (MODE == R_STRIDED) return 1.f;
    else return rowf4{1.f, 1.f, 1.f, 1.f};
}
__device__ __forceinline__ float row_dot(const rowf4& a, const rowf4& b) {
    return (a[0] * b[0] + a[1] * b[1]) + (a[2] * b[2] + a[3] * b[3]);
}
__device__ __forceinline__ float row_dot(float a, float b) { return a * b; }
__device__ __forceinline__ float row_at(const rowf4& a, int e) { return a[e]; }
__device__ __forceinline__ float row_at(float a, int) { return a; }

// The code of x at 1/scale = inv: to the nearest, ties to even; zero where the
// row's scale is no number.
__device__ __forceinline__ int q8_code(float x, float inv) {
    const float v = __builtin_rintf(x * inv);
    return v == v ? (int)v : 0;
}

// Sum, and largest unsigned value, over the NT threads of a row, the same in
// every one: a butterfly in the wave, then the waves in order through LDS.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if constexpr (NT > 64) {
        __syncthreads();              // the readers of the last use are done
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < NT / 64; ++i) v += red[i];
    }
    return v;
}
template <int NT>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    if constexpr (NT > 64) {
        uint32_t* const r = reinterpret_cast<uint32_t*>(red);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
        __syncthreads();
        v = r[0];
#pragma unroll
        for (int i = 1; i < NT / 64; ++i) v = max(v, r[i]);
    }
    return v;
}

// Largest magnitude as bits: NaN above infinity above every number, so that a
// NaN is not lost.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// NORM: RMS norm; otherwise y = x (rows put away in 8 bits).  8192 x 2048 with a
// residual, fp32 and 8-bit rows out: 48 us for 285 MB; 1 x 4096: 4.0 us, the sums'
// latency; 8192 x 4096 put away: 28-34 us.
template <int NT, int MODE, bool RES, bool NORM>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) rows_forward(RowParams p) {
    using T = RowV<MODE>;
    constexpr int V = MODE == R_STRIDED ? 1 : 4;
    constexpr int NI = RES ? kRowVals / V : 1;
    constexpr int G = NT < 256 ? 256 / NT : 1;         // rows per workgroup
    __shared__ float red[NT > 64 ? NT / 64 : 1];
    const int t = threadIdx.x % NT;
    // (a workgroup's rows go in step: NT is 64, with no barrier, or G is 1)
    for (int64_t r = (int64_t)blockIdx.x * G + threadIdx.x / NT; r < p.rows;
         r += (int64_t)gridDim.x * G) {
        auto h_at = [&](int c) {
            T v = row_load<MODE>(p.x, r, c, p.cols);
            if (NORM && p.r.p) v += row_load<MODE>(p.r, r, c, p.cols);
            return v;
        };
        T v[NI];
        float rstd = 1.f;
        if constexpr (RES) {
            // all loads in flight before the first use
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = (i * NT + t) * V;
                v[i] = c < p.cols ? row_load<MODE>(p.x, r, c, p.cols) : T{};
            }
            if (NORM && p.r.p) {
                T a[NI];
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int c = (i * NT + t) * V;
                    a[i] = c < p.cols ? row_load<MODE>(p.r, r, c, p.cols) : T{};
                }
#pragma unroll
                for (int i = 0; i < NI; ++i) v[i] += a[i];
            }
        }
        if constexpr (NORM) {
            float s = 0.f;
            auto add = [&](const T& a) { s += row_dot(a, a); };
            if constexpr (RES) {
#pragma unroll
                for (int i = 0; i < NI; ++i) add(v[i]);
            } else {
                for (int c = t * V; c < p.cols; c += NT * V) add(h_at(c));
            }
            rstd = 1.f / __builtin_sqrtf(row_sum<NT>(s, red) / (float)p.cols + p.eps);
            if (p.rstd && t == 0) p.rstd[r] = rstd;
        }
        auto y_of = [&](const T& h, int c) -> T {
            if constexpr (!NORM) return h;
            else return (h * rstd) * weight_load<MODE>(p.w, p.ws, c, p.cols);
        };
        float inv = 0.f;
        auto set_scale = [&](uint32_t m) {
            float s = __uint_as_float(row_max<NT>(m, red)) * kQ8Inv;
            s = s < kScaleMin ? kScaleMin : s;             // (a NaN stays)
            inv = 1.f / s;
            if (t == 0) p.scale[r] = s;
        };
        auto mag = [](uint32_t m, const T& a) {
#pragma unroll
            for (int e = 0; e < V; ++e) m = max(m, magnitude(row_at(a, e)));
            return m;
        };
        auto put_q = [&](const T& a, int c) {
            int8_t* const d = p.q + r * p.qs + c;
            if constexpr (MODE == R_STRIDED) {
                *d = (int8_t)q8_code(a, inv);
            } else if (MODE == R_VEC || c + 4 <= p.cols) {
                uint32_t b = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) b |= ((uint32_t)q8_code(a[e], inv) & 0xffu) << (8 * e);
                *reinterpret_cast<row_codes*>(d) = b;
            } else {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (c + e < p.cols) d[e] = (int8_t)q8_code(a[e], inv);
            }
        };
        if constexpr (RES) {
            if (NORM && p.h.p) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int c = (i * NT + t) * V;
                    if (c < p.cols) row_store<MODE>(p.h, r, c, p.cols, v[i]);
                }
            }
            if constexpr (NORM) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int c = (i * NT + t) * V;
                    if (c >= p.cols) continue;
                    v[i] = y_of(v[i], c);
                    if (p.y.p) row_store<MODE>(p.y, r, c, p.cols, v[i]);
                }
            }
            if (!p.q) continue;                            // (uniform)
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if ((i * NT + t) * V < p.cols) m = mag(m, v[i]);
            set_scale(m);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = (i * NT + t) * V;
                if (c < p.cols) put_q(v[i], c);
            }
        } else {
            if (p.q) {
                uint32_t m = 0;
                for (int c = t * V; c < p.cols; c += NT * V) m = mag(m, y_of(h_at(c), c));
                set_scale(m);
            }
            // h last, element by element after its reads: it may lie over x or r
            for (int c = t * V; c < p.cols; c += NT * V) {
                const T h = h_at(c), y = y_of(h, c);
                if (NORM && p.h.p) row_store<MODE>(p.h, r, c, p.cols, h);
                if (NORM && p.y.p) row_store<MODE>(p.y, r, c, p.cols, y);
                if (p.q) put_q(y, c);
            }
        }
    }
}

// Gradients.  A row group of NT threads walks rows row_step apart and keeps its
// part of dweight in registers (in its row of p.part where RES is false);
// the parts are summed by a launch of their own, in order.  8192 x 2048 with a
// gradient that joins: 52 us for 268 MB, and 5 for the parts.
template <int NT, int MODE, bool RES>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) rms_backward(RowBwdParams p) {
    using T = RowV<MODE>;
    constexpr int V = MODE == R_STRIDED ? 1 : 4;
    constexpr int NI = RES ? kRowVals / V : 1;
    constexpr int G = NT < 256 ? 256 / NT : 1;
    __shared__ float red[NT > 64 ? NT / 64 : 1];
    const int t = threadIdx.x % NT;
    const int64_t grp = (int64_t)blockIdx.x * G + threadIdx.x / NT;
    float* const part = p.part ? p.part + grp * p.cols : nullptr;
    const T zero{};
    T dw[NI], w[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        dw[i] = zero;
        const int c = (i * NT + t) * V;
        if constexpr (RES) w[i] = c < p.cols ? weight_load<MODE>(p.w, p.ws, c, p.cols) : zero;
    }
    bool first = true;
    for (int64_t r = grp; r < p.rows; r += p.row_step, first = false) {
        const float rstd = p.rstd[r];
        if constexpr (RES) {
            T g[NI], xh[NI];
            float s = 0.f;
            // (the next row's loads ahead of this one's sums cost a wave of the four: 61 us
            // against 50 for 8192 x 2048)
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = (i * NT + t) * V;
                g[i] = c < p.cols ? row_load<MODE>(p.dy, r, c, p.cols) : zero;
                xh[i] = (c < p.cols ? row_load<MODE>(p.h, r, c, p.cols) : zero) * rstd;
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                dw[i] += g[i] * xh[i];
                g[i] = g[i] * w[i];
                s += row_dot(g[i], xh[i]);
            }
            if (!p.dh.p) continue;                     // (uniform)
            const float mean = row_sum<NT>(s, red) / (float)p.cols;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int c = (i * NT + t) * V;
                if (c >= p.cols) continue;
                T d = rstd * (g[i] - xh[i] * mean);
                if (p.dh0.p) d += row_load<MODE>(p.dh0, r, c, p.cols);
                row_store<MODE>(p.dh, r, c, p.cols, d);
            }
        } else {
            float s = 0.f;
            for (int c = t * V; c < p.cols; c += NT * V) {
                const T dy = row_load<MODE>(p.dy, r, c, p.cols), xh = row_load<MODE>(p.h, r, c, p.cols) * rstd;
                s += row_dot(dy * weight_load<MODE>(p.w, p.ws, c, p.cols), xh);
                if (!part) continue;
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (c + e < p.cols)
                        part[c + e] = (first ? 0.f : part[c + e]) + row_at(dy, e) * row_at(xh, e);
            }
            if (!p.dh.p) continue;
            const float mean = row_sum<NT>(s, red) / (float)p.cols;
            for (int c = t * V; c < p.cols; c += NT * V) {
                const T xh = row_load<MODE>(p.h, r, c, p.cols) * rstd;
                T d = rstd * (row_load<MODE>(p.dy, r, c, p.cols) * weight_load<MODE>(p.w, p.ws, c, p.cols) - xh * mean);
                if (p.dh0.p) d += row_load<MODE>(p.dh0, r, c, p.cols);
                row_store<MODE>(p.dh, r, c, p.cols, d);
            }
        }
    }
    if (!part) return;
    if constexpr (RES) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = (i * NT + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e < p.cols) part[c + e] = row_at(dw[i], e);
        }
    } else if (first) {                                // a group without rows
        for (int c = t; c < p.cols; c += NT) part[c] = 0.f;
    }
}

// out[c] = beta*out[c] + sum over n parts, in order within each of 64 slices and then over
// the slices: 16 columns per workgroup of 1024 threads at a time.  (64 columns and 16 slices
// left most CUs without work: 5.4 us for 1024 parts of 2048.)
__global__ void __launch_bounds__(1024)
rms_dweight_sum(const float* part, int n, int cols, float* out, int64_t os, float beta) {
    __shared__ float red[64][17];
    const int l = threadIdx.x & 15, q = threadIdx.x >> 4;
    for (int64_t c0 = (int64_t)blockIdx.x * 16; c0 < cols; c0 += (int64_t)gridDim.x * 16) {
        const int64_t c = c0 + l;
        float s = 0.f;
        if (c < cols) {
#pragma unroll 8
            for (int i = q; i < n; i += 64) s += part[(int64_t)i * cols + c];
        }
        __syncthreads();                               // the readers of the columns before are done
        red[q][l] = s;
        __syncthreads();
        if (q >= 4 || c >= cols) continue;             // (one wave)
        for (int i = q + 4; i < 64; i += 4) s += red[i][l];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (q != 0) continue;
        float* const d = out + c * os;
        *d = beta != 0.f ? beta * *d + s : s;
    }
}

// y = q·scale.  UNIT: a wave takes 1024 elements of a row, four dwords of codes per lane,
// each load and store over neighbouring lanes' bytes (16 codes per lane, stored as four
// pieces 64 bytes apart, took 42 us for 8192 x 4096 where these take 26); otherwise single
// elements at any strides.
template <bool UNIT>
__global__ void __launch_bounds__(256)
dequantize_q8(const int8_t* q, int64_t qs, const float* scale, RowView y, int64_t rows, int cols) {
    if constexpr (UNIT) {
        const int lane = threadIdx.x & 63;
        const int64_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
        const int segs = (cols + 1023) >> 10;
        const int64_t n = rows * segs, step = (int64_t)gridDim.x * 4;
        for (int64_t i = wave; i < n; i += step) {
            const int64_t r = i / segs;
            const int c0 = (int)(i - r * segs) * 1024 + 4 * lane;
            const int8_t* const src = q + r * qs;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = c0 + 256 * j;
                w[j] = 0;
                if (c + 4 <= cols) {
                    w[j] = *reinterpret_cast<const row_codes*>(src + c);
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (c + e < cols) w[j] |= (uint32_t)(uint8_t)src[c + e] << (8 * e);
                }
            }
            const float s = scale[r];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = c0 + 256 * j;
                rowf4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = (float)(int8_t)(w[j] >> (8 * e)) * s;
                if (c < cols) row_store<R_TAIL>(y, r, c, cols, o);
            }
        }
    } else {
        const int64_t n = rows * cols;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n;
             i += (int64_t)gridDim.x * 256) {
            const int64_t r = i / cols;
            const int c = (int)(i - r * cols);
            y.p[r * y.rs + (int64_t)c * y.cs] = (float)q[r * qs + c] * scale[r];
        }
    }
}

}  // namespace mtk
