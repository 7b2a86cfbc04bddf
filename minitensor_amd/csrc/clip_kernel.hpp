// clip_kernel.hpp -- the norm of many tensors and their scaling (include/mtffn.h):
// norm = sqrt(sum of all squares), out = g * min(1, most / (norm + eps)).
//
// Bound by memory: every gradient is read for the norm and again to be scaled (138M elements:
// 91 us, 6.1 TB/s, and 201 us, 5.5 TB/s).  Squares of
// fp32 values are exact in fp64 and their sums are held there: nothing overflows, and a
// model's 10^9 squares lose nothing that fp32 would show.
//
// A launch takes a table of up to kClipTensors tensors in its arguments (half as many where
// they are scaled into others; no memory beside the workspace is written or read for it, so
// that a captured launch holds its own).  Dense
// tensors are cut into chunks; a workgroup takes a run of neighbouring chunks, and leaves
// one partial sum, all of which the scaling launch's workgroups add up again in the same
// order.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "row_access.hpp"

namespace mtk {

constexpr int kClipTensors = 256;     // of a launch: 14 bytes each of 4 KB of arguments
constexpr int kClipThreads = 512, kClipQuads = 4;
constexpr int kClipChunk = kClipThreads * kClipQuads * 4;   // elements
constexpr int kClipBlocks = 1024;     // workgroups of a launch, at most: four on a CU
constexpr int kClipMostParts = 4096;  // partial sums that every scaling workgroup adds up

struct ClipTable {
    float* at[kClipTensors];          // tensors, and their outputs from `to` on (0: themselves)
    uint32_t first[kClipTensors];     // chunk of the launch that the tensor starts with (past
                                      // the last tensor: the largest number)
    uint16_t last[kClipTensors];      // elements of its last chunk, less one
    int count, to;
    uint32_t chunks;
};
static_assert(kClipChunk <= 1 << 16, "a chunk's elements in 16 bits");
static_assert(sizeof(ClipTable) <= 3840, "kernel arguments");

// A tensor of any strides.
struct ClipStrided {
    const float* src;
    float* dst;
    int64_t size[3], src_stride[3], dst_stride[3];
};

struct ClipNorm {
    double* part;                     // [parts]
    int parts;
    float* norm;
    double most, eps;
};
// Gradients, in bytes, beyond which they and as many outputs do not stay in the 256 MB of the
// last cache: outputs are written past it then, and leave it to the gradients (138M elements,
// again and again: 288 us against 319).  Smaller ones stay there for whoever reads them next, not
// for the call's own sake, which written past the cache would take less (the same tensors again,
// three sets in turn; us: 38M elements 73 and 97, past it 67 and 82; 19M 35 and 45, 33 and 35).
constexpr int64_t kClipStream = (int64_t)160 << 20;

// The sum of x over a workgroup of NT, in every thread, in a fixed order.
template <int NT>
__device__ __forceinline__ double clip_block_sum(double x, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s += red[w];
    __syncthreads();
    return s;
}
// All partial sums together, the same in every workgroup.
template <int NT>
__device__ __forceinline__ double clip_total(const ClipNorm& c, double* red) {
    double s = 0;
    for (int i = threadIdx.x; i < c.parts; i += NT) s += c.part[i];
    return clip_block_sum<NT>(s, red);
}
// The factor; 1: nothing to scale.  (A NaN stays one; an infinite norm gives 0.)  It is held in
// fp64: gradients of 1e38 have one below fp32's normal range, where few digits of it are left,
// and a product that is well above it.
__device__ __forceinline__ double clip_factor(const ClipNorm& c, double total) {
    if (total == 0.0) return 1.0;
    const double f = c.most / (sqrt(total) + c.eps);
    return f >= 1.0 ? 1.0 : f;
}
__device__ __forceinline__ float clip_scaled(float x, double f) {
    asm("" : "+v"(x));                // (not its fp64 form of the squares, kept in two registers)
    return (float)((double)x * f);
}
__device__ __forceinline__ rowf4 clip_scaled(const rowf4& x, double f) {
    rowf4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = clip_scaled(x[e], f);
    return y;
}

// A workgroup's run of chunks, and what it takes of one at a time.
struct ClipRun {
    uint32_t begin, end;
};
__device__ __forceinline__ ClipRun clip_run(const ClipTable& t) {
    const uint32_t per = (t.chunks + gridDim.x - 1) / gridDim.x;
    const uint32_t begin = min(blockIdx.x * per, t.chunks);
    return {begin, min(begin + per, t.chunks)};
}
struct ClipPiece {
    const float* src;
    float* dst;
    int n;                            // elements, at most kClipChunk
};
// (the tensor of a chunk: one look at every tensor's first chunk, a lane four of them)
template <int CHUNK = kClipChunk>
__device__ __forceinline__ ClipPiece clip_piece(const ClipTable& t, uint32_t c) {
    int n = -1;
#pragma unroll
    for (int i = threadIdx.x & 63; i < kClipTensors; i += 64) n += __popcll(__ballot(t.first[i] <= c));
    const int k = __builtin_amdgcn_readfirstlane(n);
    const uint32_t end = k + 1 < t.count ? t.first[k + 1] : t.chunks;
    const int64_t at = (int64_t)(c - t.first[k]) * CHUNK;
    return {t.at[k] + at, t.at[k + t.to] + at, c + 1 == end ? t.last[k] + 1 : CHUNK};
}
// A thread's groups of four, zeros past the end, and (thread < n % 4) one of the last elements.
struct ClipValues {
    rowf4 x[kClipQuads];
    float last;
};
__device__ __forceinline__ void clip_load(const ClipPiece& p, ClipValues& v) {
    v.last = 0.f;
    if (p.n == kClipChunk) {
#pragma unroll
        for (int i = 0; i < kClipQuads; ++i)
            v.x[i] = *reinterpret_cast<const rowf4_u*>(p.src + 4 * (threadIdx.x + i * kClipThreads));
        return;
    }
    const int quads = p.n >> 2;
#pragma unroll
    for (int i = 0; i < kClipQuads; ++i) {
        const int q = threadIdx.x + i * kClipThreads;
        v.x[i] = rowf4{0.f, 0.f, 0.f, 0.f};
        if (q < quads) v.x[i] = *reinterpret_cast<const rowf4_u*>(p.src + 4 * q);
    }
    if ((int)threadIdx.x < (p.n & 3)) v.last = p.src[4 * quads + threadIdx.x];
}

__global__ void __launch_bounds__(kClipThreads) clip_squares(ClipTable t, double* part) {
    __shared__ double red[kClipThreads / 64];
    double s = 0;
    const ClipRun r = clip_run(t);
    ClipValues v, next;
    if (r.begin < r.end) clip_load(clip_piece(t, r.begin), v);
    for (uint32_t c = r.begin; c < r.end; ++c) {
        if (c + 1 < r.end) clip_load(clip_piece(t, c + 1), next);
#pragma unroll
        for (int i = 0; i < kClipQuads; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fma((double)v.x[i][e], (double)v.x[i][e], s);
        s = fma((double)v.last, (double)v.last, s);
        v = next;
    }
    s = clip_block_sum<kClipThreads>(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// From the last chunk to the first: what the squares read last is still in the cache.
// STREAM: outputs are written past the caches.
template <bool STREAM>
__global__ void __launch_bounds__(kClipThreads) clip_scale(ClipTable t, ClipNorm c) {
    __shared__ double red[kClipThreads / 64];
    const ClipRun r = clip_run(t);
    ClipPiece p{}, q{};
    ClipValues v, next;
    if (r.begin < r.end) {                            // (on its way while the sums are added up)
        p = clip_piece(t, r.end - 1);
        clip_load(p, v);
    }
    const double total = clip_total<kClipThreads>(c, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) *c.norm = (float)sqrt(total);
    const double f = clip_factor(c, total);
    for (uint32_t i = r.end; i > r.begin; --i) {
        if (i - 1 > r.begin) {
            q = clip_piece(t, i - 2);
            clip_load(q, next);
        }
        if (f != 1.0 || p.dst != p.src) {
            const int quads = p.n >> 2;
#pragma unroll
            for (int k = 0; k < kClipQuads; ++k) {
                const int at = threadIdx.x + k * kClipThreads;
                if (at >= quads) continue;
                rowf4_u* const d = reinterpret_cast<rowf4_u*>(p.dst + 4 * at);
                const rowf4 x = clip_scaled(v.x[k], f);
                if constexpr (STREAM) __builtin_nontemporal_store(x, d);
                else *d = x;
            }
            if ((int)threadIdx.x < (p.n & 3)) p.dst[4 * quads + threadIdx.x] = clip_scaled(v.last, f);
        }
        p = q;
        v = next;
    }
}

// The norm alone; or (norm nullptr) all partial sums as one, behind them.
__global__ void __launch_bounds__(kClipThreads) clip_norm(ClipNorm c) {
    __shared__ double red[kClipThreads / 64];
    const double total = clip_total<kClipThreads>(c, red);
    if (threadIdx.x != 0) return;
    if (c.norm) *c.norm = (float)sqrt(total);
    else c.part[c.parts] = total;
}

// Few elements, in one workgroup and one launch: a wave takes up to four chunks of 1024, all
// on their way at once, and holds them until the norm is there.  (Calls, one after another:
// 12288 elements 5.0 us, by two launches 8.8; 50432 7.3 and 9.0; 64000 in 64 tensors 8.9 and 11.7;
// more would not stay in registers.)
constexpr int kClipOneWaves = 16, kClipOnePieces = 4, kClipOneChunk = 1024;
template <int = 0>
__global__ void __launch_bounds__(64 * kClipOneWaves) clip_one(ClipTable t, ClipNorm c, int scale) {
    __shared__ double red[kClipOneWaves];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    ClipPiece p[kClipOnePieces];
    rowf4 x[kClipOnePieces][4];
    float last[kClipOnePieces];
#pragma unroll
    for (int i = 0; i < kClipOnePieces; ++i) {
        const uint32_t id = wave + kClipOneWaves * i;
        p[i] = ClipPiece{nullptr, nullptr, 0};
        if (id < t.chunks) p[i] = clip_piece<kClipOneChunk>(t, id);
        const int quads = p[i].n >> 2;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = lane + 64 * q;
            x[i][q] = rowf4{0.f, 0.f, 0.f, 0.f};
            if (at < quads) x[i][q] = *reinterpret_cast<const rowf4_u*>(p[i].src + 4 * at);
        }
        last[i] = lane < (p[i].n & 3) ? p[i].src[4 * quads + lane] : 0.f;
    }
    double s = 0;
#pragma unroll
    for (int i = 0; i < kClipOnePieces; ++i) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fma((double)x[i][q][e], (double)x[i][q][e], s);
        s = fma((double)last[i], (double)last[i], s);
    }
    const double total = clip_block_sum<64 * kClipOneWaves>(s, red);
    if (threadIdx.x == 0) *c.norm = (float)sqrt(total);
    if (!scale) return;
    const double f = clip_factor(c, total);
#pragma unroll
    for (int i = 0; i < kClipOnePieces; ++i) {
        if (f == 1.0 && p[i].dst == p[i].src) continue;
        const int quads = p[i].n >> 2;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (lane + 64 * q < quads)
                *reinterpret_cast<rowf4_u*>(p[i].dst + 4 * (lane + 64 * q)) = clip_scaled(x[i][q], f);
        if (lane < (p[i].n & 3)) p[i].dst[4 * quads + lane] = clip_scaled(last[i], f);
    }
}

template <class F>
__device__ __forceinline__ void clip_elements(const ClipStrided& t, F f) {
    const int64_t inner = t.size[2], rows = t.size[1], n = t.size[0] * rows * inner;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / inner, c = i - r * inner, b = r / rows, y = r - b * rows;
        f(b * t.src_stride[0] + y * t.src_stride[1] + c * t.src_stride[2],
          b * t.dst_stride[0] + y * t.dst_stride[1] + c * t.dst_stride[2]);
    }
}
__global__ void __launch_bounds__(256) clip_squares_strided(ClipStrided t, double* part) {
    __shared__ double red[4];
    double s = 0;
    clip_elements(t, [&](int64_t a, int64_t) {
        const double x = t.src[a];
        s = fma(x, x, s);
    });
    s = clip_block_sum<256>(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}
__global__ void __launch_bounds__(256) clip_scale_strided(ClipStrided t, ClipNorm c) {
    __shared__ double red[4];
    const double total = clip_total<256>(c, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) *c.norm = (float)sqrt(total);
    const double f = clip_factor(c, total);
    if (f == 1.0 && t.dst == t.src) return;
    clip_elements(t, [&](int64_t a, int64_t b) { t.dst[b] = clip_scaled(t.src[a], f); });
}

}  // namespace mtk
