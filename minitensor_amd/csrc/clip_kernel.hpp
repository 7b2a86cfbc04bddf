// clip_kernel.hpp -- the norm of many tensors and their scaling (include/mtffn.h):
// norm = sqrt(sum of all squares), out = g * min(1, most / (norm + eps)).
//
// Bound by memory: every gradient is read for the norm and again to be scaled.  Squares of
// fp32 values are exact in fp64 and their sums are held there: nothing overflows, and a
// model's 10^9 squares lose nothing that fp32 would show.
//
// A launch takes a table of up to kClipTensors tensors in its arguments (no memory beside the
// workspace is written or read for it, so that a captured launch holds its own).  Dense
// tensors are cut into chunks; a workgroup takes a run of neighbouring chunks, and leaves
// one partial sum, all of which the scaling launch's workgroups add up again in the same
// order.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "row_access.hpp"

namespace mtk {

constexpr int kClipTensors = 128;     // of a launch: 28 bytes each of 4 KB of arguments
constexpr int kClipChunk = 8192;      // elements
constexpr int kClipBlocks = 1024;     // workgroups of a launch, at most
constexpr int kClipPartials = 1 << 20;  // of a call (so that their count stays 32-bit)

struct ClipTable {
    const float* src[kClipTensors];
    float* dst[kClipTensors];
    int64_t n[kClipTensors];
    uint32_t first[kClipTensors];     // chunk of the launch that the tensor starts with
    int count;
    uint32_t chunks;
};
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

// The sum of x over a workgroup of 256, in every thread.
__device__ __forceinline__ double clip_block_sum(double x, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    const double s = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return s;
}
// All partial sums together.
__device__ __forceinline__ double clip_total(const ClipNorm& c, double* red) {
    double s = 0;
    for (int i = threadIdx.x; i < c.parts; i += 256) s += c.part[i];
    return clip_block_sum(s, red);
}
// The factor; 1: nothing to scale.  (A NaN stays one; an infinite norm gives 0.)
__device__ __forceinline__ float clip_factor(const ClipNorm& c, double total) {
    const double f = c.most / (sqrt(total) + c.eps);
    return f >= 1.0 ? 1.f : (float)f;
}

// Calls f(tensor, first element, elements) for the workgroup's chunks.
template <class F>
__device__ __forceinline__ void clip_chunks(const ClipTable& t, F f) {
    const uint32_t per = (t.chunks + gridDim.x - 1) / gridDim.x;
    uint32_t c = blockIdx.x * per;
    const uint32_t end = min(c + per, t.chunks);
    if (c >= end) return;
    int lo = 0, hi = t.count;                         // the tensor of chunk c
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    for (; c < end; ++c) {
        while (lo + 1 < t.count && t.first[lo + 1] <= c) ++lo;
        const int64_t at = (int64_t)(c - t.first[lo]) * kClipChunk;
        f(lo, at, (int)min(t.n[lo] - at, (int64_t)kClipChunk));
    }
}

__global__ void __launch_bounds__(256) clip_squares(ClipTable t, double* part) {
    __shared__ double red[4];
    double s = 0;
    clip_chunks(t, [&](int k, int64_t at, int n) {
        const float* const g = t.src[k] + at;
        const int quads = n >> 2;
        for (int i = threadIdx.x; i < quads; i += 256) {
            const rowf4 x = *reinterpret_cast<const rowf4_u*>(g + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fma((double)x[e], (double)x[e], s);
        }
        const int e = 4 * quads + threadIdx.x;
        if (e < n) s = fma((double)g[e], (double)g[e], s);
    });
    s = clip_block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ void __launch_bounds__(256) clip_scale(ClipTable t, ClipNorm c) {
    __shared__ double red[4];
    const double total = clip_total(c, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) *c.norm = (float)sqrt(total);
    const float f = clip_factor(c, total);
    clip_chunks(t, [&](int k, int64_t at, int n) {
        const float* const g = t.src[k] + at;
        float* const o = t.dst[k] + at;
        if (f == 1.f && o == g) return;
        const int quads = n >> 2;
        for (int i = threadIdx.x; i < quads; i += 256)
            *reinterpret_cast<rowf4_u*>(o + 4 * i) = *reinterpret_cast<const rowf4_u*>(g + 4 * i) * f;
        const int e = 4 * quads + threadIdx.x;
        if (e < n) o[e] = g[e] * f;
    });
}

// The norm alone.
__global__ void __launch_bounds__(256) clip_norm(ClipNorm c) {
    __shared__ double red[4];
    const double total = clip_total(c, red);
    if (threadIdx.x == 0) *c.norm = (float)sqrt(total);
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
    s = clip_block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}
__global__ void __launch_bounds__(256) clip_scale_strided(ClipStrided t, ClipNorm c) {
    __shared__ double red[4];
    const double total = clip_total(c, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) *c.norm = (float)sqrt(total);
    const float f = clip_factor(c, total);
    if (f == 1.f && t.dst == t.src) return;
    clip_elements(t, [&](int64_t a, int64_t b) { t.dst[b] = t.src[a] * f; });
}

}  // namespace mtk
