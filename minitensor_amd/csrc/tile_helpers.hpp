// tile_helpers.hpp -- what the tiled products of the language models' operators share: the
// order of tiles, a barrier for LDS, and ways to keep values where they belong.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mtk {

// Keeps the compiler from taking a packed value apart again (it rounded the low half a second
// time rather than shift it: two instructions more per pair).
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
    asm("" : "+v"(v));
    return v;
}

// p moved on by a 32-bit number of bytes: one register beside a uniform p (the compiler
// kept the number's 64 bits through the loop).
template <class T>
__device__ __forceinline__ const T* at_bytes(const T* p, uint32_t bytes) {
    asm volatile("" : "+v"(bytes));
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + bytes);
}

// The value anew, for a path beside the loop: not kept in registers through it.
__device__ __forceinline__ int anew(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// A barrier that orders LDS alone.
__device__ __forceinline__ void lb_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
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

}  // namespace mtk
