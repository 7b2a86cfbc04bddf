// row_access.hpp -- rows of fp32 and what a thread takes of one at a time.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace mtk {

typedef float rowf4 __attribute__((ext_vector_type(4)));

struct RowView {                      // fp32 rows (base nullptr: none)
    float* p;
    int64_t rs, cs;
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

// Four neighbouring columns n.. of row m, those before `end`.
__device__ __forceinline__ void put4(const RowView& v, int64_t m, int64_t n, int64_t end,
                                        const rowf4& x) {
    float* const d = v.p + m * v.rs + n * v.cs;
    if (v.cs == 1 && n + 4 <= end) {
        *reinterpret_cast<rowf4_u*>(d) = x;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < end) d[e * v.cs] = x[e];
    }
}

}  // namespace mtk
