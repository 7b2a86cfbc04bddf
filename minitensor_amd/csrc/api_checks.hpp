// api_checks.hpp -- what the entry points of include/mtlowbit.h and include/mtffn.h check
// and share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "row_access.hpp"
#include "mtlowbit.h"

namespace mtk {

// Extents are 32-bit inside the kernels, and blocks past an end stay below 2^31.
inline constexpr int64_t kMaxDim = ((int64_t)1 << 31) - (1 << 16);
inline constexpr int kCus = 256;                       // what plans fill (MI355X)
inline constexpr int64_t kMaxTiles = (int64_t)1 << 23; // of 512 threads: a grid's threads are a 32-bit number

inline int launched() {
    // (as mt_gemm_f32: a launch recorded by a stream capture reports this)
    const hipError_t e = hipGetLastError();
    return e == hipSuccess || e == hipErrorStreamCaptureUnsupported ? MT_OK : MT_ERR_HIP;
}

// A 2-D fp32 view; written: no two elements on one address.
inline bool valid(const mt_mat_f32* X, bool written) {
    if (!X || X->batch != 1 || X->rows < 0 || X->cols < 0 || X->row_stride < 0 ||
        X->col_stride < 0 || X->offset < 0 || X->rows >= kMaxDim || X->cols >= kMaxDim)
        return false;
    if (X->rows == 0 || X->cols == 0) return true;
    if (!X->base) return false;
    return !written || ((X->rows <= 1 || X->row_stride > 0) && (X->cols <= 1 || X->col_stride > 0));
}
inline bool same_shape(const mt_mat_f32* A, const mt_mat_f32* B) {
    return A->rows == B->rows && A->cols == B->cols;
}
inline bool valid(const mt_rows_q8* Q) {
    if (!Q || Q->rows < 0 || Q->cols < 0 || Q->rows >= kMaxDim || Q->cols >= kMaxDim ||
        Q->row_stride < 0 || (Q->rows > 1 && Q->row_stride < Q->cols))
        return false;
    return Q->rows == 0 || (Q->scale && (Q->cols == 0 || Q->q));
}
inline RowView view(const mt_mat_f32* X) {
    if (!X) return {nullptr, 0, 0};
    return {const_cast<float*>(X->base) + X->offset, X->row_stride, X->col_stride};
}
// Rows whose elements are neighbours (or absent).
inline bool unit(const RowView& v) { return !v.p || v.cs == 1; }

}  // namespace mtk
