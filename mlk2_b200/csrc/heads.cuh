// Strided [rows, heads, d] operands of the norm_rope and attention entries:
// 16-bit elements, the last dimension contiguous.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstdio>
#include <type_traits>

#include "common.cuh"

namespace mlkb {

constexpr int64_t kMaxHeadRows = int64_t(1) << 30;  // row indices and their tile ends stay in int32

// Checks one operand and normalises it into *v: the stride of a dimension
// with one entry is never used and may hold anything. An output's rows and
// heads may not overlap one another.
inline int checkHeads(const mlkb_heads* t, int64_t heads, int64_t d, bool output, const char* what,
                      mlkb_heads* v) {
    const char* why = nullptr;
    if (t == nullptr) {
        why = "null descriptor";
    } else {
        *v = *t;
        constexpr int64_t kMaxStride = int64_t(1) << 38;
        if (v->rows < 0 || v->rows > kMaxHeadRows) {
            why = "rows must be 0 to 2^30";
        } else if (v->rows > 0 && v->data == nullptr) {
            why = "null buffer";
        } else if (!aligned16(v->data)) {
            why = "buffer must be 16-byte aligned";
        } else {
            if (heads == 1) v->head_stride = (d + 7) / 8 * 8;
            if (v->rows <= 1) v->row_stride = heads * v->head_stride;
            if (v->head_stride <= 0 || v->row_stride <= 0 || v->head_stride % 8 != 0 ||
                v->row_stride % 8 != 0 || v->head_stride > kMaxStride || v->row_stride > kMaxStride) {
                why = "strides must be positive multiples of 8 elements";
            } else if (output) {
                const bool rowMajor = v->head_stride >= d &&
                                      v->row_stride >= (heads - 1) * v->head_stride + d;
                const bool headMajor = v->row_stride >= d &&
                                       v->head_stride >= (v->rows - 1) * v->row_stride + d;
                if (!rowMajor && !headMajor) why = "output rows overlap";
            }
        }
    }
    if (why == nullptr) return MLKB_OK;
    char msg[128];
    std::snprintf(msg, sizeof msg, "%s: %s", what, why);
    return setError(MLKB_ERR_INVALID, msg);
}

// Whether two operands have an element in common at their start. (Views may lie
// between one another's rows, so addresses alone show no other overlap.)
inline bool sameStart(const mlkb_heads& a, const mlkb_heads& b) {
    return a.rows > 0 && b.rows > 0 && a.data == b.data;
}

// MLKB_ERR_NO_DEVICE where no CUDA device can be used.
inline int needDevice() {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) return MLKB_OK;
    cudaGetLastError();
    return setCudaError(MLKB_ERR_NO_DEVICE, e, "no CUDA device");
}

// ---- 16-bit element conversions (T = __half or __nv_bfloat16) ----------------------
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
        return __half22float2(*reinterpret_cast<const __half2*>(&u));
    } else {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
    }
}

// Two values rounded to nearest even, `lo` in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t u;
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(lo, hi);
        u = *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        u = *reinterpret_cast<const uint32_t*>(&h);
    }
    return u;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

}  // namespace mlkb
