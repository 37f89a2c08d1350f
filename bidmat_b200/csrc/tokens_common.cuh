// Shared by the operators between dense token columns and sparse matrices (route.cu, top_logits.cu,
// distill.cu): element types, order keys of floats, block-wide sums and the host-side checks.
//
// A dense matrix is column-major with a leading dimension ld >= nrows in elements: one token per column.
// Elements are fp32, bf16 or fp16; everything is computed in 32 bits or more and rounded once on the way out.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/bidmat_b200.h"
#include "host_common.cuh"
#include "workspace.cuh"

namespace bidmat {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Whole numbers in the order of the floats: NaN above everything, the two zeros equal.
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    if (x != x) return 0xffffffffu;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned key) {
    if (key == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The larger one, NaN if either is.
__device__ __forceinline__ double max_nan(double a, double b) { return (a > b || a != a) ? a : b; }
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// ------------------------------------------------------------------ host side
// Rows, columns and entries are counted in ints, with room for the steps of a loop.
constexpr int kMostRows = 0x7fff0000, kMostEntries = 0x7fff0000;

// How many CTAs fill the machine is counted in its SMs: this library is built for one part.
constexpr int kSMs = 148;

inline size_t dtype_size(int dtype) { return dtype == BIDMAT_B200_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == BIDMAT_B200_F32 || dtype == BIDMAT_B200_BF16 || dtype == BIDMAT_B200_F16; }

// Finite, positive and not subnormal, so that 1.44 / temperature is a number.
inline bool temperature_ok(float t) { return isfinite(t) && t >= 1.17549435e-38f; }

// A dense operand: its leading dimension covers the rows, its address is aligned to its elements.
inline bool dense_ok(const void *p, long long ld, int nrows, int dtype) {
    return p && ld >= nrows && (reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) == 0;
}

// Dynamic shared memory above the 48 KB that every kernel may have: the kernel is allowed the most that any call asks for, not
// what this one does, so that calls from two host threads do not take it away from one another.
template <typename K> inline cudaError_t allow_shared(K kernel, size_t bytes, size_t most) {
    if (bytes <= 40000) return cudaSuccess;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
}

#define DISPATCH_DTYPE(DT, CALL)                                   \
    do {                                                           \
        if ((DT) == BIDMAT_B200_F32) { CALL(float); }              \
        else if ((DT) == BIDMAT_B200_BF16) { CALL(__nv_bfloat16); } \
        else { CALL(__half); }                                     \
    } while (0)

}  // namespace bidmat
