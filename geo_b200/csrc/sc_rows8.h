// Element types and reductions shared by the row operators on 8-bit integers and by the distillation loss.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sc_common.h"

namespace geo {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// N values of T as one load or store (N * sizeof(T) is 16, 8 or 4 bytes, or N = 1).
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T v[N]; };

template <typename T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
    return *reinterpret_cast<const Pack<T, N> *>(p);
}
template <typename T, int N> __device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &v) {
    *reinterpret_cast<Pack<T, N> *>(p) = v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

inline bool dtype_known(int dtype) { return dtype == GEO_SC_DTYPE_F32 || dtype == GEO_SC_DTYPE_BF16 || dtype == GEO_SC_DTYPE_F16; }
inline int dtype_size(int dtype) { return dtype == GEO_SC_DTYPE_F32 ? 4 : 2; }
inline bool aligned_to(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

}  // namespace geo
