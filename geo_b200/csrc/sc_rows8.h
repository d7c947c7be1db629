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
// through the packed conversions, which are not on the slow conversion pipe
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(0.f), "f"(v));
    return __ushort_as_bfloat16((unsigned short)r);
}
template <> __device__ __forceinline__ __half from_float<__half>(float v) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(0.f), "f"(v));
    return __ushort_as_half((unsigned short)r);
}

// N values of T as one load or store (N * sizeof(T) is 16, 8 or 4 bytes, or N = 1).
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T v[N]; };

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = int4; };
template <> struct Raw<8> { using type = int2; };
template <> struct Raw<4> { using type = int; };
template <> struct Raw<2> { using type = short; };
template <> struct Raw<1> { using type = signed char; };
template <typename T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
    using R = typename Raw<sizeof(Pack<T, N>)>::type;
    Pack<T, N> v;
    *reinterpret_cast<R *>(&v) = *reinterpret_cast<const R *>(p);
    return v;
}
template <typename T, int N> __device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &v) {
    using R = typename Raw<sizeof(Pack<T, N>)>::type;
    *reinterpret_cast<R *>(p) = *reinterpret_cast<const R *>(&v);
}

// Packs to and from fp32, two 16-bit values per instruction.
template <int N> __device__ __forceinline__ void unpack(const Pack<float, N> &v, float (&f)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) f[e] = v.v[e];
}
template <int N> __device__ __forceinline__ void unpack(const Pack<__nv_bfloat16, N> &v, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = __bfloat162float(v.v[0]);
    } else {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(&v);
#pragma unroll
        for (int e = 0; e < N / 2; e++) {
            f[2 * e] = __uint_as_float(w[e] << 16);
            f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
}
template <int N> __device__ __forceinline__ void unpack(const Pack<__half, N> &v, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = __half2float(v.v[0]);
    } else {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(&v);
#pragma unroll
        for (int e = 0; e < N / 2; e++)
            asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}\n" : "=f"(f[2 * e]), "=f"(f[2 * e + 1]) : "r"(w[e]));
    }
}
template <int N> __device__ __forceinline__ void pack(Pack<float, N> &v, const float (&f)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) v.v[e] = f[e];
}
template <int N> __device__ __forceinline__ void pack(Pack<__nv_bfloat16, N> &v, const float (&f)[N]) {
    if constexpr (N == 1) {
        v.v[0] = from_float<__nv_bfloat16>(f[0]);
    } else {
        uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
        for (int e = 0; e < N / 2; e++) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(f[2 * e + 1]), "f"(f[2 * e]));
    }
}
template <int N> __device__ __forceinline__ void pack(Pack<__half, N> &v, const float (&f)[N]) {
    if constexpr (N == 1) {
        v.v[0] = from_float<__half>(f[0]);
    } else {
        uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
        for (int e = 0; e < N / 2; e++) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(f[2 * e + 1]), "f"(f[2 * e]));
    }
}
// Largest value of a pack (NaN passed over); two 16-bit values per instruction.
template <int N> __device__ __forceinline__ float pack_max(const Pack<float, N> &v) {
    float m = v.v[0];
#pragma unroll
    for (int e = 1; e < N; e++) m = fmaxf(m, v.v[e]);
    return m;
}
template <int N> __device__ __forceinline__ float pack_max(const Pack<__nv_bfloat16, N> &v) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&v);
    uint32_t m = w[0];
#pragma unroll
    for (int e = 1; e < N / 2; e++) asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[e]));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}
template <int N> __device__ __forceinline__ float pack_max(const Pack<__half, N> &v) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&v);
    uint32_t m = w[0];
#pragma unroll
    for (int e = 1; e < N / 2; e++) asm("max.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[e]));
    float a, b;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}\n" : "=f"(a), "=f"(b) : "r"(m));
    return fmaxf(a, b);
}
// Four signed bytes as floats: a byte b + 128 in the low mantissa of 2^23 is the float 2^23 + 128 + b, exactly.
__device__ __forceinline__ void unpack_bytes(uint32_t w, float *f) {
    w ^= 0x80808080u;
#pragma unroll
    for (int e = 0; e < 4; e++) f[e] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + e)) - 8388736.f;
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
__device__ __forceinline__ float warp_max(float v) {   // NaN passed over
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int bytes) {   // 16 bytes, zeros past `bytes`
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> load_staged(uint32_t at) {   // 16 bytes of shared memory
    Pack<T, VEC> v;
    int4 &r = *reinterpret_cast<int4 *>(&v);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
    return v;
}
template <typename T, int VEC> __device__ __forceinline__ void store_staged(uint32_t at, const Pack<T, VEC> &v) {
    const int4 &r = *reinterpret_cast<const int4 *>(&v);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w) : "memory");
}

// These kernels are launched so that their CTAs may take their places while the kernel in front of them in the stream is
// still finishing.  ahead_of_previous(): the kernel behind this one may do the same; after_previous(): from here on the
// kernel in front has completed and its writes are visible.  Nothing in global memory is touched before that, and nothing
// is read through the read-only path (__ldg, ld.global.nc, const __restrict__): that is promised only for memory that
// nobody writes while the kernel lives, and the kernel in front writes its results while this one waits.
__device__ __forceinline__ void ahead_of_previous() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// Launch of such a kernel, in clusters of `cluster` CTAs.
template <typename... P, typename... A>
int launch_behind(void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t s, int cluster, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    GEO_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
    return GEO_SC_OK;
}

inline bool dtype_known(int dtype) { return dtype == GEO_SC_DTYPE_F32 || dtype == GEO_SC_DTYPE_BF16 || dtype == GEO_SC_DTYPE_F16; }
inline int dtype_size(int dtype) { return dtype == GEO_SC_DTYPE_F32 ? 4 : 2; }
inline bool aligned_to(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

}  // namespace geo
