// Rows of floating-point values as 8-bit integers with one scale per row, with or without a root-mean-square norm (and
// the addition of a residual stream) in front, and the integers read back.
//
//   r = round_T(x + residual)          kept in the stream's own type T and written out; the norm is of the kept value
//   p = fl32(r * weight)               the 32-bit product; p = r where there is no weight
//   q = rint(127 p / max|p|)           half to even
//   scale = max|p| * rstd / 127,       rstd = 1 / sqrt(mean(r^2) + eps), or 1 without the norm
//
// q * scale is the normalised row.  The norm's factor cancels out of q, so the integers depend on the row's values
// alone and not on the order in which the squares are added: a row gives the same integers on every launch shape.  A
// thread computes 127 p / max|p| in 32 bits and decides it in 64 only where the 32-bit value lies within 2^-14 of a
// border between two integers (its error is below 127 * 2^-23 = 2^-16): one value in about eight thousand.
//
// What bounds it: HBM.  One read of x and residual, one write of r, q and the scales; a row stays in registers between
// the statistics and the rounding.  Squares are summed in 32 bits per thread and joined in 64; a row whose sum leaves
// the range of 32 bits (values above 1e19, or so small that their squares vanish) is summed again in 64.
#include "sc_rows8.h"

namespace geo {
namespace {

struct NormParams {
    const void *x, *residual, *weight;
    void *sum_out;
    int8_t *q;
    float *scale;
    long long rows, x_stride, res_stride, q_stride;
    int cols, weight_dtype;
    float eps;
};

__device__ __forceinline__ float weight_at(const NormParams &p, int c) {
    if (p.weight_dtype == GEO_SC_DTYPE_F32) return __ldg((const float *)p.weight + c);
    if (p.weight_dtype == GEO_SC_DTYPE_BF16) return __bfloat162float(__ldg((const __nv_bfloat16 *)p.weight + c));
    return __half2float(__ldg((const __half *)p.weight + c));
}

// 127 p / top as the nearest integer, half to even (see above); |p| <= top, top > 0 and finite.
__device__ __forceinline__ int round_to_top(float p, float top, float inv) {
    const float t = p * inv;
    const float off = fabsf(t - rintf(t));
    if (off > 0.5f - 6.2e-5f || top < 1e-30f)   // next to a border, or a reciprocal outside the normal range
        return (int)rint((double)p * 127.0 / (double)top);
    return __float2int_rn(t);
}

template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> row_values(const T *x, const T *res, long long at) {
    Pack<T, VEC> v = load_pack<T, VEC>(x + at);
    if (res) {
        const Pack<T, VEC> u = load_pack<T, VEC>(res + at);
#pragma unroll
        for (int e = 0; e < VEC; e++) v.v[e] = from_float<T>(to_float(v.v[e]) + to_float(u.v[e]));
    }
    return v;
}

// TPR threads own a row, VEC values per load, NV loads kept in registers (longer rows read the rest a second time).
template <typename T, int VEC, int NV, bool NORM>
__global__ void __launch_bounds__(1024) norm_int8_kernel(NormParams pr, int tpr) {
    __shared__ float part_ss[32];
    __shared__ unsigned part_top[32];
    __shared__ double part_ss64[32];
    const int tid = threadIdx.x % tpr, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
    const bool live = row < pr.rows;
    const int nvec = live ? pr.cols / VEC : 0;
    const T *x = (const T *)pr.x + (live ? row * pr.x_stride : 0);
    const T *res = pr.residual ? (const T *)pr.residual + (live ? row * pr.res_stride : 0) : nullptr;
    T *sum_out = pr.sum_out ? (T *)pr.sum_out + (live ? row * (long long)pr.cols : 0) : nullptr;

    Pack<T, VEC> keep[NV];
    float ss = 0.f;
    unsigned top = 0;   // |p| as its bit pattern: ordered like the values, NaN above infinity, so that neither is lost
    auto take = [&](const Pack<T, VEC> &v, int i) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float r = to_float(v.v[e]);
            if (NORM) ss = fmaf(r, r, ss);
            const float p = pr.weight ? r * weight_at(pr, i * VEC + e) : r;
            top = max(top, __float_as_uint(p) & 0x7fffffffu);
        }
    };
#pragma unroll
    for (int j = 0; j < NV; j++)
        if (tid + j * tpr < nvec) keep[j] = row_values<T, VEC>(x, res, (long long)(tid + j * tpr) * VEC);
#pragma unroll
    for (int j = 0; j < NV; j++)
        if (tid + j * tpr < nvec) {
            if (sum_out) store_pack<T, VEC>(sum_out + (long long)(tid + j * tpr) * VEC, keep[j]);
            take(keep[j], tid + j * tpr);
        }
    for (int i = tid + NV * tpr; i < nvec; i += tpr) {
        const Pack<T, VEC> v = row_values<T, VEC>(x, res, (long long)i * VEC);
        if (sum_out) store_pack<T, VEC>(sum_out + (long long)i * VEC, v);
        take(v, i);
    }

    ss = warp_sum(ss);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) {
        part_ss[warp] = ss;
        part_top[warp] = top;
    }
    __syncthreads();
    // every warp of the CTA looks at every partial, so that all of them agree on whether any row is summed again
    const int warps = blockDim.x >> 5, wpr = tpr >> 5, first = (threadIdx.x / tpr) * wpr;
    double total = 0;
    bool again = false;
    top = 0;
    for (int w = 0; w < warps; w++) {
        const float s = part_ss[w];
        const unsigned t = part_top[w];
        if (NORM && t < 0x7f800000u && (!(s <= 3.0e38f) || (s < 1e-30f && t > 0))) again = true;
        if (w >= first && w < first + wpr) {
            total += (double)s;
            top = max(top, t);
        }
    }
    if (NORM && again) {
        double s64 = 0;
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (tid + j * tpr < nvec)
                for (int e = 0; e < VEC; e++) s64 += (double)to_float(keep[j].v[e]) * (double)to_float(keep[j].v[e]);
        for (int i = tid + NV * tpr; i < nvec; i += tpr) {
            const Pack<T, VEC> v = row_values<T, VEC>(x, res, (long long)i * VEC);
            for (int e = 0; e < VEC; e++) s64 += (double)to_float(v.v[e]) * (double)to_float(v.v[e]);
        }
        s64 = warp_sum(s64);
        if (lane == 0) part_ss64[warp] = s64;
        __syncthreads();
        total = 0;
        for (int w = first; w < first + wpr; w++) total += part_ss64[w];
    }
    if (!live) return;
    const float ftop = __uint_as_float(top);
    double scale = (double)ftop / 127.0;
    if (NORM && top > 0) scale /= sqrt(total / pr.cols + (double)pr.eps);
    const bool fine = top < 0x7f800000u && (float)scale <= 3.402823466e38f;
    if (tid == 0) pr.scale[row] = fine ? (float)scale : __int_as_float(0x7fc00000);

    const float inv = 127.f / ftop;
    const bool zero = !fine || top == 0;
    int8_t *q = pr.q + row * pr.q_stride;
    auto give = [&](const Pack<T, VEC> &v, int i) {
        Pack<int8_t, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float r = to_float(v.v[e]);
            const float p = pr.weight ? r * weight_at(pr, i * VEC + e) : r;
            o.v[e] = zero ? 0 : (int8_t)round_to_top(p, ftop, inv);
        }
        store_pack<int8_t, VEC>(q + (long long)i * VEC, o);
    };
#pragma unroll
    for (int j = 0; j < NV; j++)
        if (tid + j * tpr < nvec) give(keep[j], tid + j * tpr);
    for (int i = tid + NV * tpr; i < nvec; i += tpr) give(row_values<T, VEC>(x, res, (long long)i * VEC), i);
}

template <typename T, int VEC, int NV> int launch_norm_v(const NormParams &p, bool norm, cudaStream_t s) {
    const long long nvec = p.cols / VEC;
    // few rows: every load of a row in flight at once; many rows: NV loads per thread, more rows per SM
    const long long want = p.rows < 2LL * sm_count() ? nvec : (nvec + NV - 1) / NV;
    int tpr = 32;
    while (tpr < 1024 && tpr < want) tpr *= 2;
    const int threads = tpr < 128 && p.rows > 1 ? 128 : tpr;
    const long long grid = (p.rows + threads / tpr - 1) / (threads / tpr);
    if (grid > 0x7fffffffLL) return fail(GEO_SC_ERR_TOO_LARGE, "%lld rows", p.rows);
    if (norm) norm_int8_kernel<T, VEC, NV, true><<<(unsigned)grid, threads, 0, s>>>(p, tpr);
    else norm_int8_kernel<T, VEC, NV, false><<<(unsigned)grid, threads, 0, s>>>(p, tpr);
    GEO_CUDA_CHECK(cudaGetLastError());
    return GEO_SC_OK;
}

template <typename T> int launch_norm(const NormParams &p, bool norm, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    // whole 16-byte loads where every row starts on a 16-byte boundary and ends on one; else value by value
    const bool wide = p.cols % VEC == 0 && aligned_to(p.x, 16) && p.x_stride % VEC == 0 && (!p.residual || (aligned_to(p.residual, 16) && p.res_stride % VEC == 0)) &&
                      (!p.sum_out || aligned_to(p.sum_out, 16)) && aligned_to(p.q, VEC) && p.q_stride % VEC == 0;
    return wide ? launch_norm_v<T, VEC, 4>(p, norm, s) : launch_norm_v<T, 1, 16>(p, norm, s);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256) dequantize_int8_kernel(const int8_t *q, long long q_stride, const float *scale, T *out, long long rows, int cols) {
    const int nvec = cols / VEC;
    const long long n = rows * nvec;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long row = n <= 0xffffffffLL ? (long long)((unsigned)i / (unsigned)nvec) : i / nvec;
        const int c = (int)(i - row * nvec) * VEC;
        const Pack<int8_t, VEC> v = load_pack<int8_t, VEC>(q + row * q_stride + c);
        const float s = __ldg(scale + row);
        Pack<T, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; e++) o.v[e] = from_float<T>((float)v.v[e] * s);
        store_pack<T, VEC>(out + row * cols + c, o);
    }
}

template <typename T> int launch_dequantize(long long rows, int cols, const int8_t *q, long long q_stride, const float *scale, T *out, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = cols % VEC == 0 && aligned_to(q, VEC) && q_stride % VEC == 0 && aligned_to(out, 16);
    const long long n = rows * (wide ? cols / VEC : cols);
    const long long want = (n + 255) / 256, most = 16LL * sm_count();
    const unsigned grid = (unsigned)(want < most ? want : most);
    if (wide) dequantize_int8_kernel<T, VEC><<<grid, 256, 0, s>>>(q, q_stride, scale, out, rows, cols);
    else dequantize_int8_kernel<T, 1><<<grid, 256, 0, s>>>(q, q_stride, scale, out, rows, cols);
    GEO_CUDA_CHECK(cudaGetLastError());
    return GEO_SC_OK;
}

int check_rows(long long rows, int cols, int dtype) {
    if (rows < 0 || cols < 1) return fail(GEO_SC_ERR_SHAPE, "%lld rows of %d values", rows, cols);
    if (rows > (1LL << 40) / cols) return fail(GEO_SC_ERR_TOO_LARGE, "%lld rows of %d values", rows, cols);
    if (!dtype_known(dtype)) return fail(GEO_SC_ERR_UNSUPPORTED, "unknown element type %d", dtype);
    return GEO_SC_OK;
}

}  // namespace
}  // namespace geo

using namespace geo;

extern "C" {

int geo_sc_rms_norm_int8(long long rows, int cols, int dtype, const void *x, long long x_stride, const void *residual,
                         long long residual_stride, const void *weight, int weight_dtype, float eps, void *sum_out, int8_t *q,
                         long long q_stride, float *scale, void *stream) {
    int rc = check_rows(rows, cols, dtype);
    if (rc) return rc;
    if (rows == 0) return GEO_SC_OK;
    if (!x || !weight || !q || !scale) return fail(GEO_SC_ERR_NULL, "x, weight, q and scale are required");
    if ((residual == nullptr) != (sum_out == nullptr)) return fail(GEO_SC_ERR_NULL, "residual and sum_out come together");
    if (!dtype_known(weight_dtype)) return fail(GEO_SC_ERR_UNSUPPORTED, "unknown weight type %d", weight_dtype);
    if (!(eps >= 0.f) || eps > 3.402823466e38f) return fail(GEO_SC_ERR_SHAPE, "eps must be finite and not negative");
    if (x_stride < 0 || residual_stride < 0 || q_stride < cols) return fail(GEO_SC_ERR_SHAPE, "bad row stride");
    NormParams p{x, residual, weight, sum_out, q, scale, rows, x_stride, residual_stride, q_stride, cols, weight_dtype, eps};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == GEO_SC_DTYPE_F32) return launch_norm<float>(p, true, s);
    if (dtype == GEO_SC_DTYPE_BF16) return launch_norm<__nv_bfloat16>(p, true, s);
    return launch_norm<__half>(p, true, s);
}

int geo_sc_quantize_int8(long long rows, int cols, int dtype, const void *x, long long x_stride, int8_t *q, long long q_stride,
                         float *scale, void *stream) {
    int rc = check_rows(rows, cols, dtype);
    if (rc) return rc;
    if (rows == 0) return GEO_SC_OK;
    if (!x || !q || !scale) return fail(GEO_SC_ERR_NULL, "x, q and scale are required");
    if (x_stride < 0 || q_stride < cols) return fail(GEO_SC_ERR_SHAPE, "bad row stride");
    NormParams p{x, nullptr, nullptr, nullptr, q, scale, rows, x_stride, 0, q_stride, cols, GEO_SC_DTYPE_F32, 0.f};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == GEO_SC_DTYPE_F32) return launch_norm<float>(p, false, s);
    if (dtype == GEO_SC_DTYPE_BF16) return launch_norm<__nv_bfloat16>(p, false, s);
    return launch_norm<__half>(p, false, s);
}

int geo_sc_dequantize_int8(long long rows, int cols, const int8_t *q, long long q_stride, const float *scale, int dtype, void *out,
                           void *stream) {
    int rc = check_rows(rows, cols, dtype);
    if (rc) return rc;
    if (rows == 0) return GEO_SC_OK;
    if (!q || !scale || !out) return fail(GEO_SC_ERR_NULL, "q, scale and out are required");
    if (q_stride < 0) return fail(GEO_SC_ERR_SHAPE, "bad row stride");
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == GEO_SC_DTYPE_F32) return launch_dequantize<float>(rows, cols, q, q_stride, scale, (float *)out, s);
    if (dtype == GEO_SC_DTYPE_BF16) return launch_dequantize<__nv_bfloat16>(rows, cols, q, q_stride, scale, (__nv_bfloat16 *)out, s);
    return launch_dequantize<__half>(rows, cols, q, q_stride, scale, (__half *)out, s);
}

}  // extern "C"
