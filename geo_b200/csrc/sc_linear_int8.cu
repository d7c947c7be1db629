// 8-bit matrix product with a scale per token and per output channel:
//
//   out[m][n] = (sum_k x[m][k] w[n][k]) * x_scale[m] * w_scale[n] + bias[n]
//
// The sum is exact in 32-bit integers (k <= 131071, so that 2^14 k stays below 2^31); the two scales and the bias are
// applied in fp32 and the result is rounded once to the output's type.
//
// Up to 32 tokens run on linear_int8_mma_kernel below, more on the tcgen05 kernel (sc_linear_int8_tc.cu).
//
// linear_int8_mma_kernel: `mma.sync.m16n8k32` with the weights as the 16-row operand, read once from memory straight
// into fragments.  The order of k inside a product is free, so a lane takes 16 consecutive bytes of its weight row and
// the same 16 bytes of its token rows for two instructions: whole 16-byte loads, no shared memory, no shuffles.  A CTA
// of eight warps owns 16 channels and all tokens; the warps split k and join their integer sums in shared memory.
// Bound by the weights' bytes: 1 x 8192 x 8192 13.3 us (5.0 TB/s with the launch); with more tokens by the tokens' bytes
// that every CTA reads again as well.  Measured by graph replay, here and on the other kernel: 32 x 1024 x 1024 2.7 and
// 3.8 us, 9 x 4096 x 4096 5.9 and 5.9, 32 x 4096 x 4096 7.8 and 6.0, 16 x 8192 x 8192 16.0 and 14.5, 32 x 8192 x 8192 28.1
// and 14.5.  The switch at 32 tokens is right for layers of about 1000 features and too high for wide ones.
#include "sc_linear_int8.h"

namespace geo {
namespace {

// 16 bytes of a row from byte `at` on, zeros from byte k on.
__device__ __forceinline__ uint4 load16(const int8_t *row, int at, int k) {
    if (at + 16 <= k) return *(const uint4 *)(row + at);
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int b = at + 4 * i;
        v[i] = 0;
        if (b + 4 <= k) {
            v[i] = *(const uint32_t *)(row + b);
        } else if (b < k) {
            v[i] = (uint8_t)row[b];
            if (b + 1 < k) v[i] |= (uint32_t)(uint8_t)row[b + 1] << 8;
            if (b + 2 < k) v[i] |= (uint32_t)(uint8_t)row[b + 2] << 16;
        }
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int MMA_WARPS = 8;

template <typename T, int NT>
__global__ void __launch_bounds__(32 * MMA_WARPS) linear_int8_mma_kernel(LinearParams p) {
    __shared__ int sums[MMA_WARPS][NT * 8][16];
    ahead_of_previous();
    after_previous();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = (int)blockIdx.x * 16;
    // rows past the end repeat the last one; their sums are not stored
    const int8_t *wa = p.w + (long long)min(n0 + g, p.n - 1) * p.w_stride;
    const int8_t *wb = p.w + (long long)min(n0 + g + 8, p.n - 1) * p.w_stride;
    const int8_t *xr[NT];
    int acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        xr[j] = p.x + (long long)min(j * 8 + g, p.m - 1) * p.x_stride;
#pragma unroll
        for (int i = 0; i < 4; i++) acc[j][i] = 0;
    }
    auto step = [&](const uint4 &a, const uint4 &b, const uint4 (&x)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            mma_s8(acc[j], a.x, b.x, a.y, b.y, x[j].x, x[j].y);
            mma_s8(acc[j], a.z, b.z, a.w, b.w, x[j].z, x[j].w);
        }
    };
    // A warp's turn: 128 bytes (two chunks) of every row, whole lines; with few tokens two turns at a time, their weights
    // all asked for before the first is used.
    constexpr int UNROLL = NT == 1 ? 4 : 2, TURN = MMA_WARPS * 128;
    auto chunk = [&](int u) { return (u >> 1) * TURN + (u & 1) * 64 + t * 16; };
    int kc = warp * 128;
    for (; kc + (UNROLL / 2 - 1) * TURN + 128 <= p.k; kc += UNROLL / 2 * TURN) {
        uint4 a[UNROLL], b[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            a[u] = *(const uint4 *)(wa + kc + chunk(u));
            b[u] = *(const uint4 *)(wb + kc + chunk(u));
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            uint4 x[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) x[j] = *(const uint4 *)(xr[j] + kc + chunk(u));
            step(a[u], b[u], x);
        }
    }
    for (; kc < p.k; kc += TURN)
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int at = kc + chunk(u);
            const uint4 a = load16(wa, at, p.k), b = load16(wb, at, p.k);
            uint4 x[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) x[j] = load16(xr[j], at, p.k);
            step(a, b, x);
        }
#pragma unroll
    for (int j = 0; j < NT; j++) {
        sums[warp][j * 8 + t * 2][g] = acc[j][0];
        sums[warp][j * 8 + t * 2 + 1][g] = acc[j][1];
        sums[warp][j * 8 + t * 2][g + 8] = acc[j][2];
        sums[warp][j * 8 + t * 2 + 1][g + 8] = acc[j][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 8 * 16; i += blockDim.x) {
        const int m = i >> 4, ni = i & 15, n = n0 + ni;
        if (m >= p.m || n >= p.n) continue;
        int s = 0;
#pragma unroll
        for (int w = 0; w < MMA_WARPS; w++) s += sums[w][m][ni];
        float v = (float)s * p.x_scale[m] * p.w_scale[n];
        if (p.bias) v += p.bias[n];
        ((T *)p.out)[m * p.out_stride + n] = from_float<T>(v);
    }
}

template <typename T> int launch_mma(const LinearParams &p, cudaStream_t s) {
    const int nt = p.m <= 8 ? 1 : p.m <= 16 ? 2 : 4;   // 8 * nt tokens hold all m
    const auto kernel = nt == 1 ? linear_int8_mma_kernel<T, 1> : nt == 2 ? linear_int8_mma_kernel<T, 2> : linear_int8_mma_kernel<T, 4>;
    return launch_behind(kernel, (unsigned)((p.n + 15) / 16), 32 * MMA_WARPS, 0, s, 1, p);
}

}  // namespace
}  // namespace geo

using namespace geo;

extern "C" int geo_sc_linear_int8(int m, int n, int k, const int8_t *x, long long x_stride, const float *x_scale, const int8_t *w,
                                  long long w_stride, const float *w_scale, const float *bias, int dtype, void *out,
                                  long long out_stride, void *stream) {
    if (m < 0 || n < 1 || k < 1) return fail(GEO_SC_ERR_SHAPE, "product of [%d, %d] and [%d, %d]", m, k, n, k);
    if (k > 131071) return fail(GEO_SC_ERR_TOO_LARGE, "k = %d: sums of more than 131071 products may leave 32 bits", k);
    if (m > 0x7ffffe00 || n > 0x7ffffe00) return fail(GEO_SC_ERR_TOO_LARGE, "%d tokens x %d channels", m, n);
    if (!dtype_known(dtype)) return fail(GEO_SC_ERR_UNSUPPORTED, "unknown element type %d", dtype);
    if (m == 0) return GEO_SC_OK;
    if (!x || !x_scale || !w || !w_scale || !out) return fail(GEO_SC_ERR_NULL, "x, w, their scales and out are required");
    if (x_stride < k || w_stride < k || out_stride < n) return fail(GEO_SC_ERR_SHAPE, "bad row stride");
    if (!aligned_to(x, 16) || !aligned_to(w, 16) || x_stride % 16 || w_stride % 16)
        return fail(GEO_SC_ERR_UNSUPPORTED, "rows of x and w have to start on 16-byte boundaries");
    LinearParams p{x, w, x_scale, w_scale, bias, out, x_stride, w_stride, out_stride, m, n, k};
    cudaStream_t s = (cudaStream_t)stream;
    if (m > 32) return launch_linear_int8_tc(p, dtype, s);
    if (dtype == GEO_SC_DTYPE_F32) return launch_mma<float>(p, s);
    if (dtype == GEO_SC_DTYPE_BF16) return launch_mma<__nv_bfloat16>(p, s);
    return launch_mma<__half>(p, s);
}
