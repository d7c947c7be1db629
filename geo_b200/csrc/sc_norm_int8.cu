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
// border between two integers (its error is below 2^-16): one value in about eight thousand.
//
// What bounds it: HBM.  One read of x and residual, one write of r, q and the scales.  CTAs walk over rows; while a row is
// reduced and rounded, the next two are on their way into shared memory (cp.async, three stages), so that the copies do
// not stop for the barriers of the reduction.  A thread sums up to 32 squares in 32 bits; what it has beyond those (rows of
// more values than 512 threads hold) it sums in parts of at most 16, which are added up in 64 bits, so that the error does
// not grow with the row.  A row whose sum leaves the range of 32 bits (values above 1e18, or so small that their squares
// vanish) is read and summed again in 64.
//
// Measured: 16384 x 8192 fp16 with residual 165 us = 5.7 TB/s, read back 61 us = 6.6 TB/s (of 6.46 for a plain copy).
//
// norm_int8_kernel: rows that start on 16-byte boundaries and are whole numbers of 16-byte vectors.  A thread copies the
// vectors that it computes itself, so the stages need no barrier; the products stay in registers from the statistics to
// the rounding.  norm_int8_ragged_kernel: every other row.  Its 16-byte granules are copied as they lie in memory, and the
// threads read them value by value, neighbours next to each other.
#include "sc_rows8.h"

namespace geo {
namespace {

struct NormParams {
    const void *x, *residual, *weight;
    void *sum_out;
    int8_t *q;
    float *scale;
    long long rows, x_stride, res_stride, q_stride;
    int cols;
    float eps;
};

__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN is kept
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float warp_max_nan(float v) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// N products as integers: 127 p / top, half to even; |p| <= top, 1e-30 <= top, finite; inv = 127 / top in fp32.
// p * inv + 1.5 * 2^23 rounds to an integer whose two's complement is the sum's low byte.  Next to a border h between
// two integers the sign of 127 p - h top decides, whose products are exact in 64 bits.
template <int N> __device__ __forceinline__ void round_to_top(const float (&p)[N], float top, float inv, uint32_t (&m)[N]) {
    constexpr float MAGIC = 12582912.f, NEAR = 0.5f - 6.2e-5f;
    float off = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) {
        const float t = fmaf(p[e], inv, MAGIC);
        off = fmaxf(off, fabsf(fmaf(p[e], inv, MAGIC - t)));
        m[e] = __float_as_uint(t);
    }
    if (off > NEAR) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float r = __uint_as_float(m[e]) - MAGIC, f = fmaf(p[e], inv, -r);
            if (fabsf(f) > NEAR) {
                const float h = r + copysignf(0.5f, f);
                const double side = fma(127.0, (double)p[e], -(double)h * (double)top);
                m[e] = __float_as_uint(MAGIC + (side > 0 ? h + 0.5f : side < 0 ? h - 0.5f : rintf(h)));
            }
        }
    }
}
template <int VEC> __device__ __forceinline__ Pack<int8_t, VEC> round_pack(const float (&p)[VEC], float top, float inv) {
    uint32_t m[VEC];
    round_to_top<VEC>(p, top, inv, m);
    Pack<int8_t, VEC> o;
    uint32_t *word = reinterpret_cast<uint32_t *>(&o);
#pragma unroll
    for (int i = 0; i < VEC / 4; i++)
        word[i] = __byte_perm(__byte_perm(m[4 * i], m[4 * i + 1], 0x0040), __byte_perm(m[4 * i + 2], m[4 * i + 3], 0x0040), 0x5410);
    return o;
}

template <typename T, int VEC> __device__ __forceinline__ void add_pack(Pack<T, VEC> &v, const Pack<T, VEC> &u) {
    float a[VEC], b[VEC];
    unpack<VEC>(v, a);
    unpack<VEC>(u, b);
#pragma unroll
    for (int e = 0; e < VEC; e++) a[e] += b[e];
    pack<VEC>(v, a);
}

// Statistics of a row, joined over its tpr threads (one or more warps of a CTA; part_* have room for two turns).
struct RowStats {
    float ss;     // in the row's first warp
    float top;
    bool again;   // the sum of squares has to be taken again in 64 bits; the same for the whole CTA
};
template <bool NORM>
__device__ __forceinline__ RowStats join_stats(float ss, float top, int tpr, int first, float (*part_ss)[32], float (*part_top)[32], int turn) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wpr = tpr >> 5;
    if (NORM) ss = warp_sum(ss);
    RowStats r;
    r.top = warp_max_nan(top);
    r.ss = ss;
    // near the end of the range of 32 bits (32 warps add up) without a product that is infinite or NaN, or vanished without
    // being zero
    r.again = NORM && r.top <= 3.402823466e38f && (!(ss <= 1.0e37f) || (ss < 1e-30f && r.top > 0.f));
    if (tpr > 32) {
        if (lane == 0) {
            part_ss[turn][warp] = ss;
            part_top[turn][warp] = r.top;
        }
        r.again = __syncthreads_or(r.again);
        r.top = warp_max_nan(part_top[turn][first + (lane & (wpr - 1))]);
        // the sum is wanted by the warp that writes the row's scale
        if (NORM && warp == first) r.ss = warp_sum(lane < wpr ? part_ss[turn][lane + first] : 0.f);
    }
    return r;
}

// The scale of a row from its statistics; total: the sum of squares in 64 bits where it was taken again.
template <bool NORM> __device__ __forceinline__ float row_scale(const RowStats &st, double total, int cols, float eps) {
    if (!(st.top <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    if (!NORM || st.top == 0.f) return st.top / 127.f;
    if (st.again) return (float)((double)st.top / 127.0 / sqrt(total / cols + (double)eps));
    const float rms = sqrtf(st.ss / (float)cols + eps);
    const float largest = st.top / rms;   // of the normalised row: may leave the range where its 127th part does not
    return largest <= 3.402823466e38f ? largest / 127.f : st.top / 127.f / rms;
}

// Joins the 64-bit sums of a row (every thread of the CTA takes part).
__device__ __forceinline__ double join_sum64(double v, int tpr, int first, double *part) {
    v = warp_sum(v);
    if (tpr > 32) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0;
        for (int i = 0; i < tpr >> 5; i++) v += part[first + i];
        __syncthreads();
    }
    return v;
}

// tpr threads own a row, VEC values per 16-byte vector.  A warp of the row owns 32 * NV neighbouring vectors, a lane
// every 32nd of them (distances that are known when this is compiled); vectors past 32 * NV per warp are read from memory,
// twice.  W: the weight's type; without NORM there is none.
template <typename T, typename W, int NV, bool NORM>
__global__ void __launch_bounds__(NV == 4 ? 512 : 1024) norm_int8_kernel(NormParams pr, int tpr) {
    constexpr int VEC = 16 / sizeof(T), STAGES = 3;
    ahead_of_previous();
    extern __shared__ __align__(16) unsigned char norm_smem[];
    __shared__ float part_ss[2][32], part_top[2][32];
    __shared__ double part64[32];
    const int tid = threadIdx.x % tpr, rpc = blockDim.x / tpr, group = threadIdx.x / tpr, first = group * (tpr >> 5);
    const int nvec = pr.cols / VEC, v0 = (tid >> 5) * (32 * NV) + (tid & 31);
    const bool has_res = pr.residual != nullptr;
    const long long step = (long long)gridDim.x * rpc, start = (long long)blockIdx.x * rpc + group;
    // a thread's vectors: [stage][x, residual][warp][NV][lane]
    const uint32_t half = blockDim.x * 16 * NV, stage_bytes = half * (has_res ? 2 : 1);
    unsigned char *const slots = norm_smem + ((threadIdx.x >> 5) * (32 * NV) + (threadIdx.x & 31)) * 16;
    bool in[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        in[j] = v0 + j * 32 < nvec;
        if (!in[j])   // vectors past the row's end: zeros in every stage, which add nothing to its statistics
#pragma unroll
            for (int s = 0; s < STAGES; s++) {
                *(int4 *)(slots + s * stage_bytes + j * 512) = make_int4(0, 0, 0, 0);
                if (has_res) *(int4 *)(slots + s * stage_bytes + half + j * 512) = make_int4(0, 0, 0, 0);
            }
    }

    auto weight_of = [&](const W *at, float (&w)[VEC]) {
        if constexpr (VEC * sizeof(W) == 32) {   // fp32 weights of 16-bit values: two loads
            const Pack<W, VEC / 2> a = load_pack<W, VEC / 2>(at), b = load_pack<W, VEC / 2>(at + VEC / 2);
#pragma unroll
            for (int e = 0; e < VEC / 2; e++) {
                w[e] = to_float(a.v[e]);
                w[VEC / 2 + e] = to_float(b.v[e]);
            }
        } else {
            unpack<VEC>(load_pack<W, VEC>(at), w);
        }
    };
    const T *next_x = (const T *)pr.x + start * pr.x_stride + v0 * VEC, *next_r = (const T *)pr.residual + start * pr.res_stride + v0 * VEC;
    auto ask = [&](long long row, int stage) {   // the rows in turn
        if (row < pr.rows) {
            const uint32_t dst = smem_u32(slots) + stage * stage_bytes;
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (in[j]) {
                    copy_async(dst + j * 512, next_x + j * 32 * VEC, 16);
                    if (has_res) copy_async(dst + half + j * 512, next_r + j * 32 * VEC, 16);
                }
        }
        copy_commit();
        next_x += step * pr.x_stride;
        next_r += step * pr.res_stride;
    };
    after_previous();
    ask(start, 0);
    ask(start + step, 1);
    int turn = 0, stage = 0;
    T *sum_at = (T *)pr.sum_out + start * pr.cols + v0 * VEC;
    int8_t *q_at = pr.q + start * pr.q_stride + v0 * VEC;
    const W *const w_at = (const W *)pr.weight + v0 * VEC;
    // every thread of a CTA makes the same number of turns; rows past the end take part in the barriers only
    for (long long row = start; row - group < pr.rows; row += step, turn ^= 1) {
        const bool live = row < pr.rows;
        ask(row + 2 * step, stage == 0 ? 2 : stage - 1);
        copy_wait<2>();
        float p[NV][VEC], ss = 0.f, top = 0.f;
        auto take = [&](const Pack<T, VEC> &v, const W *at, float (&pv)[VEC]) {
            float r[VEC], wv[VEC];
            unpack<VEC>(v, r);
            if constexpr (NORM) weight_of(at, wv);
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                if (NORM) ss = fmaf(r[e], r[e], ss);
                pv[e] = NORM ? r[e] * wv[e] : r[e];
                top = max_nan(top, fabsf(pv[e]));
            }
        };
        // a vector from memory: past the stages' part of the row, or once more
        auto far = [&](int i, bool write) {
            Pack<T, VEC> v = load_pack<T, VEC>((const T *)pr.x + row * pr.x_stride + (long long)i * VEC);
            if (has_res) {
                add_pack<T, VEC>(v, load_pack<T, VEC>((const T *)pr.residual + row * pr.res_stride + (long long)i * VEC));
                if (write) store_pack<T, VEC>((T *)pr.sum_out + row * pr.cols + (long long)i * VEC, v);
            }
            return v;
        };
        const uint32_t at = smem_u32(slots) + stage * stage_bytes;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            Pack<T, VEC> v = load_staged<T, VEC>(at + j * 512);
            if (has_res) {
                add_pack<T, VEC>(v, load_staged<T, VEC>(at + half + j * 512));
                if (in[j] && live) store_pack<T, VEC>(sum_at + j * 32 * VEC, v);
            }
            take(v, in[j] ? w_at + j * 32 * VEC : (const W *)pr.weight, p[j]);
        }
        if (nvec > NV * tpr) {
            const float held = ss;
            double beyond = 0;
            for (int i = tid + NV * tpr; i < nvec && live; i += tpr) {
                float pv[VEC];
                ss = 0.f;
                take(far(i, true), (const W *)pr.weight + (long long)i * VEC, pv);
                beyond += (double)ss;
            }
            ss = held + (float)beyond;
        }
        stage = stage == 2 ? 0 : stage + 1;

        const RowStats st = join_stats<NORM>(ss, top, tpr, first, part_ss, part_top, turn);
        double total = 0;
        if (NORM && st.again) {
            for (int i = tid; i < nvec && live; i += tpr) {
                float r[VEC];
                unpack<VEC>(far(i, false), r);
                for (int e = 0; e < VEC; e++) total += (double)r[e] * (double)r[e];
            }
            total = join_sum64(total, tpr, first, part64);
        }
        if (live) {
            if (tid == 0) pr.scale[row] = row_scale<NORM>(st, total, pr.cols, pr.eps);
            const bool fine = st.top <= 3.402823466e38f;
            // products below the normal range of a reciprocal: the integers are those of 2^64 times the row; a row with a
            // product that is not finite, or of zeros, has zeros
            const float lift = st.top < 1e-30f ? 18446744073709551616.f : 1.f, lifted = st.top * lift;
            const float inv = fine && st.top > 0.f ? 127.f / lifted : 0.f;
            const bool plain = fine && lift == 1.f;
            if (!plain)
#pragma unroll
                for (int j = 0; j < NV; j++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) p[j][e] = fine ? p[j][e] * lift : 0.f;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const Pack<int8_t, VEC> o = round_pack<VEC>(p[j], lifted, inv);
                if (in[j]) store_pack<int8_t, VEC>(q_at + j * 32 * VEC, o);
            }
            for (int i = tid + NV * tpr; i < nvec; i += tpr) {
                float pv[VEC];
                take(far(i, false), (const W *)pr.weight + (long long)i * VEC, pv);
                if (!plain)
                    for (int e = 0; e < VEC; e++) pv[e] = fine ? pv[e] * lift : 0.f;
                store_pack<int8_t, VEC>(pr.q + row * pr.q_stride + (long long)i * VEC, round_pack<VEC>(pv, lifted, inv));
            }
        }
        sum_at += step * pr.cols;
        q_at += step * pr.q_stride;
    }
    copy_wait<0>();
}

// One row per team at a time, a team being a warp (four of them a CTA) or a CTA; any alignment.  STAGED: rows come through shared memory, `stages` (3, or 1 where three rows do
// not fit) of them; else from memory, twice.
template <typename T, typename W, int THREADS, bool NORM, bool STAGED>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) norm_int8_ragged_kernel(NormParams pr, int stages, int buf_bytes) {
    constexpr int KEEP = 8;   // products of a row that a thread keeps
    ahead_of_previous();
    extern __shared__ __align__(16) unsigned char norm_smem[];
    __shared__ float part_ss[2][32], part_top[2][32];
    __shared__ double part64[32];
    constexpr int threads = THREADS, TEAMS = THREADS == 32 ? 4 : 1;
    const int tid = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x, slot = THREADS == 32 ? threadIdx.x >> 5 : 0, cols = pr.cols;
    auto team_sync = [&]() {
        if (THREADS == 32) __syncwarp();
        else __syncthreads();
    };
    const bool has_res = pr.residual != nullptr;
    const T *const x = (const T *)pr.x, *const res = (const T *)pr.residual;
    const int stage_bytes = buf_bytes * (has_res ? 2 : 1);
    unsigned char *const bufs = norm_smem + slot * stages * stage_bytes;
    const long long step = (long long)gridDim.x * TEAMS, start = (long long)blockIdx.x * TEAMS + slot;

    // The 16-byte granules of a row, each at its own distance from the one with the row's first byte.  A granule is read
    // from the row's first byte on (value by value) where it begins before it, and up to the row's last byte.
    auto copy_row = [&](const T *row, unsigned char *buf) {
        const uintptr_t a = (uintptr_t)row, e = a + (size_t)cols * sizeof(T), g0 = a & ~(uintptr_t)15;
        const int granules = (int)((e - g0 + 15) >> 4);
        for (int i = tid; i < granules; i += threads) {
            const uintptr_t g = g0 + (uintptr_t)i * 16;
            if (g < a) {
                const int n = (int)(min(e, g + 16) - a) / (int)sizeof(T);
                for (int k = 0; k < n; k++) *(T *)(buf + (a - g0) + k * sizeof(T)) = row[k];
            } else {
                copy_async(smem_u32(buf) + i * 16, (const void *)g, (int)(min(e, g + 16) - g));
            }
        }
    };
    auto ask = [&](long long row, int stage) {
        if (row < pr.rows) {
            copy_row(x + row * pr.x_stride, bufs + stage * stage_bytes);
            if (has_res) copy_row(res + row * pr.res_stride, bufs + stage * stage_bytes + buf_bytes);
        }
        copy_commit();
    };
    after_previous();
    if (STAGED && stages == 3) {
        ask(start, 0);
        ask(start + step, 1);
    }
    int turn = 0, stage = 0;
    for (long long row = start; row < pr.rows; row += step, turn ^= 1) {
        const T *const gx = x + row * pr.x_stride, *const gr = has_res ? res + row * pr.res_stride : nullptr;
        T *const sum_out = (T *)pr.sum_out + row * cols;
        const T *sx = nullptr, *sr = nullptr;
        if (STAGED) {
            if (stages == 3) {
                ask(row + 2 * step, stage == 0 ? 2 : stage - 1);
                copy_wait<2>();
            } else {
                ask(row, 0);
                copy_wait<0>();
            }
            team_sync();
            sx = (const T *)(bufs + stage * stage_bytes + ((uintptr_t)gx & 15));
            if (has_res) sr = (const T *)(bufs + stage * stage_bytes + buf_bytes + ((uintptr_t)gr & 15));
        }
        auto value = [&](int c) {
            float r = to_float(STAGED ? sx[c] : gx[c]);
            if (has_res) r = to_float(from_float<T>(r + to_float(STAGED ? sr[c] : gr[c])));
            return r;
        };
        auto product = [&](float r, int c) {
            if constexpr (NORM) return r * to_float(((const W *)pr.weight)[c]);
            else return r;
        };
        float ss = 0.f, top = 0.f, keep[KEEP];
        auto take = [&](int c) {
            const float r = value(c);
            if (has_res) sum_out[c] = from_float<T>(r);
            if (NORM) ss = fmaf(r, r, ss);
            const float p = product(r, c);
            top = max_nan(top, fabsf(p));
            return p;
        };
#pragma unroll
        for (int j = 0; j < KEEP; j++) {
            keep[j] = 0.f;
            if ((j + 1) * threads <= cols) keep[j] = take(tid + j * threads);   // the same for every thread
            else if (tid + j * threads < cols) keep[j] = take(tid + j * threads);
        }
        if (cols > KEEP * threads) {
            const float held = ss;
            double beyond = 0;
            int c = tid + KEEP * threads;
            for (; c + 15 * threads < cols; c += 16 * threads) {
                ss = 0.f;
#pragma unroll 4
                for (int i = 0; i < 16; i++) take(c + i * threads);
                beyond += (double)ss;
            }
            ss = 0.f;
            for (; c < cols; c += threads) take(c);
            ss = held + (float)(beyond + (double)ss);
        }
        const RowStats st = join_stats<NORM>(ss, top, threads, 0, part_ss, part_top, turn);
        double total = 0;
        if (NORM && st.again) {
            for (int c = tid; c < cols; c += threads) total += (double)value(c) * (double)value(c);
            total = join_sum64(total, threads, 0, part64);
        }
        if (tid == 0) pr.scale[row] = row_scale<NORM>(st, total, cols, pr.eps);
        const bool fine = st.top <= 3.402823466e38f;
        const float lift = st.top < 1e-30f ? 18446744073709551616.f : 1.f, lifted = st.top * lift, inv = fine && st.top > 0.f ? 127.f / lifted : 0.f;
        int8_t *const q = pr.q + row * pr.q_stride;
        uint32_t m[KEEP];
        if (!fine || lift != 1.f)
#pragma unroll
            for (int j = 0; j < KEEP; j++) keep[j] = fine ? keep[j] * lift : 0.f;
        round_to_top<KEEP>(keep, lifted, inv, m);
#pragma unroll
        for (int j = 0; j < KEEP; j++)
            if (tid + j * threads < cols) q[tid + j * threads] = (int8_t)m[j];
        for (int c = tid + KEEP * threads; c < cols; c += threads) {
            const float p[1] = {fine ? product(value(c), c) * lift : 0.f};
            uint32_t o[1];
            round_to_top<1>(p, lifted, inv, o);
            q[c] = (int8_t)o[0];
        }
        if (STAGED) {
            team_sync();   // the stage may be overwritten
            if (stages == 3) stage = stage == 2 ? 0 : stage + 1;
        }
    }
    copy_wait<0>();
}

constexpr int NORM_SMEM = 200 * 1024;   // of an SM's 227 KB, shared by its CTAs

template <typename T, typename W, int NV, bool NORM> int launch_norm_nv(const NormParams &p, int tpr, cudaStream_t s) {
    const int threads = tpr < 128 && p.rows > 1 ? 128 : tpr, rpc = threads / tpr;
    const int smem = threads * 16 * NV * (p.residual ? 2 : 1) * 3;
    static PerDeviceOnce once;
    int rc = per_device_once(once, []() -> int {
        GEO_CUDA_CHECK(cudaFuncSetAttribute(norm_int8_kernel<T, W, NV, NORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_SMEM));
        return GEO_SC_OK;
    });
    if (rc) return rc;
    // as many CTAs as fit every SM's registers and the stages
    const int per_sm = max(1, min((NV == 4 ? 512 : 1024) / threads, NORM_SMEM / smem));
    const long long need = (p.rows + rpc - 1) / rpc, most = (long long)sm_count() * per_sm;
    return launch_behind(norm_int8_kernel<T, W, NV, NORM>, (unsigned)(need < most ? need : most), threads, smem, s, 1, p, tpr);
}

template <typename T, typename W, int THREADS, bool NORM> int launch_ragged(const NormParams &p, cudaStream_t s) {
    constexpr int TEAMS = THREADS == 32 ? 4 : 1, CTA = THREADS * TEAMS;
    const long long buf = ((long long)p.cols * sizeof(T) + 47) / 16 * 16, stage = buf * (p.residual ? 2 : 1) * TEAMS;
    const int stages = stage * 3 <= NORM_SMEM / 2 ? 3 : stage <= NORM_SMEM ? 1 : 0, smem = (int)(stages * stage);
    static PerDeviceOnce once;
    int rc = per_device_once(once, []() -> int {
        GEO_CUDA_CHECK(cudaFuncSetAttribute(norm_int8_ragged_kernel<T, W, THREADS, NORM, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_SMEM));
        return GEO_SC_OK;
    });
    if (rc) return rc;
    const long long need = (p.rows + TEAMS - 1) / TEAMS, most = (long long)sm_count() * max(1, min(1536 / CTA, smem ? NORM_SMEM / smem : 16));
    const unsigned grid = (unsigned)(need < most ? need : most);
    if (stages) return launch_behind(norm_int8_ragged_kernel<T, W, THREADS, NORM, true>, grid, CTA, smem, s, 1, p, stages, (int)buf);
    return launch_behind(norm_int8_ragged_kernel<T, W, THREADS, NORM, false>, grid, CTA, 0, s, 1, p, 0, 0);
}

template <typename T, typename W, bool NORM> int launch_norm(const NormParams &p, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    // whole 16-byte vectors where every row starts on a 16-byte boundary and ends on one
    const bool wide = p.cols % VEC == 0 && aligned_to(p.x, 16) && p.x_stride % VEC == 0 && (!p.residual || (aligned_to(p.residual, 16) && p.res_stride % VEC == 0)) &&
                      (!p.sum_out || aligned_to(p.sum_out, 16)) && aligned_to(p.q, VEC) && p.q_stride % VEC == 0 && (!NORM || aligned_to(p.weight, 16));
    if (wide) {
        // Few rows: one vector per thread, the shortest way through a row.  Many: two per thread for rows of up to 256
        // vectors (8192 x 1024 fp32 with read-back 30.0 us, with four 32.6), four for longer ones, which have fewer
        // reductions then (16384 x 8192 fp16: 227 us, with two 235).
        const int nvec = p.cols / VEC;
        const bool few = p.rows < 2LL * sm_count() && nvec <= 1024;
        const int most = few ? 1024 : 512, want = few ? nvec : nvec <= 256 ? (nvec + 1) / 2 : (nvec + 3) / 4;
        int tpr = 32;
        while (tpr < most && tpr < want) tpr *= 2;
        if (nvec <= tpr) return launch_norm_nv<T, W, 1, NORM>(p, tpr, s);
        if (nvec <= 2 * tpr) return launch_norm_nv<T, W, 2, NORM>(p, tpr, s);
        return launch_norm_nv<T, W, 4, NORM>(p, tpr, s);
    }
    // eight values per thread, which it keeps in registers, as long as a CTA of 512 goes round
    if (p.cols <= 256 && p.rows > 1) return launch_ragged<T, W, 32, NORM>(p, s);
    if (p.cols <= 1024) return launch_ragged<T, W, 128, NORM>(p, s);
    return p.cols <= 2048 ? launch_ragged<T, W, 256, NORM>(p, s) : launch_ragged<T, W, 512, NORM>(p, s);
}

// A warp takes STEPS x 32 vectors of a row (read VEC integers, write VEC values), all steps in flight at once.
template <typename T, int VEC, int STEPS>
__global__ void __launch_bounds__(256) dequantize_int8_kernel(const int8_t *q, long long q_stride, const float *scale, T *out, long long units, int upr,
                                                               int nvec, int cols) {
    ahead_of_previous();
    after_previous();
    const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= units) return;
    const long long row = units <= 0xffffffffLL ? (long long)((unsigned)unit / (unsigned)upr) : unit / upr;
    const int first = (int)(unit - row * upr) * (32 * STEPS) + (threadIdx.x & 31);
    q += row * q_stride;
    out += row * cols;
    Pack<int8_t, VEC> v[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; j++)
        if (first + j * 32 < nvec) v[j] = load_pack<int8_t, VEC>(q + (long long)(first + j * 32) * VEC);
    const float s = scale[row];
#pragma unroll
    for (int j = 0; j < STEPS; j++)
        if (first + j * 32 < nvec) {
            Pack<T, VEC> o;
            float f[VEC];
            if constexpr (VEC == 1) {
                f[0] = (float)v[j].v[0] * s;
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e += 4) unpack_bytes(reinterpret_cast<const uint32_t *>(&v[j])[e / 4], f + e);
#pragma unroll
                for (int e = 0; e < VEC; e++) f[e] *= s;
            }
            pack<VEC>(o, f);
            store_pack<T, VEC>(out + (long long)(first + j * 32) * VEC, o);
        }
}

template <typename T, int VEC, int STEPS> int launch_dequantize_v(long long rows, int cols, const int8_t *q, long long q_stride, const float *scale, T *out, cudaStream_t s) {
    const int nvec = cols / VEC, upr = (nvec + 32 * STEPS - 1) / (32 * STEPS);
    const long long units = rows * upr, grid = (units + 7) / 8;
    if (grid > 0x7fffffffLL) return fail(GEO_SC_ERR_TOO_LARGE, "%lld rows of %d values", rows, cols);
    return launch_behind(dequantize_int8_kernel<T, VEC, STEPS>, (unsigned)grid, 256, 0, s, 1, q, q_stride, scale, out, units, upr, nvec, cols);
}

template <typename T> int launch_dequantize(long long rows, int cols, const int8_t *q, long long q_stride, const float *scale, T *out, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = cols % VEC == 0 && aligned_to(q, VEC) && q_stride % VEC == 0 && aligned_to(out, 16);
    return wide ? launch_dequantize_v<T, VEC, 4>(rows, cols, q, q_stride, scale, out, s) : launch_dequantize_v<T, 1, 16>(rows, cols, q, q_stride, scale, out, s);
}

int check_rows(long long rows, int cols, int dtype) {
    if (rows < 0 || cols < 1) return fail(GEO_SC_ERR_SHAPE, "%lld rows of %d values", rows, cols);
    if (cols > (1 << 30) || rows > (1LL << 40) / cols) return fail(GEO_SC_ERR_TOO_LARGE, "%lld rows of %d values", rows, cols);
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
    if (weight_dtype != GEO_SC_DTYPE_F32 && weight_dtype != dtype)
        return fail(GEO_SC_ERR_UNSUPPORTED, "weight has to be fp32 or of the type of x, not type %d", weight_dtype);
    if (!(eps >= 0.f) || eps > 3.402823466e38f) return fail(GEO_SC_ERR_SHAPE, "eps must be finite and not negative");
    if (x_stride < 0 || residual_stride < 0 || q_stride < cols) return fail(GEO_SC_ERR_SHAPE, "bad row stride");
    NormParams p{x, residual, weight, sum_out, q, scale, rows, x_stride, residual_stride, q_stride, cols, eps};
    cudaStream_t s = (cudaStream_t)stream;
    const bool f32 = weight_dtype == GEO_SC_DTYPE_F32;
    if (dtype == GEO_SC_DTYPE_F32) return launch_norm<float, float, true>(p, s);
    if (dtype == GEO_SC_DTYPE_BF16) return f32 ? launch_norm<__nv_bfloat16, float, true>(p, s) : launch_norm<__nv_bfloat16, __nv_bfloat16, true>(p, s);
    return f32 ? launch_norm<__half, float, true>(p, s) : launch_norm<__half, __half, true>(p, s);
}

int geo_sc_quantize_int8(long long rows, int cols, int dtype, const void *x, long long x_stride, int8_t *q, long long q_stride,
                         float *scale, void *stream) {
    int rc = check_rows(rows, cols, dtype);
    if (rc) return rc;
    if (rows == 0) return GEO_SC_OK;
    if (!x || !q || !scale) return fail(GEO_SC_ERR_NULL, "x, q and scale are required");
    if (x_stride < 0 || q_stride < cols) return fail(GEO_SC_ERR_SHAPE, "bad row stride");
    NormParams p{x, nullptr, nullptr, nullptr, q, scale, rows, x_stride, 0, q_stride, cols, 0.f};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == GEO_SC_DTYPE_F32) return launch_norm<float, float, false>(p, s);
    if (dtype == GEO_SC_DTYPE_BF16) return launch_norm<__nv_bfloat16, __nv_bfloat16, false>(p, s);
    return launch_norm<__half, __half, false>(p, s);
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
