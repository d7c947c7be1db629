// Loss of a student's logits against a teacher's top logits, and its gradient.
//
// Row of logits z[0..vocab), entries (index_k, t_k), temperature T:
//   p_k = softmax over the entries of t_k / T          q_j = softmax over the vocabulary of z_j / T
//   loss = weight * T^2 * sum_k p_k (log p_k - log q_{index_k})
//   d loss / d z_j = weight * T * (q_j - sum of the p_k whose index is j)
// Entries with a negative index are padding, an entry of -inf has p = 0.  A row without a single entry above -inf, or
// of weight 0, has loss 0 and gradient 0, and its logits are not read.  An index at or past the vocabulary, or a
// teacher's logit that is NaN or +inf, makes the row's loss and gradient NaN; nothing is read or written through it.
//
// With m the row's largest logit, S = sum_j exp((z_j - m) / T): q_j = exp((z_j - m) / T) / S.  The difference z - m is
// taken before it is scaled, so that the terms which carry the sum have small arguments and small errors.  Every thread
// keeps a running maximum and a running sum (rescaled when the maximum grows) in one pass over the row; these pairs are
// joined in a fixed order.  Sums over the entries and over the rows are taken in 64 bits.
//
// What bounds it: HBM.  One read of the logits and, with the gradient, one write: the second pass of a team over its row
// comes from L2.  A team of one warp owns a row of a small vocabulary, a CTA one of a larger vocabulary, and where
// there are fewer rows than SMs a cluster of CTAs shares a row and joins the pairs over distributed shared memory.
#include <cooperative_groups.h>

#include "sc_rows8.h"

namespace geo {
namespace {

namespace cg = cooperative_groups;

constexpr int DISTILL_MAX_TOP = 512;
constexpr int DISTILL_WARP_VOCAB = 1024;   // vocabularies up to this: one warp per row
constexpr float NEG_INF = -INFINITY;

struct DistillParams {
    const void *logits, *indices, *teacher;
    const float *weight, *upstream;
    float *row_loss;     // [rows]
    float2 *stats;       // [rows]: m, S
    void *grad;          // [rows][vocab]
    long long rows, stride;
    int vocab, top, index64, teacher_dtype;
    int upstream_rows;   // upstream has one value per row (else one value)
    int skip_one;        // rows whose upstream is 1 keep the gradient that the forward pass has written
    float temperature, scale;
    float loss_factor, grad_factor;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Joins per-thread values of a team of TEAM threads (a warp, or the whole CTA); every thread gets the result.
template <int TEAM> struct Team {
    float *buf;   // 32 floats and 32 doubles' room, CTA teams only
    __device__ float max(float v) {
        v = warp_max(v);
        if (TEAM == 32) return v;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
        __syncthreads();
        v = buf[0];
        for (int i = 1; i < TEAM / 32; i++) v = fmaxf(v, buf[i]);
        return v;
    }
    template <typename V> __device__ V sum(V v) {
        v = warp_sum(v);
        if (TEAM == 32) return v;
        V *b = (V *)buf;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
        __syncthreads();
        v = b[0];
        for (int i = 1; i < TEAM / 32; i++) v += b[i];
        return v;
    }
    __device__ bool any(bool v) { return TEAM == 32 ? __any_sync(0xffffffffu, v) : __syncthreads_or(v); }
    __device__ void sync() {
        if (TEAM == 32) __syncwarp();
        else __syncthreads();
    }
};

__device__ __forceinline__ float teacher_at(const DistillParams &p, long long i) {
    if (p.teacher_dtype == GEO_SC_DTYPE_F32) return ((const float *)p.teacher)[i];
    if (p.teacher_dtype == GEO_SC_DTYPE_BF16) return __bfloat162float(((const __nv_bfloat16 *)p.teacher)[i]);
    return __half2float(((const __half *)p.teacher)[i]);
}

// The part of a row that a thread block owns: `head` single values up to the first 16-byte boundary (rank 0), vectors
// [v0, v1), and from `tail` on single values (last rank).
struct Slice {
    int head, v0, v1, tail;
};
template <typename T> __device__ __forceinline__ Slice slice_of(const T *row, int vocab, int rank, int ranks) {
    constexpr int VEC = 16 / sizeof(T);
    const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
    const int head = min(off ? VEC - off : 0, vocab), nvec = (vocab - head) / VEC, per = (nvec + ranks - 1) / ranks;
    Slice s;
    s.head = head;
    s.v0 = min(rank * per, nvec);
    s.v1 = min(s.v0 + per, nvec);
    s.tail = head + nvec * VEC;
    return s;
}

template <typename T, int TEAM, bool STATS, bool GRAD, bool CLUSTER>
__global__ void __launch_bounds__(TEAM == 32 ? 256 : TEAM) distill_kernel(DistillParams pr) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ __align__(16) unsigned char distill_smem[];
    __shared__ __align__(16) float reduce_buf[64];
    __shared__ float2 pair;   // this CTA's (m, S), read by the other CTAs of the cluster
    const int tid = TEAM == 32 ? (threadIdx.x & 31) : threadIdx.x;
    const int slot = TEAM == 32 ? threadIdx.x >> 5 : 0;
    int rank = 0, ranks = 1;
    if (CLUSTER) {
        rank = (int)cg::this_cluster().block_rank();
        ranks = (int)cg::this_cluster().num_blocks();
    }
    const long long row = TEAM == 32 ? (long long)blockIdx.x * (blockDim.x / 32) + slot : (long long)(blockIdx.x / ranks);
    if (TEAM == 32 && row >= pr.rows) return;
    Team<TEAM> team{reduce_buf};
    int *const idx = (int *)distill_smem + (size_t)slot * 2 * pr.top;   // an entry's index, -1 where it has no part
    float *const prob = (float *)(idx + pr.top);

    float up = 1.f;
    if (!STATS) {
        up = pr.upstream[pr.upstream_rows ? row : 0];
        if (pr.skip_one && up == 1.f) return;
    }
    const T *z = (const T *)pr.logits + row * pr.stride;
    T *grad = GRAD ? (T *)pr.grad + row * (long long)pr.vocab : nullptr;
    const float w = pr.weight ? pr.weight[row] : 1.f;
    const Slice sl = slice_of(z, pr.vocab, rank, ranks);
    const bool last = rank == ranks - 1;

    // the teacher's entries
    const float inv_t = 1.f / pr.temperature;
    float tmax = NEG_INF;
    bool bad = false;
    for (int k = tid; k < pr.top; k += TEAM) {
        const long long at = row * pr.top + k;
        const long long j = pr.index64 ? ((const long long *)pr.indices)[at] : ((const int *)pr.indices)[at];
        const float t = teacher_at(pr, at);
        const bool use = j >= 0;
        if (use && (j >= pr.vocab || !(t < INFINITY))) bad = true;
        idx[k] = use && j < pr.vocab ? (int)j : -1;
        prob[k] = use ? t : NEG_INF;
        if (use) tmax = fmaxf(tmax, t);
    }
    bad = team.any(bad);
    tmax = team.max(tmax);
    const bool dead = (!bad && tmax == NEG_INF) || w == 0.f;
    if (dead || bad) {   // the same for every CTA of a cluster
        const float v = dead ? 0.f : __int_as_float(0x7fc00000);
        if (STATS && rank == 0 && tid == 0) {
            pr.row_loss[row] = v;
            pr.stats[row] = make_float2(0.f, 1.f);
        }
        if (GRAD) {
            const int from = rank == 0 ? 0 : sl.head + sl.v0 * VEC, to = last ? pr.vocab : sl.head + sl.v1 * VEC;
            for (int j = from + tid; j < to; j += TEAM) grad[j] = from_float<T>(v);
        }
        return;
    }
    float psum = 0.f;
    for (int k = tid; k < pr.top; k += TEAM) {
        const float e = expf((prob[k] - tmax) * inv_t);   // an entry's exponential; divided by the sum when used
        if (!STATS) prob[k] = e;
        psum += e;
    }
    psum = team.sum(psum);
    const float inv_psum = 1.f / psum;

    const float c = 1.4426950408889634f * inv_t;
    float m, S;
    if (STATS) {
        m = NEG_INF;
        S = 0.f;
        auto take = [&](float v) {
            if (v > m) {
                S *= ex2((m - v) * c);
                m = v;
            }
            S += ex2((v - (m == NEG_INF ? 0.f : m)) * c);
        };
        if (rank == 0)
            for (int j = tid; j < sl.head; j += TEAM) take(to_float(z[j]));
        if (last)
            for (int j = sl.tail + tid; j < pr.vocab; j += TEAM) take(to_float(z[j]));
        const T *zv = z + sl.head;
#pragma unroll 4
        for (int i = sl.v0 + tid; i < sl.v1; i += TEAM) {
            const Pack<T, VEC> v = load_pack<T, VEC>(zv + (long long)i * VEC);
            float f[VEC], top = NEG_INF;
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                f[e] = to_float(v.v[e]);
                top = fmaxf(top, f[e]);
            }
            if (top > m) {
                S *= ex2((m - top) * c);
                m = top;
            }
            const float base = m == NEG_INF ? 0.f : m;
#pragma unroll
            for (int e = 0; e < VEC; e++) S += ex2((f[e] - base) * c);
        }
        float top = team.max(m);
        S = team.sum(S * (m == NEG_INF ? (S == 0.f ? 0.f : 1.f) : ex2((m - top) * c)));
        m = top;
        if (CLUSTER) {
            cg::cluster_group cluster = cg::this_cluster();
            if (tid == 0) pair = make_float2(m, S);
            cluster.sync();
            top = NEG_INF;
            for (int r = 0; r < ranks; r++) top = fmaxf(top, cluster.map_shared_rank(&pair, r)->x);
            S = 0.f;
            for (int r = 0; r < ranks; r++) {
                const float2 v = *cluster.map_shared_rank(&pair, r);
                S += v.y * (v.x == NEG_INF ? (v.y == 0.f ? 0.f : 1.f) : ex2((v.x - top) * c));
            }
            m = top;
            cluster.sync();   // nobody leaves while its pair may still be read
        }
        if (m == NEG_INF) S = __int_as_float(0x7fc00000);   // no logit above -inf: no distribution
        if (rank == 0) {
            const double log_s = log((double)S), log_p = log((double)psum);
            double loss = 0;
            for (int k = tid; k < pr.top; k += TEAM) {
                const float d = (prob[k] - tmax) * inv_t, e = expf(d);
                prob[k] = e;
                if (idx[k] >= 0 && e > 0.f)
                    loss += (double)e / (double)psum * (((double)d - log_p) - ((double)((to_float(z[idx[k]]) - m) * inv_t) - log_s));
            }
            loss = team.sum(loss);
            if (tid == 0) {
                const double t = pr.temperature;
                pr.row_loss[row] = (float)(loss * t * t * (double)w * (double)pr.loss_factor);
                pr.stats[row] = make_float2(m, S);
            }
        } else {
            for (int k = tid; k < pr.top; k += TEAM) prob[k] = expf((prob[k] - tmax) * inv_t);
        }
    } else {
        m = pr.stats[row].x;
        S = pr.stats[row].y;
    }
    if (!GRAD) return;

    const float a = up * pr.grad_factor * w * pr.temperature, inv_s = 1.f / S;
    const int from = rank == 0 ? 0 : sl.head + sl.v0 * VEC, to = last ? pr.vocab : sl.head + sl.v1 * VEC;
    const bool wide = ((uintptr_t)(grad + sl.head) & 15) == 0;
    if (wide) {
        if (rank == 0)
            for (int j = tid; j < sl.head; j += TEAM) grad[j] = from_float<T>(ex2((to_float(z[j]) - m) * c) * inv_s * a);
        if (last)
            for (int j = sl.tail + tid; j < pr.vocab; j += TEAM) grad[j] = from_float<T>(ex2((to_float(z[j]) - m) * c) * inv_s * a);
        const T *zv = z + sl.head;
        T *gv = grad + sl.head;
#pragma unroll 4
        for (int i = sl.v0 + tid; i < sl.v1; i += TEAM) {
            Pack<T, VEC> v = load_pack<T, VEC>(zv + (long long)i * VEC);
#pragma unroll
            for (int e = 0; e < VEC; e++) v.v[e] = from_float<T>(ex2((to_float(v.v[e]) - m) * c) * inv_s * a);
            store_pack<T, VEC>(gv + (long long)i * VEC, v);
        }
    } else {
        for (int j = from + tid; j < to; j += TEAM) grad[j] = from_float<T>(ex2((to_float(z[j]) - m) * c) * inv_s * a);
    }
    team.sync();   // the entries' places are written a second time, after the pass above
    for (int k = tid; k < pr.top; k += TEAM) {
        const int j = idx[k];
        if (j < from || j >= to) continue;
        float p = 0.f;   // the entries of one index together, by the first of them
        bool first = true;
        for (int i = 0; i < pr.top; i++)
            if (idx[i] == j) {
                if (i < k) first = false;
                p += prob[i];
            }
        if (first) grad[j] = from_float<T>((ex2((to_float(z[j]) - m) * c) * inv_s - p * inv_psum) * a);
    }
}

// The rows' losses as one value, in a fixed order.
__global__ void __launch_bounds__(1024) distill_sum_kernel(const float *row_loss, long long rows, double factor, float *loss) {
    __shared__ double part[32];
    double s = 0;
    for (long long i = threadIdx.x; i < rows; i += 1024) s += (double)row_loss[i];
    s = warp_sum(s);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 32; i++) s += part[i];
        *loss = (float)(s * factor);
    }
}

template <typename T, int TEAM, bool STATS, bool GRAD, bool CLUSTER> int launch_team(const DistillParams &p, int ranks, cudaStream_t s) {
    const int threads = TEAM == 32 ? 256 : TEAM;
    const long long grid = TEAM == 32 ? (p.rows + 7) / 8 : p.rows * ranks;
    if (grid > 0x7fffffffLL) return fail(GEO_SC_ERR_TOO_LARGE, "%lld rows", p.rows);
    const size_t smem = (size_t)(TEAM == 32 ? 8 : 1) * p.top * 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CLUSTER ? 1 : 0;
    GEO_CUDA_CHECK(cudaLaunchKernelEx(&cfg, distill_kernel<T, TEAM, STATS, GRAD, CLUSTER>, p));
    return GEO_SC_OK;
}

template <typename T, bool STATS, bool GRAD> int launch_distill(const DistillParams &p, cudaStream_t s) {
    if (p.vocab <= DISTILL_WARP_VOCAB) return launch_team<T, 32, STATS, GRAD, false>(p, 1, s);
    int ranks = 1;
    while (ranks < 8 && p.rows * ranks * 2 <= sm_count() && p.vocab / (ranks * 2) >= 2048) ranks *= 2;
    return ranks > 1 ? launch_team<T, 512, STATS, GRAD, true>(p, ranks, s) : launch_team<T, 512, STATS, GRAD, false>(p, 1, s);
}

template <bool STATS, bool GRAD> int launch_typed(const DistillParams &p, int dtype, cudaStream_t s) {
    if (dtype == GEO_SC_DTYPE_F32) return launch_distill<float, STATS, GRAD>(p, s);
    if (dtype == GEO_SC_DTYPE_BF16) return launch_distill<__nv_bfloat16, STATS, GRAD>(p, s);
    return launch_distill<__half, STATS, GRAD>(p, s);
}

int check_distill(long long rows, int vocab, int top, int dtype, const void *logits, long long stride, const void *indices,
                  int index_bits, const void *teacher, int teacher_dtype, float temperature) {
    if (rows < 0 || vocab < 1 || top < 1) return fail(GEO_SC_ERR_SHAPE, "%lld rows of %d logits, %d entries", rows, vocab, top);
    if (top > DISTILL_MAX_TOP) return fail(GEO_SC_ERR_TOO_LARGE, "%d entries per row, at most %d", top, DISTILL_MAX_TOP);
    if (rows > (1LL << 40) / vocab) return fail(GEO_SC_ERR_TOO_LARGE, "%lld rows of %d logits", rows, vocab);
    if (!dtype_known(dtype) || !dtype_known(teacher_dtype)) return fail(GEO_SC_ERR_UNSUPPORTED, "unknown element type");
    if (index_bits != 32 && index_bits != 64) return fail(GEO_SC_ERR_UNSUPPORTED, "indices of %d bits", index_bits);
    if (!(temperature >= 1e-6f && temperature <= 1e6f)) return fail(GEO_SC_ERR_SHAPE, "temperature outside [1e-6, 1e6]");
    if (stride < 0) return fail(GEO_SC_ERR_SHAPE, "bad row stride");
    if (rows > 0 && (!logits || !indices || !teacher)) return fail(GEO_SC_ERR_NULL, "logits, indices and teacher are required");
    return GEO_SC_OK;
}

}  // namespace
}  // namespace geo

using namespace geo;

extern "C" {

int geo_sc_distill_forward(long long rows, int vocab, int top, int dtype, const void *logits, long long stride, const void *indices,
                           int index_bits, const void *teacher, int teacher_dtype, const float *weight, float temperature,
                           float scale, int mean, float *row_loss, void *stats, float *loss, void *grad, void *stream) {
    int rc = check_distill(rows, vocab, top, dtype, logits, stride, indices, index_bits, teacher, teacher_dtype, temperature);
    if (rc) return rc;
    if ((rows > 0 && (!row_loss || !stats)) || (mean && !loss)) return fail(GEO_SC_ERR_NULL, "row_loss, stats and the loss are required");
    cudaStream_t s = (cudaStream_t)stream;
    const double all = mean ? (double)scale / (double)(rows > 0 ? rows : 1) : (double)scale;
    if (rows > 0) {
        DistillParams p = {};
        p.logits = logits; p.indices = indices; p.teacher = teacher; p.weight = weight;
        p.row_loss = row_loss; p.stats = (float2 *)stats; p.grad = grad;
        p.rows = rows; p.stride = stride; p.vocab = vocab; p.top = top; p.index64 = index_bits == 64; p.teacher_dtype = teacher_dtype;
        p.temperature = temperature; p.loss_factor = mean ? 1.f : scale; p.grad_factor = (float)all;
        rc = grad ? launch_typed<true, true>(p, dtype, s) : launch_typed<true, false>(p, dtype, s);
        if (rc) return rc;
    }
    if (mean) {
        distill_sum_kernel<<<1, 1024, 0, s>>>(row_loss, rows, all, loss);
        GEO_CUDA_CHECK(cudaGetLastError());
    }
    return GEO_SC_OK;
}

int geo_sc_distill_backward(long long rows, int vocab, int top, int dtype, const void *logits, long long stride, const void *indices,
                            int index_bits, const void *teacher, int teacher_dtype, const float *weight, float temperature,
                            float scale, int mean, const void *stats, const float *upstream, int skip_one, void *grad, void *stream) {
    int rc = check_distill(rows, vocab, top, dtype, logits, stride, indices, index_bits, teacher, teacher_dtype, temperature);
    if (rc) return rc;
    if (rows == 0) return GEO_SC_OK;
    if (!stats || !upstream || !grad) return fail(GEO_SC_ERR_NULL, "stats, upstream and grad are required");
    DistillParams p = {};
    p.logits = logits; p.indices = indices; p.teacher = teacher; p.weight = weight; p.upstream = upstream;
    p.stats = (float2 *)const_cast<void *>(stats); p.grad = grad;
    p.rows = rows; p.stride = stride; p.vocab = vocab; p.top = top; p.index64 = index_bits == 64; p.teacher_dtype = teacher_dtype;
    p.upstream_rows = !mean; p.skip_one = skip_one;
    p.temperature = temperature; p.grad_factor = (float)(mean ? (double)scale / (double)rows : (double)scale);
    return launch_typed<false, true>(p, dtype, (cudaStream_t)stream);
}

}  // extern "C"
