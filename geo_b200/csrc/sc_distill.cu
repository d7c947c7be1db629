// Loss of a student's logits against a teacher's top logits, and its gradient.
//
// Row of logits z[0..vocab), entries (index_k, t_k), temperature T:
//   p_k = softmax over the entries of t_k / T          q_j = softmax over the vocabulary of z_j / T
//   loss = weight * T^2 * sum_k p_k (log p_k - log q_{index_k})
//   d loss / d z_j = weight * T * (q_j - sum of the p_k whose index is j)
// Entries with a negative index are padding, an entry of -inf has p = 0.  A row without a single entry above -inf, or
// of weight 0, has loss 0 and gradient 0, whatever its logits are.  An index at or past the vocabulary, or a
// teacher's logit that is NaN or +inf, makes the row's loss and gradient NaN; nothing is read or written through it.
//
// In base 2, with c = log2(e) / T, m the row's largest logit, the reference r = fl(m c) and S = sum_j 2^(z_j c - r):
// q_j = 2^(z_j c - r) / S.  The argument is one fused multiply-add, rounded relative to itself, so the terms which carry
// the sum have small errors; that r is rounded does not matter, because every term and every partial sum is taken
// against a reference that is kept as it is.  Past |m c| = 2^30 (rows masked by the type's lowest value throughout) that
// rounding is too coarse; there two different values of any of the types are at least 64 apart in the exponent, so that in
// q logits other than m count as -inf, m as 0.  In the loss log q = (z - m) / T - log S is taken of the logit itself: it is
// finite where q is not above 0.
// Sums over the entries and over the rows are joined in a fixed order, the loss in 64 bits.
//
// What bounds it: HBM, one read of the logits and, with the gradient, one write.  A team copies its share of a row into
// shared memory (cp.async, all of it asked for at once; a thread copies the vectors that it computes), so the largest
// logit, the sum and the gradient read memory once.  Teams: a warp, a CTA of 128 or 256 threads, or a cluster of up to
// eight CTAs of 256, whichever holds the row with sixteen 16-byte vectors per thread (more threads where there are few
// rows); what a cluster of eight cannot hold is read again.  Few warps with many vectors each, because what a row costs
// a warp besides its vectors is the same for any number.  A warp of its own takes the teacher's entries of a CTA's row
// while the logits are on their way, and the loss while the gradient is written.  Measured with 4096 rows of 32768 bf16
// logits, 64 entries: 103 us for loss and gradient = 5.2 TB/s, half of the exponential pipe; 2048 x 65537 fp16, the loss
// alone: 50 us = 5.3 TB/s.
#include <cooperative_groups.h>

#include <type_traits>

#include "sc_rows8.h"

namespace geo {
namespace {

namespace cg = cooperative_groups;

constexpr int DISTILL_MAX_TOP = 512;
constexpr float NEG_INF = -INFINITY;
constexpr float FAR = 1073741824.f;   // 2^30

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
    float temperature, loss_factor, grad_factor;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

// What terms are taken against where r is the largest z c: 0 far below, where they are 0 (or NaN) and not the exponential
// of a rounding or of -inf + inf.
__device__ __forceinline__ float base_of(float r) { return r < -FAR ? 0.f : r; }
// A sum taken against base_of(from), as one against `to` >= from.
__device__ __forceinline__ float moved(float sum, float from, float to) { return from < -FAR ? sum : sum * ex2(from - to); }

constexpr int team_threads(int team) { return team == 32 ? 128 : team + 32; }   // four warps with a row each; or a team and the entries' warp
constexpr int team_blocks(int team, bool grad) { return team == 32 ? 8 : (grad ? 896 : 1280) / team; }         // that registers are left for, of an SM
// 16-byte vectors of a row that a thread holds: for the gradient, or on their way only
__host__ __device__ constexpr int held_vectors(bool grad) { return grad ? 16 : 8; }
constexpr int DISTILL_SMEM = 200 * 1024;   // of an SM's 227 KB
// a team's shared memory: 20 bytes per entry, the table that finds entries of the same index, then the team's vectors
__host__ __device__ inline int table_slots(int top) {
    int n = 64;
    while (n < 2 * top) n *= 2;
    return top <= 32 ? 0 : n;
}
__host__ __device__ inline int entry_room(int top) { return (top * 20 + table_slots(top) * 4 + 15) / 16 * 16; }

// The teacher's entries of a row in shared memory, taken by one warp.
struct Entries {
    int *idx;        // -1: no part
    float *prob;     // exp((t - largest t) / T)
    float *diff;     // (t - largest t) / T
    float *own;      // the student's logit
    float *merged;   // the probability of an index, by its first entry of those in [from, to); else -1
    int *table;
    int slots;
};
// 0: a row with entries, 1: without (or of weight 0), 2: with a bad entry.
template <typename T, int AT_ONCE>   // AT_ONCE: entries of a lane whose loads are in flight together, the index, then the logit that it names
__device__ __forceinline__ int take_entries(const DistillParams &pr, const Entries &en, long long row, const T *z, float w, float inv_t, float &psum) {
    const int lane = threadIdx.x & 31;
    float tmax = NEG_INF;
    bool bad = false;
    for (int first = lane; first < pr.top; first += 32 * AT_ONCE) {
        long long j[AT_ONCE];
        float t[AT_ONCE], own[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            const int k = first + i * 32;
            const long long at = row * pr.top + k;
            j[i] = k >= pr.top ? -1 : pr.index64 ? ((const long long *)pr.indices)[at] : ((const int *)pr.indices)[at];
            t[i] = k >= pr.top ? NEG_INF : teacher_at(pr, at);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) own[i] = j[i] >= 0 && j[i] < pr.vocab ? to_float(z[j[i]]) : 0.f;
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            const int k = first + i * 32;
            const bool use = j[i] >= 0, fits = use && j[i] < pr.vocab;
            bad |= use && (!fits || !(t[i] < INFINITY));
            if (use) tmax = fmaxf(tmax, t[i]);
            if (k < pr.top) {
                en.idx[k] = fits ? (int)j[i] : -1;
                en.own[k] = own[i];
                en.diff[k] = use ? t[i] : NEG_INF;
            }
        }
    }
    bad = __any_sync(0xffffffffu, bad);
    tmax = warp_max(tmax);
    if (w == 0.f || (!bad && tmax == NEG_INF)) return 1;
    if (bad) return 2;
    psum = 0.f;
    for (int k = lane; k < pr.top; k += 32) {
        const float d = (en.diff[k] - tmax) * inv_t, e = expf(d);
        en.diff[k] = d;
        en.prob[k] = e;
        psum += e;
    }
    psum = warp_sum(psum);
    return 0;
}

// The probability that an index in [from, to) carries, with its first entry.
__device__ __forceinline__ void merge_entries(const Entries &en, int top, int from, int to, float psum) {
    const int lane = threadIdx.x & 31;
    bool twice = false;
    if (top <= 32) {
        const int j = lane < top ? en.idx[lane] : -1;
        const unsigned same = __match_any_sync(0xffffffffu, j);
        twice = j >= 0 && (same & (same - 1)) != 0;
    } else {
        for (int i = lane; i < en.slots; i += 32) en.table[i] = -1;
        __syncwarp();
        for (int k = lane; k < top; k += 32) {
            const int j = en.idx[k];
            if (j < 0) continue;
            for (int i = (unsigned)j * 2654435769u >> 16;; i++) {   // open addressing; at most half of the slots are ever taken
                const int was = atomicCAS(&en.table[i & (en.slots - 1)], -1, j);
                twice |= was == j;
                if (was == -1 || was == j) break;
            }
        }
    }
    twice = __any_sync(0xffffffffu, twice);
    __syncwarp();
    for (int k = lane; k < top; k += 32) {
        const int j = en.idx[k];
        bool first = j >= from && j < to;
        float p = en.prob[k];
        if (twice && first) {
            p = 0.f;
            for (int i = 0; i < top; i++)
                if (en.idx[i] == j) {
                    p += en.prob[i];
                    first &= i >= k;
                }
        }
        en.merged[k] = first ? p / psum : -1.f;
    }
}

template <typename T, int TEAM, bool STATS, bool GRAD, bool CLUSTER>
__global__ void __launch_bounds__(team_threads(TEAM), team_blocks(TEAM, GRAD)) distill_kernel(DistillParams pr, int team_bytes) {
    ahead_of_previous();
    after_previous();
    if (!STATS && pr.skip_one && !pr.upstream_rows && pr.upstream[0] == 1.f) return;   // the whole gradient is there already
    constexpr int VEC = 16 / sizeof(T), WARPS = TEAM / 32, HOP = TEAM * 16;   // bytes between a thread's vectors
    constexpr int GROUP = held_vectors(GRAD) / 4;
    extern __shared__ __align__(16) unsigned char distill_smem[];
    __shared__ float2 part[8];
    __shared__ float2 pair;   // this CTA's (largest logit, sum), read by the other CTAs of the cluster
    __shared__ int row_state;
    __shared__ float row_psum;
    const int lane = threadIdx.x & 31, warp = TEAM == 32 ? 0 : threadIdx.x >> 5, slot = TEAM == 32 ? threadIdx.x >> 5 : 0;
    const int tid = TEAM == 32 ? lane : threadIdx.x;
    const bool scribe = TEAM == 32 || warp == WARPS, streams = TEAM == 32 || warp < WARPS;   // who takes the entries, who the logits
    int rank = 0, ranks = 1;
    if (CLUSTER) {
        rank = (int)cg::this_cluster().block_rank();
        ranks = (int)cg::this_cluster().num_blocks();
    }
    const bool last = rank == ranks - 1;
    auto team_sync = [&]() {
        if (TEAM == 32) __syncwarp();
        else __syncthreads();
    };
    Entries en;
    en.idx = (int *)(distill_smem + slot * team_bytes);
    en.prob = (float *)(en.idx + pr.top);
    en.diff = en.prob + pr.top;
    en.own = en.diff + pr.top;
    en.merged = en.own + pr.top;
    en.table = (int *)(en.merged + pr.top);
    en.slots = table_slots(pr.top);
    const uint32_t held = smem_u32(en.idx) + entry_room(pr.top) + tid * 16;   // a thread's vectors
    const float inv_t = 1.f / pr.temperature, c = 1.4426950408889634f * inv_t;
    auto scaled = [&](float v) { return __fmul_rn(v, c); };   // a reference: rounded, never part of a fused multiply-add

    const long long teams = TEAM == 32 ? (long long)gridDim.x * 4 : gridDim.x / ranks;
    for (long long row = TEAM == 32 ? (long long)blockIdx.x * 4 + slot : blockIdx.x / ranks; row < pr.rows; row += teams) {
        float up = 1.f;
        if (!STATS) {
            up = pr.upstream[pr.upstream_rows ? row : 0];
            if (pr.skip_one && up == 1.f) continue;
        }
        const T *const z = (const T *)pr.logits + row * pr.stride;
        T *const grad = GRAD ? (T *)pr.grad + row * (long long)pr.vocab : nullptr;
        const Slice sl = slice_of(z, pr.vocab, rank, ranks);
        const T *const zv = z + sl.head;
        const float w = pr.weight ? pr.weight[row] : 1.f;
        const int from = rank == 0 ? 0 : sl.head + sl.v0 * VEC, to = last ? pr.vocab : sl.head + sl.v1 * VEC;

        // A thread's vectors: four groups of GROUP in shared memory, asked for at once.  Where a slice is longer, the next
        // group takes the place of the one that has been read, and a second pass asks for them all again.  The lanes of a
        // warp have the same number of vectors; those past the slice are -inf.
        const int v_first = sl.v0 + tid;
        const int ahead = sl.v1 - (sl.v0 + warp * 32);   // vectors from the warp's first on
        const int count = streams ? max(0, ahead + TEAM - 1) / TEAM : 0, groups = (count + GROUP - 1) / GROUP;
        const int whole = ahead >= 32 ? ((ahead - 32) / TEAM + 1) / GROUP : 0;   // groups that every lane has all of
        auto fill = [&](int g) {
            const T *src = zv + (long long)(v_first + g * (GROUP * TEAM)) * VEC;
            const uint32_t dst = held + (g & 3) * (GROUP * HOP);
            if (g < groups) {
#pragma unroll
                for (int i = 0; i < GROUP; i++) {
                    const int h = g * GROUP + i;
                    if (v_first + h * TEAM < sl.v1) {
                        copy_async(dst + i * HOP, src + i * (TEAM * VEC), 16);
                    } else if (h < count) {
                        Pack<T, VEC> none;
#pragma unroll
                        for (int e = 0; e < VEC; e++) none.v[e] = from_float<T>(NEG_INF);
                        store_staged<T, VEC>(dst + i * HOP, none);
                    }
                }
            }
            copy_commit();
        };
        auto fill_all = [&]() {
            for (int g = 0; g < 4; g++) fill(g);
        };
        // all_of(first vector, its place) for groups that every lane has all of, one(vector, its place) for the other vectors,
        // when they have arrived; `resident`: all of them have, and stay
        auto each = [&](bool resident, auto all_of, auto one) {
            for (int g = 0; g < groups; g++) {
                if (!resident) copy_wait<3>();
                const uint32_t at = held + (g & 3) * (GROUP * HOP);
                if (g < whole) {
                    all_of(g * GROUP, at);
                } else {
#pragma unroll 1
                    for (int i = 0; i < GROUP && g * GROUP + i < count; i++) one(g * GROUP + i, at + i * HOP);
                }
                if (!resident) fill(g + 4);
            }
        };
        // the values before the first and after the last vector, one per thread
        int r_at = -1;
        float r_value = 0.f;
        if (streams) {
            fill_all();
            const int heads = rank == 0 ? sl.head : 0, ragged = heads + (last ? pr.vocab - sl.tail : 0);
            r_at = tid < heads ? tid : tid < ragged ? sl.tail + tid - heads : -1;
            if (r_at >= 0) r_value = to_float(z[r_at]);
        }
        int state = 0;
        float psum = 1.f;
        if (scribe) {
            state = take_entries<T, TEAM == 32 ? 1 : 4>(pr, en, row, z, w, inv_t, psum);
            if (TEAM > 32 && lane == 0) {
                row_state = state;
                row_psum = psum;
            }
            __syncwarp();
        }

        float m = 0.f, sum = 0.f;
        bool flat = false;   // m c out of range: a logit is either m or nothing (one that is NaN makes the sum NaN)
        auto seen = [&](float v) { return !flat ? v : v == m ? 0.f : NEG_INF; };
        auto out_of_range = [&]() { return fabsf(m) <= 3.402823466e38f && !(fabsf(scaled(m)) <= FAR); };
        // Largest logit and sum of the warp.  A thread's reference is the first largest value that it meets, and moves only
        // for one that is 2^32 times as probable (some lane would move it at nearly every vector otherwise); sums stay far
        // below 2^127.
        auto warp_stats = [&](auto is_flat, float &most, float &total) {
            constexpr bool FLAT = decltype(is_flat)::value;
            float top = r_at >= 0 ? seen(r_value) : NEG_INF, ref = scaled(top), base = base_of(ref), s1 = 0.f;
            float s0 = r_at >= 0 ? ex2(fmaf(top, c, -base)) : 0.f;
            if (FLAT && r_value != r_value) s1 = r_value;
            auto look = [&](float large) {
                top = fmaxf(top, large);
                if (scaled(large) > ref + 32.f) {
                    const float to_ref = scaled(large);
                    s0 = moved(s0, ref, to_ref);
                    s1 = moved(s1, ref, to_ref);
                    ref = to_ref;
                    base = base_of(ref);
                }
            };
            auto add = [&](const float (&f)[VEC]) {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    s0 += ex2(fmaf(f[e], c, -base));
                    s1 += ex2(fmaf(f[e + 1], c, -base));
                }
            };
            auto one = [&](int, uint32_t at) {
                float f[VEC], large = NEG_INF;
                unpack<VEC>(load_staged<T, VEC>(at), f);
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    if (FLAT) {
                        if (f[e] != f[e]) s1 = f[e];
                        f[e] = seen(f[e]);
                    }
                    large = fmaxf(large, f[e]);
                }
                look(large);
                add(f);
            };
            each(FLAT && groups <= 4, [&](int h, uint32_t at) {
                if (FLAT) {
#pragma unroll 1
                    for (int i = 0; i < GROUP; i++) one(h + i, at + i * HOP);
                } else {
                    Pack<T, VEC> v[GROUP];
                    float large = NEG_INF;
#pragma unroll
                    for (int i = 0; i < GROUP; i++) {
                        v[i] = load_staged<T, VEC>(at + i * HOP);
                        large = fmaxf(large, pack_max<VEC>(v[i]));
                    }
                    look(large);
#pragma unroll
                    for (int i = 0; i < GROUP; i++) {
                        float f[VEC];
                        unpack<VEC>(v[i], f);
                        add(f);
                    }
                }
            }, one);
            most = warp_max(top);
            total = warp_sum(moved(s0 + s1, ref, scaled(most)));
        };

        if (STATS) {
            for (;;) {
                float most = NEG_INF;
                if (streams) {
                    if (flat) warp_stats(std::true_type(), most, sum);
                    else warp_stats(std::false_type(), most, sum);
                }
                if (TEAM > 32) {
                    if (streams && lane == 0) part[warp] = make_float2(most, sum);
                    __syncthreads();
                    const float2 v = part[lane & (WARPS - 1)];
                    most = warp_max(v.x);
                    sum = warp_sum(lane < WARPS ? moved(v.y, scaled(v.x), scaled(most)) : 0.f);
                }
                if (CLUSTER) {
                    cg::cluster_group cluster = cg::this_cluster();
                    if (tid == 0) pair = make_float2(most, sum);
                    cluster.sync();
                    const float2 v = *cluster.map_shared_rank(&pair, lane & (ranks - 1));
                    cluster.sync();   // nobody leaves, or writes its next pair, while it may still be read
                    most = warp_max(v.x);
                    sum = warp_sum(lane < ranks ? moved(v.y, scaled(v.x), scaled(most)) : 0.f);
                }
                if (flat) break;
                m = most;
                if (!out_of_range()) break;
                flat = true;
                if (groups > 4) fill_all();
                team_sync();   // before the next partials
            }
            if (m == NEG_INF) sum = __int_as_float(0x7fc00000);   // no logit above -inf: no distribution
        } else {
            m = pr.stats[row].x;
            sum = pr.stats[row].y;
            flat = out_of_range();
        }
        const float ref = flat ? 0.f : scaled(m), inv_s = 1.f / sum, a = GRAD ? up * pr.grad_factor * w * pr.temperature : 0.f, a_s = a * inv_s;
        const bool wide = GRAD && ((uintptr_t)(grad + sl.head) & 15) == 0;
        auto give_all = [&]() {   // the gradient apart from the teacher's share
            if (!wide) {   // the rows of the gradient lie otherwise in memory than those of the logits (from the slice's start, so that no step leaves 31 bits)
                for (int j = tid; j < to - from; j += TEAM) grad[from + j] = from_float<T>(ex2(fmaf(seen(to_float(z[from + j])), c, -ref)) * a_s);
                return;
            }
            const bool resident = STATS && groups <= 4;
            if (STATS && !resident) fill_all();
            T *out = grad + sl.head + (long long)v_first * VEC;
            auto give = [&](auto is_flat) {
                auto share = [&](uint32_t at) {
                    float f[VEC];
                    unpack<VEC>(load_staged<T, VEC>(at), f);
#pragma unroll
                    for (int e = 0; e < VEC; e++) f[e] = ex2(fmaf(decltype(is_flat)::value ? seen(f[e]) : f[e], c, -ref)) * a_s;
                    Pack<T, VEC> o;
                    pack<VEC>(o, f);
                    return o;
                };
                each(resident, [&](int h, uint32_t at) {
#pragma unroll
                    for (int i = 0; i < GROUP; i++) store_pack<T, VEC>(out + (long long)(h + i) * (TEAM * VEC), share(at + i * HOP));
                }, [&](int h, uint32_t at) {
                    const Pack<T, VEC> o = share(at);
                    if (v_first + h * TEAM < sl.v1) store_pack<T, VEC>(out + (long long)h * (TEAM * VEC), o);
                });
            };
            if (flat) give(std::true_type());
            else give(std::false_type());
            if (r_at >= 0) grad[r_at] = from_float<T>(ex2(fmaf(seen(r_value), c, -ref)) * a_s);
        };
        if (!STATS) {   // before the entries are known: a thread writes the same places again where the row turns out to have none
            if (GRAD && streams) give_all();
            if (GRAD && scribe && state == 0) merge_entries(en, pr.top, from, to, psum);
            team_sync();
        }
        if (TEAM > 32) {
            state = row_state;
            psum = row_psum;
        }

        if (state) {   // the same for every CTA of a cluster
            const float v = state == 1 ? 0.f : __int_as_float(0x7fc00000);
            if (STATS && rank == 0 && tid == 0) {
                pr.row_loss[row] = v;
                pr.stats[row] = make_float2(0.f, 1.f);
            }
            if (GRAD && streams) {
                Pack<T, VEC> o;
#pragma unroll
                for (int e = 0; e < VEC; e++) o.v[e] = from_float<T>(v);
                if (wide) {
                    for (int i = v_first; i < sl.v1; i += TEAM) store_pack<T, VEC>(grad + sl.head + (long long)i * VEC, o);
                    if (r_at >= 0) grad[r_at] = o.v[0];
                } else {
                    for (int j = tid; j < to - from; j += TEAM) grad[from + j] = o.v[0];
                }
            }
        } else {
            if (STATS && GRAD && streams) give_all();
            if (STATS && GRAD && scribe) merge_entries(en, pr.top, from, to, psum);
            if (STATS && scribe && rank == 0) {
                const double log_s = logf(sum), log_p = logf(psum);   // half a step of about 10 at most: what is added to them is exact
                // a logit's share of log q against what S is taken against, halved: the difference stays in range
                auto half_apart = [&](float v) { return (double)(flat ? 0.5f * v - 0.5f * m : 0.5f * v); };
                double loss = 0;
                for (int k = lane; k < pr.top; k += 32)
                    if (en.idx[k] >= 0 && en.prob[k] > 0.f)
                        loss += (double)(en.prob[k] / psum) * (((double)en.diff[k] - log_p) - ((half_apart(en.own[k]) * (double)(2 * c) - (double)ref) * 0.6931471805599453 - log_s));
                loss = warp_sum(loss);
                if (lane == 0) {
                    const double t = pr.temperature;
                    pr.row_loss[row] = (float)(loss * t * t * (double)w * (double)pr.loss_factor);
                    pr.stats[row] = make_float2(m, sum);
                }
            }
            if (GRAD) {
                if (STATS) team_sync();   // the entries' places are written a second time, after the pass above
                for (int k = tid; k < pr.top; k += TEAM == 32 ? 32 : TEAM + 32)
                    if (en.merged[k] >= 0.f) grad[en.idx[k]] = from_float<T>((ex2(fmaf(seen(en.own[k]), c, -ref)) * inv_s - en.merged[k]) * a);
            }
        }
        copy_wait<0>();
        if (row + teams < pr.rows) team_sync();   // before the next row's entries
    }
}

// The rows' losses as one value, in a fixed order.
__global__ void __launch_bounds__(1024) distill_sum_kernel(const float *row_loss, long long rows, double factor, float *loss) {
    __shared__ double part[32];
    ahead_of_previous();
    after_previous();
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
    constexpr int threads = team_threads(TEAM);
    long long grid = TEAM == 32 ? (p.rows + 3) / 4 : p.rows;
    // a pass that may have nothing to do is not worth a CTA for every row: as many as are resident, walking over the rows
    const long long resident = (long long)sm_count() * team_blocks(TEAM, GRAD) / ranks;
    if ((p.skip_one || grid * ranks > 0x7fffffffLL) && grid > resident) grid = resident;
    const long long per_cta = ((long long)p.vocab * (long long)sizeof(T) / 16 + ranks - 1) / ranks;   // vectors of a CTA's slice at most
    // whole warps of vectors: the lanes past a slice have a place too
    const int team_bytes = entry_room(p.top) + (int)(per_cta < TEAM * held_vectors(GRAD) ? (per_cta + 31) / 32 * 32 : TEAM * held_vectors(GRAD)) * 16;
    static PerDeviceOnce once;
    int rc = per_device_once(once, []() -> int {
        GEO_CUDA_CHECK(cudaFuncSetAttribute(distill_kernel<T, TEAM, STATS, GRAD, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, DISTILL_SMEM));
        return GEO_SC_OK;
    });
    if (rc) return rc;
    return launch_behind(distill_kernel<T, TEAM, STATS, GRAD, CLUSTER>, (unsigned)(grid * ranks), threads, (size_t)(TEAM == 32 ? 4 : 1) * team_bytes, s, ranks, p,
                         team_bytes);
}

template <typename T, bool STATS, bool GRAD> int launch_distill(const DistillParams &p, cudaStream_t s) {
    // The smallest team that holds a row, or, for the loss alone, gives every thread some vectors; twice the team, up to
    // eight times, while that still leaves every SM one.
    const long long vectors = (long long)p.vocab * sizeof(T) / 16;
    int team = 32;
    while (team < 2048 && ((GRAD || team < 256 ? vectors > (long long)team * 16 : false) || (p.rows * team < 256LL * sm_count() && vectors > 2 * team))) team *= 2;
    if (team == 32) return launch_team<T, 32, STATS, GRAD, false>(p, 1, s);
    if (team <= 128) return launch_team<T, 128, STATS, GRAD, false>(p, 1, s);
    if (team == 256) return launch_team<T, 256, STATS, GRAD, false>(p, 1, s);
    return launch_team<T, 256, STATS, GRAD, true>(p, team / 256, s);
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
    if (!aligned_to(stats, 8)) return fail(GEO_SC_ERR_UNSUPPORTED, "stats has to start on an 8-byte boundary");
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
        return launch_behind(distill_sum_kernel, 1, 1024, 0, s, 1, (const float *)row_loss, rows, all, loss);
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
    if (!aligned_to(stats, 8)) return fail(GEO_SC_ERR_UNSUPPORTED, "stats has to start on an 8-byte boundary");
    DistillParams p = {};
    p.logits = logits; p.indices = indices; p.teacher = teacher; p.weight = weight; p.upstream = upstream;
    p.stats = (float2 *)const_cast<void *>(stats); p.grad = grad;
    p.rows = rows; p.stride = stride; p.vocab = vocab; p.top = top; p.index64 = index_bits == 64; p.teacher_dtype = teacher_dtype;
    p.upstream_rows = !mean; p.skip_one = skip_one;
    p.temperature = temperature; p.grad_factor = (float)(mean ? (double)scale / (double)rows : (double)scale);
    return launch_typed<false, true>(p, dtype, (cudaStream_t)stream);
}

}  // extern "C"
