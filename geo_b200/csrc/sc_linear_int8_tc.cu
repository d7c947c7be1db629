// The 8-bit matrix product on the fifth-generation tensor cores: tcgen05.mma kind::i8, 32-bit integer accumulators in
// tensor memory, operand tiles brought in by TMA (which fills rows and bytes past the end with zeros, so every size
// takes the same path).
//
// The weights are the 128-lane operand: an accumulator's lane is an output channel and its columns are tokens, so that
// the 32 lanes of a warp store 32 neighbouring channels of one token, for any n, and a lane keeps one weight scale and
// one bias.  A tile is 128 channels x BN tokens of one CTA, or 256 channels x 256 tokens of a pair of CTAs
// (cta_group::2): each of the pair loads its 128 channels and half of the tokens, the even CTA issues the
// instructions for both, and each keeps the accumulators of its own channels.
//
// Where there are fewer tiles than SMs a cluster of 2, 4 or 8 CTAs shares a tile: each sums a part of k and sends every
// column to the shared memory of the CTA that takes it, which adds the parts up behind one barrier of the cluster
// (integers: the order of the additions does not matter).  Sending costs the sender no waiting; fetching the parts behind
// the barrier took 3500 clocks more and a second barrier (256 x 4096 x 4096: 18 us against 12).
//
// What bounds it: with several turns of the pair's tile the time of a stage, 650 clocks for the 32 KB per CTA against 512 of
// its matrix instructions.  With a single turn the start, 3.4 to 5.6 us, and then the stages, each 0.28 to 0.32 us whether
// it brings 20 KB (32 tokens), 24 KB (64) or 32 KB (128, the pair): something fixed per stage and not the bytes, which has
// not been traced further.  So small tiles on many SMs win over large tiles on few as long as one turn holds them
// (choose_tile).  Measured: 8192 x 8192 x 8192 350 us = 3140 TOP/s at best, 400 to 450 us under the power limit,
// 1024 x 4096 x 4096 15.3 us, 256 x 4096 x 4096 10.9 us, 333 x 1001 x 2047 6.8 us.
//
// Persistent CTAs; warp 0 issues the copies, warp 1 the matrix instructions, warps 2 to 9 read finished accumulators
// out while the next tile fills the other buffer.  Every wait is bounded: one that runs out raises a count, and the
// CTA (or pair) stops waiting.  When all its warps have stopped, whichever of them it was that gave up, the copies that were
// asked for and the instructions that were issued get their time to finish (again with a bound) before a CTA leaves.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "sc_linear_int8.h"

namespace geo {

__device__ int g_linear_tc_errors = 0;

namespace {

constexpr int LT_THREADS = 320;
constexpr int LT_EPI_WARPS = 8;
constexpr int LT_KB = 128;                // bytes of k per stage: one 128-byte swizzled row
constexpr int LT_SPIN_LIMIT = 1 << 22;

template <int CTAS, int BN, bool SPLIT> struct LinearTile {
    static constexpr int X_ROWS = BN / CTAS;                                  // token rows that a CTA loads
    static constexpr int STAGE = (128 + X_ROWS) * LT_KB;
    static constexpr int JOIN = SPLIT ? BN * 128 * 4 : 0;                     // parts of the columns that a CTA takes
    static constexpr int ROOM = 212 * 1024 - JOIN;
    static constexpr int STAGES = ROOM / STAGE < 8 ? ROOM / STAGE : 8;
    static constexpr int SMEM = STAGES * STAGE + JOIN + 1024;
    static constexpr uint32_t TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;          // two accumulators
    // kind::i8: 32-bit integers out (2), signed 8-bit A and B (1), both K-major
    static constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(CTAS * 128 >> 4) << 24);
};

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t rank0_address(uint32_t addr) {   // the same place in the pair's even CTA
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(r) : "r"(addr));
    return r;
}
template <int CTAS> __device__ __forceinline__ void mbar_arrive_leader(uint32_t bar) {
    if (CTAS == 1) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
    else asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(rank0_address(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *abort) {
    for (int i = 0; i < LT_SPIN_LIMIT; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023) == 1023 && *abort) return false;
    }
    if (!*abort) {
        *abort = 1;
        atomicAdd(&g_linear_tc_errors, 1);
    }
    return false;
}
// After an abort: whatever is still in flight towards `bar` gets its time to arrive, out of `left` looks for all of them.
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity, int &left) {
    while (left > 0 && !mbar_try_wait(bar, parity)) left--;
}

template <int CTAS> __device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
    if (CTAS == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1)
                     : "memory");
    else   // the barrier is the even CTA's
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];\n"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1)
                     : "memory");
}

// Shared-memory matrix descriptor: K-major rows of 128 bytes under the 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
template <int CTAS>
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if (CTAS == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
                     ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
                     ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
                     : "memory");
}
template <int CTAS> __device__ __forceinline__ void umma_commit(uint32_t bar) {   // on the barrier of every CTA of the tile
    if (CTAS == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
                     ::"r"(bar), "h"((uint16_t)3)
                     : "memory");
}
template <int CTAS> __device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
    if (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
}
template <int CTAS> __device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    if (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(base), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(base), "r"(cols) : "memory");
}
#define LT_OUT(i) "=r"(r[i])
#define LT_INOUT(i) "+r"(r[i])
#define LT_REGS16(x) x(0), x(1), x(2), x(3), x(4), x(5), x(6), x(7), x(8), x(9), x(10), x(11), x(12), x(13), x(14), x(15)
// 16 columns of the warp's 32 lanes; the registers may be read after tmem_ld_wait (they pass through it, so that nothing
// that reads them moves up).
__device__ __forceinline__ void tmem_ld(uint32_t taddr, int (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                 : LT_REGS16(LT_OUT)
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(int (&r)[16]) { asm volatile("tcgen05.wait::ld.sync.aligned;\n" : LT_REGS16(LT_INOUT) : : "memory"); }
__device__ __forceinline__ void store_remote(uint32_t addr, int cta, int a, int b, int c, int d) {   // at the same place in another CTA of the cluster
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(cta));
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(r), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <bool CLUSTER> __device__ __forceinline__ void tile_sync() {   // all threads of the CTA, or of the cluster
    if (!CLUSTER) __syncthreads();
    else asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}

// SPLIT: a cluster shares one tile and splits k; else CTAs (or pairs of them) walk over the tiles.
template <typename T, int CTAS, int BN, bool SPLIT>
__global__ void __launch_bounds__(LT_THREADS, 1)
linear_int8_tc_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, LinearParams pr, int ntiles_n, int ntiles, int splits) {
    using Tile = LinearTile<CTAS, BN, SPLIT>;
    constexpr int ST = Tile::STAGES, COLS = BN / 2;   // columns of an epilogue warp: two warps share a lane quarter
    constexpr int CH = 16;                            // columns read out at a time
    extern __shared__ unsigned char lt_smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * ST + 5];   // full, empty, acc_full[2], acc_empty[2], drain
    __shared__ __align__(16) float scales[LT_EPI_WARPS][COLS];
    __shared__ __align__(16) float split_x[SPLIT ? BN : 1], split_w[SPLIT ? 128 : 1], split_b[SPLIT ? 128 : 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ __align__(16) int other[4];   // of the pair's other CTA, told at the end: whether it gave up, stages it asked for
    const uint32_t tiles = (smem_u32(lt_smem_raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CTAS == 1 ? 0 : (int)(blockIdx.x & 1);
    const int part = SPLIT ? (int)blockIdx.x % splits : 0;
    const int worker = SPLIT ? blockIdx.x / splits : blockIdx.x / CTAS, workers = SPLIT ? ntiles : gridDim.x / CTAS;
    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (ST + s); };
    auto accf_bar = [&](int a) { return bar0 + 8u * (2 * ST + a); };
    auto acce_bar = [&](int a) { return bar0 + 8u * (2 * ST + 2 + a); };
    const uint32_t drain_bar = bar0 + 8u * (2 * ST + 4);
    const uint32_t join = tiles + ST * Tile::STAGE;
    const int share = SPLIT ? BN / splits : BN;   // columns that a CTA takes: a power of two
    volatile int *abort = &abort_flag;

    ahead_of_previous();
    if (threadIdx.x == 32 * 2) {   // the first copies would wait for these
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map_x) : "memory");
    }
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < ST; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; a++) { mbar_init(accf_bar(a), 1); mbar_init(acce_bar(a), LT_EPI_WARPS * CTAS); }
        mbar_init(drain_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\nfence.proxy.async.shared::cta;\n" ::: "memory");
    }
    if (warp == 1) tmem_alloc<CTAS>(smem_u32(&tmem_slot), Tile::TMEM_COLS);
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    if (CTAS == 2) {
        __syncthreads();
        tile_sync<true>();
    } else if (warp == 0) {   // the first copies need the barriers only, which this warp has made: it does not wait for the others
        __syncwarp();
        asm volatile("barrier.cta.arrive.aligned 1, %0;\n" ::"n"(LT_THREADS) : "memory");
    } else {
        asm volatile("barrier.cta.sync.aligned 1, %0;\n" ::"n"(LT_THREADS) : "memory");
    }
    // SPLIT: the other CTAs have to have begun before anything is sent to them; every thread waits for that when it can
    if (SPLIT) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
    auto cluster_begun = [&]() {
        if (SPLIT) asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
    };
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem_base = CTAS == 1 && warp == 0 ? 0 : tmem_slot;   // not that warp's to read
    const int all_kb = (pr.k + LT_KB - 1) / LT_KB;
    after_previous();
    int asked = 0;   // stages that this CTA has asked for (in the thread that asks)
    const int kb0 = SPLIT ? all_kb * part / splits : 0, kb1 = SPLIT ? all_kb * (part + 1) / splits : all_kb;   // all_kb <= 1024

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (int t = worker; t < ntiles && ok; t += workers) {
                const int n0 = (t % ntiles_n) * 128 * CTAS + rank * 128, m0 = (t / ntiles_n) * BN + rank * Tile::X_ROWS;
                for (int kb = kb0; kb < kb1; kb++, asked++) {
                    const int s = asked % ST;
                    if (!(ok = mbar_wait(empty_bar(s), ((asked / ST) & 1) ^ 1, abort))) break;
                    if (rank == 0) mbar_expect_tx(full_bar(s), (uint32_t)(CTAS * Tile::STAGE));
                    const uint32_t dst = tiles + (uint32_t)s * Tile::STAGE;
                    const uint32_t bar = CTAS == 1 ? full_bar(s) : rank0_address(full_bar(s));
                    tma_load<CTAS>(dst, &map_w, bar, kb * LT_KB, n0);
                    tma_load<CTAS>(dst + 128 * LT_KB, &map_x, bar, kb * LT_KB, m0);
                }
            }
        }
        __syncwarp();
        cluster_begun();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int it = 0, n = 0;
            bool ok = true;
            for (int t = worker; t < ntiles && ok; t += workers, n++) {
                const int a = n & 1;
                if (!(ok = mbar_wait(acce_bar(a), ((n >> 1) & 1) ^ 1, abort))) break;
                for (int kb = kb0; kb < kb1; kb++, it++) {
                    const int s = it % ST;
                    if (!(ok = mbar_wait(full_bar(s), (it / ST) & 1, abort))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const uint32_t st = tiles + (uint32_t)s * Tile::STAGE;
                    const uint64_t adesc = umma_desc(st), bdesc = umma_desc(st + 128 * LT_KB);
#pragma unroll
                    for (int k = 0; k < LT_KB / 32; k++)   // 32 bytes further along k: + 2 in units of 16 bytes
                        umma_i8<CTAS>(tmem_base + a * BN, adesc + 2 * k, bdesc + 2 * k, Tile::IDESC, (kb - kb0) | k ? 1u : 0u);
                    umma_commit<CTAS>(empty_bar(s));
                }
                if (ok) umma_commit<CTAS>(accf_bar(a));
            }
        }
        __syncwarp();
        cluster_begun();
    } else {
        const int ew = warp - 2, quarter = warp & 3, half = ew >> 2;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * COLS;
        // the scales of a tile, asked for one tile ahead
        constexpr int XS = (COLS + 31) / 32;
        float xs[XS], ws = 0.f, b = 0.f;
        auto ask_scales = [&](int t) {
            const int n0 = (t % ntiles_n) * 128 * CTAS + rank * 128 + quarter * 32 + lane, m0 = (t / ntiles_n) * BN + half * COLS;
            ws = t < ntiles && n0 < pr.n ? pr.w_scale[n0] : 0.f;
            b = t < ntiles && pr.bias && n0 < pr.n ? pr.bias[n0] : 0.f;
#pragma unroll
            for (int i = 0; i < XS; i++) xs[i] = t < ntiles && i * 32 + lane < COLS && m0 + i * 32 + lane < pr.m ? pr.x_scale[m0 + i * 32 + lane] : 0.f;
        };
        ask_scales(worker);
        if (SPLIT) {   // for the whole CTA, which shares out the columns
            if (half == 0) {
                split_w[quarter * 32 + lane] = ws;
                split_b[quarter * 32 + lane] = b;
            }
            if (quarter == 0)
#pragma unroll
                for (int i = 0; i < XS; i++)
                    if (i * 32 + lane < COLS) split_x[half * COLS + i * 32 + lane] = xs[i];
        }
        cluster_begun();
        int n = 0;
        for (int t = worker; t < ntiles; t += workers, n++) {
            const int a = n & 1;
            const int ch = (t % ntiles_n) * 128 * CTAS + rank * 128 + quarter * 32 + lane, m0 = (t / ntiles_n) * BN + half * COLS;
            const float w_now = ws, b_now = b;
            if (!SPLIT) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < XS; i++)
                    if (i * 32 + lane < COLS) scales[ew][i * 32 + lane] = xs[i];
                __syncwarp();
                ask_scales(t + workers);
            }
            if (!__all_sync(0xffffffffu, mbar_wait(accf_bar(a), (n >> 1) & 1, abort))) break;   // a warp stops as a whole
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            T *out = (T *)pr.out + (long long)m0 * pr.out_stride + ch;
            const bool paired = sizeof(T) == 2 && pr.out_stride % 2 == 0 && pr.n % 2 == 0 && ((uintptr_t)pr.out & 3) == 0;
            const int tokens = min(COLS, pr.m - m0);   // of this warp's columns
            auto process = [&](const int (&v)[CH], int c) {
                if constexpr (SPLIT) {   // [part][four columns of their taker][128 channels][column]
#pragma unroll
                    for (int j = 0; j < CH; j += 4) {
                        const int col = half * COLS + c + j;
                        store_remote(join + (uint32_t)(((part * share + (col & (share - 1))) >> 2) * 128 + quarter * 32 + lane) * 16u, col / share, v[j], v[j + 1], v[j + 2], v[j + 3]);
                    }
                } else if (c + CH <= tokens && paired) {
                    // two tokens at a time: the even lane of a pair of channels stores both of one token, the odd lane of the other
                    T *at = lane & 1 ? out + pr.out_stride - 1 : out;
#pragma unroll
                    for (int j = 0; j < CH; j += 2, at += 2 * pr.out_stride) {
                        const float y0 = (float)v[j] * scales[ew][c + j] * w_now + b_now, y1 = (float)v[j + 1] * scales[ew][c + j + 1] * w_now + b_now;
                        const float other = __shfl_xor_sync(0xffffffffu, lane & 1 ? y0 : y1, 1);
                        Pack<T, 2> o;
                        const float f[2] = {lane & 1 ? other : y0, lane & 1 ? y1 : other};
                        pack<2>(o, f);
                        if (ch < pr.n) store_pack<T, 2>(at, o);
                    }
                } else if (c + CH <= tokens) {
                    T *at = out;
#pragma unroll
                    for (int j = 0; j < CH; j++, at += pr.out_stride) {
                        const T y = from_float<T>((float)v[j] * scales[ew][c + j] * w_now + b_now);
                        if (ch < pr.n) *at = y;
                    }
                } else if (c < tokens) {
                    T *at = out;
#pragma unroll
                    for (int j = 0; j < CH; j++, at += pr.out_stride)
                        if (ch < pr.n && c + j < tokens) *at = from_float<T>((float)v[j] * scales[ew][c + j] * w_now + b_now);
                }
                out += CH * pr.out_stride;
            };
            // the next columns are read out of tensor memory while these are stored
            int va[CH], vb[CH];
            tmem_ld(lane_addr + a * BN, va);
            if constexpr (COLS == CH) {
                tmem_ld_wait(va);
                process(va, 0);
            } else {
#pragma unroll 1
                for (int c = 0; c < COLS; c += 2 * CH) {
                    tmem_ld_wait(va);
                    tmem_ld(lane_addr + a * BN + c + CH, vb);
                    process(va, c);
                    tmem_ld_wait(vb);
                    if (c + 2 * CH < COLS) tmem_ld(lane_addr + a * BN + c + 2 * CH, va);
                    process(vb, c + CH);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_leader<CTAS>(acce_bar(a));
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (CTAS == 2 && threadIdx.x == 0) store_remote(smem_u32(other), rank ^ 1, abort_flag, asked, 0, 0);
    tile_sync<CTAS == 2 || SPLIT>();   // nobody leaves while another CTA may still reach its barriers; SPLIT: all parts are there
    if (abort_flag || (CTAS == 2 && other[0])) {   // the same for both of a pair
        int left = LT_SPIN_LIMIT;
        if (rank == 0 && threadIdx.x == 0) {   // copies: the stages that were asked for last, by either
            const int last = CTAS == 2 ? max(asked, other[1]) : asked;
            for (int i = last < ST ? 0 : last - ST; i < last; i++) {
                if (i >= asked) mbar_expect_tx(full_bar(i % ST), (uint32_t)Tile::STAGE);   // by the odd CTA alone
                mbar_drain(full_bar(i % ST), (i / ST) & 1, left);
            }
        } else if (rank == 0 && threadIdx.x == 32) {   // instructions: they read shared memory and write tensor memory
            umma_commit<CTAS>(drain_bar);
            mbar_drain(drain_bar, 0, left);
        }
        __syncthreads();
        tile_sync<CTAS == 2>();
    }
    if (SPLIT) {
        // a warp adds up 32 channels of four tokens
        const int n0 = (worker % ntiles_n) * 128, m0 = (worker / ntiles_n) * BN + part * share;
        for (int i = warp; i < share; i += LT_THREADS / 32) {   // share / 4 groups of tokens x 4 of channels
            const int group = i >> 2, l = (i & 3) * 32 + lane, ch = n0 + l, m = m0 + group * 4;
            if (m >= pr.m || ch >= pr.n) continue;
            int sum[4] = {0, 0, 0, 0};
            for (int r = 0; r < splits; r++) {
                int4 v;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(join + (uint32_t)((((r * share) >> 2) + group) * 128 + l) * 16u));
                sum[0] += v.x;
                sum[1] += v.y;
                sum[2] += v.z;
                sum[3] += v.w;
            }
            T *out = (T *)pr.out + (long long)m * pr.out_stride + ch;
#pragma unroll
            for (int j = 0; j < 4; j++, out += pr.out_stride)
                if (m + j < pr.m) *out = from_float<T>((float)sum[j] * split_x[part * share + group * 4 + j] * split_w[l] + split_b[l]);
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        tmem_free<CTAS>(tmem_base, Tile::TMEM_COLS);
    }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                   const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static std::once_flag once;
    static EncodeTiledFn fn = nullptr;
    std::call_once(once, []() {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)p;
    });
    return fn;
}

int encode_rows(CUtensorMap *map, const int8_t *base, int k, int rows, long long stride, int box_rows) {
    if (!encode_fn()) return fail(GEO_SC_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {LT_KB, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? GEO_SC_OK : fail(GEO_SC_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", (int)r);
}

template <typename T, int CTAS, int BN, bool SPLIT> int launch_tile(const LinearParams &p, int splits, cudaStream_t s) {
    using Tile = LinearTile<CTAS, BN, SPLIT>;
    CUtensorMap map_w, map_x;
    int rc = encode_rows(&map_w, p.w, p.k, p.n, p.w_stride, 128);
    if (!rc) rc = encode_rows(&map_x, p.x, p.k, p.m, p.x_stride, Tile::X_ROWS);
    if (rc) return rc;
    static PerDeviceOnce once;
    rc = per_device_once(once, []() -> int {
        GEO_CUDA_CHECK(cudaFuncSetAttribute(linear_int8_tc_kernel<T, CTAS, BN, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile::SMEM));
        return GEO_SC_OK;
    });
    if (rc) return rc;
    const int tn = (p.n + 128 * CTAS - 1) / (128 * CTAS);
    const long long tiles = (long long)tn * ((p.m + BN - 1) / BN);
    if (tiles > 0x3fffffff) return fail(GEO_SC_ERR_TOO_LARGE, "%d tokens x %d channels", p.m, p.n);
    const int workers = SPLIT ? (int)tiles : (int)(tiles < sm_count() / CTAS ? tiles : sm_count() / CTAS), cluster = SPLIT ? splits : CTAS;
    return launch_behind(linear_int8_tc_kernel<T, CTAS, BN, SPLIT>, (unsigned)(workers * cluster), LT_THREADS, Tile::SMEM, s, cluster, map_w, map_x, p, tn, (int)tiles, splits);
}

// The tile and the split of k with the least estimated time, in units of 10 ns.  Measured over products of 12 to 2000
// tokens (CUDA-graph replay): a call with one turn takes `start` and `stage` for each 128 bytes of k, whatever the number
// of CTAs; every further turn its stages and 0.6 us, or the stores of a tile (`stores`) where they take longer; sending
// and joining the parts of a split tile takes `join`.  So small tiles win while a turn holds them all (123 x 1920 x 944:
// 32 tokens 6.0 us, 128 tokens 7.4, a pair 8.6), large ones when there are several (378 x 6812 x 3765: a pair 15.3 us,
// 64 tokens 30.6), and a split of k pays where few tiles have a long k (50 x 500 x 8000: 6.8 us by 8, 21.0 whole).
struct TileChoice { int pair, bn, splits; };
struct TileTimes { int pair, bn, start, stage, stores, join; };
TileChoice choose_tile(const LinearParams &p) {
    constexpr TileTimes TIMES[] = {{0, 32, 340, 28, 90, 130}, {0, 64, 350, 29, 130, 200}, {0, 128, 430, 31, 250, 290}, {1, 256, 560, 32, 340, 0}};
    const long long sms = sm_count(), kb = (p.k + LT_KB - 1) / LT_KB;
    TileChoice best{0, 64, 1};
    long long least = -1;
    for (const TileTimes &t : TIMES) {
        const long long ctas = t.pair ? 2 : 1, tiles = ((p.n + 128 * ctas - 1) / (128 * ctas)) * ((p.m + t.bn - 1) / t.bn);
        for (int splits = 1; splits <= (t.pair ? 1 : 8); splits *= 2) {
            if (splits > 1 && (tiles * splits > sms || kb < 2 * splits)) break;
            const long long turns = (tiles * ctas * splits + sms - 1) / sms, stages = (kb + splits - 1) / splits * t.stage;
            const long long cost = t.start + stages + (turns - 1) * std::max(stages + 60, (long long)t.stores) + (splits > 1 ? t.join : 0);
            if (least < 0 || cost < least) {
                least = cost;
                best = TileChoice{t.pair, t.bn, splits};
            }
        }
    }
    return best;
}

template <typename T> int launch_tc(const LinearParams &p, cudaStream_t s) {
    const TileChoice c = choose_tile(p);
    if (c.pair) return launch_tile<T, 2, 256, false>(p, 1, s);
    if (c.splits > 1) {
        if (c.bn == 128) return launch_tile<T, 1, 128, true>(p, c.splits, s);
        if (c.bn == 64) return launch_tile<T, 1, 64, true>(p, c.splits, s);
        return launch_tile<T, 1, 32, true>(p, c.splits, s);
    }
    if (c.bn == 128) return launch_tile<T, 1, 128, false>(p, 1, s);
    if (c.bn == 64) return launch_tile<T, 1, 64, false>(p, 1, s);
    return launch_tile<T, 1, 32, false>(p, 1, s);
}

}  // namespace

int launch_linear_int8_tc(const LinearParams &p, int dtype, cudaStream_t s) {
    if (dtype == GEO_SC_DTYPE_F32) return launch_tc<float>(p, s);
    if (dtype == GEO_SC_DTYPE_BF16) return launch_tc<__nv_bfloat16>(p, s);
    return launch_tc<__half>(p, s);
}

int linear_int8_tc_error_count(int *count) {
    GEO_CUDA_CHECK(cudaMemcpyFromSymbol(count, g_linear_tc_errors, sizeof(int)));
    return GEO_SC_OK;
}

}  // namespace geo
