// Products grouped by expert on pairs of SMs (no reference counterpart): the forward product for many rows per expert,
// and the weight gradient.
//
//   k_mm_wide   y[t] = w[e(t)] x[t]           D = W X^T: 256 features x up to 256 of one expert's rows
//   k_mm_wgrad  dw[e] = sum_t dy[t] x[t]^T    D = dy^T x: 256 features x up to 256 columns of x, over e's rows
//
// One tcgen05.mma.cta_group::2 works on both SMs of a pair (a cluster of two CTAs): each CTA holds the accumulators of
// 128 of the 256 features, its own half of A and half of B, so a 64-element stage costs each SM 32 KB of shared memory
// and of L2 traffic for 512 cycles of products; a 128 x 256 tile on one SM would need 48 KB.  Five stages in flight, two
// accumulators of 256 TMEM columns: the epilogue of one tile overlaps the products of the next.  The grid is one pair
// per two SMs, each pair taking tiles in turn; the pipeline runs on from tile to tile.
//
// Barriers.  full[s] (used in the first CTA of the pair, the leader, whose thread issues the products): both CTAs' copies
// of stage s; empty[s] and tfull[b] (both CTAs): signalled by the products' commit to both; tempty[b] (leader): the
// sixteen epilogue warps have read accumulator b.
#include "mm.cuh"

namespace spq {
namespace {

using namespace mm;

// warps 0-7: epilogue (TMEM lanes 32 (w % 4) .., columns by w / 4), 8 and 9: copies of A and of B, 10: products.  The issue
// of the copies is on the critical path (a stage lasts 512 cycles): one warp for both operands held the weight gradient
// to 1340 TFLOP/s where two give 1500 (16384 rows, 8 experts of 5120x2048, bf16).
constexpr int THREADS = 352;
constexpr int COPY_A = 8, COPY_B = 9, PRODUCTS = 10;
constexpr int STAGES = 5;           // (four cost up to 7 %, six gave no more)
constexpr int HALF = FT * BK * 2;  // one operand half: 128 x 64 elements, 16 KB
constexpr int STAGE = 2 * HALF;
constexpr int NT = 256;            // columns of a tile
constexpr int STAGING = STAGES * STAGE;       // wgrad: 32 rows x 128 bytes of results per epilogue warp
constexpr int BARS = STAGING + 8 * 4096;
constexpr int MAPS = BARS + 256;
constexpr int FIXED = MAPS + 16 + 1024;
// wgrad: stages (of 64 rows) summed in TMEM before they are added in registers
template <typename OUT>
constexpr int DRAIN = sizeof(OUT) == 4 ? 8 : 32;

// ---- cta_group::2 forms ----
__device__ __forceinline__ void mma2_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrive on `bar` of both CTAs when every product this thread issued before has completed
__device__ __forceinline__ void commit2(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void tmem_alloc2(uint32_t* dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(dst_smem)),
                 "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// copies into this CTA's shared memory whose bytes count on a barrier of either CTA of the pair (`bar`: a cluster address)
__device__ __forceinline__ void tma2_load_3d(uint32_t smem_dst, const void* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma2_load_2d(uint32_t smem_dst, const void* map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%2, %3}], [%4];" ::"r"(smem_dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
// a tile of 32 rows x 128 bytes to global memory, one bulk group each
__device__ __forceinline__ void tma_store_3d(const void* map, int c0, int c1, int c2, uint32_t smem_src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(c0),
                 "r"(c1), "r"(c2), "r"(smem_src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// the bounded wait on a barrier that the other CTA arrives on
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, uint64_t limit_ns = 2000000000ull) {
    const uint64_t t0 = tc::globaltimer();
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(tc::smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if (tc::globaltimer() - t0 > limit_ns) return false;
    }
}

// the pair's shared state, set up before any role begins
struct Pair {
    char* sm;
    uint64_t *full, *empty, *tfull, *tempty;
    uint64_t *ragged, *zeroed;   // wgrad: this CTA's copies of a ragged stage; (leader) the other CTA's part of stage s is zeroed
    volatile int* err;
    int *start, *pre;
    uint32_t tmem;
    int rank;
    uint32_t full0, tempty0, zeroed0;   // cluster addresses of the leader's barriers
};

__device__ __forceinline__ Pair set_up(char* dyn, const int* offsets, int E, int T, int rows_per_tile) {
    Pair p;
    p.sm = dyn + ((1024u - (tc::smem_u32(dyn) & 1023u)) & 1023u);
    p.full = reinterpret_cast<uint64_t*>(p.sm + BARS);
    p.empty = p.full + STAGES;
    p.tfull = p.empty + STAGES;
    p.tempty = p.tfull + 2;
    p.ragged = p.tempty + 2;
    p.zeroed = p.ragged + 1;
    uint32_t* const slot = reinterpret_cast<uint32_t*>(p.sm + MAPS);
    p.err = reinterpret_cast<int*>(p.sm + MAPS + 4);
    p.start = reinterpret_cast<int*>(p.sm + MAPS + 16);
    p.pre = p.start + E + 1;
    p.rank = (int)cluster_rank();
    const int warp = threadIdx.x >> 5;
    if (warp == 0) map_groups(offsets, E, T, rows_per_tile, p.start, p.pre);
    if (warp == PRODUCTS) tmem_alloc2(slot, 2 * NT);
    if (threadIdx.x == 256) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&p.full[s], 1);
            tc::mbar_init(&p.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&p.tfull[b], 1);
            tc::mbar_init(&p.tempty[b], 16);
        }
        tc::mbar_init(p.ragged, 1);
        for (int s = 0; s < STAGES; ++s) tc::mbar_init(&p.zeroed[s], 1);
        tc::mbar_fence_init();
        *p.err = 0;
    }
    tc::fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    tc::fence_after_sync();
    p.tmem = *slot;
    p.full0 = mapa(tc::smem_u32(p.full), 0);
    p.tempty0 = mapa(tc::smem_u32(p.tempty), 0);
    p.zeroed0 = mapa(tc::smem_u32(p.zeroed), 0);
    return p;
}

// no CTA of the pair leaves while the other may still signal its barriers or read its operands
__device__ __forceinline__ void tear_down(const Pair& p, int* status) {
    __syncwarp();
    tc::fence_before_sync();
    cluster_sync_all();
    if ((threadIdx.x >> 5) == PRODUCTS) tmem_dealloc2(p.tmem, 2 * NT);
    if (threadIdx.x == 0 && *p.err) atomicOr(status, MM_TIMEOUT);
}

// a role's place in the ring of stages
struct Ring {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++s == STAGES) {
            s = 0;
            phase ^= 1;
        }
    }
};

// the wait for the ring's stage to be free (a barrier's first wait, for the phase before its first, returns at once)
__device__ __forceinline__ bool stage_free(const Pair& p, const Ring& r) {
    if (!*p.err && tc::mbar_wait(&p.empty[r.s], r.phase ^ 1)) return true;
    *p.err = 1;
    return false;
}
// the end of the copies: the products have released every stage (so no signal is on its way to a barrier of a CTA that
// is gone), or, after a limit ran out, the leader has seen both CTAs' copies arrive
__device__ __forceinline__ void finish_copies(const Pair& p, Ring r) {
    if (!*p.err) {
        for (int n = 0; n < STAGES; ++n, r.next())
            if (!tc::mbar_wait(&p.empty[r.s], r.phase ^ 1)) *p.err = 1;
    } else if (p.rank == 0) {
        for (int s = 0; s < STAGES; ++s) tc::mbar_wait(&p.full[s], s < r.s ? r.phase : r.phase ^ 1);
    }
}

__device__ __forceinline__ int up32(int n) { return (n + 31) & ~31; }

template <bool W_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    k_mm_wide(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx, const MmArgs a) {
    extern __shared__ char dyn[];
    const Pair p = set_up(dyn, a.offsets, a.E, a.T, NT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ntn = a.ntn, tiles = p.pre[a.E] * ntn, pairs = (int)gridDim.x / 2;
    const int kb = (a.K + BK - 1) / BK;
    struct Tile {
        int e, n0, t0, t1, cols;   // cols: the tile's rows of x, up to a multiple of 32
    };
    auto tile_at = [&](int i) {
        const int u = i / ntn;
        Tile t;
        t.n0 = (i - u * ntn) * 2 * FT;
        t.e = group_of(p.pre, a.E, u);
        t.t0 = p.start[t.e] + (u - p.pre[t.e]) * NT;
        t.t1 = min(p.start[t.e + 1], t.t0 + NT);
        t.cols = up32(t.t1 - t.t0);
        return t;
    };

    // the copy and product warps run their loops whole (their state stays in uniform registers, which TMA and tcgen05
    // operands need); one thread issues
    if (warp == COPY_A) {
        const bool one = elect();
        Ring r;
        bool ok = true;
        for (int t = (int)blockIdx.x / 2; ok && t < tiles; t += pairs) {
            const Tile d = tile_at(t);
            const int n = d.n0 + p.rank * FT;
            for (int k = 0; k < kb; ++k, r.next()) {
                if (!(ok = __all_sync(~0u, stage_free(p, r)))) break;
                if (one) {
                    const uint32_t as = tc::smem_u32(p.sm) + r.s * STAGE, bar = p.full0 + r.s * 8;
                    if (p.rank == 0) tc::mbar_expect_tx(&p.full[r.s], 2 * STAGE);
                    if (W_MN) {
                        tma2_load_3d(as, &tw, n, k * BK, d.e, bar);
                        tma2_load_3d(as + BOX_MN, &tw, n + 64, k * BK, d.e, bar);
                    } else {
                        tma2_load_3d(as, &tw, k * BK, n, d.e, bar);
                    }
                }
                __syncwarp();
            }
        }
        finish_copies(p, r);
    } else if (warp == COPY_B) {
        const bool one = elect();
        Ring r;
        bool ok = true;
        for (int t = (int)blockIdx.x / 2; ok && t < tiles; t += pairs) {
            const Tile d = tile_at(t);
            const int row = d.t0 + p.rank * (d.cols / 2);
            for (int k = 0; k < kb; ++k, r.next()) {
                if (!(ok = __all_sync(~0u, stage_free(p, r)))) break;
                if (one)
                    tma2_load_2d(tc::smem_u32(p.sm) + r.s * STAGE + HALF, &tx, k * BK, row, p.full0 + r.s * 8);
                __syncwarp();
            }
        }
    } else if (warp == PRODUCTS) {
        if (p.rank == 0) {
            const bool one = elect();
            const uint64_t a0 = sdesc<W_MN>(tc::smem_u32(p.sm)), b0 = sdesc<false>(tc::smem_u32(p.sm) + HALF);
            Ring r;
            int j = 0;
            for (int t = (int)blockIdx.x / 2; t < tiles && !*p.err; t += pairs, ++j) {
                const Tile d = tile_at(t);
                const int b = j & 1;
                const uint32_t acc = p.tmem + b * NT, id = idesc_f16(2 * FT, d.cols, a.bf16, W_MN, false);
                if (j >= 2 && !tc::mbar_wait(&p.tempty[b], (uint32_t)((j / 2 - 1) & 1))) *p.err = 1;
                tc::fence_after_sync();
                for (int k = 0; k < kb; ++k) {
                    if (*p.err || !tc::mbar_wait(&p.full[r.s], r.phase)) {
                        *p.err = 1;
                        break;
                    }
                    tc::fence_after_sync();
                    if (one) {
#pragma unroll
                        for (int q = 0; q < BK / 16; ++q)
                            mma2_f16(acc, a0 + ((r.s * STAGE + q * kstep<W_MN>()) >> 4), b0 + ((r.s * STAGE + q * kstep<false>()) >> 4),
                                     id, k > 0 || q > 0);
                        commit2(&p.empty[r.s]);
                    }
                    r.next();
                }
                if (one) commit2(&p.tfull[b]);
            }
        }
    } else {
        const bool v16 = a.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
        const int q = warp & 3, half = warp >> 2;
        const uint32_t stage = tc::smem_u32(p.sm) + STAGING + warp * Y_STAGE;
        if (a.zero_tail) {   // rows behind the last expert
            for (long long t = p.start[a.E] + (long long)blockIdx.x; t < a.T; t += gridDim.x)
                for (int n = threadIdx.x; n < a.N; n += 256) a.y[t * a.ldy + n] = 0;
        }
        int j = 0;
        for (int t = (int)blockIdx.x / 2; t < tiles; t += pairs, ++j) {
            const Tile d = tile_at(t);
            const int b = j & 1;
            const bool ok = !*p.err && tc::mbar_wait(&p.tfull[b], (uint32_t)((j / 2) & 1));
            if (!__all_sync(~0u, ok)) {
                *p.err = 1;
                break;
            }
            tc::fence_after_sync();
            const int n = d.n0 + p.rank * FT + q * 32;
            if (n < a.N)
                for (int c = half * 32; c < d.cols; c += 64)
                    store_y32(p.tmem + b * NT + c + ((uint32_t)(q * 32) << 16), stage, a.y + (long long)(d.t0 + c) * a.ldy + n,
                              a.ldy, d.t1 - d.t0 - c, a.N - n, a.bf16, v16);
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_cluster(p.tempty0 + b * 8);
        }
    }
    tear_down(p, a.status);
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// a warp's staged results to rows of dw that do not start on 16 bytes
template <typename OUT>
__device__ __forceinline__ void store_rows(const char* stage, OUT* row, int ld, int rows, int cols) {
#pragma unroll 1
    for (int x = 0; x < rows; ++x, row += ld)
#pragma unroll 1
        for (int y = threadIdx.x & 31; y < cols; y += 32) {
            const int at = y * (int)sizeof(OUT);
            row[y] = *reinterpret_cast<const OUT*>(stage + x * 128 + (((at >> 4) ^ (x & 7)) << 4) + (at & 15));
        }
    __syncwarp();
}

// whether a stage with `left` rows of its expert ends inside one product's 16
__device__ __forceinline__ bool ragged(int left) { return left < BK && left % 16 != 0; }

// The tensor core rounds toward zero each time it adds 16 products to its fp32 accumulator: over n additions of terms of
// random sign the sum comes out about n * 3e-8 of itself too small.  So the accumulator is taken every DRAIN stages and
// added to fp32 sums in registers, rounded to nearest, while the products go on in the other accumulator.  For fp32
// results every 512 rows (measured 4e-7 off in all at 5000 rows, as a sum in fp32 is); for 16-bit results, whose own
// rounding is 2^-9 or 2^-12, every 2048, which keeps the bias from growing with the length.  The reads of TMEM
// take tensor-core time: 16384 rows, 8 experts of 5120x2048 in bf16: 285 us with a drain every 256 rows, 258 every 512, 252 every 4096.
template <typename OUT, bool TMA_OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    k_mm_wgrad(const __grid_constant__ CUtensorMap tdy, const __grid_constant__ CUtensorMap tx,
               const __grid_constant__ CUtensorMap tdw, const MmWgradArgs a) {
    extern __shared__ char dyn[];
    const Pair p = set_up(dyn, a.offsets, a.E, a.T, 1 << 30);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ntn = (a.N + 2 * FT - 1) / (2 * FT), ntk = (a.K + NT - 1) / NT, per = ntn * ntk;
    const long long tiles = (long long)a.E * per;
    const int pairs = (int)gridDim.x / 2;
    struct Tile {
        int e, n0, k0, cols, r0, rows, nb;   // cols: the tile's columns of x up to a multiple of 32; nb: stages of 64 rows
    };
    auto tile_at = [&](long long i) {
        Tile t;
        t.e = (int)(i / per);
        const int l = (int)(i - (long long)t.e * per);
        t.n0 = l / ntk * 2 * FT;
        t.k0 = l % ntk * NT;
        t.cols = min(NT, up32(a.K - t.k0));
        t.r0 = p.start[t.e];
        t.rows = p.start[t.e + 1] - t.r0;
        t.nb = (t.rows + BK - 1) / BK;
        return t;
    };

    if (warp == COPY_A) {
        const bool one = elect();
        Ring r;
        uint32_t ragged_phase = 0, zeroed_phases = 0;   // (bit s: that of zeroed[s])
        bool ok = true;
        for (long long t = blockIdx.x / 2; ok && t < tiles; t += pairs) {
            const Tile d = tile_at(t);
            const int n = d.n0 + p.rank * FT, k = d.k0 + p.rank * (d.cols / 2);
            for (int c = 0; c < d.nb; ++c, r.next()) {
                if (!(ok = __all_sync(~0u, stage_free(p, r)))) break;
                const int left = d.rows - c * BK, row = d.r0 + c * BK;
                const uint32_t as = tc::smem_u32(p.sm) + r.s * STAGE;
                if (!ragged(left)) {
                    if (one) {
                        const uint32_t bar = p.full0 + r.s * 8;
                        if (p.rank == 0) tc::mbar_expect_tx(&p.full[r.s], 2 * STAGE);
                        tma2_load_2d(as, &tdy, n, row, bar);
                        tma2_load_2d(as + BOX_MN, &tdy, n + 64, row, bar);
                    }
                    __syncwarp();
                    continue;
                }
                // the expert's last rows, not a multiple of one product's 16: the rows behind them (another expert's) are
                // zeroed in both operands before the products may read the stage
                if (one) {
                    const uint32_t bar = tc::smem_u32(p.ragged);
                    tc::mbar_expect_tx(p.ragged, STAGE);
                    mm::tma_load_2d(as, &tdy, n, row, bar);
                    mm::tma_load_2d(as + BOX_MN, &tdy, n + 64, row, bar);
                    mm::tma_load_2d(as + HALF, &tx, k, row, bar);
                    mm::tma_load_2d(as + HALF + BOX_MN, &tx, k + 64, row, bar);
                }
                __syncwarp();
                ok = __all_sync(~0u, tc::mbar_wait(p.ragged, ragged_phase));
                ragged_phase ^= 1;
                if (ok) {
                    char* const st = p.sm + r.s * STAGE;   // box lane / 8, 16 bytes (lane % 8) of each row
                    for (int x = left; x < ((left + 15) & ~15); ++x)
                        *reinterpret_cast<int4*>(st + (lane >> 3) * BOX_MN + x * 128 + (lane & 7) * 16) = make_int4(0, 0, 0, 0);
                    tc::fence_async_smem();
                    __syncwarp();
                    // the leader hands the stage over when both halves are zeroed (an arrival of the second CTA on full[s]
                    // for every stage cost more than the products).  One barrier per stage: the other CTA may be several
                    // ragged stages ahead, but not past a stage that the leader has not handed over
                    if (p.rank != 0) {
                        if (one) arrive_cluster(p.zeroed0 + r.s * 8);
                    } else {
                        ok = __all_sync(~0u, wait_cluster(&p.zeroed[r.s], (zeroed_phases >> r.s) & 1));
                        zeroed_phases ^= 1u << r.s;
                        if (ok && one) tc::mbar_arrive(&p.full[r.s]);
                    }
                }
                if (!ok) {
                    *p.err = 1;
                    break;
                }
                __syncwarp();
            }
        }
        finish_copies(p, r);
    } else if (warp == COPY_B) {
        const bool one = elect();
        Ring r;
        bool ok = true;
        for (long long t = blockIdx.x / 2; ok && t < tiles; t += pairs) {
            const Tile d = tile_at(t);
            const int k = d.k0 + p.rank * (d.cols / 2);
            for (int c = 0; c < d.nb; ++c, r.next()) {
                if (!(ok = __all_sync(~0u, stage_free(p, r)))) break;
                if (one && !ragged(d.rows - c * BK)) {
                    const uint32_t bs = tc::smem_u32(p.sm) + r.s * STAGE + HALF, bar = p.full0 + r.s * 8;
                    tma2_load_2d(bs, &tx, k, d.r0 + c * BK, bar);
                    tma2_load_2d(bs + BOX_MN, &tx, k + 64, d.r0 + c * BK, bar);
                }
                __syncwarp();
            }
        }
    } else if (warp == PRODUCTS) {
        if (p.rank == 0) {
            const bool one = elect();
            const uint64_t a0 = sdesc<true>(tc::smem_u32(p.sm)), b0 = sdesc<true>(tc::smem_u32(p.sm) + HALF);
            Ring r;
            int j = 0;   // accumulators over all tiles
            for (long long t = blockIdx.x / 2; t < tiles && !*p.err; t += pairs) {
                const Tile d = tile_at(t);
                const uint32_t id = idesc_f16(2 * FT, d.cols, a.bf16, true, true);
                for (int c0 = 0; c0 < d.nb; c0 += DRAIN<OUT>, ++j) {
                    const int b = j & 1, c1 = min(c0 + DRAIN<OUT>, d.nb);
                    const uint32_t acc = p.tmem + b * NT;
                    if (j >= 2 && !tc::mbar_wait(&p.tempty[b], (uint32_t)((j / 2 - 1) & 1))) *p.err = 1;
                    tc::fence_after_sync();
                    for (int c = c0; c < c1; ++c) {
                        if (*p.err || !tc::mbar_wait(&p.full[r.s], r.phase)) {
                            *p.err = 1;
                            break;
                        }
                        tc::fence_after_sync();
                        const int left = d.rows - c * BK;
                        if (one) {
#pragma unroll
                            for (int q = 0; q < BK / 16; ++q)
                                if (q * 16 < left)
                                    mma2_f16(acc, a0 + ((r.s * STAGE + q * kstep<true>()) >> 4), b0 + ((r.s * STAGE + q * kstep<true>()) >> 4),
                                             id, c > c0 || q > 0);
                            commit2(&p.empty[r.s]);
                        }
                        r.next();
                    }
                    if (one) commit2(&p.tfull[b]);
                }
            }
        }
    } else {
        constexpr int COLS = 128 / sizeof(OUT);
        const int q = warp & 3, half = warp >> 2;
        const bool one = elect();
        char* const stage = p.sm + STAGING + warp * 4096;
        int j = 0;
        bool ok = true;
        for (long long t = blockIdx.x / 2; ok && t < tiles; t += pairs) {
            const Tile d = tile_at(t);
            float sum[NT / 2];
#pragma unroll
            for (int c = 0; c < NT / 2; ++c) sum[c] = 0.f;
            for (int c = 0; c < d.nb; c += DRAIN<OUT>, ++j) {
                const int b = j & 1;
                ok = !*p.err && tc::mbar_wait(&p.tfull[b], (uint32_t)((j / 2) & 1));
                if (!__all_sync(~0u, ok)) {
                    *p.err = 1;
                    ok = false;
                    break;
                }
                tc::fence_after_sync();
                const uint32_t at = p.tmem + b * NT + half * (NT / 2) + ((uint32_t)(q * 32) << 16);
#pragma unroll
                for (int c0 = 0; c0 < NT / 2; c0 += 16) {
                    if (half * (NT / 2) + c0 < d.cols) {
                        float v[16];
                        tc::tmem_ld16(at + c0, v);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 16; ++x) sum[c0 + x] += v[x];
                    }
                }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_cluster(p.tempty0 + b * 8);
            }
            if (!ok) break;
            // 32 rows x 128 bytes at a time through shared memory (in the swizzled layout, so that the lanes' rows meet no
            // bank twice), then one TMA store: lanes that write their own rows to memory touch 32 lines per instruction,
            // which took longer than the products (16 experts of 2048x5120 in fp32: 328 us so)
            const int n = d.n0 + p.rank * FT + q * 32, k = d.k0 + half * (NT / 2);
            const uint32_t mine = tc::smem_u32(stage) + lane * 128;
#pragma unroll
            for (int c = 0; c < NT / 2; c += COLS) {
                if (n < a.N && k + c < a.K) {
                    if (one) bulk_wait_read();
                    __syncwarp();
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const uint32_t at = mine + ((x ^ (lane & 7)) << 4);
                        if constexpr (sizeof(OUT) == 4) {
                            const float* v = sum + c + 4 * x;
                            st_shared16(at, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                        } else {
                            const float* v = sum + c + 8 * x;
                            st_shared16(at, pack16(v[0], v[1], a.bf16), pack16(v[2], v[3], a.bf16), pack16(v[4], v[5], a.bf16),
                                        pack16(v[6], v[7], a.bf16));
                        }
                    }
                    if (TMA_OUT) {
                        tc::fence_async_smem();
                        __syncwarp();
                        if (one) tma_store_3d(&tdw, k + c, n, d.e, tc::smem_u32(stage));
                    } else {
                        __syncwarp();
                        store_rows(stage, static_cast<OUT*>(a.dw) + ((long long)d.e * a.N + n) * a.K + k + c, a.K,
                                   min(32, a.N - n), min(COLS, a.K - k - c));
                    }
                }
            }
        }
        if (one) bulk_wait();   // the last results have left shared memory before it goes
    }
    tear_down(p, a.status);
}

template <auto kernel, typename... A>
cudaError_t go(long long tiles, int E, cudaStream_t st, const A&... args) {
    int nsm = 0;
    cudaError_t e = sm_count(&nsm);
    const int smem = FIXED + 2 * (E + 1) * (int)sizeof(int);
    static SmemOnce once;   // of this kernel
    if (e == cudaSuccess) e = once.allow(reinterpret_cast<const void*>(kernel), FIXED + 2 * (MM_MAX_E + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return e;
    const long long pairs = tiles < nsm / 2 ? tiles : nsm / 2;
    kernel<<<(unsigned)(2 * pairs), THREADS, smem, st>>>(args...);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mm_wide(const MmOperand& x, const MmOperand& w, const MmArgs& args, cudaStream_t st) {
    MmArgs a = args;
    a.ntn = (a.N + 2 * FT - 1) / (2 * FT);
    alignas(64) CUtensorMap tw, tx;
    cudaError_t e = encode_mm(&tx, x, a.type(), BK, FT);
    if (e == cudaSuccess) e = w.mn ? encode_mm(&tw, w, a.type(), 64, BK) : encode_mm(&tw, w, a.type(), BK, FT);
    if (e != cudaSuccess) return e;
    const long long tiles = ((long long)(a.T / NT) + (a.T < a.E ? a.T : a.E)) * a.ntn;   // the most the offsets could give
    if (tiles > (1LL << 30)) return cudaErrorInvalidValue;
    return w.mn ? go<k_mm_wide<true>>(tiles, a.E, st, tw, tx, a) : go<k_mm_wide<false>>(tiles, a.E, st, tw, tx, a);
}

cudaError_t launch_mm_wgrad(const MmOperand& dy, const MmOperand& x, const MmWgradArgs& a, cudaStream_t st) {
    const int size = a.out32 ? 4 : 2;
    const bool rows16 = reinterpret_cast<uintptr_t>(a.dw) % 16 == 0 && (long long)a.K * size % 16 == 0;
    alignas(64) CUtensorMap tdy, tx, tdw{};
    cudaError_t e = encode_mm(&tdy, dy, a.type(), 64, BK);
    if (e == cudaSuccess) e = encode_mm(&tx, x, a.type(), 64, BK);
    if (e == cudaSuccess && rows16)
        e = encode_mm(&tdw, MmOperand{a.dw, a.K, a.N, a.K, a.E, (long long)a.N * a.K, false}, a.out32 ? DT_F32 : a.type(),
                      128 / size, 32);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)a.E * ((a.N + 2 * FT - 1) / (2 * FT)) * ((a.K + NT - 1) / NT);
    if (rows16)
        return a.out32 ? go<k_mm_wgrad<float, true>>(tiles, a.E, st, tdy, tx, tdw, a)
                       : go<k_mm_wgrad<uint16_t, true>>(tiles, a.E, st, tdy, tx, tdw, a);
    return a.out32 ? go<k_mm_wgrad<float, false>>(tiles, a.E, st, tdy, tx, tdw, a)
                   : go<k_mm_wgrad<uint16_t, false>>(tiles, a.E, st, tdy, tx, tdw, a);
}

}  // namespace spq
