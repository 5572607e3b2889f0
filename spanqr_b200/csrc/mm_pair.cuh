// Pairs of SMs: what the kernels that work on one tile of a product with two SMs share (k_mm_wide.cu, k_mm_wgrad.cu).
//
// One tcgen05.mma.cta_group::2 works on both SMs of a pair (a cluster of two CTAs): each CTA holds the accumulators of
// 128 of a tile's 256 features, its own half of A and half of B, so a 64-element stage of a 256 x 256 tile costs each SM
// 32 KB of shared memory and of L2 traffic for 512 cycles of products; a 128 x 256 tile on one SM would need 48 KB.  Two
// accumulators: the epilogue of one overlaps the products of the next.  The grid is one pair per two SMs; the pipeline
// runs on from tile to tile.
//
// Barriers.  full[s] (used in the first CTA of the pair, the leader, whose thread issues the products): both CTAs' copies
// of stage s; empty[s] and tfull[b] (both CTAs): signalled by the products' commit to both; tempty[b] (leader): the
// sixteen epilogue warps have read accumulator b.
#pragma once
#include "mm.cuh"

namespace spq {
namespace mm {

// warps 0-7: epilogue (TMEM lanes 32 (w % 4) .., columns by w / 4), 8 and 9: copies of A and of B, 10: products.  The issue
// of the copies is on the critical path (a stage lasts 512 cycles): one warp for both operands held the weight gradient
// to 1340 TFLOP/s where two give 1500 (16384 rows, 8 experts of 5120x2048, bf16).
constexpr int THREADS = 352;
constexpr int COPY_A = 8, COPY_B = 9, PRODUCTS = 10;
constexpr int A_BYTES = FT * BK * 2;   // one CTA's half of A: 128 x 64 elements, 16 KB

// NT: columns of a tile (and of each accumulator); ST: stages; OUT: bytes through which the results leave
template <int NT_, int ST, int OUT>
struct PairCfg {
    static constexpr int NT = NT_, STAGES = ST;
    static constexpr int STAGE = A_BYTES + NT / 2 * BK * 2;
    static constexpr int STAGING = STAGES * STAGE;
    static constexpr int BARS = STAGING + OUT;
    static constexpr int MAPS = BARS + 384;        // tmem slot, error flag, then the group map
    static constexpr int FIXED = MAPS + 16 + 1024; // + 1024: the base is aligned up
    static_assert((3 * STAGES + 5) * 8 <= 384, "barriers");
    static_assert(FIXED + 2 * (MM_MAX_E + 1) * 4 <= 227 * 1024, "shared memory");
};

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

constexpr uint64_t WAIT_NS = 2000000000ull;   // the limit of every wait (only the self-test gives another)

// the bounded wait on a barrier that the other CTA arrives on
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, uint64_t limit_ns = WAIT_NS) {
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
    uint64_t *ragged, *zeroed;   // wgrad: this CTA's copies of a ragged stage; (leader) the other has zeroed its part of stage s
    volatile int* err;
    int *start, *pre;
    uint32_t tmem;
    int rank;
    uint32_t full0, tempty0, zeroed0;   // cluster addresses of the leader's barriers
};

template <typename C>
__device__ __forceinline__ Pair set_up(char* dyn, const int* offsets, int E, int T, int rows_per_tile) {
    constexpr int STAGES = C::STAGES;
    Pair p;
    p.sm = dyn + ((1024u - (tc::smem_u32(dyn) & 1023u)) & 1023u);
    p.full = reinterpret_cast<uint64_t*>(p.sm + C::BARS);
    p.empty = p.full + STAGES;
    p.zeroed = p.empty + STAGES;
    p.tfull = p.zeroed + STAGES;
    p.tempty = p.tfull + 2;
    p.ragged = p.tempty + 2;
    uint32_t* const slot = reinterpret_cast<uint32_t*>(p.sm + C::MAPS);
    p.err = reinterpret_cast<int*>(p.sm + C::MAPS + 4);
    p.start = reinterpret_cast<int*>(p.sm + C::MAPS + 16);
    p.pre = p.start + E + 1;
    p.rank = (int)cluster_rank();
    const int warp = threadIdx.x >> 5;
    if (warp == 0) map_groups(offsets, E, T, rows_per_tile, p.start, p.pre);
    if (warp == PRODUCTS) tmem_alloc2(slot, 2 * C::NT);
    if (threadIdx.x == 32 * COPY_A) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&p.full[s], 1);
            tc::mbar_init(&p.empty[s], 1);
            tc::mbar_init(&p.zeroed[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(&p.tfull[b], 1);
            tc::mbar_init(&p.tempty[b], 16);
        }
        tc::mbar_init(p.ragged, 1);
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
    wait_primary();   // (the offsets, read above, are no copy's result)
    return p;
}

// No CTA of the pair leaves while the other may still signal its barriers or read its operands.  When all went well the roles
// have seen every signal and copy by now.  After a wait that ran out they have not: the products' signals to both CTAs and
// the second CTA's copies may be under way still.  Whoever finds the flag set stays for GRACE_NS, thousands of times what
// either takes, so that all it issued has landed.
constexpr uint64_t GRACE_NS = 10000000ull;

template <typename C>
__device__ __forceinline__ void tear_down(const Pair& p, int* status) {
    if (*p.err)
        for (const uint64_t t0 = tc::globaltimer(); tc::globaltimer() - t0 < GRACE_NS;) __nanosleep(1000);
    __syncwarp();
    tc::fence_before_sync();
    cluster_sync_all();
    if ((threadIdx.x >> 5) == PRODUCTS) tmem_dealloc2(p.tmem, 2 * C::NT);
    if (threadIdx.x == 0 && *p.err) atomicOr(status, MM_TIMEOUT);
}

// a role's place in the ring of stages
template <typename C>
struct Ring {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++s == C::STAGES) {
            s = 0;
            phase ^= 1;
        }
    }
};

// the wait for the ring's stage to be free (a barrier's first wait, for the phase before its first, returns at once)
template <typename C>
__device__ __forceinline__ bool stage_free(const Pair& p, const Ring<C>& r, uint64_t limit_ns = WAIT_NS) {
    if (!*p.err && tc::mbar_wait(&p.empty[r.s], r.phase ^ 1, limit_ns)) return true;
    *p.err = 1;
    return false;
}
// the end of the copies: the products have released every stage (so no signal is on its way to a barrier of a CTA that
// is gone), or, after a limit ran out, the leader has seen both CTAs' copies arrive
template <typename C>
__device__ __forceinline__ void finish_copies(const Pair& p, Ring<C> r, uint64_t limit_ns = WAIT_NS) {
    if (!*p.err) {
        for (int n = 0; n < C::STAGES; ++n, r.next())
            if (!tc::mbar_wait(&p.empty[r.s], r.phase ^ 1, limit_ns)) *p.err = 1;
    } else if (p.rank == 0) {
        for (int s = 0; s < C::STAGES; ++s) tc::mbar_wait(&p.full[s], s < r.s ? r.phase : r.phase ^ 1, limit_ns);
    }
}

__device__ __forceinline__ int up32(int n) { return (n + 31) & ~31; }

// ---- stages split evenly ----
// With fewer tiles than pairs the stages of all tiles, in order, are cut into equal runs, one per pair, of at least
// MIN_RUN stages.  A run that begins or ends inside a tile leaves that tile's partial sums in its slot of the
// workspace: slot 2 pair for the run's first tile, 2 pair + 1 for its last when that begins in the run.  A second kernel
// adds a tile's parts in their order, so the bits depend on the sizes and offsets alone.
__host__ __device__ __forceinline__ int run_count(long long total, int pairs, int min_run) {
    const long long most = total / min_run;
    return most < 1 ? 1 : most < pairs ? (int)most : pairs;
}
__host__ __device__ __forceinline__ long long run_begin(long long total, int runs, int i) {
    return i < runs ? total * i / runs : total;
}

// a pair kernel's launch (behind: the copies of its operands precede it)
template <typename C, auto kernel, typename... A>
cudaError_t launch_pairs(int pairs, int E, bool behind, cudaStream_t st, const A&... args) {
    static SmemOnce once;   // of this kernel
    const void* const fn = reinterpret_cast<const void*>(kernel);
    const int most = C::FIXED + 2 * (MM_MAX_E + 1) * (int)sizeof(int), smem = C::FIXED + 2 * (E + 1) * (int)sizeof(int);
    cudaError_t e = once.allow(fn, most);
    if (e != cudaSuccess) return e;
    for (int attempt = 0;; ++attempt) {
        if (behind) {
            e = launch_behind(kernel, dim3(2 * pairs), THREADS, smem, st, args...);
        } else {
            kernel<<<2 * pairs, THREADS, smem, st>>>(args...);
            e = cudaGetLastError();
        }
        // a device that was reset since has forgotten the limit
        if (e != cudaErrorInvalidValue || attempt > 0) return e;
        cudaGetLastError();
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
    }
}

}  // namespace mm
}  // namespace spq
