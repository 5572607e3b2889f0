// Self-test of the pair kernels' waits (mm_pair.cuh): their set-up, their bounded waits and their way out, with no copies
// and no products.  With `arrive` the roles hand a ring of stages and an accumulator round once.  Without it every wait runs
// out after the limit: the second CTA's copy warp on a stage that is not released, the leader's on the other CTA, its
// product warp on a stage that is not filled, the epilogue warps on an accumulator that is not finished.  The pair then
// leaves as a production kernel does, and reports in the same word.
#include "mm_pair.cuh"

namespace spq {
namespace {

using namespace mm;
using C = PairCfg<32, 4, 0>;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    k_mm_selftest(int arrive, unsigned long long limit_ns, int* status) {
    extern __shared__ char dyn[];
    const Pair p = set_up<C>(dyn, nullptr, 0, 0, 32);   // (no experts: the offsets are not read)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == COPY_A) {
        Ring<C> r;
        for (int s = 0; s < C::STAGES; ++s, r.next()) stage_free(p, r, limit_ns);   // (free before their first use)
        // the leader hands the stages on when the other CTA has passed them too, so that no release comes before its wait
        if (p.rank != 0) {
            if (arrive && lane == 0) arrive_cluster(p.zeroed0);
        } else if (!wait_cluster(&p.zeroed[0], 0, limit_ns)) {
            *p.err = 1;
        } else if (lane == 0) {
            for (int s = 0; s < C::STAGES; ++s) tc::mbar_arrive(&p.full[s]);
        }
        __syncwarp();
        stage_free(p, r, limit_ns);
        finish_copies(p, r, limit_ns);
    } else if (warp == PRODUCTS && p.rank == 0) {
        bool ok = true;
        for (int s = 0; ok && s < C::STAGES; ++s) ok = __all_sync(~0u, tc::mbar_wait(&p.full[s], 0, limit_ns));
        if (ok && lane < 2) {   // lane: the CTA
            for (int s = 0; s < C::STAGES; ++s) arrive_cluster(mapa(tc::smem_u32(&p.empty[s]), lane));
            arrive_cluster(mapa(tc::smem_u32(&p.tfull[0]), lane));
        }
        __syncwarp();
        if (!ok || !tc::mbar_wait(&p.tempty[0], 0, limit_ns)) *p.err = 1;
    } else if (warp < COPY_A) {
        const bool ok = __all_sync(~0u, tc::mbar_wait(&p.tfull[0], 0, limit_ns));
        if (!ok) *p.err = 1;
        else if (lane == 0) arrive_cluster(p.tempty0);
    }
    tear_down<C>(p, status);
}

}  // namespace

cudaError_t launch_mm_selftest(int arrive, unsigned long long limit_ns, int* status, cudaStream_t st) {
    return launch_pairs<C, k_mm_selftest>(1, 0, false, st, arrive, limit_ns, status);
}

}  // namespace spq
