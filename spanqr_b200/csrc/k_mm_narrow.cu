// y[t] = w[e(t)] x[t] for few rows per expert: decoding steps, short prompts (no reference counterpart).
//
// Every weight is used for a handful of rows, so the kernel is bound by reading w once from HBM.  The product is
// taken as D = W X^T: 128 features are the rows of the tensor-core tile (their operand is the weights, streamed by TMA),
// TN in {16, 32, 64} of one expert's rows are its columns.  A tensor-core product costs the same time at any N up to
// 256, so a narrow tile wastes tensor time that nobody waits for.
//
// One cluster of S CTAs takes one tile; its CTAs split the contracted dimension, so that a few experts still fill
// every SM, and join through distributed shared memory: each owns TN / S of the tile's rows, receives the others' fp32
// sums for them and adds all S in rank order (the bits depend on S, never on timing).  No workspace, no atomics.  A CTA
// keeps below half of an SM's shared memory, so two are resident and one's start and epilogue hide behind the other's
// stream.
#include "mm.cuh"

namespace spq {
namespace {

using namespace mm;

constexpr int THREADS = 192;   // warps 0-3: epilogue (TMEM lanes 32 w ..), 4: copies, 5: products

template <int TN>
struct Cfg {
    static constexpr int STAGES = TN == 16 ? 5 : TN == 32 ? 4 : 3;
    static constexpr int A_BYTES = FT * BK * 2, B_BYTES = TN * BK * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int RECV = STAGES * STAGE;                    // TN x 128 floats: the partial sums of the CTA's rows
    static constexpr int BARS = RECV + TN * FT * 4;                // full[STAGES], empty[STAGES], done
    static constexpr int MAPS = BARS + 128;                        // tmem slot, error flag, then the group map
    static constexpr int FIXED = MAPS + 16 + 1024;                 // + 1024: the base is aligned up
    static constexpr uint32_t TCOLS = TN < 32 ? 32 : TN;
    static_assert((2 * STAGES + 1) * 8 <= 128, "barriers");
};

template <int TN, bool W_MN>
__global__ void __launch_bounds__(THREADS, 2) k_mm_narrow(const __grid_constant__ CUtensorMap tw,
                                                          const __grid_constant__ CUtensorMap tx, const MmArgs a) {
    using C = Cfg<TN>;
    extern __shared__ char dyn[];
    char* const sm = dyn + ((1024u - (tc::smem_u32(dyn) & 1023u)) & 1023u);
    float* const recv = reinterpret_cast<float*>(sm + C::RECV);
    uint64_t* const full = reinterpret_cast<uint64_t*>(sm + C::BARS);
    uint64_t* const empty = full + C::STAGES;
    uint64_t* const done = empty + C::STAGES;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sm + C::MAPS);
    volatile int* const err = reinterpret_cast<int*>(sm + C::MAPS + 4);
    int* const start = reinterpret_cast<int*>(sm + C::MAPS + 16);
    int* const pre = start + a.E + 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = (int)cluster_size(), rank = (int)cluster_rank();

    if (warp == 0) map_groups(a.offsets, a.E, a.T, TN, start, pre);
    if (tid == 160) {
        prefetch_map(&tw);
        prefetch_map(&tx);
        for (int s = 0; s < C::STAGES; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        tc::mbar_init(done, 1);
        tc::mbar_fence_init();
        *err = 0;
    }
    __syncthreads();

    if (a.zero_tail) {   // rows behind the last expert
        for (long long t = start[a.E] + (long long)blockIdx.x; t < a.T; t += gridDim.x)
            for (int n = tid; n < a.N; n += THREADS) a.y[t * a.ldy + n] = 0;
    }
    const int tile = (int)blockIdx.x / S, u = tile / a.ntn, n0 = (tile - u * a.ntn) * FT;
    if (u >= pre[a.E]) return;   // the grid covers the most tiles the offsets could give (the whole cluster leaves)
    const int e = group_of(pre, a.E, u);
    const int t0 = start[e] + (u - pre[e]) * TN, t1 = start[e + 1];
    const int kb = (a.K + BK - 1) / BK;
    const int kb0 = (int)((long long)kb * rank / S), nk = (int)((long long)kb * (rank + 1) / S) - kb0;

    if (warp == 5) tc::tmem_alloc(tmem_slot, C::TCOLS);
    tc::fence_before_sync();
    cluster_sync_all();          // every CTA of the cluster runs before its shared memory is written
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const uint32_t sbase = tc::smem_u32(sm);

    if (warp == 4) {
        if (lane == 0) {
            int i = 0;
            for (; i < nk; ++i) {
                const int s = i % C::STAGES;
                if (i >= C::STAGES && (*err || !tc::mbar_wait(&empty[s], (uint32_t)((i / C::STAGES - 1) & 1)))) {
                    *err = 1;
                    break;
                }
                const uint32_t bar = tc::smem_u32(&full[s]), as = sbase + s * C::STAGE, bs = as + C::A_BYTES;
                const int k = (kb0 + i) * BK;
                tc::mbar_expect_tx(&full[s], C::STAGE);
                if (W_MN) {
                    tma_load_3d(as, &tw, n0, k, e, bar);
                    tma_load_3d(as + BOX_MN, &tw, n0 + 64, k, e, bar);
                } else {
                    tma_load_3d(as, &tw, k, n0, e, bar);
                }
                tma_load_2d(bs, &tx, k, t0, bar);
            }
            // the products have released the last stages or, after a limit ran out, their copies have arrived
            uint64_t* const last = *err ? full : empty;
            for (int j = max(0, i - C::STAGES); j < i; ++j)
                if (!tc::mbar_wait(&last[j % C::STAGES], (uint32_t)((j / C::STAGES) & 1))) *err = 1;
        }
        __syncwarp();
    } else if (warp == 5) {
        if (lane == 0) {
            const uint32_t id = idesc_f16(FT, TN, a.bf16, W_MN, false);
            for (int i = 0; i < nk; ++i) {
                const int s = i % C::STAGES;
                if (*err || !tc::mbar_wait(&full[s], (uint32_t)((i / C::STAGES) & 1))) {
                    *err = 1;
                    break;
                }
                tc::fence_after_sync();
                const uint32_t as = sbase + s * C::STAGE, bs = as + C::A_BYTES;
#pragma unroll
                for (int k = 0; k < BK / 16; ++k)
                    mma_f16(tmem, sdesc<W_MN>(as + k * kstep<W_MN>()), sdesc<false>(bs + k * kstep<false>()), id,
                            i > 0 || k > 0);
                tc::mma_commit(&empty[s]);
            }
            tc::mma_commit(done);
        }
        __syncwarp();
    } else {
        // this CTA's sums of column c (row t0 + c) go to the CTA that owns it
        const bool ok = nk == 0 || tc::mbar_wait(done, 0u);
        if (!ok) *err = 1;
        __syncwarp();
        tc::fence_after_sync();
        const int per = TN / S, f = warp * 32 + lane;
#pragma unroll
        for (int c0 = 0; c0 < TN; c0 += 16) {
            float v[16];
            if (nk > 0) {
                tc::tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c0, v);
                tc::tmem_wait_ld();
            } else {   // fewer stages of the contracted dimension than CTAs
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int c = c0 + j, owner = c / per;
                const uint32_t dst = tc::smem_u32(recv + ((size_t)rank * per + (c - owner * per)) * FT + f);
                st_cluster(mapa(dst, (uint32_t)owner), v[j]);
            }
        }
        tc::fence_before_sync();
    }
    cluster_sync_all();          // every sum has arrived; from here on no CTA touches another's memory
    if (warp == 5) tc::tmem_dealloc(tmem, C::TCOLS);
    if (*err && tid == 0) atomicOr(a.status, MM_TIMEOUT);
    if (warp < 4) {
        const int per = TN / S, f = 2 * (tid & 63), n = n0 + f;
        const bool pairs = a.ldy % 2 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 3) == 0;
        for (int c = tid >> 6; c < per; c += 2) {
            const int t = t0 + rank * per + c;
            if (t >= t1 || n >= a.N) continue;
            float2 v = make_float2(0.f, 0.f);
            for (int s = 0; s < S; ++s) {
                const float2 p = *reinterpret_cast<const float2*>(recv + ((size_t)s * per + c) * FT + f);
                v.x += p.x;
                v.y += p.y;
            }
            uint16_t* const y = a.y + (long long)t * a.ldy + n;
            if (pairs && n + 1 < a.N) {
                *reinterpret_cast<uint32_t*>(y) = pack16(v.x, v.y, a.bf16);
            } else {
                y[0] = to16(v.x, a.bf16);
                if (n + 1 < a.N) y[1] = to16(v.y, a.bf16);
            }
        }
    }
}

template <int TN, bool W_MN>
cudaError_t launch(const CUtensorMap& tw, const CUtensorMap& tx, const MmArgs& a, int tiles, int S, cudaStream_t st) {
    const int smem = Cfg<TN>::FIXED + 2 * (a.E + 1) * (int)sizeof(int);
    static SmemOnce once;
    cudaError_t e = once.allow(reinterpret_cast<const void*>(k_mm_narrow<TN, W_MN>),
                               Cfg<TN>::FIXED + 2 * (MM_MAX_E + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)tiles * S);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {(unsigned)S, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_mm_narrow<TN, W_MN>, tw, tx, a);
}

template <int TN>
cudaError_t run(const MmOperand& x, const MmOperand& w, MmArgs a, cudaStream_t st) {
    alignas(64) CUtensorMap tw, tx;
    cudaError_t e = encode_mm(&tx, x, a.type(), BK, TN);
    if (e == cudaSuccess) e = w.mn ? encode_mm(&tw, w, a.type(), 64, BK) : encode_mm(&tw, w, a.type(), BK, FT);
    int nsm = 0;
    if (e == cudaSuccess) e = sm_count(&nsm);
    if (e != cudaSuccess) return e;
    // the most row tiles: every expert's last tile may hold a single row
    const long long most = (long long)(a.T / TN) + (a.T < a.E ? a.T : a.E), tiles = most * a.ntn;
    if (tiles > (1LL << 28)) return cudaErrorInvalidValue;
    // CTAs per tile: as many as keep within two per SM, with at least four stages of the contracted dimension each
    const int kb = (a.K + BK - 1) / BK;
    int S = 1;
    while (S < 8 && tiles * S * 2 <= 2LL * nsm && kb >= 8 * S) S *= 2;
    return w.mn ? launch<TN, true>(tw, tx, a, (int)tiles, S, st) : launch<TN, false>(tw, tx, a, (int)tiles, S, st);
}

}  // namespace

cudaError_t launch_mm_narrow(const MmOperand& x, const MmOperand& w, const MmArgs& a, int tn, cudaStream_t st) {
    return tn == 16 ? run<16>(x, w, a, st) : tn == 32 ? run<32>(x, w, a, st) : run<64>(x, w, a, st);
}

}  // namespace spq
