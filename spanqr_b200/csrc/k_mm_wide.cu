// y[t] = w[e(t)] x[t], rows sorted by expert (no reference counterpart): D = W X^T in tiles of 256 features x up to NT of
// one expert's rows, on pairs of SMs (mm_pair.cuh).
//
// The weights are the tensor core's first operand whatever the number of rows: with few rows the kernel streams them once
// from HBM, with many it is bound by the products, and a tile's last rows cost products in steps of 32 columns, not of
// 128.  NT is 32 to 256 by the rows per expert and the tiles that leaves (mm_plan): the smaller the tile, the more of
// the weights are in flight and the more pairs have work.  Where even tiles of 32 rows leave pairs idle, the stages of the
// contracted dimension are split evenly over the pairs and joined by a second kernel.
//
// Measured (bf16, inputs out of the caches, rows split evenly): 16384 rows, 8 experts of 5120x2048: 222 us (1546 TFLOP/s;
// cuBLAS with one matrix at this size, in the same run: 217 us); the same rows unevenly (997 to 4092 each): 268 us; 1024
// rows, 128 experts of 1024x1024: 49 us (5.6 TB/s); 64 rows, 8 experts of 5120x2048: 35 us (4.8 TB/s); one row and next to
// no work: 5 us.
#include "mm_pair.cuh"

namespace spq {
namespace {

using namespace mm;

template <int NT>
using Cfg = PairCfg<NT, NT == 256 ? 5 : NT == 128 ? 7 : NT == 64 ? 8 : 9, 8 * Y_STAGE>;
constexpr int MIN_RUN = 4;   // stages
template <int NT>
constexpr bool CAN_SPLIT = NT == 32;

// a pair's tiles or parts of tiles in turn: tile, stages k0 .. k1
struct Part {
    int tile, k0, k1;
    bool whole;
};
struct Parts {
    int tile, k0, step, kb;
    long long left;
    __device__ __forceinline__ Parts(bool split, int tiles, int kb, int pair, int pairs) : kb(kb) {
        const long long total = (long long)tiles * kb;
        if (split) {
            const int runs = run_count(total, pairs, MIN_RUN);
            const long long b = run_begin(total, runs, pair);
            left = run_begin(total, runs, pair + 1) - b;
            tile = (int)(b / kb);
            k0 = (int)(b - (long long)tile * kb);
            step = 1;
        } else {
            left = pair < tiles ? (long long)((tiles - pair + pairs - 1) / pairs) * kb : 0;
            tile = pair;
            k0 = 0;
            step = pairs;
        }
    }
    __device__ __forceinline__ bool next(Part& p) {
        if (left <= 0) return false;
        p.tile = tile;
        p.k0 = k0;
        p.k1 = (int)min((long long)kb, k0 + left);
        p.whole = p.k0 == 0 && p.k1 == kb;
        left -= p.k1 - p.k0;
        tile += step;
        k0 = 0;
        return true;
    }
};

struct Tile {
    int e, n0, t0, rows, cols;   // cols: the rows up to a multiple of 32
};
template <int NT>
__device__ __forceinline__ Tile tile_at(const int* start, const int* pre, int E, int ntn, int i) {
    const int u = i / ntn;
    Tile t;
    t.n0 = (i - u * ntn) * 2 * FT;
    t.e = group_of(pre, E, u);
    t.t0 = start[t.e] + (u - pre[t.e]) * NT;
    t.rows = min(NT, start[t.e + 1] - t.t0);
    t.cols = up32(t.rows);
    return t;
}

template <bool W_MN, int NT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    k_mm_wide(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx, const MmArgs a) {
    using C = Cfg<NT>;
    extern __shared__ char dyn[];
    const bool split = CAN_SPLIT<NT> && a.part != nullptr;
    if (split) launch_dependents();
    const Pair p = set_up<C>(dyn, a.offsets, a.E, a.T, NT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ntn = a.ntn, pair = (int)blockIdx.x / 2;
    Parts parts(split, p.pre[a.E] * ntn, (a.K + BK - 1) / BK, pair, (int)gridDim.x / 2);
    Part t;

    // the copy and product warps run their loops whole (their state stays in uniform registers, which TMA and tcgen05
    // operands need); one thread issues
    if (warp == COPY_A) {
        const bool one = elect();
        if (one) prefetch_map(&tw);
        Ring<C> r;
        bool ok = true;
        while (ok && parts.next(t)) {
            const Tile d = tile_at<NT>(p.start, p.pre, a.E, ntn, t.tile);
            const int n = d.n0 + p.rank * FT;
            for (int k = t.k0; k < t.k1; ++k, r.next()) {
                if (!(ok = __all_sync(~0u, stage_free(p, r)))) break;
                if (one) {
                    const uint32_t as = tc::smem_u32(p.sm) + r.s * C::STAGE, bar = p.full0 + r.s * 8;
                    if (p.rank == 0) tc::mbar_expect_tx(&p.full[r.s], 2 * C::STAGE);
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
        if (one) prefetch_map(&tx);
        Ring<C> r;
        bool ok = true;
        while (ok && parts.next(t)) {
            const Tile d = tile_at<NT>(p.start, p.pre, a.E, ntn, t.tile);
            const int row = d.t0 + p.rank * (d.cols / 2);
            for (int k = t.k0; k < t.k1; ++k, r.next()) {
                if (!(ok = __all_sync(~0u, stage_free(p, r)))) break;
                if (one) tma2_load_2d(tc::smem_u32(p.sm) + r.s * C::STAGE + A_BYTES, &tx, k * BK, row, p.full0 + r.s * 8);
                __syncwarp();
            }
        }
    } else if (warp == PRODUCTS) {
        if (p.rank == 0) {
            const bool one = elect();
            const uint64_t a0 = sdesc<W_MN>(tc::smem_u32(p.sm)), b0 = sdesc<false>(tc::smem_u32(p.sm) + A_BYTES);
            Ring<C> r;
            int j = 0;
            while (!*p.err && parts.next(t)) {
                const Tile d = tile_at<NT>(p.start, p.pre, a.E, ntn, t.tile);
                const int b = j & 1;
                const uint32_t acc = p.tmem + b * NT, id = idesc_f16(2 * FT, d.cols, a.bf16, W_MN, false);
                if (j >= 2 && !tc::mbar_wait(&p.tempty[b], (uint32_t)((j / 2 - 1) & 1))) *p.err = 1;
                tc::fence_after_sync();
                for (int k = t.k0; k < t.k1; ++k, r.next()) {
                    if (*p.err || !tc::mbar_wait(&p.full[r.s], r.phase)) {
                        *p.err = 1;
                        break;
                    }
                    tc::fence_after_sync();
                    if (one) {
#pragma unroll
                        for (int q = 0; q < BK / 16; ++q)
                            mma2_f16(acc, a0 + ((r.s * C::STAGE + q * kstep<W_MN>()) >> 4),
                                     b0 + ((r.s * C::STAGE + q * kstep<false>()) >> 4), id, k > t.k0 || q > 0);
                        commit2(&p.empty[r.s]);
                    }
                }
                if (one) commit2(&p.tfull[b]);
                ++j;
            }
        }
    } else {
        const bool v16 = a.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
        const int q = warp & 3, half = warp >> 2;
        const uint32_t stage = tc::smem_u32(p.sm) + C::STAGING + warp * Y_STAGE;
        if (a.zero_tail) {   // rows behind the last expert
            const int whole = v16 ? a.N / 8 * 8 : 0;
            for (long long r = p.start[a.E] + (long long)blockIdx.x; r < a.T; r += gridDim.x) {
                uint16_t* const y = a.y + r * a.ldy;
                for (int n = threadIdx.x * 8; n < whole; n += 256 * 8) *reinterpret_cast<uint4*>(y + n) = make_uint4(0, 0, 0, 0);
                for (int n = whole + threadIdx.x; n < a.N; n += 256) y[n] = 0;
            }
        }
        for (int j = 0; parts.next(t); ++j) {
            const Tile d = tile_at<NT>(p.start, p.pre, a.E, ntn, t.tile);
            const int b = j & 1, f = p.rank * FT + q * 32, n = d.n0 + f;
            const bool ok = !*p.err && tc::mbar_wait(&p.tfull[b], (uint32_t)((j / 2) & 1));
            if (!__all_sync(~0u, ok)) {
                *p.err = 1;
                break;
            }
            tc::fence_after_sync();
            const uint32_t acc = p.tmem + b * NT + ((uint32_t)(q * 32) << 16);
            if (n < a.N) {
                if (!CAN_SPLIT<NT> || t.whole) {
                    store_y(acc, stage, a.y + (long long)d.t0 * a.ldy + n, a.ldy, half * 32, 64, d.cols, d.rows, a.N - n,
                            a.bf16, v16);
                } else {   // the part's slot: [column][feature]
                    float* const out = a.part + (size_t)(2 * pair + (t.k0 == 0)) * NT * 256 + f + lane;
                    for (int c = half * 32; c < d.cols; c += 64) {
                        float v[32];
                        tc::tmem_ld32(acc + c, v);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; ++x) out[(c + x) * 256] = v[x];
                    }
                }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_cluster(p.tempty0 + b * 8);
        }
    }
    tear_down<C>(p, a.status);
}

// The split tiles' parts, added in order: CTA (c, s) takes the tile that run c begins inside, if it is the first to, and of
// it the columns s, s + gridDim.y, ...; a thread is a feature.
template <int NT>
__global__ void __launch_bounds__(256) k_mm_join(const MmArgs a, int pairs) {
    extern __shared__ int map[];
    int *const start = map, *const pre = map + a.E + 1;
    if (threadIdx.x < 32) map_groups(a.offsets, a.E, a.T, NT, start, pre);
    __syncthreads();
    const int kb = (a.K + BK - 1) / BK, c = (int)blockIdx.x + 1;
    const long long total = (long long)pre[a.E] * a.ntn * kb;
    const int runs = run_count(total, pairs, MIN_RUN);
    const long long b = run_begin(total, runs, c);
    const int tile = (int)(b / kb);
    const long long lo = (long long)tile * kb, hi = lo + kb;
    wait_primary();
    if (c >= runs || b == lo || run_begin(total, runs, c - 1) > lo) return;
    int last = c;   // the last run in the tile
    while (last + 1 < runs && run_begin(total, runs, last + 1) < hi) ++last;
    const Tile d = tile_at<NT>(start, pre, a.E, a.ntn, tile);
    const int n = d.n0 + (int)threadIdx.x;
    if (n >= a.N) return;
    constexpr size_t SLOT = (size_t)NT * 256;
    for (int col = blockIdx.y; col < d.rows; col += gridDim.y) {
        const float* const p = a.part + (size_t)col * 256 + threadIdx.x;
        float s = p[(2 * (c - 1) + 1) * SLOT];
        int i = c;
        for (; i + 8 <= last + 1; i += 8) {   // eight loads in flight, added in order
            float v[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = p[2 * (i + x) * SLOT];
#pragma unroll
            for (int x = 0; x < 8; ++x) s += v[x];
        }
        for (; i <= last; ++i) s += p[2 * i * SLOT];
        a.y[(long long)(d.t0 + col) * a.ldy + n] = to16(s, a.bf16);
    }
}

template <int NT>
cudaError_t run(const MmOperand& x, const MmOperand& w, const MmArgs& a, const MmPlan& pl, cudaStream_t st) {
    using C = Cfg<NT>;
    alignas(64) CUtensorMap tw, tx;
    cudaError_t e = encode_mm(&tx, x, a.type(), BK, NT / 2);
    if (e == cudaSuccess) e = w.mn ? encode_mm(&tw, w, a.type(), 64, BK) : encode_mm(&tw, w, a.type(), BK, FT);
    if (e == cudaSuccess)
        e = w.mn ? launch_pairs<C, k_mm_wide<true, NT>>(pl.pairs, a.E, a.behind, st, tw, tx, a)
                 : launch_pairs<C, k_mm_wide<false, NT>>(pl.pairs, a.E, a.behind, st, tw, tx, a);
    if constexpr (CAN_SPLIT<NT>) {
        if (e == cudaSuccess && pl.split)
            e = launch_behind(k_mm_join<NT>, dim3(pl.pairs - 1, NT / 2), 256, 2 * (a.E + 1) * (int)sizeof(int), st, a,
                              pl.pairs);
    }
    return e;
}

}  // namespace

MmPlan mm_plan(int T, int E, int N, int K, int nsm) {
    MmPlan p;
    const long long ntn = (N + 2 * FT - 1) / (2 * FT), some = T < E ? T : E;
    const int pairs = nsm / 2;
    auto tiles = [&](int nt) { return ntn * (T / nt + (some + 1) / 2); };   // as many as to expect
    // Tiles that hold an average expert with room to spare (a second tile reads its weights again), halved while a quarter
    // of the pairs would idle.  Measured (us at 32 / 64 / 128 / 256 rows): 16 experts of 2048x2048 with 256 rows in all:
    // 26 / 27 / 27 / 28; 1024: 38 / 31 / 28 / 29; 4096: 95 / 58 / 45 / 43; one expert of 2048x2048 with 512 rows (two tiles
    // of 256 for each of 8 in its features): 18 / 13 / 14 / 19.
    p.nt = T <= 20LL * E ? 32 : T <= 44LL * E ? 64 : T <= 96LL * E ? 128 : 256;
    while (p.nt > 32 && tiles(p.nt) * 4 < 3 * pairs) p.nt /= 2;
    // Whole, a pair takes about 0.165 us for each of a tile's kb stages, the others idling.  Split, all pairs take 0.2 us a
    // stage out of L2, and all the weights that are read for the first time come at HBM's rate (0.48 us a stage and pair);
    // the partial sums and the second kernel cost 6.5 us.  Measured (us whole / split, bf16): 8 rows and one matrix of
    // 256x8192 (one tile of 128 stages): 26 / 15; 256x4096: 16 / 11; 256x2048: 10 / 10; 2048x6144 (8 of 96): 21 / 16;
    // 4096x4096 (16 of 64): 16 / 17; 6144x6144 (24 of 96): 21 / 23; 256 rows and 768x17408 (24 tiles of 272 stages over the
    // weights of 3): 50 / 29; 16 rows over 16 experts of 1024x2048 (4 tiles of 32 for each expert that has rows, some ten of
    // them): 14 / 19.
    const long long kb = (K + BK - 1) / BK, first = ntn * some, all = tiles(32);
    p.split = p.nt == 32 && kb * (10 * pairs - (12 * all > 30 * first ? 12 * all : 30 * first)) > 400LL * pairs;
    const long long most = ntn * (T / p.nt + some);
    p.tiles = most;
    p.pairs = p.split || most > pairs ? pairs : (int)most;
    p.ws = p.split ? (size_t)2 * pairs * p.nt * 256 * sizeof(float) : 0;
    return p;
}

cudaError_t launch_mm(const MmOperand& x, const MmOperand& w, const MmArgs& a, const MmPlan& p, cudaStream_t st) {
    if (p.tiles > (1LL << 30)) return cudaErrorInvalidValue;
    return p.nt == 32 ? run<32>(x, w, a, p, st) : p.nt == 64 ? run<64>(x, w, a, p, st)
         : p.nt == 128 ? run<128>(x, w, a, p, st) : run<256>(x, w, a, p, st);
}

}  // namespace spq
