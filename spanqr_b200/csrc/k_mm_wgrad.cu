// dw[e] = sum over expert e's rows of dy[t] x[t]^T (no reference counterpart): D = dy^T x in tiles of 256 features x 256
// columns of x, on pairs of SMs (mm_pair.cuh).  Both operands are read as they lie, row by row (MN-major), in stages of 64
// rows.  Where the tiles are fewer than the pairs, each expert's rows are cut into `splits` runs of whole stages with a
// partial result each, and a second kernel adds those in order: the bits depend on the sizes, the offsets and the device's
// number of SMs, from one call to the next they are the same.
//
// Measured (inputs out of the caches): 32768 rows, 8 experts of 5120x2048, rows split evenly, fp16 to fp32: 527 us (1304
// TFLOP/s), to fp16 553 us; in a row, under the power limit, 556 and 544 us; 8191 rows, 32 experts of 768x512, bf16 to fp32
// (50 MB, a fill of which takes 21 us): 40 us evenly, 44 us with 18 to 1505 rows each.
#include "mm_pair.cuh"

namespace spq {
namespace {

using namespace mm;

constexpr int NT = 256;
// five stages (four cost up to 7 %, six gave no more); 32 rows x 128 bytes of results per epilogue warp
using C = PairCfg<NT, 5, 8 * 4096>;
// stages (of 64 rows) summed in TMEM before they are added in registers
template <typename OUT>
constexpr int DRAIN = sizeof(OUT) == 4 ? 8 : 32;

__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// a warp's staged results to rows of dw that do not start on 16 bytes: a lane is a column (two of 16 bits)
template <typename OUT>
__device__ __forceinline__ void store_rows(const char* stage, OUT* row, int ld, int rows, int cols) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int x = 0; x < rows; x += 8) {
#pragma unroll
        for (int z = 0; z < 8; ++z) {
#pragma unroll
            for (int y = lane; y < 128 / (int)sizeof(OUT); y += 32) {
                const int at = y * (int)sizeof(OUT), r = x + z;   // (r & 7 == z)
                const OUT v = *reinterpret_cast<const OUT*>(stage + r * 128 + (((at >> 4) ^ z) << 4) + (at & 15));
                if (r < rows && y < cols) row[(long long)r * ld + y] = v;
            }
        }
    }
    __syncwarp();
}

// whether a stage with `left` rows of its expert ends inside one product's 16
__device__ __forceinline__ bool ragged(int left) { return left < BK && left % 16 != 0; }

// The tensor core rounds toward zero each time it adds 16 products to its fp32 accumulator: over n additions of terms of
// random sign the sum comes out about n * 1.5e-8 of itself too small (measured on 4096x4096 results: 8.1e-7 at 1000 rows,
// 4.6e-6 at 5000, 2.0e-5 at 20000, 1.0e-4 at 100000).  So the accumulator is taken every DRAIN stages and added to fp32 sums
// in registers, rounded to nearest, while the products go on in the other accumulator: every 512 rows for fp32 results,
// which are then 4.6e-7 to 5.4e-7 off in all at those lengths (sums of fp32 products in fp32: 2.5e-7 to 4.6e-6); every 2048
// for 16-bit results, whose own rounding is 2^-9 or 2^-12, so that the bias does not grow with the length.  The reads of TMEM
// take tensor-core time: 16384 rows, 8 experts of 5120x2048 in bf16, with one copy warp: 285 us drained every 256 rows, 258
// every 512, 252 every 4096.
template <typename OUT, bool TMA_OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    k_mm_wgrad(const __grid_constant__ CUtensorMap tdy, const __grid_constant__ CUtensorMap tx,
               const __grid_constant__ CUtensorMap tdw, const MmWgradArgs a) {
    extern __shared__ char dyn[];
    if (a.splits > 1) launch_dependents();
    const Pair p = set_up<C>(dyn, a.offsets, a.E, a.T, BK);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ntn = (a.N + 2 * FT - 1) / (2 * FT), ntk = (a.K + NT - 1) / NT, per = ntn * ntk;
    const long long tiles = (long long)a.E * a.splits * per;
    const int pairs = (int)gridDim.x / 2;
    struct Tile {
        // plane: of the result, expert by expert and run by run; cols: the tile's columns of x up to a multiple of 32; rows
        // r0 .. r0 + rows in nb stages
        int plane, n0, k0, cols, r0, rows, nb;
    };
    auto tile_at = [&](long long i) {
        Tile t;
        t.plane = (int)(i / per);
        const int l = (int)(i - (long long)t.plane * per), e = t.plane / a.splits, run = t.plane - e * a.splits;
        t.n0 = l / ntk * 2 * FT;
        t.k0 = l % ntk * NT;
        t.cols = min(NT, up32(a.K - t.k0));
        const int all = p.pre[e + 1] - p.pre[e], each = (all + a.splits - 1) / a.splits;   // stages of 64 rows
        const int c0 = min(run * each, all);
        t.nb = min(each, all - c0);
        t.r0 = p.start[e] + c0 * BK;
        t.rows = min(p.start[e + 1] - t.r0, t.nb * BK);
        return t;
    };

    if (warp == COPY_A) {
        const bool one = elect();
        Ring<C> r;
        uint32_t ragged_phase = 0, zeroed_phases = 0;   // (bit s: that of zeroed[s])
        bool ok = true;
        for (long long t = blockIdx.x / 2; ok && t < tiles; t += pairs) {
            const Tile d = tile_at(t);
            const int n = d.n0 + p.rank * FT, k = d.k0 + p.rank * (d.cols / 2);
            for (int c = 0; c < d.nb; ++c, r.next()) {
                if (!(ok = __all_sync(~0u, stage_free(p, r)))) break;
                const int left = d.rows - c * BK, row = d.r0 + c * BK;
                const uint32_t as = tc::smem_u32(p.sm) + r.s * C::STAGE;
                if (!ragged(left)) {
                    if (one) {
                        const uint32_t bar = p.full0 + r.s * 8;
                        if (p.rank == 0) tc::mbar_expect_tx(&p.full[r.s], 2 * C::STAGE);
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
                    tc::mbar_expect_tx(p.ragged, C::STAGE);
                    mm::tma_load_2d(as, &tdy, n, row, bar);
                    mm::tma_load_2d(as + BOX_MN, &tdy, n + 64, row, bar);
                    mm::tma_load_2d(as + A_BYTES, &tx, k, row, bar);
                    mm::tma_load_2d(as + A_BYTES + BOX_MN, &tx, k + 64, row, bar);
                }
                __syncwarp();
                ok = __all_sync(~0u, tc::mbar_wait(p.ragged, ragged_phase));
                ragged_phase ^= 1;
                if (ok) {
                    char* const st = p.sm + r.s * C::STAGE;   // box lane / 8, 16 bytes (lane % 8) of each row
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
        Ring<C> r;
        bool ok = true;
        for (long long t = blockIdx.x / 2; ok && t < tiles; t += pairs) {
            const Tile d = tile_at(t);
            const int k = d.k0 + p.rank * (d.cols / 2);
            for (int c = 0; c < d.nb; ++c, r.next()) {
                if (!(ok = __all_sync(~0u, stage_free(p, r)))) break;
                if (one && !ragged(d.rows - c * BK)) {
                    const uint32_t bs = tc::smem_u32(p.sm) + r.s * C::STAGE + A_BYTES, bar = p.full0 + r.s * 8;
                    tma2_load_2d(bs, &tx, k, d.r0 + c * BK, bar);
                    tma2_load_2d(bs + BOX_MN, &tx, k + 64, d.r0 + c * BK, bar);
                }
                __syncwarp();
            }
        }
    } else if (warp == PRODUCTS) {
        if (p.rank == 0) {
            const bool one = elect();
            const uint64_t a0 = sdesc<true>(tc::smem_u32(p.sm)), b0 = sdesc<true>(tc::smem_u32(p.sm) + A_BYTES);
            Ring<C> r;
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
                                    mma2_f16(acc, a0 + ((r.s * C::STAGE + q * kstep<true>()) >> 4),
                                             b0 + ((r.s * C::STAGE + q * kstep<true>()) >> 4), id, c > c0 || q > 0);
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
        char* const stage = p.sm + C::STAGING + warp * 4096;
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
                            st_shared16(at, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                        __float_as_uint(v[3]));
                        } else {
                            const float* v = sum + c + 8 * x;
                            st_shared16(at, pack16(v[0], v[1], a.bf16), pack16(v[2], v[3], a.bf16), pack16(v[4], v[5], a.bf16),
                                        pack16(v[6], v[7], a.bf16));
                        }
                    }
                    if (TMA_OUT) {
                        tc::fence_async_smem();
                        __syncwarp();
                        if (one) tma_store_3d(&tdw, k + c, n, d.plane, tc::smem_u32(stage));
                    } else {
                        __syncwarp();
                        store_rows(stage, static_cast<OUT*>(a.dw) + ((long long)d.plane * a.N + n) * a.K + k + c, a.K,
                                   min(32, a.N - n), min(COLS, a.K - k - c));
                    }
                }
            }
        }
        if (one) bulk_wait();   // the last results have left shared memory before it goes
    }
    tear_down<C>(p, a.status);
}

// the runs' partial results (rows of ldp floats, a multiple of 4), added in order: one thread, four columns of one row.
// (part is not __restrict__: the kernel before still writes it when this one starts.)
template <typename OUT>
__global__ void __launch_bounds__(256) k_mm_wgrad_join(const MmWgradArgs a, const float* part, int ldp) {
    const int quads = ldp / 4;
    const long long plane = (long long)a.N * ldp, all = (long long)a.E * a.N * quads;
    wait_primary();
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const long long row = i / quads;   // of all experts
        const int k = (int)(i - row * quads) * 4;
        const long long e = row / a.N;
        const float* p = part + e * a.splits * plane + (row - e * a.N) * ldp + k;
        float4 s = *reinterpret_cast<const float4*>(p);
#pragma unroll 4
        for (int r = 1; r < a.splits; ++r) {
            p += plane;
            const float4 v = *reinterpret_cast<const float4*>(p);
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        OUT* const o = static_cast<OUT*>(a.dw) + row * a.K + k;
        const float v[4] = {s.x, s.y, s.z, s.w};
        if (k + 4 <= a.K && reinterpret_cast<uintptr_t>(o) % (4 * sizeof(OUT)) == 0) {
            if constexpr (sizeof(OUT) == 4) *reinterpret_cast<float4*>(o) = s;
            else *reinterpret_cast<uint2*>(o) = make_uint2(pack16(s.x, s.y, a.bf16), pack16(s.z, s.w, a.bf16));
        } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (k + x < a.K) {
                    if constexpr (sizeof(OUT) == 4) o[x] = v[x];
                    else o[x] = to16(v[x], a.bf16);
                }
            }
        }
    }
}

constexpr int MIN_STAGES = 8;   // of a run

}  // namespace

MmWgradPlan mm_wgrad_plan(int T, int E, int N, int K, int nsm) {
    MmWgradPlan p;
    const long long tiles = (long long)E * ((N + 2 * FT - 1) / (2 * FT)) * ((K + NT - 1) / NT);
    const long long stages = T / BK / E;   // of an average expert
    long long s = nsm / 2 / tiles;
    if (s > stages / MIN_STAGES) s = stages / MIN_STAGES;
    // a stage takes about 0.3 us, the partial results and the second kernel about 4 us.  Measured (us, fp32 results): 2048
    // rows, one expert of 768x512: 17.7 whole, 15.1 split four ways (24 of 32 stages saved); 4096 rows, 4 experts of 512x512:
    // 15.8 whole, 17.4 split two ways (8 of 16); 32768 rows, one expert of 768x512: 162 whole, 35 split twelve ways
    p.splits = s > 1 && stages * (s - 1) >= 16 * s ? (int)s : 1;
    p.ldp = (K + 3) / 4 * 4;
    p.tiles = tiles * p.splits;
    p.ws = p.splits > 1 ? (size_t)E * p.splits * N * p.ldp * sizeof(float) : 0;
    return p;
}

cudaError_t launch_mm_wgrad(const MmOperand& dy, const MmOperand& x, const MmWgradArgs& args, const MmWgradPlan& pl, float* ws,
                            cudaStream_t st) {
    MmWgradArgs a = args;
    a.splits = pl.splits;
    const bool split = pl.splits > 1;
    if (split) a.dw = ws;   // the first kernel writes the partial results, in fp32
    const bool out32 = a.out32 || split;
    const int size = out32 ? 4 : 2, ld = split ? pl.ldp : a.K;
    const bool rows16 = reinterpret_cast<uintptr_t>(a.dw) % 16 == 0 && (long long)ld * size % 16 == 0;
    alignas(64) CUtensorMap tdy, tx, tdw{};
    cudaError_t e = encode_mm(&tdy, dy, a.type(), 64, BK);
    if (e == cudaSuccess) e = encode_mm(&tx, x, a.type(), 64, BK);
    if (e == cudaSuccess && rows16)
        e = encode_mm(&tdw, MmOperand{a.dw, a.K, a.N, ld, a.E * a.splits, (long long)a.N * ld, false},
                      out32 ? DT_F32 : a.type(), 128 / size, 32);
    int nsm = 0;
    if (e == cudaSuccess) e = sm_count(&nsm);
    if (e != cudaSuccess) return e;
    const int pairs = (int)(pl.tiles < nsm / 2 ? pl.tiles : nsm / 2);
    if (rows16)
        e = out32 ? launch_pairs<C, k_mm_wgrad<float, true>>(pairs, a.E, a.behind, st, tdy, tx, tdw, a)
                  : launch_pairs<C, k_mm_wgrad<uint16_t, true>>(pairs, a.E, a.behind, st, tdy, tx, tdw, a);
    else
        e = out32 ? launch_pairs<C, k_mm_wgrad<float, false>>(pairs, a.E, a.behind, st, tdy, tx, tdw, a)
                  : launch_pairs<C, k_mm_wgrad<uint16_t, false>>(pairs, a.E, a.behind, st, tdy, tx, tdw, a);
    if (e != cudaSuccess || !split) return e;
    a.dw = args.dw;
    const long long quads = (long long)a.E * a.N * (pl.ldp / 4), ctas = (quads + 255) / 256;
    const dim3 grid((unsigned)(ctas < 8LL * nsm ? ctas : 8LL * nsm));
    return a.out32 ? launch_behind(k_mm_wgrad_join<float>, grid, 256, 0, st, a, (const float*)ws, pl.ldp)
                   : launch_behind(k_mm_wgrad_join<uint16_t>, grid, 256, 0, st, a, (const float*)ws, pl.ldp);
}

}  // namespace spq
