// What the products grouped by expert share: 16-bit tcgen05 products, TMA loads, and the map from offsets to tiles.
//
// Operand tiles hold 64 elements of the contracted dimension.  K-major (the contracted dimension contiguous in memory):
// R rows of 128 bytes, one TMA box, 8-row atoms of 1024 bytes with the 16-byte chunks of row m at chunk ^ (m % 8).
// MN-major (the other dimension contiguous): boxes of 64 columns x 64 contracted rows (8 KB), the same swizzle; one
// product of 16 contracted rows then starts 2048 bytes after the last.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "tc.cuh"

namespace spq {
namespace mm {

constexpr int BK = 64;                 // contracted elements per pipeline stage
constexpr int FT = 128;                // features (rows of TMEM) per CTA
constexpr int BOX_MN = 64 * 128;       // bytes of one MN-major box

// ---- products: 16-bit operands of one type, fp32 accumulation ----
// instruction descriptor: D fp32, A and B both bf16 or both fp16, each K-major or MN-major, M x N
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool bf16, bool a_mn, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) |
           ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// shared-memory descriptor of an MN-major 128-byte-swizzled tile: 64-column boxes 8 KB apart (leading byte offset),
// groups of 8 contracted rows 1024 bytes apart (stride byte offset)
__device__ __forceinline__ uint64_t sdesc_mn128(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(BOX_MN >> 4) << 16) | ((uint64_t)64u << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
template <bool MN>
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr) {
    return MN ? sdesc_mn128(saddr) : tc::sdesc_k128(saddr);
}
// bytes from one product's operand start to the next one's (16 contracted elements)
template <bool MN>
__device__ __forceinline__ constexpr uint32_t kstep() { return MN ? 2048u : 32u; }

// one thread of a whole warp, the same each time
__device__ __forceinline__ bool elect() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r != 0;
}

__device__ __forceinline__ void tma_load_2d(uint32_t smem_dst, const void* map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_dst), "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const void* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// the address in CTA `rank` of this cluster of a shared-memory address of this CTA
__device__ __forceinline__ uint32_t mapa(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}

// ---- 16-bit results ----
__device__ __forceinline__ uint16_t to16(float x, bool bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&b);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- accumulators (TMEM lanes = features, columns = rows of y) to row-major 16-bit rows of y ----
// 16 lanes x 32 columns as four fragments of 16 x 8: v[4 i + {0, 1}] of thread t is lane t / 4, columns 8 i + 2 (t % 4) + {0,
// 1}; v[4 i + {2, 3}] the same 8 lanes on
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// four 8 x 8 matrices of 16-bit values, each transposed: lane 8 i + r gives the address of row r of matrix i as stored
__device__ __forceinline__ void stmatrix4t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
                 "r"(d)
                 : "memory");
}
constexpr int Y_PITCH = 80;            // bytes from one staged row of y to the next: 32 features and 16 bytes against conflicts
constexpr int Y_STAGE = 2 * 32 * Y_PITCH;   // per warp: two blocks of 32 rows in turn

// This warp's 32 features of a tile's rows c0, c0 + step, ... (blocks of 32, below cols): TMEM at `taddr` (this warp's lanes,
// the tile's first column) through `stage` to y + r * ldy, rows r < rows and features f < features.  v16: every row of y and
// the first feature are on 16 bytes.  The next block's accumulators are read while this one is stored.
__device__ __forceinline__ void store_y(uint32_t taddr, uint32_t stage, uint16_t* y, long long ldy, int c0, int step, int cols,
                                        int rows, int features, bool bf16, bool v16) {
    const int lane = threadIdx.x & 31, f = (lane & 3) * 8;
    const uint32_t at = ((lane >> 4) * 8 + (lane & 7)) * Y_PITCH + ((lane >> 3) & 1) * 16;
    float v[2][16];
    if (c0 < cols) {
        tmem_ld_frag(taddr + c0, v[0]);
        tmem_ld_frag(taddr + c0 + (16u << 16), v[1]);
    }
    uint32_t other = stage + 32 * Y_PITCH;
    for (int c = c0; c < cols; c += step) {
        tc::tmem_wait_ld();
        uint32_t w[2][8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i) w[h][i] = pack16(v[h][2 * i], v[h][2 * i + 1], bf16);
        if (c + step < cols) {
            tmem_ld_frag(taddr + c + step, v[0]);
            tmem_ld_frag(taddr + c + step + (16u << 16), v[1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            stmatrix4t(stage + at + h * 32, w[h][0], w[h][1], w[h][2], w[h][3]);
            stmatrix4t(stage + at + h * 32 + 16 * Y_PITCH, w[h][4], w[h][5], w[h][6], w[h][7]);
        }
        __syncwarp();   // (the buffer's last readers passed the block in between)
        if (v16) {   // 16 bytes a lane, 64 of each of 8 rows at a time
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 2);
                uint32_t u[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
                             : "r"(stage + r * Y_PITCH + f * 2)
                             : "memory");
                if (c + r >= rows) continue;
                uint16_t* const o = y + (long long)(c + r) * ldy + f;
                if (f + 8 <= features) {
                    *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[2], u[3]);
                } else {
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        if (f + x < features) o[x] = (uint16_t)(u[x >> 1] >> (16 * (x & 1)));
                }
            }
        } else {     // rows at any address: a lane is a feature
            const int last = min(32, rows - c);
            for (int r = 0; r < last; ++r) {
                uint16_t u;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(stage + r * Y_PITCH + lane * 2) : "memory");
                if (lane < features) y[(long long)(c + r) * ldy + lane] = u;
            }
        }
        const uint32_t next = other;
        other = stage;
        stage = next;
    }
}

// ---- offsets -> tiles ----
// start[e], start[e + 1]: the rows of expert e; pre[e]: tiles of `rows` rows before it (both E + 1 long, in shared
// memory).  offsets[e] is the end of expert e's rows; ends are clamped to [previous end, T], so that no offsets make a
// kernel leave its tensors.  Run by one whole warp.
__device__ __forceinline__ void map_groups(const int* __restrict__ offsets, int E, int T, int rows, int* start, int* pre) {
    const int lane = threadIdx.x & 31;
    int end = 0, tiles = 0;
    int next = lane < E ? offsets[lane] : 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
        int v = min(max(next, 0), T);
        if (e0 + 32 + lane < E) next = offsets[e0 + 32 + lane];
        else next = 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(~0u, v, o);
            if (lane >= o) v = max(v, u);
        }
        v = max(v, end);
        int before = __shfl_up_sync(~0u, v, 1);
        if (lane == 0) before = end;
        int s = (v - before + rows - 1) / rows;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(~0u, s, o);
            if (lane >= o) s += u;
        }
        if (e0 + lane < E) {
            start[e0 + lane + 1] = v;
            pre[e0 + lane + 1] = tiles + s;
        }
        end = __shfl_sync(~0u, v, 31);
        tiles += __shfl_sync(~0u, s, 31);
    }
    if (lane == 0) start[0] = pre[0] = 0;
}

// the expert that holds row tile u < pre[E]
__device__ __forceinline__ int group_of(const int* pre, int E, int u) {
    int lo = 0, hi = E - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid + 1] > u) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

}  // namespace mm
}  // namespace spq
