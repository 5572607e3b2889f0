// 16-bit rows copied to rows that start on 16 bytes, for the operands of the products grouped by expert (no reference
// counterpart).  Bound by HBM: every element read and written once.  A thread makes 16 bytes of a destination row from the
// two aligned 16-byte blocks of the source that hold them, shifted against each other (rows of odd length start at every
// even address); a block is read only if it holds an element of the row.
#include "kernels.h"

namespace spq {
namespace {

// the 16 bytes that begin `shift` bytes (even, below 16) into lo : hi
__device__ __forceinline__ uint4 align16(uint4 lo, uint4 hi, int shift) {
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t o[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {   // whole words by selection (registers have no addresses), then half a word
        if (shift >> 2 == s) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i] = (shift & 2) ? __funnelshift_r(w[s + i], s + i + 1 < 8 ? w[s + i + 1] : 0u, 16) : w[s + i];
        }
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// rows [plane][row] of `cols` elements, ld and plane_stride elements apart -> rows of ldd elements (a multiple of 8)
__global__ void __launch_bounds__(256) k_pad_rows(const uint16_t* __restrict__ src, long long plane_stride, long long ld,
                                                  int rows, int cols, uint16_t* __restrict__ dst, int ldd, long long vecs) {
    const int per = ldd / 8;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < vecs; i += (long long)gridDim.x * 256) {
        const long long row = i / per, plane = row / rows;
        const int c = (int)(i - row * per) * 8;
        const uintptr_t first = reinterpret_cast<uintptr_t>(src + plane * plane_stride + (row - plane * rows) * ld);
        const uintptr_t a = first + 2 * (uintptr_t)c, end = first + 2 * (uintptr_t)cols, block = a & ~uintptr_t(15);
        const uint4 lo = *reinterpret_cast<const uint4*>(block);
        uint4 hi = make_uint4(0, 0, 0, 0);
        if (block != a && block + 16 < end) hi = *reinterpret_cast<const uint4*>(block + 16);
        *reinterpret_cast<uint4*>(dst + i * 8) = align16(lo, hi, (int)(a - block));
    }
}

}  // namespace

cudaError_t launch_pad_rows(const void* src, long long plane_stride, long long ld, int planes, int rows, int cols, void* dst,
                            int ldd, cudaStream_t st) {
    int nsm = 0;
    const cudaError_t e = sm_count(&nsm);
    if (e != cudaSuccess) return e;
    const long long vecs = (long long)planes * rows * (ldd / 8), ctas = (vecs + 255) / 256;
    k_pad_rows<<<(unsigned)(ctas < 16LL * nsm ? ctas : 16LL * nsm), 256, 0, st>>>(
        static_cast<const uint16_t*>(src), plane_stride, ld, rows, cols, static_cast<uint16_t*>(dst), ldd, vecs);
    return cudaGetLastError();
}

}  // namespace spq
