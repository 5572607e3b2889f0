// 16-bit rows copied to rows that start on 16 bytes, for the operands of the products grouped by expert (no reference
// counterpart).  Bound by HBM: every element read and written once.  A thread makes 16 bytes of a destination row from the
// two aligned 16-byte blocks of the source that hold them, shifted against each other (rows of odd length start at every
// even address); a block is read only if it holds an element of the row.  1537 rows and 24 experts of 1001x1111 (57 MB): 26
// us, of which writing 57 MB alone takes 20.
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

struct Jobs {
    PadJob j[2];
    long long vecs[2];   // 16-byte pieces of the destinations
};

__global__ void __launch_bounds__(256) k_pad_rows(const Jobs jobs) {
    const long long all = jobs.vecs[0] + jobs.vecs[1];
    for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < all; g += (long long)gridDim.x * 256) {
        const bool second = g >= jobs.vecs[0];
        const PadJob& j = jobs.j[second];
        const long long i = second ? g - jobs.vecs[0] : g;
        const int per = (j.cols + 7) / 8;
        const long long row = i / per, plane = row / j.rows;
        const int c = (int)(i - row * per) * 8;
        const uintptr_t first =
            reinterpret_cast<uintptr_t>(static_cast<const uint16_t*>(j.src) + plane * j.plane + (row - plane * j.rows) * j.ld);
        const uintptr_t a = first + 2 * (uintptr_t)c, end = first + 2 * (uintptr_t)j.cols, block = a & ~uintptr_t(15);
        const uint4 lo = *reinterpret_cast<const uint4*>(block);
        uint4 hi = make_uint4(0, 0, 0, 0);
        if (block != a && block + 16 < end) hi = *reinterpret_cast<const uint4*>(block + 16);
        reinterpret_cast<uint4*>(j.dst)[i] = align16(lo, hi, (int)(a - block));
    }
}

}  // namespace

cudaError_t launch_pad_rows(const PadJob* jobs, int count, cudaStream_t st) {
    int nsm = 0;
    const cudaError_t e = sm_count(&nsm);
    if (e != cudaSuccess) return e;
    Jobs js{};
    long long all = 0;
    for (int i = 0; i < count; ++i) {
        js.j[i] = jobs[i];
        all += js.vecs[i] = (long long)jobs[i].planes * jobs[i].rows * ((jobs[i].cols + 7) / 8);
    }
    const long long ctas = (all + 255) / 256;
    k_pad_rows<<<(unsigned)(ctas < 16LL * nsm ? ctas : 16LL * nsm), 256, 0, st>>>(js);
    return cudaGetLastError();
}

}  // namespace spq
