// 16-bit rows copied to rows that start on 16 bytes, for the operands of the products grouped by expert (no reference
// counterpart).  Bound by HBM: every element read and written once.  A thread makes 16 bytes of a destination row from the
// four or five aligned 4-byte words of the source that hold them (rows of odd length start at every even address); a word
// is read only if it holds an element of the row.  1537 rows and 24 experts of 1001x1111, 57 MB each way: 28 us, where a
// copy of as much takes 27.
#include "kernels.h"

namespace spq {
namespace {

// `lanes` threads (a power of two up to a warp) copy one row, then the one `groups` rows on: the plane is carried along,
// because 64-bit divisions for every 16 bytes took longer than the copy
__device__ __forceinline__ void pad_rows(const PadJob& j, int lanes, long long group, long long groups, int lane) {
    const int per = (j.cols + 7) / 8;
    const int step_planes = (int)(groups / j.rows), step_rows = (int)(groups - (long long)step_planes * j.rows);
    int plane = (int)min(group / j.rows, (long long)j.planes), row = (int)(group - (long long)plane * j.rows);
    while (plane < j.planes) {
        // (an end that is not above the one before it leaves its expert empty, whatever the others are)
        if (!j.ends || j.ends[plane] > (plane ? j.ends[plane - 1] : 0)) {
            const uintptr_t first = reinterpret_cast<uintptr_t>(static_cast<const uint16_t*>(j.src) + plane * j.plane + row * j.ld);
            const uint32_t* const src = reinterpret_cast<const uint32_t*>(first & ~uintptr_t(3));
            const int odd = (int)(first >> 1) & 1, words = (j.cols + odd + 1) / 2;   // words that hold elements of the row
            uint4* const dst = static_cast<uint4*>(j.dst) + ((long long)plane * j.rows + row) * per;
            const int full = (words - odd) / 4;   // pieces whose words all do
#pragma unroll 4
            for (int i = lane; i < full; i += lanes) {
                const uint32_t* const p = src + 4 * i;
                uint4 v = make_uint4(p[0], p[1], p[2], p[3]);
                if (odd)
                    v = make_uint4(__funnelshift_r(v.x, v.y, 16), __funnelshift_r(v.y, v.z, 16), __funnelshift_r(v.z, v.w, 16),
                                   __funnelshift_r(v.w, p[4], 16));
                dst[i] = v;
            }
            if (full < per && lane == (full & (lanes - 1))) {   // the last piece
                uint32_t w[5];
#pragma unroll
                for (int k = 0; k < 5; ++k) w[k] = 4 * full + k < words ? src[4 * full + k] : 0u;
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = odd ? __funnelshift_r(w[k], w[k + 1], 16) : w[k];
                dst[full] = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        plane += step_planes;
        row += step_rows;
        if (row >= j.rows) {
            row -= j.rows;
            ++plane;
        }
    }
}

constexpr int CTAS_PER_SM = 6;   // all resident at once: a second round of a few CTAs took as long as the first

struct Jobs {
    PadJob j[2];
    int lanes[2];
    int ctas[2];   // blocks 0 .. ctas[0] - 1 take the first job
};

__global__ void __launch_bounds__(256, CTAS_PER_SM) k_pad_rows(const __grid_constant__ Jobs jobs) {
    auto take = [&](const PadJob& j, int lanes, int ctas, int block) {
        const int per_cta = 256 / lanes;
        pad_rows(j, lanes, (long long)block * per_cta + threadIdx.x / lanes, (long long)ctas * per_cta, threadIdx.x & (lanes - 1));
    };
    launch_dependents();
    // (not jobs.j[i]: parameters under a variable index are copied to local memory first)
    const int block = (int)blockIdx.x - jobs.ctas[0];
    if (block < 0) take(jobs.j[0], jobs.lanes[0], jobs.ctas[0], (int)blockIdx.x);
    else take(jobs.j[1], jobs.lanes[1], jobs.ctas[1], block);
}

}  // namespace

cudaError_t launch_pad_rows(const PadJob* jobs, int count, cudaStream_t st) {
    int nsm = 0;
    const cudaError_t e = sm_count(&nsm);
    if (e != cudaSuccess) return e;
    Jobs js{};
    double all = 0.0;
    for (int i = 0; i < count; ++i) all += (double)jobs[i].planes * jobs[i].rows * jobs[i].cols;
    for (int i = 0; i < count; ++i) {   // the CTAs by the jobs' sizes
        js.j[i] = jobs[i];
        int lanes = 1;
        while (lanes < 32 && lanes * 8 < jobs[i].cols) lanes *= 2;
        js.lanes[i] = lanes;
        const double n = (double)jobs[i].planes * jobs[i].rows, need = (n * lanes + 255) / 256;
        const double share = (CTAS_PER_SM * nsm - 1) * (n * jobs[i].cols / all);
        js.ctas[i] = need < share ? (int)need : share < 1 ? 1 : (int)share;
    }
    k_pad_rows<<<js.ctas[0] + js.ctas[1], 256, 0, st>>>(js);
    return cudaGetLastError();
}

}  // namespace spq
