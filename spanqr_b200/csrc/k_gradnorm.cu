// The global L2 norm of a list of gradients, and the list scaled to a maximal norm (no reference counterpart).
//
//   n = sqrt(sum_i sum_j x_ij^2),   y_ij = x_ij * min(1, max_norm / (n + 1e-6))
//
// Both passes are bound by HBM: the norm reads every element once, the scaling reads and writes it once.  A list of
// hundreds of tensors of any sizes is cut into chunks of CHUNK bytes (each inside one tensor, its start rounded down to
// 32 bytes so that every load but a tensor's first and last is one aligned 32-byte vector); the persistent grid takes
// the chunks in turn.  The table of tensors travels in the kernel's parameters, so a call copies nothing to the device
// and a captured call keeps its table.
//
// Arithmetic: 32 bytes of squares (8 fp32 or 16 sixteen-bit values) are summed in fp32 and added to an fp64 sum: one
// conversion per vector, because fp32 -> fp64 conversions run at about 10 per clock per SM, which at one per element
// would cost more than the reads.  Squares leave fp32's range long before the norm does, so a vector whose sum is
// outside [2^-80, 2^120] is summed again, its values scaled by 2^100 (all are below 2^-40, and the smallest subnormal's
// square is then 2^-98) or by 2^-80 (one is above 2^58, and the largest square is then 2^96).
// Every CTA's sum goes to its own slot; the slots are added in one fixed order, so a list gives the same bits each time.
//
// Measured: the norm of 2.3 GB of bf16 in 313 us (7.3 TB/s); 1.7 GB of fp32 clipped to new tensors in 816 us (6.3 TB/s over
// the three passes); 14 tensors of 768x512 in 7 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "tc.cuh"

namespace spq {
namespace {

constexpr int THREADS = 256;
constexpr int UNROLL = 4;                              // 32-byte vectors in flight per thread
constexpr int CHUNK = THREADS * UNROLL * 32;           // bytes of input per chunk (32 KB)

template <int CAP>
struct Table {
    GradEntry e[CAP];
    unsigned first[CAP + 1];   // first chunk of each tensor in this launch; first[count] = all chunks
    int count;
    bool in_place;             // every output is its input
};

// the tensor that holds chunk c
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& t, unsigned c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

struct Vec {
    uint32_t w[8];
};

__device__ __forceinline__ Vec load32(const char* p) {
    Vec v;
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]),
                   "=r"(v.w[7])
                 : "l"(p));
    return v;
}
__device__ __forceinline__ void store32(char* p, const Vec& v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]),
                 "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
                 : "memory");
}

// one value at byte address p
template <int TYPE>
__device__ __forceinline__ float load1(const char* p) {
    if constexpr (TYPE == DT_F32) return *reinterpret_cast<const float*>(p);
    if constexpr (TYPE == DT_F16) return __half2float(*reinterpret_cast<const __half*>(p));
    return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
}
template <int TYPE>
__device__ __forceinline__ void store1(char* p, float x) {
    if constexpr (TYPE == DT_F32) *reinterpret_cast<float*>(p) = x;
    else if constexpr (TYPE == DT_F16) *reinterpret_cast<__half*>(p) = __float2half_rn(x);
    else *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(x);
}

// the values of a vector: 8 fp32 or 16 sixteen-bit ones
template <int TYPE>
struct Values {
    static constexpr int N = TYPE == DT_F32 ? 8 : 16;
    float x[N];
};
template <int TYPE>
__device__ __forceinline__ Values<TYPE> values(const Vec& v) {
    Values<TYPE> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (TYPE == DT_F32) {
            r.x[i] = __uint_as_float(v.w[i]);
        } else if constexpr (TYPE == DT_BF16) {
            r.x[2 * i] = __uint_as_float(v.w[i] << 16);
            r.x[2 * i + 1] = __uint_as_float(v.w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
            r.x[2 * i] = f.x;
            r.x[2 * i + 1] = f.y;
        }
    }
    return r;
}

// sum of squares of one vector (see the head of the file)
template <int TYPE>
__device__ __forceinline__ double sumsq(const Vec& v) {
    const Values<TYPE> r = values<TYPE>(v);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < r.N; ++i) s = __fmaf_rn(r.x[i], r.x[i], s);
    if (TYPE != DT_F16 && !(s >= 0x1p-80f && s <= 0x1p120f)) {   // out of range, zero, infinite or NaN
        const bool big = !(s < 1.0f);
        const float f = big ? 0x1p-80f : 0x1p100f;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < r.N; ++i) {
            const float t = r.x[i] * f;
            s = __fmaf_rn(t, t, s);
        }
        return (double)s * (big ? 0x1p160 : 0x1p-200);
    }
    return (double)s;
}

__device__ __forceinline__ uintptr_t down32(uintptr_t a) { return a & ~uintptr_t(31); }

// one chunk of a tensor: whole(the thread's vectors, the first one's address) where the chunk lies inside the tensor,
// else vector(v, address) and element(address) for what of it does
template <int TYPE, typename W, typename V, typename E>
__device__ __forceinline__ void for_chunk(const GradEntry& e, unsigned local, W&& whole, V&& vector, E&& element) {
    constexpr int ES = TYPE == DT_F32 ? 4 : 2;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(e.in), end = begin + (uintptr_t)e.n * ES;
    const uintptr_t chunk = down32(begin) + (uintptr_t)local * CHUNK, base = chunk + threadIdx.x * 32;
    if (chunk >= begin && chunk + CHUNK <= end) {
        Vec v[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) v[k] = load32(reinterpret_cast<const char*>(base + k * THREADS * 32));
        whole(v, base);
        return;
    }
#pragma unroll 1
    for (int k = 0; k < UNROLL; ++k) {
        const uintptr_t a = base + k * THREADS * 32;
        if (a >= begin && a + 32 <= end) {
            vector(load32(reinterpret_cast<const char*>(a)), a);
        } else {
#pragma unroll 1
            for (uintptr_t b = a; b < a + 32; b += ES)
                if (b >= begin && b < end) element(b);
        }
    }
}

template <int TYPE>
__device__ __forceinline__ double chunk_sumsq(const GradEntry& e, unsigned local) {
    double acc = 0.0;
    for_chunk<TYPE>(
        e, local,
        [&](const Vec(&v)[UNROLL], uintptr_t) {
#pragma unroll
            for (int k = 0; k < UNROLL; ++k) acc += sumsq<TYPE>(v[k]);
        },
        [&](const Vec& v, uintptr_t) { acc += sumsq<TYPE>(v); },
        [&](uintptr_t a) {
            const double x = (double)load1<TYPE>(reinterpret_cast<const char*>(a));
            acc += x * x;
        });
    return acc;
}

template <int CAP>
__global__ void __launch_bounds__(THREADS, GRAD_CTAS_PER_SM)
    k_grad_sumsq(const __grid_constant__ Table<CAP> t, double* __restrict__ part) {
    double acc = 0.0;
    const unsigned all = t.first[t.count];
    launch_dependents();   // the kernel that adds the slots starts while the last chunks are read
    for (unsigned c = blockIdx.x; c < all; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const GradEntry& e = t.e[i];
        const unsigned local = c - t.first[i];
        acc += e.in_type == DT_F32 ? chunk_sumsq<DT_F32>(e, local)
                                   : (e.in_type == DT_F16 ? chunk_sumsq<DT_F16>(e, local) : chunk_sumsq<DT_BF16>(e, local));
    }
    __shared__ double red[THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(~0u, acc, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = red[0];
#pragma unroll
        for (int w = 1; w < THREADS / 32; ++w) s += red[w];
        part[blockIdx.x] = s;
    }
}

// the slots' sum, the same bits in every CTA that takes it.  (Not __restrict__, here and in the kernels that call this: a
// kernel that starts before its predecessor's end must not read what that still writes as data that nobody changes.)
__device__ double total(const double* part, int nparts) {
    __shared__ double red[THREADS / 32];
    double acc = 0.0;
    wait_primary();   // the slots are written
    for (int i = threadIdx.x; i < nparts; i += THREADS) acc += part[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(~0u, acc, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
    __syncthreads();
    double s = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) s += red[w];
    return s;
}

__global__ void __launch_bounds__(THREADS) k_grad_finish(const double* part, int nparts, double* sumsq_out,
                                                         float* norm) {
    const double s = total(part, nparts);
    if (threadIdx.x == 0) {
        if (sumsq_out) *sumsq_out = s;
        if (norm) *norm = (float)sqrt(s);
    }
}

struct Coef {
    float c, p;
};

template <int IN, int OUT>
__device__ __forceinline__ void scale_vec(const GradEntry& e, const Vec& v, uintptr_t a, Coef coef) {
    constexpr int ES = IN == DT_F32 ? 4 : 2, OS = OUT == DT_F32 ? 4 : 2;
    Values<IN> r = values<IN>(v);
#pragma unroll
    for (int i = 0; i < r.N; ++i) r.x[i] = r.x[i] * coef.c * coef.p;
    char* o = static_cast<char*>(e.out) + (a - reinterpret_cast<uintptr_t>(e.in)) / ES * OS;
    if ((reinterpret_cast<uintptr_t>(o) & 31) == 0) {
        constexpr int PER = 32 / OS;   // values of one output vector
#pragma unroll
        for (int h = 0; h < r.N / PER; ++h) {
            Vec w;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (OUT == DT_F32) {
                    w.w[i] = __float_as_uint(r.x[h * PER + i]);
                } else if constexpr (OUT == DT_BF16) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(r.x[2 * i], r.x[2 * i + 1]);
                    w.w[i] = *reinterpret_cast<const uint32_t*>(&b);
                } else {
                    const __half2 b = __floats2half2_rn(r.x[2 * i], r.x[2 * i + 1]);
                    w.w[i] = *reinterpret_cast<const uint32_t*>(&b);
                }
            }
            store32(o + 32 * h, w);
        }
    } else {   // an output whose address differs from the input's modulo 32 bytes
#pragma unroll
        for (int i = 0; i < r.N; ++i) store1<OUT>(o + i * OS, r.x[i]);
    }
}

template <int IN, int OUT>
__device__ __forceinline__ void chunk_scale(const GradEntry& e, unsigned local, Coef coef) {
    constexpr int ES = IN == DT_F32 ? 4 : 2, OS = OUT == DT_F32 ? 4 : 2;
    for_chunk<IN>(
        e, local,
        [&](const Vec(&v)[UNROLL], uintptr_t base) {
#pragma unroll
            for (int k = 0; k < UNROLL; ++k) scale_vec<IN, OUT>(e, v[k], base + k * THREADS * 32, coef);
        },
        [&](const Vec& v, uintptr_t a) { scale_vec<IN, OUT>(e, v, a, coef); },
        [&](uintptr_t a) {
            char* o = static_cast<char*>(e.out) + (a - reinterpret_cast<uintptr_t>(e.in)) / ES * OS;
            store1<OUT>(o, load1<IN>(reinterpret_cast<const char*>(a)) * coef.c * coef.p);
        });
}

// Every CTA adds the slots itself (a few KB out of L2; a launch of its own for the sum would cost more), then scales
// its chunks, the list's last ones first: those are the ones the norm's pass left in the caches.  A coefficient of
// one leaves tensors clipped in place unread and unwritten.
template <int CAP>
__global__ void __launch_bounds__(THREADS, GRAD_CTAS_PER_SM)
    k_grad_scale(const __grid_constant__ Table<CAP> t, const double* part, int nparts, double max_norm, float* norm) {
    const double n = sqrt(total(part, nparts));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double c = n == INFINITY ? 0.0 : max_norm / (n + 1e-6);   // (zero for an infinite max_norm too)
    // x * coef as (x * c32) * p, so that a coefficient below fp32's normal range (a norm near or above fp32's largest value,
    // or a small max_norm) keeps its bits: c32 = c * 2^64 down to 2^-190, c * 2^149 below (and below 2^-278 every product
    // rounds to zero), p the other power; else p = 1.  x * c32 stays in range, and normal where the result is not zero
    const double up = c < 0x1p-190 ? 0x1p149 : c < 0x1p-100 ? 0x1p64 : 1.0;
    const Coef coef{(float)(c >= 1.0 ? 1.0 : c * up), (float)(1.0 / up)};   // a NaN norm gives NaN
    const bool unchanged = coef.c == 1.0f && coef.p == 1.0f;
    if (unchanged && t.in_place) return;
    const unsigned all = t.first[t.count];
    for (unsigned k = blockIdx.x; k < all; k += gridDim.x) {
        const unsigned ch = all - 1 - k;
        const int i = tensor_of(t, ch);
        const GradEntry& e = t.e[i];
        if (unchanged && e.in == e.out) continue;
        const unsigned local = ch - t.first[i];
        if (e.in_type == DT_F32) chunk_scale<DT_F32, DT_F32>(e, local, coef);
        else if (e.in_type == DT_F16 && e.out_type == DT_F16) chunk_scale<DT_F16, DT_F16>(e, local, coef);
        else if (e.in_type == DT_F16) chunk_scale<DT_F16, DT_F32>(e, local, coef);
        else if (e.out_type == DT_BF16) chunk_scale<DT_BF16, DT_BF16>(e, local, coef);
        else chunk_scale<DT_BF16, DT_F32>(e, local, coef);
    }
}

// a launch's table: two capacities, because the parameters of every launch are copied whole (2.3 KB and 32 KB)
constexpr int CAP_SMALL = 64, CAP_LARGE = 900;

template <int CAP>
unsigned fill(Table<CAP>& t, const GradEntry* e, int count) {
    unsigned c = 0;
    t.in_place = true;
    for (int i = 0; i < count; ++i) {
        t.in_place = t.in_place && e[i].in == e[i].out;
        t.e[i] = e[i];
        t.first[i] = c;
        const uintptr_t b = reinterpret_cast<uintptr_t>(e[i].in);
        const uintptr_t bytes = (uintptr_t)e[i].n * (e[i].in_type == DT_F32 ? 4 : 2) + (b & 31);
        c += (unsigned)((bytes + CHUNK - 1) / CHUNK);
    }
    t.first[count] = c;
    t.count = count;
    return c;
}

int grid_for(unsigned chunks, int nsm) {
    const unsigned most = (unsigned)(nsm * GRAD_CTAS_PER_SM);
    return (int)(chunks < most ? (chunks ? chunks : 1) : most);
}

template <int CAP>
cudaError_t sumsq_launch(const GradEntry* e, int count, int nsm, double* part, int* nparts, cudaStream_t st) {
    Table<CAP> t;
    const int grid = grid_for(fill(t, e, count), nsm);
    k_grad_sumsq<CAP><<<grid, THREADS, 0, st>>>(t, part);
    *nparts += grid;
    return cudaGetLastError();
}

template <int CAP>
cudaError_t scale_launch(const GradEntry* e, int count, int nsm, const double* part, int nparts, double max_norm,
                         float* norm, bool behind, cudaStream_t st) {
    Table<CAP> t;
    const int grid = grid_for(fill(t, e, count), nsm);
    if (behind) return launch_behind(k_grad_scale<CAP>, dim3(grid), THREADS, 0, st, t, part, nparts, max_norm, norm);
    k_grad_scale<CAP><<<grid, THREADS, 0, st>>>(t, part, nparts, max_norm, norm);
    return cudaGetLastError();
}

}  // namespace

int grad_launches(int count) { return count <= CAP_SMALL ? 1 : (count + CAP_LARGE - 1) / CAP_LARGE; }

cudaError_t launch_grad_sumsq(const GradEntry* e, int count, double* part, int* nparts, cudaStream_t st) {
    int nsm = 0;
    cudaError_t err = sm_count(&nsm);
    *nparts = 0;
    if (err == cudaSuccess && count <= CAP_SMALL) return sumsq_launch<CAP_SMALL>(e, count, nsm, part, nparts, st);
    for (int i = 0; err == cudaSuccess && i < count; i += CAP_LARGE)
        err = sumsq_launch<CAP_LARGE>(e + i, count - i < CAP_LARGE ? count - i : CAP_LARGE, nsm, part + *nparts, nparts, st);
    return err;
}

cudaError_t launch_grad_finish(const double* part, int nparts, double* sumsq, float* norm, bool behind, cudaStream_t st) {
    if (behind) return launch_behind(k_grad_finish, dim3(1), THREADS, 0, st, part, nparts, sumsq, norm);
    k_grad_finish<<<1, THREADS, 0, st>>>(part, nparts, sumsq, norm);
    return cudaGetLastError();
}

cudaError_t launch_grad_scale(const GradEntry* e, int count, const double* part, int nparts, double max_norm, float* norm,
                              bool behind, cudaStream_t st) {
    int nsm = 0;
    cudaError_t err = sm_count(&nsm);
    if (err == cudaSuccess && count <= CAP_SMALL)
        return scale_launch<CAP_SMALL>(e, count, nsm, part, nparts, max_norm, norm, behind, st);
    if (err == cudaSuccess && count <= CAP_LARGE)
        return scale_launch<CAP_LARGE>(e, count, nsm, part, nparts, max_norm, norm, behind, st);
    for (int i = (count - 1) / CAP_LARGE * CAP_LARGE; err == cudaSuccess && i >= 0; i -= CAP_LARGE)   // the last part first
        err = scale_launch<CAP_LARGE>(e + i, count - i < CAP_LARGE ? count - i : CAP_LARGE, nsm, part, nparts, max_norm,
                                      i == 0 ? norm : nullptr, false, st);
    return err;
}

}  // namespace spq
