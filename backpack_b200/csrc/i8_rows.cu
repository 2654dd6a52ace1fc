// Rows to 8 bits: residual addition, root-mean-square norm and symmetric quantisation with one scale per row, one pass.
//
// For a row of K values (all in float; x, r and the sum may be stored in 16 bits)
//   v = x + r,   p = v * w,   a = max |p|,   rstd = 1 / sqrt(mean(v^2) + eps)
//   code = round_half_even(127 p / a),   scale = a * rstd / 127
// rstd is a factor of the whole row and of its largest value, so the codes do not depend on it: they are computed from the
// exact quotient and never differ with the order of a sum.  In float the quotient is off by at most 127 * 3 * 2^-24 = 2.3e-5
// (the product, 127/a and their product are rounded); a quotient that lies nearer than 4e-5 to the middle between two codes
// is computed again in double from the exact product (48 bits) and the exact a.
//
// Memory bound (13 bytes a value with a float residual stream).  A row's values stay in registers between the two halves
// (statistics, codes); the reduction in between takes one barrier.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "q4k_common.cuh"

namespace bpq4k {

namespace {

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// E elements with one access: 16 bytes, or a single element on rows that are not 16-byte aligned.
template <typename T, int E>
struct Pack {
    T v[E];
};
template <typename T, int E>
__device__ __forceinline__ Pack<T, E> load_pack(const T* p) {
    Pack<T, E> r;
    if constexpr (E == 1) {
        r.v[0] = *p;
    } else {
        static_assert(sizeof(T) * E == 16, "16 bytes");
        *reinterpret_cast<uint4*>(r.v) = *reinterpret_cast<const uint4*>(p);
    }
    return r;
}
template <typename T, int E>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, E>& r) {
    if constexpr (E == 1)
        *p = r.v[0];
    else
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.v);
}

// Monotonic map of a float to an unsigned word, and back.
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t b = __float_as_uint(f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

// A thread holds PT values: PT / E accesses, blockDim.x of them apart.
template <typename T, int E, int PT, bool NORM, bool RES>
__global__ void __launch_bounds__(1024) rows_i8_kernel(const __grid_constant__ RowsI8Args a) {
    constexpr int NV = PT / E;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, warps = blockDim.x >> 5;
    const T* x = static_cast<const T*>(a.X) + (uint64_t)row * a.ldx;
    const T* r = RES ? static_cast<const T*>(a.R) + (uint64_t)row * a.ldr : nullptr;
    T* sum = RES && a.sum ? static_cast<T*>(a.sum) + (uint64_t)row * a.lds : nullptr;
    int8_t* codes = a.codes + (uint64_t)row * a.ldc;

    auto weights = [&](uint32_t e, float (&w)[E]) {
        if constexpr (E == 1) {
            w[0] = __ldg(a.w + e);
        } else {
#pragma unroll
            for (int j = 0; j < E; j += 4) {
                const float4 t = __ldg(reinterpret_cast<const float4*>(a.w + e + j));
                w[j] = t.x, w[j + 1] = t.y, w[j + 2] = t.z, w[j + 3] = t.w;
            }
        }
    };

    float v[PT];
    float ss = 0.f, lo = 0.f;
    uint32_t hi = 0u;  // the largest |p| as bits: a NaN or an infinity is the largest of all; `lo` its exact rounding error
    {
        Pack<T, E> xv[NV], rv[RES ? NV : 1];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const uint32_t e = (tid + i * blockDim.x) * E;
            if (e < a.K) xv[i] = load_pack<T, E>(x + e);
        }
        if constexpr (RES) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const uint32_t e = (tid + i * blockDim.x) * E;
                if (e < a.K) rv[i] = load_pack<T, E>(r + e);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const uint32_t e = (tid + i * blockDim.x) * E;
            if (e >= a.K) {
#pragma unroll
                for (int j = 0; j < E; j++) v[i * E + j] = 0.f;
                continue;
            }
            float w[E];
            if constexpr (NORM) weights(e, w);
#pragma unroll
            for (int j = 0; j < E; j++) {
                float s = Elem<T>::get(xv[i].v[j]);
                if constexpr (RES) s += Elem<T>::get(rv[i].v[j]);
                v[i * E + j] = s;
                if constexpr (NORM) {
                    ss = fmaf(s, s, ss);
                    const float p = fabsf(s * w[j]);
                    const uint32_t b = __float_as_uint(p);
                    if (b >= hi) {
                        const float l = fmaf(fabsf(s), fabsf(w[j]), -p);
                        lo = b > hi ? l : fmaxf(lo, l);
                        hi = b;
                    }
                } else {
                    hi = max(hi, __float_as_uint(fabsf(s)));
                }
            }
            if (RES && sum) {
                Pack<T, E> o;
#pragma unroll
                for (int j = 0; j < E; j++) o.v[j] = Elem<T>::put(v[i * E + j]);
                if (BPQ4K_CHECK(e + E <= a.K, a.status)) store_pack<T, E>(sum + e, o);
            }
        }
    }

    __shared__ uint32_t s_hi[32], s_lo[32];
    __shared__ float s_ss[32];
    __shared__ double s_sq[32], s_peak[32];
    // the largest (hi, lo) of lanes: the largest hi, and the largest lo beside it
    auto largest = [](uint32_t& h, uint32_t& l) {
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, h);
        l = __reduce_max_sync(0xFFFFFFFFu, h == top ? l : 0u);
        h = top;
    };
    uint32_t low = ordered(lo);
    largest(hi, low);
    if constexpr (NORM) {
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    }
    if (lane == 0) s_hi[warp] = hi, s_lo[warp] = low, s_ss[warp] = ss;
    __syncthreads();
    hi = lane < warps ? s_hi[lane] : 0u;
    low = lane < warps ? s_lo[lane] : 0u;
    largest(hi, low);
    double rstd = 1.0, peak = (double)__uint_as_float(hi) + (NORM ? (double)unordered(low) : 0.0);
    if constexpr (NORM) {
        ss = lane < warps ? s_ss[lane] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        double sq = ss;
        // squares, or low parts of products, beyond what a float holds well (every thread sees the same, so all or none come here)
        if (!(ss > 1e-20f && ss < 1e30f) || __uint_as_float(hi) < 1e-30f) {
            sq = 0.0, peak = 0.0;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const uint32_t e = (tid + i * blockDim.x) * E;
                if (e >= a.K) continue;
                float w[E];
                weights(e, w);
#pragma unroll
                for (int j = 0; j < E; j++) {
                    const double s = (double)v[i * E + j];
                    sq += s * s;
                    peak = fmax(peak, fabs(s * (double)w[j]));
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                sq += __shfl_xor_sync(0xFFFFFFFFu, sq, o);
                peak = fmax(peak, __shfl_xor_sync(0xFFFFFFFFu, peak, o));
            }
            if (lane == 0) s_sq[warp] = sq, s_peak[warp] = peak;
            __syncthreads();
            sq = lane < warps ? s_sq[lane] : 0.0;
            peak = lane < warps ? s_peak[lane] : 0.0;
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                sq += __shfl_xor_sync(0xFFFFFFFFu, sq, o);
                peak = fmax(peak, __shfl_xor_sync(0xFFFFFFFFu, peak, o));
            }
        }
        rstd = rsqrt(sq / (double)a.K + (double)a.eps);
    }
    const bool bad = hi >= 0x7F800000u;
    if (tid == 0) a.scales[row] = bad ? __uint_as_float(0x7FC00000u) : peak == 0.0 ? 0.f : (float)(peak * rstd / 127.0);

    const float inv = 127.f / (float)peak;
    const bool zero = bad || peak == 0.0, tiny = peak < 1e-30;  // (127 / a, or the low parts of products, leave the float range)
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const uint32_t e = (tid + i * blockDim.x) * E;
        if (e >= a.K) continue;
        float w[E];
        if constexpr (NORM) weights(e, w);
        uint32_t q[E];
#pragma unroll
        for (int j = 0; j < E; j++) {
            const float s = v[i * E + j];
            const float t = (NORM ? s * w[j] : s) * inv;
            const float c = t + 12582912.f;  // 1.5 * 2^23: the low byte of the sum is the rounded quotient
            q[j] = __float_as_uint(c);
            if (zero) {
                q[j] = 0u;
            } else if (tiny || fabsf(t - (c - 12582912.f)) > 0.5f - 4e-5f) {
                const double p = NORM ? (double)s * (double)w[j] : (double)s;
                q[j] = (uint32_t)(int32_t)rint(127.0 * p / peak);
            }
        }
        if (!BPQ4K_CHECK(e + E <= a.K && row < a.M, a.status)) continue;
        if constexpr (E == 1) {
            codes[e] = (int8_t)(q[0] & 0xFFu);
        } else {
#pragma unroll
            for (int j = 0; j < E; j += 4) {
                const uint32_t word = __byte_perm(__byte_perm(q[j], q[j + 1], 0x0040), __byte_perm(q[j + 2], q[j + 3], 0x0040), 0x5410);
                q[j / 4] = word;
            }
            if constexpr (E == 4)
                *reinterpret_cast<uint32_t*>(codes + e) = q[0];
            else
                *reinterpret_cast<uint2*>(codes + e) = make_uint2(q[0], q[1]);
        }
    }
}

template <typename T, int E, int PT>
cudaError_t launch_pt(const RowsI8Args& a, cudaStream_t stream) {
    const uint32_t units = (a.K + PT - 1u) / PT, threads = (units + 31u) & ~31u;
    if (a.w && a.R)
        rows_i8_kernel<T, E, PT, true, true><<<a.M, threads, 0, stream>>>(a);
    else if (a.w)
        rows_i8_kernel<T, E, PT, true, false><<<a.M, threads, 0, stream>>>(a);
    else
        rows_i8_kernel<T, E, PT, false, false><<<a.M, threads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const RowsI8Args& a, cudaStream_t stream) {
    constexpr int E = 16 / sizeof(T);
    auto off = [](const void* p, uint32_t ld) { return p && ((reinterpret_cast<uintptr_t>(p) & 15u) || (uint64_t)ld * sizeof(T) % 16u); };
    const bool single = a.K % E || off(a.X, a.ldx) || off(a.R, a.ldr) || off(a.sum, a.lds) || (reinterpret_cast<uintptr_t>(a.w) & 15u);
    if (single) return a.K <= 8192u ? launch_pt<T, 1, 8>(a, stream) : launch_pt<T, 1, 32>(a, stream);
    return a.K <= 8192u ? launch_pt<T, E, 8>(a, stream) : launch_pt<T, E, 32>(a, stream);
}

}  // namespace

cudaError_t launch_rows_i8(const RowsI8Args& a, int ftype, cudaStream_t stream) {
    if (a.M == 0) return cudaSuccess;
    if (a.K == 0 || a.K > kRowsI8MaxK || (a.R && !a.w)) return cudaErrorInvalidValue;
    switch (ftype) {
        case 0: return launch_type<float>(a, stream);
        case 1: return launch_type<__half>(a, stream);
        case 30: return launch_type<__nv_bfloat16>(a, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace bpq4k
