// Matrix product of 8-bit rows with 8-bit weights: Y[m][n] = (sum_k x[m][k] * w[n][k]) * xs[m] * ws[n] + bias[n].
//
// The sum is an exact 32-bit integer (K <= 131071), so no order of it changes a bit of the result.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "q4k_common.cuh"

namespace bpq4k {

namespace {

template <typename T>
__device__ __forceinline__ T to_elem(float v);
template <>
__device__ __forceinline__ float to_elem<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half to_elem<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 to_elem<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 codes from byte k of a row on, zeros from byte K on (the bytes behind a row's codes may be anything).
__device__ __forceinline__ int4 codes16(const int8_t* row, uint32_t k, uint32_t K) {
    int4 v = __ldg(reinterpret_cast<const int4*>(row + k));
    if (k + 16u > K) {
        const uint32_t n = K - k;  // 1..15 codes
        auto keep = [n](int w, uint32_t first) { return n >= first + 4u ? w : n <= first ? 0 : w & (int)((1u << (8u * (n - first))) - 1u); };
        v.x = keep(v.x, 0), v.y = keep(v.y, 4), v.z = keep(v.z, 8), v.w = keep(v.w, 12);
    }
    return v;
}

// One warp per weight row, MT activation rows at a time.
template <typename T, int MT>
__global__ void __launch_bounds__(256) matmul_i8_dot_kernel(const __grid_constant__ MatmulI8Args a) {
    const uint32_t n = blockIdx.x * 8u + (threadIdx.x >> 5), lane = threadIdx.x & 31u, m0 = blockIdx.y * MT;
    if (n >= a.N) return;
    const int8_t* w = a.W + (uint64_t)n * a.ldw;
    int acc[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) acc[i] = 0;
    for (uint32_t k = lane * 16u; k < a.K; k += 512u) {
        const int4 wv = codes16(w, k, a.K);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            if (m0 + i >= a.M) break;
            const int4 xv = codes16(a.X + (uint64_t)(m0 + i) * a.ldx, k, a.K);
            acc[i] = __dp4a(xv.x, wv.x, __dp4a(xv.y, wv.y, __dp4a(xv.z, wv.z, __dp4a(xv.w, wv.w, acc[i]))));
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int s = __reduce_add_sync(0xFFFFFFFFu, acc[i]);
        if (lane == (uint32_t)i && m0 + i < a.M) {
            float y = (float)s * a.xs[m0 + i] * a.ws[n];
            if (a.bias) y += a.bias[n];
            static_cast<T*>(a.Y)[(uint64_t)(m0 + i) * a.ldy + n] = to_elem<T>(y);
        }
    }
}

template <typename T>
cudaError_t launch_type(const MatmulI8Args& a, cudaStream_t stream) {
    matmul_i8_dot_kernel<T, 8><<<dim3((a.N + 7u) / 8u, (a.M + 7u) / 8u), 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_matmul_i8(const MatmulI8Args& a, int ftype, int* status_dev, int sm_count, cudaStream_t stream, int* launches) {
    (void)status_dev, (void)sm_count;
    if (a.M == 0 || a.N == 0) return cudaSuccess;
    ++*launches;
    switch (ftype) {
        case 0: return launch_type<float>(a, stream);
        case 1: return launch_type<__half>(a, stream);
        case 30: return launch_type<__nv_bfloat16>(a, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace bpq4k
