// Rows to 8 bits: residual addition, root-mean-square norm and symmetric quantisation with one scale per row, one pass.
//
// For a row of K values (all in float; x, r and the sum may be stored in 16 bits)
//   v = x + r,   p = v * w,   a = max |p|,   rstd = 1 / sqrt(mean(v^2) + eps)
//   code = round_half_even(127 p / a),   scale = a * rstd / 127
// rstd is a factor of the whole row and of its largest value, so the codes do not depend on it: they are computed from the
// exact quotient and never differ with the order of a sum.  In float the quotient is off by at most 127 * 3 * 2^-24 = 2.3e-5
// (the product, a and 127/a are rounded; the quotient's distance from its code is not, it is a multiply-add).  Where one lies
// nearer than 3e-5 to the middle between two codes, its code is computed again in double, from the exact product (48 bits) and
// the exact a.
// Values of 16 bits without a norm need none of that, and have what costs it most: where a/2 is among them, 63.5 is exact.  With
// p = m 2^-t and a = n (whole mantissas of at most 11 bits), a quotient is a border or at least 2^-12 2^-t away from one, and a float's
// error is below 254 * 2^-23 * 2^-t: only exact borders can go wrong, 254 m = (2k+1) n 2^t.  127 divides 2k+1 or n.  If not n, k = 63,
// and 127/a rounded up makes that 64 (the even code), so a multiply-add is all there is to a code.  If n, as above (one row in 64).
// Almost half of the warps' instructions went into borders before (2048 x 14336 bfloat16 31.3 us, now 20.9).
//
// Memory bound (13 bytes a value with a float residual stream).  A row's values stay in registers between the two halves
// (statistics, codes), one CTA to a row, several rows to an SM, so that one row's loads overlap another's arithmetic; that runs on
// pairs (.f32x2).  2048 x 8192 float with a residual: 35 us, 0.95 of the copy rate.  With 16-bit streams (bfloat16 27 us, 0.67)
// neither DRAM (55 % in the profile) nor the issue slots (50 %, 24 instructions a value) are full: warps wait for loads and at the
// barrier between the halves, with too few rows on an SM to cover it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "kernels.h"
#include "q4k_common.cuh"

namespace bpq4k {

namespace {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

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
// E floats, rounded to the element type (two at a time: a single conversion to 16 bits has a sixteenth of the rate).
template <typename T, int E>
__device__ __forceinline__ void store_pack(T* p, const float* v) {
    if constexpr (sizeof(T) == 4 && E == 1) {
        *p = v[0];
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        T2 w[(E + 1) / 2];
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            const float second = E == 1 ? 0.f : v[j + (E > 1)];
            if constexpr (std::is_same<T, __half>::value)
                w[j / 2] = __floats2half2_rn(v[j], second);
            else
                w[j / 2] = __floats2bfloat162_rn(v[j], second);
        }
        if constexpr (E == 1)
            *p = w[0].x;
        else
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
    }
}

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN if either is one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float kNear = 0.5f - 3e-5f;  // a quotient further from its code than this may belong to the next one

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: added to a quotient, it leaves the rounded quotient in the low byte

// The code of 127 p / peak, which lies in [k, k + 1): on which side of k + 1/2 it is.  Single values have 24 bits, and a double holds
// both sides of the comparison.  Products of two (PRODUCTS) have 48, so the sides can have 56 and are rounded: they compare like the
// exact ones unless they round to the same double, and then their rests, which a multiply-add gives exactly, decide.
template <bool PRODUCTS>
__device__ __forceinline__ uint32_t exact_code(double p, double peak, int k) {
    const double n = 2 * k + 1;
    double l = 254.0 * p, r = n * peak;
    if (PRODUCTS && l == r) l = fma(254.0, p, -l), r = fma(n, peak, -r);
    return (uint32_t)(l < r || (l == r && (k & 1) == 0) ? k : k + 1);
}

template <int E>
__device__ __forceinline__ void store_codes(int8_t* at, const uint32_t (&q)[E]) {
    if constexpr (E == 1) {
        *at = (int8_t)(q[0] & 0xFFu);
    } else {
        uint32_t w[E / 4];
#pragma unroll
        for (int j = 0; j < E; j += 4)
            w[j / 4] = __byte_perm(__byte_perm(q[j], q[j + 1], 0x0040), __byte_perm(q[j + 2], q[j + 3], 0x0040), 0x5410);
        if constexpr (E == 4)
            *reinterpret_cast<uint32_t*>(at) = w[0];
        else
            *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
    }
}

// Two floats in a register pair.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// A warp takes 32 * PT neighbouring values of the row, a lane PT / E accesses 32 * E apart, so that all offsets are constants.
// Values stay as they were loaded, or (RES) as their sums in float; behind the row they are zeros.
// Without a norm, 32 registers a thread, for twice the warps (2048 x 8192 float 14.8 us, 512 x 14336 bfloat16 8.1, with up to 64
// 10.1; not for 32 floats in accesses of 16 bytes, which spill: 512 x 28672 float 23.4, with 64 17.5).  With one there is no gain
// in fewer (2048 x 8192 float with a residual 40.6 us with 40, 34.9 with 64).
template <typename T, int E, int PT, bool NORM, bool RES>
__global__ void __launch_bounds__(1024, NORM || (PT == 32 && E == 4) ? 1 : 2) rows_i8_kernel(const __grid_constant__ RowsI8Args a) {
    constexpr int NV = PT / E, G = E == 1 ? 2 : E;  // G: values of a group, which the arithmetic takes in pairs
    const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, warps = blockDim.x >> 5;
    const uint32_t e0 = warp * (32u * PT) + lane * E;
    const T* x = static_cast<const T*>(a.X) + (uint64_t)row * a.ldx + e0;
    const T* r = RES ? static_cast<const T*>(a.R) + (uint64_t)row * a.ldr + e0 : nullptr;
    T* sum = RES && a.sum ? static_cast<T*>(a.sum) + (uint64_t)row * a.lds + e0 : nullptr;
    int8_t* codes = a.codes + (uint64_t)row * a.ldc + e0;
    const float* wp = a.w + e0;
    auto in = [&](int i) { return e0 + (uint32_t)i * (32u * E) < a.K; };
    auto weights = [&](int g, float (&w)[G]) {  // of group g
        if constexpr (E == 1) {
            w[0] = in(2 * g) ? __ldg(wp + 64 * g) : 0.f;
            w[1] = in(2 * g + 1) ? __ldg(wp + 64 * g + 32) : 0.f;
        } else {
#pragma unroll
            for (int j = 0; j < E; j += 4) {
                const float4 t = in(g) ? __ldg(reinterpret_cast<const float4*>(wp + 32 * E * g + j)) : make_float4(0.f, 0.f, 0.f, 0.f);
                w[j] = t.x, w[j + 1] = t.y, w[j + 2] = t.z, w[j + 3] = t.w;
            }
        }
    };

    Pack<T, E> xv[NV] = {};
    float v[RES ? PT : 1] = {};
    // Products stay too where a value has two accesses of weights at half their rate (a lane's are 32 bytes apart): these are fetched
    // once, not twice (512 x 8192 bfloat16 8.0 -> 7.3 us, 2048 x 8192 bfloat16 R 27.2 -> 26.8; with single accesses or for floats,
    // which spill, nothing: 301 x 5001 half 5.3 -> 5.7).
    constexpr bool kKeep = NORM && PT <= 16 && E == 8;
    float product[kKeep ? PT : 1];
    auto value = [&](int t) { return RES ? v[RES ? t : 0] : to_float(xv[t / E].v[t % E]); };
    float hi = 0.f;          // (an infinity or a NaN reaches hi)
    uint64_t ss2 = 0ull;
    {
        Pack<T, E> rv[RES ? NV : 1] = {};
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (in(i)) xv[i] = load_pack<T, E>(x + 32 * E * i);
        if constexpr (RES) {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (in(i)) rv[i] = load_pack<T, E>(r + 32 * E * i);
        }
#pragma unroll
        for (int g = 0; g < PT / G; g++) {
            float w[G];
            if constexpr (NORM) weights(g, w);
#pragma unroll
            for (int j = 0; j < G; j += 2) {
                const int t = g * G + j;
                uint64_t s = pair(to_float(xv[t / E].v[t % E]), to_float(xv[(t + 1) / E].v[(t + 1) % E]));
                if constexpr (RES) {
                    s = add2(s, pair(to_float(rv[t / E].v[t % E]), to_float(rv[(t + 1) / E].v[(t + 1) % E])));
                    v[t] = halves(s).x, v[t + 1] = halves(s).y;
                }
                if constexpr (NORM) ss2 = fma2(s, s, ss2);
                const float2 p = halves(NORM ? mul2(s, pair(w[j], w[j + 1])) : s);
                if constexpr (kKeep) product[t] = p.x, product[t + 1] = p.y;
                hi = max_nan(max_nan(hi, fabsf(p.x)), fabsf(p.y));
            }
        }
        if constexpr (RES) {
            if (sum) {
#pragma unroll
                for (int i = 0; i < NV; i++)
                    if (in(i) && BPQ4K_CHECK(e0 + 32u * E * i + E <= a.K, a.status)) store_pack<T, E>(sum + 32 * E * i, v + i * E);
            }
        }
    }
    float ss = halves(ss2).x + halves(ss2).y;

    __shared__ uint32_t s_hi[32];
    __shared__ float s_ss[32];
    __shared__ double s_sq[32], s_peak[32];
    __shared__ unsigned long long s_exact;  // the exact a, as the bits of a double (positive ones order like whole numbers)
    const uint32_t mine = __float_as_uint(hi);
    const uint32_t warp_hi = __reduce_max_sync(0xFFFFFFFFu, mine);
    if constexpr (NORM) {
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    }
    if (lane == 0) s_hi[warp] = warp_hi, s_ss[warp] = ss;
    if (tid == 0) s_exact = 0ull;
    __syncthreads();
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? s_hi[lane] : 0u);
    const float peak = __uint_as_float(top);
    const bool bad = !(peak < __uint_as_float(0x7F800000u)), tiny = peak < 1e-30f;  // (tiny: products and 127 / a leave the float range)
    double largest = (double)peak, sq = 0.0;
    if constexpr (NORM) {
        ss = lane < warps ? s_ss[lane] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        sq = ss;
        // squares or products beyond what a float holds well (every thread sees the same, so all or none come here)
        if (!(ss > 1e-20f && ss < 1e30f) || tiny) {
            sq = 0.0;
            double big = 0.0;
#pragma unroll
            for (int g = 0; g < PT / G; g++) {
                float w[G];
                weights(g, w);
#pragma unroll
                for (int j = 0; j < G; j++) {
                    const double s = (double)value(g * G + j);
                    sq += s * s;
                    big = fmax(big, fabs(s * (double)w[j]));
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                sq += __shfl_xor_sync(0xFFFFFFFFu, sq, o);
                big = fmax(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
            }
            if (lane == 0) s_sq[warp] = sq, s_peak[warp] = big;
            __syncthreads();
            sq = lane < warps ? s_sq[lane] : 0.0;
            largest = lane < warps ? s_peak[lane] : 0.0;
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                sq += __shfl_xor_sync(0xFFFFFFFFu, sq, o);
                largest = fmax(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, o));
            }
        }
    }
    const bool zero = bad || largest == 0.0;
    if (tid == 0) {
        const double rstd = NORM ? rsqrt(sq / (double)a.K + (double)a.eps) : 1.0;
        a.scales[row] = bad ? __uint_as_float(0x7FC00000u) : zero ? 0.f : (float)(largest * rstd / 127.0);
    }
    if (zero) {  // (a whole row)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const uint32_t none[E] = {};
            if (in(i) && BPQ4K_CHECK(e0 + 32u * E * i + E <= a.K, a.status)) store_codes<E>(codes + 32 * E * i, none);
        }
        return;
    }

    if constexpr (!NORM) {
        constexpr bool kShort = sizeof(T) == 2;  // (with 127 no divisor of the mantissa of a)
        bool exactly = tiny || (kShort && ((top & 0x7FFFFFu) | 0x800000u) % 127u == 0u);
        if (!exactly) {
            const float inv = kShort ? __fdiv_ru(127.f, peak) : 127.f / peak;
            float far = 0.f;  // the largest distance of a quotient from its code
#pragma unroll
            for (int i = 0; i < NV; i++) {
                uint32_t q[E];
#pragma unroll
                for (int j = 0; j < E; j++) {
                    const float p = value(i * E + j), c = fmaf(p, inv, kMagic);
                    q[j] = __float_as_uint(c);
                    if (!kShort) far = fmaxf(far, fabsf(fmaf(p, inv, kMagic - c)));
                }
                if (in(i) && BPQ4K_CHECK(e0 + 32u * E * i + E <= a.K && row < a.M, a.status)) store_codes<E>(codes + 32 * E * i, q);
            }
            exactly = far > kNear;
        }
        if (exactly) {
            const double by = 127.0 / (double)peak;
#pragma unroll 1  // (and read again: the values need no registers up to here)
            for (int i = 0; i < NV; i++) {
                if (!in(i)) continue;
                const Pack<T, E> again = load_pack<T, E>(x + 32 * E * i);
                uint32_t q[E];
#pragma unroll
                for (int j = 0; j < E; j++) {
                    const double p = to_float(again.v[j]);
                    q[j] = exact_code<false>(p, (double)peak, (int)floor(p * by));
                }
                if (BPQ4K_CHECK(e0 + 32u * E * i + E <= a.K && row < a.M, a.status)) store_codes<E>(codes + 32 * E * i, q);
            }
        }
        return;
    }

    // one product, or a few that round to the same float, is the largest: whoever holds it knows a exactly
    if (mine == top || tiny) {
        double big = 0.0;
#pragma unroll
        for (int g = 0; g < PT / G; g++) {
            float w[G];
            weights(g, w);
#pragma unroll
            for (int j = 0; j < G; j++) big = fmax(big, fabs((double)value(g * G + j) * (double)w[j]));
        }
        atomicMax(&s_exact, (unsigned long long)__double_as_longlong(big));
    }
    const float inv = tiny ? 0.f : 127.f / peak;
    const uint64_t inv2 = pair(inv, inv), magic2 = pair(kMagic, kMagic), minus2 = pair(-1.f, -1.f);
    float far = tiny ? 1.f : 0.f;  // the largest distance of a quotient from its code
#pragma unroll
    for (int g = 0; g < PT / G; g++) {
        float w[G];
        if constexpr (!kKeep) weights(g, w);
        uint32_t q[G];
#pragma unroll
        for (int j = 0; j < G; j += 2) {
            const int t = g * G + j;
            const uint64_t p = kKeep ? pair(product[kKeep ? t : 0], product[kKeep ? t + 1 : 0]) : mul2(pair(value(t), value(t + 1)), pair(w[j], w[j + 1]));
            const uint64_t c = fma2(p, inv2, magic2);
            const float2 f = halves(c), d = halves(fma2(p, inv2, fma2(c, minus2, magic2)));
            q[j] = __float_as_uint(f.x), q[j + 1] = __float_as_uint(f.y);
            far = fmaxf(fmaxf(far, fabsf(d.x)), fabsf(d.y));
        }
#pragma unroll
        for (int l = 0; l < G / E; l++) {
            const int i = g * (G / E) + l;
            if (in(i) && BPQ4K_CHECK(e0 + 32u * E * i + E <= a.K && row < a.M, a.status))
                store_codes<E>(codes + 32 * E * i, reinterpret_cast<const uint32_t(&)[E]>(q[l * E]));
        }
    }
    __syncthreads();
    if (far > kNear) {
        const double exact = __longlong_as_double((long long)s_exact), by = tiny ? 127.0 / exact : 0.0;
#pragma unroll
        for (int g = 0; g < PT / G; g++) {
            float w[G];
            weights(g, w);
            uint32_t q[G];
#pragma unroll
            for (int j = 0; j < G; j++) {
                const float s = value(g * G + j), p = s * w[j], c = fmaf(p, inv, kMagic), d = fmaf(p, inv, -(c - kMagic));
                q[j] = __float_as_uint(c);
                if (tiny || fabsf(d) > kNear) {
                    const double pp = (double)s * (double)w[j];
                    q[j] = exact_code<true>(pp, exact, tiny ? (int)floor(pp * by) : __float2int_rn(c - kMagic) - (d < 0.f ? 1 : 0));
                }
            }
#pragma unroll
            for (int l = 0; l < G / E; l++) {
                const int i = g * (G / E) + l;
                if (in(i) && BPQ4K_CHECK(e0 + 32u * E * i + E <= a.K && row < a.M, a.status))
                    store_codes<E>(codes + 32 * E * i, reinterpret_cast<const uint32_t(&)[E]>(q[l * E]));
            }
        }
    }
}

template <typename T, int E, int PT>
cudaError_t launch_pt(const RowsI8Args& a, cudaStream_t stream) {
    const uint32_t warps = (a.K + 32u * PT - 1u) / (32u * PT);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.M);
    cfg.blockDim = dim3(warps * 32u);
    cfg.stream = stream;
    if (a.w && a.R) return cudaLaunchKernelEx(&cfg, rows_i8_kernel<T, E, PT, true, true>, a);
    if (a.w) return cudaLaunchKernelEx(&cfg, rows_i8_kernel<T, E, PT, true, false>, a);
    return cudaLaunchKernelEx(&cfg, rows_i8_kernel<T, E, PT, false, false>, a);
}

// Values of a thread (us on B200; R: with a residual, Q: no norm).  8: the shortest way through a row, for rows that have an SM each
// (1 x 4096 float R 3.0, with 16 3.4; Q 1.8, 2.0) and short rows (2048 x 768 float R 5.8, 7.2; 2048 x 1025 bfloat16 R, single
// accesses, 8.1, 9.6; 4096 x 1024 float Q 5.3, 6.1).  16 for the others: most loads in flight with the warps to hide them (2048 x 8192
// float R 34.9, with 8 45.4, with 32 39.9; bfloat16 R 27.3, 37.7, 26.5; 700 x 8192 bfloat16 R 11.8, 13.9, 12.9; 2048 x 14336 float Q
// 26.7, with 32 38.0; 2048 x 5001 half R, single accesses, 22.8, with 32 37.9).  32 where 1024 threads need them.
template <typename T, int E>
cudaError_t launch_vec(const RowsI8Args& a, int sm_count, cudaStream_t stream) {
    const uint32_t sms = (uint32_t)sm_count;
    if (a.K <= 8192u && (a.M <= sms || a.K <= (E == 1 ? 2048u : 1024u))) return launch_pt<T, E, 8>(a, stream);
    if (a.K <= 16384u) return launch_pt<T, E, 16>(a, stream);
    return launch_pt<T, E, 32>(a, stream);
}

template <typename T>
cudaError_t launch_type(const RowsI8Args& a, int sm_count, cudaStream_t stream) {
    constexpr int E = 16 / sizeof(T);
    auto off = [](const void* p, uint32_t ld) { return p && ((reinterpret_cast<uintptr_t>(p) & 15u) || (uint64_t)ld * sizeof(T) % 16u); };
    const bool single = a.K % E || off(a.X, a.ldx) || off(a.R, a.ldr) || off(a.sum, a.lds) || (reinterpret_cast<uintptr_t>(a.w) & 15u);
    return single ? launch_vec<T, 1>(a, sm_count, stream) : launch_vec<T, E>(a, sm_count, stream);
}

}  // namespace

cudaError_t launch_rows_i8(const RowsI8Args& a, int ftype, int sm_count, cudaStream_t stream) {
    if (a.M == 0) return cudaSuccess;
    if (a.K == 0 || a.K > kRowsI8MaxK || (a.R && !a.w)) return cudaErrorInvalidValue;
    switch (ftype) {
        case 0: return launch_type<float>(a, sm_count, stream);
        case 1: return launch_type<__half>(a, sm_count, stream);
        case 30: return launch_type<__nv_bfloat16>(a, sm_count, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace bpq4k
