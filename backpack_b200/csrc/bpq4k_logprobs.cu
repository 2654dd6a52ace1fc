// What a row of logits says: log probabilities of given tokens, the entropy, the most likely tokens.  One pass over the row.
//
//   m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m):   log p(i) = x_i - m - ln S,   H = ln S - T / S
//
// S and T are kept relative to a running maximum and rescaled when it grows (T' = (T + S d) e^d, S' = S e^d with
// d = old - new maximum).  Both terms of H are at least zero, so nothing cancels.
//
// The most likely tokens: every warp keeps the best 32 of what it has seen, sorted over its lanes, as 64-bit keys (the value
// in the order of unsigned words, below it the inverted index: the larger key is the larger value or, among equal values, the
// lower index).  A value that is not larger than the warp's k-th best is passed over after one comparison: later values have
// higher indexes, so an equal one loses.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "q4k_common.cuh"

namespace bpq4k {

namespace {

constexpr uint32_t kFull = 0xFFFFFFFFu;
constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kThreads = 512, kWarps = kThreads / 32u;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

union Pack16 {
    uint4 q;
    uint16_t h[8];
    float f[4];
};

struct Stats {
    float m, s, t;
    // (x - m) of a maximum that is still -infinity is taken from 0
    __device__ __forceinline__ float ref() const { return m == -kInf ? 0.f : m; }
    __device__ __forceinline__ void add(const Stats& o) {
        const float n = fmaxf(m, o.m);
        // (-infinity less -infinity is a NaN, and fmaxf drops it; e^-200 is 0 as a float)
        const float d = fmaxf(m - n, -200.f), od = fmaxf(o.m - n, -200.f);
        const float f = exp2_fast(d * kLog2e), of = exp2_fast(od * kLog2e);
        t = f * fmaf(s, d, t) + of * fmaf(o.s, od, o.t);
        s = s * f + o.s * of;
        m = n;
    }
    __device__ __forceinline__ void add_lanes() {  // over the warp; the result is lane 0's
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const Stats other{__shfl_down_sync(kFull, m, o), __shfl_down_sync(kFull, s, o), __shfl_down_sync(kFull, t, o)};
            add(other);
        }
        m = __shfl_sync(kFull, m, 0), s = __shfl_sync(kFull, s, 0), t = __shfl_sync(kFull, t, 0);
    }
};

__device__ __forceinline__ unsigned long long make_key(float v, uint32_t idx) {
    const uint32_t b = __float_as_uint(v + 0.f);  // (-0 and +0 are equal)
    return ((unsigned long long)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long k) { return ~(uint32_t)k; }

// Keys of a warp in descending order over its lanes.
__device__ __forceinline__ unsigned long long sort_warp(unsigned long long k, uint32_t lane) {
#pragma unroll
    for (uint32_t size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (uint32_t step = size >> 1; step; step >>= 1) {
            const unsigned long long o = __shfl_xor_sync(kFull, k, step);
            const bool larger = ((lane & step) == 0u) == ((lane & size) == 0u || size == 32u);
            k = (k > o) == larger ? k : o;
        }
    return k;
}
// The best 32 of two descending lists of 32, descending.
__device__ __forceinline__ unsigned long long merge_warp(unsigned long long a, unsigned long long b, uint32_t lane) {
    const unsigned long long r = __shfl_sync(kFull, b, 31u - lane);
    unsigned long long k = a > r ? a : r;
#pragma unroll
    for (uint32_t step = 16; step; step >>= 1) {
        const unsigned long long o = __shfl_xor_sync(kFull, k, step);
        k = (k > o) == ((lane & step) == 0u) ? k : o;
    }
    return k;
}

// The best 32 keys of a warp's values, and the k-th of them.  Key 0 stands for none.
struct TopList {
    unsigned long long mine = 0ull;  // lane i: the i-th best
    unsigned long long least = 0ull;
    float bar = -kInf;       // value of `least`
    bool open = true;                // fewer than k so far: every value is taken

    __device__ __forceinline__ void update(uint32_t k) {
        least = __shfl_sync(kFull, mine, k - 1u);
        open = least == 0ull;
        bar = key_value(least);
    }
    __device__ __forceinline__ void insert(unsigned long long key, uint32_t k, uint32_t lane) {
        const uint32_t pos = __popc(__ballot_sync(kFull, mine > key));
        const unsigned long long up = __shfl_up_sync(kFull, mine, 1);
        if (lane >= pos) mine = lane == pos ? key : up;
        least = __shfl_sync(kFull, mine, k - 1u);
    }
    // Values of a lane: v[j] has the index first + j / E * gap + j % E.  The whole warp comes here.
    template <int N, int E>
    __device__ __forceinline__ void take(const float (&v)[N], uint32_t valid, uint32_t first, uint32_t gap, uint32_t k, uint32_t lane) {
        uint32_t left = valid;
        if (open) {  // the lanes' own best first: sorted at once, they bar nearly everything else
            unsigned long long best = 0ull;
            int at = 0;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const unsigned long long key = (valid >> j) & 1u ? make_key(v[j], first + (uint32_t)(j / E) * gap + (uint32_t)(j % E)) : 0ull;
                if (key > best) best = key, at = j;
            }
            if (best) left &= ~(1u << at);
            mine = merge_warp(mine, sort_warp(best, lane), lane);
            least = __shfl_sync(kFull, mine, k - 1u);
        }
#pragma unroll
        for (int j = 0; j < N; j++) {
            const unsigned long long key = (left >> j) & 1u ? make_key(v[j], first + (uint32_t)(j / E) * gap + (uint32_t)(j % E)) : 0ull;
            uint32_t who = __ballot_sync(kFull, key > least);
            while (who) {
                const uint32_t src = __ffs(who) - 1u;
                const unsigned long long c = __shfl_sync(kFull, key, src);
                if (c > least) insert(c, k, lane);
                who &= who - 1u;
            }
        }
        update(k);
    }
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const __grid_constant__ LogprobsArgs a) {
    constexpr int E = 16 / sizeof(T), U = 16 / E, N = U * E;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const T* x = static_cast<const T*>(a.logits) + (uint64_t)row * a.ld;
    // whole 16-byte accesses between the first and the last boundary inside the row; what lies outside comes one by one
    const uint32_t head = min(a.V, (uint32_t)((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (uint32_t)sizeof(T));
    const uint32_t nv = (a.V - head) / E, tail = head + nv * E;

    Stats st{-kInf, 0.f, 0.f};
    TopList top;
    auto take = [&](const float(&v)[N], uint32_t valid, uint32_t first, uint32_t gap) {
        float mx = v[0];
#pragma unroll
        for (int j = 1; j < N; j++) mx = fmaxf(mx, v[j]);
        if (mx > st.m) {
            const float n = mx, d = fmaxf(st.ref() - n, -200.f), f = exp2_fast(d * kLog2e);
            // (a sum that has nothing yet has no reference)
            st.t = st.s == 0.f ? 0.f : f * fmaf(st.s, d, st.t);
            st.s = st.s == 0.f ? 0.f : st.s * f;
            st.m = n;
        }
        const float ref = st.ref();
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float u = v[j] - ref, e = exp2_fast(u * kLog2e);
            st.s += e;
            st.t = fmaf(e, fmaxf(u, -200.f), st.t);
        }
        if constexpr (TOP) {
            if (__any_sync(kFull, top.open ? valid != 0u : mx > top.bar)) top.take<N, E>(v, valid, first, gap, a.nTop, lane);
        }
    };
    auto single = [&](uint32_t first, uint32_t last) {  // at most E - 1 values, one to a lane
        float v[N];
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = -kInf;
        const uint32_t i = first + lane;
        if (i < last) v[0] = to_float(x[i]);
        take(v, i < last ? 1u : 0u, i, 0u);
    };
    if (warp == 0 && head) single(0u, head);
    for (uint32_t b = warp * 32u; b < nv; b += kThreads * U) {
        Pack16 p[U];
        float v[N];
        uint32_t valid = 0u;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = b + lane + (uint32_t)u * kThreads;
            if (i < nv) p[u].q = __ldg(reinterpret_cast<const uint4*>(x + head) + i), valid |= ((1u << E) - 1u) << (u * E);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < E; j++)
                v[u * E + j] = (valid >> (u * E)) & 1u ? to_float(reinterpret_cast<const T*>(&p[u])[j]) : -kInf;
        take(v, valid, head + (b + lane) * E, kThreads * E);
    }

    if (warp == 0 && tail < a.V) single(tail, a.V);

    __shared__ unsigned long long s_keys[kWarps][32];
    __shared__ float s_m[kWarps], s_s[kWarps], s_t[kWarps];
    st.add_lanes();
    if (lane == 0) s_m[warp] = st.m, s_s[warp] = st.s, s_t[warp] = st.t;
    if constexpr (TOP) s_keys[warp][lane] = top.mine;
    __syncthreads();
    if (warp) return;
    st = lane < kWarps ? Stats{s_m[lane], s_s[lane], s_t[lane]} : Stats{-kInf, 0.f, 0.f};
    st.add_lanes();
    const bool none = st.m == -kInf && st.s == 0.f;  // the row's mask leaves nothing
    const bool bad = !(st.s == st.s);                        // a NaN or +infinity
    const float ln_s = logf(st.s);
    auto logp = [&](float v) { return bad ? __uint_as_float(0x7FC00000u) : none || v == -kInf ? -kInf : (float)((double)v - (double)st.m - (double)ln_s); };
    if (a.entropy && lane == 0) a.entropy[row] = bad ? __uint_as_float(0x7FC00000u) : none ? 0.f : ln_s - st.t / st.s;
    for (uint32_t g = lane; g < a.nGiven; g += 32u) {
        const int32_t id = a.given[(uint64_t)row * a.nGiven + g];
        a.given_lp[(uint64_t)row * a.nGiven + g] = id < 0 || (uint32_t)id >= a.V ? __uint_as_float(0x7FC00000u) : logp(to_float(x[id]));
    }
    if constexpr (TOP) {
        unsigned long long k = s_keys[0][lane];
        for (uint32_t w = 1; w < kWarps; w++) k = merge_warp(k, s_keys[w][lane], lane);
        if (lane < a.nTop) {
            a.top_ids[(uint64_t)row * a.nTop + lane] = bad ? -1 : (int32_t)key_index(k);
            a.top_lp[(uint64_t)row * a.nTop + lane] = logp(key_value(k));
        }
    }
}

template <typename T>
cudaError_t launch_type(const LogprobsArgs& a, cudaStream_t stream) {
    if (a.nTop)
        logprobs_kernel<T, true><<<a.M, kThreads, 0, stream>>>(a);
    else
        logprobs_kernel<T, false><<<a.M, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs& a, int ftype, cudaStream_t stream) {
    if (a.M == 0) return cudaSuccess;
    switch (ftype) {
        case 0: return launch_type<float>(a, stream);
        case 1: return launch_type<__half>(a, stream);
        case 30: return launch_type<__nv_bfloat16>(a, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace bpq4k
