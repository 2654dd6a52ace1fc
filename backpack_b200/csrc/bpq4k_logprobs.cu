// What a row of logits says: log probabilities of given tokens, the entropy, the most likely tokens.  One pass over the row.
//
//   m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m):   log p(i) = x_i - m - ln S,   H = ln S - T / S
//
// S and T are kept by every thread relative to its own running maximum and rescaled when that grows.  The difference to the
// maximum is taken before anything else, so logits of any magnitude are sound and the largest has the weight 1 exactly; the
// arithmetic is on pairs (add, mul and fma .f32x2: half an instruction a value each).  Both terms of H are at least zero, so
// nothing cancels.
//
// The most likely tokens cost the pass nothing.  Values are compared as 64-bit keys (the value in the order of unsigned words,
// below it the inverted index: the larger key is the larger value or, among equal ones, the lower index; no two are equal).
// Every thread knows its largest value; of the keys of these, the k-th largest bounds the k-th largest of all from below, and
// only the k threads at or above it can hold a larger one.  Their shares are read once more (k of 512 threads' values, from L2).
//
// Few rows: CTAs of a cluster share a row, so that no working memory is needed; the first of them gathers.
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
constexpr uint32_t kMaxGroup = 8;  // CTAs that share a row: the largest cluster that every device takes

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN if either is one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
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

// Maximum, S and T of some values, T in units of ln 2.
struct Stats {
    float m, s, t;
    __device__ __forceinline__ void add(const Stats& o) {
        const float n = max_nan(m, o.m);
        // (-infinity less -infinity is a NaN, and fmaxf drops it; 2^-300 is 0 as a float)
        const float d = fmaxf((m - n) * kLog2e, -300.f), od = fmaxf((o.m - n) * kLog2e, -300.f);
        const float f = exp2_fast(d), of = exp2_fast(od);
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

// The value at this place of the first CTA of the cluster.
template <typename V>
__device__ __forceinline__ void store_cluster(V* at, const V& v) {
    static_assert(sizeof(V) % 4 == 0, "words");
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(at)));
    uint32_t w[sizeof(V) / 4];
    memcpy(w, &v, sizeof(V));
#pragma unroll
    for (uint32_t i = 0; i < sizeof(V) / 4; i++) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 4u * i), "r"(w[i]) : "memory");
}

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

// The best 32 of the lists of all warps, in every warp's `list`.  keys: 32 per warp; the whole CTA comes here.
__device__ __forceinline__ unsigned long long merge_cta(unsigned long long list, unsigned long long (*keys)[32], uint32_t warp, uint32_t lane) {
    keys[warp][lane] = list;
#pragma unroll
    for (uint32_t step = kWarps / 2u; step; step >>= 1) {
        __syncthreads();
        if (warp < step) keys[warp][lane] = list = merge_warp(list, keys[warp + step][lane], lane);
    }
    __syncthreads();
    return keys[0][lane];
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 2) logprobs_kernel(const __grid_constant__ LogprobsArgs a, const uint32_t group) {
    constexpr uint32_t E = 16 / sizeof(T), U = 16 / E, N = U * E;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    uint32_t rank = 0;
    if (group > 1u) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for before anything crosses over)
    }
    const uint32_t row = blockIdx.x / group;
    const T* x = static_cast<const T*>(a.logits) + (uint64_t)row * a.ld;
    // whole 16-byte accesses between the first and the last boundary inside the row; what lies outside comes one by one
    const uint32_t head = min(a.V, (uint32_t)((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (uint32_t)sizeof(T));
    const uint32_t nv = (a.V - head) / E, tail = head + nv * E;
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    const uint32_t v0 = (uint32_t)((uint64_t)nv * rank / group), v1 = (uint32_t)((uint64_t)nv * (rank + 1u) / group);
    // a value outside the accesses for this thread: before them, or behind them
    uint32_t single = a.V;
    if (rank == 0 && tid < head) single = tid;
    if (rank == group - 1u && tid >= 32u && tail + tid - 32u < a.V) single = tail + tid - 32u;

    float m = -kInf;
    uint64_t s2 = 0ull, t2 = 0ull;  // S and T of every other value
    uint32_t at = 0;                // the step in which the maximum was seen first
    const uint64_t log2e2 = pair(kLog2e, kLog2e);
    auto raise = [&](float to, uint32_t n) {
        const float d = fmaxf((m - to) * kLog2e, -300.f), f = exp2_fast(d);
        const uint64_t d2 = pair(d, d), f2 = pair(f, f);
        t2 = mul2(f2, fma2(s2, d2, t2));
        s2 = mul2(f2, s2);
        m = to, at = n;
    };
    auto take = [&](float v, float w) {  // (fmaxf drops the NaN of an infinity less an infinity)
        const float2 l = halves(mul2(add2(pair(v, w), pair(-m, -m)), log2e2));
        const float lv = fmaxf(l.x, -300.f), lw = fmaxf(l.y, -300.f);
        const uint64_t e2 = pair(exp2_fast(lv), exp2_fast(lw));
        s2 = add2(s2, e2);
        t2 = fma2(e2, pair(lv, lw), t2);
    };
    for (uint32_t n = 0; v0 + tid + n * kThreads < v1; n += U) {
        uint4 p[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint32_t i = v0 + tid + (n + u) * kThreads;
            p[u] = __ldg(xv + (i < v1 ? i : v0 + tid + n * kThreads));
        }
        float v[N];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const bool in = v0 + tid + (n + u) * kThreads < v1;
#pragma unroll
            for (uint32_t j = 0; j < E; j++) {
                v[u * E + j] = to_float(reinterpret_cast<const T*>(&p[u])[j]);
                if (u) v[u * E + j] = in ? v[u * E + j] : -kInf;
            }
        }
        float mx = v[0];
#pragma unroll
        for (uint32_t j = 1; j < N; j++) mx = max_nan(mx, v[j]);
        if (!(mx <= m)) raise(max_nan(mx, m), n);
#pragma unroll
        for (uint32_t j = 0; j < N; j += 2u) take(v[j], v[j + 1u]);
    }
    const float own = m;  // of the accesses alone
    const uint32_t own_at = at;
    if (single < a.V) {
        const float v = to_float(x[single]);
        if (!(v <= m)) raise(max_nan(v, m), 0u);
        take(v, -kInf);
    }
    Stats st{m, halves(s2).x + halves(s2).y, halves(t2).x + halves(t2).y};

    __shared__ unsigned long long s_keys[kWarps][32];
    __shared__ Stats s_stats[kWarps];
    __shared__ unsigned long long c_keys[TOP ? kMaxGroup : 1][32];
    __shared__ Stats c_stats[kMaxGroup];
    st.add_lanes();
    if (lane == 0) s_stats[warp] = st;
    unsigned long long list = 0ull;
    if constexpr (TOP) {
        unsigned long long key = 0ull;
        if (v0 + tid < v1) {  // where in its step the maximum is
            uint32_t idx = 0xFFFFFFFFu;
#pragma unroll
            for (uint32_t u = U; u-- > 0u;) {
                const uint32_t i = v0 + tid + (own_at + u) * kThreads;
                if (i >= v1) continue;
                const uint4 p = __ldg(xv + i);
#pragma unroll
                for (uint32_t j = E; j-- > 0u;)
                    if (to_float(reinterpret_cast<const T*>(&p)[j]) == own) idx = head + i * E + j;
            }
            key = make_key(own, idx);
        }
        const unsigned long long best = merge_cta(sort_warp(key, lane), s_keys, warp, lane);  // lane i: the i-th of the threads' best keys
        const unsigned long long bound = __shfl_sync(kFull, best, a.nTop - 1u);
        unsigned long long least = bound ? bound - 1ull : 0ull;  // what a key has to exceed
        auto offer = [&](unsigned long long k) {  // a key of every lane, 0: none
            uint32_t who = __ballot_sync(kFull, k > least);
            while (who) {
                const unsigned long long c = __shfl_sync(kFull, k, __ffs(who) - 1u);
                who &= who - 1u;
                if (c <= least) continue;
                const uint32_t pos = __popc(__ballot_sync(kFull, list > c));
                const unsigned long long up = __shfl_up_sync(kFull, list, 1);
                if (lane >= pos) list = lane == pos ? c : up;
                const unsigned long long last = __shfl_sync(kFull, list, a.nTop - 1u);
                least = last > least ? last : least;
            }
        };
        for (uint32_t w = warp; w < a.nTop; w += kWarps) {
            const unsigned long long k = __shfl_sync(kFull, best, w);
            if (k == 0ull) break;
            const uint32_t t = ((key_index(k) - head) / E - v0) % kThreads;
            for (uint32_t i0 = v0 + t; i0 < v1; i0 += 32u * kThreads) {
                const uint32_t i = i0 + lane * kThreads;
                uint4 p = make_uint4(0u, 0u, 0u, 0u);
                if (BPQ4K_CHECK(t < kThreads, a.status) && i < v1) p = __ldg(xv + i);
#pragma unroll
                for (uint32_t j = 0; j < E; j++) offer(i < v1 ? make_key(to_float(reinterpret_cast<const T*>(&p)[j]), head + i * E + j) : 0ull);
            }
        }
        if (warp < 2u) offer(single < a.V ? make_key(to_float(x[single]), single) : 0ull);
        __syncthreads();
        list = merge_cta(list, s_keys, warp, lane);
    } else {
        __syncthreads();
    }
    st = lane < kWarps ? s_stats[lane] : Stats{-kInf, 0.f, 0.f};
    st.add_lanes();
    if (group > 1u) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (warp == 0) {
            if constexpr (TOP) store_cluster(&c_keys[rank][lane], list);
            if (lane == 0) store_cluster(&c_stats[rank], st);
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank) return;
        st = lane < group ? c_stats[lane] : Stats{-kInf, 0.f, 0.f};
        st.add_lanes();
        if constexpr (TOP) {
            list = c_keys[0][lane];
            for (uint32_t g = 1; g < group; g++) list = merge_warp(list, c_keys[g][lane], lane);
        }
    }
    const bool bad = !(st.m < kInf);      // a NaN or +infinity
    const bool none = st.m == -kInf;      // the row's mask leaves nothing
    const float ln_s = logf(st.s), nan = __uint_as_float(0x7FC00000u);
    auto logp = [&](float v) { return bad ? nan : none || v == -kInf ? -kInf : (float)((double)v - (double)st.m - (double)ln_s); };
    if (a.entropy && tid == 0) a.entropy[row] = bad ? nan : none ? 0.f : ln_s - 0.69314718056f * (st.t / st.s);
    for (uint32_t g = tid; g < a.nGiven; g += kThreads) {
        const int32_t id = a.given[(uint64_t)row * a.nGiven + g];
        a.given_lp[(uint64_t)row * a.nGiven + g] = id < 0 || (uint32_t)id >= a.V ? nan : logp(to_float(x[id]));
    }
    if (TOP && tid < a.nTop) {
        a.top_ids[(uint64_t)row * a.nTop + tid] = bad ? -1 : (int32_t)key_index(list);
        a.top_lp[(uint64_t)row * a.nTop + tid] = logp(key_value(list));
    }
}

template <typename T, bool TOP>
cudaError_t launch_rows(const LogprobsArgs& a, uint32_t group, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.M * group);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = group, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = group > 1u ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, TOP>, a, group);
}

template <typename T>
cudaError_t launch_type(const LogprobsArgs& a, int sm_count, cudaStream_t stream) {
    // CTAs that share a row: while there are SMs without one, and a thread has a step's work
    uint32_t group = 1;
    while (group < kMaxGroup && a.M * group * 2u <= 2u * (uint32_t)sm_count && a.V >= group * 2u * kThreads * 8u) group *= 2u;
    return a.nTop ? launch_rows<T, true>(a, group, stream) : launch_rows<T, false>(a, group, stream);
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs& a, int ftype, int sm_count, cudaStream_t stream) {
    if (a.M == 0) return cudaSuccess;
    switch (ftype) {
        case 0: return launch_type<float>(a, sm_count, stream);
        case 1: return launch_type<__half>(a, sm_count, stream);
        case 30: return launch_type<__nv_bfloat16>(a, sm_count, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace bpq4k
