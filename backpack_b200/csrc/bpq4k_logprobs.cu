// What a row of logits says: log probabilities of given tokens, the entropy, the most likely tokens.  One pass over the row.
//
//   m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m):   log p(i) = x_i - m - ln S,   H = ln S - T / S
//
// A warp takes 1024 neighbouring values at a time.  S and T are kept relative to the running maximum of what the warp has seen and
// rescaled when that grows.  The difference to the maximum is taken before anything else, so logits of any magnitude are sound and
// the largest has the weight 1 exactly; the arithmetic is on pairs (add, mul and fma .f32x2: half an instruction a value each).
// Both terms of H are at least zero, so nothing cancels.
//
// The most likely tokens cost the pass next to nothing.  Values are compared as 64-bit keys (the value in the order of unsigned
// words, below it the inverted index: the larger key is the larger value or, among equal ones, the lower index; no two are equal).
// The pass leaves the largest value of every block (1024 values, 512 bytes of them in short rows); the k best tokens lie in the k blocks
// that are first by largest value and, among equal ones, by position: whatever lies elsewhere has a value of each of these before it.
// These blocks, or the lines of 512 bytes in them that matter, are read once more (a thread's own values, 16 bytes here and there,
// would cost 64 bytes of DRAM for each 16: 512 x 128256, 32 tokens, 77 us against 54).
//
// Few rows: CTAs of a cluster share a row, so that no working memory is needed; the first of them gathers.  Which values a thread
// adds up, and so the last bits of S and T, follows from that and from where the row lies between 16-byte boundaries.
//
// What bounds it.  Float logits: DRAM (512 x 128256: 42 us without alternatives, 0.95 of the copy rate; 48 with five: a row's last
// 5 us, the selection, have no other row to overlap).  16-bit logits: instructions, about 11 a value (32 us, 0.63; the exponentials
// alone are 15).  Few rows: the chain load, reduce, select, gather (1 x 128256: 4.9 us, with 20 alternatives 9.6).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>
#include <type_traits>

#include "kernels.h"
#include "q4k_common.cuh"

namespace bpq4k {

namespace {

constexpr uint32_t kFull = 0xFFFFFFFFu;
constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kBlockValues = 1024;  // values of a step, and of the smallest block that is not fine
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

__device__ __forceinline__ float warp_max_nan(float v) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
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

// The largest of the values of U accesses, a NaN if one is; 16-bit values are compared as they are, two at a time.
template <uint32_t U>
__device__ __forceinline__ float largest(const uint4 (&p)[U], float) {
    float m = __uint_as_float(p[0].x);
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
        m = max_nan(max_nan(max_nan(m, __uint_as_float(p[u].x)), __uint_as_float(p[u].y)), max_nan(__uint_as_float(p[u].z), __uint_as_float(p[u].w)));
    return m;
}
template <uint32_t U, typename T>
__device__ __forceinline__ float largest(const uint4 (&p)[U], T) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 m = reinterpret_cast<const T2&>(p[0].x);
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
        m = __hmax2_nan(__hmax2_nan(__hmax2_nan(m, reinterpret_cast<const T2&>(p[u].x)), reinterpret_cast<const T2&>(p[u].y)),
                        __hmax2_nan(reinterpret_cast<const T2&>(p[u].z), reinterpret_cast<const T2&>(p[u].w)));
    return max_nan(to_float(m.x), to_float(m.y));
}

// Maximum, S and T of some values, T in units of ln 2.
struct Stats {
    float m, s, t;
};
// The sum of the first n lanes' (n a power of two), in all lanes.
__device__ __forceinline__ Stats add_lanes(Stats v, uint32_t n) {
    float m = v.m;
    for (uint32_t o = n >> 1; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(kFull, m, o));
    // (-infinity less -infinity is a NaN, and fmaxf drops it; 2^-300 is 0 as a float)
    const float d = fmaxf((v.m - m) * kLog2e, -300.f), f = exp2_fast(d);
    v.t = f * fmaf(v.s, d, v.t);
    v.s *= f;
    for (uint32_t o = n >> 1; o; o >>= 1) v.s += __shfl_xor_sync(kFull, v.s, o), v.t += __shfl_xor_sync(kFull, v.t, o);
    return {__shfl_sync(kFull, m, 0), __shfl_sync(kFull, v.s, 0), __shfl_sync(kFull, v.t, 0)};
}

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

// How many of n keys are larger than `mine`; keys[n] may be read and is 0 where n is odd.  All keys differ, so this is the key's
// place in descending order: for the few hundred keys here, reads that do not wait for one another, where a sort is a chain of
// exchanges (lists of the warps, sorted and merged in a tree: 8 x 128256, 5 tokens 8.5 us, by places 8.1; 512 x 4000 7.9, 7.3;
// only 1 x 128256, 20 tokens 8.8, 9.6).
__device__ __forceinline__ uint32_t place_of(const unsigned long long* keys, uint32_t n, unsigned long long mine) {
    uint32_t place = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < n; i += 2u) {
        const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(keys + i);
        place += (k.x > mine ? 1u : 0u) + (k.y > mine ? 1u : 0u);
    }
    return place;
}

// FINE: a block is one access of a warp (a line), else a step or more.  LINES: a block is a step, and the lines' largest values are
// kept beside the blocks', so that only lines are read again that have a value like the k-th block's.
template <typename T, bool TOP, bool FINE, bool LINES, uint32_t kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logprobs_kernel(const __grid_constant__ LogprobsArgs a, const uint32_t group) {
    constexpr uint32_t kWarps = kThreads / 32u;
    // (half of either: float 48.3 and 60.5 us for 512 x 128256, bfloat16 36.9 and 43.2; twice, bfloat16: 37.8)
    constexpr uint32_t E = 16 / sizeof(T), U = 32 / E, kLog = U == 8u ? 3u : 2u;
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
    // lines of 32 accesses; 2^shift of them are a block
    constexpr uint32_t kStep = 32u * U;
    const uint32_t steps = (v1 - v0 + kStep - 1u) / kStep, lines = (v1 - v0 + 31u) / 32u;
    uint32_t shift = FINE ? 0u : kLog;
    while (!FINE && (lines >> shift) >= kThreads) shift++;  // a thread to a block; fine ones are few enough (launch_type)
    const uint32_t blocks = (lines + (1u << shift) - 1u) >> shift;
    __shared__ __align__(16) unsigned long long s_keys[TOP ? kThreads : 1];  // of the blocks: the largest value, the position
    __shared__ float s_line[LINES ? kThreads * U : 1];
    if (TOP && tid >= blocks) s_keys[tid] = 0ull;

    // the given tokens' logits, the first of each thread: fetched now, needed at the end
    int32_t id = -1;
    float id_logit = 0.f;
    if (rank == 0 && tid < a.nGiven) {
        id = a.given[(uint64_t)row * a.nGiven + tid];
        if (id >= 0 && (uint32_t)id < a.V) id_logit = to_float(x[id]);
    }

    const uint64_t log2e2 = pair(kLog2e, kLog2e);
    float m = -kInf;                // of the warp
    uint64_t s2 = 0ull, t2 = 0ull;  // S and T of every other value
    auto raise = [&](float to) {
        const float d = fmaxf((m - to) * kLog2e, -300.f), f = exp2_fast(d);
        const uint64_t d2 = pair(d, d), f2 = pair(f, f);
        t2 = mul2(f2, fma2(s2, d2, t2));
        s2 = mul2(f2, s2);
        m = to;
    };
    auto take = [&](float v, float w) {  // (fmaxf drops the NaN of an infinity less an infinity)
        const float2 l = halves(mul2(add2(pair(v, w), pair(-m, -m)), log2e2));
        const float lv = fmaxf(l.x, -300.f), lw = fmaxf(l.y, -300.f);
        const uint64_t e2 = pair(exp2_fast(lv), exp2_fast(lw));
        s2 = add2(s2, e2);
        t2 = fma2(e2, pair(lv, lw), t2);
    };
    auto take_access = [&](const uint4& p) {
#pragma unroll
        for (uint32_t j = 0; j < E; j += 2u) take(to_float(reinterpret_cast<const T*>(&p)[j]), to_float(reinterpret_cast<const T*>(&p)[j + 1u]));
    };
    const uint32_t block_steps = FINE ? 1u : 1u << (shift - kLog);
    for (uint32_t b = warp; b * block_steps < steps; b += kWarps) {
        float block = -kInf;
        for (uint32_t step = b * block_steps; step < min(steps, (b + 1u) * block_steps); step++) {
            const uint32_t i = v0 + step * kStep + lane;
            uint4 p[U];
            float mx = -kInf;
            const bool whole = v0 + (step + 1u) * kStep <= v1;
            if (!FINE && !LINES && whole) {
#pragma unroll
                for (uint32_t u = 0; u < U; u++) p[u] = __ldg(xv + i + 32u * u);
                mx = warp_max_nan(largest<U>(p, T(0.f)));
            } else {
#pragma unroll
                for (uint32_t u = 0; u < U; u++)
                    if (whole || i + 32u * u < v1) p[u] = __ldg(xv + i + 32u * u);
#pragma unroll
                for (uint32_t u = 0; u < U; u++) {
                    const uint4 one[1] = {p[u]};
                    const float line = warp_max_nan(whole || i + 32u * u < v1 ? largest<1>(one, T(0.f)) : -kInf);
                    mx = max_nan(mx, line);
                    if (LINES && lane == u && BPQ4K_CHECK(step < kThreads, a.status)) s_line[step * U + u] = line;
                    if (TOP && FINE && lane == 0 && step * U + u < lines && BPQ4K_CHECK(lines <= kThreads, a.status)) s_keys[step * U + u] = make_key(line, step * U + u);
                }
            }
            if (!(mx <= m)) raise(max_nan(mx, m));
            block = fmaxf(block, mx);
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                if (whole || i + 32u * u < v1) take_access(p[u]);
        }
        if (TOP && !FINE && lane == 0 && BPQ4K_CHECK(b < kThreads, a.status)) s_keys[b] = make_key(block, b);
    }
    if (warp < 2u) {
        const float v = single < a.V ? to_float(x[single]) : -kInf, mx = warp_max_nan(v);
        if (!(mx <= m)) raise(max_nan(mx, m));
        take(v, -kInf);
    }
    Stats st{m, halves(s2).x + halves(s2).y, halves(t2).x + halves(t2).y};

    __shared__ Stats s_stats[kWarps];
    __shared__ __align__(16) unsigned long long s_found[TOP ? kThreads : 1];
    __shared__ unsigned long long s_list[32];  // the first blocks, then the largest keys, in descending order; 0 behind the last
    __shared__ uint32_t s_count, s_lines;
    __shared__ uint32_t s_again[LINES ? 32u * U : 1];  // the lines to be read again
    __shared__ __align__(16) unsigned long long c_keys[TOP ? kMaxGroup * 32u : 1];
    __shared__ Stats c_stats[kMaxGroup];
#pragma unroll
    for (int o = 16; o; o >>= 1) st.s += __shfl_xor_sync(kFull, st.s, o), st.t += __shfl_xor_sync(kFull, st.t, o);  // (one maximum a warp)
    if (lane == 0) s_stats[warp] = st;
    if constexpr (TOP) {
        if (tid < 32u) s_list[tid] = 0ull;
        if (tid == 0) s_lines = 0u;
        __syncthreads();
        // the k first blocks
        const unsigned long long own = s_keys[tid];
        if (own) {
            const uint32_t place = place_of(s_keys, blocks, own);
            if (place < a.nTop) s_list[place] = own;
        }
        __syncthreads();
        const unsigned long long best = s_list[lane], bound = s_list[a.nTop - 1u];
        // what a key has to exceed: the k-th block has a value like its largest, at its end if nowhere else
        unsigned long long least = 0ull;
        if (bound) least = make_key(key_value(bound), head + min(v1, v0 + ((key_index(bound) + 1u) << shift) * 32u) * E - 1u) - 1ull;
        uint32_t first_lines = __popc(__ballot_sync(kFull, best != 0ull)) << shift;  // (lane i has the i-th block; none behind the k-th)
        if constexpr (LINES) {
            const float like = bound ? key_value(bound) : -kInf;
            for (uint32_t l = tid; l < first_lines; l += kThreads) {
                const uint32_t line = key_index(s_list[l >> kLog]) * U + l % U;
                if (line < lines && !(s_line[line] < like)) s_again[atomicAdd(&s_lines, 1u)] = line;
            }
            __syncthreads();
            first_lines = s_lines;
        }
        // Keys above `least` are collected, a few more than k as a rule.  Should they not fit, the k-th of those that did is a better
        // bound, and the blocks are read again.
        for (;;) {
            if (tid == 0) s_count = 0u;
            s_found[tid] = 0ull;
            __syncthreads();
            auto offer = [&](unsigned long long k) {
                if (k <= least) return;
                const uint32_t at = atomicAdd(&s_count, 1u);
                if (at < kThreads) s_found[at] = k;
            };
            // the lines of the blocks, dealt to the warps, R of each in flight
            constexpr uint32_t R = 4;
            for (uint32_t l0 = warp; l0 < first_lines; l0 += R * kWarps) {
                uint4 p[R];
                uint32_t at[R];
#pragma unroll
                for (uint32_t u = 0; u < R; u++) {
                    const uint32_t l = l0 + u * kWarps;
                    uint32_t line;
                    if constexpr (LINES)
                        line = s_again[min(l, 32u * U - 1u)];
                    else
                        line = (key_index(__shfl_sync(kFull, best, min(l >> shift, 31u))) << shift) + (l & ((1u << shift) - 1u));
                    at[u] = l < first_lines ? v0 + line * 32u + lane : v1;
                    if (BPQ4K_CHECK(l >= first_lines || line >> shift < blocks, a.status) && at[u] < v1) p[u] = __ldg(xv + at[u]);
                }
#pragma unroll
                for (uint32_t u = 0; u < R; u++)
#pragma unroll
                    for (uint32_t j = 0; j < E; j++)
                        if (at[u] < v1) offer(make_key(to_float(reinterpret_cast<const T*>(&p[u])[j]), head + at[u] * E + j));
            }
            if (single < a.V) offer(make_key(to_float(x[single]), single));
            __syncthreads();
            const uint32_t found = s_count, kept = min(found, kThreads);
            const unsigned long long key = s_found[tid];
            if (tid < 32u) s_list[tid] = 0ull;
            __syncthreads();
            if (key) {
                const uint32_t place = place_of(s_found, kept, key);
                if (place < 32u) s_list[place] = key;
            }
            __syncthreads();
            if (found <= kThreads) break;
            least = s_list[a.nTop - 1u] - 1ull;
        }
    } else {
        __syncthreads();
    }
    st = add_lanes(s_stats[lane % kWarps], kWarps);
    if (group > 1u) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (warp == 0) {
            if (TOP && lane < a.nTop) store_cluster(&c_keys[rank * a.nTop + lane], s_list[lane]);
            if (lane == 0) store_cluster(&c_stats[rank], st);
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (rank) return;
        st = add_lanes(c_stats[lane % group], group);
        if constexpr (TOP) {
            if (tid < 32u) s_list[tid] = 0ull;
            __syncthreads();
            for (uint32_t i = tid; i < group * a.nTop; i += kThreads) {  // (an even number: clusters are)
                const unsigned long long key = c_keys[i];
                if (key == 0ull) continue;
                const uint32_t place = place_of(c_keys, group * a.nTop, key);
                if (place < a.nTop) s_list[place] = key;
            }
            __syncthreads();
        }
    }
    const bool bad = !(st.m < kInf);      // a NaN or +infinity
    const bool none = st.m == -kInf;      // the row's mask leaves nothing
    const float ln_s = logf(st.s), nan = __uint_as_float(0x7FC00000u);
    auto logp = [&](float v) { return bad ? nan : none || v == -kInf ? -kInf : (float)((double)v - (double)st.m - (double)ln_s); };
    if (a.entropy && tid == 0) a.entropy[row] = bad ? nan : none ? 0.f : ln_s - 0.69314718056f * (st.t / st.s);
    auto is_token = [&](int32_t i) { return i >= 0 && (uint32_t)i < a.V; };
    if (tid < a.nGiven) a.given_lp[(uint64_t)row * a.nGiven + tid] = is_token(id) ? logp(id_logit) : nan;
    for (uint32_t g = tid + kThreads; g < a.nGiven; g += kThreads) {
        id = a.given[(uint64_t)row * a.nGiven + g];
        a.given_lp[(uint64_t)row * a.nGiven + g] = is_token(id) ? logp(to_float(x[id])) : nan;
    }
    if (TOP && tid < a.nTop) {
        const unsigned long long key = s_list[tid];
        a.top_ids[(uint64_t)row * a.nTop + tid] = bad ? -1 : (int32_t)key_index(key);
        a.top_lp[(uint64_t)row * a.nTop + tid] = logp(key_value(key));
    }
}

template <typename T, bool TOP, bool FINE, bool LINES, uint32_t kThreads>
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
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, TOP, FINE, LINES, kThreads>, a, group);
}

template <typename T>
cudaError_t launch_group(const LogprobsArgs& a, uint32_t group, cudaStream_t stream) {
    if (!a.nTop) return launch_rows<T, false, false, false, 256>(a, group, stream);
    // fine blocks where a CTA's part of a row has fewer of the others than tokens are asked for
    if (a.V / group >= a.nTop * kBlockValues) {
        // Lines cost the pass 5 us of 46 (512 x 128256 float), and the second read, of few of them, no longer grows with k: 5 tokens 51.9 us,
        // without 47.8; 16 tokens 52.4, 52.5; 32 tokens 54.0, 59.5; 512 x 32000 float, 20 tokens 19.4, 23.6; bfloat16, 5 tokens 14.0, 13.8;
        // 64 x 128256, four CTAs a row, 5 tokens 13.7, 14.3.  So: where k blocks are an eighth of the row.
        if ((uint64_t)a.nTop * 8u * kBlockValues >= a.V / group && a.V / group <= 255u * kBlockValues) return launch_rows<T, true, false, true, 256>(a, group, stream);
        return launch_rows<T, true, false, false, 256>(a, group, stream);
    }
    // (512 x 4000 float: 128 threads 7.7 us, 256 8.7; 8 x 128256, eight CTAs a row: 11.0 and 9.0)
    if (a.V / group > 4096u) return launch_rows<T, true, true, false, 256>(a, group, stream);
    return launch_rows<T, true, true, false, 128>(a, group, stream);
}

template <typename T>
cudaError_t launch_type(const LogprobsArgs& a, int sm_count, cudaStream_t stream) {
    // CTAs that share a row: while they are fewer than the machine holds at once, and a thread has 16 values
    uint32_t group = 1;
    while (group < kMaxGroup && (uint64_t)a.M * group * 2u <= 4ull * sm_count && a.V >= group * 2u * 4096u) group *= 2u;
    cudaError_t e = launch_group<T>(a, group, stream);
    if (e != cudaSuccess && group > 1u) {  // a context that cannot place clusters (restricted SM sets): a CTA to a row
        cudaGetLastError();
        e = launch_group<T>(a, 1u, stream);
    }
    return e;
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
