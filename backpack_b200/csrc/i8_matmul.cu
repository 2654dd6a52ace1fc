// Matrix product of 8-bit rows with 8-bit weights: Y[m][n] = (sum_k x[m][k] * w[n][k]) * xs[m] * ws[n] + bias[n].
//
// The sum is an exact 32-bit integer (K <= 131071), so neither the order of it nor the split of K changes a bit of the result.
//
// tcgen05.mma.kind::i8 with the weights as the M side (128 rows of a CTA, 256 of a pair) and up to 256 activation rows as the N
// side: one lane of tensor memory is one output channel, so a warp's store of one activation row is 32 neighbouring outputs.
// Both operands come by TMA in steps of 128 codes (128-byte swizzle); rows behind M, N and codes behind K arrive as zeros.
//   one CTA    few activation rows.  Bound by reading the weights; CTAs of a cluster share the K range of a tile where there
//              are fewer tiles than SMs, and each adds up and stores its share of the tile's columns.
//   a pair     many activation rows (tcgen05 cta_group::2): each CTA loads half of either operand.
// What bounds it (us; "against": the larger of the bytes at the measured copy rate, 6542 GB/s, and the operations at twice the
// measured bfloat16 rate; a yardstick, not a bound: reads alone can run faster than a copy, and the clock varies under the power cap).
// 2048 x 28672 x 8192: 292 to 305 against 294, the tensor cores under the power cap.  1 x 128256 x 4096: 79 against 80, DRAM.
// Between, whole rounds of tiles (256 x 28672 x 8192: 112 tiles on 74 pairs, 57 against 41) and the 4.6 us from a kernel's start to
// its first sum and from the last to the end (13 x 6144 x 4096: 9.2 against 3.9).
// Roles (12 warps): warp 0 TMA, warp 1 mma, warp 2 tensor memory, warps 4-11 epilogue.  Persistent over the tiles; two
// accumulators, so that a tile accumulates while the one before it is stored.
//
// A CTA takes more than half of an SM's shared memory, so two that allocate tensor memory never meet on one SM: with kernels on
// several streams no allocation waits for a CTA that waits in a cluster for a third.
//
// Every wait is bounded: on a time-out the role raises the abort flag of every CTA of its cluster and the device status word, and
// waits that would block return at once from then on.  All threads of the cluster meet at the end, where the flag is final: if it
// is raised, copies and mmas in flight are waited for (bounded too), whichever role gave up, before tensor memory is freed.
#include <cuda.h>
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

// The same three roundings in every kernel: the sum to a float, its product with xs, and that times ws plus the bias.
__device__ __forceinline__ float finish(int s, float xs, float ws, float bias) { return fmaf(__fmul_rn((float)s, xs), ws, bias); }

// ---- few activation rows: weights straight into registers ---------------------------------------------------------------


// 16 codes from byte k of a row on: zeros behind the row, and (`clean`) in place of the bytes behind code K.
__device__ __forceinline__ int4 codes16(const int8_t* row, uint32_t k, uint32_t K, bool clean) {
    if (k >= K) return make_int4(0, 0, 0, 0);
    int4 v = __ldg(reinterpret_cast<const int4*>(row + k));
    if (clean && k + 16u > K) {
        const uint32_t n = K - k;  // 1..15 codes
        auto keep = [n](int w, uint32_t first) { return n >= first + 4u ? w : n <= first ? 0 : w & (int)((1u << (8u * (n - first))) - 1u); };
        v.x = keep(v.x, 0), v.y = keep(v.y, 4), v.z = keep(v.z, 8), v.w = keep(v.w, 12);
    }
    return v;
}
__device__ __forceinline__ void mma_i8(int (&c)[4], int a0, int a1, int a2, int a3, int b0, int b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr uint32_t kStreamRows = 8;  // activation rows at most: the mma's columns

// A warp takes 16 weight rows and a share of K; 2^wk_log warps of the CTA share the rows.  Lane (g, t) = (lane / 4, lane % 4) loads
// the 16 bytes 64 p + 16 t of rows g and g + 8 and of activation row g: which codes of K meet in one mma does not matter as long as
// both operands agree, so a lane's 16 bytes are the fragments of two mmas as they are.  No shared memory, tensor memory or barrier
// stands between the launch and the first load: 1 x 1024 x 4096 3.7 us, by the kernel below 6.0; 1 x 4096 x 4096 5.7 and 7.6;
// 4 x 6144 x 4096 8.1 and 9.4.  Its loads are 64 bytes of 16 rows at a time, which DRAM likes less than whole boxes: 1 x 14336 x
// 4096 12.8 us both, 8 x 28672 x 8192 50 and 44.
template <typename T, uint32_t kStreamWarps>
__global__ void __launch_bounds__(kStreamWarps * 32, 1024 / (kStreamWarps * 32)) matmul_i8_stream_kernel(const __grid_constant__ MatmulI8Args a, const uint32_t wk_log) {
    constexpr uint32_t kStreamThreads = kStreamWarps * 32, kPieces = 4;  // 64-byte pieces of a row in flight
    __shared__ int parts[kStreamWarps][16][8];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t tiles = kStreamWarps >> wk_log, n0 = (blockIdx.x * tiles + (warp >> wk_log)) * 16u, share = warp & ((1u << wk_log) - 1u);
    const uint32_t pieces = (a.K + 63u) / 64u;
    const uint32_t p0 = (uint32_t)((uint64_t)pieces * share >> wk_log), p1 = (uint32_t)((uint64_t)pieces * (share + 1u) >> wk_log);
    const int8_t* w0 = a.W + (uint64_t)min(n0 + g, a.N - 1u) * a.ldw;
    const int8_t* w1 = a.W + (uint64_t)min(n0 + g + 8u, a.N - 1u) * a.ldw;
    const int8_t* x = a.X + (uint64_t)min(g, a.M - 1u) * a.ldx;
    int c[4] = {};
    asm volatile("griddepcontrol.wait;" ::: "memory");  // all that is read comes from earlier kernels
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // the scales of this thread's first output: needed at the end, fetched now
    const uint32_t rows = tiles * 16u, m_first = threadIdx.x / rows, n_first = blockIdx.x * rows + threadIdx.x % rows;
    const bool first = m_first < a.M && n_first < a.N;
    const float xs_first = first ? __ldg(a.xs + m_first) : 0.f, ws_first = first ? __ldg(a.ws + n_first) : 0.f;
    const float bias_first = first && a.bias ? __ldg(a.bias + n_first) : 0.f;
    for (uint32_t p = p0; p < p1; p += kPieces) {
        int4 u[kPieces], v[kPieces];
#pragma unroll
        for (uint32_t i = 0; i < kPieces; i++) {
            const uint32_t k = p + i < p1 ? (p + i) * 64u + t * 16u : a.K;
            u[i] = codes16(w0, k, a.K, false);
            v[i] = codes16(w1, k, a.K, false);
        }
#pragma unroll
        for (uint32_t i = 0; i < kPieces; i++) {
            const uint32_t k = p + i < p1 ? (p + i) * 64u + t * 16u : a.K;
            const int4 b = codes16(x, k, a.K, true);
            mma_i8(c, u[i].x, v[i].x, u[i].y, v[i].y, b.x, b.y);
            mma_i8(c, u[i].z, v[i].z, u[i].w, v[i].w, b.z, b.w);
        }
    }
    *reinterpret_cast<int2*>(&parts[warp][g][2u * t]) = make_int2(c[0], c[1]);
    *reinterpret_cast<int2*>(&parts[warp][g + 8u][2u * t]) = make_int2(c[2], c[3]);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < rows * a.M; i += kStreamThreads) {
        const uint32_t m = i / rows, r = i - m * rows, n = blockIdx.x * rows + r;
        if (n >= a.N || !BPQ4K_CHECK(m < a.M && m < kStreamRows, a.status)) continue;
        int sum = 0;
        for (uint32_t s = 0; s < 1u << wk_log; s++) sum += parts[((r >> 4) << wk_log) + s][r & 15u][m];
        static_cast<T*>(a.Y)[(uint64_t)m * a.ldy + n] = to_elem<T>(
            i < kStreamThreads ? finish(sum, xs_first, ws_first, bias_first) : finish(sum, __ldg(a.xs + m), __ldg(a.ws + n), a.bias ? __ldg(a.bias + n) : 0.f));
    }
}

template <typename T, uint32_t kStreamWarps>
cudaError_t launch_stream(const MatmulI8Args& m, uint32_t wk_log, cudaStream_t stream) {
    const uint32_t rows = (kStreamWarps >> wk_log) * 16u;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((m.N + rows - 1u) / rows);
    cfg.blockDim = dim3(kStreamWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, matmul_i8_stream_kernel<T, kStreamWarps>, m, wk_log);
}

// ---- tensor cores -------------------------------------------------------------------------------------------------------

#ifdef BPQ4K_DEBUG_CHECKS
constexpr uint32_t kWaitLimit = 1u << 28;             // polls of some 20 ns
#else
constexpr uint32_t kWaitLimit = 1u << 21;             // polls of up to 4 us
constexpr uint32_t kSuspendNs = 1000;
#endif
constexpr uint32_t kStep = 128;                       // codes of a row per ring stage: the swizzle's row
constexpr uint32_t kEpilogueWarps = 8, kThreads = (4 + kEpilogueWarps) * 32;
constexpr uint32_t kMaxStages = 12;
constexpr uint32_t kMaxSplits = 8;                    // CTAs that share a tile: the largest cluster that every device takes
constexpr uint32_t kMaxTile = 256;                    // activation rows of a tile

struct TcArgs {
    CUtensorMap tmap_w, tmap_x;  // [rows][K] bytes, boxes of 128 codes x 128 weight rows | tile / CTAs of the pair activation rows
    const float* xs;
    const float* ws;
    const float* bias;
    void* Y;
    uint32_t M, N, ldy;
    uint32_t tile, m_tiles, tiles, chunks;  // activation rows of a tile, tiles along M, tiles in all, steps along K
    uint32_t splits;                        // CTAs that share a tile's K range (one CTA form)
    uint32_t in_ring;                       // where they exchange their sums: 1 the ring (once it is free), 0 behind the barriers
    uint32_t stages, tmem_cols;
    uint32_t wait_limit;                    // polls after which a wait gives up
    int* status;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// One poll.  The product build is suspended meanwhile, for 4 us at most, whatever time is asked for; the debug build is not, so that a
// short limit ends waits anywhere in the kernel.  (A branch between the two in the product build: 2048 x 28672 x 8192 305 -> 336 us.)
__device__ __forceinline__ uint32_t mbar_poll(uint32_t bar, uint32_t parity) {
    uint32_t ok;
#ifdef BPQ4K_DEBUG_CHECKS
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
#else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kSuspendNs)
        : "memory");
#endif
    return ok;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// Raises the abort flag of every CTA of the cluster (of this one, where there is no cluster).
__device__ __forceinline__ void raise_abort(volatile int* abort_flag) {
    const uint32_t at = smem_u32(const_cast<const int*>(abort_flag));
    uint32_t ctas;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
    for (uint32_t q = 0; q < ctas; q++) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(at, q)), "r"(1) : "memory");
}
// Bounded wait; false if it ran out, or at once if it would block while the cluster aborts (the caller carries on without what it
// waited for, so that barriers of the CTA stay matched).
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int* abort_flag, const TcArgs& a) {
    if (mbar_poll(bar, parity)) return true;
    for (uint32_t i = 1; i < a.wait_limit; i++) {
        if (mbar_poll(bar, parity)) return true;
        if ((i & 63u) == 1u && *abort_flag) return false;
    }
    raise_abort(abort_flag);
    if (a.status) atomicExch(a.status, kDeviceTimeout);
    return false;
}
// The same for what is in flight when the cluster aborts.
__device__ __forceinline__ void wait_in_flight(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < kWaitLimit; i++)
        if (mbar_poll(bar, parity)) return;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A tile load into this CTA; its completion is counted on `bar`, for a pair on the leader's (a cluster address).
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* tmap, uint32_t x, uint32_t y, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(tmap), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(tmap), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
// K-major shared-memory descriptor, version 1 (sm_100): rows of 128 B, 128-byte swizzle, 8-row groups 1024 B apart.
__device__ __forceinline__ uint64_t desc_128(uint32_t a) { return (uint64_t)((a >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61); }
template <int CG>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Arrives on the barrier (of a pair: at this offset in both CTAs) when the mmas issued so far are done.
template <int CG>
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    if constexpr (CG == 1) {
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    } else {
        const uint16_t both = 3;
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(both)
                     : "memory");
    }
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// (the values are there after tmem_wait)
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr));
}
// Waits for the reads so far; the registers pass through, so that nothing that uses them moves ahead of it.
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                   "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueWarps * 32) : "memory"); }

// Shared memory behind the ring: activation scales of two tiles, barriers, flags; the exchange of a shared tile.
constexpr uint32_t kScaleBytes = 2u * kMaxTile * 4u, kBarBytes = 512u;
constexpr uint32_t stage_bytes(uint32_t tile, uint32_t cg) { return 128u * kStep + tile / cg * kStep; }
constexpr uint32_t exchange_bytes(uint32_t tile) { return tile * 128u * 4u; }
constexpr uint32_t smem_bytes(uint32_t stages, uint32_t tile, uint32_t cg, bool exchange) {
    return 1024u + stages * stage_bytes(tile, cg) + kScaleBytes + kBarBytes + (exchange ? exchange_bytes(tile) : 0u);
}

template <int CG, typename T>
__global__ void __launch_bounds__(kThreads, 2) matmul_i8_kernel(const __grid_constant__ TcArgs a) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t sbytes = stage_bytes(a.tile, CG), off_scale = a.stages * sbytes, off_bar = off_scale + kScaleBytes;
    float* scale = reinterpret_cast<float*>(base_ptr + off_scale);
    const uint32_t bar0 = base + off_bar, off_exchange = a.in_ring ? 0u : off_bar + kBarBytes;
    auto full = [&](uint32_t s) { return bar0 + s * 8u; };
    auto empty = [&](uint32_t s) { return bar0 + (kMaxStages + s) * 8u; };
    auto acc_full = [&](uint32_t b) { return bar0 + (2u * kMaxStages + b) * 8u; };
    auto acc_empty = [&](uint32_t b) { return bar0 + (2u * kMaxStages + 2u + b) * 8u; };
    const uint32_t parts_bar = bar0 + (2u * kMaxStages + 4u) * 8u, done_bar = parts_bar + 8u, ready_bar = parts_bar + 24u, issued_at = parts_bar + 32u;
    static_assert((2u * kMaxStages + 9u) * 8u <= kBarBytes, "barrier area");
    volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + off_bar + (2u * kMaxStages + 6u) * 8u);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + off_bar + (2u * kMaxStages + 6u) * 8u + 4u);
    const uint32_t* issued_steps = reinterpret_cast<const uint32_t*>(base_ptr + off_bar + (2u * kMaxStages + 8u) * 8u);  // by either half

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    uint32_t rank = 0;
    const uint32_t group = CG == 2 ? 2u : a.splits;            // CTAs of a cluster
    if (group > 1u) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const uint32_t first_tile = blockIdx.x / group, step_tile = gridDim.x / group;
    const uint32_t half = CG == 2 ? rank : 0u;                 // which half of the pair's operands
    const uint32_t part = CG == 2 ? 0u : rank;                 // which share of K
    const bool leader = half == 0u;
    const uint32_t c0 = (uint32_t)((uint64_t)a.chunks * part / a.splits), c1 = (uint32_t)((uint64_t)a.chunks * (part + 1u) / a.splits);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < a.stages; s++) mbar_init(full(s), 1), mbar_init(empty(s), 1);
        for (uint32_t b = 0; b < 2; b++) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), CG * kEpilogueWarps);
        mbar_init(parts_bar, a.splits * kEpilogueWarps);
        mbar_init(ready_bar, a.splits);
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a.tmap_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a.tmap_x) : "memory");
    }
    if (warp == 2) {
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(a.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(a.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    fence_before();
    if (group > 1u) cluster_sync_all();  // barriers and tensor memory are ready before anything crosses over
    else __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // all that is read comes from earlier kernels
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- operands ----------------
            uint32_t s = 0, it = 0, issued = 0;
            const uint32_t full0 = CG == 2 ? peer_addr(full(0), 0u) : full(0);
            bool ok = true;
            for (uint32_t t = first_tile; t < a.tiles && ok; t += step_tile) {
                const uint32_t rt = t / a.m_tiles, n0 = (rt * CG + half) * 128u, m0 = (t - rt * a.m_tiles) * a.tile + half * (a.tile / CG);
                for (uint32_t c = c0; c < c1; c++) {
                    ok = it == 0 || wait_bar(empty(s), (it - 1u) & 1u, abort_flag, a);
                    if (!ok) break;
                    const uint32_t dst = base + s * sbytes, bar = full0 + s * 8u;
                    if (!BPQ4K_CHECK(s < a.stages && c < a.chunks && rt * CG * 128u < a.N, a.status)) {
                        raise_abort(abort_flag), ok = false;
                        break;
                    }
                    if (leader) mbar_expect_tx(full(s), CG * sbytes);
                    tma_load<CG>(dst, &a.tmap_w, c * kStep, n0, bar);
                    tma_load<CG>(dst + 128u * kStep, &a.tmap_x, c * kStep, m0, bar);
                    issued++;
                    if (++s == a.stages) s = 0, it++;
                }
            }
            for (uint32_t q = 0; q < CG; q++)  // (both of a pair know how far both came)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(issued_at + half * 4u, CG == 2 ? q : rank)), "r"(issued) : "memory");
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            // ---------------- products ----------------
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((a.tile >> 3) << 17) | ((CG * 128u >> 4) << 24);  // s32 += s8 * s8, K-major
            uint32_t s = 0, it = 0, i = 0;
            bool ok = true;
            for (uint32_t t = first_tile; t < a.tiles && ok; t += step_tile, i++) {
                const uint32_t buf = i & 1u, d = tmem + buf * a.tile;
                ok = i < 2u || wait_bar(acc_empty(buf), ((i >> 1) - 1u) & 1u, abort_flag, a);
                fence_after();
                for (uint32_t c = c0; c < c1 && ok; c++) {
                    ok = wait_bar(full(s), it & 1u, abort_flag, a);
                    if (!ok) break;
                    fence_after();
                    const uint64_t da = desc_128(base + s * sbytes), db = desc_128(base + s * sbytes + 128u * kStep);
#pragma unroll
                    for (uint32_t k = 0; k < kStep / 32u; k++) umma<CG>(d, da + k * 2u, db + k * 2u, idesc, (c > c0 || k) ? 1u : 0u);
                    umma_commit<CG>(empty(s));
                    if (++s == a.stages) s = 0, it++;
                }
                if (ok) umma_commit<CG>(acc_full(buf));
            }
        }
    } else if (warp >= 4) {
        // ---------------- epilogue ----------------
        const uint32_t e = threadIdx.x - 128u, quad = warp & 3u, side = (warp - 4u) >> 2, r = quad * 32u + lane;
        T* Y = static_cast<T*>(a.Y);
        uint32_t i = 0;
        bool ok = true;
        for (uint32_t t = first_tile; t < a.tiles; t += step_tile, i++) {
            const uint32_t rt = t / a.m_tiles, n = (rt * CG + half) * 128u + r, m0 = (t - rt * a.m_tiles) * a.tile, buf = i & 1u;
            const uint32_t cols = min(a.tile, a.M - m0);
            const bool live = n < a.N;
            const float wscale = live ? __ldg(a.ws + n) : 0.f, bias = live && a.bias ? __ldg(a.bias + n) : 0.f;
            float* xscale = scale + buf * kMaxTile;
            if (e < cols) xscale[e] = __ldg(a.xs + m0 + e);
            epilogue_sync();
            // (a whole warp reads tensor memory, or none of it; after a wait that ran out it reads no more, stores no more and arrives nowhere)
            ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(acc_full(buf), (i >> 1) & 1u, abort_flag, a));
            fence_after();
            const uint32_t acc = tmem + ((quad * 32u) << 16) + buf * a.tile;
            if (CG == 2 || a.splits == 1u) {
                auto store = [&](uint32_t c, const uint32_t (&v)[16]) {
                    T* y = Y + (uint64_t)(m0 + c) * a.ldy + n;
                    if (live) {
#pragma unroll
                        for (uint32_t j = 0; j < 16; j++)
                            if (c + j < cols) y[(uint64_t)j * a.ldy] = to_elem<T>(finish((int)v[j], xscale[c + j], wscale, bias));
                    }
                };
                if constexpr (CG == 2) {  // one read ahead of the stores (in the one CTA form its registers cost the exchange more: 100 x 4096 x 4096 10.0 -> 11.3 us)
                    uint32_t v[16], next[16];
                    if (side * 16u < cols && ok) tmem_ld16(acc + side * 16u, v);
                    for (uint32_t c = side * 16u; c < cols && ok; c += 64u) {
                        tmem_wait(v);
                        if (c + 32u < cols) tmem_ld16(acc + c + 32u, next);
                        store(c, v);
                        if (c + 32u < cols) {
                            tmem_wait(next);
                            if (c + 64u < cols) tmem_ld16(acc + c + 64u, v);
                            store(c + 32u, next);
                        }
                    }
                } else {
                    for (uint32_t c = side * 16u; c < cols && ok; c += 32u) {
                        uint32_t v[16];
                        tmem_ld16(acc + c, v);
                        tmem_wait(v);
                        store(c, v);
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0 && ok) mbar_arrive_cluster(peer_addr(acc_empty(buf), CG == 2 ? 0u : rank));
            } else {
                // every CTA of the cluster has a part of each sum: CTA q adds up and stores the columns that are q modulo the CTAs
                const uint32_t mask = a.splits - 1u, log = 31u - __clz(a.splits), cols_each = a.tile >> log;
                const uint32_t slot = base + off_exchange + (part * cols_each * 128u + r) * 4u;
                bool ready = ok;
                if (a.in_ring && ok) {  // this CTA's mmas are done with its ring; the others'?
                    if (e < a.splits) mbar_arrive_cluster(peer_addr(ready_bar, e));
                    ready = __all_sync(0xFFFFFFFFu, wait_bar(ready_bar, 0u, abort_flag, a));
                }
                // (tiles of 16 columns: eight to either side)
                auto send = [&](uint32_t c, const uint32_t* v, uint32_t n) {
#pragma unroll
                    for (uint32_t j = 0; j < n; j++)
                        if (c + j < cols)
                            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(slot + ((c + j) >> log) * 512u, j & mask)), "r"(v[j]) : "memory");
                };
                if (a.tile == 16u) {
                    uint32_t v[8];
                    if (ready) tmem_ld8(acc + side * 8u, v), send(side * 8u, v, 8u);
                } else {
                    for (uint32_t c = side * 16u; c < cols && ready; c += 32u) {
                        uint32_t v[16];
                        tmem_ld16(acc + c, v);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        send(c, v, 16u);
                    }
                }
                asm volatile("fence.acq_rel.cluster;" ::: "memory");
                __syncwarp();
                if (lane < a.splits && ready) mbar_arrive_cluster(peer_addr(parts_bar, lane));
                const bool all = ready && wait_bar(parts_bar, 0u, abort_flag, a);
                const int* parts = reinterpret_cast<const int*>(base_ptr + off_exchange) + r;
                if (all && live) {
#pragma unroll 4
                    for (uint32_t c = side; part + (c << log) < cols; c += 2u) {
                        int sum = 0;
#pragma unroll
                        for (uint32_t p = 0; p < kMaxSplits; p++)
                            if (p < a.splits) sum += parts[(p * cols_each + c) * 128u];
                        const uint32_t m = part + (c << log);
                        Y[(uint64_t)(m0 + m) * a.ldy + n] = to_elem<T>(finish(sum, xscale[m], wscale, bias));
                    }
                }
            }
        }
    }
    __syncwarp();
    fence_before();
    if (group > 1u) cluster_sync_all();  // nothing crosses over any more
    else __syncthreads();
    if (*abort_flag) {  // (the same in the whole cluster)
        if (warp == 0 && lane == 0) {
            // A pair's copies are counted by the leader, whose barriers expect both halves of a step: whoever is behind issues as many
            // steps as the other, whatever is in them.  The stages are free: the one ahead has seen the pair's mmas done with them.
            const uint32_t steps = CG == 2 ? max(issued_steps[0], issued_steps[1]) : issued_steps[0];
            for (uint32_t i = issued_steps[half]; i < steps; i++) {
                const uint32_t s = i % a.stages, dst = base + s * sbytes, bar = (CG == 2 ? peer_addr(full(0), 0u) : full(0)) + s * 8u;
                if (leader) mbar_expect_tx(full(s), CG * sbytes);
                tma_load<CG>(dst, &a.tmap_w, 0u, 0u, bar);
                tma_load<CG>(dst + 128u * kStep, &a.tmap_x, 0u, 0u, bar);
            }
            if (leader)
                for (uint32_t i = steps > a.stages ? steps - a.stages : 0u; i < steps; i++) wait_in_flight(full(i % a.stages), (i / a.stages) & 1u);
        } else if (warp == 1 && lane == 0) {
            if (leader) umma_commit<CG>(done_bar);  // (of a pair: arrives in both)
            wait_in_flight(done_bar, 0u);
        }
        __syncwarp();
        if (group > 1u) cluster_sync_all();
        else __syncthreads();
    }
    if (warp == 2) {
        fence_after();
        if constexpr (CG == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
    }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = []() -> EncodeTiledFn {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            return nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}
bool encode_rows(CUtensorMap* map, const int8_t* codes, uint32_t rows, uint32_t K, uint32_t ld, uint32_t box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t gdim[2] = {K, rows}, gstride[1] = {ld};
    const cuuint32_t box[2] = {kStep, box_rows}, estr[2] = {1u, 1u};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(codes), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a product is cut: activation rows of a tile, tiles, CTAs that share a tile's K range.
struct Cut {
    uint32_t tile, m_tiles, splits;
    uint64_t tiles;
    double us;  // estimate of what differs between cuts
};
// An SM takes in about 92 GB/s (32 SMs streaming weights; 128 x 256 tiles of a pair), so a step costs what both operands' bytes of a
// stage do; a shared tile costs an exchange.  (128 x 4096 x 14336: a pair 33 us, four CTAs to a tile 17.7.)
constexpr uint32_t kSmem = 226u * 1024u;

// Clusters of `size` CTAs (one an SM) that the device runs at once: not every SM of every GPC finds partners.  0: none, or the
// question failed (which is asked again then).  The answer is the handle's: it depends on the context that is current.
uint32_t max_clusters(const MatmulI8Args& m, uint32_t size, int sm_count);

template <int CG>
Cut cut_of(const MatmulI8Args& m, int sm_count, bool clusters) {
    Cut c{};
    const uint32_t most = CG == 1 ? kMaxTile / 2u : kMaxTile, unit = CG * 16u;  // (the mma's step of N)
    c.m_tiles = (m.M + most - 1u) / most;
    c.tile = ((m.M + c.m_tiles - 1u) / c.m_tiles + unit - 1u) / unit * unit;
    c.m_tiles = (m.M + c.tile - 1u) / c.tile;
    c.tiles = (uint64_t)((m.N + CG * 128u - 1u) / (CG * 128u)) * c.m_tiles;
    c.splits = 1;
    const uint32_t chunks = (m.K + kStep - 1u) / kStep;
    if (CG == 1 && clusters)
        while (c.splits < kMaxSplits && c.tiles <= max_clusters(m, c.splits * 2u, sm_count) && chunks >= c.splits * 8u) c.splits *= 2u;
    const uint64_t groups = CG * c.splits == 1u ? (uint32_t)sm_count : max_clusters(m, CG * c.splits, sm_count);
    if (groups == 0) {  // (a context whose SMs have no partners)
        c.us = 1e30;
        return c;
    }
    const uint64_t rounds = (c.tiles + groups - 1u) / groups;
    c.us = (double)rounds * ((chunks + c.splits - 1u) / c.splits) * stage_bytes(c.tile, CG) / 92e3 + (c.splits > 1u ? 1.0 + 0.012 * c.tile : 0.0);
    return c;
}

uint32_t max_clusters(const MatmulI8Args& m, uint32_t size, int sm_count) {
    uint32_t& known = m.clusters->known[size == 2u ? 0 : size == 4u ? 1 : 2];  // (asked for once: a few calls a product)
    if (known) return known - 1u;
    static KernelConfig kcfg;
    const void* func = reinterpret_cast<const void*>(matmul_i8_kernel<1, float>);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((uint32_t)sm_count / size * size);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (kcfg.prepare(func, kThreads, kSmem, nullptr) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, func, &cfg) != cudaSuccess || n < 0) {
        cudaGetLastError();
        return 0;
    }
    known = (uint32_t)n + 1u;
    return (uint32_t)n;
}

template <int CG, typename T>
cudaError_t launch_tc(const MatmulI8Args& m, const Cut& cut, int sm_count, cudaStream_t stream) {
    TcArgs a{};
    a.xs = m.xs, a.ws = m.ws, a.bias = m.bias, a.Y = m.Y, a.M = m.M, a.N = m.N, a.ldy = m.ldy, a.status = m.status, a.wait_limit = m.wait_polls ? m.wait_polls : kWaitLimit;
    a.chunks = (m.K + kStep - 1u) / kStep;
    if (cut.tiles > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    a.tile = cut.tile, a.m_tiles = cut.m_tiles, a.tiles = (uint32_t)cut.tiles, a.splits = cut.splits;
    const uint32_t group = CG == 2 ? 2u : a.splits;
    // (a shorter ring is faster where little else than weights is read: 1 x 128256 x 4096 79 us with 150 KB, 85 with 226)
    const uint32_t budget = a.tile <= 48u ? 150u * 1024u : kSmem;
    // room of its own for the exchange while it is small; else the ring's, for one more hand-shake
    const bool exchange = a.splits > 1u && a.tile <= 48u;
    a.in_ring = a.splits > 1u && !exchange;
    a.stages = (budget - smem_bytes(0, a.tile, CG, exchange)) / stage_bytes(a.tile, CG);
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    if (a.stages < 2u || smem_bytes(a.stages, a.tile, CG, exchange) <= 114u * 1024u || (a.in_ring && a.stages * stage_bytes(a.tile, CG) < exchange_bytes(a.tile))) return cudaErrorInvalidValue;
    a.tmem_cols = 32;
    while (a.tmem_cols < (a.splits > 1u ? 1u : 2u) * a.tile) a.tmem_cols *= 2u;
    uint32_t groups = group == 1u ? (uint32_t)sm_count : max_clusters(m, group, sm_count);
    if (a.splits > 1u || groups > a.tiles) groups = a.tiles;  // (a shared tile is a cluster's only one)
    if (!encode_rows(&a.tmap_w, m.W, m.N, m.K, m.ldw, 128u) || !encode_rows(&a.tmap_x, m.X, m.M, m.K, m.ldx, a.tile / CG)) return cudaErrorInvalidValue;
    const uint32_t smem = smem_bytes(a.stages, a.tile, CG, exchange);
    static KernelConfig kcfg;
    if (cudaError_t e = kcfg.prepare(reinterpret_cast<const void*>(matmul_i8_kernel<CG, T>), kThreads, kSmem, nullptr)) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(groups * group);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = group, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = group > 1u ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, matmul_i8_kernel<CG, T>, a);
}

template <typename T>
cudaError_t launch_type(const MatmulI8Args& a, int sm_count, cudaStream_t stream) {
    if (a.M <= kStreamRows && (uint64_t)a.N * a.K <= 32u << 20) {
        // warps that share a row tile: as many as keep all warps on the machine at once (32 an SM) and leave each a fetch of its own
        const uint64_t tiles = (a.N + 15u) / 16u, fetches = (a.K + 255u) / 256u;
        uint32_t wk_log = 0;
        while (wk_log < 4u && tiles << (wk_log + 1u) <= 32u * (uint64_t)sm_count && fetches >> (wk_log + 1u)) wk_log++;
        return wk_log == 4u ? launch_stream<T, 16>(a, wk_log, stream) : launch_stream<T, 8>(a, wk_log, stream);
    }
    const Cut one = cut_of<1>(a, sm_count, true), pair = cut_of<2>(a, sm_count, true);
    // (of equals the one CTA form, which spreads over more SMs: 512 x 4096 x 4096 14.3 us, a pair 16.4)
    const bool single = one.us <= pair.us;
    cudaError_t e = single ? launch_tc<1, T>(a, one, sm_count, stream) : launch_tc<2, T>(a, pair, sm_count, stream);
    if (e != cudaSuccess && !(single && one.splits == 1u)) {  // another context than the one that was asked, which cannot place clusters
        cudaGetLastError();
        e = launch_tc<1, T>(a, cut_of<1>(a, sm_count, false), sm_count, stream);
    }
    return e;
}

}  // namespace

cudaError_t launch_matmul_i8(const MatmulI8Args& a, int ftype, int sm_count, cudaStream_t stream, int* launches) {
    if (a.M == 0 || a.N == 0) return cudaSuccess;
    ++*launches;
    switch (ftype) {
        case 0: return launch_type<float>(a, sm_count, stream);
        case 1: return launch_type<__half>(a, sm_count, stream);
        case 30: return launch_type<__nv_bfloat16>(a, sm_count, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace bpq4k
