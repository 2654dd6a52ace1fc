// A CUDA runtime that launches nothing: it writes down what would be launched, and refuses what the test says.  Linked with the
// objects of kernels whose host code (which kernel, which grid, what if a launch is refused) is tested without a GPU.
#include <cuda.h>
#include <cuda_runtime_api.h>

#include <cstring>
#include <map>
#include <string>
#include <vector>

#include "../backpack_b200/csrc/kernels.h"

namespace {
std::map<const void*, std::string>& names() {
    static std::map<const void*, std::string> m;
    return m;
}
struct Launch {
    std::string name;
    unsigned grid, block, cluster;
    bool refused;
};
std::vector<Launch> launches;
unsigned largest_cluster = 16;      // larger ones are refused
int cluster_error = 0;              // what the occupancy query returns
unsigned sms = 148;                 // that the occupancy query spreads clusters over
unsigned queries = 0;
cudaError_t last = cudaSuccess;

unsigned cluster_of(const cudaLaunchConfig_t* c) {
    for (unsigned i = 0; i < c->numAttrs; i++)
        if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) return c->attrs[i].val.clusterDim.x;
    return 1;
}
CUresult encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}
}  // namespace

extern "C" {
void** __cudaRegisterFatBinary(void*) {
    static void* handle;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char* host, char*, const char* name, int, uint3*, uint3*, dim3*, dim3*, int*) { names()[host] = name; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, void*) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* func, void**) {
    const unsigned cluster = cluster_of(c);
    const bool refused = cluster > largest_cluster;
    launches.push_back({names()[func], c->gridDim.x, c->blockDim.x, cluster, refused});
    return refused ? last = cudaErrorLaunchOutOfResources : cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaGetLastError() {
    const cudaError_t e = last;
    last = cudaSuccess;
    return e;
}
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t* c) {
    queries++;
    if (cluster_error) return last = (cudaError_t)cluster_error;
    const unsigned cluster = cluster_of(c);
    *n = cluster > largest_cluster ? 0 : (int)(sms / cluster);
    return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char*, void** p, unsigned long long, cudaDriverEntryPointQueryResult* q) {
    *p = reinterpret_cast<void*>(&encode);
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}

// ---- what the test calls ----
__attribute__((visibility("default"))) void fake_reset(unsigned largest, int error, unsigned sm) {
    launches.clear(), largest_cluster = largest, cluster_error = error, sms = sm, queries = 0, last = cudaSuccess;
}
__attribute__((visibility("default"))) int fake_count() { return (int)launches.size(); }
__attribute__((visibility("default"))) int fake_queries() { return (int)queries; }
__attribute__((visibility("default"))) int fake_last_error() { return (int)last; }
__attribute__((visibility("default"))) const char* fake_launch(int i, unsigned* out) {
    const Launch& l = launches[i];
    out[0] = l.grid, out[1] = l.block, out[2] = l.cluster, out[3] = l.refused;
    return l.name.c_str();
}
__attribute__((visibility("default"))) int fake_logprobs(int ftype, unsigned M, unsigned V, unsigned nTop, int sm_count) {
    bpq4k::LogprobsArgs a{};
    a.M = M, a.V = a.ld = V, a.nTop = nTop;
    return (int)bpq4k::launch_logprobs(a, ftype, sm_count, nullptr);
}
// One handle's products: what it knows of clusters is kept between the calls, or forgotten (a new handle).
__attribute__((visibility("default"))) int fake_matmul(int new_handle, int ftype, unsigned M, unsigned N, unsigned K, int sm_count) {
    static bpq4k::ClusterCounts handle;
    if (new_handle) handle = bpq4k::ClusterCounts();
    bpq4k::MatmulI8Args a{};
    a.M = M, a.N = N, a.K = K, a.ldx = a.ldw = (K + 15) / 16 * 16, a.ldy = N, a.clusters = &handle;
    int launched = 0;
    return (int)bpq4k::launch_matmul_i8(a, ftype, sm_count, nullptr, &launched);
}
}
