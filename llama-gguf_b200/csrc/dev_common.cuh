// dev_common.cuh — what the operators on device tensors (device_ops.cu) share: element types, the 4-bit cache's layout, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/llama_b200.h"

namespace dev {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements at p as f32 / f32 to N elements; VEC: p is on 16 bytes (on N elements where those are fewer) and they go as words
template <typename T, int N, bool VEC> __device__ __forceinline__ void load_n(const T* p, float (&f)[N]) {
    if constexpr (VEC) {
        constexpr int B = N * (int)sizeof(T) < 16 ? N * (int)sizeof(T) : 16, E = B / (int)sizeof(T);
        struct __align__(B) W { T v[E]; };
#pragma unroll
        for (int i = 0; i < N / E; i++) {
            const W w = reinterpret_cast<const W*>(p)[i];
#pragma unroll
            for (int j = 0; j < E; j++) f[i * E + j] = to_f(w.v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = to_f(p[i]);
    }
}
template <typename T, int N, bool VEC> __device__ __forceinline__ void store_n(T* p, const float (&f)[N]) {
    if constexpr (VEC) {
        constexpr int B = N * (int)sizeof(T) < 16 ? N * (int)sizeof(T) : 16, E = B / (int)sizeof(T);
        struct __align__(B) W { T v[E]; };
#pragma unroll
        for (int i = 0; i < N / E; i++) {
            W w;
#pragma unroll
            for (int j = 0; j < E; j++) w.v[j] = from_f<T>(f[i * E + j]);
            reinterpret_cast<W*>(p)[i] = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = from_f<T>(f[i]);
    }
}

__device__ __forceinline__ float max_nan(float a, float b) {      // NaN where either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// magnitudes below this count as zero, so that 1 / scale and 127 / magnitude stay finite
constexpr float kTiny = 1.504632769052528e-36f;      // 2^-119
constexpr uint32_t kInfBits = 0x7f800000u;

// one kv head's block of a page (include/llama_b200.h, b200_q4_pages)
struct Q4Block {
    const uint8_t *k, *v;
    const float *ks, *vs;
};
__device__ __forceinline__ Q4Block q4_block(const b200_q4_pages& c, int64_t page, int head) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(c.data) + (page * c.n_kv_heads + head) * ((int64_t)c.page_size * (c.head_dim + 8));
    const int rows = c.page_size * c.head_dim / 2;
    return Q4Block{p, p + rows, reinterpret_cast<const float*>(p + 2 * rows), reinterpret_cast<const float*>(p + 2 * rows) + c.page_size};
}

// 16 or 8 bytes to shared memory
template <int N> __device__ __forceinline__ void copy_all(uint32_t to, const void* from) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(N) : "memory");
}
// ... zeros where `there` is not set (the address is a valid one all the same)
template <int N> __device__ __forceinline__ void copy_where(uint32_t to, const void* from, bool there) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(N), "r"(there ? N : 0) : "memory");
}

// Clusters: barriers, and what lies in another block's shared memory
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
    uint32_t p;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(addr), "r"(rank));
    return p;
}
__device__ __forceinline__ int peer_s32(uint32_t addr, uint32_t rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at_rank(addr, rank)));      // (behind a barrier: nothing to be ordered with)
    return v;
}
__device__ __forceinline__ float4 peer_f32x4(uint32_t addr, uint32_t rank) {      // (a block without a cluster is rank 0 of its own)
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at_rank(addr, rank)) : "memory");
    return v;
}

// Programmatic launches: a kernel may be scheduled while the one before it on the stream ends.  Every block of every kernel here calls before() first thing, ahead of any access to global memory (it
// returns when all that came before is done and visible), and so no kernel can end before its predecessors have.
__device__ __forceinline__ void before() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... P, typename... A> cudaError_t launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, int cluster, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// SMs of the current device (asked for once per device, of 64 devices)
inline cudaError_t sm_count(int* sms) {
    static std::atomic<int> known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    *sms = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
    if (*sms) return cudaSuccess;
    e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess && dev < 64) known[dev].store(*sms, std::memory_order_relaxed);
    return e;
}
// A kernel's dynamic shared memory is allowed once per device (64 devices; further ones ask every time).  One per kernel, by its address.
struct SmemAllowed {
    std::atomic<uint64_t> done{0};
    cudaError_t operator()(const void* kernel, size_t bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
        if (bit && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
        return e;
    }
};
// a launch of KERNEL, which is allowed up to `most` bytes of dynamic shared memory
template <auto KERNEL, typename A> cudaError_t launch_with(size_t most, dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const A& a) {
    static SmemAllowed allowed;
    const cudaError_t e = allowed(reinterpret_cast<const void*>(KERNEL), most);
    return e != cudaSuccess ? e : launch(KERNEL, grid, threads, smem, 1, st, a);
}

}  // namespace dev
