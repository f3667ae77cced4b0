// dev_common.cuh — what the operators on device tensors (device_ops.cu) share: element types, the 4-bit cache's layout, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

}  // namespace dev
