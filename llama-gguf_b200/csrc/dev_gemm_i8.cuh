// dev_gemm_i8.cuh — products of 8-bit integers with scales per token and per output channel (b200_dev_mat_mat_i8).
#pragma once
#include "dev_common.cuh"

namespace dev {

struct GemmI8Args {
    const int8_t *a, *w;
    const float *as, *ws, *bias;
    void* out;
    int64_t lda, ldw, ldo;
    int t, k, n;
};
template <typename T> __device__ __forceinline__ T i8_result(const GemmI8Args& g, int acc, float a_scale, float w_scale, float bias) {
    const float v = __fmul_rn(__fmul_rn((float)acc, a_scale), w_scale);
    return from_f<T>(g.bias ? __fadd_rn(v, bias) : v);
}

template <typename T> __global__ void __launch_bounds__(256) gemm_i8_plain_kernel(const GemmI8Args g) {
    const int n = blockIdx.x * 16 + (threadIdx.x & 15), t = blockIdx.y * 16 + (threadIdx.x >> 4);
    if (n >= g.n || t >= g.t) return;
    const int8_t *a = g.a + t * g.lda, *w = g.w + n * g.ldw;
    int acc = 0, k = 0;
    for (; k + 4 <= g.k; k += 4) acc = __dp4a(*reinterpret_cast<const int*>(a + k), *reinterpret_cast<const int*>(w + k), acc);
    for (; k < g.k; k++) acc += (int)a[k] * (int)w[k];
    reinterpret_cast<T*>(g.out)[t * g.ldo + n] = i8_result<T>(g, acc, g.as[t], g.ws[n], g.bias ? g.bias[n] : 0.0f);
}

template <typename T> cudaError_t gemm_i8(const GemmI8Args& g, cudaStream_t st) {
    gemm_i8_plain_kernel<T><<<dim3((g.n + 15) / 16, (g.t + 15) / 16), 256, 0, st>>>(g);
    return cudaGetLastError();
}

}  // namespace dev
