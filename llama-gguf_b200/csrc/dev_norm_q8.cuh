// dev_norm_q8.cuh — RMS norm of a residual sum with the result in 8 bits and a scale per row (b200_dev_add_rms_norm_q8).
#pragma once
#include "dev_common.cuh"

namespace dev {

struct NormQ8Args {
    const void *x, *residual;
    void* sum;
    const float* weight;
    int8_t* q;
    float* scales;
    int64_t ldx, ldr, lds, ldq, rows;
    int hidden;
    float eps;
};

// sum over the block of a double and maximum of an unsigned word; `s`: one word per warp
__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (blockDim.x == 32) return v;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < (int)blockDim.x / 32; i++) v += s[i];
    return v;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* s) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (blockDim.x == 32) return v;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < (int)blockDim.x / 32; i++) v = max(v, s[i]);
    return v;
}

// Rows of any length and alignment: a block per row, which is read once per step (sum of squares, maximum, result); the sum is read back where it was written, each element by the
// thread that wrote it.
template <typename T> __global__ void __launch_bounds__(256) add_rms_norm_q8_any_kernel(const NormQ8Args a) {
    __shared__ double s_sum[32];
    __shared__ uint32_t s_max[32];
    const int64_t row = blockIdx.x;
    const T *x = reinterpret_cast<const T*>(a.x) + row * a.ldx, *res = a.residual ? reinterpret_cast<const T*>(a.residual) + row * a.ldr : nullptr;
    T* sum = a.residual ? reinterpret_cast<T*>(a.sum) + row * a.lds : nullptr;
    double ss = 0;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        float r = to_f(x[i]);
        if (res) {
            const T t = from_f<T>(r + to_f(res[i]));
            sum[i] = t;
            r = to_f(t);
        }
        ss += (double)r * r;
    }
    const float rstd = (float)(1.0 / sqrt(block_sum(ss, s_sum) / a.hidden + (double)a.eps));
    const T* r = res ? sum : x;
    uint32_t top = 0;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) top = max(top, __float_as_uint(fabsf(__fmul_rn(__fmul_rn(to_f(r[i]), rstd), a.weight[i]))));
    top = block_max(top, s_max);
    const float m = __uint_as_float(top);
    const bool live = top < kInfBits && m >= kTiny;
    const float inv = live ? __fdiv_rn(127.0f, m) : 0.0f;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x)
        a.q[row * a.ldq + i] = live ? (int8_t)__float2int_rn(__fmul_rn(__fmul_rn(__fmul_rn(to_f(r[i]), rstd), a.weight[i]), inv)) : (int8_t)0;
    if (threadIdx.x == 0) a.scales[row] = top >= kInfBits ? __uint_as_float(0x7fffffffu) : live ? __fdiv_rn(m, 127.0f) : 0.0f;
}

template <typename T> cudaError_t add_rms_norm_q8(const NormQ8Args& a, cudaStream_t st) {
    add_rms_norm_q8_any_kernel<T><<<(unsigned)a.rows, 256, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace dev
