// dev_glu_q8.cuh — gated unit of a row's two halves with the result in 8 bits and a scale per row (b200_dev_glu_q8).
//
// y = act(g) * u; scale = max |y| / 127; q = round(y * 127 / max |y|), halves to even, all of it as if y were exact: it is made in f32, and again in 64 bits where that could decide otherwise (the
// largest value of the row, and what lies next to the border between two numbers).
#pragma once
#include <algorithm>

#include "dev_norm_q8.cuh"

namespace dev {

enum { GLU_SILU = 0, GLU_GELU = 1, GLU_RELU = 2 };

struct GluQ8Args {
    const void* x;
    int8_t* q;
    float* scales;
    int64_t ldx, ldq, rows;
    int ff, act;
};

__device__ __noinline__ double glu_exact(float gate, float up, int act) {
    const double g = gate;
    const double z = act == GLU_GELU ? 1.5957691216057308 * (g + 0.044715 * g * g * g) : g;      // 0.5 (1 + tanh(z)) is 1 / (1 + exp(-2 z))
    return (act == GLU_RELU ? (isnan(g) ? g : fmax(g, 0.0)) : g / (1.0 + exp(-z))) * up;
}

// largest of the block of values that are not negative
__device__ __forceinline__ double block_max_double(double v, double* s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (blockDim.x == 32) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (int)blockDim.x / 32 ? s[lane] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// A block per row, read twice, everything in 64 bits.
template <typename T> __global__ void __launch_bounds__(256) glu_q8_any_kernel(const GluQ8Args a) {
    before();
    __shared__ double s_max[32];
    const int64_t row = blockIdx.x;
    const T *g = reinterpret_cast<const T*>(a.x) + row * a.ldx, *u = g + a.ff;
    double top = 0;
    bool bad = false;
    for (int i = threadIdx.x; i < a.ff; i += blockDim.x) {
        const double y = glu_exact(to_f(g[i]), to_f(u[i]), a.act);
        bad |= !isfinite(y);
        top = fmax(top, fabs(y));
    }
    if (bad) top = INFINITY;
    top = block_max_double(top, s_max);
    const bool live = top >= (double)kTiny && top < INFINITY;
    const double inv = live ? 127.0 / top : 0.0;
    for (int i = threadIdx.x; i < a.ff; i += blockDim.x) a.q[row * a.ldq + i] = live ? (int8_t)__double2int_rn(glu_exact(to_f(g[i]), to_f(u[i]), a.act) * inv) : (int8_t)0;
    if (threadIdx.x == 0) a.scales[row] = top == INFINITY ? NAN : live ? (float)(top / 127.0) : 0.0f;
}

template <typename T> cudaError_t glu_q8(const GluQ8Args& a, cudaStream_t st) { return launch(glu_q8_any_kernel<T>, dim3((unsigned)a.rows), 256, 0, 1, st, a); }

}  // namespace dev
