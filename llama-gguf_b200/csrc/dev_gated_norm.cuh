// dev_gated_norm.cuh — a block's output onto the residual stream and the next norm's rows in 8 bits (b200_dev_add_gated_norm_q8).
//
// m = y, or the sum over j of mix[j] * y[j] (in that order, products and sums rounded to f32); p = m * rstd(m) * post_weight, or m; r = residual + scale * (p * gate), every product and the sum in f32, r
// rounded to the type; q, scales = the RMS norm of r times weight in 8 bits, as add_rms_norm_q8 makes it.
#pragma once
#include <algorithm>

#include "dev_norm_q8.cuh"

namespace dev {

struct GatedNormArgs {
    const void *y, *residual, *gate;
    void* sum;
    const float *mix, *post_weight, *weight;
    int8_t* q;
    float* scales;
    int64_t ldy, ldr, lds, ldq, gate_row, gate_col, rows;
    int hidden, top;      // rows of y per row (mix)
    float scale, eps;
};

// Rows of any length and alignment: a block per row; what it makes of a row is kept in the sum's place.
template <typename T> __global__ void __launch_bounds__(256) add_gated_norm_any_kernel(const GatedNormArgs a) {
    before();
    __shared__ double s_sum[32], s_sum2[32];
    __shared__ uint32_t s_max[32];
    const int64_t row = blockIdx.x;
    const T *y = reinterpret_cast<const T*>(a.y) + row * a.top * a.ldy, *res = reinterpret_cast<const T*>(a.residual) + row * a.ldr;
    const T* gate = a.gate ? reinterpret_cast<const T*>(a.gate) + row * a.gate_row : nullptr;
    T* sum = reinterpret_cast<T*>(a.sum) + row * a.lds;
    auto mixed = [&](int i) {
        if (!a.mix) return to_f(y[i]);
        float m = __fmul_rn(a.mix[row * a.top], to_f(y[i]));
        for (int j = 1; j < a.top; j++) m = __fadd_rn(m, __fmul_rn(a.mix[row * a.top + j], to_f(y[j * a.ldy + i])));
        return m;
    };
    float post = 1;
    if (a.post_weight) {
        double ss = 0;
        for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
            const double m = mixed(i);
            ss += m * m;
        }
        post = q8_rstd(block_sum(ss, s_sum), a.hidden, a.eps);
    }
    double ss = 0;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        float p = mixed(i);
        if (a.post_weight) p = __fmul_rn(__fmul_rn(p, post), a.post_weight[i]);
        if (gate) p = __fmul_rn(p, to_f(gate[i * a.gate_col]));
        const T r = from_f<T>(__fadd_rn(to_f(res[i]), __fmul_rn(p, a.scale)));
        sum[i] = r;
        ss += (double)to_f(r) * to_f(r);
    }
    if (!a.weight) return;
    const float rstd = q8_rstd(block_sum(ss, s_sum2), a.hidden, a.eps);
    uint32_t top = 0;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) top = max(top, __float_as_uint(fabsf(__fmul_rn(__fmul_rn(to_f(sum[i]), rstd), a.weight[i]))));
    const Q8Row q = q8_row(block_max(top, s_max));
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x)
        a.q[row * a.ldq + i] = q.inv == 0.0f ? (int8_t)0 : (int8_t)__float2int_rn(__fmul_rn(__fmul_rn(__fmul_rn(to_f(sum[i]), rstd), a.weight[i]), q.inv));
    if (threadIdx.x == 0) a.scales[row] = q.scale;
}

template <typename T> cudaError_t add_gated_norm(const GatedNormArgs& a, cudaStream_t st) { return launch(add_gated_norm_any_kernel<T>, dim3((unsigned)a.rows), 256, 0, 1, st, a); }

}  // namespace dev
