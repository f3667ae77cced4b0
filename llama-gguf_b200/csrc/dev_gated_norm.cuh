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

// Rows of whole 16-byte words on 16 bytes: blocks stride over the rows; a row stays in registers (V words per thread) from its loads on, the next one's words are asked for before this one's sums, and with one word per
// thread both weights are kept.  GATE: 0 none, 1 one number per row, 2 words (of this row, or of all rows).
template <typename T, int V, int GATE, bool POST> __global__ void __launch_bounds__(1024) add_gated_norm_kernel(const GatedNormArgs a) {
    before();
    constexpr int E = 16 / (int)sizeof(T);
    constexpr bool AHEAD = V < 4, KEPT = V == 1;
    __shared__ double s_sum[2][32];
    __shared__ uint32_t s_max[32];
    const int words = a.hidden / E, tid = threadIdx.x;
    uint4 d[V], w[V], h[V];
    auto load = [&](int64_t row) {
        const uint4 *res = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.residual) + row * a.ldr), *y = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.y) + row * a.top * a.ldy),
                    *gate = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.gate) + row * a.gate_row);
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = v * blockDim.x + tid;
            w[v] = i < words ? y[i] : make_uint4(0, 0, 0, 0);
            d[v] = i < words ? res[i] : make_uint4(0, 0, 0, 0);
            if (GATE == 2) h[v] = i < words ? gate[i] : make_uint4(0, 0, 0, 0);
        }
    };
    float pw[KEPT ? E : 1], nw[KEPT ? E : 1];
    if constexpr (KEPT)
        if (tid < words) {
            if constexpr (POST) load_n<float, E, true>(a.post_weight + tid * E, pw);
            if (a.weight) load_n<float, E, true>(a.weight + tid * E, nw);
        }
    if (AHEAD) load(blockIdx.x);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (!AHEAD) load(row);
        const float one = GATE == 1 ? to_f(reinterpret_cast<const T*>(a.gate)[row * a.gate_row]) : 1.0f;
        float r[V][E];
        const float* mix = a.mix ? a.mix + row * a.top : nullptr;
        const float m0 = mix ? mix[0] : 1.0f;
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int e = 0; e < E; e++) r[v][e] = __fmul_rn(m0, to_f(reinterpret_cast<const T*>(&w[v])[e]));      // (by one: nothing changes)
        for (int j = 1; j < a.top; j++) {
            const float m = mix[j];
            const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.y) + (row * a.top + j) * a.ldy);
#pragma unroll
            for (int v = 0; v < V; v++) {
                const int i = v * blockDim.x + tid;
                w[v] = i < words ? p[i] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int e = 0; e < E; e++) r[v][e] = __fadd_rn(r[v][e], __fmul_rn(m, to_f(reinterpret_cast<const T*>(&w[v])[e])));
        }
        if constexpr (POST) {
            double ss = 0;
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int e = 0; e < E; e++) ss += (double)r[v][e] * r[v][e];
            const float post = q8_rstd(block_sum(ss, s_sum[0]), a.hidden, a.eps);
#pragma unroll
            for (int v = 0; v < V; v++) {
                const int i = v * blockDim.x + tid;
                if (i < words) {
                    float g[E];
                    if constexpr (!KEPT) load_n<float, E, true>(a.post_weight + i * E, g);
#pragma unroll
                    for (int e = 0; e < E; e++) r[v][e] = __fmul_rn(__fmul_rn(r[v][e], post), KEPT ? pw[KEPT ? e : 0] : g[e]);
                }
            }
        }
        uint4* sum = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.sum) + row * a.lds);
        double ss = 0;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = v * blockDim.x + tid;
            T* p = reinterpret_cast<T*>(&d[v]);
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (GATE == 1) r[v][e] = __fmul_rn(r[v][e], one);
                if (GATE == 2) r[v][e] = __fmul_rn(r[v][e], to_f(reinterpret_cast<const T*>(&h[v])[e]));
                p[e] = from_f<T>(__fadd_rn(to_f(p[e]), __fmul_rn(r[v][e], a.scale)));
                r[v][e] = to_f(p[e]);
                ss += std::is_same<T, __half>::value ? (double)(r[v][e] * r[v][e]) : (double)r[v][e] * r[v][e];      // (squares of f16 are exact in f32)
            }
            if (i < words) sum[i] = d[v];
        }
        if (AHEAD && row + gridDim.x < a.rows) load(row + gridDim.x);      // (sum may be residual: other rows)
        if (!a.weight) {
            if (POST) __syncthreads();      // (the next row writes what this one's sums are read from)
            continue;
        }
        const float rstd = q8_rstd(block_sum(ss, s_sum[1]), a.hidden, a.eps);
        uint32_t top = 0;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = v * blockDim.x + tid;
            if (i < words) {
                float g[E];
                if constexpr (!KEPT) load_n<float, E, true>(a.weight + i * E, g);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    r[v][e] = __fmul_rn(__fmul_rn(r[v][e], rstd), KEPT ? nw[KEPT ? e : 0] : g[e]);
                    top = max(top, __float_as_uint(fabsf(r[v][e])));
                }
            }
        }
        const Q8Row q = q8_row(block_max(top, s_max));
        int8_t* out = a.q + row * a.ldq;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = v * blockDim.x + tid;
            if (i < words) store_q8<E>(out + i * E, r[v], q.inv);
        }
        if (tid == 0) a.scales[row] = q.scale;
    }
}

template <typename T, int V> cudaError_t add_gated_norm_words(const GatedNormArgs& a, int threads, int blocks, cudaStream_t st) {
    auto go = [&](auto kernel) { return launch(kernel, dim3((unsigned)std::min<int64_t>(a.rows, blocks)), threads, 0, 1, st, a); };
    const int gate = !a.gate ? 0 : a.gate_col == 0 ? 1 : 2;
    if (a.post_weight) return gate == 0 ? go(add_gated_norm_kernel<T, V, 0, true>) : gate == 1 ? go(add_gated_norm_kernel<T, V, 1, true>) : go(add_gated_norm_kernel<T, V, 2, true>);
    return gate == 0 ? go(add_gated_norm_kernel<T, V, 0, false>) : gate == 1 ? go(add_gated_norm_kernel<T, V, 1, false>) : go(add_gated_norm_kernel<T, V, 2, false>);
}
// As many threads as a row has words, up to 1024; the SMs' 65 536 registers hold 1024 threads.
template <typename T> cudaError_t add_gated_norm(const GatedNormArgs& a, cudaStream_t st) {
    constexpr int E = 16 / (int)sizeof(T);
    auto off = [](const void* p, int64_t ld, int bytes, int size) { return reinterpret_cast<uintptr_t>(p) % bytes || ld * size % bytes; };
    const bool words = a.hidden % E == 0 && a.hidden / E <= 4096 && !off(a.y, a.ldy, 16, sizeof(T)) && !off(a.residual, a.ldr, 16, sizeof(T)) && !off(a.sum, a.lds, 16, sizeof(T)) &&
                       (!a.post_weight || !off(a.post_weight, 0, 16, 4)) && (!a.weight || (!off(a.weight, 0, 16, 4) && !off(a.q, a.ldq, E, 1))) &&
                       (!a.gate || a.gate_col == 0 || (a.gate_col == 1 && !off(a.gate, a.gate_row, 16, sizeof(T))));
    if (!words) return launch(add_gated_norm_any_kernel<T>, dim3((unsigned)a.rows), 256, 0, 1, st, a);
    int sms = 0;
    const cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    const int n = a.hidden / E, v = n > 2048 ? 4 : n > 1024 ? 2 : 1, threads = ((n + v - 1) / v + 31) / 32 * 32, blocks = sms * std::max(1, 1024 / threads);
    return v == 4 ? add_gated_norm_words<T, 4>(a, threads, blocks, st) : v == 2 ? add_gated_norm_words<T, 2>(a, threads, blocks, st) : add_gated_norm_words<T, 1>(a, threads, blocks, st);
}

}  // namespace dev
