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
    double per;      // 1 / hidden
};

// 1 / sqrt(sum / hidden + eps), rounded to f32 once: the root's first bits from rsqrt.approx, then two steps of Newton's method in 64 bits (2^-50 off).  (A division and a root in 64 bits took a third of the kernel's
// instructions.)
__device__ __forceinline__ float gated_rstd(double sum, double per, float eps) {
    const double x = fma(sum, per, (double)eps);
    double r;
    asm("rsqrt.approx.ftz.f64 %0, %1;" : "=d"(r) : "d"(x));
    if (!(x > 1e-300 && x < 1e300)) return (float)(1.0 / sqrt(x));
    const double h = 0.5 * x;
    r = r * fma(-h * r, r, 1.5);
    r = r * fma(-h * r, r, 1.5);
    return (float)r;
}
// Rows of any alignment: a block per row, which stays in registers where V blocks have its length (V > 0), element by element; longer ones (V = 0) in the sum's place, each element by the thread that wrote it.
template <typename T, int V> __global__ void __launch_bounds__(1024) add_gated_norm_row_kernel(const GatedNormArgs a) {
    before();
    __shared__ double s_sum[32], s_sum2[32];
    __shared__ uint32_t s_max[32];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, step = blockDim.x;
    const T *y = reinterpret_cast<const T*>(a.y) + row * a.top * a.ldy, *res = reinterpret_cast<const T*>(a.residual) + row * a.ldr;
    const T* gate = a.gate ? reinterpret_cast<const T*>(a.gate) + row * a.gate_row : nullptr;
    T* sum = reinterpret_cast<T*>(a.sum) + row * a.lds;
    constexpr int N = V > 0 ? V : 1;
    float r[N];
    // every element of this thread, with its place in r and whether it is one (a place behind the last is read as the last, so that loads need no branch)
    auto each = [&](auto&& f) {
        if constexpr (V > 0) {
#pragma unroll
            for (int v = 0; v < V; v++) f(min(v * step + tid, a.hidden - 1), r[v], v * step + tid < a.hidden);
        } else {
            for (int i = tid; i < a.hidden; i += step) f(i, r[0], true);
        }
    };
    auto mixed = [&](int i) {
        if (!a.mix) return to_f(y[i]);
        float m = __fmul_rn(a.mix[row * a.top], to_f(y[i]));
        for (int j = 1; j < a.top; j++) m = __fadd_rn(m, __fmul_rn(a.mix[row * a.top + j], to_f(y[j * a.ldy + i])));
        return m;
    };
    float post = 1;
    if (a.post_weight) {
        double ss = 0;
        if (V > 0) each([&](int i, float& x, bool) { x = mixed(i); });
        each([&](int i, float& x, bool there) {
            if (V == 0) x = mixed(i);
            ss += there ? (double)x * x : 0.0;
        });
        post = gated_rstd(block_sum(ss, s_sum), a.per, a.eps);
    }
    double ss = 0;
    if (V > 0 && !a.post_weight) each([&](int i, float& x, bool) { x = mixed(i); });
    each([&](int i, float& x, bool there) {
        if (V == 0) x = mixed(i);
        if (a.post_weight) x = __fmul_rn(__fmul_rn(x, post), a.post_weight[i]);
        if (gate) x = __fmul_rn(x, to_f(gate[i * a.gate_col]));
        const T t = from_f<T>(__fadd_rn(there ? to_f(res[i]) : 0.0f, __fmul_rn(x, a.scale)));      // (sum may be residual: no thread reads another's element)
        if (there) sum[i] = t;
        x = to_f(t);
        ss += there ? (double)x * x : 0.0;
    });
    if (!a.weight) return;
    const float rstd = gated_rstd(block_sum(ss, s_sum2), a.per, a.eps);
    float top = 0;
    each([&](int i, float& x, bool there) {
        if (V == 0) x = to_f(sum[i]);
        x = __fmul_rn(__fmul_rn(x, rstd), a.weight[i]);
        if (there) top = max_nan(top, fabsf(x));
    });
    const Q8Row q = q8_row(block_max(__float_as_uint(top), s_max));
    each([&](int i, float& x, bool there) {
        if (V == 0) x = __fmul_rn(__fmul_rn(to_f(sum[i]), rstd), a.weight[i]);
        if (there) a.q[row * a.ldq + i] = q.inv == 0.0f ? (int8_t)0 : (int8_t)(__float_as_uint(__fadd_rn(__fmul_rn(x, q.inv), kRoundHere)) & 0xff);
    });
    if (tid == 0) a.scales[row] = q.scale;
}

// Rows of whole 16-byte words on 16 bytes: a block per row, which stays in registers (V words per thread) from its copy to shared memory on (cp.async: each thread reads what it has copied itself, when it needs it).  With one word per thread
// both weights are asked for at once and kept.  GATE: 0 none, 1 one number per row, 2 words (of this row, or of all rows).
// What bounds it: 64-bit sums (a conversion of each element for each norm), reductions, and the weights' bytes from L2 behind a sum that they do not need (2048 x 4096 bf16 with both norms and a gate per channel: 15.9 us by itself, 67 MB: 10.2
// at the measured rate; without the first norm 10.3).  Blocks that strode over the rows with the next row's words on their way took 18.4 and 12.5, with the weights asked for ahead of the sums (128 registers, half the blocks) 18.8.
template <typename T, int V, int GATE, bool POST> __global__ void __launch_bounds__(1024) add_gated_norm_kernel(const GatedNormArgs a) {
    before();
    constexpr int E = 16 / (int)sizeof(T);
    constexpr bool KEPT = V == 1;
    extern __shared__ uint4 gated_words[];      // [y, residual, gate][V][threads]
    __shared__ double s_sum[2][32];
    __shared__ uint32_t s_max[32];
    const int words = a.hidden / E, tid = threadIdx.x, step = blockDim.x;
    const uint4* mine = gated_words + tid;
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(mine);
    const int64_t row = blockIdx.x;
    const uint4 *res = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.residual) + row * a.ldr) + tid, *y = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.y) + row * a.top * a.ldy) + tid,
                *gate = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.gate) + row * a.gate_row) + tid;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const bool there = v * step + tid < words;
        copy_where<16>(to + v * step * 16, there ? y + v * step : a.y, there);
        copy_where<16>(to + (V + v) * step * 16, there ? res + v * step : a.y, there);
        if (GATE == 2) copy_where<16>(to + (2 * V + v) * step * 16, there ? gate + v * step : a.y, there);
    }
    float pw[KEPT ? E : 1], nw[KEPT ? E : 1];
    if constexpr (KEPT)
        if (tid < words) {
            if constexpr (POST) load_n<float, E, true>(a.post_weight + tid * E, pw);
            if (a.weight) load_n<float, E, true>(a.weight + tid * E, nw);
        }
    const float one = GATE == 1 ? to_f(reinterpret_cast<const T*>(a.gate)[row * a.gate_row]) : 1.0f;
    float r[V][E];
    const float* mix = a.mix ? a.mix + row * a.top : nullptr;
    const float m0 = mix ? mix[0] : 1.0f;
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int v = 0; v < V; v++) {
        const uint4 w = mine[v * step];
#pragma unroll
        for (int e = 0; e < E; e++) r[v][e] = to_f(reinterpret_cast<const T*>(&w)[e]);
    }
    if (mix) {
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int e = 0; e < E; e++) r[v][e] = __fmul_rn(m0, r[v][e]);
    }
    for (int j = 1; j < a.top; j++) {
        const float m = mix[j];
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.y) + (row * a.top + j) * a.ldy);
        uint4 w[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = v * step + tid;
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
        const float post = gated_rstd(block_sum(ss, s_sum[0]), a.per, a.eps);
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = v * step + tid;
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
        const int i = v * step + tid;
        uint4 d = mine[(V + v) * step];
        const uint4 h = GATE == 2 ? mine[(2 * V + v) * step] : make_uint4(0, 0, 0, 0);
        T* p = reinterpret_cast<T*>(&d);
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (GATE == 1) r[v][e] = __fmul_rn(r[v][e], one);
            if (GATE == 2) r[v][e] = __fmul_rn(r[v][e], to_f(reinterpret_cast<const T*>(&h)[e]));
            p[e] = from_f<T>(__fadd_rn(to_f(p[e]), __fmul_rn(r[v][e], a.scale)));
            r[v][e] = to_f(p[e]);
            ss += std::is_same<T, __half>::value ? (double)(r[v][e] * r[v][e]) : (double)r[v][e] * r[v][e];      // (squares of f16 are exact in f32)
        }
        if (i < words) sum[i] = d;
    }
    if (!a.weight) return;
    const float rstd = gated_rstd(block_sum(ss, s_sum[1]), a.per, a.eps);
    float top = 0;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int i = v * step + tid;
        if (i < words) {
            float g[E];
            if constexpr (!KEPT) load_n<float, E, true>(a.weight + i * E, g);
#pragma unroll
            for (int e = 0; e < E; e++) {
                r[v][e] = __fmul_rn(__fmul_rn(r[v][e], rstd), KEPT ? nw[KEPT ? e : 0] : g[e]);
                top = max_nan(top, fabsf(r[v][e]));
            }
        }
    }
    const Q8Row q = q8_row(block_max(__float_as_uint(top), s_max));
    int8_t* out = a.q + row * a.ldq;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int i = v * step + tid;
        if (i < words) store_q8<E>(out + i * E, r[v], q.inv);
    }
    if (tid == 0) a.scales[row] = q.scale;
}

template <typename T, int V> cudaError_t add_gated_norm_words(const GatedNormArgs& a, int threads, cudaStream_t st) {
    const int gate = !a.gate ? 0 : a.gate_col == 0 ? 1 : 2;
    const dim3 grid((unsigned)a.rows);
    const size_t most = V * 1024 * 48, smem = V * threads * (gate == 2 ? 48 : 32);
    if (a.post_weight)
        return gate == 0   ? launch_with<add_gated_norm_kernel<T, V, 0, true>>(most, grid, threads, smem, st, a)
               : gate == 1 ? launch_with<add_gated_norm_kernel<T, V, 1, true>>(most, grid, threads, smem, st, a)
                           : launch_with<add_gated_norm_kernel<T, V, 2, true>>(most, grid, threads, smem, st, a);
    return gate == 0   ? launch_with<add_gated_norm_kernel<T, V, 0, false>>(most, grid, threads, smem, st, a)
           : gate == 1 ? launch_with<add_gated_norm_kernel<T, V, 1, false>>(most, grid, threads, smem, st, a)
                       : launch_with<add_gated_norm_kernel<T, V, 2, false>>(most, grid, threads, smem, st, a);
}
// Few rows: as many threads as a row has words, up to 1024 (latency).  Many rows: four words per thread, so that several blocks of an SM (its 65 536 registers hold 1024 threads) cover one another's barriers, and the sums over
// a block take fewer instructions.
template <typename T> cudaError_t add_gated_norm(const GatedNormArgs& a, cudaStream_t st) {
    constexpr int E = 16 / (int)sizeof(T);
    auto off = [](const void* p, int64_t ld, int bytes, int size) { return reinterpret_cast<uintptr_t>(p) % bytes || ld * size % bytes; };
    const bool words = a.hidden % E == 0 && a.hidden / E <= 4096 && !off(a.y, a.ldy, 16, sizeof(T)) && !off(a.residual, a.ldr, 16, sizeof(T)) && !off(a.sum, a.lds, 16, sizeof(T)) &&
                       (!a.post_weight || !off(a.post_weight, 0, 16, 4)) && (!a.weight || (!off(a.weight, 0, 16, 4) && !off(a.q, a.ldq, E, 1))) &&
                       (!a.gate || a.gate_col == 0 || (a.gate_col == 1 && !off(a.gate, a.gate_row, 16, sizeof(T))));
    if (!words) {
        auto go = [&](auto kernel, int v) { return launch(kernel, dim3((unsigned)a.rows), ((a.hidden + v - 1) / v + 31) / 32 * 32, 0, 1, st, a); };
        return a.hidden <= 1024 ? go(add_gated_norm_row_kernel<T, 4>, 4) : a.hidden <= 16384 ? go(add_gated_norm_row_kernel<T, 16>, 16) : launch(add_gated_norm_row_kernel<T, 0>, dim3((unsigned)a.rows), 1024, 0, 1, st, a);
    }
    int sms = 0;
    const cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    const int n = a.hidden / E, many = a.rows > 2 * sms, v = n > 2048 || (many && n >= 256) ? 4 : n > 1024 || (many && n >= 64) ? 2 : 1, threads = ((n + v - 1) / v + 31) / 32 * 32;
    return v == 4 ? add_gated_norm_words<T, 4>(a, threads, st) : v == 2 ? add_gated_norm_words<T, 2>(a, threads, st) : add_gated_norm_words<T, 1>(a, threads, st);
}

}  // namespace dev
