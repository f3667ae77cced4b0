// dev_norm_q8.cuh — RMS norm of a residual sum with the result in 8 bits and a scale per row (b200_dev_add_rms_norm_q8).
#pragma once
#include <algorithm>
#include <type_traits>

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

// sum over the block of a double, and the maximum of an unsigned word; `s`: one word per warp
__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (blockDim.x == 32) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (int)blockDim.x / 32 ? s[lane] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* s) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (blockDim.x == 32) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, lane < (int)blockDim.x / 32 ? s[lane] : 0u);
}
__device__ __forceinline__ float q8_rstd(double sum, int hidden, float eps) { return (float)(1.0 / sqrt(sum / hidden + (double)eps)); }
// the row's scale and 127 / maximum (0: the row is zeros) from the bits of its maximum
struct Q8Row {
    float scale, inv;
};
__device__ __forceinline__ Q8Row q8_row(uint32_t top) {
    const float m = __uint_as_float(top);
    const bool live = top < kInfBits && m >= kTiny;
    return Q8Row{top >= kInfBits ? __uint_as_float(0x7fffffffu) : live ? __fdiv_rn(m, 127.0f) : 0.0f, live ? __fdiv_rn(127.0f, m) : 0.0f};
}

constexpr float kRoundHere = 12582912.0f;      // 1.5 * 2^23: the low bits of a sum with it are the other number (up to 2^22) rounded to an integer, halves to even
// the low bytes of E words at `out`, as a word of them
template <int E> __device__ __forceinline__ void store_bytes(int8_t* out, const uint32_t (&n)[E]) {
    uint32_t o[E / 4];
#pragma unroll
    for (int e = 0; e < E; e += 4) o[e / 4] = __byte_perm(__byte_perm(n[e], n[e + 1], 0x0040), __byte_perm(n[e + 2], n[e + 3], 0x0040), 0x5410);
    if constexpr (E == 8) *reinterpret_cast<uint2*>(out) = make_uint2(o[0], o[1]);
    else *reinterpret_cast<uint32_t*>(out) = o[0];
}
// E values times `inv` (at most 127 and its roundings) as 8-bit numbers (inv 0: zeros)
template <int E> __device__ __forceinline__ void store_q8(int8_t* out, const float (&y)[E], float inv) {
    uint32_t n[E] = {};
    if (inv != 0.0f) {
#pragma unroll
        for (int e = 0; e < E; e++) n[e] = __float_as_uint(__fadd_rn(__fmul_rn(y[e], inv), kRoundHere));
    }
    store_bytes<E>(out, n);
}

// Rows of whole 16-byte words on 16 bytes: a block per row, which stays in registers (V words per thread, asked for together) from its only load on.
// A square has twice its element's bits and exponent: f16's fits f32, bf16's passes its range both ways, so that one and f32's are made and added in 64 bits.  (A sum of them is rounded, and
// its order that of the kernel: at 2^-53 of the sum, which only a reciprocal root next to a border of f32 shows.)
template <typename T, int V> __global__ void __launch_bounds__(1024) add_rms_norm_q8_kernel(const NormQ8Args a) {
    before();
    constexpr int E = 16 / (int)sizeof(T);
    __shared__ double s_sum[32];
    __shared__ uint32_t s_max[32];
    const int64_t row = blockIdx.x;
    const int words = a.hidden / E;
    const uint4* x = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.x) + row * a.ldx);
    const uint4* res = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.residual) + row * a.ldr);
    uint4* sum = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.sum) + row * a.lds);
    uint4 w[V], d[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int i = v * blockDim.x + threadIdx.x;
        w[v] = i < words ? x[i] : make_uint4(0, 0, 0, 0);
        if (a.residual && i < words) d[v] = res[i];
    }
    float r[V][E];
    double ss = 0;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int i = v * blockDim.x + threadIdx.x;
        if (a.residual && i < words) {
            T *p = reinterpret_cast<T*>(&w[v]), *q = reinterpret_cast<T*>(&d[v]);
#pragma unroll
            for (int e = 0; e < E; e++) p[e] = from_f<T>(to_f(p[e]) + to_f(q[e]));
            sum[i] = w[v];
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
            r[v][e] = to_f(reinterpret_cast<T*>(&w[v])[e]);
            ss += std::is_same<T, __half>::value ? (double)(r[v][e] * r[v][e]) : (double)r[v][e] * r[v][e];
        }
    }
    const float rstd = q8_rstd(block_sum(ss, s_sum), a.hidden, a.eps);
    uint32_t top = 0;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int i = v * blockDim.x + threadIdx.x;
        if (i < words) {
            float g[E];
            load_n<float, E, true>(a.weight + i * E, g);
#pragma unroll
            for (int e = 0; e < E; e++) {
                r[v][e] = __fmul_rn(__fmul_rn(r[v][e], rstd), g[e]);
                top = max(top, __float_as_uint(fabsf(r[v][e])));
            }
        }
    }
    const Q8Row q = q8_row(block_max(top, s_max));
    int8_t* out = a.q + row * a.ldq;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int i = v * blockDim.x + threadIdx.x;
        if (i < words) store_q8<E>(out + i * E, r[v], q.inv);
    }
    if (threadIdx.x == 0) a.scales[row] = q.scale;
}

// Rows of any length and alignment: a block per row, which is read once per step (sum of squares, maximum, result); the sum is read back where it was written, each element by the
// thread that wrote it.
template <typename T> __global__ void __launch_bounds__(256) add_rms_norm_q8_any_kernel(const NormQ8Args a) {
    before();
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
    const float rstd = q8_rstd(block_sum(ss, s_sum), a.hidden, a.eps);
    const T* r = res ? sum : x;
    uint32_t top = 0;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) top = max(top, __float_as_uint(fabsf(__fmul_rn(__fmul_rn(to_f(r[i]), rstd), a.weight[i]))));
    const Q8Row q = q8_row(block_max(top, s_max));
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x)
        a.q[row * a.ldq + i] = q.inv == 0.0f ? (int8_t)0 : (int8_t)__float2int_rn(__fmul_rn(__fmul_rn(__fmul_rn(to_f(r[i]), rstd), a.weight[i]), q.inv));
    if (threadIdx.x == 0) a.scales[row] = q.scale;
}

template <typename T, int V> cudaError_t add_rms_norm_q8_words(const NormQ8Args& a, int threads, cudaStream_t st) {
    return launch(add_rms_norm_q8_kernel<T, V>, dim3((unsigned)a.rows), threads, 0, 1, st, a);
}
// Bound by the rows' bytes where there are many (2048 x 4096 bf16 with a residual: 58.7 MB in 15 us by itself, 13 among others), by the launch and two reductions where there are few (one row of 4096: 5 us by itself).
// A block per row with two reads of it took 42 and 22.
// Few rows: as many threads as the row has words, up to 1024 (one token of 4096 in bf16: latency).  Many rows: four words per thread, so that a block has fewer warps to wait for and the loads of a
// thread cover one another.  Rows of more than 4 x 1024 words do not fit the registers.
template <typename T> cudaError_t add_rms_norm_q8(const NormQ8Args& a, cudaStream_t st) {
    constexpr int E = 16 / (int)sizeof(T);
    auto off = [](const void* p, int64_t ld, int bytes, int size) { return reinterpret_cast<uintptr_t>(p) % bytes || ld * size % bytes; };
    const bool words = a.hidden % E == 0 && a.hidden / E <= 4096 && !off(a.x, a.ldx, 16, sizeof(T)) && !off(a.weight, 0, 16, 4) && !off(a.q, a.ldq, E, 1) &&
                       (!a.residual || (!off(a.residual, a.ldr, 16, sizeof(T)) && !off(a.sum, a.lds, 16, sizeof(T))));
    if (!words) return launch(add_rms_norm_q8_any_kernel<T>, dim3((unsigned)a.rows), 256, 0, 1, st, a);
    const int n = a.hidden / E, few = a.rows <= 296;
    const int v = n > 2048 || (!few && n >= 256) ? 4 : n > 1024 || (!few && n >= 128) ? 2 : 1, threads = ((n + v - 1) / v + 31) / 32 * 32;
    return v == 4 ? add_rms_norm_q8_words<T, 4>(a, threads, st) : v == 2 ? add_rms_norm_q8_words<T, 2>(a, threads, st) : add_rms_norm_q8_words<T, 1>(a, threads, st);
}

// Rows in 8 bits as values: sixteen neighbours per thread and step, or one where rows are not on 16 bytes.  Blocks (x) along a row, (y) over rows.
struct ReadQ8Args {
    const int8_t* q;
    const float* scales;
    void* out;
    int64_t ldq, ldo, rows, n;
};
template <typename T, int E> __global__ void __launch_bounds__(256) read_q8_kernel(const ReadQ8Args a) {
    before();
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float s = a.scales[row];
        for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * E; i < a.n; i += (int64_t)gridDim.x * 256 * E) {
            struct __align__(E) W { int8_t v[E]; };
            const W w = *reinterpret_cast<const W*>(a.q + row * a.ldq + i);
            float f[E];
#pragma unroll
            for (int e = 0; e < E; e++) f[e] = (float)w.v[e] * s;
            store_n<T, E, (E > 1)>(reinterpret_cast<T*>(a.out) + row * a.ldo + i, f);
        }
    }
}
template <typename T> cudaError_t read_q8(const ReadQ8Args& a, cudaStream_t st) {
    const bool words = a.n % 16 == 0 && !((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) & 15) && a.ldq % 16 == 0 && a.ldo * sizeof(T) % 16 == 0;
    const int64_t per = words ? 4096 : 256;
    const dim3 grid((unsigned)std::min<int64_t>((a.n + per - 1) / per, 1024), (unsigned)std::min<int64_t>(a.rows, 16384));
    return words ? launch(read_q8_kernel<T, 16>, grid, 256, 0, 1, st, a) : launch(read_q8_kernel<T, 1>, grid, 256, 0, 1, st, a);
}

}  // namespace dev
