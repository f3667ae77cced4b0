// dev_glu_q8.cuh — gated unit of a row's two halves with the result in 8 bits and a scale per row (b200_dev_glu_q8).
//
// y = act(g) * u; scale = max |y| / 127; q = round(y * 127 / max |y|), halves to even, all of it as if y were exact: it is made in f32, and again in 64 bits where that could decide otherwise (the
// largest value of the row, and what lies next to the border between two numbers).  In 64 bits throughout 4096 x 14336 bf16 took 495 us.
//
// What bounds it: instructions and their latency (4096 x 14336 bf16 77 us by itself, 294 MB: 45 at the measured rate; relu, without the exponentials, 51, gelu 146; f32 rows of half as many, 264 MB, 50; rows of zeros 295, each of whose values may be the largest).  Steps: one block a row and a barrier on either side of
// the largest value's 64 bits 99 us; every warp making its own largest one in 64 bits, which leaves one barrier, and rounding from both ends of what y may be (two FMA and an exclusive or for a product, two sums, a difference and
// a comparison) 76.
#pragma once
#include <algorithm>
#include <type_traits>

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
    if (act == GLU_RELU) return (isnan(g) ? g : fmax(g, 0.0)) * up;
    const double d = 1.0 + exp(-z);
    if (!(d < 1e300)) return g / d * up;
    double r;      // 1 / d: its first bits, then two steps of Newton's method
    asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(r) : "d"(d));
    r = fma(r, fma(-d, r, 1.0), r);
    r = fma(r, fma(-d, r, 1.0), r);
    return g * r * up;
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

// largest magnitude whose f32 is finite
constexpr double kGluMost = 3.4028235677973366e38;      // 2^128 - 2^103
__device__ __forceinline__ bool glu_live(double top) { return top >= (double)kTiny && top < kGluMost; }
__device__ __forceinline__ float glu_scale(double top) { return !(top < kGluMost) ? NAN : glu_live(top) ? (float)(top / 127.0) : 0.0f; }
// Rows that no registers hold: a block per row, read twice, everything in 64 bits.
template <typename T> __global__ void __launch_bounds__(1024) glu_q8_any_kernel(const GluQ8Args a) {
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
    top = block_max_double(bad ? INFINITY : top, s_max);
    const double inv = glu_live(top) ? 127.0 / top : 0.0;
    for (int i = threadIdx.x; i < a.ff; i += blockDim.x) a.q[row * a.ldq + i] = inv != 0 ? (int8_t)__double2int_rn(glu_exact(to_f(g[i]), to_f(u[i]), a.act) * inv) : (int8_t)0;
    if (threadIdx.x == 0) a.scales[row] = glu_scale(top);
}

// y in f32.  With z = g (SiLU) or its tanh form's argument (GELU), 1 / (1 + exp(-z)) by ex2.approx (2^-22 off) and rcp.approx (2^-23); the exponential's argument is off by up to 1.5 2^-24 of itself (GELU: 2^-21.7), which counts
// where z is negative.  With the products' roundings, y and y times rcp.approx of (maximum / 127) are off by less than 2^-19 + |z| 2^-21 of themselves (the roundings alone by half of that).  Where z <= -16 y is made
// in 64 bits.  The gate is multiplied with last: it may be as small as 2^-149, where half of it has too few bits and a large up brings it back.  An up is that small in rows that count (from 2^-119 on) too, but then what
// r * up loses, 2^-150, is small beside y: for r < 1 the gate is below 17, and a number that is not 0 is of a y from 2^-119 / 254 on, so that 17 * 2^-150 is less than 2^-18 of it; in rows from 2^-112 on less than 2^-25.
constexpr float kGluOff = 1.9073486328125e-6f, kGluOffZ = 4.76837158203125e-7f, kGluOffMost = 1.1444091796875e-5f;      // 2^-19, 2^-21, both for z = -16 and a half more
constexpr float kGluOffSmall = 3.814697265625e-6f;      // 2^-18
template <int ACT> __device__ __forceinline__ float glu_z(float g) { return ACT == GLU_GELU ? 1.5957691216057308f * fmaf(0.044715f * g * g, g, g) : g; }
template <int ACT> __device__ __forceinline__ float glu_near(float g, float u) {
    if constexpr (ACT == GLU_RELU) return (g > 0 ? g : g == g ? 0.0f : g) * u;
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(glu_z<ACT>(g) * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return g * (r * u);
}
// the gate down to which y is made in f32 (z = -16, and -15.6)
template <int ACT> __device__ __forceinline__ constexpr float glu_least() { return ACT == GLU_GELU ? -4.8f : -16.0f; }
// ... and y made there may come out infinite where the exact one, next to the largest f32, does not: then it is made in 64 bits too.  (RELU's product is rounded once, as the exact one's.)
template <int ACT> __device__ __forceinline__ float glu_y(float g, float u) {
    const float y = glu_near<ACT>(g, u);
    return ACT != GLU_RELU && (g <= glu_least<ACT>() || !(fabsf(y) < INFINITY)) ? (float)glu_exact(g, u, ACT) : y;
}
// what a number of a row may be off by, of itself: `low` the least of its gates, `exact` the row's largest value
template <int ACT> __device__ __forceinline__ float glu_off(float low, double exact) {
    return kGluOff - fmaxf(glu_z<ACT>(fmaxf(low, glu_least<ACT>())), -16.0f) * kGluOffZ + (exact < 0x1p-112 ? kGluOffSmall : 0.0f);
}
// the smallest of `least` and a word's elements (NaN does not count)
template <typename T> __device__ __forceinline__ float word_min(const uint4& w, float least) {
    if constexpr (sizeof(T) == 4) {
        return fminf(fminf(least, fminf(__uint_as_float(w.x), __uint_as_float(w.y))), fminf(__uint_as_float(w.z), __uint_as_float(w.w)));
    } else {
        using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
        const T2* p = reinterpret_cast<const T2*>(&w);
        const T2 m = __hmin2(__hmin2(p[0], p[1]), __hmin2(p[2], p[3]));
        return fminf(least, fminf(to_f(m.x), to_f(m.y)));
    }
}
// Rows of whole 16-byte words on 16 bytes: blocks stride over the rows; a row stays in registers as y (V words of each half per thread), the next one's words are on their way to shared memory meanwhile, where each thread
// reads what it has copied itself.  A warp finds its largest value among the f32 ones and makes those that may be it again in 64 bits, so that the block needs one barrier a row; a number next to the border between
// two 8-bit ones is made again too (some of a hundred thousand).
template <typename T, int V, int ACT> __global__ void __launch_bounds__(1024) glu_q8_kernel(const GluQ8Args a) {
    before();
    constexpr int E = 16 / (int)sizeof(T);
    extern __shared__ uint4 glu_words[];      // [gate, up][V][threads]
    __shared__ double s_top[2][32];
    const int words = a.ff / E, tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5, step = blockDim.x;
    const uint4 *g = glu_words + tid, *u = g + V * step;
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(g);
    auto copy = [&](int64_t row) {
        if (row < a.rows) {
            const uint4 *p = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.x) + row * a.ldx) + tid, *q = p + words;
#pragma unroll
            for (int v = 0; v < V; v++) {
                const bool there = v * step + tid < words;
                copy_where<16>(to + v * step * 16, there ? p + v * step : a.x, there);
                copy_where<16>(to + (V + v) * step * 16, there ? q + v * step : a.x, there);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    copy(blockIdx.x);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        float y[V][E], most_of[V], top = 0, low = 0;
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
        for (int v = 0; v < V; v++) {
            const uint4 gw = g[v * step], uw = u[v * step];
#pragma unroll
            for (int e = 0; e < E; e++) y[v][e] = glu_near<ACT>(to_f(reinterpret_cast<const T*>(&gw)[e]), to_f(reinterpret_cast<const T*>(&uw)[e]));
            if constexpr (ACT != GLU_RELU) {
                const float least = word_min<T>(gw, 0.0f);
                low = fminf(low, least);
                if (least <= glu_least<ACT>()) {
#pragma unroll
                    for (int e = 0; e < E; e++) y[v][e] = glu_y<ACT>(to_f(reinterpret_cast<const T*>(&gw)[e]), to_f(reinterpret_cast<const T*>(&uw)[e]));
                }
            }
            most_of[v] = 0;
#pragma unroll
            for (int e = 0; e < E; e++) most_of[v] = max_nan(most_of[v], fabsf(y[v][e]));
            top = max_nan(top, most_of[v]);
        }
        uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if (ACT != GLU_RELU && most >= kInfBits) {
            uint32_t far = 0;
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int e = 0; e < E; e++) far |= fabsf(y[v][e]) < INFINITY ? 0u : 1u << (v * E + e);
            for (; far; far &= far - 1) {
                const int o = __ffs(far) - 1;
                const float x = (float)glu_exact(to_f(reinterpret_cast<const T*>(g + o / E * step)[o % E]), to_f(reinterpret_cast<const T*>(u + o / E * step)[o % E]), ACT);
#pragma unroll
                for (int v = 0; v < V; v++)
#pragma unroll
                    for (int e = 0; e < E; e++) y[v][e] = v * E + e == o ? x : y[v][e];
            }
            top = 0;
#pragma unroll
            for (int v = 0; v < V; v++) {
                most_of[v] = 0;
#pragma unroll
                for (int e = 0; e < E; e++) most_of[v] = max_nan(most_of[v], fabsf(y[v][e]));
                top = max_nan(top, most_of[v]);
            }
            most = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        }
        const float least = __uint_as_float(most) * (1.0f - 2 * kGluOffMost);
        double mine = most < kInfBits ? 0.0 : INFINITY;
        if (most < kInfBits && top >= least) {
            uint32_t which = 0;
#pragma unroll
            for (int v = 0; v < V; v++)
                if (most_of[v] >= least) {
#pragma unroll
                    for (int e = 0; e < E; e++) which |= fabsf(y[v][e]) >= least ? 1u << (v * E + e) : 0u;
                }
            for (; which; which &= which - 1) {
                const int o = __ffs(which) - 1;
                mine = fmax(mine, fabs(glu_exact(to_f(reinterpret_cast<const T*>(g + o / E * step)[o % E]), to_f(reinterpret_cast<const T*>(u + o / E * step)[o % E]), ACT)));
            }
        }
        // (largest of the warp: the lanes' doubles are not negative, so that their bits ascend as they do)
        const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)__double2hiint(mine)), lo = __reduce_max_sync(0xffffffffu, (uint32_t)__double2hiint(mine) == hi ? (uint32_t)__double2loint(mine) : 0u);
        if (lane == 0) s_top[turn][tid >> 5] = __hiloint2double((int)hi, (int)lo);
        copy(row + gridDim.x);
        __syncthreads();
        const double other = lane < warps ? s_top[turn][lane] : 0.0;
        const uint32_t bh = __reduce_max_sync(0xffffffffu, (uint32_t)__double2hiint(other)), bl = __reduce_max_sync(0xffffffffu, (uint32_t)__double2hiint(other) == bh ? (uint32_t)__double2loint(other) : 0u);
        const double exact = __hiloint2double((int)bh, (int)bl);
        if (tid == 0) a.scales[row] = glu_scale(exact);
        int8_t* out = a.q + row * a.ldq;
        if (!glu_live(exact)) {
            const uint32_t none[E] = {};
#pragma unroll
            for (int v = 0; v < V; v++)
                if (v * step + tid < words) store_bytes<E>(out + (v * step + tid) * E, none);
            continue;
        }
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"((float)exact * (1.0f / 127.0f)));      // (from 2^-126 to 2^121: neither side leaves the range)
        // rounded from both ends of what y may be: where the two are one number it is that
        const float off = glu_off<ACT>(low, exact), up = inv + inv * off, down = inv - inv * off;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = v * step + tid;
            if (i < words) {
                uint32_t n[E], differ = 0;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    n[e] = __float_as_uint(fmaf(y[v][e], up, kRoundHere));
                    differ |= n[e] ^ __float_as_uint(fmaf(y[v][e], down, kRoundHere));
                }
                store_bytes<E>(out + i * E, n);
                if (differ) {      // (the row's words are from memory again: the next one's have their place)
                    const T *p = reinterpret_cast<const T*>(a.x) + row * a.ldx + i * E, *q = p + a.ff;
#pragma unroll 1
                    for (int e = 0; e < E; e++) {
                        const float x = to_f(p[e]), z = to_f(q[e]), f = glu_y<ACT>(x, z);
                        if (fmaf(f, up, kRoundHere) != fmaf(f, down, kRoundHere)) out[i * E + e] = (int8_t)__double2int_rn(glu_exact(x, z, ACT) * (127.0 / exact));
                    }
                }
            }
        }
    }
}

// The same for rows of any length up to V blocks and any alignment: element by element, from memory again where something is made again.
template <typename T, int V, int ACT> __global__ void __launch_bounds__(1024) glu_q8_row_kernel(const GluQ8Args a) {
    before();
    __shared__ double s_top[32];
    const int64_t row = blockIdx.x;
    const T *gate = reinterpret_cast<const T*>(a.x) + row * a.ldx, *up_ = gate + a.ff;
    const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5;
    float y[V], top = 0, low = 0;
    uint32_t far = 0;      // where the gate is too far down for f32 (and then what came out infinite)
    {
        T g[V], u[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int i = min(v * (int)blockDim.x + tid, a.ff - 1);
            g[v] = gate[i];
            u[v] = up_[i];
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
            const bool there = v * (int)blockDim.x + tid < a.ff;
            const float x = to_f(g[v]);
            y[v] = there ? glu_near<ACT>(x, to_f(u[v])) : 0.0f;
            low = fminf(low, x);
            if (ACT != GLU_RELU && there && x <= glu_least<ACT>()) far |= 1u << v;
        }
    }
    uint32_t most;
    for (bool again = ACT != GLU_RELU;; again = false) {
        for (; far; far &= far - 1) {
            const int k = __ffs(far) - 1, i = k * blockDim.x + tid;
            const float x = (float)glu_exact(to_f(gate[i]), to_f(up_[i]), ACT);
#pragma unroll
            for (int v = 0; v < V; v++) y[v] = v == k ? x : y[v];
        }
        top = 0;
#pragma unroll
        for (int v = 0; v < V; v++) top = max_nan(top, fabsf(y[v]));
        most = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if (!again || most < kInfBits) break;
#pragma unroll
        for (int v = 0; v < V; v++) far |= fabsf(y[v]) < INFINITY ? 0u : 1u << v;      // (behind the row's last element y is 0)
    }
    const float least = __uint_as_float(most) * (1.0f - 2 * kGluOffMost);
    double mine = most < kInfBits ? 0.0 : INFINITY;
    if (most < kInfBits && top >= least) {
        uint32_t which = 0;
#pragma unroll
        for (int v = 0; v < V; v++) which |= fabsf(y[v]) >= least ? 1u << v : 0u;
        for (; which; which &= which - 1) {
            const int i = (__ffs(which) - 1) * blockDim.x + tid;
            if (i < a.ff) mine = fmax(mine, fabs(glu_exact(to_f(gate[i]), to_f(up_[i]), ACT)));
        }
    }
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)__double2hiint(mine)), lo = __reduce_max_sync(0xffffffffu, (uint32_t)__double2hiint(mine) == hi ? (uint32_t)__double2loint(mine) : 0u);
    if (lane == 0) s_top[tid >> 5] = __hiloint2double((int)hi, (int)lo);
    __syncthreads();
    const double other = lane < warps ? s_top[lane] : 0.0;
    const uint32_t bh = __reduce_max_sync(0xffffffffu, (uint32_t)__double2hiint(other)), bl = __reduce_max_sync(0xffffffffu, (uint32_t)__double2hiint(other) == bh ? (uint32_t)__double2loint(other) : 0u);
    const double exact = __hiloint2double((int)bh, (int)bl);
    if (tid == 0) a.scales[row] = glu_scale(exact);
    const bool live = glu_live(exact);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"((float)exact * (1.0f / 127.0f)));
    const float off = glu_off<ACT>(low, exact), up = inv + inv * off, down = inv - inv * off;
    int8_t* out = a.q + row * a.ldq;
    uint32_t close = 0;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int i = v * blockDim.x + tid;
        const uint32_t n = __float_as_uint(fmaf(y[v], up, kRoundHere));
        if (i < a.ff) {
            if (n != __float_as_uint(fmaf(y[v], down, kRoundHere))) close |= 1u << v;
            out[i] = live ? (int8_t)(n & 0xff) : (int8_t)0;
        }
    }
    if (live)
        for (; close; close &= close - 1) {
            const int i = (__ffs(close) - 1) * blockDim.x + tid;
            out[i] = (int8_t)__double2int_rn(glu_exact(to_f(gate[i]), to_f(up_[i]), ACT) * (127.0 / exact));
        }
}
template <typename T, int V> cudaError_t glu_q8_row(const GluQ8Args& a, cudaStream_t st) {
    const unsigned threads = ((a.ff + V - 1) / V + 31) / 32 * 32;
    auto go = [&](auto kernel) { return launch(kernel, dim3((unsigned)a.rows), threads, 0, 1, st, a); };
    return a.act == GLU_SILU ? go(glu_q8_row_kernel<T, V, GLU_SILU>) : a.act == GLU_GELU ? go(glu_q8_row_kernel<T, V, GLU_GELU>) : go(glu_q8_row_kernel<T, V, GLU_RELU>);
}

template <typename T, int V> cudaError_t glu_q8_words(const GluQ8Args& a, int threads, int blocks, cudaStream_t st) {
    const dim3 grid((unsigned)std::min<int64_t>(a.rows, blocks));
    const size_t most = V * 1024 * 32, smem = V * threads * 32;
    return a.act == GLU_SILU   ? launch_with<glu_q8_kernel<T, V, GLU_SILU>>(most, grid, threads, smem, st, a)
           : a.act == GLU_GELU ? launch_with<glu_q8_kernel<T, V, GLU_GELU>>(most, grid, threads, smem, st, a)
                               : launch_with<glu_q8_kernel<T, V, GLU_RELU>>(most, grid, threads, smem, st, a);
}
// Few rows: as many threads as a half has words, up to 1024 (latency: two rows of 14336 4 us by themselves).  Many rows: four words per thread, so that two and more blocks of an SM (its 65 536 registers hold 1024 threads) cover one another's barriers.
template <typename T> cudaError_t glu_q8(const GluQ8Args& a, cudaStream_t st) {
    constexpr int E = 16 / (int)sizeof(T);
    const bool words = a.ff % E == 0 && a.ff / E <= 4096 && !(reinterpret_cast<uintptr_t>(a.x) & 15) && a.ldx % E == 0 && !(reinterpret_cast<uintptr_t>(a.q) % E) && a.ldq % E == 0;
    // (2000 x 16383 bf16: 104 us, 215 in 64 bits throughout; 16384 wide rows, as words, 41 for as many)
    if (!words) return a.ff <= 1024 ? glu_q8_row<T, 4>(a, st) : a.ff <= 16384 ? glu_q8_row<T, 16>(a, st) : launch(glu_q8_any_kernel<T>, dim3((unsigned)a.rows), 1024, 0, 1, st, a);
    int sms = 0;
    const cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    const int n = a.ff / E, v = n > 2048 || (a.rows > 2 * sms && n >= 256) ? 4 : n > 1024 || (a.rows > 2 * sms && n >= 64) ? 2 : 1, threads = ((n + v - 1) / v + 31) / 32 * 32, blocks = sms * std::max(1, 1024 / threads);
    return v == 4 ? glu_q8_words<T, 4>(a, threads, blocks, st) : v == 2 ? glu_q8_words<T, 2>(a, threads, blocks, st) : glu_q8_words<T, 1>(a, threads, blocks, st);
}

}  // namespace dev
