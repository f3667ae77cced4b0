// dev_route.cuh — routing to experts (b200_dev_route_experts): a router's logits to each token's experts and their weights.
//
// p = softmax(z) or 1 / (1 + exp(-z)); c = z, or p + correction; experts by c, the lower number first among equals; weights p, or p over the sum of the chosen ones', times a factor.
// What decides is made in 64 bits: scores of 32 bits next to one another would be chosen by their rounding.
//
// A warp per token; expert e is lane e % 32's value e / 32.  A choice is the largest key of all lanes (keys are the values' bits, so that they ascend as unsigned numbers) by redux.sync, its
// high word, then its low word among those that have it, then the lowest expert.
#pragma once
#include <algorithm>

#include "dev_common.cuh"

namespace dev {

enum { ROUTE_MOST = 1024, ROUTE_GROUPS = 32, ROUTE_WARPS = 4 };

struct RouteArgs {
    const void* logits;
    const float* correction;
    int32_t* experts;
    float* weights;
    int64_t ld, tokens;
    int n, top, groups, top_groups, sigmoid, renormalise;
    float scale;
};

// ascending as unsigned; 0: not to be chosen
__device__ __forceinline__ uint64_t route_key(double c) {
    if (!(c > -INFINITY)) return 0;
    const uint64_t b = (uint64_t)__double_as_longlong(c + 0.0);      // (+ 0.0: there is one zero)
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double route_value(uint64_t key) { return __longlong_as_double((long long)(key >> 63 ? key & 0x7fffffffffffffffull : ~key)); }
// the largest key of the warp
__device__ __forceinline__ uint64_t route_max(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (uint64_t)hi << 32 | lo;
}

template <typename T, int V> __global__ void __launch_bounds__(ROUTE_WARPS * 32) route_experts_kernel(const RouteArgs a) {
    before();
    __shared__ uint64_t s_key[ROUTE_WARPS][V * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t token = (int64_t)blockIdx.x * ROUTE_WARPS + warp;
    if (token >= a.tokens) return;
    const T* z = reinterpret_cast<const T*>(a.logits) + token * a.ld;
    float x[V];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; v++) {
        x[v] = v * 32 + lane < a.n ? to_f(z[v * 32 + lane]) : -INFINITY;
        nan |= isnan(x[v]) || (!a.sigmoid && x[v] == INFINITY);
    }
    nan = __any_sync(0xffffffffu, nan);      // (no weights then; the choice goes by the logits)
    float most = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; v++) most = fmaxf(most, x[v]);
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    double total = 0;
    if (!a.sigmoid) {
#pragma unroll
        for (int v = 0; v < V; v++) total += x[v] > -INFINITY ? exp((double)x[v] - most) : 0.0;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    auto score = [&](float v) { return !(v > -INFINITY) ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : exp((double)v - most) / total; };
    const bool by_score = a.correction && !nan;
    uint64_t key[V];
#pragma unroll
    for (int v = 0; v < V; v++) key[v] = !(x[v] > -INFINITY) ? 0 : route_key(by_score ? score(x[v]) + a.correction[v * 32 + lane] : (double)x[v]);
    if (a.groups > 1) {
        // a lane per group: its two best
        const int each = a.n / a.groups;
#pragma unroll
        for (int v = 0; v < V; v++) s_key[warp][v * 32 + lane] = by_score || nan ? key[v] : key[v] ? route_key(score(x[v])) : 0;
        __syncwarp();
        uint64_t first = 0, second = 0;
        if (lane < a.groups)
            for (int i = 0; i < each; i++) {
                const uint64_t k = s_key[warp][lane * each + i];
                second = max(second, min(first, k));
                first = max(first, k);
            }
        uint64_t value = second && !nan ? route_key(route_value(first) + route_value(second)) : first;
        uint32_t kept = 0;
        for (int i = 0; i < a.top_groups; i++) {
            const uint64_t best = route_max(value);
            const int who = __reduce_min_sync(0xffffffffu, value == best ? lane : 32);
            if (best) kept |= 1u << who;
            if (lane == who) value = 0;
        }
#pragma unroll
        for (int v = 0; v < V; v++)
            if (v * 32 + lane < a.n && !(kept >> ((v * 32 + lane) / each) & 1)) key[v] = 0;
    }
    int mine = -1;      // lane j: the token's expert j
    float at = -INFINITY;
    for (int j = 0; j < a.top; j++) {
        uint64_t k = 0;
        int e = 0;
        float l = 0;
#pragma unroll
        for (int v = V - 1; v >= 0; v--)
            if (key[v] >= k) k = key[v], e = v * 32 + lane, l = x[v];
        const uint64_t best = route_max(k);
        const int who = best ? (int)__reduce_min_sync(0xffffffffu, k == best ? (uint32_t)e : 0xffffffffu) : -1;
        const float value = __shfl_sync(0xffffffffu, l, who & 31);
        if (lane == j) mine = who, at = best ? value : -INFINITY;
#pragma unroll
        for (int v = 0; v < V; v++)
            if (v * 32 + lane == who) key[v] = 0;
    }
    double p = score(at);
    if (a.renormalise) {
        double sum = p;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        p = sum > 0 ? p / sum : p;
    }
    if (lane < a.top) {
        a.experts[token * a.top + lane] = mine;
        a.weights[token * a.top + lane] = nan && mine >= 0 ? NAN : (float)(p * a.scale);
    }
}

template <typename T> cudaError_t route_experts(const RouteArgs& a, cudaStream_t st) {
    const dim3 grid((unsigned)((a.tokens + ROUTE_WARPS - 1) / ROUTE_WARPS));
    auto go = [&](auto kernel) { return launch(kernel, grid, ROUTE_WARPS * 32, 0, 1, st, a); };
    return a.n <= 32 ? go(route_experts_kernel<T, 1>) : a.n <= 64 ? go(route_experts_kernel<T, 2>) : a.n <= 128 ? go(route_experts_kernel<T, 4>) : a.n <= 256 ? go(route_experts_kernel<T, 8>)
         : a.n <= 512 ? go(route_experts_kernel<T, 16>) : go(route_experts_kernel<T, 32>);
}

}  // namespace dev
