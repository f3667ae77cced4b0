// dev_route.cuh — routing to experts (b200_dev_route_experts): a router's logits to each token's experts and their weights.
//
// p = softmax(z) or 1 / (1 + exp(-z)); c = z, or p + correction; experts by c, the lower number first among equals; weights p, or p over the sum of the chosen ones', times a factor.
// What decides is made in 64 bits: scores of 32 bits next to one another would be chosen by their rounding.
//
// A warp per token; expert e is lane e % 32's value e / 32.  Keys ascend as unsigned numbers: 22 bits of the value (16-bit logits whole, f32 logits' first bits, scores in fixed point between the token's least and
// largest), then 1023 - e, so that one redux.sync gives a choice and its expert, the lower one among equals; each lane's keys are sorted once and the chosen one's lane moves up.  Scores are made in f32 (off by less
// than 2^-21).  Where two that follow one another are closer than all that may be off, the token (some of a hundred) is chosen for again with 64-bit scores and keys, which took 34 us for 8192 tokens of 256
// experts in 8 groups where all did.
// What bounds it: instructions, some 1560 a token with groups (8192 tokens of 256 experts, sigmoid with a correction, 8 of them in 4 of 8 groups: 22.6 us; without groups 15.3, softmax by logits 9.9; the logits' bytes 0.6).  One token: 2 us by itself.
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
    uint32_t per_group;      // 2^20 / experts of a group, rounded up: e * per_group >> 20 is expert e's group
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

// Group `lane`'s two best keys (of `each` neighbours in s_key; `of` lanes share a group's): read in turns, so that lanes of different groups meet different banks.
template <typename K> __device__ __forceinline__ void route_two(const K* s_key, int lane, int groups, int each, K& first, K& second) {
    int of = 1;
    while (of * 2 * groups <= 32) of *= 2;
    const int mine = lane / of, part = lane % of, turn = each % of == 0 ? mine * of % each : 0;
    first = second = 0;
    if (mine < groups)
        for (int i = part; i < each; i += of) {
            const int at = i + turn;      // (the places of a lane are those of its part, whichever it begins at)
            const K k = s_key[mine * each + (at < each ? at : at - each)];
            second = max(second, min(first, k));
            first = max(first, k);
        }
    for (int o = 1; o < of; o <<= 1) {
        const K f = __shfl_xor_sync(0xffffffffu, first, o), s = __shfl_xor_sync(0xffffffffu, second, o);
        second = max(min(first, f), max(second, s));
        first = max(first, f);
    }
    // lane g: group g's
    const int from = lane * of & 31;
    const K f = __shfl_sync(0xffffffffu, first, from), s = __shfl_sync(0xffffffffu, second, from);
    first = lane < groups ? f : 0;
    second = lane < groups ? s : 0;
}

// One token in 64 bits.  x: its logits, most: their largest; returns this lane's (place's) expert, and its logit in `at`.
template <int V> __device__ __noinline__ int route_exactly(const RouteArgs& a, const float* x, float most, bool by_score, bool nan, uint64_t* s_key, int lane, float* at) {
    double total = 0;
    if (!a.sigmoid) {
        for (int v = 0; v < V; v++) total += x[v] > -INFINITY ? exp((double)x[v] - most) : 0.0;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    auto score = [&](float v) { return a.sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : exp((double)v - most) / total; };
    uint64_t key[V];
#pragma unroll
    for (int v = 0; v < V; v++) key[v] = !(x[v] > -INFINITY) ? 0 : route_key(by_score ? score(x[v]) + a.correction[v * 32 + lane] : (double)x[v]);
    if (a.groups > 1) {
        const int each = a.n / a.groups;
#pragma unroll
        for (int v = 0; v < V; v++) s_key[v * 32 + lane] = by_score || nan ? key[v] : key[v] ? route_key(score(x[v])) : 0;
        __syncwarp();
        uint64_t first, second;
        route_two<uint64_t>(s_key, lane, a.groups, each, first, second);
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
    int mine = -1;
    *at = -INFINITY;
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
        if (lane == j) mine = who, *at = best ? value : -INFINITY;
#pragma unroll
        for (int v = 0; v < V; v++)
            if (v * 32 + lane == who) key[v] = 0;
    }
    return mine;
}

__device__ __forceinline__ uint32_t route_key32(float c) {
    if (!(c > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(c + 0.0f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float route_value32(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

// descending
template <int V> __device__ __forceinline__ void route_sort(uint32_t (&k)[V]) {
#pragma unroll
    for (int size = 2; size <= V; size *= 2)
#pragma unroll
        for (int apart = size / 2; apart; apart /= 2)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int o = i ^ apart;
                if (o > i) {
                    const uint32_t hi = max(k[i], k[o]), lo = min(k[i], k[o]);
                    k[i] = i & size ? lo : hi;
                    k[o] = i & size ? hi : lo;
                }
            }
}

template <typename T, int V> __global__ void __launch_bounds__(ROUTE_WARPS * 32, V <= 4 ? 12 : V == 8 ? 8 : 4) route_experts_kernel(const RouteArgs a) {
    before();
    __shared__ uint64_t s_key[ROUTE_WARPS][V * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t token = (int64_t)blockIdx.x * ROUTE_WARPS + warp;
    if (token >= a.tokens) return;
    const T* z = reinterpret_cast<const T*>(a.logits) + token * a.ld;
    float x[V], most = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; v++) x[v] = v * 32 + lane < a.n ? to_f(z[v * 32 + lane]) : -INFINITY;
#pragma unroll
    for (int v = 0; v < V; v++) {
        nan |= isnan(x[v]) || (!a.sigmoid && x[v] == INFINITY);
        most = fmaxf(most, x[v]);
    }
    nan = __any_sync(0xffffffffu, nan);      // (no weights then; the choice goes by the logits)
    if (!a.sigmoid || nan) {
        const uint32_t k = __reduce_max_sync(0xffffffffu, route_key32(most));
        most = k ? route_value32(k) : -INFINITY;
    }
    const bool by_score = a.correction && !nan, scores = by_score || (a.groups > 1 && !nan);
    bool close = false;      // the choice may be another one in 64 bits
    float c[V];              // scores (with the correction)
    if (scores) {
        float per = 1.0f;
        if (!a.sigmoid) {
            double total = 0;
#pragma unroll
            for (int v = 0; v < V; v++) {
                c[v] = expf(x[v] - most);
                total += x[v] > -INFINITY ? c[v] : 0.0f;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            per = (float)(1.0 / total);
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
            float p = c[v] * per;
            if (a.sigmoid) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(1.0f + __expf(-x[v])));
            c[v] = !(x[v] > -INFINITY) ? -INFINITY : by_score ? p + a.correction[v * 32 + lane] : p;
        }
    }
    uint32_t kept = 0xffffffffu;
    if (a.groups > 1) {
        uint32_t* s_key32 = reinterpret_cast<uint32_t*>(s_key[warp]);
#pragma unroll
        for (int v = 0; v < V; v++) s_key32[v * 32 + lane] = route_key32(scores ? c[v] : x[v]);
        __syncwarp();
        uint32_t first, second, least = 0;
        route_two<uint32_t>(s_key32, lane, a.groups, a.n / a.groups, first, second);
        uint32_t value = second && !nan ? route_key32(route_value32(first) + route_value32(second)) : first;
        kept = 0;
        for (int i = 0; i < a.top_groups; i++) {
            least = __reduce_max_sync(0xffffffffu, value);
            const int who = __reduce_min_sync(0xffffffffu, value == least ? lane : 32);
            if (least) kept |= 1u << who;
            if (lane == who) value = 0;
        }
        const uint32_t next = __reduce_max_sync(0xffffffffu, value);
        if (scores) {      // (a sum of two: 2^-20, and its rounding and theirs, which are those of the largest where they cancel)
            const float most_of = fmaxf(first ? fabsf(route_value32(first)) : 0.0f, second ? fabsf(route_value32(second)) : 0.0f), largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most_of)));
            if (next && least) close = !(route_value32(least) - route_value32(next) > 0x1p-18f + 0x1p-21f * largest);
            close |= largest > 1e38f;      // (a sum may leave the range)
        }
    }
    // keys, and by how much (in their 22 bits) a choice must be ahead of what follows it
    uint32_t key[V], ahead = sizeof(T) == 2 ? 0 : 1;
    if (by_score) {
        float lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int v = 0; v < V; v++) {
            hi = fmaxf(hi, c[v]);
            if (c[v] > -INFINITY) lo = fminf(lo, c[v]);
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, route_key32(hi)), bottom = __reduce_min_sync(0xffffffffu, lo < INFINITY ? route_key32(lo) : 0xffffffffu);
        hi = route_value32(top);
        lo = route_value32(bottom);
        const float range = fmaxf(hi - lo, 0x1p-10f), per = 4194000.0f / range;      // (below 2^22 - 2 for any rounding)
        close |= !(range < 1e30f) && top;
        ahead = (uint32_t)fminf((0x1p-19f + 0x1p-22f * fmaxf(fabsf(lo), fabsf(hi))) * per + 3.0f, 4e6f);
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = c[v] > -INFINITY ? ((uint32_t)fminf((c[v] - lo) * per, 4194000.0f) + 1) << 10 : 0;
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) {
            const uint32_t k = route_key32(x[v]);      // (16-bit numbers: the last 13 or 16 bits are all zeros or all ones)
            key[v] = k ? (k >> 10 ? k & ~1023u : 1024u) : 0;
        }
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int e = v * 32 + lane;
        key[v] = key[v] && kept >> ((uint32_t)e * a.per_group >> 20 & 31) & 1 ? key[v] | (uint32_t)(1023 - e) : 0;
    }
    route_sort<V>(key);
    int mine = -1;      // lane j: the token's expert j
    uint32_t last = 0xffffffffu;
    for (int j = 0; j <= a.top; j++) {
        const uint32_t best = __reduce_max_sync(0xffffffffu, key[0]);
        if (!best) break;
        close |= (last >> 10) - (best >> 10) < ahead;
        last = best;
        if (lane == j && j < a.top) mine = 1023 - (int)(best & 1023u);
        if (key[0] == best) {
#pragma unroll
            for (int v = 0; v + 1 < V; v++) key[v] = key[v + 1];
            key[V - 1] = 0;
        }
    }
    float at = mine >= 0 ? to_f(z[mine]) : -INFINITY;
    if (close) mine = route_exactly<V>(a, x, most, by_score, nan, s_key[warp], lane, &at);
    // weights: in 64 bits
    double p = 0;
    if (at > -INFINITY) p = a.sigmoid ? 1.0 / (1.0 + exp(-(double)at)) : exp((double)at - most);
    double total = 0;
    if (a.renormalise) {
        total = p;
    } else if (!a.sigmoid) {
#pragma unroll
        for (int v = 0; v < V; v++) total += x[v] > -INFINITY ? exp((double)x[v] - most) : 0.0;
    }
    if (a.renormalise || !a.sigmoid) {
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        p = total > 0 ? p / total : p;
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
