// dev_q4_attn.cuh — attention over the paged 4-bit cache (b200_dev_attention_paged_q4).
#pragma once
#include "dev_common.cuh"

namespace dev {

template <typename T, int HD> __global__ void __launch_bounds__(128) attention_q4_plain_kernel(const b200_q4_attention a) {
    constexpr int E = HD / 32;
    const int64_t item = (int64_t)blockIdx.x * 4 + threadIdx.x / 32, s = item / a.n_heads;
    const int h = (int)(item - s * a.n_heads), lane = threadIdx.x & 31, kv = h / (a.n_heads / a.cache.n_kv_heads), page_size = a.cache.page_size;
    if (s >= a.seqs) return;
    const int64_t first = a.q_starts ? a.q_starts[s] : s, end = a.q_starts ? a.q_starts[s + 1] : s + 1, count = end - first;
    const int64_t cap = (int64_t)a.table_pages * page_size;
    int64_t len = a.kv_lens[s];
    if (len < 0 || len > cap || first < 0 || count < 0 || end > a.tokens) {
        if (a.status && lane == 0) atomicOr(a.status, (int)B200_STATUS_BAD_LENGTH);
        len = len < 0 ? 0 : len > cap ? cap : len;
        if (first < 0 || count < 0 || end > a.tokens) return;
    }
    for (int64_t t = first + blockIdx.y; t < end; t += gridDim.y) {
    const int64_t pos = len - count + (t - first), begin = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) {
        q[i] = to_f(reinterpret_cast<const T*>(a.q)[t * a.q_token + h * a.q_head + lane * E + i]) * a.scale * 1.44269504f;
        o[i] = 0.0f;
    }
    for (int64_t j = begin; j <= pos; j++) {
        const int64_t page = a.page_table[s * a.table_stride + j / page_size];
        if (page < 0 || page >= a.cache.n_pages) {
            if (a.status && lane == 0) atomicOr(a.status, (int)B200_STATUS_BAD_PAGE);
            continue;
        }
        const Q4Block b = q4_block(a.cache, page, kv);
        const int at = (int)(j % page_size);
        float z = 0.0f;
        float vv[E];
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int c = lane * E + i;
            z += q[i] * (float)(((b.k[at * (HD / 2) + c / 2] >> (4 * (c & 1))) & 15) - 8);
            vv[i] = (float)(((b.v[at * (HD / 2) + c / 2] >> (4 * (c & 1))) & 15) - 8) * b.vs[at];
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
        z *= b.ks[at];
        const float top = fmaxf(m, z), f = m == top ? 1.0f : exp2f(m - top), p = z == top ? 1.0f : exp2f(z - top);
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < E; i++) o[i] = o[i] * f + p * vv[i];
        m = top;
    }
#pragma unroll
    for (int i = 0; i < E; i++) reinterpret_cast<T*>(a.out)[t * a.out_token + h * a.out_head + lane * E + i] = from_f<T>(l == 0.0f ? 0.0f : o[i] / l);
    }
}

template <typename T, int HD> cudaError_t attention_q4(const b200_q4_attention& a, cudaStream_t st) {
    const int64_t items = (int64_t)a.seqs * a.n_heads;
    attention_q4_plain_kernel<T, HD><<<dim3((unsigned)((items + 3) / 4), (unsigned)(a.tokens > a.seqs ? 256 : 1)), 128, 0, st>>>(a);
    return cudaGetLastError();
}
inline size_t attention_q4_workspace(const b200_q4_attention&) { return 0; }

}  // namespace dev
