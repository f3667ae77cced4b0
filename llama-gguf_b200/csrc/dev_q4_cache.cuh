// dev_q4_cache.cuh — rotation, and keys and values into the paged 4-bit cache (b200_dev_rope_append_q4); cached rows as values (b200_dev_read_q4).
#pragma once
#include "dev_common.cuh"

namespace dev {

// Eight neighbouring channels per lane, head_dim / 8 lanes per row; a row is a head of a token's query, key or value.  VEC: every row starts on 16 bytes and rot_dims / 2 is a
// multiple of 8, so that a lane's channels, and those they are paired with, are words.
template <typename T, int HD, bool VEC> __global__ void __launch_bounds__(256) rope_append_q4_kernel(const b200_q4_append a) {
    constexpr int L = HD / 8;
    const int nkv = a.cache.n_kv_heads, heads = (a.q ? a.n_heads : 0) + 2 * nkv, half = a.rot_dims / 2;
    const int64_t item = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L, t = item / heads;
    const bool there = t < a.tokens;
    int h = (int)(item - t * heads);
    const int c = (threadIdx.x % L) * 8;
    const int kind = !a.q ? 1 + (h >= nkv) : h < a.n_heads ? 0 : 1 + (h - a.n_heads >= nkv);      // 0 query, 1 key, 2 value
    if (kind) h -= (a.q ? a.n_heads : 0) + (kind - 1) * nkv;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = 0.0f;
    bool placed = false;
    if (there) {
        const T* row = kind == 0   ? reinterpret_cast<const T*>(a.q) + t * a.q_token + h * a.q_head
                       : kind == 1 ? reinterpret_cast<const T*>(a.k) + t * a.k_token + h * a.k_head
                                   : reinterpret_cast<const T*>(a.v) + t * a.v_token + h * a.v_head;
        load_n<T, 8, VEC>(row + c, x);
        const int64_t pos = a.positions[t];
        placed = pos >= 0 && pos < a.table_rows;
        if (kind < 2 && placed && c < a.rot_dims) {
            const float* cs = a.cos_sin + pos * a.rot_dims;
            float y[8], cosv[8], sinv[8];
            if (VEC && a.use_neox) {
                const int i = c < half ? c : c - half;
                load_n<T, 8, true>(row + (c < half ? c + half : c - half), y);
                load_n<float, 8, false>(cs + i, cosv);
                load_n<float, 8, false>(cs + half + i, sinv);
                const float sign = c < half ? -1.0f : 1.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = __fadd_rn(__fmul_rn(x[j], cosv[j]), sign * __fmul_rn(y[j], sinv[j]));
            } else if (a.use_neox) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int ch = c + j;
                    if (ch < a.rot_dims) {
                        const bool lo = ch < half;
                        const int i = lo ? ch : ch - half;
                        const float other = __fmul_rn(to_f(row[lo ? ch + half : ch - half]), cs[half + i]);
                        x[j] = __fadd_rn(__fmul_rn(x[j], cs[i]), lo ? -other : other);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (c + 2 * j < a.rot_dims) {
                        const float co = cs[c / 2 + j], si = cs[half + c / 2 + j], u = x[2 * j], w = x[2 * j + 1];
                        x[2 * j] = __fsub_rn(__fmul_rn(u, co), __fmul_rn(w, si));
                        x[2 * j + 1] = __fadd_rn(__fmul_rn(w, co), __fmul_rn(u, si));
                    }
            }
        }
        if (!placed && a.status && threadIdx.x % L == 0) atomicOr(a.status, (int)B200_STATUS_BAD_POSITION);
    }
    __syncwarp();      // (q_out may be q: a row's lanes have read it all)
    if (there && kind == 0) {
        if (!placed) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __uint_as_float(0x7fffffffu);
        }
        store_n<T, 8, VEC>(reinterpret_cast<T*>(a.q_out) + t * a.q_out_token + h * a.q_out_head + c, x);
    }
    // the row's largest magnitude (as bits: infinities and NaN are above all numbers), and its value
    float hi = x[0], lo = x[0];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        hi = fmaxf(hi, x[i]);
        lo = fminf(lo, x[i]);
        top = max(top, __float_as_uint(fabsf(x[i])));
    }
#pragma unroll
    for (int o = L / 2; o; o >>= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (!there || kind == 0 || !placed) return;
    const int64_t slot = a.slots[t], page = slot / a.cache.page_size;
    if (slot < 0) return;
    if (page >= a.cache.n_pages) {
        if (a.status && threadIdx.x % L == 0) atomicOr(a.status, (int)B200_STATUS_BAD_SLOT);
        return;
    }
    const float m = __uint_as_float(top);
    const bool live = top < kInfBits && m >= kTiny;
    const float scale = live ? __fmul_rn(hi >= -lo ? hi : lo, -0.125f) : 0.0f, inv = live ? __fdiv_rn(1.0f, scale) : 0.0f;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int n = live ? min(15, __float2int_rn(__fmul_rn(x[i], inv)) + 8) : 8;
        word |= (uint32_t)n << (4 * i);
    }
    const int at = (int)(slot - page * a.cache.page_size);
    const Q4Block b = q4_block(a.cache, page, h);
    *reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(kind == 1 ? b.k : b.v) + at * (HD / 2) + c / 2) = word;
    if (threadIdx.x % L == 0) const_cast<float*>(kind == 1 ? b.ks : b.vs)[at] = top >= kInfBits ? __uint_as_float(0x7fffffffu) : scale;
}

struct ReadQ4Args {
    b200_q4_pages cache;
    const int64_t* slots;
    int64_t tokens;
    void *k_out, *v_out;
    int32_t* status;
};
template <typename T, int HD> __global__ void __launch_bounds__(256) read_q4_kernel(const ReadQ4Args a) {
    constexpr int L = HD / 8;
    const int nkv = a.cache.n_kv_heads;
    const int64_t item = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L, t = item / (2 * nkv);
    if (t >= a.tokens) return;
    const int u = (int)(item - t * 2 * nkv), kind = u >= nkv, h = kind ? u - nkv : u, c = (threadIdx.x % L) * 8;
    T* out = reinterpret_cast<T*>(kind ? a.v_out : a.k_out);
    if (!out) return;
    const int64_t slot = a.slots[t], page = slot / a.cache.page_size;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = 0.0f;
    if (slot >= 0 && page < a.cache.n_pages) {
        const int at = (int)(slot - page * a.cache.page_size);
        const Q4Block b = q4_block(a.cache, page, h);
        const uint32_t word = *reinterpret_cast<const uint32_t*>((kind ? b.v : b.k) + at * (HD / 2) + c / 2);
        const float scale = (kind ? b.vs : b.ks)[at];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = scale * (float)((int)((word >> (4 * i)) & 15u) - 8);
    } else if (slot >= 0 && a.status && threadIdx.x % L == 0) {
        atomicOr(a.status, (int)B200_STATUS_BAD_SLOT);
    }
    store_n<T, 8, true>(out + (t * nkv + h) * HD + c, x);
}

template <typename T, int HD> cudaError_t rope_append_q4(const b200_q4_append& a, bool vec, cudaStream_t st) {
    const int64_t rows = a.tokens * ((a.q ? a.n_heads : 0) + 2 * a.cache.n_kv_heads), per = 256 / (HD / 8), grid = (rows + per - 1) / per;
    if (vec) rope_append_q4_kernel<T, HD, true><<<(unsigned)grid, 256, 0, st>>>(a);
    else rope_append_q4_kernel<T, HD, false><<<(unsigned)grid, 256, 0, st>>>(a);
    return cudaGetLastError();
}
template <typename T, int HD> cudaError_t read_q4(const ReadQ4Args& a, cudaStream_t st) {
    const int64_t rows = a.tokens * 2 * a.cache.n_kv_heads, per = 256 / (HD / 8);
    read_q4_kernel<T, HD><<<(unsigned)((rows + per - 1) / per), 256, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace dev
