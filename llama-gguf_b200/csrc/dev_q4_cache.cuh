// dev_q4_cache.cuh — rotation, and keys and values into the paged 4-bit cache (b200_dev_rope_append_q4); cached rows as values (b200_dev_read_q4).
#pragma once
#include "dev_common.cuh"

namespace dev {

// n / d for n < 2^31: (n * m) >> 32 with m = ceil(2^32 / d) is at most one too large, which the product tells
struct Divisor {
    uint32_t d, m;
    explicit Divisor(uint32_t d_) : d(d_), m((uint32_t)((((uint64_t)1 << 32) + d_ - 1) / d_)) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        if (d == 1) return n;
        const uint32_t q = __umulhi(n, m);
        return q * d > n ? q - 1 : q;
    }
};

// Eight neighbouring channels per lane, head_dim / 8 lanes per row; a row is a head of a token's query, key or value.  VEC: every row starts on 16 bytes, rot_dims / 2 is a
// multiple of 8 and the table starts on 16 bytes, so that a lane's channels, those they are paired with, and their cosines and sines are words.
// Bound by the rows' bytes (queries read and written, keys and values read) where there are many tokens, by the launch and one chain of loads (position, table, row) where there are few.
// 4001 tokens of 32 + 4 + 4 heads of 64 in f16: @APPEND@.
template <typename T, int HD, bool VEC> __global__ void __launch_bounds__(256) rope_append_q4_kernel(const b200_q4_append a, const Divisor heads) {
    constexpr int L = HD / 8;
    const int nkv = a.cache.n_kv_heads, nh = a.q ? a.n_heads : 0, half = a.rot_dims / 2;
    const uint32_t item = blockIdx.x * (256 / L) + threadIdx.x / L, t = heads(item);      // (rows of one call are fewer than 2^31)
    const bool there = t < a.tokens;
    int h = (int)(item - t * heads.d);
    const int c = (threadIdx.x % L) * 8;
    const int kind = h < nh ? 0 : 1 + (h - nh >= nkv);      // 0 query, 1 key, 2 value
    if (kind) h -= nh + (kind - 1) * nkv;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = 0.0f;
    bool placed = false;
    int64_t slot = -1;
    if (there) {
        const T* row = kind == 0   ? reinterpret_cast<const T*>(a.q) + t * a.q_token + h * a.q_head
                       : kind == 1 ? reinterpret_cast<const T*>(a.k) + t * a.k_token + h * a.k_head
                                   : reinterpret_cast<const T*>(a.v) + t * a.v_token + h * a.v_head;
        const int64_t pos = a.positions[t];
        if (kind) slot = a.slots[t];
        load_n<T, 8, VEC>(row + c, x);
        placed = pos >= 0 && pos < a.table_rows;
        if (kind < 2 && placed && c < a.rot_dims) {
            const float* cs = a.cos_sin + pos * a.rot_dims;
            if (VEC && a.use_neox) {
                float y[8], cosv[8], sinv[8];
                const int i = c < half ? c : c - half;
                load_n<T, 8, true>(row + (c < half ? c + half : c - half), y);
                load_n<float, 8, true>(cs + i, cosv);
                load_n<float, 8, true>(cs + half + i, sinv);
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
                float co[4], si[4];
                if (VEC) {
                    load_n<float, 4, true>(cs + c / 2, co);
                    load_n<float, 4, true>(cs + half + c / 2, si);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const bool in = c + 2 * j < a.rot_dims;
                        co[j] = in ? cs[c / 2 + j] : 1.0f;
                        si[j] = in ? cs[half + c / 2 + j] : 0.0f;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (VEC || c + 2 * j < a.rot_dims) {
                        const float u = x[2 * j], w = x[2 * j + 1];
                        x[2 * j] = __fsub_rn(__fmul_rn(u, co[j]), __fmul_rn(w, si[j]));
                        x[2 * j + 1] = __fadd_rn(__fmul_rn(w, co[j]), __fmul_rn(u, si[j]));
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
    if (!__any_sync(0xffffffffu, there && kind)) return;      // (queries alone)
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
    if (!there || kind == 0 || !placed || slot < 0) return;
    const int64_t page = slot / a.cache.page_size;
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
template <typename T, int HD> __global__ void __launch_bounds__(256) read_q4_kernel(const ReadQ4Args a, const Divisor rows) {
    constexpr int L = HD / 8;
    const int nkv = a.cache.n_kv_heads;
    const uint32_t item = blockIdx.x * (256 / L) + threadIdx.x / L;
    const int64_t t = rows(item);
    if (t >= a.tokens) return;
    const int u = (int)(item - (uint32_t)t * rows.d), kind = u >= nkv, h = kind ? u - nkv : u, c = (threadIdx.x % L) * 8;
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
    const uint32_t heads = (a.q ? a.n_heads : 0) + 2 * a.cache.n_kv_heads;
    const int64_t per = 256 / (HD / 8), grid = (a.tokens * heads + per - 1) / per;
    if (vec) rope_append_q4_kernel<T, HD, true><<<(unsigned)grid, 256, 0, st>>>(a, Divisor(heads));
    else rope_append_q4_kernel<T, HD, false><<<(unsigned)grid, 256, 0, st>>>(a, Divisor(heads));
    return cudaGetLastError();
}
template <typename T, int HD> cudaError_t read_q4(const ReadQ4Args& a, cudaStream_t st) {
    const uint32_t rows = 2 * a.cache.n_kv_heads;
    const int64_t per = 256 / (HD / 8);
    read_q4_kernel<T, HD><<<(unsigned)((a.tokens * rows + per - 1) / per), 256, 0, st>>>(a, Divisor(rows));
    return cudaGetLastError();
}

}  // namespace dev
