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

// Eight neighbouring channels per lane, head_dim / 8 lanes per row; a row is a head of a token's query, key or value.  The first blocks have the keys and values, a row per group of lanes; the others
// the queries, QPER rows of a token per group of lanes, their loads together, with one load of the token's cosines and sines.  VEC: every row starts on 16 bytes, rot_dims / 2 is a multiple of 8 and the
// table starts on 16 bytes, so that a lane's channels, those they are paired with, and their cosines and sines are words.
// Bound by the rows' bytes (queries read and written, keys and values read) where there are many tokens, by the launch and one chain of loads (position, table, row) where there are few.  Measured (cold, by itself):
// 4001 tokens of 32 + 4 + 4 heads of 64 in f16 14.3 us (39.1 MB, 2.7 TB/s; four rows there 14.0, one 16.4), 32 tokens of 32 + 8 + 8 heads of 128 in bf16 5.8.
template <typename T, int HD, bool VEC> struct RopeLane {
    static constexpr int L = HD / 8;
    int c, half, rot;
    bool neox, lo, turned;
    float co[8], si[8];
    __device__ __forceinline__ explicit RopeLane(const b200_q4_append& a)
        : c((threadIdx.x % L) * 8), half(a.rot_dims / 2), rot(a.rot_dims), neox(a.use_neox != 0), lo(c < half), turned(c < rot) {}
    __device__ __forceinline__ void table(const float* cs) {      // a token's row
        if (!turned) return;
        const int at = neox ? (lo ? c : c - half) : c / 2;
        if (VEC) {
            load_n<float, 4, true>(cs + at, reinterpret_cast<float(&)[4]>(co[0]));
            load_n<float, 4, true>(cs + half + at, reinterpret_cast<float(&)[4]>(si[0]));
            if (neox) {
                load_n<float, 4, true>(cs + at + 4, reinterpret_cast<float(&)[4]>(co[4]));
                load_n<float, 4, true>(cs + half + at + 4, reinterpret_cast<float(&)[4]>(si[4]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = neox ? (c + j < half ? c + j : c + j - half) : c / 2 + j;
                const bool in = neox ? c + j < rot : j < 4 && c + 2 * j < rot;
                co[j] = in ? cs[i] : 1.0f;
                si[j] = in ? cs[half + i] : 0.0f;
            }
        }
    }
    // a row's channels, and those they are paired with (halves)
    __device__ __forceinline__ void load(const T* row, T (&x)[8], T (&y)[8]) const {
        if (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) {
                reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(row + c)[i];
                if (neox && turned) reinterpret_cast<uint4*>(y)[i] = reinterpret_cast<const uint4*>(row + (lo ? c + half : c - half))[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[j] = row[c + j];
                if (neox && c + j < rot) y[j] = row[c + j < half ? c + j + half : c + j - half];
            }
        }
    }
    __device__ __forceinline__ void turn(const T (&x)[8], const T (&y)[8], float (&f)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = to_f(x[j]);
        if (!turned) return;
        if (neox) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (VEC || c + j < rot) {
                    const float u = __fmul_rn(to_f(y[j]), si[j]);
                    f[j] = __fadd_rn(__fmul_rn(f[j], co[j]), (VEC ? lo : c + j < half) ? -u : u);
                }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (VEC || c + 2 * j < rot) {
                    const float u = f[2 * j], w = f[2 * j + 1];
                    f[2 * j] = __fsub_rn(__fmul_rn(u, co[j]), __fmul_rn(w, si[j]));
                    f[2 * j + 1] = __fadd_rn(__fmul_rn(w, co[j]), __fmul_rn(u, si[j]));
                }
        }
    }
};

template <typename T, int HD, bool VEC, int QPER>
__global__ void __launch_bounds__(256) rope_append_q4_kernel(const b200_q4_append a, const Divisor kv_rows, const Divisor q_groups, unsigned kv_blocks, const Divisor page16) {
    before();
    constexpr int L = HD / 8, PB = 256 / L;
    RopeLane<T, HD, VEC> lane(a);
    const bool leader = threadIdx.x % L == 0;
    const int nkv = a.cache.n_kv_heads;
    if (blockIdx.x >= kv_blocks) {
        // ---- queries
        const uint32_t item = (blockIdx.x - kv_blocks) * PB + threadIdx.x / L;      // (rows of one call are fewer than 2^31)
        const int64_t t = q_groups(item);
        const int first = (int)(item - (uint32_t)t * q_groups.d) * QPER, n = t < a.tokens ? min(QPER, a.n_heads - first) : 0;
        __align__(16) T x[QPER][8], y[QPER][8];
        bool placed = false;
        if (n > 0) {
            const int64_t pos = a.positions[t];
            const T* row = reinterpret_cast<const T*>(a.q) + t * a.q_token + first * a.q_head;
#pragma unroll
            for (int i = 0; i < QPER; i++, row += a.q_head)
                if (i < n) lane.load(row, x[i], y[i]);
            placed = pos >= 0 && pos < a.table_rows;
            if (placed) lane.table(a.cos_sin + pos * a.rot_dims);
            else if (a.status && leader) atomicOr(a.status, (int)B200_STATUS_BAD_POSITION);
        }
        __syncwarp();      // (q_out may be q: a row's lanes have read it all)
        T* to = reinterpret_cast<T*>(a.q_out) + t * a.q_out_token + first * a.q_out_head + lane.c;
#pragma unroll
        for (int i = 0; i < QPER; i++, to += a.q_out_head)
            if (i < n) {
                float f[8];
                lane.turn(x[i], y[i], f);
                if (!placed) {
#pragma unroll
                    for (int j = 0; j < 8; j++) f[j] = __uint_as_float(0x7fffffffu);
                }
                store_n<T, 8, VEC>(to, f);
            }
        return;
    }
    // ---- keys and values
    const uint32_t item = blockIdx.x * PB + threadIdx.x / L;
    const int64_t t = kv_rows(item);
    const int r = (int)(item - (uint32_t)t * kv_rows.d), h = r < nkv ? r : r - nkv;
    const bool key = r < nkv, there = t < a.tokens;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = 0.0f;
    int64_t slot = -1;
    if (there) {
        __align__(16) T x[8], y[8];
        const int64_t pos = a.positions[t];
        slot = a.slots[t];
        const T* row = key ? reinterpret_cast<const T*>(a.k) + t * a.k_token + h * a.k_head : reinterpret_cast<const T*>(a.v) + t * a.v_token + h * a.v_head;
        lane.load(row, x, y);
        if (pos < 0 || pos >= a.table_rows) {
            slot = -1;
            if (a.status && leader) atomicOr(a.status, (int)B200_STATUS_BAD_POSITION);
        } else if (key) {
            lane.table(a.cos_sin + pos * a.rot_dims);
            lane.turn(x, y, f);
        }
        if (!key) {
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = to_f(x[j]);
        }
    }
    // the row's largest magnitude (as bits: infinities and NaN are above all numbers), and its value
    float high = f[0], low = f[0];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        high = fmaxf(high, f[j]);
        low = fminf(low, f[j]);
        top = max(top, __float_as_uint(fabsf(f[j])));
    }
#pragma unroll
    for (int o = L / 2; o; o >>= 1) {
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (slot < 0) return;
    // (sixteens of slots: a page has a whole number of them)
    const int64_t page = (slot >> 35) == 0 ? (int64_t)page16((uint32_t)(slot >> 4)) : slot / a.cache.page_size;
    if (page >= a.cache.n_pages) {
        if (a.status && leader) atomicOr(a.status, (int)B200_STATUS_BAD_SLOT);
        return;
    }
    const float m = __uint_as_float(top);
    const bool live = top < kInfBits && m >= kTiny;
    const float scale = live ? __fmul_rn(high >= -low ? high : low, -0.125f) : 0.0f, inv = live ? __fdiv_rn(1.0f, scale) : 0.0f;
    uint32_t word = 0x88888888u;
    if (live) {
        word = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) word |= (uint32_t)min(15, __float2int_rn(__fmul_rn(f[j], inv)) + 8) << (4 * j);
    }
    const int at = (int)(slot - page * a.cache.page_size);
    const Q4Block b = q4_block(a.cache, page, h);
    *reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(key ? b.k : b.v) + at * (HD / 2) + lane.c / 2) = word;
    if (leader) const_cast<float*>(key ? b.ks : b.vs)[at] = top >= kInfBits ? __uint_as_float(0x7fffffffu) : scale;
}

struct ReadQ4Args {
    b200_q4_pages cache;
    const int64_t* slots;
    int64_t tokens;
    void *k_out, *v_out;
    int32_t* status;
};
template <typename T, int HD> __global__ void __launch_bounds__(256) read_q4_kernel(const ReadQ4Args a, const Divisor rows) {
    before();
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

template <typename T, int HD, bool VEC, int QPER> cudaError_t rope_append_q4_by(const b200_q4_append& a, cudaStream_t st) {
    const int64_t per = 256 / (HD / 8), kv = 2 * a.cache.n_kv_heads, kv_blocks = (a.tokens * kv + per - 1) / per, groups = a.q ? (a.n_heads + QPER - 1) / QPER : 1;
    const int64_t q_blocks = a.q ? (a.tokens * groups + per - 1) / per : 0;
    return launch(rope_append_q4_kernel<T, HD, VEC, QPER>, dim3((unsigned)(kv_blocks + q_blocks)), 256, 0, 1, st, a, Divisor((uint32_t)kv), Divisor((uint32_t)groups), (unsigned)kv_blocks,
                  Divisor((uint32_t)a.cache.page_size / 16));
}
// Four query rows per group of lanes where one each would be more than all SMs hold at once (2048 threads each): fewer instructions per row.  Below that one: more rows on their way.
template <typename T, int HD> cudaError_t rope_append_q4(const b200_q4_append& a, bool vec, cudaStream_t st) {
    return !vec ? rope_append_q4_by<T, HD, false, 1>(a, st) : a.q && a.tokens * a.n_heads * (HD / 8) > 148 * 2048 ? rope_append_q4_by<T, HD, true, 4>(a, st) : rope_append_q4_by<T, HD, true, 1>(a, st);
}
template <typename T, int HD> cudaError_t read_q4(const ReadQ4Args& a, cudaStream_t st) {
    const uint32_t rows = 2 * a.cache.n_kv_heads;
    const int64_t per = 256 / (HD / 8);
    return launch(read_q4_kernel<T, HD>, dim3((unsigned)((a.tokens * rows + per - 1) / per)), 256, 0, 1, st, a, Divisor(rows));
}

}  // namespace dev
