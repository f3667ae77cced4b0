// dev_q4_prompt.cuh — attention of many query tokens over the paged 4-bit cache, on tcgen05 (the sequences of b200_dev_attention_paged_q4 with many rows).
//
// The same function as dev_q4_attn.cuh.  A block has 128 query rows (row = token * G + head) of one sequence and kv head and walks the keys they see in tiles of 128:
//   warps 8-15  read a tile's nibbles (a page's row is one to four 16-byte words) and write them to shared memory as operands: 128 + n is n in the low bits of the bf16 128, 1024 + n those of the
//               fp16 1024; minus 136 or 1032 it is n - 8 (keys have the queries' type, values are fp16).  Keys as they lie, their channels in groups of eight in the order 0 4 1 5 2 6 3 7 (one shift and one and give two of them), which the
//               queries have too; values transposed, two positions per 32-bit word.
//   warp 16     issues S = Q K^T (128 x 128, K = hd) and O += P V (N = hd, K = 128).
//   warps 0-7   one thread per row, two groups of four warps that take every second tile with sums, maximum and statistics of their own, so that one group's exponentials run under the other's
//               products; the two are joined at the end.  P goes back to tensor memory in place of S.
// Keys' scales multiply the scores, values' scales the weights.  f32 queries are pairs of fp16 numbers scaled by a power of two.  Passes:
//   first   The reference of a row's exponentials need only be near: it is the largest score of the first tile that the row sees, and stays.  So no tile waits for another: one O, three buffers of scores,
//           each score read once.  A weight p_j d_j is two fp16 numbers (what the first leaves over is the second: 2^-22), 2^3 or 2^4 where the reference was set.
//   scan, again   Where a row passes fp16's range, or the last bits of its weights may have cost too much of its result (Q4Weights), or its result is not finite, the block goes over the keys twice more: once for
//           the scores alone, which gives each row its largest score m and its largest weight, and once as above with these for references: probabilities 2^(z_j - m), weights p_j d_j 2^e of up to 2^14 in pairs of fp16
//           numbers, whose last bit, 2^-25, is 2^-38 of the largest.
// What bounds it: per row and tile 128 x (hd + hd) products (three times that for f32), 128 exponentials with some ten instructions each, and shared memory: both operands of S and the values of P V are
// read from it, and 48 KB of them written per tile.  A tile takes 1.8 us at hd 128 (f32 2.1), on one SM as on all; issue slots are 59 % used, the tensor pipe 41 %, and the three roles slow one another at the schedulers.
// Measured: 2048 query tokens after 2048 others, 32 heads over 8 of 128: bf16 and f16 204 us, 512 blocks of 17 to 32 tiles, 505 TFLOP/s of the products that the mask leaves; f32 237.  bf16 results with single fp16 weights
// (2^-11) took 182, and then 20 more with keys made behind the values of the tile before.  Where every block goes over its keys again 545 (bf16), 556 (f16), 597 (f32): a scan takes 145 over the first pass, the pass behind it
// as long as the first.  (A second pass whose references moved, with pairs of bf16, took as long, and lost bits; with pairs of fp16 640.)  Blocks that need it: scores that pass a row's first tile by 2^12 or so, and rows whose
// largest channel is small next to the sum of their weights.  Gaussian scores of up to 4000 keys none; a first position with e^12 of the others' weight each and a twentieth of their values none in bf16, most in f16;
// f32 rows of Gaussian scores from some 5000 keys on.
#pragma once
#include <type_traits>

#include "dev_q4_attn.cuh"

namespace dev {

enum { QP_ROWS = 128, QP_KEYS = 128, QP_SOFT = 8, QP_MAKE = 8, QP_MMA = 16, QP_THREADS = 544 };

// By the result's type: the weights' place, 2^-kUp at the reference, so that scores have room for 2^(16 + kUp) above it (9 and 8.3 in natural logarithms), and the part of a row's largest channel that its weights' last
// bits, 2^-25 of each times a value of up to 8, may have cost at most, had they all one sign: half a step of bf16 and of f16 results, 2^-16 of f32 ones.
// (2^6 for Gaussian scores of standard deviation 2: some rows of 2048 tokens behind 2048 pass 2^10, and the call takes a third longer; 2^4: now and then a call has such a row; 1: a first position that draws most of the
// weight and has a twentieth of the others' values costs too many bits there already.)
template <typename T> struct Q4Weights { static constexpr float kUp = -3.0f, kOff = 1.0f / (1 << 8); };
template <> struct Q4Weights<__half> { static constexpr float kUp = -3.0f, kOff = 1.0f / (1 << 11); };
template <> struct Q4Weights<float> { static constexpr float kUp = -4.0f, kOff = 1.0f / (1 << 16); };

template <typename T, int HD> struct Q4PromptSmem {
    static constexpr int NQ = sizeof(T) == 4 ? 2 : 1;
    static constexpr int SLAB = 128 * 128, Q = NQ * (HD / 64) * SLAB, K = (HD / 64) * SLAB, V = 2 * HD * 128;      // rows of 128 bytes, SWIZZLE_128B
    static constexpr int K_AT = Q, V_AT = K_AT + 2 * K, META_AT = V_AT + 2 * V, META = 128 * 4 * 2 + 16, STAT_AT = META_AT + 4 * META, BAR_AT = STAT_AT + 2 * 128 * 8, BARS = 21, BYTES = BAR_AT + 3 * BARS * 8;
};
template <bool BF> __device__ __forceinline__ uint32_t sub_2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (BF) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// two nibbles (bits 0-3 and 16-19 of v) as n - 8
template <bool BF> __device__ __forceinline__ uint32_t nibbles(uint32_t v, uint32_t mask) { return sub_2<BF>(masked_or(v, mask, BF ? 0x43004300u : 0x64006400u), BF ? 0x43084308u : 0x64086408u); }
__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t at, uint32_t a) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(a) : "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
        "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
        "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
        : "memory");
}
// take(j, columns 32 j .. 32 j + 31) for a tile's 128 (a loop: the code of all of them at once does not stay in the instruction cache)
template <typename F> __device__ __forceinline__ void by_32(uint32_t taddr, F&& take) {
#pragma unroll 1
    for (int j = 0; j < 4; j++) {
        uint32_t v[32];
        tmem_ld32(v, taddr + 32 * j);
        take(j, v);
    }
}
// two f32 operations in one instruction
__device__ __forceinline__ uint64_t two(float2 v) { return (uint64_t)__float_as_uint(v.x) | (uint64_t)__float_as_uint(v.y) << 32; }
__device__ __forceinline__ float2 two(uint64_t v) { return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(a)), "l"(two(b)));
    return two(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(a)), "l"(two(b)));
    return two(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(two(a)), "l"(two(b)), "l"(two(c)));
    return two(r);
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// D = f32, A = B = bf16 (1) or fp16 (0), K-major
__device__ __forceinline__ uint32_t f16_idesc(bool bf, int M, int N) { return (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// passes; the two that few blocks make have code and registers of their own (by copy: nothing of the first one gets an address)
enum { QP_FIRST, QP_SCAN, QP_AGAIN };
template <typename F> __device__ __noinline__ void once_more(F pass) {
    pass(std::integral_constant<int, QP_SCAN>{});
    pass(std::integral_constant<int, QP_AGAIN>{});
}

template <typename T, int HD> __global__ void __launch_bounds__(QP_THREADS, 1) attention_q4_prompt_kernel(const b200_q4_attention a, uint64_t page16, int64_t limit) {
    before();
    using Sm = Q4PromptSmem<T, HD>;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    constexpr int NQ = Sm::NQ, SLABS = HD / 64;
    constexpr float kUp = Q4Weights<T>::kUp, kOff = Q4Weights<T>::kOff;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_item[2], s_bad;
    __shared__ float s_above;
    uint8_t* smem = smem_raw + ((1024u - (sm_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = sm_u32(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nkv = a.cache.n_kv_heads, G = a.n_heads / nkv, page_size = a.cache.page_size;

    // ---- this block's rows.  The last ones of a sequence see the most keys and come first.
    const int id = (int)(gridDim.x - 1 - blockIdx.x), h = id % nkv, item = id / nkv;
    if (warp == 0) {
        int at = item, seq = -1, rb = 0;
        for (int s0 = 0; s0 < a.seqs && seq < 0; s0 += 32) {
            int blocks = 0;
            if (s0 + lane < a.seqs) {
                const int64_t rows = (int64_t)q4_seq(a, s0 + lane, false).count * G;
                blocks = rows > limit ? (int)((rows + QP_ROWS - 1) / QP_ROWS) : 0;
            }
            int upto = blocks;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, at < upto);
            if (hit) {
                const int l = __ffs(hit) - 1;
                seq = s0 + l;
                rb = at - __shfl_sync(0xffffffffu, upto - blocks, l);
            } else {
                at -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (lane == 0) {
            s_item[0] = seq;
            s_item[1] = rb;
        }
    }
    // barriers of each pass (see below): keys there, used; values there, used (2 each); scores there (6); weights there, their products done (3 each; the scan: scores read, 6); all products done
    if (warp == 1) {
        for (int i = lane; i < 3 * Sm::BARS; i += 32) {
            const int b = i % Sm::BARS;
            bar_init(base + Sm::BAR_AT + 8 * i, b < 2 || b == 4 || b == 5 ? QP_MMA - QP_MAKE : b >= 14 && b < (i / Sm::BARS == QP_SCAN ? 20 : 17) ? 4 : 1);
        }
        bar_init_done();
        if (lane == 0) s_bad = 0;
    }
    __syncthreads();
    const int s = s_item[0], rb = s_item[1];
    if (s < 0) return;      // (the whole block)
    const Q4Seq q = q4_seq(a, s, false);
    const int rows = min(QP_ROWS, q.count * G - rb * QP_ROWS), first = rb * QP_ROWS / G, last = (rb * QP_ROWS + rows - 1) / G;
    const int64_t at0 = q.len - q.count;      // position of the sequence's first query token
    const int hi = (int)max((int64_t)0, at0 + last + 1), hi_min = (int)max((int64_t)0, at0 + first + 1);
    const int lo_min = a.window > 0 ? (int)max((int64_t)0, at0 + first + 1 - a.window) : 0, lo_max = a.window > 0 ? (int)max((int64_t)0, at0 + last + 1 - a.window) : 0;
    const int begin = lo_min & ~15, n = (hi - begin + QP_KEYS - 1) / QP_KEYS;      // tiles (0: nothing is seen)
    if (warp == QP_MMA) tmem_alloc<false>(&s_tmem, 512);

    // ---- queries: thread = row, half the channels each of two; pairs of fp16 for f32; scaled so that the row's elements are below 2^14 (bf16 too: sums of products with 8 stay in f32)
    float alpha = 0.0f;      // what a row's scores are multiplied with (its sign is in the queries)
    if (warp < QP_SOFT) {
        const int r = tid & 127, half = tid >> 7;
        const bool live = r < rows;
        const int rr = rb * QP_ROWS + (live ? r : 0), token = rr / G;
        const T* p = reinterpret_cast<const T*>(a.q) + (q.first + token) * a.q_token + (h * G + rr - token * G) * a.q_head;
        const bool vec = (reinterpret_cast<uintptr_t>(p) & 15) == 0;
        float* tops = reinterpret_cast<float*>(smem + Sm::STAT_AT);
        __align__(16) T x[HD / 2];
        if (vec) {
#pragma unroll
            for (int i = 0; i < HD / 32 * (int)sizeof(T); i++) reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(p + half * (HD / 2))[i];
        } else {
#pragma unroll
            for (int i = 0; i < HD / 2; i++) x[i] = p[half * (HD / 2) + i];
        }
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 2; i++) top = fmaxf(top, fabsf(to_f(x[i])));
        tops[tid] = top;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        top = fmaxf(tops[r], tops[128 + r]);
        const int e = top < INFINITY ? 140 - (int)(__float_as_uint(top) >> 23) : 0;
        float f1 = __int_as_float((127 + e / 2) << 23);
        const float f2 = __int_as_float((127 + e - e / 2) << 23);
        alpha = ldexpf(fabsf(a.scale) * 1.4426950408889634f, -e);
        if (a.scale < 0.0f) f1 = -f1;
#pragma unroll
        for (int g = 0; g < HD / 16; g++) {
            uint32_t o[4], ol[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float u = live ? to_f(x[8 * g + k]) * f1 * f2 : 0.0f, v = live ? to_f(x[8 * g + k + 4]) * f1 * f2 : 0.0f;
                if (BF) {
                    o[k] = pack_bf2(u, v);
                } else {
                    o[k] = pack_h2(u, v);
                    if (NQ == 2) {
                        const float2 b = unpack_h2(o[k]);
                        ol[k] = pack_h2(u - b.x, v - b.y);
                    }
                }
            }
            const int i = half * (HD / 16) + g;
            const uint32_t to = base + (i >> 3) * Sm::SLAB + r * 128 + (((i & 7) ^ (r & 7)) << 4);
            sts128(to, o[0], o[1], o[2], o[3]);
            if (NQ == 2) sts128(to + SLABS * Sm::SLAB, ol[0], ol[1], ol[2], ol[3]);
        }
        async_fence();
    }
    umma_before_sync();
    __syncthreads();
    umma_after_sync();
    const uint32_t tmem = s_tmem;
    bool alive = true;

    // one pass over the keys
    auto pass = [=](auto mode) mutable {
        constexpr int PASS = decltype(mode)::value;
        const uint32_t bars = base + Sm::BAR_AT + PASS * Sm::BARS * 8;
        const uint32_t k_full = bars, k_empty = bars + 16, v_full = bars + 32, v_empty = bars + 48, s_full = bars + 64, p_full = bars + 112, pv_done = bars + 136, all_done = bars + 160;
        if (warp >= QP_MAKE && warp < QP_MMA) {
            // ---- operands of keys and values
            const int pw = warp - QP_MAKE;
            constexpr int CH = HD / 32, PER = 32 / CH;              // 16-byte words of a row; rows a warp reads at once
            constexpr int KN = 16 / PER, VW = HD / 32;              // 16-byte words of keys per thread; 32-bit words of each of two values
            const int block = page_size * (HD + 8), v_off = page_size * (HD / 2);
            const uint8_t* head = reinterpret_cast<const uint8_t*>(a.cache.data) + (int64_t)h * block;
            const int64_t page_bytes = (int64_t)nkv * block;
            const int32_t* table = a.page_table + (int64_t)s * a.table_stride;
            uint32_t mask = 0x000f000fu;
            asm("" : "+r"(mask));      // (kept in a register: an instruction has room for one constant)
            // this warp's keys: the sixteen pw; its values: pairs of half the tile's positions, a quarter of the channels
            const int v_key = 64 * (pw & 1) + 2 * lane, v_word = (pw >> 1) * VW;
            // The page of the next tile's rows is looked up when this one's are asked for; those are asked for as soon as the registers of the tile before are free.
            const int tile_pages = QP_KEYS / page_size, tile_rows = QP_KEYS - tile_pages * page_size;
            const uint32_t n_pages = (uint32_t)min(a.cache.n_pages, (int64_t)INT32_MAX);
            struct Place {
                uint32_t page[1];
                int p, index, row;      // the first of sixteen positions, all in a page: its number, its page's place in the table, its row there
                bool wanted;
            } of_keys, of_values;
            auto look = [&](Place& w) {
                w.wanted = w.p < hi;
                load_where<1>(w.page, table + w.index, w.wanted);
            };
            auto first_look = [&](Place& w, int key) {
                w.p = begin + key;
                w.index = (int)(((uint64_t)(w.p >> 4) * page16) >> 36);
                w.row = w.p - w.index * page_size;
                look(w);
            };
            auto next_look = [&](Place& w) {
                w.p += QP_KEYS;      // (a call's positions end 2^20 before 2^31)
                w.row += tile_rows;
                w.index += tile_pages;
                if (w.row >= page_size) {
                    w.row -= page_size;
                    w.index++;
                }
                look(w);
            };
            auto at = [&](const Place& w) -> const uint8_t* {
                const bool good = w.wanted && w.page[0] < n_pages;
                if (w.wanted && !good && a.status) atomicOr(a.status, (int)B200_STATUS_BAD_PAGE);
                return good ? head + (int64_t)w.page[0] * page_bytes + w.row * (HD / 2) : nullptr;
            };
            struct Keys {
                uint32_t k[KN][4];
                uint32_t scale[1];      // of key 16 pw + lane, or of the value there (lanes from 16 on)
                bool there;
            } keys;
            struct Values {
                uint32_t v[2][VW];
            } values;
            auto ask_values = [&]() {
                const uint8_t* from = at(of_values);
                const bool there = from != nullptr;
                next_look(of_values);
#pragma unroll
                for (int u = 0; u < 2; u++) load_where<VW>(values.v[u], from + v_off + ((v_key & 15) + u) * (HD / 2) + v_word * 4, there);
            };
            auto ask_keys = [&]() {
                const uint8_t* from = at(of_keys);
                const bool there = from != nullptr;
                const uint8_t* scales = from + 2 * v_off - of_keys.row * (HD / 2 - 4) + ((lane & 15) + (lane < 16 ? 0 : page_size)) * 4;
                keys.there = there && of_keys.p + (lane & 15) < hi;
                next_look(of_keys);
#pragma unroll
                for (int i = 0; i < KN; i++) load_where<4>(keys.k[i], from + (i * PER + lane / CH) * (HD / 2) + (lane % CH) * 16, there);
                load_where<1>(keys.scale, scales, keys.there);
            };
            auto make_keys = [&](int t) {
                const Keys& w = keys;
                const uint32_t kt = base + Sm::K_AT + (t & 1) * Sm::K;
#pragma unroll
                for (int i = 0; i < KN; i++) {
                    const int r = pw * 16 + i * PER + lane / CH;
                    // (the second half of a row's lanes take their words in another order: the same chunk of both slabs is in the same banks)
                    const bool far = HD == 128 && (lane & 2);
                    const uint32_t x[4] = {far ? w.k[i][2] : w.k[i][0], far ? w.k[i][3] : w.k[i][1], far ? w.k[i][0] : w.k[i][2], far ? w.k[i][1] : w.k[i][3]};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int g = (lane % CH) * 4 + (far ? j ^ 2 : j);          // eight channels
                        sts128(kt + (g >> 3) * Sm::SLAB + r * 128 + (((g & 7) ^ (r & 7)) << 4), nibbles<BF>(x[j], mask), nibbles<BF>(x[j] >> 4, mask),
                               nibbles<BF>(x[j] >> 8, mask), nibbles<BF>(x[j] >> 12, mask));
                    }
                }
                uint8_t* meta = smem + Sm::META_AT + (t & 3) * Sm::META;
                // (the scan wants the values' scales as powers of two)
                reinterpret_cast<uint32_t*>(meta)[(lane < 16 ? 0 : 128) + 16 * pw + (lane & 15)] = PASS == QP_SCAN && lane >= 16 ? __float_as_uint(__log2f(fabsf(__uint_as_float(w.scale[0])))) : w.scale[0];
                const uint32_t gone = ~__ballot_sync(0xffffffffu, w.there);
                if (lane == 0) reinterpret_cast<uint16_t*>(meta + 1024)[pw] = (uint16_t)gone;
            };
            auto make_values = [&](int t) {
                const Values& w = values;
                const uint32_t vt = base + Sm::V_AT + (t & 1) * Sm::V + (pw & 1) * (HD * 128) + (lane & 3) * 4;
                const uint32_t c8 = lane >> 2;
#pragma unroll
                for (int j = 0; j < VW; j++) {
                    const uint32_t x[2] = {__byte_perm(w.v[0][j], w.v[1][j], 0x5410), __byte_perm(w.v[0][j], w.v[1][j], 0x7632)};
#pragma unroll
                    for (int k = 0; k < 8; k++) sts32(vt + ((v_word + j) * 8 + k) * 128 + ((c8 ^ k) << 4), nibbles<false>(x[k >> 2] >> (4 * (k & 3)), mask));
                }
            };
            first_look(of_keys, 16 * pw);
            if (PASS != QP_SCAN) first_look(of_values, v_key & ~15);
            if (n > 0) {
                ask_keys();
                if (PASS != QP_SCAN) ask_values();
            }
            // (a tile's keys before the values of the one ahead of it: these wait for products that need a row's exponentials, those only for the scores two tiles ago)
#pragma unroll 1
            for (int t = 0; t < n + (n > 0); t++) {
                if (t < n) {
                    const int st = t & 1;
                    bar_wait(k_empty + 8 * st, ((t >> 1) & 1) ^ 1u, alive, 11);
                    // (the scales of the tile four ago have been read: where values are made, those of two tiles ago were behind the products of its weights)
                    if (PASS == QP_SCAN && t >= 4) bar_wait(p_full + 8 * ((t - 4) % 6), ((t - 4) / 6) & 1, alive, 19);
                    make_keys(t);
                    async_fence();
                    __syncwarp();
                    if (lane == 0) bar_arrive(k_full + 8 * st);
                    ask_keys();
                }
                if (PASS != QP_SCAN && t > 0) {
                    const int st = (t - 1) & 1;
                    bar_wait(v_empty + 8 * st, (((t - 1) >> 1) & 1) ^ 1u, alive, 12);
                    make_values(t - 1);
                    async_fence();
                    __syncwarp();
                    if (lane == 0) bar_arrive(v_full + 8 * st);
                    ask_values();
                }
            }
        } else if (warp == QP_MMA) {
            const uint32_t iqk = f16_idesc(BF, 128, QP_KEYS), ipv = f16_idesc(false, 128, HD);
            constexpr int nb = 3, ns = 6;      // buffers of scores, barriers of theirs
            auto scores = [&](int t) {
                const int st = t & 1;
                bar_wait(k_full + 8 * st, (t >> 1) & 1, alive, 13);
                alive = __all_sync(0xffffffffu, alive);
                umma_after_sync();
                const uint32_t to = tmem + (t % nb) * 128, done = s_full + 8 * (t % ns);
                if (elect()) {
                    if (alive) {
                        const uint64_t dk = umma_desc(base + Sm::K_AT + st * Sm::K);
#pragma unroll
                        for (int u = 0; u < NQ; u++)
#pragma unroll
                            for (int sl = 0; sl < SLABS; sl++)
#pragma unroll
                                for (int kk = 0; kk < 4; kk++)
                                    mma_ss(to, umma_desc(base + (u * SLABS + sl) * Sm::SLAB) + 2 * kk, dk + (uint64_t)(sl * (Sm::SLAB >> 4) + 2 * kk), iqk, u + sl + kk > 0);
                    }
                    umma_commit<false>(k_empty + 8 * st);
                    umma_commit<false>(done);
                }
                __syncwarp();
            };
            for (int t = 0; t < min(n, nb); t++) scores(t);
            for (int t = 0; t < n; t++) {
                const int st = t & 1, b = t % nb;
                if constexpr (PASS == QP_SCAN) {      // whose scores go where those of t have been read
                    if (t + nb < n) {
                        bar_wait(p_full + 8 * (t % 6), (t / 6) & 1, alive, 15);
                        umma_after_sync();
                        scores(t + nb);
                    }
                    continue;
                }
                bar_wait(v_full + 8 * st, (t >> 1) & 1, alive, 14);
                bar_wait(p_full + 8 * b, (t / nb) & 1, alive, 15);
                alive = __all_sync(0xffffffffu, alive);
                umma_after_sync();
                const uint32_t to = tmem + 384, from = tmem + b * 128;
                if (elect()) {
                    if (alive) {
                        const uint64_t dv = umma_desc(base + Sm::V_AT + st * Sm::V);
#pragma unroll
                        for (int kk = 0; kk < 8; kk++)
#pragma unroll
                            for (int u = 0; u < 2; u++)
                                mma_ts(to, from + 32 * (kk >> 1) + 8 * (kk & 1) + 16 * u, dv + (uint64_t)((kk >> 2) * (HD * 128 >> 4) + 2 * (kk & 3)), ipv, t >= 1 || kk + u > 0);
                    }
                    umma_commit<false>(v_empty + 8 * st);
                    umma_commit<false>(pv_done + 8 * b);
                    if (t == n - 1) umma_commit<false>(all_done);
                }
                __syncwarp();
                if (t + nb < n) {      // whose scores go where the weights of t are
                    bar_wait(pv_done + 8 * b, (t / nb) & 1, alive, 16);
                    scores(t + nb);
                }
            }
        } else {
            // ---- rows
            const int r = tid & 127, grp = warp >> 2, rr = rb * QP_ROWS + r, token = rr / G;
            const bool live = r < rows;
            const int row_hi = live ? (int)max((int64_t)0, at0 + token + 1) : INT32_MAX, row_lo = live && a.window > 0 ? (int)max((int64_t)0, at0 + token + 1 - a.window) : 0;
            const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            float* refs = reinterpret_cast<float*>(smem + Sm::STAT_AT);      // first: after the first tile, after the second, then the two groups' sums; scan to again: m, e
            float m = -INFINITY, l = 0.0f;
            float above = 0.0f, heavy = -INFINITY;      // (scan: the largest log2 of a weight)
            int e = 0;                                  // again: weights are p d 2^e
            if constexpr (PASS == QP_AGAIN) {
                m = refs[r];
                e = (int)refs[128 + r];
            }
            const float unit = PASS == QP_AGAIN ? __int_as_float((127 + e) << 23) : 1.0f;
            bool write = true;
            for (int t = grp; t < n; t += 2) {
                const int p0 = begin + t * QP_KEYS;
                const uint8_t* meta = smem + Sm::META_AT + (t & 3) * Sm::META;
                const int b = t % 3;
                const uint32_t S = lanes + b * 128;
                bar_wait(s_full + 8 * (t % 6), (t / 6) & 1, alive, 17);
                __syncwarp();
                umma_after_sync();
                const uint4 gone = *reinterpret_cast<const uint4*>(meta + 1024);
                const bool all = p0 >= lo_max && p0 + QP_KEYS <= hi_min && !(gone.x | gone.y | gone.z | gone.w);      // (uniform)
                // a bit per key of a batch of 32 that this row does not see
                auto hidden = [&](int j) {
                    const int p = p0 + 32 * j, above = row_hi - p, below_ = row_lo - p;
                    uint32_t b = reinterpret_cast<const uint32_t*>(meta + 1024)[j];
                    if (above < 32) b |= above <= 0 ? 0xffffffffu : 0xffffffffu << above;
                    if (below_ > 0) b |= below_ >= 32 ? 0xffffffffu : ~(0xffffffffu << below_);
                    return b;
                };
                const float4* k4 = reinterpret_cast<const float4*>(meta);
                // the largest score
                auto largest = [&](auto whole) {
                    constexpr bool ALL = decltype(whole)::value;
                    float top[2] = {-INFINITY, -INFINITY};
                    const float2 al = make_float2(alpha, alpha);
                    auto take = [&](int j, const uint32_t (&v)[32]) {
                        const uint32_t hid = ALL ? 0u : hidden(j);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float4 k = k4[8 * j + i];
                            const float2 x = mul2(mul2(make_float2(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1])), al), make_float2(k.x, k.y)),
                                         y = mul2(mul2(make_float2(__uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3])), al), make_float2(k.z, k.w));
                            if (ALL) {
                                top[0] = fmaxf(fmaxf(x.x, x.y), top[0]);
                                top[1] = fmaxf(fmaxf(y.x, y.y), top[1]);
                            } else {
                                const float z[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
                                for (int u = 0; u < 4; u++)
                                    if (!((hid >> (4 * i + u)) & 1u)) top[0] = fmaxf(top[0], z[u]);
                            }
                        }
                    };
                    by_32(S, take);
                    return fmaxf(top[0], top[1]);
                };
                if constexpr (PASS == QP_SCAN) {
                    // the largest score so far, and the largest weight, as a power of two and with that score for reference
                    auto scan = [&](auto whole) {
                        constexpr bool ALL = decltype(whole)::value;
                        const float2 al = make_float2(alpha, alpha);
                        auto take = [&](int j, const uint32_t (&v)[32]) {
                            const uint32_t hid = ALL ? 0u : hidden(j);
                            float2 z[16];
                            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const float4 k = k4[8 * j + i];
#pragma unroll
                                for (int u = 0; u < 2; u++) {
                                    z[2 * i + u] = mul2(make_float2(__uint_as_float(v[4 * i + 2 * u]), __uint_as_float(v[4 * i + 2 * u + 1])), al);
                                    const float2 y = mul2(z[2 * i + u], u ? make_float2(k.z, k.w) : make_float2(k.x, k.y));
                                    if (ALL) {
                                        top[u] = fmaxf(fmaxf(y.x, y.y), top[u]);
                                    } else {
                                        if (!((hid >> (4 * i + 2 * u)) & 1u)) top[u] = fmaxf(top[u], y.x);
                                        if (!((hid >> (4 * i + 2 * u + 1)) & 1u)) top[u] = fmaxf(top[u], y.y);
                                    }
                                }
                            }
                            const float was = m;
                            m = fmaxf(m, fmaxf(top[0], top[1]));
                            heavy += below(was, m);
                            float most[2] = {heavy, heavy};
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const float4 k = k4[8 * j + i], d = k4[32 + 8 * j + i];
#pragma unroll
                                for (int u = 0; u < 2; u++) {
                                    const float2 w = add2(fma2(z[2 * i + u], u ? make_float2(k.z, k.w) : make_float2(k.x, k.y), make_float2(-m, -m)), u ? make_float2(d.z, d.w) : make_float2(d.x, d.y));
                                    if (ALL) {
                                        most[u] = fmaxf(fmaxf(w.x, w.y), most[u]);
                                    } else {
                                        if (!((hid >> (4 * i + 2 * u)) & 1u)) most[u] = fmaxf(most[u], w.x);
                                        if (!((hid >> (4 * i + 2 * u + 1)) & 1u)) most[u] = fmaxf(most[u], w.y);
                                    }
                                }
                            }
                            heavy = fmaxf(most[0], most[1]);
                        };
                        by_32(S, take);
                    };
                    if (all) scan(std::true_type{});
                    else scan(std::false_type{});
                    umma_before_sync();
                    __syncwarp();
                    if (lane == 0) bar_arrive(p_full + 8 * (t % 6));
                    continue;
                }
                if (PASS == QP_FIRST && t == 1) {
                    asm volatile("bar.sync 2, 256;" ::: "memory");
                    m = refs[r];
                    above = s_above;
                } else if (PASS == QP_FIRST && t == 2) {
                    asm volatile("bar.sync 3, 256;" ::: "memory");
                    m = refs[128 + r];
                }
                if (PASS == QP_FIRST && t < 2 && __any_sync(0xffffffffu, m == -INFINITY)) {
                    const float top = all ? largest(std::true_type{}) : largest(std::false_type{});
                    if (t == 0) {
                        // the largest value scale of the tile, as a power of two: with the reference that much higher (and kUp more) its weights are fp16 numbers of about 2^-kUp
                        // (of those that are numbers: a row that sees another one has no other result than NaN)
                        const float4 d = k4[32 + lane];
                        auto size = [](float v) { return (__float_as_uint(v) & 0x7fffffffu) < kInfBits ? fabsf(v) : 0.0f; };
                        const uint32_t big = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(size(d.x), size(d.y)), fmaxf(size(d.z), size(d.w)))));
                        above = (big ? (float)((int)(big >> 23) - 127) : 0.0f) + kUp;
                        if (tid == 0) s_above = above;
                    }
                    if (m == -INFINITY) m = fmaxf(m, top + above);
                }
                if (PASS == QP_FIRST && t < 2) {      // for the other group's first tile, or this one's next
                    refs[128 * t + r] = m;
                    __threadfence_block();
                    if (t == 0 && n > 1) asm volatile("bar.arrive 2, 256;" ::: "memory");
                    if (t == 1 && n > 2) asm volatile("bar.arrive 3, 256;" ::: "memory");
                }
                // the weights, in place of the scores: of 32 columns the first sixteen words are theirs, the others what those leave over
                auto weights = [&](auto whole) {
                    constexpr bool ALL = decltype(whole)::value;
                    const float2 al = make_float2(alpha, alpha);
                    const float ref = m == -INFINITY ? 0.0f : m;
                    float2 sum = make_float2(0.0f, 0.0f);
                    auto take = [&](int j, const uint32_t (&v)[32]) {
                        const uint32_t hid = ALL ? 0u : hidden(j);
                        float2 x[16];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float4 k = k4[8 * j + i];
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                // (alpha first: scaled queries times the scale of a large key would leave f32)
                                const float2 z = mul2(make_float2(__uint_as_float(v[4 * i + 2 * u]), __uint_as_float(v[4 * i + 2 * u + 1])), al);
                                float2 y = fma2(z, u ? make_float2(k.z, k.w) : make_float2(k.x, k.y), make_float2(-ref, -ref));
                                if (!ALL) {
                                    if ((hid >> (4 * i + 2 * u)) & 1u) y.x = -INFINITY;
                                    if ((hid >> (4 * i + 2 * u + 1)) & 1u) y.y = -INFINITY;
                                }
                                x[2 * i + u] = y;
                            }
                        }
                        uint32_t o[32];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float4 d = k4[32 + 8 * j + i];
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const float2 p = make_float2(ex2(x[2 * i + u].x), ex2(x[2 * i + u].y));
                                float2 w = mul2(p, u ? make_float2(d.z, d.w) : make_float2(d.x, d.y));
                                if (PASS == QP_AGAIN) w = mul2(w, make_float2(unit, unit));
                                if (!ALL) {      // (a scale that other rows see may be NaN)
                                    if ((hid >> (4 * i + 2 * u)) & 1u) w.x = 0.0f;
                                    if ((hid >> (4 * i + 2 * u + 1)) & 1u) w.y = 0.0f;
                                }
                                sum = add2(sum, p);
                                o[2 * i + u] = pack_h2(w.x, w.y);
                                const float2 f = unpack_h2(o[2 * i + u]);
                                o[16 + 2 * i + u] = pack_h2(w.x - f.x, w.y - f.y);
                            }
                        }
                        tmem_st32(S + 32 * j, o);      // (over columns that have been read)
                    };
                    by_32(S, take);
                    l += sum.x + sum.y;
                };
                if (all) weights(std::true_type{});
                else weights(std::false_type{});
                tmem_st_done();
                umma_before_sync();
                __syncwarp();
                if (lane == 0) bar_arrive(p_full + 8 * b);
            }
            if constexpr (PASS == QP_SCAN) {
                float2* stat = reinterpret_cast<float2*>(refs);
                stat[grp * 128 + r] = make_float2(m, heavy);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float2 s0 = stat[r], s1 = stat[128 + r];
                m = fmaxf(s0.x, s1.x);
                heavy = fmaxf(s0.y + below(s0.x, m), s1.y + below(s1.x, m));
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (grp == 0) {
                    refs[r] = m;
                    refs[128 + r] = m > -INFINITY && heavy > -INFINITY ? fminf(fmaxf(14.0f - ceilf(heavy), -126.0f), 126.0f) : 0.0f;
                }
            }
            if constexpr (PASS != QP_SCAN) {
                // ---- each thread has its row's half of the channels
                refs[256 + grp * 128 + r] = l;
                if (n > 0) bar_wait(all_done, 0, alive, 18);
                __syncwarp();
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float sum = refs[256 + r] + refs[384 + r];
                __syncwarp();
                umma_after_sync();
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                T* to = reinterpret_cast<T*>(a.out) + (q.first + token) * a.out_token + (h * G + rr - token * G) * a.out_head + grp * (HD / 2);
                const bool vec = (reinterpret_cast<uintptr_t>(to) & 15) == 0;
                auto result = [&](int j, float (&y)[32]) {
#pragma unroll
                    for (int i = 0; i < 32; i++) y[i] = 0.0f;
                    if (n > 0) {
                        uint32_t v[32];
                        tmem_ld32(v, lanes + 384 + grp * (HD / 2) + 32 * j);
#pragma unroll
                        for (int i = 0; i < 32; i++) y[i] = __uint_as_float(v[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 32; i++) y[i] = sum == 0.0f ? 0.0f : PASS == QP_AGAIN ? ldexpf(y[i] * inv, -e) : y[i] * inv;
                };
                if (PASS == QP_FIRST) {
                    // what is not finite may be so with another reference; sums of fp16 weights far below one have lost bits
                    float zero = sum * 0.0f, most = 0.0f;
#pragma unroll 1
                    for (int j = 0; j < HD / 64; j++) {
                        float y[32];
                        result(j, y);
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            zero = fmaf(y[i], 0.0f, zero);
                            most = fmaxf(most, fabsf(y[i]));
                        }
                    }
                    refs[grp * 128 + r] = m == -INFINITY ? -1.0f : most;      // (-1: the row has no reference, as far as this group knows)
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                    const float size = fmaxf(refs[r], refs[128 + r]);
                    // (none at all: its first two tiles lie in pages that are not there, and what follows them, if anything does, went without one)
                    const bool small = size < 0.0f ? row_hi > begin + 2 * QP_KEYS : !(size * sum * kOff >= (float)(n * QP_KEYS) * (1.0f / (1 << 22)));
                    // (values from 2^60 on: under their reference probabilities leave f32 below while they count)
                    if (__any_sync(0xffffffffu, live && (small || zero != 0.0f || above > 60.0f)) && lane == 0) atomicOr(&s_bad, 1);
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                    if (s_bad) write = false;
                }
#pragma unroll 1
                for (int j = 0; write && j < HD / 64; j++) {
                    float y[32];
                    result(j, y);
                    if (live) {
                        if (vec) store_n<T, 32, true>(to + 32 * j, y);
                        else store_n<T, 32, false>(to + 32 * j, y);
                    }
                }
            }
        }
        __syncwarp();
        umma_before_sync();
        __syncthreads();
        umma_after_sync();
    };
    pass(std::integral_constant<int, QP_FIRST>{});
    if (s_bad) once_more(pass);      // (uniform: written before the pass's last barrier)
    if (warp == QP_MMA) tmem_free<false>(tmem, 512);
}

// ------------------------------------------------------------------------------------------------------------------- host
// Sequences with more rows than this go to attention_q4_prompt_kernel, where a call's rows make it worth while.
constexpr int64_t kPromptRows = 32;
// blocks of 128 rows of a kv head, at most: whole ones, and a last one of each sequence that has more rows than kPromptRows
inline int64_t attention_q4_prompt_blocks(const b200_q4_attention& a) {
    const int64_t rows = a.tokens * (a.n_heads / a.cache.n_kv_heads);
    return rows / QP_ROWS + std::min<int64_t>(a.seqs, rows / (kPromptRows + 1));
}
// Whether a call's long sequences go there, by what the host knows.  A block of 128 rows takes 1.8 us for 128 keys (f32 2.1), whether alone or on every SM, and some 12 more; the other kernel spreads any number of rows
// over all SMs, a unit of eight of them some 0.04 us and 0.03 for 1000 keys.  So the units are compared with what a wave of 148 blocks is worth, 170 units where keys are few and up to 310 where they are many.  Of the keys
// the host knows the page table's width, or the window.  (Wider tables than a call needs: 310 for 190, rows that would take 31 us there take up to 40.)  Measured (32 heads over 8, hd 128, bf16, one sequence; units of the call:
// us there, here): 256 keys 128: 26, 28, 192: 30, 28; 500 keys 128: 30, 30, 256: 36, 32; 1000 keys 128: 32, 38, 192: 40, 38, 256: 44, 38; 2000 keys 192: 46, 52, 256: 54, 52; 4000 keys 256: 71, 83, 384: 93, 81;
// 16 000 keys 256: 167, 253, 384: 239, 249, 512: 304, 243.  Eight sequences with 1000 keys 288: 44, 38, with 4000 288: 77, 83, 384: 93, 83.  f32: 500 keys 192: 38, 38; 1000 keys 256: 46, 46; 4000 keys 256: 77, 93,
// 384: 104, 91.  32 heads over 4, hd 64: 1000 keys 128: 32, 34, 192: 38, 32; 4000 keys 256: 61, 67, 384: 81, 67.
inline bool attention_q4_has_prompts(const b200_q4_attention& a) {
    const int64_t G = a.n_heads / a.cache.n_kv_heads, nkv = a.cache.n_kv_heads;
    if (!a.q_starts || (a.max_q ? a.max_q : a.tokens) * G <= kPromptRows) return false;
    const int64_t width = (int64_t)a.table_pages * a.cache.page_size, keys = a.window > 0 ? std::min<int64_t>(width, (int64_t)a.window + QP_ROWS) : width;
    return (a.tokens * G + 7) / 8 * nkv > std::min<int64_t>(310, 170 + keys * 35 / 1000) * ((attention_q4_prompt_blocks(a) * nkv + 147) / 148);
}
template <typename T, int HD> cudaError_t attention_q4_prompt(const b200_q4_attention& a, cudaStream_t st) {
    using Sm = Q4PromptSmem<T, HD>;
    static SmemAllowed allowed;
    const auto kernel = attention_q4_prompt_kernel<T, HD>;
    const cudaError_t e = allowed((const void*)kernel, Sm::BYTES + 1024);
    if (e != cudaSuccess) return e;
    const uint64_t d = (uint64_t)a.cache.page_size / 16, page16 = (((uint64_t)1 << 36) + d - 1) / d;
    return launch(kernel, dim3((unsigned)(attention_q4_prompt_blocks(a) * a.cache.n_kv_heads)), QP_THREADS, Sm::BYTES + 1024, 1, st, a, page16, kPromptRows);
}
template <typename T, int HD> cudaError_t attention_q4(const b200_q4_attention& a, cudaStream_t st) {
    const bool prompts = attention_q4_has_prompts(a);
    if (prompts) {
        const cudaError_t e = attention_q4_prompt<T, HD>(a, st);
        if (e != cudaSuccess) return e;
    }
    return attention_q4_rows<T, HD>(a, prompts ? kPromptRows : INT64_MAX, st);
}

}  // namespace dev
