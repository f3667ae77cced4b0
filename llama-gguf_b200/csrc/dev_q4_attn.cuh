// dev_q4_attn.cuh — attention over the paged 4-bit cache (b200_dev_attention_paged_q4).
//
// One pass over the keys with a running maximum: o = sum_j p_j d_j (n_j - 8) / sum_j p_j, p_j = 2^(z_j - m), z_j = log2(e) scale k_j q . (n_j - 8), k_j and d_j the scales of key and value j.
//
// Work.  An item is eight query rows of one sequence and kv head (row = token * G + head, G query heads per kv head) with the keys they see, in tiles of 16 W positions (W warps).  All items
// lie on one line, sequence after sequence, QA_START units for what an item takes by itself and one for each of its tiles, and every block takes an equal stretch of it, so that a long sequence among
// short ones, or alone, keeps every SM busy; lengths are read on the device only.  A stretch that ends inside an item leaves its sums in the workspace, and the second kernel joins them.
// (Without the units for the start 32 sequences of up to 8000 took 60 us for 46 of longer ones: the block with the shortest sequences took twice the others' time.)
//
// A warp takes 16 positions at a time (never more than one page) through a ring in shared memory (cp.async, 16 bytes per lane) and multiplies with mma.m16n8k16 (fp16, f32 sums), the
// positions (scores) or channels (values) as its 16 rows and the eight query rows as its columns:
//   scores  a nibble in the low bits of an fp16 is the number n 2^-24 exactly (four bits further up: 16 n 2^-24, and that channel's query element is divided by 16): one shift
//           and four ands turn eight nibbles into operands.  - 8 sum q is taken off afterwards in f32 (not for f32 results, which that would cost three bits: theirs are made as the values').
//   values  1024 + n is n in the low bits of the fp16 1024; minus 1032 it is n - 8.  (Sums of n alone would grow with the keys while the result does not: f32 sums would lose 1e-4 of it.)
// Queries are scaled by a power of two into fp16's range.  Weights are two fp16 numbers (what the first leaves over is the second: 2^-22), and so are f32 queries: the second ones go through another mma into the
// same sums.  f16 and bf16 queries are one exactly.  (Weights of one number, 2^-11, took a tenth less time for bf16 results, which they moved to the next number now and then.)
// The weight of a value is p_j d_j.  Its reference is not m but m + r, the largest z_j + log2 |d_j| so far less 7: p_j d_j stays in fp16's range whatever the values' scales are, from 2^7 to 2^15 where it is largest,
// so that fp16's last bit, 2^-25, is 2^-32 of that (r is kept by itself: large scores leave no bits of log2 |d_j| in a sum).  Both references move only when something passes them by 2^8, so the usual step has no exchange between lanes but the 8 x 8 transposition that makes operands of the weights.
// What bounds it: the bytes of the cache, hd + 8 per position and kv head.  Measured (both kernels, cold): one token over 131072 positions, 64 heads over 8 of 128, bf16 and f16: 50 us for 143 MB (2.8 TB/s): about 7 us until
// every block knows its stretch and has its first tiles, some 33 of stream (a kernel of the same copies without the arithmetic: 36 altogether), a spread of the blocks' ends, 4 of the join; f32 56.  Issue slots are 54 % used.  32 sequences of
// up to 8000: 43 us for 96 MB.  With single weights (bf16) 46 and 39.  A warp takes 32 positions a step (two of the above, so that its chains of mma cover each other).  When single weights were the rule, warps of an SM and positions of a step (us, the two cases): 12 and 32 46.5, 38.7;
// 16 and 32 51, 44.6; 16 and 16 52, 43; 8 and 48 43.9 to 45, 39.5 to 43: the first of these is the best of the two together and the steadier.
#pragma once
#include <type_traits>

#include "dev_umma.cuh"

namespace dev {

enum { QA_ROWS = 8, QA_START = 4, QA_WARPS = 12, QA_STAGES = 3 };      // rows of an item, units of its start, warps of an SM
constexpr float QA_UP = 7.0f;                                           // log2 of the weight that a reference is set to

struct Q4Seq {
    int first, count;      // query tokens
    int64_t len;           // cached positions
};
// a sequence's query tokens (none where the tokens do not lie within the call's, or there are more than `limit` rows)
__device__ __forceinline__ Q4Seq q4_seq(const b200_q4_attention& a, int s, bool report, int64_t limit = INT64_MAX) {
    Q4Seq q;
    const int64_t b = a.q_starts ? a.q_starts[s] : s, e = a.q_starts ? a.q_starts[s + 1] : s + 1, cap = (int64_t)a.table_pages * a.cache.page_size;
    q.len = a.kv_lens[s];
    const bool wrong = b < 0 || e < b || e > a.tokens;
    if (report && a.status && (wrong || q.len < 0 || q.len > cap)) atomicOr(a.status, (int)B200_STATUS_BAD_LENGTH);
    q.len = q.len < 0 ? 0 : q.len > cap ? cap : q.len;
    q.first = wrong ? 0 : (int)b;
    q.count = wrong || (e - b) * (a.n_heads / a.cache.n_kv_heads) > limit ? 0 : (int)(e - b);
    return q;
}
// positions [base, hi) that the rows of block rb see, in `tiles` tiles; rows that see nothing have one tile all the same (it writes their zeros)
struct Q4Span {
    int base, hi, tiles;
};
template <int TILE> __device__ __forceinline__ Q4Span q4_span(const b200_q4_attention& a, const Q4Seq& q, int G, int rb) {
    const int last = (min(rb * QA_ROWS + QA_ROWS, q.count * G) - 1) / G, first = rb * QA_ROWS / G;
    const int64_t at = q.len - q.count;
    Q4Span s;
    s.hi = (int)max((int64_t)0, at + last + 1);
    s.base = a.window > 0 ? (int)max((int64_t)0, at + first + 1 - a.window) / TILE * TILE : 0;
    s.tiles = max(1, (s.hi - s.base + TILE - 1) / TILE);
    return s;
}

// the workspace: per block, two parts of [8][HD] sums, [8][4] (m, r, l, -); then per block what its first stretch ends
struct Q4End {
    int first_cta, first_slot, token, rb, head, rows;      // the sequence's first query token; rows of the item (0: nothing ends)
};
template <int HD> __host__ __device__ constexpr int q4_part_floats() { return QA_ROWS * (HD + 4); }

// where block i of `grid` begins on a line of `total` units: floor(total i / grid), without a division of 64 bits
__device__ __forceinline__ long long q4_begin(long long total, int i, int grid) {
    if (total >> 32) return total * i / grid;
    const uint32_t each = (uint32_t)total / (uint32_t)grid, over = (uint32_t)total - each * (uint32_t)grid;
    return (long long)each * i + over * (uint32_t)i / (uint32_t)grid;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// a reference's distance to one that is at least as high (0 where both are -infinity)
__device__ __forceinline__ float below(float x, float top) { return x == top ? 0.0f : x - top; }
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// ... with sums that begin here
__device__ __forceinline__ void mma16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// (v & mask) | set in one instruction
__device__ __forceinline__ uint32_t masked_or(uint32_t v, uint32_t mask, uint32_t set) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(set));
    return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ uint32_t sub_h2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// an 8 x 8 matrix of 16-bit numbers, two neighbours of row lane / 4 per lane
__device__ __forceinline__ uint32_t transposed8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// loads that are made where `there` holds, and zeros elsewhere, without a choice after the load, which would wait for it
template <int N> __device__ __forceinline__ void load_where(uint32_t (&v)[N], const void* p, bool there) {
    if constexpr (N == 4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t@p ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}"
                     : "=&r"(v[0]), "=&r"(v[1]), "=&r"(v[2]), "=&r"(v[3])
                     : "l"(p), "r"((uint32_t)there)
                     : "memory");
    else if constexpr (N == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t@p ld.global.v2.u32 {%0,%1}, [%2];\n\t}" : "=&r"(v[0]), "=&r"(v[1]) : "l"(p), "r"((uint32_t)there) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.u32 %0, 0;\n\t@p ld.global.u32 %0, [%1];\n\t}" : "=&r"(v[0]) : "l"(p), "r"((uint32_t)there) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void lds(uint32_t (&v)[N], uint32_t at) {
    if constexpr (N == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
    else if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at) : "memory");
    else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(at) : "memory");
}

// a stage of a warp's ring: 16 key rows as they are, 16 value rows in 16-byte pieces, 16 + 16 scales.  Piece q of value row r is at q4_piece(r, q): the words that a step reads together (rows of one
// parity and half, neighbouring words) are in different banks.
template <int HD> struct Q4Stage {
    static constexpr int ROW = HD / 2, V = 16 * ROW, KS = 32 * ROW, VS = KS + 64, BYTES = KS + 128;
};
__device__ __forceinline__ int q4_piece(int row, int q) { return (((row & 1) | ((row >> 3) & 1) << 1 | (q >> 1) << 2) << 3) | (q & 1) | ((row >> 1) & 3) << 1; }

template <int HD, int W, int U> struct Q4Smem {      // (the warps' sums lie over the drained ring)
    static constexpr int TILE = 16 * W * U, STAGES = QA_STAGES, RING = W * STAGES * U * Q4Stage<HD>::BYTES, MERGE = W * QA_ROWS * (HD + 4) * 4 + W * QA_ROWS * 16, BYTES = RING > MERGE ? RING : MERGE;
};

template <typename T, int HD, int W, int U> __global__ void __launch_bounds__(32 * W, QA_WARPS / W) attention_q4_kernel(const b200_q4_attention a, uint64_t page16, int64_t limit) {
    using St = Q4Stage<HD>;
    using Sm = Q4Smem<HD, W, U>;
    constexpr int STAGES = Sm::STAGES, TILE = Sm::TILE, WORDS = HD / 32, NT = HD / 16;      // words of a key row per lane; row tiles of the values
    constexpr bool Q2 = sizeof(T) == 4;
    before();
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ long long s_sum[W];
    __shared__ int s_item[4];      // sequence, row block, head, unit of the item
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int nkv = a.cache.n_kv_heads, G = a.n_heads / nkv, page_size = a.cache.page_size;

    // ---- the line of all tiles, and where this block's stretch begins
    const int chunk = (a.seqs + 32 * W - 1) / (32 * W), s_beg = min(a.seqs, tid * chunk), s_end = min(a.seqs, s_beg + chunk);
    auto tiles_of = [&](const Q4Seq& q) {
        long long n = 0;
        for (int rb = 0; rb * QA_ROWS < q.count * G; rb++) n += QA_START + q4_span<TILE>(a, q, G, rb).tiles;
        return n * nkv;
    };
    long long mine = 0;
    for (int s = s_beg; s < s_end; s++) mine += tiles_of(q4_seq(a, s, blockIdx.x == 0, limit));
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) s_sum[warp] = before;
    __syncthreads();
    long long total = 0;
    before -= mine;
#pragma unroll
    for (int w = 0; w < W; w++) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    const long long grid = min((long long)gridDim.x, total);
    Q4End* ends = reinterpret_cast<Q4End*>(reinterpret_cast<float*>(a.workspace) + (size_t)gridDim.x * 2 * q4_part_floats<HD>()) + blockIdx.x;
    if (blockIdx.x >= grid) {      // (the whole block)
        if (tid == 0) ends->rows = 0;
        return;
    }
    const long long c0 = q4_begin(total, blockIdx.x, (int)grid), c1 = q4_begin(total, blockIdx.x + 1, (int)grid);
    if (before <= c0 && c0 < before + mine) {
        long long at = c0 - before;
        for (int s = s_beg; s < s_end; s++) {
            const Q4Seq q = q4_seq(a, s, false, limit);
            const long long n = tiles_of(q);
            if (at >= n) { at -= n; continue; }
            for (int rb = 0;; rb++) {
                const int per = QA_START + q4_span<TILE>(a, q, G, rb).tiles;
                if (at >= (long long)per * nkv) { at -= (long long)per * nkv; continue; }
                s_item[0] = s;
                s_item[1] = rb;
                const int head = (int)(at >> 32 ? at / per : (uint32_t)at / (uint32_t)per);
                s_item[2] = head;
                s_item[3] = (int)(at - (long long)head * per);
                break;
            }
            break;
        }
    }
    __syncthreads();
    int s = s_item[0], rb = s_item[1], h = s_item[2], unit = s_item[3];

    const uint32_t ring = sm_u32(smem) + warp * STAGES * U * St::BYTES;
    float* merge = reinterpret_cast<float*>(smem);                        // [W][8][HD + 4]
    float* stat = merge + W * QA_ROWS * (HD + 4);                         // [W][8][4]
    // where this lane's words of a stage are: keys of positions g and g + 8; values of positions 2 c + (0, 1, 8, 9), words g and g + 8
    const uint32_t k_at = g * St::ROW + c * (WORDS * 4), v_at = St::V + q4_piece(2 * c, g >> 2) * 16 + (g & 3) * 4;
    constexpr int P = St::ROW / 16;                                       // pieces of a row
    // where it puts what it fetches, and from which offsets of a kv head's block (lane * 16 into the rows of a position)
    const uint32_t v_to = St::V + q4_piece(lane / P, lane % P) * 16;
    const int block = page_size * (HD + 8), page_bytes = nkv * block, v_off = page_size * St::ROW, s_off = 2 * v_off + (lane < 4 ? 0 : page_size * 4 - 64);
    const unsigned n_pages = (unsigned)a.cache.n_pages;
    const int tile_pages = TILE / page_size, tile_rows = TILE - tile_pages * page_size;
    Q4Seq q = q4_seq(a, s, false, limit);
    bool first = true;      // no part of this block's yet
    Q4End end{};
    auto next_item = [&]() {
        unit = 0;
        if (++h == nkv) {
            h = 0;
            rb++;
            while (rb * QA_ROWS >= q.count * G) {      // (there is one: the line goes on)
                rb = 0;
                q = q4_seq(a, ++s, false, limit);
            }
        }
    };
    for (long long cur = c0; cur < c1;) {
        const Q4Span sp = q4_span<TILE>(a, q, G, rb);
        const int unit_end = (int)min((long long)sp.tiles + QA_START, unit + (c1 - cur)), tile = max(0, unit - QA_START), stop = max(0, unit_end - QA_START);
        const long long start = cur - unit;      // the item's first unit
        cur += unit_end - unit;
        if (stop == tile) {                      // (nothing but units of the start)
            if (cur < c1) next_item();
            continue;
        }

        // ---- the ring.  The page of a step is looked up one step before its rows are asked for.
        const int32_t* table = a.page_table + (int64_t)s * a.table_stride;
        const uint8_t* mine_k = reinterpret_cast<const uint8_t*>(a.cache.data) + (int64_t)h * block + lane * 16;
        int p_look = sp.base + tile * TILE + warp * 16 * U, index = (int)(((uint64_t)(p_look >> 4) * page16) >> 36), row_look = p_look - index * page_size;
        int p_fetch = p_look, page[U], row[U];
        const int p_stop = min(sp.hi, sp.base + stop * TILE);
        bool odd_page = false;      // a page that is none of the cache's came by in this item
#pragma unroll
        for (int b = 0; b < U; b++) page[b] = row[b] = 0;
        auto look = [&]() {
#pragma unroll
            for (int b = 0; b < U; b++) {
                int over = 0;      // pages further on
                row[b] = row_look + 16 * b;
#pragma unroll
                for (int i = 0; i < b; i++)
                    if (row[b] >= page_size) {
                        row[b] -= page_size;
                        over++;
                    }
                uint32_t got[1];
                load_where<1>(got, table + index + over, p_look + 16 * b < p_stop);
                page[b] = (int)got[0];
            }
            p_look += TILE;
            index += tile_pages;
            row_look += tile_rows;
            if (row_look >= page_size) {
                row_look -= page_size;
                index++;
            }
        };
        auto fetch = [&](int stage) {
#pragma unroll
            for (int b = 0; b < U; b++)
                if (p_fetch + 16 * b < p_stop) {
                    if ((unsigned)page[b] >= n_pages) {      // (masked below)
                        odd_page = true;
                        page[b] = 0;
                        if (a.status && lane == 0) atomicOr(a.status, (int)B200_STATUS_BAD_PAGE);
                    }
                    const uint8_t* k = mine_k + (int64_t)page[b] * page_bytes + row[b] * St::ROW;
                    const uint32_t at = ring + (stage * U + b) * St::BYTES;
#pragma unroll
                    for (int i = 0; i < 16 * P; i += 32) {
                        cp16(at + lane * 16 + i * 16, k + i * 16);
                        cp16(at + v_to + q4_piece(i / P, 0) * 16, k + v_off + i * 16);
                    }
                    // (lanes 0-3 key scales, 4-7 value scales, which follow page_size floats later: lane * 16 is in k, 64 of it too much for those)
                    if (lane < 8) cp16(at + St::KS + lane * 16, k - row[b] * (St::ROW - 4) + s_off);
                }
            cp_commit();
            p_fetch += TILE;
        };
        // the first steps' pages, the query row, the first steps' rows: each is asked for before the one ahead of it is there
        int pages[STAGES][U], rows[STAGES][U];
#pragma unroll
        for (int i = 0; i < STAGES; i++) {
            look();
#pragma unroll
            for (int b = 0; b < U; b++) {
                pages[i][b] = page[b];
                rows[i][b] = row[b];
            }
        }
        const int r = rb * QA_ROWS + g, token = r / G;
        const bool live = r < q.count * G;
        const int64_t pos = q.len - q.count + token;
        // (rows behind the last one compute along with the first: nothing of theirs is written)
        const int row_hi = live ? (int)max((int64_t)0, pos + 1) : INT32_MAX, row_lo = live && a.window > 0 ? (int)max((int64_t)0, pos + 1 - a.window) : 0;
        float x[HD / 4];
        const T* p = reinterpret_cast<const T*>(a.q) + (q.first + (live ? token : 0)) * a.q_token + (h * G + (live ? r - token * G : 0)) * a.q_head + c * (HD / 4);
        if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) load_n<T, HD / 4, true>(p, x);
        else load_n<T, HD / 4, false>(p, x);
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) {
#pragma unroll
            for (int b = 0; b < U; b++) {
                page[b] = pages[i][b];
                row[b] = rows[i][b];
            }
            fetch(i);
        }
#pragma unroll
        for (int b = 0; b < U; b++) {
            page[b] = pages[STAGES - 1][b];
            row[b] = rows[STAGES - 1][b];
        }

        // ---- query row g as operand; what scores of rows 2 c and 2 c + 1 need
        uint32_t qb[WORDS][2][2], ql[Q2 ? WORDS : 1][2][2];
        float alpha[2], q8[2], m[2], mr[2], l[2], acc[NT][4];
        int hi[2], lo[2], hi_min, lo_max;
        {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 4; i++) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // elements times 2^e are below 2^14: fp16 holds the fp16 of them and what that leaves over
            // (e is at most 140: two factors, each a number)
            const int e = top < INFINITY ? 140 - (int)(__float_as_uint(top) >> 23) : 0;
            const float e1 = __int_as_float((127 + e / 2) << 23), e2 = __int_as_float((127 + e - e / 2) << 23);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 4; i++) x[i] = x[i] * e1 * e2;
            auto part = [&](float u, float v, float f, uint32_t& first, uint32_t& second) {
                first = pack_h2(u * f, v * f);
                const float2 b = unpack_h2(first);
                sum += (b.x + b.y) / f;
                if (Q2) {
                    second = pack_h2(u * f - b.x, v * f - b.y);
                    const float2 d = unpack_h2(second);
                    sum += (d.x + d.y) / f;
                }
            };
#pragma unroll
            for (int j = 0; j < WORDS; j++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    part(x[8 * j + 2 * u], x[8 * j + 2 * u + 4], 1.0f, qb[j][u][0], ql[Q2 ? j : 0][u][0]);
                    part(x[8 * j + 2 * u + 1], x[8 * j + 2 * u + 5], 0.0625f, qb[j][u][1], ql[Q2 ? j : 0][u][1]);
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const float row_q8 = sum * (8.0f / 16384.0f);                  // in units of 2^-10: (sums of n 2^-24) * 2^10
            const float row_alpha = ldexpf(a.scale * 1.4426950408889634f, Q2 ? -e : 14 - e);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                q8[k] = __shfl_sync(0xffffffffu, row_q8, 4 * (2 * c + k));
                alpha[k] = __shfl_sync(0xffffffffu, row_alpha, 4 * (2 * c + k));
                hi[k] = __shfl_sync(0xffffffffu, row_hi, 4 * (2 * c + k));
                lo[k] = __shfl_sync(0xffffffffu, row_lo, 4 * (2 * c + k));
                m[k] = mr[k] = -INFINITY;
                l[k] = 0.0f;
            }
            hi_min = __reduce_min_sync(0xffffffffu, row_hi);
            lo_max = __reduce_max_sync(0xffffffffu, row_lo);
        }
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) acc[i][k] = 0.0f;

        int stage = 0, stage_to = STAGES - 1;
        uint32_t magic = 0x64006400u;
        asm("" : "+r"(magic));      // (kept in a register: an instruction has room for one constant)
        for (int p0 = sp.base + tile * TILE + warp * 16 * U; p0 < p_stop; p0 += TILE) {
            cp_wait<STAGES - 2>();
            __syncwarp();
            fetch(stage_to);
            look();
            const uint32_t at0 = ring + stage * U * St::BYTES;
            stage_to = stage;
            stage = stage == STAGES - 1 ? 0 : stage + 1;
            // scores: [16 positions][position g, g + 8][row 2 c, 2 c + 1]
            float z[U][2][2];
            uint32_t vs[U][2];
#pragma unroll
            for (int b = 0; b < U; b++) {
                const uint32_t at = at0 + b * St::BYTES;
                uint32_t w[2][WORDS], ks[2][1];
                float d[4];
#pragma unroll
                for (int u = 0; u < 2; u++) lds<WORDS>(w[u], at + k_at + u * 8 * St::ROW);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t v[1];
                    lds<1>(ks[u], at + St::KS + (8 * u + g) * 4);
                    lds<1>(v, at + St::VS + (8 * u + g) * 4);
                    vs[b][u] = v[0];
                }
#pragma unroll
                for (int j = 0; j < WORDS; j++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const uint32_t x = t ? w[0][j] >> 8 : w[0][j], y = t ? w[1][j] >> 8 : w[1][j];
                        const uint32_t k0 = Q2 ? sub_h2(masked_or(x, 0x000f000fu, magic), 0x64086408u) : x & 0x000f000fu, k1 = Q2 ? sub_h2(masked_or(y, 0x000f000fu, magic), 0x64086408u) : y & 0x000f000fu;
                        const uint32_t k2 = Q2 ? sub_h2(masked_or(x, 0x00f000f0u, magic), 0x64806480u) : x & 0x00f000f0u, k3 = Q2 ? sub_h2(masked_or(y, 0x00f000f0u, magic), 0x64806480u) : y & 0x00f000f0u;
                        if (j + t == 0) mma16_first(d, k0, k1, k2, k3, qb[j][t][0], qb[j][t][1]);
                        else mma16(d, k0, k1, k2, k3, qb[j][t][0], qb[j][t][1]);
                        if (Q2) mma16(d, k0, k1, k2, k3, ql[Q2 ? j : 0][t][0], ql[Q2 ? j : 0][t][1]);
                    }
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int k = 0; k < 2; k++) z[b][u][k] = (Q2 ? d[2 * u + k] * alpha[k] : fmaf(d[2 * u + k], 1024.0f, -q8[k]) * alpha[k]) * __uint_as_float(ks[u][0]);
            }
            const bool all = !odd_page && p0 >= lo_max && p0 + 16 * U <= hi_min;
            uint32_t hidden = 0;      // bit 4 b + 2 u + k
            if (!all) {               // (uniform)
#pragma unroll
                for (int b = 0; b < U; b++) {
                    // (a block of 16 behind the stop was not fetched)
                    const bool there = p0 + 16 * b < p_stop && (unsigned)table[(int)(((uint64_t)((p0 + 16 * b) >> 4) * page16) >> 36)] < n_pages;
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int j = p0 + 16 * b + 8 * u + g;
                        // (a scale of a position that nobody sees may be NaN)
                        if (!there || !((j >= lo[0] && j < hi[0]) || (j >= lo[1] && j < hi[1]))) vs[b][u] = 0;
#pragma unroll
                        for (int k = 0; k < 2; k++)
                            if (!there || j < lo[k] || j >= hi[k]) {
                                z[b][u][k] = -INFINITY;
                                hidden |= 1u << (4 * b + 2 * u + k);
                            }
                    }
                }
            }
            float x[U][2][2], y[U][2][2], ex[U][2];      // log2 p, log2 of the weight's magnitude, log2 of the value's scale
            bool past = false;
#pragma unroll
            for (int b = 0; b < U; b++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    // (a scale of zero: as 2^-1000, which leaves nothing of it; NaN stays)
                    asm("{\n\t.reg .f32 t;\n\tlg2.approx.f32 t, %1;\n\tmax.NaN.f32 %0, t, 0fC47A0000;\n\t}" : "=f"(ex[b][u]) : "f"(fabsf(__uint_as_float(vs[b][u]))));
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        x[b][u][k] = z[b][u][k] - m[k];
                        y[b][u][k] = x[b][u][k] + (ex[b][u] - mr[k]);
                        past |= x[b][u][k] > 8.0f || y[b][u][k] > 8.0f + QA_UP;
                    }
                }
            if (__any_sync(0xffffffffu, past)) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float top = z[0][0][k];
#pragma unroll
                    for (int b = 0; b < U; b++) top = fmaxf(top, fmaxf(z[b][0][k], z[b][1][k]));
#pragma unroll
                    for (int o = 4; o <= 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    top = fmaxf(top, m[k]);
                    const float up = below(m[k], top), was = mr[k] + up;
                    float topr = -INFINITY;
#pragma unroll
                    for (int b = 0; b < U; b++) topr = fmaxf(topr, fmaxf(z[b][0][k] - top + ex[b][0], z[b][1][k] - top + ex[b][1]));
#pragma unroll
                    for (int o = 4; o <= 16; o <<= 1) topr = fmaxf(topr, __shfl_xor_sync(0xffffffffu, topr, o));
                    topr = fmaxf(topr - QA_UP, was);
                    l[k] *= ex2(up);
                    const float f = ex2(below(was, topr));
#pragma unroll
                    for (int i = 0; i < NT; i++) {
                        acc[i][k] *= f;
                        acc[i][k + 2] *= f;
                    }
                    m[k] = top;
                    mr[k] = topr;
#pragma unroll
                    for (int b = 0; b < U; b++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            x[b][u][k] = z[b][u][k] - top;
                            y[b][u][k] = x[b][u][k] + (ex[b][u] - topr);
                        }
                }
            }
            if (!all) {      // (a row that has seen nothing yet has no reference, and a scale that another row sees may be NaN)
#pragma unroll
                for (int b = 0; b < U; b++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int k = 0; k < 2; k++)
                            if ((hidden >> (4 * b + 2 * u + k)) & 1u) x[b][u][k] = y[b][u][k] = -INFINITY;
            }
#pragma unroll
            for (int b = 0; b < U; b++) {
                const uint32_t at = at0 + b * St::BYTES;
                uint32_t pb[2], pl[2];      // the weights of positions 2 c, 2 c + 1 (+ 8) for row g, and what their fp16 leave over
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    float w[2];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        l[k] += ex2(x[b][u][k]);
                        w[k] = __uint_as_float(__float_as_uint(ex2(y[b][u][k])) ^ (vs[b][u] & 0x80000000u));
                    }
                    pb[u] = pack_h2(w[0], w[1]);
                    const float2 f = unpack_h2(pb[u]);
                    pl[u] = transposed8x8(pack_h2(w[0] - f.x, w[1] - f.y));
                    pb[u] = transposed8x8(pb[u]);
                }
                // values: [positions 2 c, 2 c + 1; + 8][word g, word g + 8], channels 0-3 and 4-7 of the word
                uint32_t t[HD / 64][2][2];
#pragma unroll
                for (int half = 0; half < HD / 64; half++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        uint32_t w0[1], w1[1];
                        lds<1>(w0, at + v_at + q4_piece(8 * u, 2 * half) * 16);
                        lds<1>(w1, at + v_at + q4_piece(8 * u + 1, 2 * half) * 16);
                        t[half][u][0] = __byte_perm(w0[0], w1[0], 0x5410);
                        t[half][u][1] = __byte_perm(w0[0], w1[0], 0x7632);
                    }
                // nibble i of its word; odd ones 16 times too large, which is put right at the end
                auto nibble = [&](int half, int u, int i) {
                    const uint32_t v = (i & 2) ? t[half][u][i >> 2] >> 8 : t[half][u][i >> 2];
                    return sub_h2(masked_or(v, (i & 1) ? 0x00f000f0u : 0x000f000fu, magic), (i & 1) ? 0x64806480u : 0x64086408u);
                };
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    uint32_t v[4];      // rows g of the tile: word g, nibble i; rows g + 8: word g + 8 (hd 64: nibble i + 4)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        v[2 * u] = nibble(0, u, i);
                        v[2 * u + 1] = HD == 128 ? nibble(HD / 64 - 1, u, i) : nibble(0, u, i + 4);
                    }
                    mma16(acc[i], v[0], v[1], v[2], v[3], pb[0], pb[1]);
                    mma16(acc[i], v[0], v[1], v[2], v[3], pl[0], pl[1]);
                }
            }
        }
        cp_wait<0>();
        __syncthreads();

        // ---- the warps' sums into one
#pragma unroll
        for (int k = 0; k < 2; k++) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], o);
            if (g == 0) *reinterpret_cast<float4*>(stat + (warp * QA_ROWS + 2 * c + k) * 4) = make_float4(m[k], mr[k], l[k], 0.0f);
            float* to = merge + (warp * QA_ROWS + 2 * c + k) * (HD + 4) + 8 * g;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const float f = (i & 1) ? 0.0625f : 1.0f;
                to[i] = acc[i][k] * f;
                to[HD == 128 ? 64 + i : 4 + i] = acc[i][k + 2] * f;
            }
        }
        __syncthreads();
        const bool whole = tile == 0 && stop == sp.tiles;
        float* part = reinterpret_cast<float*>(a.workspace) + ((size_t)blockIdx.x * 2 + (first ? 0 : 1)) * q4_part_floats<HD>();
        for (int i = tid; i < QA_ROWS * (HD / 4); i += 32 * W) {
            const int row = i / (HD / 4), ch = (i % (HD / 4)) * 4;
            float top = -INFINITY, topr = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) top = fmaxf(top, stat[(w * QA_ROWS + row) * 4]);
#pragma unroll
            for (int w = 0; w < W; w++) topr = fmaxf(topr, stat[(w * QA_ROWS + row) * 4 + 1] + below(stat[(w * QA_ROWS + row) * 4], top));
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float4 st = *reinterpret_cast<const float4*>(stat + (w * QA_ROWS + row) * 4), v = *reinterpret_cast<const float4*>(merge + (w * QA_ROWS + row) * (HD + 4) + ch);
                const float d = below(st.x, top), f = ex2(below(st.y + d, topr));
                sum += st.z * ex2(d);
                o.x += v.x * f;
                o.y += v.y * f;
                o.z += v.z * f;
                o.w += v.w * f;
            }
            if (whole) {
                const int rr = rb * QA_ROWS + row;
                if (rr < q.count * G) {
                    // (l = 0: the row saw nothing, and the sums are zeros)
                    const float f = sum == 0.0f ? 0.0f : 1.0f / sum, e = topr == -INFINITY ? 0.0f : topr;
                    const float v[4] = {o.x, o.y, o.z, o.w};
                    T* p = reinterpret_cast<T*>(a.out) + (q.first + rr / G) * a.out_token + (h * G + rr % G) * a.out_head + ch;
#pragma unroll
                    for (int k = 0; k < 4; k++) p[k] = from_f<T>(sum == 0.0f ? 0.0f : ldexpf(v[k] * f, (int)floorf(e)) * ex2(e - floorf(e)));
                }
            } else {
                *reinterpret_cast<float4*>(part + row * HD + ch) = o;
                if (ch == 0) *reinterpret_cast<float4*>(part + QA_ROWS * HD + row * 4) = make_float4(top, topr, sum, 0.0f);
            }
        }
        if (first && tile > 0 && stop == sp.tiles) {      // (a part, and the last one)
            // the block that has the first tile; this item is its first one unless its stretch begins ahead of the item
            end.first_cta = (int)(((start + QA_START + 1) * grid - 1) / total);
            end.first_slot = q4_begin(total, end.first_cta, (int)grid) < start;
            end.token = q.first;
            end.rb = rb;
            end.head = h;
            end.rows = min((int)QA_ROWS, q.count * G - rb * QA_ROWS);
        }
        first = false;
        __syncthreads();
        if (cur < c1) next_item();
    }
    if (tid == 0) *ends = end;
}

// Joins the parts of the items that ended in a block's first stretch: block (x, y) = that block, a row.
template <typename T, int HD> __global__ void __launch_bounds__(256) attention_q4_join_kernel(const b200_q4_attention a, int grid) {
    before();
    constexpr int LANES = HD / 4, GROUPS = 256 / LANES, PART = q4_part_floats<HD>(), AHEAD = 8;
    __shared__ __align__(16) float s_o[GROUPS][HD];
    __shared__ float s_l[GROUPS];
    const float* ws = reinterpret_cast<const float*>(a.workspace);
    const Q4End e = reinterpret_cast<const Q4End*>(ws + (size_t)grid * 2 * PART)[blockIdx.x];
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, n = (int)blockIdx.x - e.first_cta + 1, G = a.n_heads / a.cache.n_kv_heads, rr = e.rb * QA_ROWS + row;
    if (row >= e.rows) return;
    auto part = [&](int i) { return ws + ((size_t)(e.first_cta + i) * 2 + (i == 0 ? e.first_slot : 0)) * PART; };
    // every group's first parts are asked for before anything waits
    float4 st[AHEAD], v[AHEAD];
    auto ask = [&](int i0) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int i = i0 + u * GROUPS;
            if (i < n) {
                st[u] = *reinterpret_cast<const float4*>(part(i) + QA_ROWS * HD + row * 4);
                v[u] = *reinterpret_cast<const float4*>(part(i) + row * HD + (tid % LANES) * 4);
            }
        }
    };
    ask(tid / LANES);
    float top = -INFINITY, topr = -INFINITY, sum = 0.0f;
    // (a warp has both maxima by itself: no exchange between warps)
#pragma unroll 4
    for (int i = lane; i < n; i += 32) {
        const float2 x = *reinterpret_cast<const float2*>(part(i) + QA_ROWS * HD + row * 4);
        const float was = top;
        top = fmaxf(top, x.x);
        topr = fmaxf(topr + below(was, top), x.y + below(x.x, top));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float x = __shfl_xor_sync(0xffffffffu, top, o), y = __shfl_xor_sync(0xffffffffu, topr, o), was = top;
        top = fmaxf(top, x);
        topr = fmaxf(topr + below(was, top), y + below(x, top));
    }
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = tid / LANES; i0 < n; i0 += AHEAD * GROUPS) {
        if (i0 >= AHEAD * GROUPS) ask(i0);
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
            if (i0 + u * GROUPS < n) {
                const float d = below(st[u].x, top), f = ex2(below(st[u].y + d, topr));
                sum += st[u].z * ex2(d);
                o.x += v[u].x * f;
                o.y += v[u].y * f;
                o.z += v[u].z * f;
                o.w += v[u].w * f;
            }
    }
    *reinterpret_cast<float4*>(&s_o[tid / LANES][(tid % LANES) * 4]) = o;
    if (tid % LANES == 0) s_l[tid / LANES] = sum;
    __syncthreads();
    if (tid < HD) {
        float x = 0.0f, l = 0.0f;
#pragma unroll
        for (int k = 0; k < GROUPS; k++) {
            x += s_o[k][tid];
            l += s_l[k];
        }
        const float r = topr == -INFINITY ? 0.0f : topr;
        reinterpret_cast<T*>(a.out)[(int64_t)(e.token + rr / G) * a.out_token + (e.head * G + rr % G) * a.out_head + tid] =
            from_f<T>(l == 0.0f ? 0.0f : ldexpf(x * (1.0f / l), (int)floorf(r)) * ex2(r - floorf(r)));
    }
}

// ------------------------------------------------------------------------------------------------------------------- host
constexpr int QA_W = 4, QA_U = 2;      // warps of a block, 16 positions a warp takes at a time
// blocks of the first kernel: as many as run at once on 148 SMs, fewer where even one tile each could not be found
inline int attention_q4_grid(const b200_q4_attention& a) {
    const int64_t G = a.n_heads / a.cache.n_kv_heads, blocks = (a.tokens * G + QA_ROWS - 1) / QA_ROWS + a.seqs;
    const int64_t tiles = blocks * a.cache.n_kv_heads * (((int64_t)a.table_pages * a.cache.page_size + 16 * QA_W * QA_U - 1) / (16 * QA_W * QA_U) + 1 + QA_START);
    return (int)std::min<int64_t>(148 * (QA_WARPS / QA_W), tiles);
}
inline size_t attention_q4_workspace(const b200_q4_attention& a) {
    const size_t grid = (size_t)attention_q4_grid(a), part = QA_ROWS * (a.cache.head_dim + 4) * 4;
    return grid * (2 * part + sizeof(Q4End));
}
// limit: sequences with more rows are left out
template <typename T, int HD> cudaError_t attention_q4_rows(const b200_q4_attention& a, int64_t limit, cudaStream_t st) {
    using Sm = Q4Smem<HD, QA_W, QA_U>;
    static SmemAllowed allowed;
    const auto kernel = attention_q4_kernel<T, HD, QA_W, QA_U>;
    cudaError_t e = allowed((const void*)kernel, Sm::BYTES);
    if (e != cudaSuccess) return e;
    const uint64_t d = (uint64_t)a.cache.page_size / 16, page16 = (((uint64_t)1 << 36) + d - 1) / d;      // n / d = n * page16 >> 36 for n < 2^27
    const int grid = attention_q4_grid(a);
    e = launch(kernel, dim3(grid), 32 * QA_W, Sm::BYTES, 1, st, a, page16, limit);
    if (e != cudaSuccess) return e;
    return launch(attention_q4_join_kernel<T, HD>, dim3(grid, (unsigned)std::min<int64_t>(QA_ROWS, a.q_starts ? QA_ROWS : a.n_heads / a.cache.n_kv_heads)), 256, 0, 1, st, a, grid);
}

}  // namespace dev
