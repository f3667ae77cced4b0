// dev_mat_i4.cuh — product of rows in 8 bits with 4-bit weights that have a scale per group of channels, of one matrix or of each token's experts (b200_dev_mat_mat_i4).
//
// out[p][n] = a_scales[r] * sum_g ws[e][n][g] * (sum over the channels k of group g of a[r][k] * w[e][n][k]) + bias[e][n], r the row of a and e the expert of output row p.
// The inner sums are integers and exact; the outer one is f32, in an order that the sizes decide and, with experts, how many pairs each expert has (columns of a unit, and where warps and blocks cut a unit's channels).
//
// A tile of weights is 16 rows x 64 channels in 512 bytes, placed so that the 16 bytes of a lane are the operands of two mma.m16n8k32 (s8, s32 sums): a word has four channels in the low
// halves of its bytes and the next four in the high halves; (word << 4) & 0xf0f0f0f0 and word & 0xf0f0f0f0 are those values times sixteen as signed bytes, three instructions for eight weights.  Eight rows of a are
// the columns.
//
// Work.  A unit is one or eight tiles of weight rows and as many rows of a as the kernel takes at once.  Each lane copies the bytes that it will read itself into a ring in shared memory (cp.async), some steps ahead, so that no warp waits
// for another's weights.  With experts every block lists the pairs (token, expert) by expert first, all in the same order; up to that many pairs of an expert are a unit for each tile.
//   few rows (up to 16): the weights' bytes.  Two blocks per SM have consecutive units of one tile each; its warps share their steps of 256 channels evenly, whichever unit they are of, and leave the sums of a unit that two or
//   more warps have a part of in shared memory for the end.  Rows of a come from L1 and L2.
//   more rows (up to 64 at a time): rows of a cost as much as weights.  A block has eight tiles; its teams of four warps have a part of the channels each, whose rows of a serve all eight.  With few units the
//   blocks of a cluster share the channels of one.
// What bounds it.  Few rows: the weights' bytes from some 30 MB on (one token through two of eight experts, 28672 x 4096 in groups of 32 with f16 scales: 25.2 us for 132 MB, 5.2 TB/s, of which 6.5 us are launch, list, first bytes and the last
// sums; 4096 to 8192 channels of one matrix add 66 MB in 10 us), below that the launch and a chain of loads (6144 x 4096: 7.0 us; a call of nothing 3.4).  Sixteen tokens' units of up to eight rows: waits for rows of a
// and issue slots (55 %), 50 to 58 us for 263 MB, by what the tokens choose.  More rows: the latency of a team's step, with issue slots at 44 % (33 rows of 4096 x 14336 20.4 us, of 8192 x 28672 56, 2.2 TB/s; the integer pipe is active 24 %).  Measured on the way: loads to registers, two steps ahead, 55 us (token, two experts);
// the ring, 64-bit arithmetic in every unit, 47; shared steps 38; several groups in the columns 26.  More rows: rows of a from L1 51 us (33 rows); a ring of four tiles a warp 33; sixteen warps on one step 25; teams of eight
// warps with one tile 24, of four with two 20; a warp that copies for all by bulk copies (of 128 bytes for a row) 73.  Copies with nothing computed per step but an addition took 100 instructions a step off.
#pragma once
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dev_common.cuh"
#include "dev_mat_i4_plan.cuh"

namespace dev {

struct MatI4Args {
    const int8_t* a;
    const float* a_scales;
    const uint8_t* w;
    const void* ws;
    const float* bias;
    const int32_t* experts;
    void* out;
    int32_t* status;
    int64_t lda, ldo;
    int rows, k, n, div, n_experts, steps, groups, tiles;      // rows of out; row p of out is of row p / div of a; steps of 64 channels
    uint32_t out_type;
    int tokens;     // rows of `experts`
    int first;      // the first row of out that this launch makes; `rows` counts from there
    int split;      // blocks of a cluster, which share a unit's channels
    int most, ring;      // more rows: rows that a step has room for (a multiple of eight), steps of a team's ring
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// ... with sums that begin here
__device__ __forceinline__ void mma_s8_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ float i4_sum(int sum) { return (float)sum; }
// Pairs by expert, in shared memory: expert e's pairs are list[end[e - 1]] .. list[end[e] - 1] (those without an expert come last), its first chunk is chunk[e].
struct I4List {
    int *end, *chunk;
    uint16_t *list, *of;
};
__device__ __forceinline__ I4List i4_list(void* smem, const MatI4Args& a) {
    int* p = reinterpret_cast<int*>(smem);
    uint16_t* q = reinterpret_cast<uint16_t*>(p + 2 * (a.n_experts + 2));
    return I4List{p, p + a.n_experts + 2, q, q + a.rows};
}
__device__ __forceinline__ void i4_lists(const MatI4Args& a, const I4List& l, int per_chunk) {
    const int E = a.n_experts + 1, tid = threadIdx.x, lane = tid & 31;
    for (int e = tid; e <= E; e += blockDim.x) l.end[e] = 0;
    __syncthreads();
    for (int p = tid; p < a.rows; p += blockDim.x) {
        const int x = a.experts[a.first + p], e = x >= 0 && x < a.n_experts ? x : a.n_experts;
        if (x < -1 || x >= a.n_experts) {
            if (a.status && blockIdx.x == 0) atomicOr(a.status, (int)B200_STATUS_BAD_EXPERT);
        }
        l.of[p] = (uint16_t)e;
        atomicAdd(&l.end[e], 1);
    }
    __syncthreads();
    if (tid < 32) {
        int pairs = 0, chunks = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int n = e0 + lane < E ? l.end[e0 + lane] : 0, c = e0 + lane < a.n_experts ? (n + per_chunk - 1) / per_chunk : 0;
            int sn = n, sc = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int un = __shfl_up_sync(0xffffffffu, sn, o), uc = __shfl_up_sync(0xffffffffu, sc, o);
                if (lane >= o) sn += un, sc += uc;
            }
            if (e0 + lane < E) {
                l.end[e0 + lane] = pairs + sn - n;
                l.chunk[e0 + lane] = chunks + sc - c;
            }
            pairs += __shfl_sync(0xffffffffu, sn, 31);
            chunks += __shfl_sync(0xffffffffu, sc, 31);
        }
        __syncwarp();
        // (in order of the pairs, so that all blocks have the same list; end[e] is counted up from where e's pairs begin)
        for (int p0 = 0; p0 < a.rows; p0 += 32) {
            const int p = p0 + lane, e = p < a.rows ? l.of[p] : -1;
            const uint32_t same = __match_any_sync(0xffffffffu, e), ahead = __popc(same & ((1u << lane) - 1));
            const int at = e >= 0 ? l.end[e] : 0;
            __syncwarp();
            if (e >= 0) {
                l.list[at + ahead] = (uint16_t)p;
                if (ahead == 0) l.end[e] = at + __popc(same);
            }
            __syncwarp();
        }
    }
    __syncthreads();
}
// A chunk: its expert, the first of its pairs (rows, without experts), how many.
struct I4Chunk {
    int e, lo, many;
};
template <int MOST> __device__ __forceinline__ I4Chunk i4_chunk(const MatI4Args& a, const I4List& l, int c) {
    if (!a.experts) return I4Chunk{0, c * MOST, min(MOST, a.rows - c * MOST)};
    int e = 0, top = a.n_experts;      // the last expert whose first chunk is not behind c: that one has it
    while (e < top) {
        const int mid = (e + top + 1) / 2;
        if (l.chunk[mid] <= c) e = mid;
        else top = mid - 1;
    }
    const int lo = (e ? l.end[e - 1] : 0) + (c - l.chunk[e]) * MOST;
    return I4Chunk{e, lo, min(MOST, l.end[e] - lo)};
}
__device__ __forceinline__ int i4_pair(const MatI4Args& a, const I4List& l, int i) { return a.experts ? l.list[i] : i; }
__device__ __forceinline__ float i4_row_scale(const MatI4Args& a, int p) { return a.a_scales[(a.first + p) / a.div]; }
__device__ __forceinline__ void i4_put(const MatI4Args& a, int e, int p, int n, float sum, float scale) {
    float y = (sum * 0.0625f) * scale;      // (the products are sixteen times the values; a scale may be as small as 2^-126, and a sixteenth of that has fewer bits)
    if (a.bias) y += a.bias[(int64_t)e * a.n + n];
    const int64_t to = (int64_t)(a.first + p) * a.ldo + n;
    if (a.out_type == B200_TYPE_F32) reinterpret_cast<float*>(a.out)[to] = y;
    else if (a.out_type == B200_TYPE_F16) reinterpret_cast<__half*>(a.out)[to] = __float2half_rn(y);
    else reinterpret_cast<__nv_bfloat16*>(a.out)[to] = __float2bfloat16_rn(y);
}
// zeros for the pairs without an expert; the blocks of the launch share them
__device__ __forceinline__ void i4_zeros(const MatI4Args& a, const I4List& l) {
    const int lo = l.end[a.n_experts - 1], hi = l.end[a.n_experts];
    for (int i = lo; i < hi; i++) {
        const int64_t to = (int64_t)(a.first + l.list[i]) * a.ldo;
        for (int n = blockIdx.x * blockDim.x + threadIdx.x; n < a.n; n += gridDim.x * blockDim.x) {
            if (a.out_type == B200_TYPE_F32) reinterpret_cast<float*>(a.out)[to + n] = 0.0f;
            else reinterpret_cast<uint16_t*>(a.out)[to + n] = 0;
        }
    }
}
// the scales of rows g and g + 8 of a tile for one group
template <typename S> __device__ __forceinline__ float2 i4_scales(const uint8_t* p) {
    struct __align__(2 * sizeof(S)) W { S lo, hi; };
    const W w = *reinterpret_cast<const W*>(p);
    return make_float2(to_f(w.lo), to_f(w.hi));
}
// A step of C tiles' channels of one tile of rows (i4_slot) copied to a ring, from w (this lane's 16 bytes of the step's first tile) and d (its 8 bytes of the scales).  A whole step, with nothing to be asked; and the last one of a tile, with zeros behind the last channel.
template <typename S, int GROUP, int C> __device__ __forceinline__ void i4_copy(uint32_t to, const uint8_t* w, const uint8_t* d, int lane) {
    constexpr int WORDS = 64 * C / GROUP * 2 * (int)sizeof(S);      // 8-byte words of the scales
#pragma unroll
    for (int c = 0; c < C; c++) copy_all<16>(to + c * I4_TILE + lane * 16, w + c * I4_TILE);
#pragma unroll
    for (int c = 0; c < WORDS; c += 32)
        if (c + 32 <= WORDS || lane < WORDS - c) copy_all<8>(to + C * I4_TILE + c * 8 + lane * 8, d + c * 8);
}
template <typename S, int GROUP, int C> __device__ __noinline__ void i4_copy_last(uint32_t to, const uint8_t* w, const uint8_t* d, int tiles, int groups, int lane) {      // how many there are left
    constexpr int WORDS = 64 * C / GROUP * 2 * (int)sizeof(S);
    const uint8_t* any = w - lane * 16;
    for (int c = 0; c < C; c++) copy_where<16>(to + c * I4_TILE + lane * 16, c < tiles ? w + c * I4_TILE : any, c < tiles);
    for (int c = lane; c < WORDS; c += 32) copy_where<8>(to + C * I4_TILE + c * 8, c < groups * 2 * (int)sizeof(S) ? d + (c - lane) * 8 : any, c < groups * 2 * (int)sizeof(S));
}

// ------------------------------------------------------------------------------------------------------------- few rows
// A step's sums of one tile with TC rows of a (1, 2, 4; 8: eight rows each in NT blocks of columns).  TC rows are TC of the eight columns; with fewer than eight the other columns take the same rows' other
// groups: column n has row n % TC and group n / TC of the (up to) 8 / TC that one set of sums has, so that what a group's sum costs afterwards (a conversion and a product in each lane) is paid once for all
// of them.  (One row in one column took 240 instructions for 128 channels.)
template <typename S, int GROUP, int TC, int NT> struct I4Step {
    static constexpr int GC = GROUP / 32, GS = 256 / GROUP, SETS = GS * TC > 8 ? GS * TC / 8 : 1, PER = GS / SETS;      // chunks (of 32 channels) of a group, groups of a step, sets of sums, groups of a set
    static constexpr int SB = 16 * (int)sizeof(S);
    uint2 b[NT][SETS * GC];
    // this lane's bytes of the rows; `at`: row g % TC, channel 8 t; columns that no group has, and channels behind the last one, are zeros
    __device__ __forceinline__ void load(const int8_t* const (&at)[NT], int s, int k, int g) {
        const int group = g / TC, from = s * 256 + group * GROUP;
        const bool used = PER * TC == 8 || group < PER;
        if ((s + 1) * 256 <= k) {
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int i = 0; i < SETS * GC; i++) b[j][i] = used ? *reinterpret_cast<const uint2*>(at[j] + from + i / GC * PER * GROUP + i % GC * 32) : make_uint2(0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int i = 0; i < SETS * GC; i++) {
                    const int ch = from + i / GC * PER * GROUP + i % GC * 32;
                    b[j][i] = used && ch < k ? *reinterpret_cast<const uint2*>(at[j] + ch) : make_uint2(0, 0);
                }
        }
    }
    __device__ __forceinline__ void add(float (&acc)[NT][4], const uint8_t* in, int lane) const {
        const int g = lane >> 2, t = lane & 3, group = g / TC;
        const uint8_t* scales = in + 4 * I4_TILE + g * 2 * sizeof(S);
        uint4 tile;
#pragma unroll
        for (int z = 0; z < SETS; z++) {
            int sum[NT][4];
#pragma unroll
            for (int i = 0; i < PER * GC; i++) {
                const int k = z * PER * GC + i;      // the chunk: half a tile
                if (k % 2 == 0) tile = *reinterpret_cast<const uint4*>(in + (k / 2) * I4_TILE + lane * 16);
                const uint2 v = k % 2 ? make_uint2(tile.z, tile.w) : make_uint2(tile.x, tile.y);
                const uint32_t a0 = (v.x << 4) & 0xf0f0f0f0u, a1 = (v.y << 4) & 0xf0f0f0f0u, a2 = v.x & 0xf0f0f0f0u, a3 = v.y & 0xf0f0f0f0u;
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const uint2 w = b[j][z * GC + i % GC];
                    const uint32_t b0 = PER == 1 || group == i / GC ? w.x : 0, b1 = PER == 1 || group == i / GC ? w.y : 0;
                    if (i == 0) mma_s8_first(sum[j], a0, a1, a2, a3, b0, b1);
                    else mma_s8(sum[j], a0, a1, a2, a3, b0, b1);
                }
            }
            // columns 2t and 2t + 1: one group's, but for TC = 1
            const int q0 = 2 * t / TC, q1 = (2 * t + 1) / TC;
            float2 d0 = i4_scales<S>(scales + (z * PER + (PER > 1 ? min(q0, PER - 1) : 0)) * SB), d1 = d0;
            if constexpr (TC == 1) d1 = i4_scales<S>(scales + (z * PER + (PER > 1 ? min(q1, PER - 1) : 0)) * SB);
            if constexpr (PER * TC < 8) {      // (columns that no group has)
                if (q0 >= PER) d0 = make_float2(0, 0);
                if (q1 >= PER) d1 = make_float2(0, 0);
            }
#pragma unroll
            for (int j = 0; j < NT; j++) {
                acc[j][0] = fmaf(d0.x, i4_sum(sum[j][0]), acc[j][0]);
                acc[j][1] = fmaf(d1.x, i4_sum(sum[j][1]), acc[j][1]);
                acc[j][2] = fmaf(d0.y, i4_sum(sum[j][2]), acc[j][2]);
                acc[j][3] = fmaf(d1.y, i4_sum(sum[j][3]), acc[j][3]);
            }
        }
    }
};

template <int NT> __host__ __device__ constexpr int i4_few_warps() { return NT == 1 ? 12 : 8; }
template <typename S, int GROUP, int NT> __global__ void __launch_bounds__(i4_few_warps<NT>() * 32, 2) mat_mat_i4_few_kernel(const MatI4Args a) {
    before();
    constexpr int SLOT = i4_slot(sizeof(S), GROUP, 4), SB = 16 * (int)sizeof(S), CHUNK = 8 * NT, WARPS = i4_few_warps<NT>();
    extern __shared__ __align__(16) uint8_t i4_smem[];
    float4* parts = reinterpret_cast<float4*>(i4_smem + WARPS * I4_RING * SLOT);      // [warps][its first unit, its last][NT][32]
    const I4List l = i4_list(parts + WARPS * 2 * NT * 32, a);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, whole = (a.steps + 3) / 4;
    const uint8_t* slots = i4_smem + warp * I4_RING * SLOT;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(slots);
    int chunks = (a.rows + CHUNK - 1) / CHUNK;
    if (a.experts) {
        i4_lists(a, l, CHUNK);
        chunks = l.chunk[a.n_experts];
        i4_zeros(a, l);
    }
    // this block's units (of fewer than 2^31, see mat_mat_i4), their steps one after the other, and this warp's of those
    const uint32_t units = (uint32_t)chunks * (uint32_t)a.tiles, each = units / gridDim.x, over = units - each * gridDim.x, u0 = each * blockIdx.x + min(over, blockIdx.x);
    const int many = (int)(each + (blockIdx.x < over)), steps = many * whole, part = steps / WARPS, rest = steps - part * WARPS;
    auto begin = [&](int w) { return part * w + min(rest, w); };
    // sums over a row's columns, and the results of a unit
    auto row_scales = [&](float2 (&d)[NT], const I4Chunk& x) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int col = 8 * j + 2 * t;
            d[j] = make_float2(col < x.many ? i4_row_scale(a, i4_pair(a, l, x.lo + col)) : 0.0f, col + 1 < x.many ? i4_row_scale(a, i4_pair(a, l, x.lo + col + 1)) : 0.0f);
        }
    };
    auto finish = [&](float4 (&y)[NT], const float2 (&d)[NT], const I4Chunk& x, int tile) {
        const int tc = x.many > 4 ? 8 : x.many > 2 ? 4 : x.many;      // (columns of one row are 1, 2, 4 apart)
        if (tc == 1) y[0].x += y[0].y, y[0].z += y[0].w;
        if (tc < 4) {
            y[0].x += __shfl_xor_sync(0xffffffffu, y[0].x, 1);
            y[0].y += __shfl_xor_sync(0xffffffffu, y[0].y, 1);
            y[0].z += __shfl_xor_sync(0xffffffffu, y[0].z, 1);
            y[0].w += __shfl_xor_sync(0xffffffffu, y[0].w, 1);
        }
        if (tc < 8) {
            y[0].x += __shfl_xor_sync(0xffffffffu, y[0].x, 2);
            y[0].y += __shfl_xor_sync(0xffffffffu, y[0].y, 2);
            y[0].z += __shfl_xor_sync(0xffffffffu, y[0].z, 2);
            y[0].w += __shfl_xor_sync(0xffffffffu, y[0].w, 2);
        }
        const int n = tile * 16 + g;
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const int col = 8 * j + 2 * t + q;
                if (col < x.many) {
                    const int p = i4_pair(a, l, x.lo + col);
                    if (n < a.n) i4_put(a, x.e, p, n, q ? y[j].y : y[j].x, q ? d[j].y : d[j].x);
                    if (n + 8 < a.n) i4_put(a, x.e, p, n + 8, q ? y[j].w : y[j].z, q ? d[j].y : d[j].x);
                }
            }
    };
    const int f0 = begin(warp), f1 = begin(warp + 1);
    if (f0 < f1) {
        const int v0 = f0 / whole;
        int c = (int)((u0 + v0) / (uint32_t)a.tiles), tile = (int)(u0 + v0 - (uint32_t)c * a.tiles), s = f0 - v0 * whole;
        I4Chunk x = i4_chunk<CHUNK>(a, l, c);
        // copies, I4_RING - 1 steps ahead of the products
        int cc = c, ct = tile, ce = x.e, cs = s, left = f1 - f0;
        const int full = a.k / 256;      // whole steps of a tile
        uint32_t into = ring;
        const uint8_t *cw = nullptr, *cd = nullptr;
        auto place = [&]() {
            const int64_t at = (int64_t)ce * a.tiles + ct;
            cw = a.w + (at * a.steps + cs * 4) * I4_TILE + lane * 16;
            cd = reinterpret_cast<const uint8_t*>(a.ws) + (at * a.groups + cs * (256 / GROUP)) * SB + lane * 8;
        };
        place();
        auto copy = [&]() {
            if (left > 0) {
                if (cs < full) i4_copy<S, GROUP, 4>(into, cw, cd, lane);
                else i4_copy_last<S, GROUP, 4>(into, cw, cd, a.steps - cs * 4, a.groups - cs * (256 / GROUP), lane);
                cw += 4 * I4_TILE;
                cd += 256 / GROUP * SB;
                into = into + SLOT == ring + I4_RING * SLOT ? ring : into + SLOT;
                left--;
                if (++cs == whole && left > 0) {
                    cs = 0;
                    if (++ct == a.tiles) {
                        ct = 0;
                        ce = i4_chunk<CHUNK>(a, l, ++cc).e;
                    }
                    place();
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < I4_RING - 1; i++) copy();
        const uint8_t* slot = slots;
        for (int f = f0; f < f1;) {
            const int sa = s, sb = min(whole, s + f1 - f);
            float acc[NT][4];
            float2 d[NT];
            row_scales(d, x);
#pragma unroll
            for (int j = 0; j < NT; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0;
            auto products = [&](auto step, auto& sums) {
                constexpr int N = sizeof(sums) / sizeof(sums[0]);
                const int tc = x.many > 4 ? 8 : x.many > 2 ? 4 : x.many;
                const int8_t* at[N];
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const int col = 8 * j + (g & (tc - 1));      // (columns without a row take another's: nothing reads their sums)
                    at[j] = a.a + (int64_t)((a.first + i4_pair(a, l, x.lo + (col < x.many ? col : 0))) / a.div) * a.lda + 8 * t;
                }
                for (; s < sb; s++) {
                    step.load(at, s, a.k, g);
                    asm volatile("cp.async.wait_group %0;" ::"n"(I4_RING - 2) : "memory");
                    __syncwarp();
                    copy();
                    step.add(sums, slot, lane);
                    slot = slot + SLOT == slots + I4_RING * SLOT ? slots : slot + SLOT;
                }
            };
            auto& one = reinterpret_cast<float(&)[1][4]>(acc);
            if (NT > 1 && x.many > 8) products(I4Step<S, GROUP, 8, NT>(), acc);
            else if (x.many > 4) products(I4Step<S, GROUP, 8, 1>(), one);
            else if (x.many > 2) products(I4Step<S, GROUP, 4, 1>(), one);
            else if (x.many > 1) products(I4Step<S, GROUP, 2, 1>(), one);
            else products(I4Step<S, GROUP, 1, 1>(), one);
            float4 y[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) y[j] = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
            if (sa == 0 && sb == whole) {
                finish(y, d, x, tile);
            } else {
#pragma unroll
                for (int j = 0; j < NT; j++) parts[((warp * 2 + (f != f0)) * NT + j) * 32 + lane] = y[j];
            }
            f += sb - sa;
            if (f < f1) {
                s = 0;
                if (++tile == a.tiles) {
                    tile = 0;
                    x = i4_chunk<CHUNK>(a, l, ++c);
                }
            }
        }
    }
    __syncthreads();
    // units that several warps have a part of, a warp for each; the parts are added in the order of the channels
    for (int v = warp; v < many; v += WARPS) {
        const int f = v * whole;
        int w = f < rest * (part + 1) ? f / (part + 1) : rest + (f - rest * (part + 1)) / part;      // the warp that has the unit's first step
        if (begin(w + 1) >= (v + 1) * whole) continue;      // one warp's: written
        float4 y[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) y[j] = make_float4(0, 0, 0, 0);
        for (; w < WARPS && begin(w) < (v + 1) * whole; w++) {
            const int b = begin(w);
            if (b == begin(w + 1)) continue;
            const int which = b / whole != v;
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const float4 z = parts[((w * 2 + which) * NT + j) * 32 + lane];
                y[j].x += z.x, y[j].y += z.y, y[j].z += z.z, y[j].w += z.w;
            }
        }
        const int c = (int)((u0 + v) / (uint32_t)a.tiles);
        const I4Chunk x = i4_chunk<CHUNK>(a, l, c);
        float2 d[NT];
        row_scales(d, x);
        finish(y, d, x, (int)(u0 + v - (uint32_t)c * a.tiles));
    }
}

// ------------------------------------------------------------------------------------------------------------- more rows
// Four teams of four warps; a team has a part of the channels, 128 at a time, and its own ring, so that the teams' copies, products and sums overlap.  A warp has two of the unit's eight tiles; the rows of a are the
// team's.  As many blocks of columns are computed as i4_many_blocks says, and a step has room for the rows of all of them (i4_many_plan).

template <typename S, int GROUP> __global__ void __launch_bounds__(I4_TEAMS * I4_TEAM_WARPS * 32, 1) mat_mat_i4_many_kernel(const MatI4Args a) {
    before();
    constexpr int T = I4_TEAM_TILES, WSLOT = i4_slot(sizeof(S), GROUP, 2), GS = 128 / GROUP, SB = 16 * (int)sizeof(S), GC = GROUP / 32;
    extern __shared__ __align__(16) uint8_t i4_smem[];
    __shared__ float s_scale[I4_MANY_ROWS];
    __shared__ int s_pair[I4_MANY_ROWS];      // the unit's rows of out, their scales, where their rows of a begin
    __shared__ int64_t s_from[I4_MANY_ROWS];
    const int RING = a.ring, SLOT = i4_many_slot(sizeof(S), GROUP, a.most), most_nt = a.most / 8;
    const I4List l = i4_list(i4_smem + I4_TEAMS * RING * SLOT, a);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, team = warp / I4_TEAM_WARPS, member = warp % I4_TEAM_WARPS, g = lane >> 2, t = lane & 3;
    uint8_t* slots = i4_smem + team * RING * SLOT;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(slots), wrap = ring + RING * SLOT;
    const int blocks = (a.tiles + T - 1) / T, whole = (a.steps + 1) / 2, full = a.k / 128;
    int chunks = (a.rows + I4_MANY_ROWS - 1) / I4_MANY_ROWS;
    if (a.experts) {
        i4_lists(a, l, I4_MANY_ROWS);
        chunks = l.chunk[a.n_experts];
        i4_zeros(a, l);
    }
    const int rank = blockIdx.x % a.split, parts = I4_TEAMS * a.split, part = rank * I4_TEAMS + team, s0 = (int)((int64_t)whole * part / parts), s1 = (int)((int64_t)whole * (part + 1) / parts);
    auto together = [&] { asm volatile("bar.sync %0, 128;" ::"r"(team + 1) : "memory"); };
    for (int64_t u = blockIdx.x / a.split; u < (int64_t)chunks * blocks; u += gridDim.x / a.split) {
        const int c = (int)(u / blocks), tile0 = (int)(u - (int64_t)c * blocks) * T;
        const I4Chunk x = i4_chunk<I4_MANY_ROWS>(a, l, c);
        const int nt = (x.many + 7) / 8;
        // this warp's tiles (where there are none others': nothing reads their sums), and the rows of a that this thread copies 16 bytes of: at the next step to be copied
        const int first = min(tile0 + member * 2, a.tiles - 1);
        const int64_t at = (int64_t)x.e * a.tiles + first, tile_w = first + 1 < a.tiles ? (int64_t)a.steps * I4_TILE : 0, tile_d = first + 1 < a.tiles ? (int64_t)a.groups * SB : 0;
        const uint8_t *w = a.w + (at * a.steps + 2 * s0) * I4_TILE + lane * 16, *d = reinterpret_cast<const uint8_t*>(a.ws) + (at * a.groups + s0 * GS) * SB + lane * 8;
        const int unit = tid & 7, row0 = (tid & 127) >> 3;
        const int8_t* from = a.a + s0 * 128 + unit * 16;
        if (tid < I4_MANY_ROWS) {
            const int p = i4_pair(a, l, x.lo + (tid < x.many ? tid : 0));
            s_pair[tid] = p;
            s_from[tid] = (int64_t)((a.first + p) / a.div) * a.lda;
            s_scale[tid] = i4_row_scale(a, p);
        }
        __syncthreads();
        // rows of 128 bytes; 16 bytes u of row i lie at u ^ (2 (i % 4)), so that the eight rows of a block of columns are read without bank conflicts
        const uint32_t row_to = T * WSLOT + row0 * 128 + ((unit ^ ((row0 & 3) << 1)) << 4), tile_to = member * 2 * WSLOT;
        int cs = s0;
        uint32_t into = ring;
        auto copy = [&]() {
            if (cs < s1) {
                const bool there = cs < full || cs * 128 + unit * 16 < a.k;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (i * 16 + row0 < nt * 8) copy_where<16>(into + row_to + i * 2048, there ? from + s_from[i * 16 + row0] : a.a, there);
                from += 128;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    if (cs < full) i4_copy<S, GROUP, 2>(into + tile_to + r * WSLOT, w + r * tile_w, d + r * tile_d, lane);
                    else i4_copy_last<S, GROUP, 2>(into + tile_to + r * WSLOT, w + r * tile_w, d + r * tile_d, a.steps - cs * 2, a.groups - cs * GS, lane);
                }
                w += 2 * I4_TILE;
                d += GS * SB;
                cs++;
                into = into + SLOT == wrap ? ring : into + SLOT;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int i = 0; i < RING - 1; i++) copy();
        auto products = [&](auto blocks_of_columns) {
            constexpr int N = decltype(blocks_of_columns)::value, AT_ONCE = N * GC > 12 ? 1 : 2;      // (both tiles at once, or one after the other where registers do not hold both)
            float acc[2][N][4];
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int j = 0; j < N; j++) acc[r][j][0] = acc[r][j][1] = acc[r][j][2] = acc[r][j][3] = 0;
            uint32_t slot = 0;
            for (int s = s0; s < s1; s++) {
                if (RING == 4) asm volatile("cp.async.wait_group 2;" ::: "memory");
                else if (RING == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
                else asm volatile("cp.async.wait_group 0;" ::: "memory");
                together();      // (all copies of this step are there, and all warps are done with the step before)
                copy();
                const uint8_t *in = slots + slot, *mine = in + tile_to, *rows = in + T * WSLOT + g * 128;
                slot = slot + SLOT == RING * SLOT ? 0 : slot + SLOT;
#pragma unroll
                for (int q = 0; q < GS; q++)
#pragma unroll
                    for (int r0 = 0; r0 < 2; r0 += AT_ONCE) {
                        uint32_t lo[AT_ONCE][2 * GC], hi[AT_ONCE][2 * GC];
                        float2 e[AT_ONCE];
#pragma unroll
                        for (int r = 0; r < AT_ONCE; r++) {
                            const uint8_t* tile = mine + (r0 + r) * WSLOT;
#pragma unroll
                            for (int i = 0; i < GC; i++) {
                                const int h = q * GC + i;
                                const uint2 v = *reinterpret_cast<const uint2*>(tile + (h / 2) * I4_TILE + lane * 16 + (h % 2) * 8);
                                lo[r][2 * i] = (v.x << 4) & 0xf0f0f0f0u, lo[r][2 * i + 1] = (v.y << 4) & 0xf0f0f0f0u;
                                hi[r][2 * i] = v.x & 0xf0f0f0f0u, hi[r][2 * i + 1] = v.y & 0xf0f0f0f0u;
                            }
                            e[r] = i4_scales<S>(tile + 2 * I4_TILE + q * SB + g * 2 * sizeof(S));
                        }
#pragma unroll
                        for (int j = 0; j < N; j++) {
                            uint2 b[GC];
#pragma unroll
                            for (int i = 0; i < GC; i++) b[i] = *reinterpret_cast<const uint2*>(rows + j * 1024 + ((((q * GC + i) * 2 + (t >> 1)) ^ ((g & 3) << 1)) << 4) + (t & 1) * 8);
#pragma unroll
                            for (int r = 0; r < AT_ONCE; r++) {
                                int sum[4];
#pragma unroll
                                for (int i = 0; i < GC; i++) {
                                    if (i == 0) mma_s8_first(sum, lo[r][0], lo[r][1], hi[r][0], hi[r][1], b[0].x, b[0].y);
                                    else mma_s8(sum, lo[r][2 * i], lo[r][2 * i + 1], hi[r][2 * i], hi[r][2 * i + 1], b[i].x, b[i].y);
                                }
                                float(&y)[4] = acc[r0 + r][j];
                                y[0] = fmaf(e[r].x, i4_sum(sum[0]), y[0]);
                                y[1] = fmaf(e[r].x, i4_sum(sum[1]), y[1]);
                                y[2] = fmaf(e[r].y, i4_sum(sum[2]), y[2]);
                                y[3] = fmaf(e[r].y, i4_sum(sum[3]), y[3]);
                            }
                        }
                    }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            together();
            // sums to the team's ring's place
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (j < nt) reinterpret_cast<float4*>(slots)[((member * 2 + r) * most_nt + j) * 32 + lane] = make_float4(acc[r][j][0], acc[r][j][1], acc[r][j][2], acc[r][j][3]);
        };
        auto columns = [](auto blocks) { return std::integral_constant<int, i4_many_blocks(decltype(blocks)::value)>(); };
        static_assert(i4_many_blocks(1) == i4_many_blocks(2) && i4_many_blocks(7) == i4_many_blocks(8), "one case each below");
        if (nt <= 2) products(columns(std::integral_constant<int, 2>()));
        else if (nt <= 3) products(columns(std::integral_constant<int, 3>()));
        else if (nt <= 4) products(columns(std::integral_constant<int, 4>()));
        else if (nt <= 5) products(columns(std::integral_constant<int, 5>()));
        else if (nt <= 6) products(columns(std::integral_constant<int, 6>()));
        else products(columns(std::integral_constant<int, 8>()));
        __syncwarp();
        if (a.split > 1) cluster_sync();
        else __syncthreads();
        // a warp for every tile and block of columns; the cluster's blocks take turns
        for (int o = warp * a.split + rank; o < T * nt; o += I4_TEAMS * I4_TEAM_WARPS * a.split) {
            const int i = o % T, j = o / T, col = 8 * j + 2 * t, n = (tile0 + i) * 16 + g;
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(i4_smem) + ((i * most_nt + j) * 32 + lane) * 16;
            float4 y = make_float4(0, 0, 0, 0);
            for (int b = 0; b < a.split; b++)
#pragma unroll
                for (int k = 0; k < I4_TEAMS; k++) {
                    const float4 z = peer_f32x4(at + k * RING * SLOT, b);
                    y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
                }
#pragma unroll
            for (int q = 0; q < 2; q++)
                if (col + q < x.many) {
                    if (n < a.n) i4_put(a, x.e, s_pair[col + q], n, q ? y.y : y.x, s_scale[col + q]);
                    if (n + 8 < a.n) i4_put(a, x.e, s_pair[col + q], n + 8, q ? y.w : y.z, s_scale[col + q]);
                }
        }
        __syncwarp();
        if (a.split > 1) cluster_sync();
        else __syncthreads();
    }
}

// ----------------------------------------------------------------------------------------------------------------- host
// (a launch's list of pairs is bounded: more pairs are more launches)
template <int CHUNK, int R, int WARPS, int PER_SM, typename F> cudaError_t mat_mat_i4_launch(MatI4Args a, F kernel, SmemAllowed& allowed, size_t base, size_t most, int sms, cudaStream_t st) {
    cudaError_t e = allowed(reinterpret_cast<const void*>(kernel), most);
    const int rows = a.rows, per = a.experts ? I4_PAIRS / a.div * a.div : rows;
    const int64_t blocks = (a.tiles + R - 1) / R;
    for (int first = 0; e == cudaSuccess && first < rows; first += per) {
        a.first = first;
        a.rows = std::min(per, rows - first);
        const int64_t units = (a.experts ? std::min<int64_t>(a.rows, a.n_experts + a.rows / CHUNK) : (a.rows + CHUNK - 1) / CHUNK) * blocks;
        a.split = 1;
        // clusters of two, four or eight while there are SMs for all at once (clusters of three leave too many of a GPC's SMs over: 48 of them took 24 us where 48 of two take 16) and a step for each team
        if (R > 1)
            while (a.split < 8 && units * a.split * 2 <= sms && a.steps >= 16 * a.split) a.split *= 2;
        e = launch(kernel, dim3((unsigned)(std::min<int64_t>(units, PER_SM * sms / a.split) * a.split)), WARPS * 32, base + (a.experts ? i4_list_bytes(a.n_experts, a.rows) : 0), a.split, st, a);
    }
    return e;
}
template <typename S, int GROUP, int NT> cudaError_t mat_mat_i4_few(const MatI4Args& a, int sms, cudaStream_t st) {
    static SmemAllowed allowed;
    constexpr size_t base = i4_few_warps<NT>() * (I4_RING * i4_slot(sizeof(S), GROUP, 4) + 2 * NT * 512);
    return mat_mat_i4_launch<8 * NT, 1, i4_few_warps<NT>(), 2>(a, mat_mat_i4_few_kernel<S, GROUP, NT>, allowed, base, base + i4_list_bytes(1024, I4_PAIRS), sms, st);
}
template <typename S, int GROUP> cudaError_t mat_mat_i4_many(MatI4Args a, int sms, cudaStream_t st) {
    static SmemAllowed allowed;
    const I4ManyPlan p = i4_many_plan(sizeof(S), GROUP, a.rows, a.n_experts);
    a.most = p.most;
    a.ring = p.ring;
    return mat_mat_i4_launch<I4_MANY_ROWS, I4_TEAM_TILES, I4_TEAMS * I4_TEAM_WARPS, 1>(a, mat_mat_i4_many_kernel<S, GROUP>, allowed, p.smem, I4_MANY_MOST, sms, st);
}
template <typename S, int GROUP> cudaError_t mat_mat_i4(const MatI4Args& a, cudaStream_t st) {
    int sms = 0;
    const cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    // rows of a that meet the same weights: all of them, or with experts no more than there are tokens, and seldom more than two standard deviations above the average
    int64_t rows = a.rows;
    if (a.experts) {
        const double each = (double)a.rows / a.n_experts;
        rows = std::min<int64_t>(a.tokens, (int64_t)std::ceil(each + 2 * std::sqrt(each)));
    }
    // five to eight rows of one matrix: eight columns each, which the kernel of sixteen rows has registers to make faster (8 rows of 6144 x 4096: 8.7 us for 9.4, of 4096 x 14336 12.2 for 13.2); experts' units mostly have fewer,
    // where more warps count (sixteen tokens through two of eight experts, 4096 x 14336: 50 us for 57)
    return rows <= (a.experts ? 8 : 4) ? mat_mat_i4_few<S, GROUP, 1>(a, sms, st) : rows <= 16 ? mat_mat_i4_few<S, GROUP, 2>(a, sms, st) : mat_mat_i4_many<S, GROUP>(a, sms, st);
}

}  // namespace dev
