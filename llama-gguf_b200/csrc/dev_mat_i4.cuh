// dev_mat_i4.cuh — product of rows in 8 bits with 4-bit weights that have a scale per group of channels, of one matrix or of each token's experts (b200_dev_mat_mat_i4).
//
// out[p][n] = a_scales[r] * sum_g ws[e][n][g] * (sum over the channels k of group g of a[r][k] * w[e][n][k]) + bias[e][n], r the row of a and e the expert of output row p.
// The inner sums are integers and exact; the outer one is f32, in an order that only the sizes decide.
//
// A tile of weights is 16 rows x 64 channels in 512 bytes, placed so that the 16 bytes of a lane are the operands of two mma.m16n8k32 (s8, s32 sums): a word has four channels in the low
// halves of its bytes and the next four in the high halves; (word << 4) & 0xf0f0f0f0 and word & 0xf0f0f0f0 are those values times sixteen as signed bytes, three instructions for eight weights.  Eight rows of a are
// the columns.  Sums begin at the bits of 1.5 * 2^23, so that read as f32 they are that plus the sum (|16 sum| <= 2^21).
//
// Work.  A unit is R tiles of weight rows and up to 8 NT rows of a; its channels go 128 at a time (a step: two tiles, a whole number of groups).  Each lane copies the bytes that it will read itself into a
// ring of its warp (cp.async), some steps ahead, so that no warp waits for another.  With experts every block lists the pairs (token, expert) by expert first, all in the same order; a chunk of up to
// 8 NT pairs of an expert is a unit for each R tiles.
//   few rows (NT 1 or 2, R 1): the weights' bytes.  A block per SM has consecutive units; its warps share their steps evenly, whichever unit they are of, and leave the sums of a unit that two or more warps have a part of in
//   shared memory for the end.  Rows of a come from L1.
//   more rows (NT 4 or 8, R 4): rows of a cost as much as weights.  A block's warps share a unit's steps, with clusters the blocks of one too; the rows' bytes go through the ring with the weights', and
//   serve four tiles.
#pragma once
#include <algorithm>
#include <cmath>

#include "dev_common.cuh"

namespace dev {

enum { I4_TILE = 512, I4_PAIRS = 2048, I4_RING = 3 };      // bytes of a tile, pairs of a launch, steps of a warp's ring (few rows)

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
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int kI4Zero = 0x4B400000;      // the bits of 1.5 * 2^23
// ... with sums that begin there
__device__ __forceinline__ void mma_s8_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kI4Zero));
}
__device__ __forceinline__ float i4_sum(int bits) { return __int_as_float(bits) - 12582912.0f; }
// 16 or 8 bytes to shared memory, zeros where `there` is not set (the address is a valid one all the same)
template <int N> __device__ __forceinline__ void copy_where(uint32_t to, const void* from, bool there) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(N), "r"(there ? N : 0) : "memory");
}

// Pairs by expert, in shared memory: expert e's pairs are list[end[e - 1]] .. list[end[e] - 1] (those without an expert come last), its first chunk is chunk[e].
struct I4List {
    int *end, *chunk;
    uint16_t *list, *of;
};
__host__ __device__ constexpr size_t i4_list_bytes(int experts, int pairs) { return (size_t)(2 * (experts + 2)) * 4 + (size_t)pairs * 4; }
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
__device__ __forceinline__ void i4_put(const MatI4Args& a, int e, int p, int n, float sum) {
    float y = sum * 0.0625f * a.a_scales[(a.first + p) / a.div];
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
// What a ring holds of a step (C tiles' channels of R tiles of rows): the weights of each, then the groups' scales of each.
template <typename S, int GROUP, int R, int C> __host__ __device__ constexpr int i4_slot() { return R * (C * I4_TILE + 16 * (int)sizeof(S) * (64 * C / GROUP)); }
// ... copied: step s of R tiles from `tile` on, whose weights and scales are at w and d
template <typename S, int GROUP, int R, int C> __device__ __forceinline__ void i4_copy(const MatI4Args& a, uint32_t to, const uint8_t* w, const uint8_t* d, int tile, int s, int lane) {
    constexpr int GS = 64 * C / GROUP, SB = 16 * (int)sizeof(S), WORDS = GS * SB / 8;
    const uint8_t *p = w + (int64_t)s * (C * I4_TILE) + lane * 16, *q = d + (int64_t)s * (GS * SB) + lane * 8;
    const int room = a.steps - s * C, scales = (a.groups - s * GS) * (SB / 8);      // tiles of the step, and 8-byte words of its scales
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool in = R == 1 || tile + r < a.tiles;
#pragma unroll
        for (int c = 0; c < C; c++) copy_where<16>(to + (r * C + c) * I4_TILE + lane * 16, in && c < room ? p + c * I4_TILE : a.w, in && c < room);
#pragma unroll
        for (int c = 0; c < WORDS; c += 32)
            if (c + 32 <= WORDS || lane < WORDS - c) {
                const bool there = in && c + lane < scales;
                copy_where<8>(to + R * C * I4_TILE + r * GS * SB + c * 8 + lane * 8, there ? q + c * 8 : a.w, there);
            }
        p += (int64_t)a.steps * I4_TILE;
        q += (int64_t)a.groups * SB;
    }
}

// ------------------------------------------------------------------------------------------------------------- few rows
// TC rows of a are TC of the eight columns; with fewer than eight the other columns take the same rows' other groups: column n has row n % TC and group n / TC of the (up to) 8 / TC that one set of sums
// has, so that what a group's sum costs afterwards (a subtraction and a multiplication in each lane) is paid once for all of them.  (One row in all columns took 240 instructions for 128 channels.)
// NT > 1: TC = 8, and that many times eight columns.
template <int NT> __host__ __device__ constexpr int i4_few_warps() { return NT == 1 ? 24 : 16; }
template <typename S, int GROUP, int TC, int NT> __global__ void __launch_bounds__(i4_few_warps<NT>() * 32, 1) mat_mat_i4_few_kernel(const MatI4Args a) {
    before();
    constexpr int C = 4, SLOT = i4_slot<S, GROUP, 1, C>(), SB = 16 * (int)sizeof(S), CHUNK = TC * NT, WARPS = i4_few_warps<NT>();
    constexpr int GC = GROUP / 32, GS = 256 / GROUP, SETS = GS * TC > 8 ? GS * TC / 8 : 1, PER = GS / SETS;      // chunks (of 32 channels) of a group, groups of a step, sets of sums, groups of a set
    extern __shared__ __align__(16) uint8_t i4_smem[];
    float4* parts = reinterpret_cast<float4*>(i4_smem + WARPS * I4_RING * SLOT);      // [warps][its first unit, its last][NT][32]
    const I4List l = i4_list(parts + WARPS * 2 * NT * 32, a);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, whole = (a.steps + C - 1) / C;
    const uint8_t* slots = i4_smem + warp * I4_RING * SLOT;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(slots);
    int chunks = (a.rows + CHUNK - 1) / CHUNK;
    if (a.experts) {
        i4_lists(a, l, CHUNK);
        chunks = l.chunk[a.n_experts];
        i4_zeros(a, l);
    }
    // this block's units, their steps one after the other, and this warp's of those
    const int64_t units = (int64_t)chunks * a.tiles, u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
    const int many = (int)(u1 - u0), steps = many * whole;
    auto begin = [&](int w) { return (int)((int64_t)steps * w / WARPS); };
    // sums over a row's columns, and the results of a unit
    auto finish = [&](float4 (&y)[NT], const I4Chunk& x, int tile) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            if constexpr (TC == 1) y[j].x += y[j].y, y[j].z += y[j].w;
#pragma unroll
            for (int o = TC == 4 ? 2 : 1; o < 4 && TC < 8; o <<= 1) {
                y[j].x += __shfl_xor_sync(0xffffffffu, y[j].x, o);
                y[j].z += __shfl_xor_sync(0xffffffffu, y[j].z, o);
                if constexpr (TC > 1) {
                    y[j].y += __shfl_xor_sync(0xffffffffu, y[j].y, o);
                    y[j].w += __shfl_xor_sync(0xffffffffu, y[j].w, o);
                }
            }
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const int col = 8 * j + 2 * t + q, n = tile * 16 + g;
                if (col < (TC < 8 ? min(TC, x.many) : x.many)) {
                    const int p = i4_pair(a, l, x.lo + col);
                    if (n < a.n) i4_put(a, x.e, p, n, q ? y[j].y : y[j].x);
                    if (n + 8 < a.n) i4_put(a, x.e, p, n + 8, q ? y[j].w : y[j].z);
                }
            }
        }
    };
    const int f0 = begin(warp), f1 = begin(warp + 1);
    if (f0 < f1) {
        const int v0 = f0 / whole;
        int c = (int)((u0 + v0) / a.tiles), tile = (int)(u0 + v0 - (int64_t)c * a.tiles), s = f0 - v0 * whole;
        I4Chunk x = i4_chunk<CHUNK>(a, l, c);
        // copies, I4_RING - 1 steps ahead of the products
        int cc = c, ct = tile, ce = x.e, cs = s, left = f1 - f0, into = 0;
        const uint8_t *cw = nullptr, *cd = nullptr;
        auto place = [&]() {
            const int64_t at = (int64_t)ce * a.tiles + ct;
            cw = a.w + at * a.steps * I4_TILE;
            cd = reinterpret_cast<const uint8_t*>(a.ws) + at * a.groups * SB;
        };
        place();
        auto copy = [&]() {
            if (left > 0) {
                i4_copy<S, GROUP, 1, C>(a, ring + into * SLOT, cw, cd, ct, cs, lane);
                into = into + 1 == I4_RING ? 0 : into + 1;
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
        const int group = g / TC;      // this column's, of a set's
        int slot = 0;
        for (int f = f0; f < f1;) {
            const int sa = s, sb = min(whole, s + f1 - f);
            float acc[NT][4];
            const int8_t* rows[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0;
                // (columns without a row take another's: nothing reads their sums)
                const int col = 8 * j + g % TC;
                rows[j] = a.a + (int64_t)((a.first + i4_pair(a, l, x.lo + (col < x.many ? col : 0))) / a.div) * a.lda + group * GROUP + 8 * t;
            }
            for (; s < sb; s++) {
                uint2 b[NT][SETS * GC];
                const int room = a.k - s * 256 - group * GROUP;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int z = 0; z < SETS; z++)
#pragma unroll
                        for (int h = 0; h < GC; h++)
                            b[j][z * GC + h] = z * PER * GROUP + h * 32 < room && (PER * TC == 8 || group < PER) && (j == 0 || 8 * j < x.many)
                                                   ? *reinterpret_cast<const uint2*>(rows[j] + s * 256 + z * PER * GROUP + h * 32) : make_uint2(0, 0);
                asm volatile("cp.async.wait_group %0;" ::"n"(I4_RING - 2) : "memory");
                __syncwarp();
                const uint8_t *in = slots + slot * SLOT, *scales = in + C * I4_TILE + g * 2 * sizeof(S);
                copy();
                slot = slot + 1 == I4_RING ? 0 : slot + 1;
#pragma unroll
                for (int z = 0; z < SETS; z++) {
                    int sum[NT][4];
#pragma unroll
                    for (int q = 0; q < PER; q++)
#pragma unroll
                        for (int h = 0; h < GC; h++) {
                            const int k = (z * PER + q) * GC + h;      // the chunk: half a tile
                            const uint2 v = *reinterpret_cast<const uint2*>(in + (k / 2) * I4_TILE + lane * 16 + (k % 2) * 8);
                            const uint32_t a0 = (v.x << 4) & 0xf0f0f0f0u, a1 = (v.y << 4) & 0xf0f0f0f0u, a2 = v.x & 0xf0f0f0f0u, a3 = v.y & 0xf0f0f0f0u;
#pragma unroll
                            for (int j = 0; j < NT; j++) {
                                if (j && 8 * j >= x.many) break;
                                const uint32_t b0 = PER == 1 || group == q ? b[j][z * GC + h].x : 0, b1 = PER == 1 || group == q ? b[j][z * GC + h].y : 0;
                                if (q == 0 && h == 0) mma_s8_first(sum[j], a0, a1, a2, a3, b0, b1);
                                else mma_s8(sum[j], a0, a1, a2, a3, b0, b1);
                            }
                        }
                    // columns 2t and 2t + 1: one group's, but for TC = 1
                    const int q0 = 2 * t / TC, q1 = (2 * t + 1) / TC;
                    float2 d0 = i4_scales<S>(scales + (z * PER + (PER > 1 ? min(q0, PER - 1) : 0)) * SB), d1 = d0;
                    if constexpr (TC == 1) d1 = i4_scales<S>(scales + (z * PER + (PER > 1 ? min(q1, PER - 1) : 0)) * SB);
                    if (PER * TC < 8) {      // (columns that no group has)
                        if (q0 >= PER) d0 = make_float2(0, 0);
                        if (q1 >= PER) d1 = make_float2(0, 0);
                    }
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        if (j && 8 * j >= x.many) break;
                        acc[j][0] = fmaf(d0.x, i4_sum(sum[j][0]), acc[j][0]);
                        acc[j][1] = fmaf(d1.x, i4_sum(sum[j][1]), acc[j][1]);
                        acc[j][2] = fmaf(d0.y, i4_sum(sum[j][2]), acc[j][2]);
                        acc[j][3] = fmaf(d1.y, i4_sum(sum[j][3]), acc[j][3]);
                    }
                }
            }
            float4 y[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) y[j] = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
            if (sa == 0 && sb == whole) {
                finish(y, x, tile);
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
        int w = (int)((int64_t)v * whole * WARPS / steps);      // the warp that has the unit's first step
        while (begin(w + 1) <= v * whole) w++;
        while (begin(w) > v * whole) w--;
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
        const int c = (int)((u0 + v) / a.tiles);
        finish(y, i4_chunk<CHUNK>(a, l, c), (int)(u0 + v - (int64_t)c * a.tiles));
    }
}

// ------------------------------------------------------------------------------------------------------------- more rows
// A block has four tiles of rows and its eight pairs of warps a part of the channels each: a pair's warps have two tiles each, and the same rows of a, which both copy a half of.
enum { I4_PAIRS_OF_WARPS = 8, I4_R = 2 };
template <typename S, int GROUP, int NT> __host__ __device__ constexpr int i4_many_slot() { return 2 * i4_slot<S, GROUP, I4_R, 2>() + NT * 8 * 128; }
template <typename S, int GROUP, int NT> __host__ __device__ constexpr int i4_many_ring() {      // steps of a pair's ring: as many as fit a block's 227 KiB with the longest lists, up to four
    const int fit = (int)(227 * 1024 - 1024 - i4_list_bytes(1024, I4_PAIRS)) / (I4_PAIRS_OF_WARPS * i4_many_slot<S, GROUP, NT>());
    return fit < 4 ? fit : 4;
}

template <typename S, int GROUP, int NT> __global__ void __launch_bounds__(I4_PAIRS_OF_WARPS * 64, 1) mat_mat_i4_many_kernel(const MatI4Args a) {
    before();
    constexpr int R = I4_R, P = I4_PAIRS_OF_WARPS, RING = i4_many_ring<S, GROUP, NT>(), WSLOT = i4_slot<S, GROUP, R, 2>(), SLOT = i4_many_slot<S, GROUP, NT>(), GS = 128 / GROUP, SB = 16 * (int)sizeof(S),
                  GC = GROUP / 32, J = NT < 4 ? NT : 4;
    static_assert(RING >= 2 && RING * SLOT >= 2 * R * NT * 512, "a pair's sums take its ring's place");
    extern __shared__ __align__(16) uint8_t i4_smem[];
    __shared__ int64_t s_row[8 * NT];      // where the unit's rows of a begin
    const I4List l = i4_list(i4_smem + P * RING * SLOT, a);
    const int tid = threadIdx.x, lane = tid & 31, pair = tid >> 6, half = (tid >> 5) & 1, g = lane >> 2, t = lane & 3;
    uint8_t* slots = i4_smem + pair * RING * SLOT;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(slots);
    const int blocks = (a.tiles + 2 * R - 1) / (2 * R), whole = (a.steps + 1) / 2;
    int chunks = (a.rows + 8 * NT - 1) / (8 * NT);
    if (a.experts) {
        i4_lists(a, l, 8 * NT);
        chunks = l.chunk[a.n_experts];
        i4_zeros(a, l);
    }
    const int rank = blockIdx.x % a.split, parts = P * a.split, part = rank * P + pair, s0 = (int)((int64_t)whole * part / parts), s1 = (int)((int64_t)whole * (part + 1) / parts);
    auto together = [&] { asm volatile("bar.sync %0, 64;" ::"r"(pair + 1) : "memory"); };
    for (int64_t u = blockIdx.x / a.split; u < (int64_t)chunks * blocks; u += gridDim.x / a.split) {
        const int c = (int)(u / blocks), tile = (int)(u - (int64_t)c * blocks) * 2 * R + half * R;
        const I4Chunk x = i4_chunk<8 * NT>(a, l, c);
        if (tid < 8 * NT) s_row[tid] = tid < x.many ? (int64_t)((a.first + i4_pair(a, l, x.lo + tid)) / a.div) * a.lda : 0;
        __syncthreads();
        const int64_t at = (int64_t)x.e * a.tiles + tile;
        const uint8_t *w = a.w + at * a.steps * I4_TILE, *d = reinterpret_cast<const uint8_t*>(a.ws) + at * a.groups * SB;
        // rows of 128 bytes; 16 bytes u of row i lie at u ^ (2 (i % 4)), so that the eight rows of a column block are read without bank conflicts
        auto copy = [&](int s, int into) {
            if (s < s1) {
                const int unit = lane & 7, ch = s * 128 + unit * 16;
                const uint32_t to = ring + into * SLOT + 2 * WSLOT;
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    const int row = i * 8 + half * 4 + (lane >> 3);
                    if (i * 8 < x.many) {
                        const bool there = row < x.many && ch < a.k;
                        copy_where<16>(to + row * 128 + ((unit ^ ((row & 3) << 1)) << 4), there ? a.a + s_row[row] + ch : a.a, there);
                    }
                }
                i4_copy<S, GROUP, R, 2>(a, ring + into * SLOT + half * WSLOT, w, d, tile, s, lane);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < RING - 1; i++) copy(s0 + i, i);
        float acc[R][NT][4];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[r][j][0] = acc[r][j][1] = acc[r][j][2] = acc[r][j][3] = 0;
        int slot = 0, into = RING - 1;
        for (int s = s0; s < s1; s++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory");
            together();      // (both warps' copies of this step are there, and both are done with the step before)
            copy(s + RING - 1, into);
            const uint8_t *in = slots + slot * SLOT, *mine = in + half * WSLOT;
            into = into + 1 == RING ? 0 : into + 1;
            slot = slot + 1 == RING ? 0 : slot + 1;
#pragma unroll
            for (int j0 = 0; j0 < NT; j0 += J) {
                if (j0 * 8 >= x.many) break;
#pragma unroll
                for (int q = 0; q < GS; q++) {
                    uint2 b[J][GC];
#pragma unroll
                    for (int j = 0; j < J; j++)
#pragma unroll
                        for (int h = 0; h < GC; h++)
                            b[j][h] = *reinterpret_cast<const uint2*>(in + 2 * WSLOT + ((j0 + j) * 8 + g) * 128 + ((((q * GC + h) * 2 + (t >> 1)) ^ ((g & 3) << 1)) << 4) + (t & 1) * 8);
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        uint2 v[GC];
#pragma unroll
                        for (int h = 0; h < GC; h++) v[h] = *reinterpret_cast<const uint2*>(mine + (r * 2 + (q * GC + h) / 2) * I4_TILE + lane * 16 + (q * GC + h) % 2 * 8);
                        const float2 e = i4_scales<S>(mine + R * 2 * I4_TILE + (r * GS + q) * SB + g * 2 * sizeof(S));
#pragma unroll
                        for (int j = 0; j < J; j++) {
                            if ((j0 + j) * 8 >= x.many) break;
                            int sum[4];
#pragma unroll
                            for (int h = 0; h < GC; h++) {
                                const uint32_t a0 = (v[h].x << 4) & 0xf0f0f0f0u, a1 = (v[h].y << 4) & 0xf0f0f0f0u, a2 = v[h].x & 0xf0f0f0f0u, a3 = v[h].y & 0xf0f0f0f0u;
                                if (h == 0) mma_s8_first(sum, a0, a1, a2, a3, b[j][h].x, b[j][h].y);
                                else mma_s8(sum, a0, a1, a2, a3, b[j][h].x, b[j][h].y);
                            }
                            acc[r][j0 + j][0] = fmaf(e.x, i4_sum(sum[0]), acc[r][j0 + j][0]);
                            acc[r][j0 + j][1] = fmaf(e.x, i4_sum(sum[1]), acc[r][j0 + j][1]);
                            acc[r][j0 + j][2] = fmaf(e.y, i4_sum(sum[2]), acc[r][j0 + j][2]);
                            acc[r][j0 + j][3] = fmaf(e.y, i4_sum(sum[3]), acc[r][j0 + j][3]);
                        }
                    }
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        together();
        // sums to this pair's part of the ring
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NT; j++)
                reinterpret_cast<float4*>(slots)[((half * R + r) * NT + j) * 32 + lane] = make_float4(acc[r][j][0], acc[r][j][1], acc[r][j][2], acc[r][j][3]);
        __syncwarp();
        if (a.split > 1) cluster_sync();
        else __syncthreads();
        for (int o = tid + rank * P * 64; o < 32 * R * x.many; o += P * 64 * a.split) {      // row i of the unit's, column q
            const int i = o % (32 * R), q = o / (32 * R), n = (tile - half * R) * 16 + i;
            if (n >= a.n) continue;
            const uint8_t* from = i4_smem + (((i / 16 * NT + q / 8) * 32 + (i % 8) * 4 + q % 8 / 2) * 4 + (i % 16) / 8 * 2 + q % 2) * 4;
            float y = 0;
            for (int b = 0; b < a.split; b++)
#pragma unroll
                for (int w = 0; w < P; w++) {
                    const uint8_t* f = from + w * RING * SLOT;
                    y += a.split > 1 ? peer_f32((uint32_t)__cvta_generic_to_shared(f), b) : *reinterpret_cast<const float*>(f);
                }
            i4_put(a, x.e, i4_pair(a, l, x.lo + q), n, y);
        }
        __syncwarp();
        if (a.split > 1) cluster_sync();
        else __syncthreads();
    }
}

// ----------------------------------------------------------------------------------------------------------------- host
// (a launch's list of pairs is bounded: more pairs are more launches)
template <int CHUNK, int R, int WARPS, typename F> cudaError_t mat_mat_i4_launch(MatI4Args a, F kernel, SmemAllowed& allowed, size_t base, int sms, cudaStream_t st) {
    cudaError_t e = allowed(reinterpret_cast<const void*>(kernel), base + i4_list_bytes(1024, I4_PAIRS));
    const int rows = a.rows, per = a.experts ? I4_PAIRS / a.div * a.div : rows;
    const int64_t blocks = (a.tiles + R - 1) / R;
    for (int first = 0; e == cudaSuccess && first < rows; first += per) {
        a.first = first;
        a.rows = std::min(per, rows - first);
        const int64_t units = (a.experts ? std::min<int64_t>(a.rows, a.n_experts + a.rows / CHUNK) : (a.rows + CHUNK - 1) / CHUNK) * blocks;
        a.split = 1;
        if (R > 1)
            while (a.split < 8 && units * a.split * 2 <= sms && a.steps >= 32 * a.split) a.split *= 2;
        e = launch(kernel, dim3((unsigned)(std::min<int64_t>(units, sms / a.split) * a.split)), WARPS * 32, base + (a.experts ? i4_list_bytes(a.n_experts, a.rows) : 0), a.split, st, a);
    }
    return e;
}
template <typename S, int GROUP, int TC, int NT> cudaError_t mat_mat_i4_few(const MatI4Args& a, int sms, cudaStream_t st) {
    static SmemAllowed allowed;
    return mat_mat_i4_launch<TC * NT, 1, i4_few_warps<NT>()>(a, mat_mat_i4_few_kernel<S, GROUP, TC, NT>, allowed, i4_few_warps<NT>() * (I4_RING * i4_slot<S, GROUP, 1, 4>() + 2 * NT * 512), sms, st);
}
template <typename S, int GROUP, int NT> cudaError_t mat_mat_i4_many(const MatI4Args& a, int sms, cudaStream_t st) {
    static SmemAllowed allowed;
    return mat_mat_i4_launch<NT * 8, 2 * I4_R, 2 * I4_PAIRS_OF_WARPS>(a, mat_mat_i4_many_kernel<S, GROUP, NT>, allowed, I4_PAIRS_OF_WARPS * i4_many_ring<S, GROUP, NT>() * i4_many_slot<S, GROUP, NT>(), sms, st);
}
template <typename S, int GROUP> cudaError_t mat_mat_i4(const MatI4Args& a, cudaStream_t st) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    // rows of a that meet the same weights: all of them, or with experts no more than there are tokens, and seldom more than two standard deviations above the average
    int64_t rows = a.rows;
    if (a.experts) {
        const double each = (double)a.rows / a.n_experts;
        rows = std::min<int64_t>(a.tokens, (int64_t)std::ceil(each + 2 * std::sqrt(each)));
    }
    return rows <= 1 ? mat_mat_i4_few<S, GROUP, 1, 1>(a, sms, st) : rows <= 2 ? mat_mat_i4_few<S, GROUP, 2, 1>(a, sms, st) : rows <= 4 ? mat_mat_i4_few<S, GROUP, 4, 1>(a, sms, st)
         : rows <= 8 ? mat_mat_i4_few<S, GROUP, 8, 1>(a, sms, st) : rows <= 16 ? mat_mat_i4_few<S, GROUP, 8, 2>(a, sms, st) : rows <= 32 ? mat_mat_i4_many<S, GROUP, 4>(a, sms, st)
         : mat_mat_i4_many<S, GROUP, 8>(a, sms, st);
}

}  // namespace dev
