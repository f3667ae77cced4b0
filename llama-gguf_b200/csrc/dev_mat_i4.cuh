// dev_mat_i4.cuh — product of rows in 8 bits with 4-bit weights that have a scale per group of channels, of one matrix or of each token's experts (b200_dev_mat_mat_i4).
//
// out[p][n] = a_scales[r] * sum_g ws[e][n][g] * (sum over the channels k of group g of a[r][k] * w[e][n][k]) + bias[e][n], r the row of a and e the expert of output row p.
// The inner sums are integers and exact; the outer one is f32, in an order that only the sizes decide.
//
// A tile of weights is 16 rows x 64 channels in 512 bytes, placed so that the 16 bytes of a lane are the operands of two mma.m16n8k32 (s8, s32 sums): a word has four channels in the low
// halves of its bytes and the next four in the high halves; (word << 4) & 0xf0f0f0f0 and word & 0xf0f0f0f0 are those values times sixteen as signed bytes, three instructions for eight weights.  Eight rows of a are
// the columns.  Sums begin at the bits of 1.5 * 2^23, so that read as f32 they are that plus the sum (|16 sum| <= 2^21).
//
// Work.  A unit is 16 R rows of weights and up to 8 NT rows of a; a block's eight warps share its channels and add their sums up in shared memory.  Blocks stride over the units.  With experts every
// block lists the pairs (token, expert) by expert first, all in the same order; a chunk of up to 8 NT pairs of an expert is one unit per 16 R rows.
#pragma once
#include <algorithm>

#include "dev_common.cuh"

namespace dev {

enum { I4_WARPS = 8, I4_TILE = 512, I4_PAIRS = 4096 };      // warps of a block, bytes of a tile, pairs of a launch

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
    int rows, k, n, div, n_experts, steps, groups, tiles;      // rows of out; row p of out is of row p / div of a
    uint32_t out_type;
    int first;      // the first row of out that this launch makes; `rows` counts from there
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int kI4Zero = 0x4B400000;      // the bits of 1.5 * 2^23
__device__ __forceinline__ float i4_sum(int bits) { return __int_as_float(bits) - 12582912.0f; }

// the scales of rows g and g + 8 of a tile for one group
template <typename S> __device__ __forceinline__ float2 i4_scales(const S* p) {
    struct __align__(2 * sizeof(S)) W { S lo, hi; };
    const W w = *reinterpret_cast<const W*>(p);
    return make_float2(to_f(w.lo), to_f(w.hi));
}

// Pairs by expert, in shared memory: first[e] the place of expert e's first pair in `list`, chunk[e] its first chunk; e = n_experts: the pairs without an expert (their rows are zeros).
struct I4List {
    int *first, *chunk, *list;
};
__device__ __forceinline__ int i4_expert(const MatI4Args& a, int p) {
    const int e = a.experts[a.first + p];
    return e >= 0 && e < a.n_experts ? e : a.n_experts;
}
__device__ __forceinline__ void i4_lists(const MatI4Args& a, const I4List& l, int per_chunk) {
    const int E = a.n_experts + 1, tid = threadIdx.x, lane = tid & 31;
    for (int e = tid; e <= E; e += blockDim.x) l.first[e] = 0;
    __syncthreads();
    for (int p = tid; p < a.rows; p += blockDim.x) {
        const int e = i4_expert(a, p);
        if (e == a.n_experts && a.status && blockIdx.x == 0 && a.experts[a.first + p] != -1) atomicOr(a.status, (int)B200_STATUS_BAD_EXPERT);
        atomicAdd(&l.first[e], 1);
    }
    __syncthreads();
    if (tid < 32) {
        int pairs = 0, chunks = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int n = e0 + lane < E ? l.first[e0 + lane] : 0, c = (n + per_chunk - 1) / per_chunk;
            int sn = n, sc = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int un = __shfl_up_sync(0xffffffffu, sn, o), uc = __shfl_up_sync(0xffffffffu, sc, o);
                if (lane >= o) sn += un, sc += uc;
            }
            if (e0 + lane < E) {
                l.first[e0 + lane] = pairs + sn - n;
                l.chunk[e0 + lane] = chunks + sc - c;
            }
            pairs += __shfl_sync(0xffffffffu, sn, 31);
            chunks += __shfl_sync(0xffffffffu, sc, 31);
        }
        if (lane == 0) {
            l.first[E] = pairs;
            l.chunk[E] = chunks;
        }
        __syncwarp();
        // (in order of the pairs, so that all blocks have the same list: first[e] is counted up, and afterwards is where e's pairs end)
        for (int p0 = 0; p0 < a.rows; p0 += 32) {
            const int p = p0 + lane, e = p < a.rows ? i4_expert(a, p) : -1;
            const uint32_t same = __match_any_sync(0xffffffffu, e), ahead = __popc(same & ((1u << lane) - 1));
            const int at = e >= 0 ? l.first[e] : 0;
            __syncwarp();
            if (e >= 0) {
                l.list[at + ahead] = p;
                if (ahead == 0) l.first[e] = at + __popc(same);
            }
            __syncwarp();
        }
    }
    __syncthreads();
}

template <typename S, int GROUP, int NT, int R> __global__ void __launch_bounds__(I4_WARPS * 32) mat_mat_i4_kernel(const MatI4Args a) {
    before();
    extern __shared__ __align__(16) int i4_smem[];
    float4* red = reinterpret_cast<float4*>(i4_smem);      // [warps][R * NT][32]
    __shared__ int s_row[8 * NT];                           // the unit's rows of out (-1: none)
    const I4List l{i4_smem + I4_WARPS * R * NT * 128, i4_smem + I4_WARPS * R * NT * 128 + a.n_experts + 2, i4_smem + I4_WARPS * R * NT * 128 + 2 * (a.n_experts + 2)};
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int blocks = (a.tiles + R - 1) / R;
    int chunks = (a.rows + 8 * NT - 1) / (8 * NT);
    if (a.experts) {
        i4_lists(a, l, 8 * NT);
        chunks = l.chunk[a.n_experts + 1];
    }
    // this warp's steps: whole groups
    constexpr int PER = GROUP > 64 ? GROUP / 64 : 1;
    const int whole = (a.steps + PER - 1) / PER, s0 = whole * warp / I4_WARPS * PER, s1 = min(a.steps, whole * (warp + 1) / I4_WARPS * PER);
    for (int64_t u = blockIdx.x; u < (int64_t)chunks * blocks; u += gridDim.x) {
        const int c = (int)(u / blocks), tile0 = (int)(u - (int64_t)c * blocks) * R;
        int e = 0, lo = c * 8 * NT, hi = a.rows;
        if (a.experts) {
            int top = a.n_experts;      // the last expert whose first chunk is not behind c and that has one
            while (e < top) {
                const int mid = (e + top + 1) / 2;
                if (l.chunk[mid] <= c) e = mid;
                else top = mid - 1;
            }
            hi = l.first[e];
            lo = (e ? l.first[e - 1] : 0) + (c - l.chunk[e]) * 8 * NT;
        }
        const int many = min(8 * NT, hi - lo);
        if (tid < 8 * NT) s_row[tid] = tid < many ? (a.experts ? l.list[lo + tid] : lo + tid) : -1;
        __syncthreads();
        float acc[R][NT][4];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[r][j][0] = acc[r][j][1] = acc[r][j][2] = acc[r][j][3] = 0;
        if (e < max(1, a.n_experts)) {
            const int8_t* rows[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int p = s_row[8 * j + g];
                rows[j] = p >= 0 ? a.a + (int64_t)((a.first + p) / a.div) * a.lda + 8 * t : nullptr;
            }
            const uint8_t* w = a.w + ((int64_t)e * a.tiles + tile0) * a.steps * I4_TILE + lane * 16;
            const S* ws = reinterpret_cast<const S*>(a.ws) + ((int64_t)e * a.tiles + tile0) * a.groups * 16 + g * 2;
            int sum[R][NT][4];
#pragma unroll 2
            for (int s = s0; s < s1; s++) {
                uint4 v[R];
#pragma unroll
                for (int r = 0; r < R; r++) v[r] = tile0 + r < a.tiles ? *reinterpret_cast<const uint4*>(w + ((int64_t)r * a.steps + s) * I4_TILE) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int k0 = s * 64 + h * 32;
                    uint2 b[NT];
#pragma unroll
                    for (int j = 0; j < NT; j++) b[j] = rows[j] && k0 < a.k ? *reinterpret_cast<const uint2*>(rows[j] + k0) : make_uint2(0, 0);
                    const bool begins = GROUP == 32 || (GROUP == 64 && h == 0) || (GROUP == 128 && h == 0 && s % 2 == 0);
                    const bool ends = GROUP == 32 || (GROUP == 64 && h == 1) || (GROUP == 128 && h == 1 && s % 2 == 1);
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        const uint32_t x = h ? v[r].z : v[r].x, y = h ? v[r].w : v[r].y;
                        const uint32_t a0 = (x << 4) & 0xf0f0f0f0u, a1 = (y << 4) & 0xf0f0f0f0u, a2 = x & 0xf0f0f0f0u, a3 = y & 0xf0f0f0f0u;
                        float2 d = make_float2(0, 0);
                        if (ends && tile0 + r < a.tiles && k0 / GROUP < a.groups) d = i4_scales(ws + ((int64_t)r * a.groups + k0 / GROUP) * 16);
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            if (begins) sum[r][j][0] = sum[r][j][1] = sum[r][j][2] = sum[r][j][3] = kI4Zero;
                            mma_s8(sum[r][j], a0, a1, a2, a3, b[j].x, b[j].y);
                            if (ends) {
                                acc[r][j][0] += d.x * i4_sum(sum[r][j][0]);
                                acc[r][j][1] += d.x * i4_sum(sum[r][j][1]);
                                acc[r][j][2] += d.y * i4_sum(sum[r][j][2]);
                                acc[r][j][3] += d.y * i4_sum(sum[r][j][3]);
                            }
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < NT; j++) red[(warp * R * NT + r * NT + j) * 32 + lane] = make_float4(acc[r][j][0], acc[r][j][1], acc[r][j][2], acc[r][j][3]);
        __syncthreads();
        // one output per thread and step: row i of the unit's 16 R, column (row of a) q
        for (int o = tid; o < 16 * R * many; o += I4_WARPS * 32) {
            const int i = o % (16 * R), q = o / (16 * R), n = tile0 * 16 + i;
            if (n >= a.n) continue;
            const int r = i / 16, j = q / 8, at = (r * NT + j) * 128 + ((i % 8) * 4 + q % 8 / 2) * 4 + (i % 16) / 8 * 2 + q % 2;
            const float* f = reinterpret_cast<const float*>(red) + at;
            float y = 0;
#pragma unroll
            for (int x = 0; x < I4_WARPS; x++) y += f[x * R * NT * 128];
            const int p = s_row[q];
            if (e < max(1, a.n_experts)) {
                y = y * 0.0625f * a.a_scales[(a.first + p) / a.div];
                if (a.bias) y += a.bias[(int64_t)e * a.n + n];
            }
            const int64_t to = (int64_t)(a.first + p) * a.ldo + n;
            if (a.out_type == B200_TYPE_F32) reinterpret_cast<float*>(a.out)[to] = y;
            else if (a.out_type == B200_TYPE_F16) reinterpret_cast<__half*>(a.out)[to] = __float2half_rn(y);
            else reinterpret_cast<__nv_bfloat16*>(a.out)[to] = __float2bfloat16_rn(y);
        }
        __syncthreads();
    }
}

template <typename S, int GROUP, int NT, int R> cudaError_t mat_mat_i4_as(MatI4Args a, int sms, cudaStream_t st) {
    static SmemAllowed allowed;
    const size_t smem = I4_WARPS * R * NT * 512 + (a.experts ? (2 * (a.n_experts + 2) + std::min<int>(a.rows, I4_PAIRS)) * 4 : 0);
    cudaError_t e = smem > 48 * 1024 ? allowed(reinterpret_cast<const void*>(mat_mat_i4_kernel<S, GROUP, NT, R>), 128 * 1024) : cudaSuccess;
    const int rows = a.rows, per = a.experts ? I4_PAIRS / a.div * a.div : rows;      // (a launch's list of pairs is bounded)
    for (int first = 0; e == cudaSuccess && first < rows; first += per) {
        a.first = first;
        a.rows = std::min(per, rows - first);
        const int64_t chunks = a.experts ? std::min<int64_t>(a.rows, a.n_experts + 1 + a.rows / (8 * NT)) : (a.rows + 8 * NT - 1) / (8 * NT);
        e = launch(mat_mat_i4_kernel<S, GROUP, NT, R>, dim3((unsigned)std::min<int64_t>(chunks * ((a.tiles + R - 1) / R), 4 * sms)), I4_WARPS * 32, smem, 1, st, a);
    }
    return e;
}
template <typename S, int GROUP> cudaError_t mat_mat_i4(const MatI4Args& a, cudaStream_t st) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    const int many = a.rows;
    if (many <= 8) return mat_mat_i4_as<S, GROUP, 1, 1>(a, sms, st);
    return mat_mat_i4_as<S, GROUP, 4, 1>(a, sms, st);
}

}  // namespace dev
