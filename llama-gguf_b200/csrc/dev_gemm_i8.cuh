// dev_gemm_i8.cuh — products of 8-bit integers with scales per token and per output channel (b200_dev_mat_mat_i8) on tcgen05.mma kind::i8.
//
// out[t][n] = a_scale[t] * w_scale[n] * sum_k a[t][k] w[n][k] + bias[n].  The sums are exact in s32, so cutting K and the order of the parts change nothing.
// A tile is 128 weight rows (the M of the MMA: lanes of tensor memory) by TN tokens (its N: columns).  A step is 128 bytes of K = one row of a SWIZZLE_128B atom; one warp asks the TMA
// unit for the weight rows of a step, one for its token rows, an mbarrier ring runs between them and the warp that issues the MMAs (four of K = 32 a step).  What lies past
// k, n and t arrives as zeros, so ragged sizes need no code in the loop.
//   gemm_i8_wide_kernel    many tokens: a CTA per SM walks tiles, two accumulators in tensor memory, so that a tile's epilogue runs under the next one's products.  PAIR: two CTAs share a
//                          tile of 256 x 256 (cta_group::2), each with its own weight rows and half of the token rows: 32 KB a step per CTA instead of 48.
//   gemm_i8_split_kernel   few tiles: S CTAs of a cluster share a tile's steps and add their sums through distributed shared memory.  With one token the weights' bytes are all there is
//                          to do, and a ring of up to 192 KB per SM keeps enough of them on the way.
// Measured (tokens x n x k): 2048 x 14336 x 4096 101 us in a loop (2400 TOP/s; 88 us by itself), bound by the tensor pipe (79 % of cycles, 91 on the SMs with the most tiles) and a last wave; 4 x 14336 x 4096 13.3 us for 59 MB (4.4 TB/s).
#pragma once
#include "dev_umma.cuh"

namespace dev {

struct GemmI8Args {
    const float *as, *ws, *bias;
    void* out;
    int64_t ldo;
    int t, k, n, splits;
};
enum { GI_EPI_WARPS = 8, GI_LOAD_W = 8, GI_LOAD_A = 9, GI_MMA = 10, GI_THREADS = 352, GI_STEP = 128, GI_M = 128 };
constexpr int GI_RING = 196608;

template <typename T> __device__ __forceinline__ T i8_result(int acc, float a_scale, float w_scale, float bias) {
    return from_f<T>(__fadd_rn(__fmul_rn(__fmul_rn((float)acc, a_scale), w_scale), bias));      // (without a bias: + 0, which changes no value)
}
// D = s32 (2 at bit 4), A and B signed (1 at bits 7 and 10), K-major, N >> 3 at bit 17, M >> 4 at bit 24
__device__ __forceinline__ uint32_t i8_idesc(int M, int N) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
template <bool PAIR> __device__ __forceinline__ void i8_mma_step(uint32_t acc, uint32_t w, uint32_t a, uint32_t idesc, bool first) {
    const uint64_t dw = umma_desc(w), da = umma_desc(a);
#pragma unroll
    for (int kk = 0; kk < GI_STEP / 32; kk++) {      // 32 bytes along the swizzled row: start address + 2
        const uint32_t accum = (!first || kk > 0) ? 1u : 0u;
        if constexpr (PAIR)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(acc), "l"(dw + (uint64_t)(2 * kk)),
                         "l"(da + (uint64_t)(2 * kk)), "r"(idesc), "r"(accum)
                         : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(acc), "l"(dw + (uint64_t)(2 * kk)),
                         "l"(da + (uint64_t)(2 * kk)), "r"(idesc), "r"(accum)
                         : "memory");
    }
}
// barriers and tensor memory; bars: [stages] full (both loaders), [stages] empty, [n_acc] accumulator done, [n_acc] accumulator read
template <bool PAIR> __device__ __forceinline__ void i8_setup(uint32_t bar, int stages, int n_acc, uint32_t* s_tmem, uint32_t cols) {
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; i++) {
            bar_init(bar + 8u * i, 2);
            bar_init(bar + 8u * (stages + i), 1);
        }
        for (int i = 0; i < n_acc; i++) {
            bar_init(bar + 8u * (2 * stages + i), 1);
            bar_init(bar + 8u * (2 * stages + n_acc + i), PAIR ? 2 * GI_EPI_WARPS : GI_EPI_WARPS);
        }
        bar_init_done();
    }
    if ((threadIdx.x >> 5) == GI_MMA) tmem_alloc<PAIR>(s_tmem, cols);
    umma_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync();      // (the other CTA's barriers are there)
    umma_after_sync();
}
// a loader that gave up at stage s: the copies that it has asked for land before it goes on (bounded)
__device__ __forceinline__ void i8_drain(uint32_t full, int stages, uint32_t s, uint32_t ph) {
    for (uint32_t i = 0; i < (uint32_t)stages; i++) {
        bool wait = true;
        bar_wait(full + 8u * i, i < s ? ph ^ 1u : ph, wait, 0);
    }
}

template <typename T, int TN, bool PAIR>
__global__ void __launch_bounds__(GI_THREADS, 1) gemm_i8_wide_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap wmap, const GemmI8Args g) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int W_BYTES = GI_M * GI_STEP, A_BYTES = (PAIR ? TN / 2 : TN) * GI_STEP, STAGE = W_BYTES + A_BYTES, NS = GI_RING / STAGE;
    __shared__ __align__(8) unsigned long long s_bar[2 * NS + 4];
    __shared__ uint32_t s_tmem;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = (sm_u32(smem) + 1023u) & ~1023u;      // (the swizzle is on absolute address bits)
    const uint32_t full = sm_u32(s_bar), empty = full + 8u * NS, acc_full = full + 16u * NS, acc_empty = acc_full + 16u;
    i8_setup<PAIR>(full, NS, 2, &s_tmem, 2 * TN);
    before();
    const uint32_t tmem = s_tmem, rank = PAIR ? cluster_rank() : 0u;
    const int steps = (g.k + GI_STEP - 1) / GI_STEP, mt = (g.n + GI_M - 1) / GI_M, per = PAIR ? (mt + 1) / 2 : mt, nt = (g.t + TN - 1) / TN, tiles = per * nt;
    const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x, stride = PAIR ? gridDim.x >> 1 : gridDim.x;
    bool alive = true;
    if (warp == GI_LOAD_W || warp == GI_LOAD_A) {
        const bool is_w = warp == GI_LOAD_W;
        uint32_t s = 0, ph = 1;
        for (int item = first; alive && item < tiles; item += stride) {
            const int m = PAIR ? 2 * (item / nt) + (int)rank : item / nt, row = is_w ? m * GI_M : (item % nt) * TN + (PAIR ? (int)rank * (TN / 2) : 0);
            for (int k = 0; k < steps; k++) {
                bar_wait(empty + 8u * s, ph, alive, 1);
                alive = __all_sync(0xffffffffu, alive);
                if (!alive) break;
                if (elect()) {
                    if (rank == 0) bar_expect(full + 8u * s, (PAIR ? 2 : 1) * (is_w ? W_BYTES : A_BYTES));      // (both CTAs' bytes)
                    tma_2d<PAIR>(ring + s * STAGE + (is_w ? 0 : W_BYTES), is_w ? &wmap : &amap, k * GI_STEP, row, PAIR ? at_rank(full + 8u * s, 0) : full + 8u * s);
                }
                __syncwarp();
                if (++s == NS) { s = 0; ph ^= 1u; }
            }
        }
        if (!alive && rank == 0) i8_drain(full, NS, s, ph);
    } else if (warp == GI_MMA) {
        const uint32_t idesc = i8_idesc(PAIR ? 2 * GI_M : GI_M, TN);
        uint32_t s = 0, ph = 0, it = 0;
        if (!PAIR || rank == 0)
            for (int item = first; item < tiles; item += stride, it++) {
                const uint32_t buf = it & 1u;
                bar_wait(acc_empty + 8u * buf, ((it >> 1) & 1u) ^ 1u, alive, 2);
                if (PAIR) asm volatile("fence.acq_rel.cluster;" ::: "memory");
                umma_after_sync();
                for (int k = 0; k < steps; k++) {
                    bar_wait(full + 8u * s, ph, alive, 3);
                    alive = __all_sync(0xffffffffu, alive);
                    umma_after_sync();
                    if (elect()) {
                        if (alive) i8_mma_step<PAIR>(tmem + buf * TN, ring + s * STAGE, ring + s * STAGE + W_BYTES, idesc, k == 0);
                        umma_commit<PAIR>(empty + 8u * s);
                        if (k == steps - 1) umma_commit<PAIR>(acc_full + 8u * buf);
                    }
                    __syncwarp();
                    if (++s == NS) { s = 0; ph ^= 1u; }
                }
            }
    } else {
        // warps w and w + 4 read the lanes 32 (w & 3) .. + 31 (weight rows), every second batch of 32 tokens each
        uint32_t it = 0;
        for (int item = first; item < tiles; item += stride, it++) {
            const uint32_t buf = it & 1u;
            const int m = PAIR ? 2 * (item / nt) + (int)rank : item / nt, t0 = (item % nt) * TN, n = m * GI_M + (threadIdx.x & 127), rows = min(TN, g.t - t0);
            const bool live = n < g.n;
            const float ws = live ? g.ws[n] : 0.0f, bias = live && g.bias ? g.bias[n] : 0.0f;
            bar_wait(acc_full + 8u * buf, (it >> 1) & 1u, alive, 4);
            umma_after_sync();
#pragma unroll 1
            for (int c0 = 32 * (warp >> 2); c0 < rows; c0 += 64) {
                uint32_t v[32];
                tmem_ld32(v, tmem + buf * TN + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c0);
                const float as = c0 + lane < rows ? g.as[t0 + c0 + lane] : 0.0f;
                T* out = reinterpret_cast<T*>(g.out) + (int64_t)(t0 + c0) * g.ldo + n;
#pragma unroll
                for (int c = 0; c < 32; c++) {
                    const float sc = __shfl_sync(0xffffffffu, as, c);
                    if (live && c0 + c < rows) out[c * g.ldo] = i8_result<T>((int)v[c], sc, ws, bias);
                }
            }
            umma_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(at_rank(acc_empty + 8u * buf, 0)) : "memory");
                else bar_arrive(acc_empty + 8u * buf);
            }
        }
    }
    __syncwarp();
    umma_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync();      // nobody leaves while the other's copies, commits or arrivals may still come here
    if (warp == GI_MMA) tmem_free<PAIR>(tmem, 2 * TN);
}

template <int TN> struct SplitRing {
    static constexpr int W_BYTES = GI_M * GI_STEP, A_BYTES = TN * GI_STEP, STAGE = W_BYTES + A_BYTES, NS = GI_RING / STAGE < 10 ? GI_RING / STAGE : 10;
    static constexpr size_t SMEM = (size_t)NS * STAGE + 1024;
    static_assert(TN * GI_M * 4 <= NS * STAGE, "the partial sums lie over the drained ring");
};
template <typename T, int TN>
__global__ void __launch_bounds__(GI_THREADS, 1) gemm_i8_split_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap wmap, const GemmI8Args g) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using Ring = SplitRing<TN>;
    constexpr int NS = Ring::NS, COLS = TN < 32 ? 32 : TN;
    __shared__ __align__(8) unsigned long long s_bar[2 * NS + 2];
    __shared__ uint32_t s_tmem;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, S = g.splits, rank = blockIdx.x % S, m = blockIdx.x / S, t0 = blockIdx.y * TN;
    const uint32_t ring = (sm_u32(smem) + 1023u) & ~1023u;
    const uint32_t full = sm_u32(s_bar), empty = full + 8u * NS, acc_full = full + 16u * NS;
    i8_setup<false>(full, NS, 1, &s_tmem, COLS);
    before();
    const uint32_t tmem = s_tmem;
    const int all = (g.k + GI_STEP - 1) / GI_STEP, k_beg = (int)((int64_t)rank * all / S), k_end = (int)((int64_t)(rank + 1) * all / S);      // (S <= all)
    bool alive = true;
    if (warp == GI_LOAD_W || warp == GI_LOAD_A) {
        const bool is_w = warp == GI_LOAD_W;
        uint32_t s = 0, ph = 1;
        for (int k = k_beg; k < k_end; k++) {
            bar_wait(empty + 8u * s, ph, alive, 1);
            alive = __all_sync(0xffffffffu, alive);
            if (!alive) break;
            if (elect()) {
                bar_expect(full + 8u * s, is_w ? Ring::W_BYTES : Ring::A_BYTES);
                tma_2d<false>(ring + s * Ring::STAGE + (is_w ? 0 : Ring::W_BYTES), is_w ? &wmap : &amap, k * GI_STEP, is_w ? m * GI_M : t0, full + 8u * s);
            }
            __syncwarp();
            if (++s == NS) { s = 0; ph ^= 1u; }
        }
        if (!alive) i8_drain(full, NS, s, ph);
    } else if (warp == GI_MMA) {
        const uint32_t idesc = i8_idesc(GI_M, TN);
        uint32_t s = 0, ph = 0;
        for (int k = k_beg; k < k_end; k++) {
            bar_wait(full + 8u * s, ph, alive, 3);
            alive = __all_sync(0xffffffffu, alive);
            umma_after_sync();
            if (elect()) {
                if (alive) i8_mma_step<false>(tmem, ring + s * Ring::STAGE, ring + s * Ring::STAGE + Ring::W_BYTES, idesc, k == k_beg);
                umma_commit<false>(empty + 8u * s);
                if (k == k_end - 1) umma_commit<false>(acc_full);
            }
            __syncwarp();
            if (++s == NS) { s = 0; ph ^= 1u; }
        }
    }
    __syncwarp();
    const int rows = min(TN, g.t - t0), row = threadIdx.x & 127, n = m * GI_M + row;
    const bool live = n < g.n;
    int* part = reinterpret_cast<int*>(smem + (ring - sm_u32(smem)));      // [TN tokens][128 rows] over the drained ring
    if (warp < GI_EPI_WARPS) {
        const float ws = live && S == 1 ? g.ws[n] : 0.0f, bias = live && S == 1 && g.bias ? g.bias[n] : 0.0f;
        bar_wait(acc_full, 0, alive, 4);
        umma_after_sync();
#pragma unroll 1
        for (int c0 = 32 * (warp >> 2); c0 < rows; c0 += 64) {
            uint32_t v[32];
            tmem_ld32(v, tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c0);
            if (S == 1) {
                const float as = c0 + lane < rows ? g.as[t0 + c0 + lane] : 0.0f;
                T* out = reinterpret_cast<T*>(g.out) + (int64_t)(t0 + c0) * g.ldo + n;
#pragma unroll
                for (int c = 0; c < 32; c++) {
                    const float sc = __shfl_sync(0xffffffffu, as, c);
                    if (live && c0 + c < rows) out[c * g.ldo] = i8_result<T>((int)v[c], sc, ws, bias);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 32; c++)
                    if (c0 + c < rows) part[(c0 + c) * GI_M + row] = (int)v[c];
            }
        }
    }
    umma_before_sync();
    if (S > 1) {
        cluster_sync();
        if (warp < GI_EPI_WARPS) {
            const int c_beg = rank * rows / S, c_end = (rank + 1) * rows / S;
            const float ws = live ? g.ws[n] : 0.0f, bias = live && g.bias ? g.bias[n] : 0.0f;
            constexpr int AT_ONCE = 4;      // tokens whose sums a thread asks for together
            for (int c0 = c_beg + (int)(threadIdx.x >> 7); c0 < c_end; c0 += 2 * AT_ONCE) {
                int v[AT_ONCE][8], sum[AT_ONCE];
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
                    for (int r = 0; r < 8; r++)
                        if (r < S) v[u][r] = peer_s32(ring + (uint32_t)(min(c0 + 2 * u, c_end - 1) * GI_M + row) * 4u, (uint32_t)r);
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++) {
                    sum[u] = 0;
#pragma unroll
                    for (int r = 0; r < 8; r++) sum[u] += r < S ? v[u][r] : 0;
                    const int c = c0 + 2 * u;
                    if (live && c < c_end) reinterpret_cast<T*>(g.out)[(int64_t)(t0 + c) * g.ldo + n] = i8_result<T>(sum[u], g.as[t0 + c], ws, bias);
                }
            }
        }
        cluster_sync();      // nobody leaves while its sums are read
    } else {
        __syncthreads();
    }
    umma_after_sync();
    if (warp == GI_MMA) tmem_free<false>(tmem, COLS);
}

// ------------------------------------------------------------------------------------------------------------------- host
struct GemmI8Plan {
    int tn, splits;
    bool wide, pair;
};
// The kernel of least estimated time (ns) on 148 SMs, by what each one measured (bf16 results, weights from DRAM): a step of 128 bytes of K takes 225 + 0.4 TN (wide: 280 with 128 tokens, 361 with 256, 300 for a
// pair), whatever its MMAs, since it is a step's copies that bound it (a pair's MMAs take 276 of its 300); a launch 2300 + 20 TN for its first bytes and its last sums, the exchange of a cut 400 and 30 per token and CTA; a wide kernel's start and last tile
// 5900, 8200 and 9500.  Clusters of 8 do not tile the chip's groups of SMs: 112 of their CTAs run at once.
// Measured (us; t x n x k): 1 x 4096 x 4096 10.2 in one piece, 7.5 in two, 6.6 in four, 13.7 in eight; 160 x 4096 x 4096 in tiles of 64 tokens 11.9, of 128 13.8; 2048 x 2048 x 2048 wide 13.8, 128 and 14.9 of 128 tokens;
// 384 x 14336 x 4096 28.6 in pairs, 32.8 and 33.6 without.
inline GemmI8Plan gemm_i8_plan(int64_t t, int64_t k, int64_t n) {
    const int64_t steps = (k + GI_STEP - 1) / GI_STEP, mt = (n + GI_M - 1) / GI_M;
    GemmI8Plan best{128, 1, false, false};
    int64_t least = -1;
    auto offer = [&](GemmI8Plan p, int64_t cost) {
        if (least < 0 || cost < least) { least = cost; best = p; }
    };
    for (int tn : {16, 32, 64, 128}) {
        if ((tn < 64 && t > tn) || (t + tn - 1) / tn > 65535) continue;      // (the grid's second dimension; such a call has enough tiles for the wide kernels)
        for (int s : {1, 2, 4, 8}) {
            if (s > steps) break;
            const int64_t fit = s == 8 ? 112 : s == 4 ? 140 : 148, waves = (mt * ((t + tn - 1) / tn) * s + fit - 1) / fit;
            offer({tn, s, false, false}, 300 + waves * ((steps + s - 1) / s * (225 + 2 * tn / 5) + 2000 + 20 * tn + (s > 1 ? 400 + 30 * tn / s : 0)));
        }
        if (t <= tn) break;
    }
    if (t > 128 || least < 0) {
        offer({128, 1, true, false}, 5900 + (mt * ((t + 127) / 128) + 147) / 148 * steps * 280);
        offer({256, 1, true, false}, 8200 + (mt * ((t + 255) / 256) + 147) / 148 * steps * 361);
        offer({256, 1, true, true}, 9500 + ((mt + 1) / 2 * ((t + 255) / 256) + 73) / 74 * steps * 300);
    }
    return best;
}
struct GemmI8Call {
    CUtensorMap amap, wmap;
    GemmI8Args g;
    GemmI8Plan plan;
    cudaStream_t st;
};
template <typename T, int TN, bool PAIR> cudaError_t gemm_i8_wide(const GemmI8Call& c) {
    static SmemAllowed allowed;
    const auto kernel = gemm_i8_wide_kernel<T, TN, PAIR>;
    const cudaError_t e = allowed((const void*)kernel, GI_RING + 1024);
    if (e != cudaSuccess) return e;
    const int64_t mt = (c.g.n + GI_M - 1) / GI_M, nt = (c.g.t + TN - 1) / TN;
    const int64_t grid = PAIR ? 2 * std::min<int64_t>((mt + 1) / 2 * nt, 74) : std::min<int64_t>(mt * nt, 148);
    return launch(kernel, dim3((unsigned)grid), GI_THREADS, GI_RING + 1024, PAIR ? 2 : 1, c.st, c.amap, c.wmap, c.g);
}
template <typename T, int TN> cudaError_t gemm_i8_split(const GemmI8Call& c) {
    static SmemAllowed allowed;
    const auto kernel = gemm_i8_split_kernel<T, TN>;
    const cudaError_t e = allowed((const void*)kernel, SplitRing<TN>::SMEM);
    if (e != cudaSuccess) return e;
    return launch(kernel, dim3((unsigned)((c.g.n + GI_M - 1) / GI_M * c.g.splits), (unsigned)((c.g.t + TN - 1) / TN)), GI_THREADS, SplitRing<TN>::SMEM, c.g.splits, c.st, c.amap, c.wmap, c.g);
}
template <typename T> cudaError_t gemm_i8(const int8_t* a, int64_t lda, const int8_t* w, int64_t ldw, GemmI8Args g, cudaStream_t st) {
    GemmI8Call c{};
    c.plan = gemm_i8_plan(g.t, g.k, g.n);
    c.g = g;
    c.g.splits = c.plan.splits;
    c.st = st;
    if (!byte_map(&c.amap, a, g.k, g.t, lda, c.plan.pair ? c.plan.tn / 2 : c.plan.tn) || !byte_map(&c.wmap, w, g.k, g.n, ldw, GI_M)) return cudaErrorInvalidValue;
    if (c.plan.wide) return c.plan.pair ? gemm_i8_wide<T, 256, true>(c) : c.plan.tn == 256 ? gemm_i8_wide<T, 256, false>(c) : gemm_i8_wide<T, 128, false>(c);
    return c.plan.tn == 16 ? gemm_i8_split<T, 16>(c) : c.plan.tn == 32 ? gemm_i8_split<T, 32>(c) : c.plan.tn == 64 ? gemm_i8_split<T, 64>(c) : gemm_i8_split<T, 128>(c);
}

}  // namespace dev
