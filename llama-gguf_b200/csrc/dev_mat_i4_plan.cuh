// dev_mat_i4_plan.cuh — what the kernels of dev_mat_i4.cuh hold in shared memory, and how many of its bytes they read.  Plain arithmetic (compiled by the host compiler in tests/test_device_experts_plan_host.py).
#pragma once
#include <stddef.h>

#if defined(__CUDACC__)
#define I4_FN __host__ __device__ constexpr
#else
#define I4_FN constexpr
#endif

namespace dev {

enum { I4_TILE = 512, I4_PAIRS = 2048, I4_RING = 3 };      // bytes of a tile, pairs of a launch, steps of a warp's ring (few rows)
enum { I4_TEAMS = 4, I4_TEAM_WARPS = 4, I4_TEAM_TILES = 8, I4_MANY_ROWS = 64, I4_MANY_RING = 4 };      // more rows

// the lists of pairs by expert (I4List)
I4_FN size_t i4_list_bytes(int experts, int pairs) { return (size_t)(2 * (experts + 2)) * 4 + (size_t)pairs * 4; }
// What a ring holds of a step of `tiles` tiles' channels of one tile of rows: the weights, then the groups' scales.
I4_FN int i4_slot(int scale_bytes, int group, int tiles) { return tiles * I4_TILE + 16 * scale_bytes * (64 * tiles / group); }

// More rows: a step of a team's ring, the unit's weights and `rows` rows of 128 channels of a.
I4_FN int i4_many_slot(int scale_bytes, int group, int rows) { return I4_TEAM_TILES * i4_slot(scale_bytes, group, 2) + rows * 128; }
// Blocks of eight columns that are computed (and whose rows of a are read from a step) where `blocks` of them have a row
I4_FN int i4_many_blocks(int blocks) { return blocks <= 2 ? 2 : blocks == 7 ? 8 : blocks; }
struct I4ManyPlan {
    int most, ring;      // rows that a step has room for, steps of a team's ring
    size_t smem;         // bytes of the launch
};
enum { I4_MANY_OWN = I4_MANY_ROWS * 16, I4_MANY_MOST = 227 * 1024 - I4_MANY_OWN };      // the kernel's own places of rows; what is left for a launch to ask for
// rows: of out in the call; n_experts 0: one matrix
I4_FN I4ManyPlan i4_many_plan(int scale_bytes, int group, int rows, int n_experts) {
    I4ManyPlan p{};
    const int listed = rows < I4_PAIRS ? rows : I4_PAIRS, lists = n_experts ? (int)i4_list_bytes(n_experts, listed) : 0;
    p.most = 8 * i4_many_blocks((rows < I4_MANY_ROWS ? rows + 7 : I4_MANY_ROWS) / 8);      // (whole blocks as they are computed: 49 to 56 rows have eight)
    const int step = I4_TEAMS * i4_many_slot(scale_bytes, group, p.most), fit = (I4_MANY_MOST - lists) / step;
    p.ring = fit < I4_MANY_RING ? fit : I4_MANY_RING;      // (two at least: 144 KiB and the longest lists' 16)
    p.smem = (size_t)p.ring * step;
    return p;
}

}  // namespace dev
