// A choice of blocks and attention over it in one launch: a workgroup of 8 wavefronts for a token and a head of the cache.
//
// A batch of answers has few tokens, and what its choice reads - 2 D bytes a block, then the chosen blocks - is little: four
// launches (scores, choice, attention, join) wait for each other longer than they work.
#pragma once
#include "attend_few.h"
#include "select_device.h"

constexpr int kStepWaves = 8;

template <int D, int NS, int C>
__global__ __launch_bounds__(512) void attend_step_kernel(AttendArgs a, SelectArgs s) {
    typedef JoinLds<kStepWaves> Join;
    extern __shared__ __attribute__((aligned(16))) char lds[];  // scores [blocks] and then the join's sums; behind them the list [count]
    __shared__ ScoreLds<kStepWaves> s_score;
    __shared__ ChooseLds<kStepWaves> s_choose;
    uint32_t *const keys = (uint32_t *)lds;
    const size_t front = max(sizeof(Join), (size_t)s.t.blocks * 4 + 15 & ~(size_t)15);
    int32_t *const list = (int32_t *)(lds + front);

    const int row = blockIdx.x / a.c.heads, h = blockIdx.x % a.c.heads;
    const int lane = threadIdx.x & 63, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Standing at = standing_of(a.t, row);
    if (!at.real) return;
    const int b = __builtin_amdgcn_readfirstlane(at.b), blocks = __builtin_amdgcn_readfirstlane(at.blocks);
    const Scored what = {b, h, at.token, 1, at.place0, at.length, row - at.token};
    const bool real = r < a.group;
    score_blocks<D, NS, kStepWaves, false>(s, what, 0, blocks, keys, 0, s_score);
    __syncthreads();
    int32_t *const out = s.out + ((int64_t)row * a.c.heads + h) * s.count;
    const int found = choose<kStepWaves>(keys, blocks, s.count, s_choose, [&](int k, int i) {
        out[k] = i;
        list[k] = i;
    });
    for (int i = found + threadIdx.x; i < s.count; i += 512) out[i] = VL_MAXINT;
    __syncthreads();

    const int sees = max(min(at.place0 + at.token + 1, at.length), 0);
    QueryLoads<D, NS> f;
    load_queries<D, NS>(f, a, real, row, h * a.group + r);
    RowState<D> st;
    start_rows<D>(st);
    const int most = __builtin_amdgcn_readfirstlane(sees), length = __builtin_amdgcn_readfirstlane(at.length);
    take_blocks<D, NS, C>(st, a, f, real, {list, wave, kStepWaves, found}, b, h, C < 16 || real ? sees : 0, most, most, length);
    __syncthreads();
    join_waves<D, NS, kStepWaves, C>(st, *(Join *)lds, a, 0, [&](int r) { return r < a.group ? (int64_t)row * a.heads_q + h * a.group + r : -1; });
}
