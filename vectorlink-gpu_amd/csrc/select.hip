// The choice of blocks for rows that attend_step_kernel does not take.
#include "select_device.h"

namespace {

constexpr int kChunk = 64;  // blocks that a workgroup of score_kernel scores: a tile for every wavefront
constexpr int kLdsKeys = 16384 - 2048;  // scores that a workgroup of choose_kernel keeps in LDS: two workgroups on a compute unit

// Tokens that share a workgroup of choose_kernel; 0: one token's scores are too many
int tokens_together(const SelectArgs &a) {
    const int fit = kLdsKeys / (a.t.blocks > 1 ? a.t.blocks : 1), T = tokens_a_tile(a.group);
    return fit < T ? fit : T;
}

// What a workgroup of choose_kernel has of LDS beside the scores
struct ChooseKernelLds {
    ScoreLds<4> score;
    ChooseLds<1> choose[4];
};

// A workgroup scores all blocks of T tokens for one head into LDS, then every wavefront chooses for a token at a time.
template <int D, int NS, bool WHOLE>
__global__ __launch_bounds__(256) void choose_kernel(SelectArgs a, int T) {
    extern __shared__ uint32_t s_keys[];  // [T][a.t.blocks]
    __shared__ ChooseKernelLds s;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    Piece w = {(int)blockIdx.x, 0};
    if (a.t.offsets) w = find_piece(a.t.sequences, blockIdx.x, [&](int b) { return (row_count(a.t, b) + T - 1) / T; });
    if (w.sequence < 0) return;
    const int b = w.sequence, all = row_count(a.t, b), length = length_of(a.t, b);
    const int place0 = (int)min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all;
    const Scored what = {b, (int)blockIdx.y, w.piece * T, min(T, all - w.piece * T), place0, length, first_row(a.t, b)};
    const int last = min(place0 + what.token0 + what.tokens, length) - 1;
    const int blocks = last < 0 ? 0 : last / kPage + 1;
    score_blocks<D, NS, 4, WHOLE>(a, what, 0, blocks, s_keys, a.t.blocks, s.score);
    __syncthreads();
    for (int token = wave; token < what.tokens; token += 4) {
        const int place = min(place0 + what.token0 + token, length - 1), n = place < 0 ? 0 : place / kPage + 1;
        int32_t *const out = a.out + ((what.row0 + what.token0 + token) * a.c.heads + what.h) * a.count;
        const int found = choose<1>(s_keys + token * a.t.blocks, n, a.count, s.choose[wave], [&](int at, int i) { out[at] = i; });
        for (int i = found + lane; i < a.count; i += 64) out[i] = VL_MAXINT;
    }
}

// A workgroup scores kChunk blocks of one token and head.
template <int D, int NS, bool WHOLE>
__global__ __launch_bounds__(256) void score_kernel(SelectArgs a, int chunks) {
    __shared__ ScoreLds<4> s_score;
    const int row = blockIdx.x / chunks, from = blockIdx.x % chunks * kChunk, h = blockIdx.y;
    const Standing at = standing_of(a.t, row);
    if (!at.real || from >= at.blocks) return;
    const Scored s = {at.b, h, at.token, 1, at.place0, at.length, row - at.token};
    score_blocks<D, NS, 4, WHOLE>(a, s, from, min(from + kChunk, at.blocks), a.keys + ((int64_t)row * a.c.heads + h) * a.t.blocks, 0, s_score);
}
__global__ __launch_bounds__(512) void select_kernel(SelectArgs a) {
    __shared__ ChooseLds<8> s_choose;
    const int row = blockIdx.x, h = blockIdx.y;
    const Standing at = standing_of(a.t, row);
    if (!at.real) return;
    int32_t *const out = a.out + ((int64_t)row * a.c.heads + h) * a.count;
    const int found = choose<8>(a.keys + ((int64_t)row * a.c.heads + h) * a.t.blocks, at.blocks, a.count, s_choose, [&](int k, int i) { out[k] = i; });
    for (int i = found + threadIdx.x; i < a.count; i += 512) out[i] = VL_MAXINT;
}

template <int NS, bool WHOLE>
int launch(const SelectArgs &a, hipStream_t stream) {
    hipError_t e = hipSuccess;
    if (chosen_in_one(a)) {
        const int T = tokens_together(a);
        const int64_t tiles = a.t.offsets ? a.t.rows / T + sequences_with_rows(a.t) : a.t.rows;
        VL_REQUIRE(tiles <= 4 * kMaxBlocks, "more rows than one call takes: %lld", (long long)tiles);
        const size_t lds = (size_t)T * a.t.blocks * 4;
        for_dim(a.c.dim, [&](auto d) {
            constexpr int D = decltype(d)::value;
            e = vl_allow_lds(choose_kernel<D, NS, WHOLE>, lds + sizeof(ChooseKernelLds));  // both count towards a launch's 64 KiB
            if (e == hipSuccess) choose_kernel<D, NS, WHOLE><<<dim3((unsigned)tiles, (unsigned)a.c.heads), 256, lds, stream>>>(a, T);
        });
    } else {
        const int chunks = (a.t.blocks + kChunk - 1) / kChunk;
        VL_REQUIRE((int64_t)a.t.rows * chunks <= 4 * kMaxBlocks, "more rows than one call takes: %d of %d blocks", a.t.rows, a.t.blocks);
        for_dim(a.c.dim, [&](auto d) {
            score_kernel<decltype(d)::value, NS, WHOLE><<<dim3((unsigned)(a.t.rows * chunks), (unsigned)a.c.heads), 256, 0, stream>>>(a, chunks);
        });
        VL_LAUNCH_CHECK("score_kernel");
        select_kernel<<<dim3((unsigned)a.t.rows, (unsigned)a.c.heads), 512, 0, stream>>>(a);
    }
    VL_HIP(e);
    VL_LAUNCH_CHECK("select_kernel");
    return VL_OK;
}

}  // namespace

bool chosen_in_one(const SelectArgs &a) { return tokens_together(a) > 0 && (a.t.blocks <= 1024 || (int64_t)a.t.rows * a.c.heads >= kComputeUnits); }

int64_t select_workspace_bytes(const SelectArgs &a) {
    return chosen_in_one(a) ? 0 : ((int64_t)a.t.rows * a.c.heads * a.t.blocks * 4 + 255) / 256 * 256;
}

int launch_select(const SelectArgs &a, int type, hipStream_t stream) {
    if (a.group > 16)
        return type == VL_BF16 ? launch<1, true>(a, stream) : type == VL_F16 ? launch<2, true>(a, stream) : launch<3, true>(a, stream);
    return type == VL_BF16 ? launch<1, false>(a, stream) : type == VL_F16 ? launch<2, false>(a, stream) : launch<3, false>(a, stream);
}
