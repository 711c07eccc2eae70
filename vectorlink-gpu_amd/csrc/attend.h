// Attention over the cache: what its kernels and their launchers share.
#pragma once
#include "select.h"

// S = scale <query, key>, P = softmax of S over the tokens that a row sees, out = P values.
struct AttendArgs {
    CacheView c;
    Tokens t;
    const void *queries;
    int64_t q_row, q_head;  // strides in elements
    void *out;              // [rows, heads_q, D]
    float *lse;             // [rows, heads_q] or null
    const int32_t *list;    // [rows, c.heads, count] blocks of every row and head, or null: all blocks
    int count;
    int group, heads_q;     // queries that share a head of the cache; c.heads * group
    int causal;
    float scale;            // |scale| log2(e): exponentials are powers of two here
    float turn;             // the scale's sign, 0 for no scale at all: what the queries are multiplied with
    int splits;             // workgroups that share a tile
    int waves;              // of attend_few_kernel: wavefronts of a workgroup that share a tile, 4 or 8; 1: four have one each
    float *part;            // splits > 1: [rows * heads_q, splits, D] sums, then [rows * heads_q, splits, 2] maxima and sums of weights
};
constexpr int kMaxSplits = 64;

// 16 rows at a time, the tokens split over wavefronts and workgroups
template <int NS>
int launch_attend_few(const AttendArgs &a, int64_t tiles, hipStream_t stream);
// 32 rows a wavefront, all of a workgroup's on the same pages: 8 wavefronts, or 4 where a row's registers are many
constexpr int many_waves(int dim) { return dim <= 128 ? 8 : 4; }
constexpr bool many_built(int dim, int parts) { return dim * parts <= 256; }
// pages a round: two where two sets of them fit LDS (2,048 rows over 16,384 tokens of 128: 503 us with one, 492 with two; of 64: 365
// and 333)
constexpr int many_pages(int dim) { return dim <= 128 ? 2 : 1; }
template <int NS>
int launch_attend_many(const AttendArgs &a, int64_t tiles, hipStream_t stream);
// a choice of blocks and attention over it, a workgroup for a token and head; longer rows of other types do not fit the registers
constexpr bool step_built(int dim, int parts) { return dim <= 128 || parts == 1; }
template <int NS>
int launch_attend_step(const AttendArgs &a, const SelectArgs &s, hipStream_t stream);
extern template int launch_attend_few<1>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_few<2>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_few<3>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<1>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<2>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<3>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_step<1>(const AttendArgs &, const SelectArgs &, hipStream_t);
extern template int launch_attend_step<2>(const AttendArgs &, const SelectArgs &, hipStream_t);
extern template int launch_attend_step<3>(const AttendArgs &, const SelectArgs &, hipStream_t);
