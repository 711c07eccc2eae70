// Attention over the cache: what its kernels and their launchers share.
#pragma once
#include "cache8.h"
#include "select.h"

// S = scale <query, key>, P = softmax of S over the tokens that a row sees, out = P values.
struct AttendArgs {
    CacheView c;
    int bits;               // 4 or 8
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
    // of a cache in 8 bits whose tokens' weights are added up
    float *ends;            // [rows, heads_q, 2] or null: the maximum of a row's scores and the sum of its weights
    float *scores;          // [rows, c.heads, t.blocks, group, 64] or null: the scores of single tokens, unscaled
    float *part;            // splits > 1: [rows * heads_q, splits, D] sums, then [rows * heads_q, splits, 2] maxima and sums of weights
};
constexpr int kMaxSplits = 64;

// Weights are exp2(scale s - top) with one rounding, of the difference, where top is rounded: a largest score of 2^k finds itself up to
// 2^(k - 24) above or below it, which its row's sum takes out again, until it leaves no float32 - the row would be NaN, or zeros.
// Where top is beyond 2^28 (16 either way) the scores are rounded as it is.
__device__ inline bool is_far(float top) { return __builtin_fabsf(top) > 0x1p28f; }

// 16 rows at a time, the tokens split over wavefronts and workgroups
template <int NS, int BITS = 4>
int launch_attend_few(const AttendArgs &a, int64_t tiles, hipStream_t stream);
// 32 rows a wavefront, all of a workgroup's on the same pages: 8 wavefronts, or 4 where a row's registers are many
constexpr int many_waves(int dim) { return dim <= 128 ? 8 : 4; }
constexpr bool many_built(int dim, int parts) { return dim * parts <= 256; }
// pages a round: two where two sets of them fit LDS (2,048 rows over 16,384 tokens of 128: 503 us with one, 492 with two; of 64: 365
// and 333)
constexpr int many_pages(int dim) { return dim <= 128 ? 2 : 1; }
template <int NS, int BITS = 4>
int launch_attend_many(const AttendArgs &a, int64_t tiles, hipStream_t stream);
// a choice of blocks and attention over it, a workgroup for a token and head; longer rows of other types do not fit the registers
constexpr bool step_built(int dim, int parts) { return dim <= 128 || parts == 1; }
template <int NS>
int launch_attend_step(const AttendArgs &a, const SelectArgs &s, hipStream_t stream);
// the weights that the rows' queries give the tokens, added to the cache's: from the scores of a call, or from the keys once more
int launch_weigh_scores(const AttendArgs &a, hipStream_t stream);
template <int NS>
int launch_weigh_rows(const AttendArgs &a, hipStream_t stream);
extern template int launch_attend_few<1, 4>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<1, 4>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_few<1, 8>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<1, 8>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_step<1>(const AttendArgs &, const SelectArgs &, hipStream_t);
extern template int launch_weigh_rows<1>(const AttendArgs &, hipStream_t);
extern template int launch_attend_few<2, 4>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<2, 4>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_few<2, 8>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<2, 8>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_step<2>(const AttendArgs &, const SelectArgs &, hipStream_t);
extern template int launch_weigh_rows<2>(const AttendArgs &, hipStream_t);
extern template int launch_attend_few<3, 4>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<3, 4>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_few<3, 8>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_many<3, 8>(const AttendArgs &, int64_t, hipStream_t);
extern template int launch_attend_step<3>(const AttendArgs &, const SelectArgs &, hipStream_t);
extern template int launch_weigh_rows<3>(const AttendArgs &, hipStream_t);
