// Attention over the cache: entry points, their checks, and how a call is cut into workgroups.
#include "attend.h"

#include <math.h>


namespace {

// Tokens times heads up to which one launch may take a choice and its attention: a workgroup for each compute unit (512 workgroups over
// 8,192 tokens each: 56 us, in several launches 45).
constexpr int64_t kStepItems = 256;

float in_powers_of_two(double scale) { return (float)(fabs(scale) * 1.4426950408889634); }

int cache_of(const vl_cache *cache, AttendArgs *a) {
    a->bits = 4;
    return vl_cache_of(cache, &a->c);
}
int cache_of(const vl_cache8 *cache, AttendArgs *a) {
    a->bits = 8;
    return vl_cache8_of(cache, &a->c);
}

template <class Cache>
int attend_args(const Cache *cache, const vl_tokens *tokens, const vl_queries *q, bool data, AttendArgs *a) {
    *a = {};
    int rc = cache_of(cache, a);
    if (rc == VL_OK) rc = vl_tokens_of(tokens, &a->t);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(q != nullptr, "queries is null");
    VL_REQUIRE(q->type >= VL_BF16 && q->type <= VL_F32, "type: %d", q->type);
    VL_REQUIRE(q->heads >= 1 && q->heads <= (1 << 24) && q->heads % a->c.heads == 0, "%lld heads of queries for %d of the cache",
               (long long)q->heads, a->c.heads);
    VL_REQUIRE(q->form == 0 || q->form == VL_ATTEND_FEW || (q->form == VL_ATTEND_MANY && many_built(a->c.dim, q->type)), "form: %lld",
               (long long)q->form);
    const int size = q->type == VL_F32 ? 4 : 2;
    if (data && a->t.rows) {
        VL_REQUIRE(q->queries && q->out, "queries or out is null");
        VL_REQUIRE((uintptr_t)q->queries % size == 0, "queries not aligned to their type");
        VL_REQUIRE(((uintptr_t)q->out & 15) == 0, "out not on a 16-byte boundary");
        VL_REQUIRE(isfinite(in_powers_of_two(q->scale)), "scale: %g is not finite, or too large for float32", q->scale);
    }
    a->queries = q->queries;
    a->q_row = q->row_stride;
    a->q_head = q->head_stride;
    a->out = q->out;
    a->lse = q->lse;
    a->heads_q = (int)q->heads;
    a->group = (int)(q->heads / a->c.heads);
    a->causal = q->causal != 0;
    a->scale = in_powers_of_two(q->scale);
    a->turn = q->scale < 0 ? -1.0f : 1.0f;
    if (a->scale == 0) {  // 0 times the -inf that masks a score would be none: the queries take the 0
        a->scale = 1;
        a->turn = 0;
    }
    a->splits = 1;
    return VL_OK;
}

// Tiles of 16 rows: rows of a sequence and a head come one after the other, and every sequence may end inside a tile.
int64_t few_tiles(const AttendArgs &a) {
    const int64_t per = (a.group + 15) / 16;
    if (a.count || !a.t.offsets) return a.t.rows * per;
    return (int64_t)a.t.rows * a.group / 16 + sequences_with_rows(a.t);
}

// How the pages of a tile are shared out.  A tile for every wavefront where that alone gives every SIMD two.  A workgroup of 8
// wavefronts for a tile where that leaves each at most four pages, two of a list, which takes no second launch to join (1,000 tokens, 32
// heads: 14.5 us in two launches, 10.3 in one; 8 tiles with lists of 16, 20 and 32 blocks, in a graph: 9.0, 9.7 and 12.3 us in one, 9.5,
// 9.5 and 9.6 in two).  Else workgroups of 4, as many a tile as give every compute unit one (two for float32,
// which is three times the products), but two pages (one) for every wavefront: parts cost their starts and ends, and joining them.
// One workgroup a compute unit and two: one sequence of 65,536 tokens 27 us and 36, 32 of 4,096 to 8,192 with 8 heads of 8 47 and 53,
// in float32 68 and 59.  Two pages a wavefront and one: 2 sequences of 16,384 19 us and 27.
struct Shares {
    int waves, splits;
};
Shares shares_for(const AttendArgs &a, int type, int64_t tiles) {
    const int64_t entries = a.count ? a.count : a.t.blocks;
    const int64_t items = tiles * a.c.heads;
    if (items == 0) return {4, 1};
    if (items >= 8 * kComputeUnits) return {1, 1};
    // of 8 bits 4 wavefronts are enough: 1,000 tokens 10.1 us with 4 and with 8, 1,536 11.8 and 12.6 (two launches 13.6), 2,048 13.8
    // and 14.7 (13.6), 32 sequences of 2,048 20.5 and 20.8 (23.7)
    if (a.bits == 8 && items <= kComputeUnits && entries <= 32) return {4, 1};
    if (a.c.dim <= 128 && items <= kComputeUnits && entries <= (a.count ? 16 : 32)) return {8, 1};
    const int64_t groups = (type == VL_F32 ? 2 : 1) * kComputeUnits, pages = type == VL_F32 ? 4 : 8;
    int64_t s = (groups + items - 1) / items;
    s = s < (entries + pages - 1) / pages ? s : (entries + pages - 1) / pages;
    return {4, (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s)};
}

int64_t part_bytes(const AttendArgs &a, int splits) {
    if (splits <= 1) return 0;
    return ((int64_t)a.t.rows * a.heads_q * splits * (a.c.dim + 2) * 4 + 255) / 256 * 256;
}

// Tiles of the rows of a workgroup of attend_many_kernel: at most, and about
int64_t many_tiles(const AttendArgs &a) { return (int64_t)a.t.rows * a.group / (32 * many_waves(a.c.dim)) + sequences_with_rows(a.t); }
int64_t many_tiles_about(const AttendArgs &a) {
    if (a.t.rows == 0) return 0;  // and perhaps no sequences either
    const int64_t sequences = sequences_with_rows(a.t);
    const int64_t rows = 32 * many_waves(a.c.dim), each = (int64_t)a.t.rows * a.group / sequences;
    return sequences * (each / rows + (each % rows != 0));
}

// Pages that the busiest compute unit takes one after the other, a workgroup's start and end counted as kEnds, if the tokens of a
// tile are split over `splits` workgroups.
constexpr int64_t kEnds = 3;
int64_t many_pages_in_turn(const AttendArgs &a, int64_t splits) {
    const int64_t groups = many_tiles_about(a) * a.c.heads * splits;
    return (groups + kComputeUnits - 1) / kComputeUnits * ((a.t.blocks + splits - 1) / splits + kEnds);
}
int many_splits(const AttendArgs &a) {
    int best = 1;
    for (int s = 2; s <= 32 && a.t.blocks / s >= 4; s++)
        if (many_pages_in_turn(a, s) < many_pages_in_turn(a, best)) best = s;
    return best;
}

// The form whose compute units are done first.  A page of a workgroup of attend_many_kernel takes a compute unit about as long as 8
// pages of 16 rows in attend_few_kernel take it (11 where queries are two or three parts): at 8,192 rows and 128 dimensions 2.0
// us against 0.26, half precision 3.4 and 0.28, so of a tile's 256 rows more than half have to be there; 6 for the 128 rows of longer
// ones (256 dimensions: 3.6 and 0.58).  Where a row's
// registers leave one wavefront a SIMD (half precision of 192, float32 of 96 and more) the few-row form is never slower: 256
// dimensions of float32 1026 us against 699.
bool takes_many(const AttendArgs &a, const vl_queries *q) {
    const int type = q->type;
    if (q->form) return q->form == VL_ATTEND_MANY;
    if (!a.t.offsets || !many_built(a.c.dim, type) || a.t.sequences == 0) return false;
    const int64_t few = ((int64_t)a.t.rows * a.group + 15) / 16 * a.c.heads * a.t.blocks / kComputeUnits;
    // Of 8 bits a page is twice the bytes for every tile that reads it, and what it takes to turn it into bfloat16 no more: 8 sequences of
    // 8,192, 32 heads on 8 of 128, us few and many: 8 rows each 57 and 68, 16 rows 103 and 70, 32 rows 160 and 77; one sequence 15 and 19,
    // 24 and 21, 29 and 25; 16 of 1,024 tokens with 16 rows 25 and 30, with 32 44 and 36.  64 dimensions change sides at 16 rows (54 and
    // 53), 32 at 24; half precision takes 91 for the 70, and changes sides at 14 and at 24 rows of 64; float32 of 64 at 50.  One figure does
    // for all longer rows: 8 sequences of 8,192 with 12 rows each and with 16, of 96 dimensions 46 and 60, 77 and 62, of 192 89 and 95, 122
    // and 96, of 256 115 and 115, 163 and 117; 10 rows, which are three tiles as 12 are, 98 and 94 of 192, 129 and 115 of 256.
    if (a.bits == 8) {
        const int at = a.c.dim <= 32 ? 0 : a.c.dim <= 64 ? 1 : 2;
        const int quarters[3][3] = {{24, 16, 12}, {28, 20, 14}, {44, 44, 44}};  // of such a unit, a page of the form for many rows
        return many_pages_in_turn(a, many_splits(a)) * quarters[type - VL_BF16][at] < few * 4;
    }
    return many_pages_in_turn(a, many_splits(a)) * (type != VL_BF16 ? 11 : a.c.dim <= 128 ? 8 : 6) < few;
}

int check_workspace(int64_t need, const void *workspace, int64_t bytes) {
    if (need > bytes || (need && !workspace)) {
        vl_set_error("workspace too small: %lld bytes needed, %lld given", (long long)need, (long long)bytes);
        return VL_ERR_WORKSPACE;
    }
    VL_REQUIRE(((uintptr_t)workspace & 15) == 0, "workspace not on a 16-byte boundary");
    return VL_OK;
}

template <int BITS = 4>
int attend_few(AttendArgs &a, int type, void *workspace, int64_t bytes, hipStream_t stream) {
    const int64_t tiles = few_tiles(a);
    const Shares shares = shares_for(a, type, tiles);
    a.waves = shares.waves;
    a.splits = shares.splits;
    const int rc = check_workspace(part_bytes(a, a.splits), workspace, bytes);
    if (rc != VL_OK) return rc;
    a.part = (float *)workspace;
    return type == VL_BF16 ? launch_attend_few<1, BITS>(a, tiles, stream) : type == VL_F16 ? launch_attend_few<2, BITS>(a, tiles, stream)
                                                                                         : launch_attend_few<3, BITS>(a, tiles, stream);
}

template <int BITS = 4>
int attend_many(AttendArgs &a, int type, void *workspace, int64_t bytes, hipStream_t stream) {
    const int64_t tiles = many_tiles(a);
    a.splits = many_splits(a);
    const int rc = check_workspace(part_bytes(a, a.splits), workspace, bytes);
    if (rc != VL_OK) return rc;
    a.part = (float *)workspace;
    return type == VL_BF16 ? launch_attend_many<1, BITS>(a, tiles, stream) : type == VL_F16 ? launch_attend_many<2, BITS>(a, tiles, stream)
                                                                                          : launch_attend_many<3, BITS>(a, tiles, stream);
}

// What a call over a cache in 8 bits has of its workspace: parts, and where weights are added up the rows' ends and, of single tokens
// whose queries are one tile, their scores.
struct Space {
    int64_t part, ends, scores;
    int64_t bytes() const { return part + ends + scores; }
};
Space space_of(const AttendArgs &a, const vl_queries *q, bool accumulate) {
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    const bool many = takes_many(a, q);
    Space s = {part_bytes(a, many ? many_splits(a) : shares_for(a, q->type, few_tiles(a)).splits), 0, 0};
    if (!accumulate || a.c.pages == 0) return s;  // without pages no token has a weight, nor are there any to read
    s.ends = up((int64_t)a.t.rows * a.heads_q * 8);
    // the scores of a token and head are reached by 31 bits; where tables are so wide that they would take more than 4 GiB, they are
    // made once more from the keys
    const int64_t scores = up((int64_t)a.t.rows * a.heads_q * a.t.blocks * kPage * 4);
    if (!many && !a.t.offsets && a.group <= 16 && a.t.blocks <= 1 << 18 && scores <= (int64_t)1 << 32) s.scores = scores;
    return s;
}

int check_count(int64_t count) {
    VL_REQUIRE(count >= 1 && count < (1 << 24), "count: %lld", (long long)count);
    return VL_OK;
}

SelectArgs select_args(const AttendArgs &a, int64_t count) {
    return {a.c, a.t, a.queries, a.q_row, a.q_head, a.group, (int)count, 0, nullptr, nullptr};
}

int choose(const AttendArgs &a, int type, int64_t count, bool turned, int32_t *blocks, void *workspace, int64_t bytes, hipStream_t stream) {
    SelectArgs s = select_args(a, count);
    s.turned = turned;
    const int rc = check_workspace(select_workspace_bytes(s), workspace, bytes);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(blocks, "blocks is null");
    s.out = blocks;
    s.keys = (uint32_t *)workspace;
    return launch_select(s, type, stream);
}

// What the single launch takes, in ns beside what both ways have in common: its workgroup works on one block after the other.
int64_t step_takes(const AttendArgs &a, int type, int64_t count) {
    const int64_t chosen = count * (40 + a.c.dim * 7 / 5);  // bfloat16
    return a.t.blocks * (36 + a.c.dim) / 18 + (type == VL_BF16 ? chosen : type == VL_F16 ? chosen * 11 / 10 : chosen * 3 / 2);
}
// What several launches take: one or two more, and 1 us because fewer are to be had for the same; a choice by a workgroup for a token,
// or scores by many (0.13 ns each) and a choice from them; the chosen pages at about 6 TB/s.
int64_t several_take(const AttendArgs &a, int64_t count) {
    const int64_t items = (int64_t)a.t.rows * a.c.heads, pages = items * count * (kPage * (a.c.dim + a.c.dim / 16)) / 6000;
    const int64_t choice = chosen_in_one(select_args(a, count)) ? a.t.blocks * (420 + a.c.dim) / 28 : 5000 + items * a.t.blocks * 13 / 100;
    return 2500 + 12 * a.c.dim + choice + pages;
}
// Whether attend_step_kernel takes a choice and the attention over it.  us in one launch and in several, next to where the rule changes
// sides, for 8 tokens times heads (bfloat16 of 128): 32 of 256 blocks 20.4 and 21.3, 64 of 256 26.9 and 21.2, 64 of 1,024 33.1 and 35.0, 128
// of 1,024 45.8 and 35.4, 16 of 1,024 23.8 and 33.6, 16 of 1,040 24.3 and 21.6; for 64: 64 of 300 28.2 and 25.2, of 1,000 34.8 and 38.5, of
// 2,000 43.5 and 36.2, 16 of 2,000 33.0 and 32.3; for 128: 256 of 300 67.1 and 61.3, of 1,000 73.5 and 74.4.  64 and 256 dimensions, half
// precision and float32 change sides as the figures above have it, to 2 us of 20 to 50.
bool in_one_step(const AttendArgs &a, int type, int64_t count) {
    return step_built(a.c.dim, type) && a.group <= 16 && a.t.blocks <= 16384 && count <= 2048 && (int64_t)a.t.rows * a.c.heads <= kStepItems &&
           step_takes(a, type, count) <= several_take(a, count);
}

}  // namespace

VL_EXPORT int vl_attend_form(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries) {
    AttendArgs a;
    const int rc = attend_args(cache, tokens, queries, false, &a);
    return rc != VL_OK ? rc : takes_many(a, queries) ? VL_ATTEND_MANY : VL_ATTEND_FEW;
}

VL_EXPORT int64_t vl_attend_workspace_bytes(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries) {
    AttendArgs a;
    const int rc = attend_args(cache, tokens, queries, false, &a);
    if (rc != VL_OK) return rc;
    if (takes_many(a, queries)) return part_bytes(a, many_splits(a));
    return part_bytes(a, shares_for(a, queries->type, few_tiles(a)).splits);
}

VL_EXPORT int vl_attend(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries, void *workspace,
                        int64_t workspace_bytes, void *stream) {
    AttendArgs a;
    const int rc = attend_args(cache, tokens, queries, true, &a);
    if (rc != VL_OK || a.t.rows == 0) return rc;
    return takes_many(a, queries) ? attend_many(a, queries->type, workspace, workspace_bytes, (hipStream_t)stream)
                                        : attend_few(a, queries->type, workspace, workspace_bytes, (hipStream_t)stream);
}

VL_EXPORT int vl_attend8_form(const vl_cache8 *cache, const vl_tokens *tokens, const vl_queries *queries) {
    AttendArgs a;
    const int rc = attend_args(cache, tokens, queries, false, &a);
    return rc != VL_OK ? rc : takes_many(a, queries) ? VL_ATTEND_MANY : VL_ATTEND_FEW;
}

VL_EXPORT int64_t vl_attend8_workspace_bytes(const vl_cache8 *cache, const vl_tokens *tokens, const vl_queries *queries, int accumulate) {
    AttendArgs a;
    const int rc = attend_args(cache, tokens, queries, false, &a);
    return rc != VL_OK ? rc : space_of(a, queries, accumulate != 0).bytes();
}

VL_EXPORT int vl_attend8(const vl_cache8 *cache, const vl_tokens *tokens, const vl_queries *queries, int accumulate, void *workspace,
                         int64_t workspace_bytes, void *stream) {
    AttendArgs a;
    int rc = attend_args(cache, tokens, queries, true, &a);
    if (rc != VL_OK || a.t.rows == 0) return rc;
    VL_REQUIRE(!accumulate || a.c.weights || a.c.pages == 0, "the cache has no weights");
    const Space space = space_of(a, queries, accumulate != 0);
    rc = check_workspace(space.bytes(), workspace, workspace_bytes);
    if (rc != VL_OK) return rc;
    if (space.ends) a.ends = (float *)((uint8_t *)workspace + space.part);
    if (space.scores) a.scores = (float *)((uint8_t *)workspace + space.part + space.ends);
    const hipStream_t s = (hipStream_t)stream;
    const int type = queries->type;
    rc = takes_many(a, queries) ? attend_many<8>(a, type, workspace, space.part, s) : attend_few<8>(a, type, workspace, space.part, s);
    if (rc != VL_OK || !accumulate) return rc;
    if (a.scores) return a.splits > 1 ? launch_weigh_scores(a, s) : VL_OK;  // one workgroup's alone are added by it
    return type == VL_BF16 ? launch_weigh_rows<1>(a, s) : type == VL_F16 ? launch_weigh_rows<2>(a, s) : launch_weigh_rows<3>(a, s);
}

VL_EXPORT int64_t vl_select_blocks_workspace_bytes(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries,
                                                   int64_t count) {
    AttendArgs a;
    int rc = attend_args(cache, tokens, queries, false, &a);
    if (rc == VL_OK) rc = check_count(count);
    return rc != VL_OK ? rc : select_workspace_bytes(select_args(a, count));
}

VL_EXPORT int vl_select_blocks(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries, int64_t count,
                               int32_t *blocks, void *workspace, int64_t workspace_bytes, void *stream) {
    AttendArgs a;
    int rc = attend_args(cache, tokens, queries, false, &a);
    if (rc == VL_OK) rc = check_count(count);
    if (rc != VL_OK || a.t.rows == 0) return rc;
    VL_REQUIRE(a.queries && (uintptr_t)a.queries % (queries->type == VL_F32 ? 4 : 2) == 0, "queries is null or not aligned to its type");
    return choose(a, queries->type, count, false, blocks, workspace, workspace_bytes, (hipStream_t)stream);
}

VL_EXPORT int64_t vl_attend_blocks_workspace_bytes(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries,
                                                   int64_t count) {
    AttendArgs a;
    int rc = attend_args(cache, tokens, queries, false, &a);
    if (rc == VL_OK) rc = check_count(count);
    a.count = (int)count;
    return rc != VL_OK ? rc : part_bytes(a, shares_for(a, queries->type, few_tiles(a)).splits);
}

VL_EXPORT int vl_attend_blocks(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries, const int32_t *blocks,
                               int64_t count, void *workspace, int64_t workspace_bytes, void *stream) {
    AttendArgs a;
    int rc = attend_args(cache, tokens, queries, true, &a);
    if (rc == VL_OK) rc = check_count(count);
    if (rc != VL_OK || a.t.rows == 0) return rc;
    VL_REQUIRE(blocks, "blocks is null");
    a.list = blocks;
    a.count = (int)count;
    return attend_few(a, queries->type, workspace, workspace_bytes, (hipStream_t)stream);
}

VL_EXPORT int64_t vl_attend_selected_workspace_bytes(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries,
                                                     int64_t count) {
    AttendArgs a;
    int rc = attend_args(cache, tokens, queries, false, &a);
    if (rc == VL_OK) rc = check_count(count);
    if (rc != VL_OK) return rc;
    if (in_one_step(a, queries->type, count)) return 0;
    a.count = (int)count;
    return select_workspace_bytes(select_args(a, count)) + part_bytes(a, shares_for(a, queries->type, few_tiles(a)).splits);
}

VL_EXPORT int vl_attend_selected(const vl_cache *cache, const vl_tokens *tokens, const vl_queries *queries, int64_t count,
                                 int32_t *blocks, void *workspace, int64_t workspace_bytes, void *stream) {
    AttendArgs a;
    int rc = attend_args(cache, tokens, queries, true, &a);
    if (rc == VL_OK) rc = check_count(count);
    if (rc != VL_OK || a.t.rows == 0) return rc;
    if (in_one_step(a, queries->type, count)) {
        VL_REQUIRE(blocks, "blocks is null");
        SelectArgs s = select_args(a, count);
        s.out = blocks;
        s.turned = queries->scale < 0;
        const hipStream_t at = (hipStream_t)stream;
        return queries->type == VL_BF16 ? launch_attend_step<1>(a, s, at) : queries->type == VL_F16 ? launch_attend_step<2>(a, s, at) : launch_attend_step<3>(a, s, at);
    }
    rc = choose(a, queries->type, count, queries->scale < 0, blocks, workspace, workspace_bytes, (hipStream_t)stream);
    if (rc != VL_OK) return rc;
    const int64_t used = select_workspace_bytes(select_args(a, count));
    a.list = blocks;
    a.count = (int)count;
    return attend_few(a, queries->type, workspace ? (uint8_t *)workspace + used : nullptr, workspace_bytes - used, (hipStream_t)stream);
}
