// The choice of blocks for every row and head of the cache.
#pragma once
#include "cache.h"

struct SelectArgs {
    CacheView c;
    Tokens t;
    const void *queries;
    int64_t q_row, q_head;
    int group;
    int count;
    int turned;      // 1: the queries' signs are turned, for scores that a negative scale will be multiplied with
    int32_t *out;    // [rows, c.heads, count]
    uint32_t *keys;  // [rows, c.heads, t.blocks]: scores, in an order that unsigned numbers have
};
// One workgroup a token scores and chooses where that fills the GPU or the blocks are few; else they are scored by many.
bool chosen_in_one(const SelectArgs &a);
int64_t select_workspace_bytes(const SelectArgs &a);
int launch_select(const SelectArgs &a, int type, hipStream_t stream);
