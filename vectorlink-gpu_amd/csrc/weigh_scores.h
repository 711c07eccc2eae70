// The weights that attention gave the tokens of a cache in 8 bits, added to those that it holds: w_t += sum over rows and the queries
// that share a head of exp2(scale s_t - max) / sum, with each row's maximum and sum as attention left them.  Here from the scores that
// a single token's attention left: by the workgroup that made them, or by a launch of its own where several made them.
#pragma once
#include "attend.h"

// What a row's scores are turned into weights with: exp2(scale s - max) * by.  A row that saw nothing, or something that is not finite,
// gives no weight to anything: exp2(s - inf) * 0, for scores that are finite.
struct RowEnds {
    float minus, by;
    bool fine;
};
__device__ inline RowEnds row_ends(float top, float total) {
    RowEnds r;
    r.fine = top > -INFINITY && top < INFINITY && total > 0 && total < INFINITY;
    r.minus = r.fine ? -top : -INFINITY;
    r.by = r.fine ? 1.0f / total : 0.0f;
    return r;
}

// Places from, from + STEP, ... < sees of a sequence and head, four at a time: the scores of the queries that share the head (at most G)
// are asked for all at once, and for U turns, 16 loads of scores.  ends(g): (max, sum) of query g.
template <int G, int STEP, class F>
__device__ inline void weigh_places(const AttendArgs &a, int b, int h, int from, int sees, F ends) {
    constexpr int U = 16 / G;
    const float *const scores = a.scores + ((int64_t)b * a.c.heads + h) * ((int64_t)a.t.blocks * a.group * kPage);
    for (; from < sees; from += U * STEP) {
        int64_t page[U];
        f32x4 s[U][G], w[U];
#pragma unroll
        for (int u = 0; u < U; u++) page[u] = from + u * STEP < sees ? page_of(a.t, a.c, b, (from + u * STEP) / kPage) : -1;
#pragma unroll
        for (int u = 0; u < U; u++) {  // of no page: loads of the cache's first, which there is, and nothing is made of them
            const int place = min(from + u * STEP, (sees - 1) & ~3);
            const float *const at = scores + (int64_t)(place / kPage) * a.group * kPage + place % kPage;
#pragma unroll
            for (int g = 0; g < G; g++) s[u][g] = *reinterpret_cast<const f32x4 *>(at + min(g, a.group - 1) * kPage);
            w[u] = *reinterpret_cast<const f32x4 *>(a.c.weights + (max(page[u], (int64_t)0) * a.c.heads + h) * kPage + place % kPage);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (page[u] < 0) continue;
            f32x4 sum = {0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < G; g++) {
                const RowEnds e = ends(min(g, a.group - 1));
                if (g >= a.group || !e.fine) continue;
                const bool far = is_far(e.minus);
                const f32x4 x = far ? s[u][g] * a.scale : s[u][g];
                const float by = far ? 1.0f : a.scale;
#pragma unroll
                for (int i = 0; i < 4; i++) sum[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(x[i], by, e.minus)), e.by, sum[i]);
            }
            const int place = from + u * STEP;
#pragma unroll
            for (int i = 0; i < 4; i++) w[u][i] = place + i < sees ? w[u][i] + sum[i] : w[u][i];
            *reinterpret_cast<f32x4 *>(a.c.weights + (page[u] * a.c.heads + h) * kPage + place % kPage) = w[u];
        }
    }
}
