// Weights of tokens from the scores that attention over single tokens left.
#include "weigh.h"

namespace {

// Four places of a sequence and head a thread, 1,024 a workgroup; the scores of the queries that share the head, read once.
__global__ __launch_bounds__(256) void weigh_scores_kernel(AttendArgs a, int64_t units, int pieces) {
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int piece = (int)(u % pieces), h = (int)(u / pieces % a.c.heads), b = (int)(u / pieces / a.c.heads);
        const int sees = length_of(a.t, b), place = piece * 1024 + threadIdx.x * 4;  // one row, the last
        if (place >= sees) continue;
        const int64_t page = page_of(a.t, a.c, b, place / kPage);
        if (page < 0) continue;
        const int64_t row = (int64_t)b * a.heads_q + h * a.group, wide = (int64_t)a.t.blocks * kPage;
        f32x4 sum = {0, 0, 0, 0};
        for (int g = 0; g < a.group; g++) {
            const RowEnds ends = row_ends(a.ends, row + g);
            if (!ends.fine) continue;
            const f32x4 s = *reinterpret_cast<const f32x4 *>(a.scores + (row + g) * wide + place);
#pragma unroll
            for (int i = 0; i < 4; i++) sum[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale, ends.minus)), ends.by, sum[i]);
        }
        float *const to = a.c.weights + (page * a.c.heads + h) * kPage + place % kPage;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (place + i < sees) to[i] += sum[i];
    }
}

}  // namespace

int launch_weigh_scores(const AttendArgs &a, hipStream_t stream) {
    const int pieces = (a.t.blocks * kPage + 1023) / 1024;
    const int64_t units = (int64_t)a.t.rows * a.c.heads * pieces;
    if (units == 0) return VL_OK;
    weigh_scores_kernel<<<vl_grid_for(units, 1), 256, 0, stream>>>(a, units, pieces);
    VL_LAUNCH_CHECK("weigh_scores_kernel");
    return VL_OK;
}
