// Weights of tokens from the scores that attention over single tokens left.
#include "weigh_scores.h"

namespace {

// 2,048 places of a sequence and head a workgroup: one round of 256 threads with 8 queries a head, two with more; of 4 or fewer half of a
// round's loads lie behind the piece's end
template <int G>
__global__ __launch_bounds__(256) void weigh_scores_kernel(AttendArgs a, int64_t units, int pieces) {
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int piece = (int)(u % pieces), h = (int)(u / pieces % a.c.heads), b = (int)(u / pieces / a.c.heads);
        const int sees = length_of(a.t, b);  // one row, the last
        const float *const at = a.ends + ((int64_t)b * a.heads_q + h * a.group) * 2;
        weigh_places<G, 1024>(a, b, h, piece * 2048 + threadIdx.x * 4, min(sees, (piece + 1) * 2048), [&](int g) { return row_ends(at[2 * g], at[2 * g + 1]); });
    }
}

}  // namespace

int launch_weigh_scores(const AttendArgs &a, hipStream_t stream) {
    const int pieces = (a.t.blocks * kPage + 2047) / 2048;
    const int64_t units = (int64_t)a.t.rows * a.c.heads * pieces;
    if (units == 0) return VL_OK;
    auto launch = [&](auto g) { weigh_scores_kernel<decltype(g)::value><<<vl_grid_for(units, 1), 256, 0, stream>>>(a, units, pieces); };
    if (a.group <= 4) launch(std::integral_constant<int, 4>());
    else if (a.group <= 8) launch(std::integral_constant<int, 8>());
    else launch(std::integral_constant<int, 16>());
    VL_LAUNCH_CHECK("weigh_scores_kernel");
    return VL_OK;
}
