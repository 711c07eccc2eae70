// The weights of weigh_scores.h from the keys once more.
//
// A page and head is one workgroup's (two pages of one sequence are two), so sums have one order and nothing is atomic.
#pragma once
#include "attend_few.h"

// Many rows, or several tokens of a sequence: the scores of a page are made once more.  A workgroup has one page of one head; its
// wavefronts hold the page's keys in registers as bfloat16 (32 tokens a tile, two tiles) and take every fourth tile of 32 rows.
// S^T = K Q^T as in attend_many_kernel; a lane's 32 sums are those of its column of rows, added over lanes and wavefronts at the end.
template <int D, int NS>
__global__ __launch_bounds__(256) void weigh_rows_kernel(AttendArgs a, int64_t units) {
    typedef typename ElementOf<NS>::type E;
    __shared__ float s_sum[4][kPage];
    const int lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int h = (int)(u % a.c.heads);
        const int64_t rest = u / a.c.heads;
        const int block = (int)(rest % a.t.blocks), b = (int)(rest / a.t.blocks);
        const int length = length_of(a.t, b), all = row_count(a.t, b), first = block * kPage;
        if (first >= length || all == 0) continue;
        const int64_t page = page_of(a.t, a.c, b, block);
        if (page < 0) continue;
        const int64_t unit = page * a.c.heads + h;
        const uint32_t scales = a.c.scales[unit];
        const bool marked = is_marked(scales);
        const int row0 = first_row(a.t, b), place0 = (int)min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all;
        bf16x8 k[2][D / 16];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            u32x4 x[D / 32];
            const uint8_t *const at = a.c.keys + unit * (kPage * D) + (t * 32 + col) * D + hi * 16;
#pragma unroll
            for (int c = 0; c < D / 32; c++) x[c] = *reinterpret_cast<const u32x4 *>(at + c * 32);
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                k[t][2 * c] = eight_of_bytes(x[c][0], x[c][1], scale_of_keys(scales));
                k[t][2 * c + 1] = eight_of_bytes(x[c][2], x[c][3], scale_of_keys(scales));
            }
        }
        float sum[2][16];
#pragma unroll
        for (int i = 0; i < 32; i++) sum[i >> 4][i & 15] = 0;
        const int64_t rows = (int64_t)all * a.group;
        // the first row that sees the page
        const int64_t from = a.causal ? (int64_t)max(first - place0, 0) * a.group / 32 : 0;
        for (int64_t tile = from + wave; tile * 32 < rows; tile += 4) {
            const int64_t index = tile * 32 + col;
            const int token = (int)(index / a.group), head = h * a.group + (int)(index % a.group);
            const bool real = index < rows;
            const int64_t row = row0 + (int64_t)token;
            f32x2 top_and_total = *reinterpret_cast<const f32x2 *>(a.ends + (real ? row * a.heads_q + head : 0) * 2);
            const RowEnds ends = row_ends(top_and_total[0], top_and_total[1]);
            const int sees = !real || !ends.fine ? 0 : a.causal ? min(max(place0 + token + 1, 0), length) : length;
            const E *const at = (const E *)a.queries + (real ? row * a.q_row + head * a.q_head : 0) + hi * 16;
            f32x16 s[2], small[2];
#pragma unroll
            for (int i = 0; i < 16; i++) s[0][i] = s[1][i] = small[0][i] = small[1][i] = 0;
            Eight<NS> x[D / 16];
#pragma unroll
            for (int c = 0; c < D / 16; c++) x[c] = load8<NS>(at + (c >> 1) * 32 + (c & 1) * 8);
#pragma unroll
            for (int c = 0; c < D / 16; c++) {
                bf16x8 q[NS];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    __bf16 p[NS];
                    split_into<NS>((float)x[c][i] * a.turn, p);
#pragma unroll
                    for (int n = 0; n < NS; n++) q[n][i] = p[n];
                }
#pragma unroll
                for (int n = 0; n < NS; n++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        f32x16 &to = NS == 3 && n > 0 ? small[t] : s[t];
                        to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[t][c], q[n], to, 0, 0, 0);
                    }
            }
            if (marked || __ballot(sees < first + kPage)) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int place = first + t * 32 + 8 * (i >> 2) + 4 * hi + (i & 3);
                        const float score = NS == 3 ? s[t][i] + small[t][i] : s[t][i];
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(score, a.scale, ends.minus)) * ends.by;
                        sum[t][i] += place < sees ? p : 0.0f;
                    }
            } else {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float score = NS == 3 ? s[t][i] + small[t][i] : s[t][i];
                        sum[t][i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(score, a.scale, ends.minus)), ends.by, sum[t][i]);
                    }
            }
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) sum[t][i] += __shfl_xor(sum[t][i], d);
                if (col == 0) s_sum[wave][t * 32 + 8 * (i >> 2) + 4 * hi + (i & 3)] = sum[t][i];
            }
        __syncthreads();
        if (threadIdx.x < kPage && first + (int)threadIdx.x < length)
            a.c.weights[unit * kPage + threadIdx.x] += (s_sum[0][threadIdx.x] + s_sum[1][threadIdx.x]) + (s_sum[2][threadIdx.x] + s_sum[3][threadIdx.x]);
        __syncthreads();
    }
}

template <int NS>
int launch_weigh_rows(const AttendArgs &a, hipStream_t stream) {
    const int64_t units = (int64_t)a.t.sequences * a.t.blocks * a.c.heads;
    if (units == 0) return VL_OK;
    VL_REQUIRE((double)a.t.sequences * a.t.blocks * a.c.heads < 9e18, "more pages than one call takes: %d sequences of %d blocks", a.t.sequences, a.t.blocks);
    for_dim(a.c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        weigh_rows_kernel<D, NS><<<vl_grid_for(units, 1), 256, 0, stream>>>(a, units);
    });
    VL_LAUNCH_CHECK("weigh_rows_kernel");
    return VL_OK;
}
