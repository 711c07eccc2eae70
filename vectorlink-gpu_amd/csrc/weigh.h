// The weights of weigh_scores.h from the keys once more.
//
// A page and head is one workgroup's (weigh_rows_kernel) or one wavefront's (weigh_pages_kernel), which takes all rows, so sums have one
// order and nothing is atomic.
#pragma once
#include "attend_few.h"

// Many rows, or several tokens of a sequence: the scores of a page are made once more.  A wavefront holds a page's keys in registers (two
// tiles of 32 tokens) and takes tiles of 32 rows; S^T = K Q^T as in attend_many_kernel.  A lane's 32 sums are those of its column of rows,
// added over the lanes at the end.  What bounds it are the exponentials, a quarter of the vector units' rate, and half of attention's
// matrix products.
//
// Queries of half precision meet the codes as half precision, which is one product where bfloat16 parts of them would be two; those of
// float32 are split into three parts.
template <int NS>
using Operand = typename std::conditional<NS == 2, f16x8, bf16x8>::type;
constexpr int query_parts(int NS) { return NS == 3 ? 3 : 1; }

template <int D, int NS>
struct PageKeys {
    Operand<NS> k[2][D / 16];
    float ahead, scale;  // of the scores: see scale_with
    bool apart;          // a token may not be finite, or ahead is not 1
};
template <int D, int NS>
__device__ inline void load_keys(PageKeys<D, NS> &g, const AttendArgs &a, int64_t unit) {
    const int col = threadIdx.x & 31, hi = threadIdx.x >> 5 & 1;
    const uint32_t scales = a.c.scales[unit];
    g.ahead = NS == 2 ? power_ahead(a.scale, scale_of_keys(scales)) : 1.0f;
    g.apart = is_marked(scales) || g.ahead != 1.0f;
    g.scale = (NS == 2 ? scale_with(a.scale, scale_of_keys(scales)) : a.scale) * (NS == 3 ? 1.0f : a.turn);
    // Without a scale all scores are 0, and 0 times a product beyond float32 would be none: the keys are 0 then.  (Queries of float32 are.)
    const uint32_t there = NS < 3 && a.turn == 0 ? 0 : ~0u;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        u32x4 x[D / 32];
        const uint8_t *const at = a.c.keys + unit * (kPage * D) + (t * 32 + col) * D + hi * 16;
#pragma unroll
        for (int c = 0; c < D / 32; c++) x[c] = *reinterpret_cast<const u32x4 *>(at + c * 32) & there;
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            if constexpr (NS == 2) {
                g.k[t][2 * c] = eight_halves(x[c][0], x[c][1]);
                g.k[t][2 * c + 1] = eight_halves(x[c][2], x[c][3]);
            } else {
                g.k[t][2 * c] = eight_of_bytes(x[c][0], x[c][1], scale_of_keys(scales));
                g.k[t][2 * c + 1] = eight_of_bytes(x[c][2], x[c][3], scale_of_keys(scales));
            }
        }
    }
}
// Where chunk c of 16 dimensions of a row is, in elements: as load_keys brings the keys, 16 bytes for two of them.
__device__ inline int chunk_at(int c) { return (c >> 1) * 32 + (threadIdx.x >> 5 & 1) * 16 + (c & 1) * 8; }

// A tile of 32 rows, of which this lane's sees the first `mine` of the page's places that are its own: query(c, n) is part n of chunk c.
template <int D, int NS, class F>
__device__ inline void weigh_tile(float (&sum)[32], const PageKeys<D, NS> &g, float minus, float by, int sees, F query) {
    f32x16 s[2], small[2];  // products with the second and third part of a query have sums of their own: a score is rounded less often
#pragma unroll
    for (int i = 0; i < 16; i++) s[0][i] = s[1][i] = small[0][i] = small[1][i] = 0;
#pragma unroll
    for (int c = 0; c < D / 16; c++) {
        Operand<NS> q[query_parts(NS)];
        query(c, q);
#pragma unroll
        for (int n = 0; n < query_parts(NS); n++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                f32x16 &to = n > 0 ? small[t] : s[t];
                if constexpr (NS == 2) to = __builtin_amdgcn_mfma_f32_32x32x16_f16(g.k[t][c], q[n], to, 0, 0, 0);
                else to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(g.k[t][c], q[n], to, 0, 0, 0);
            }
    }
    auto score = [&](int i) { return NS == 3 ? s[i >> 4][i & 15] + small[i >> 4][i & 15] : s[i >> 4][i & 15]; };
    auto weight = [&](float x, float scale) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, minus)); };
    // These scores are sums in another order than attention's: beyond 2^16 the largest may be far above what the row ends with, and no
    // weight is more than 1.
    if (g.apart || __ballot(sees < kPage || __builtin_fabsf(minus) > 0x1p16f)) {
        const int mine = sees - 4 * (threadIdx.x >> 5 & 1);
        const bool far = is_far(minus);
        const float then = far ? g.scale : 1.0f, scale = far ? 1.0f : g.scale;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            if (i % 8 == 0) __builtin_amdgcn_sched_barrier(0);
            const float p = fminf(fmaxf(weight((NS == 2 ? score(i) * g.ahead : score(i)) * then, scale) * by, 0.0f), 1.0f);
            sum[i] += (i >> 4) * 32 + 8 * (i >> 2 & 3) + (i & 3) < mine ? p : 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) {
            if (i % 8 == 0) __builtin_amdgcn_sched_barrier(0);  // a few exponentials at a time: all 32 at once take the registers
            sum[i] = __builtin_fmaf(weight(score(i), g.scale), by, sum[i]);
        }
    }
}
// The sums over the columns: of what is left of its sums a lane passes on half and keeps the other, until it has one, that of place
// place_of_lane() of the page.
__device__ inline float sum_of_columns(float (&sum)[32]) {
    auto halve = [&](auto half) {
        constexpr int d = decltype(half)::value;
        const bool upper = threadIdx.x & d;
#pragma unroll
        for (int i = 0; i < d; i++) {
            const float pass = upper ? sum[i] : sum[i + d];
            sum[i] = (upper ? sum[i + d] : sum[i]) + __shfl_xor(pass, d);
        }
    };
    halve(std::integral_constant<int, 16>());
    halve(std::integral_constant<int, 8>());
    halve(std::integral_constant<int, 4>());
    halve(std::integral_constant<int, 2>());
    halve(std::integral_constant<int, 1>());
    return sum[0];
}
__device__ inline int place_of_lane() {
    const int col = threadIdx.x & 31;
    return (col >> 4) * 32 + 8 * (col >> 2 & 3) + 4 * (threadIdx.x >> 5 & 1) + (col & 3);
}

// The rows of a sequence and head that come one after the other, from `first` on: which token and query they are, and how far they see.
struct RowWalk {
    int64_t rows, token;  // of the sequence; of the row that `at` counts from
    int64_t place0;
    int row0, index, length;
    __device__ inline RowWalk(const AttendArgs &a, int b, int64_t first) {
        const int all = row_count(a.t, b);
        rows = (int64_t)all * a.group;
        row0 = first_row(a.t, b);
        length = length_of(a.t, b);
        place0 = min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all;
        token = first / a.group;
        index = (int)(first % a.group);
    }
    // behind the last row: the sequence's first, which sees nothing; first: the row that `at` counts from
    __device__ inline int look(const AttendArgs &a, int64_t first, int at, int h, int64_t &row, int &head) const {
        const bool real = first + at < rows;
        const int64_t mine = real ? token + (index + at) / a.group : 0;
        row = row0 + mine;
        head = h * a.group + (real ? (index + at) % a.group : 0);
        return !real ? 0 : a.causal ? (int)min(max(place0 + mine + 1, (int64_t)0), (int64_t)length) : length;
    }
    __device__ inline void step(const AttendArgs &a, int n) {
        token += n / a.group;
        index += n % a.group;
        if (index >= a.group) {
            index -= a.group;
            token++;
        }
    }
};

// Few pages: a workgroup has one, and its wavefronts take every fourth tile of rows, the next one's queries on their way.  With two tiles'
// queries beside the page 128 dimensions of bfloat16 and half precision spill 9 and 12 of 256 vector registers; 512 rows over 4,096 tokens, 32
// heads on 4 of 128, take 34 us for their weights beside 54 and 67 for the attention, float32 (one tile's queries, no spills) 69 beside 94.
template <int D, int NS>
__global__ __launch_bounds__(256, D <= 128 && NS < 3 ? 2 : 1) void weigh_rows_kernel(AttendArgs a, int64_t units) {
    typedef typename ElementOf<NS>::type E;
    constexpr bool kAhead = NS < 3;  // float32 queries fill the registers once
    __shared__ float s_sum[4][kPage];
    const int col = threadIdx.x & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int h = (int)(u % a.c.heads);
        const int64_t rest = u / a.c.heads;
        const int block = (int)(rest % a.t.blocks), b = (int)(rest / a.t.blocks), first = block * kPage;
        const int length = length_of(a.t, b), all = row_count(a.t, b);
        if (first >= length || all == 0) continue;
        const int64_t page = page_of(a.t, a.c, b, block);
        if (page < 0) continue;
        const int64_t unit = page * a.c.heads + h;
        // from the first row on that sees the page
        const int64_t place0 = min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all, tiles = ((int64_t)all * a.group + 31) / 32;
        const int64_t from = (a.causal ? max(first - place0, (int64_t)0) * a.group / 32 : 0) + wave;
        RowWalk walk(a, b, from * 32);
        struct Tile {
            Eight<NS> x[D / 16];
            f32x2 ends;
            int sees;
        };
        auto load = [&](Tile &t, int64_t tile) {
            int64_t row;
            int head;
            t.sees = walk.look(a, tile * 32, col, h, row, head);
            t.ends = *reinterpret_cast<const f32x2 *>(a.ends + (row * a.heads_q + head) * 2);
            const E *const q = (const E *)a.queries + row * a.q_row + head * a.q_head;
#pragma unroll
            for (int c = 0; c < D / 16; c++) t.x[c] = load8<NS>(q + chunk_at(c));
            walk.step(a, 128);
        };
        Tile x;
        if (from < tiles) load(x, from);
        PageKeys<D, NS> g;
        load_keys<D, NS>(g, a, unit);
        float sum[32];
#pragma unroll
        for (int i = 0; i < 32; i++) sum[i] = 0;
        auto take = [&](const Tile &tile) {
            const RowEnds ends = row_ends(tile.ends[0], tile.ends[1]);
            weigh_tile<D, NS>(sum, g, ends.minus, ends.by, (ends.fine ? tile.sees : 0) - first, [&](int c, Operand<NS>(&q)[query_parts(NS)]) {
                if constexpr (NS == 3) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        __bf16 p[NS];
                        split_into<NS>((float)tile.x[c][i] * a.turn, p);
#pragma unroll
                        for (int n = 0; n < NS; n++) q[n][i] = p[n];
                    }
                } else {
                    q[0] = __builtin_bit_cast(Operand<NS>, tile.x[c]);
                }
            });
        };
        if (from < tiles) {
            if constexpr (kAhead) {
                Tile y;
                for (int64_t tile = from;; tile += 8) {
                    load(y, tile + 4);
                    take(x);
                    if (tile + 4 >= tiles) break;
                    load(x, tile + 8);
                    take(y);
                    if (tile + 8 >= tiles) break;
                }
            } else {
                for (int64_t tile = from;;) {
                    take(x);
                    tile += 4;
                    if (tile >= tiles) break;
                    load(x, tile);
                }
            }
        }
        s_sum[wave][place_of_lane()] = sum_of_columns(sum);
        __syncthreads();
        if (threadIdx.x < kPage && first + (int)threadIdx.x < length)
            a.c.weights[unit * kPage + threadIdx.x] += (s_sum[0][threadIdx.x] + s_sum[1][threadIdx.x]) + (s_sum[2][threadIdx.x] + s_sum[3][threadIdx.x]);
        __syncthreads();
    }
}

// Many pages: each of a workgroup's wavefronts has one, four neighbours of a head, and all of them take the same rows, which go through
// LDS, brought there row after row while the last are worked on.  As the products want them, 32 rows at a time, they are lines that the
// caches do not give in that time (2,048 rows over 16,384 tokens, 32 heads on 8 of 128: 476 us from the caches, 384 from LDS).
template <int D, int NS>
struct QueryTiles {
    static constexpr int kTiles = D * query_parts(NS) <= 256 ? 2 : 1, kRows = 32 * kTiles;  // of a step
    static constexpr int kRow = D * 2 + 16;  // bytes: 16 lanes' rows lie in different banks
    static constexpr int kPart = kRows * kRow, kBytes = query_parts(NS) * kPart + kRows * 16;  // and what the rows end with
    static constexpr int kUnits = (kRows * D / 8 + 255) / 256;                                  // of 8 elements, of a thread
};
template <int D, int NS>
__global__ __launch_bounds__(256, D <= 128 && NS < 3 ? 2 : 1) void weigh_pages_kernel(AttendArgs a, int64_t units) {
    typedef QueryTiles<D, NS> Q;
    typedef typename ElementOf<NS>::type E;
    extern __shared__ __attribute__((aligned(16))) char lds[];  // two of Q::kBytes
    const int col = threadIdx.x & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int groups = (a.t.blocks + 3) / 4;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int h = (int)(u % a.c.heads);
        const int64_t rest = u / a.c.heads;
        const int block0 = (int)(rest % groups) * 4, block = block0 + wave, b = (int)(rest / groups), first = block * kPage;
        const int length = length_of(a.t, b), all = row_count(a.t, b);
        if (block0 * kPage >= length || all == 0) continue;
        // a wavefront without a page takes part with the cache's first, and adds its sums to nothing
        const int64_t page = first < length ? page_of(a.t, a.c, b, block) : -1, unit = max(page, (int64_t)0) * a.c.heads + h;
        const int64_t rows = (int64_t)all * a.group, steps = (rows + Q::kRows - 1) / Q::kRows;
        // from the first row on that sees the first page
        const int64_t place0 = min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all;
        const int64_t from = a.causal ? min(max(block0 * kPage - place0, (int64_t)0) * a.group / Q::kRows, steps) : 0;
        RowWalk walk(a, b, from * Q::kRows);
        Eight<NS> x[Q::kUnits];
        f32x2 ends = {0, 0};
        int sees = 0;
        auto fetch = [&](int64_t step) {
            int64_t row;
            int head;
#pragma unroll
            for (int k = 0; k < Q::kUnits; k++) {
                const int i = k * 256 + threadIdx.x;
                walk.look(a, step * Q::kRows, min(i / (D / 8), Q::kRows - 1), h, row, head);
                x[k] = load8<NS>((const E *)a.queries + row * a.q_row + head * a.q_head + i % (D / 8) * 8);
            }
            if (threadIdx.x < Q::kRows) {
                sees = walk.look(a, step * Q::kRows, threadIdx.x, h, row, head);
                ends = *reinterpret_cast<const f32x2 *>(a.ends + (row * a.heads_q + head) * 2);
            }
            walk.step(a, Q::kRows);
        };
        auto store = [&](char *to) {
#pragma unroll
            for (int k = 0; k < Q::kUnits; k++) {
                const int i = k * 256 + threadIdx.x;
                if (i >= Q::kRows * D / 8) continue;
                char *const at = to + i / (D / 8) * Q::kRow + i % (D / 8) * 16;
                if constexpr (NS == 3) {
                    bf16x8 part[3];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        __bf16 p[3];
                        split_into<3>((float)x[k][e] * a.turn, p);
#pragma unroll
                        for (int n = 0; n < 3; n++) part[n][e] = p[n];
                    }
#pragma unroll
                    for (int n = 0; n < 3; n++) *reinterpret_cast<bf16x8 *>(at + n * Q::kPart) = part[n];
                } else {
                    *reinterpret_cast<Eight<NS> *>(at) = x[k];
                }
            }
            if (threadIdx.x < Q::kRows) {
                const RowEnds e = row_ends(ends[0], ends[1]);
                *reinterpret_cast<f32x4 *>(to + query_parts(NS) * Q::kPart + threadIdx.x * 16) =
                    f32x4{e.minus, e.by, __builtin_bit_cast(float, e.fine ? sees : 0), 0};
            }
        };
        if (from < steps) fetch(from);
        PageKeys<D, NS> g;
        load_keys<D, NS>(g, a, unit);
        float sum[32];
#pragma unroll
        for (int i = 0; i < 32; i++) sum[i] = 0;
        if (from < steps) store(lds);
        __syncthreads();
        for (int64_t step = from, turn = 0; step < steps; step++, turn ^= 1) {
            const bool more = step + 1 < steps;
            if (more) fetch(step + 1);
#pragma unroll 1
            for (int t = 0; t < Q::kTiles; t++) {
                const char *const in = lds + turn * Q::kBytes, *const my = in + (t * 32 + col) * Q::kRow;
                const f32x4 end = *reinterpret_cast<const f32x4 *>(in + query_parts(NS) * Q::kPart + (t * 32 + col) * 16);
                const float bits = end[2];
                weigh_tile<D, NS>(sum, g, end[0], end[1], __builtin_bit_cast(int, bits) - first, [&](int c, Operand<NS>(&q)[query_parts(NS)]) {
#pragma unroll
                    for (int n = 0; n < query_parts(NS); n++) q[n] = *reinterpret_cast<const Operand<NS> *>(my + n * Q::kPart + chunk_at(c) * 2);
                });
            }
            if (more) store(lds + (turn ^ 1) * Q::kBytes);
            __syncthreads();
        }
        const float all_rows = sum_of_columns(sum);
        if (page >= 0 && first + place_of_lane() < length) a.c.weights[unit * kPage + place_of_lane()] += all_rows;
    }
}

template <int NS>
int launch_weigh_rows(const AttendArgs &a, hipStream_t stream) {
    if (a.c.pages == 0) return VL_OK;
    VL_REQUIRE((double)a.t.sequences * a.t.blocks * a.c.heads < 9e18, "more pages than one call takes: %d sequences of %d blocks", a.t.sequences, a.t.blocks);
    const int64_t units = (int64_t)a.t.sequences * a.t.blocks * a.c.heads, fours = (int64_t)a.t.sequences * ((a.t.blocks + 3) / 4) * a.c.heads;
    if (units == 0) return VL_OK;
    hipError_t e = hipSuccess;
    for_dim(a.c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        // Two pages for every SIMD of the card: 64 rows of 4 sequences of 16,384 tokens 65 us with four pages a workgroup, 170 with one; 1,024 rows of
        // 4 of 1,024 tokens 94 us and 65.
        if (units >= 8 * kComputeUnits) {
            constexpr size_t lds = 2 * QueryTiles<D, NS>::kBytes;
            e = vl_allow_lds(weigh_pages_kernel<D, NS>, lds);
            if (e == hipSuccess) weigh_pages_kernel<D, NS><<<vl_grid_for(fours, 1), 256, lds, stream>>>(a, fours);
        } else {
            weigh_rows_kernel<D, NS><<<vl_grid_for(units, 1), 256, 0, stream>>>(a, units);
        }
    });
    VL_HIP(e);
    VL_LAUNCH_CHECK("launch_weigh_rows");
    return VL_OK;
}
