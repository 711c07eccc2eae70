// The choice of blocks: scores of all blocks of a row from their bounds, then the best of them.
#include "select.h"

namespace {

constexpr uint32_t kOwn = 0xFFFFFFFFu;        // the row's own block
constexpr uint32_t kUnbounded = 0xFFFFFFFEu;  // a block without bounds; every other score is finite and lower
constexpr int kChunk = 256;                   // blocks a workgroup scores

// Tokens of a sequence that share a tile of 16 queries
__device__ __host__ inline int tokens_a_tile(int group) { return group >= 16 ? 1 : 16 / group; }

// Scores of up to 256 blocks for one tile of 16 (token, query of the head) pairs.
//
// score = max over the queries of sum_j max(u_j, 0) hi_j + min(u_j, 0) lo_j: one sum over 2 D channels of 8-bit products, which
// the matrix cores make of 16 blocks x 16 queries at once; it is a whole number below 2^22, exact in float32, and so is its
// product with the block's power of two.  What bounds it is the bounds' bytes, 2 D a block.
template <int D, int NS>
__global__ __launch_bounds__(256) void score_kernel(SelectArgs a, int chunks) {
    typedef typename ElementOf<NS>::type E;
    constexpr int kSteps = 2 * D / 64;
    __shared__ float s_top[4][16];
    __shared__ int s_score[4][16][17];
    const int h = blockIdx.y, chunk = blockIdx.x % chunks, tile = blockIdx.x / chunks;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15, wave = threadIdx.x >> 6;
    const int T = tokens_a_tile(a.group);
    Piece w = {tile, 0};
    if (a.t.offsets) w = find_piece(a.t.sequences, tile, [&](int b) { return (row_count(a.t, b) + T - 1) / T; });
    if (w.sequence < 0) return;
    const int b = w.sequence, all = row_count(a.t, b), length = length_of(a.t, b);
    const int64_t row0 = first_row(a.t, b);
    const int place0 = (int)min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all;  // of the sequence's first row
    const int token0 = w.piece * T, tokens = min(T, all - token0);
    const int last = min(place0 + token0 + tokens, length) - 1;                    // the last place of the tile
    if (last < 0 || chunk * kChunk > last / kPage) return;
    const int ways = (a.group + 15) / 16;  // tiles of 16 queries; more than one only where a token fills them

    // the largest magnitude of a token's queries
    float top = 0;
    bool finite = true;
    auto query = [&](int way, int step, float(&x)[16]) {
        const int token = a.group >= 16 ? 0 : r / a.group, g = a.group >= 16 ? way * 16 + r : r % a.group;
        const bool real = token < tokens && g < a.group;
        const int d = (step * 64 + q * 16) % D;  // D is a multiple of 32: 16 channels are all of the upper or all of the lower bounds
        float y[8];
#pragma unroll
        for (int half = 0; half < 2; half++) {
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = 0;
            if (real) load8<NS>((const E *)a.queries + (row0 + token0 + token) * a.q_row + (h * a.group + g) * a.q_head + d + half * 8, a.aligned, y);
#pragma unroll
            for (int i = 0; i < 8; i++) x[half * 8 + i] = y[i];
        }
    };
    for (int way = 0; way < ways; way++) {
#pragma unroll
        for (int step = 0; step < (D + 63) / 64; step++) {
            float x[16];
            query(way, step, x);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                finite &= (__builtin_bit_cast(uint32_t, x[i]) & 0x7F800000u) != 0x7F800000u;
                top = fmaxf(top, fabsf(x[i]));
            }
        }
    }
    if (!finite) top = INFINITY;
    top = max_over_quads(top);
    if (q == 0) s_top[wave][r] = top;
    __syncthreads();
    {
        const int first = a.group >= 16 ? 0 : r / a.group * a.group, n = a.group >= 16 ? 16 : a.group;
        for (int i = first; i < min(first + n, 16); i++) top = fmaxf(top, s_top[wave][i]);
    }
    // its exponent becomes 6; queries that are not finite, or so small that this leaves the range, count as zeros
    const int e = max((int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127 - 6, -100);
    const float unit = top < INFINITY ? __builtin_bit_cast(float, (uint32_t)(127 - e) << 23) : 0.0f;

    const int end = min(min((chunk + 1) * kChunk, a.t.blocks), last / kPage + 1);
    for (int first = chunk * kChunk + wave * 16; first < chunk * kChunk + kChunk; first += 64) {
        const bool some = first < end;  // the same for the wavefront
        i32x4 best = {INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN};
        int64_t page = some && first + r < end ? page_of(a.t, a.c, b, first + r) : -1;
        if (some) {
            const int8_t *const at = a.c.bounds + (max(page, (int64_t)0) * a.c.heads + h) * (2 * D) + q * 16;
            i32x4 edges[kSteps];
#pragma unroll
            for (int step = 0; step < kSteps; step++) {
                edges[step] = i32x4{0, 0, 0, 0};
                if (page >= 0) edges[step] = *reinterpret_cast<const i32x4 *>(at + step * 64);
            }
            for (int way = 0; way < ways; way++) {
                i32x4 sum = {0, 0, 0, 0};
#pragma unroll
                for (int step = 0; step < kSteps; step++) {
                    float x[16];
                    query(way, step, x);
                    const bool upper = step * 64 + q * 16 < D;
                    i32x4 u = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        int v = 0;
                        if (unit != 0.0f) v = (int)fminf(fmaxf(rintf(x[i] * unit), -127.0f), 127.0f);
                        v = upper ? max(v, 0) : min(v, 0);
                        u[i >> 2] |= (v & 255) << (8 * (i & 3));
                    }
                    sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(edges[step], u, sum, 0, 0, 0);
                }
                if (a.group >= 16 && way * 16 + r >= a.group) continue;  // no such query: its zeros are no score
#pragma unroll
                for (int i = 0; i < 4; i++) best[i] = max(best[i], sum[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s_score[wave][q * 4 + i][r] = best[i];
        __syncthreads();
        if (some) {
            const int spans = a.group >= 16 ? 16 : a.group;
            for (int i = lane; i < tokens * 16; i += 64) {
                const int token = i >> 4, block = first + (i & 15);
                int score = INT32_MIN;
                for (int g = 0; g < spans; g++) score = max(score, s_score[wave][i & 15][token * spans + g]);
                const int own = min(place0 + token0 + token, length - 1) / kPage;  // a place below 0 has no own block, see select
                if (block >= end || block > own) continue;
                const int64_t p = page_of(a.t, a.c, b, block);
                uint32_t key = 0;
                if (p >= 0) {
                    const int s = a.c.bound_scales[p * a.c.heads + h];
                    key = s == kBoundless ? kUnbounded : vl_float_key((float)score * __builtin_bit_cast(float, (uint32_t)(s + 127) << 23));
                }
                if (block == own) key = kOwn;
                a.keys[((row0 + token0 + token) * a.c.heads + h) * a.t.blocks + block] = key;
            }
        }
        __syncthreads();
    }
}

// A workgroup chooses for one row and head: the `count` largest keys by counting their bytes from the top, ties to the lower
// block, written in the order of the blocks.
__global__ __launch_bounds__(256) void select_kernel(SelectArgs a) {
    __shared__ int s_count[256];
    __shared__ int s_wave[4][2];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int64_t row = blockIdx.x;
    const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t *const out = a.out + (row * a.c.heads + h) * a.count;
    const int b = sequence_of(a.t, (int)row);
    const int all = row_count(a.t, b), length = length_of(a.t, b);
    const int64_t place = min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all + row - first_row(a.t, b);
    const int n = place < 0 || length == 0 ? 0 : (int)min(place, (int64_t)length - 1) / kPage + 1;
    const uint32_t *const keys = a.keys + (row * a.c.heads + h) * a.t.blocks;
    uint32_t least = 1;  // keys below are not candidates
    int ties = 0;        // of those equal to it this many are taken
    if (n > a.count) {
        if (threadIdx.x == 0) {
            s_prefix = 0;
            s_need = a.count;
        }
        for (int shift = 24; shift >= 0; shift -= 8) {
            s_count[threadIdx.x] = 0;
            __syncthreads();
            const uint32_t prefix = s_prefix;
            const int need = s_need;
            for (int i = threadIdx.x; i < n; i += 256) {
                const uint32_t key = keys[i];
                if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&s_count[key >> shift & 255], 1);
            }
            __syncthreads();
            if (wave == 0) {
                // lane l has the bytes 255 - 4 l and the three below it; keys above them, from the top
                int c[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    c[i] = s_count[255 - 4 * lane - i];
                    sum += c[i];
                }
                int upto = sum;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int other = __shfl_up(upto, d);
                    if (lane >= d) upto += other;
                }
                int above = upto - sum;
                if (above < need && upto >= need) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (above < need && above + c[i] >= need) {
                            s_prefix = prefix << 8 | (uint32_t)(255 - 4 * lane - i);
                            s_need = need - above;
                            above = need;  // found
                        } else {
                            above += c[i];
                        }
                    }
                }
            }
            __syncthreads();
        }
        least = s_prefix;
        ties = s_need;
    }
    if (n <= a.count || least == 0) {  // all candidates fit
        least = 0;
        ties = 0;
    }
    int more = 0, equal = 0;  // larger and equal ones so far
    for (int i0 = 0; i0 < n; i0 += 256) {
        const int i = i0 + threadIdx.x;
        const uint32_t key = i < n ? keys[i] : 0;
        const bool gt = key > least, eq = key == least && i < n;
        const uint64_t gts = __ballot(gt), eqs = __ballot(eq), before = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) {
            s_wave[wave][0] = __popcll(gts);
            s_wave[wave][1] = __popcll(eqs);
        }
        __syncthreads();
        int m = more + __popcll(gts & before), e = equal + __popcll(eqs & before);
        for (int k = 0; k < 4; k++) {
            if (k < wave) {
                m += s_wave[k][0];
                e += s_wave[k][1];
            }
            more += s_wave[k][0];
            equal += s_wave[k][1];
        }
        if (gt || (eq && e < ties)) out[m + min(e, ties)] = i;
    }
    for (int i = more + min(equal, ties) + threadIdx.x; i < a.count; i += 256) out[i] = VL_MAXINT;
}

template <int NS>
void launch_score(const SelectArgs &a, int64_t tiles, int chunks, hipStream_t stream) {
    for_dim(a.c.dim, [&](auto d) {
        score_kernel<decltype(d)::value, NS><<<dim3((unsigned)(tiles * chunks), (unsigned)a.c.heads), 256, 0, stream>>>(a, chunks);
    });
}

}  // namespace

int64_t select_workspace_bytes(const SelectArgs &a) {
    return ((int64_t)a.t.rows * a.c.heads * a.t.blocks * 4 + 255) / 256 * 256;
}

int launch_select(const SelectArgs &a, int type, hipStream_t stream) {
    const int chunks = (a.t.blocks + kChunk - 1) / kChunk;
    const int T = tokens_a_tile(a.group);
    const int64_t tiles = a.t.offsets ? a.t.rows / T + (int64_t)a.t.sequences : a.t.rows;
    VL_REQUIRE(tiles * chunks <= 4 * kMaxBlocks && a.t.rows <= 4 * kMaxBlocks, "more rows than one call takes: %d of %d blocks",
               a.t.rows, a.t.blocks);
    if (chunks) {
        if (type == VL_BF16) launch_score<1>(a, tiles, chunks, stream);
        else if (type == VL_F16) launch_score<2>(a, tiles, chunks, stream);
        else launch_score<3>(a, tiles, chunks, stream);
        VL_LAUNCH_CHECK("score_kernel");
    }
    select_kernel<<<dim3((unsigned)a.t.rows, (unsigned)a.c.heads), 256, 0, stream>>>(a);
    VL_LAUNCH_CHECK("select_kernel");
    return VL_OK;
}
