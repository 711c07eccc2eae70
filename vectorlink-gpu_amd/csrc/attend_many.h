// Attention of many rows over the same tokens: a prompt, or a piece of one, against everything before it.
//
// What bounds it is the two matrix products, 4 D operations a row and token, and beside them the vector units' work on every
// score (maximum, exponential, sum, rounding).  A workgroup has kRows = 32 WAVES rows of one head - tokens and the queries that
// share the head, one after the other - and takes a page of 64 tokens at a time: all wavefronts turn its bytes into bfloat16
// in LDS once, then each reads all of it for 32 rows of its own.  PAGES pages a round, two sets of buffers, one barrier a round:
// the next pages' bytes are on their way while these are worked on, and are turned into the other buffers after them.  Measured:
// 2,048 rows over 16,384 tokens, 32 heads on 8 of 128, 478 us (1,080 TFLOP/s; a large library product of bfloat16 1,216 to 1,248),
// matrix units busy 46 % and vector units 49 % of the time; some cards take 500.
//
// S^T = K Q^T in tiles of 32 tokens x 32 rows: lane l holds row l % 32, and of a tile the tokens 8 (i / 4) + 4 (l / 32) + i % 4.
// out^T = V^T P^T takes P^T as it lies, 16 tokens a step: of half l / 32 the tokens 16 s + 4 (l / 32) + j and those 8 further, so
// values lie in LDS as [dimension][token] in that order, 8 tokens of a half in 16 bytes.  Both images are swizzled by 16 bytes
// so that the rows that 16 lanes read at once lie in different banks.
#pragma once
#include "attend.h"
#include "attend_few.h"

template <int D>
struct Images {
    static constexpr int kRow = D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256;  // elements of a key's row
    static constexpr int kChunks = kRow / 8;                                        // of 16 bytes
    static constexpr int kPerBanks = kRow >= 128 ? 1 : 128 / kRow;                  // rows in 256 bytes
    static constexpr int kKeys = kPage * kRow * 2, kValues = D * kPage * 2, kBytes = kKeys + kValues;
    __device__ static int key(int token, int chunk) {  // byte of a chunk
        return token * (kRow * 2) + (chunk ^ (token / kPerBanks & (kChunks < 16 ? kChunks - 1 : 15))) * 16;
    }
    __device__ static int value(int d, int chunk) { return kKeys + d * (kPage * 2) + (chunk ^ (d >> 1 & 7)) * 16; }
};

// What a thread brings of a page: keys of D / 4 dimensions of a token, values of 8 dimensions of 4 tokens.
template <int D>
struct KeyPart {
    uint32_t w[D / 32];
    uint8_t scale[D / 32];
};
template <int D>
struct ValuePart {
    static constexpr int kUnits = D <= 128 ? 1 : 2;
    u32x4 w[kUnits];
    uint32_t scale[kUnits];
};

template <int D>
__device__ inline void fetch_keys(KeyPart<D> &g, const CacheView &c, int64_t unit, int id) {
    const int token = (id >> 6) * 16 + (id & 15), q = id >> 4 & 3;
    const uint8_t *const at = c.keys + unit * (kPage * D / 2) + token * (D / 2) + q * (D / 8);
    const uint8_t *const ks = c.key_scales + unit * (kPage * D / 32) + token;
    if (D % 128 == 0) {
#pragma unroll
        for (int i = 0; i < D / 128; i++) {
            const u32x4 x = reinterpret_cast<const u32x4 *>(at)[i];
#pragma unroll
            for (int k = 0; k < 4; k++) g.w[4 * i + k] = x[k];
        }
    } else if (D % 64 == 0) {
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            const u32x2 x = reinterpret_cast<const u32x2 *>(at)[i];
            g.w[2 * i] = x[0];
            g.w[2 * i + 1] = x[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < D / 32; i++) g.w[i] = reinterpret_cast<const uint32_t *>(at)[i];
    }
    if (D % 128 == 0) {
#pragma unroll
        for (int i = 0; i < D / 32; i++) g.scale[i] = ks[(q * (D / 128) + i / 4) * kPage];
    } else {
#pragma unroll
        for (int i = 0; i < D / 32; i++) g.scale[i] = ks[(q * (D / 32) + i) / 4 * kPage];
    }
}

template <int D>
__device__ inline void store_keys(const KeyPart<D> &g, char *lds, int id) {
    typedef Images<D> I;
    const int token = (id >> 6) * 16 + (id & 15), q = id >> 4 & 3;
#pragma unroll
    for (int i = 0; i < D / 32; i++)
        *reinterpret_cast<bf16x8 *>(lds + I::key(token, q * (D / 32) + i)) = eight_values(g.w[i], __builtin_bit_cast(float, (uint32_t)g.scale[i] << 23));
}

template <int D>
__device__ inline void fetch_values(ValuePart<D> &g, const CacheView &c, int64_t unit, int id) {
    const int four = id & 15;
    const uint8_t *const vc = c.values + unit * (kPage * D / 2), *const vs = c.value_scales + unit * (kPage * D / 32);
#pragma unroll
    for (int u = 0; u < ValuePart<D>::kUnits; u++) {
        const int seg = (id >> 4) + u * 16;
        if (seg < D / 8) {
            g.w[u] = *reinterpret_cast<const u32x4 *>(vc + (four * (D / 8) + seg) * 16);
            g.scale[u] = *reinterpret_cast<const uint32_t *>(vs + (seg >> 2) * kPage + four * 4);
        }
    }
}

// spoilt: 64 bytes that say which tokens' values are not finite (looked at on edge pages alone)
template <int D>
__device__ inline void store_values(const ValuePart<D> &g, char *lds, uint8_t *spoilt, int id, bool edge, int written) {
    typedef Images<D> I;
    const int four = id & 15;
    // tokens 4 * four ...: step four / 4, half four % 2, the upper or lower 4 of its 8
    const int chunk = (four >> 2) * 2 + (four & 1), half = four >> 1 & 1;
#pragma unroll
    for (int u = 0; u < ValuePart<D>::kUnits; u++) {
        const int seg = (id >> 4) + u * 16;
        if (seg >= D / 8) continue;
        uint32_t scale = g.scale[u];
        if (edge) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool bad = (scale >> (8 * i) & 255) == kNotFinite;
                if (seg == 0) spoilt[four * 4 + i] = bad;
                if (bad || four * 4 + i >= written) scale = (scale & ~(255u << (8 * i))) | (127u << (8 * i));  // see take_page
            }
        }
        const float s[4] = {scale_at(scale, 0), scale_at(scale, 1), scale_at(scale, 2), scale_at(scale, 3)};
#define VL_TWO_ROWS(B)                                                                                                          \
    {                                                                                                                           \
        const uint32_t x0 = two_values<B>(g.w[u][0], s[0]), x1 = two_values<B>(g.w[u][1], s[1]);                                \
        const uint32_t x2 = two_values<B>(g.w[u][2], s[2]), x3 = two_values<B>(g.w[u][3], s[3]);                                \
        *reinterpret_cast<u32x2 *>(lds + I::value(seg * 8 + 2 * B, chunk) + half * 8) =                                         \
            u32x2{__builtin_amdgcn_perm(x1, x0, 0x05040100), __builtin_amdgcn_perm(x3, x2, 0x05040100)};                        \
        *reinterpret_cast<u32x2 *>(lds + I::value(seg * 8 + 2 * B + 1, chunk) + half * 8) =                                     \
            u32x2{__builtin_amdgcn_perm(x1, x0, 0x07060302), __builtin_amdgcn_perm(x3, x2, 0x07060302)};                        \
    }
        VL_TWO_ROWS(0)
        VL_TWO_ROWS(1)
        VL_TWO_ROWS(2)
        VL_TWO_ROWS(3)
#undef VL_TWO_ROWS
    }
}

__device__ inline float max_of_halves(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    return fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
}
__device__ inline float sum_of_halves(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    return __builtin_bit_cast(float, a0) + __builtin_bit_cast(float, a1);
}

template <int D, int NS, int WAVES, int PAGES>
__global__ __launch_bounds__(WAVES * 64) void attend_many_kernel(AttendArgs a, int tiles) {
    typedef Images<D> I;
    typedef typename ElementOf<NS>::type E;
    constexpr int kRows = 32 * WAVES, kBuffer = I::kBytes + kPage;
    // Parts of a weight, as many as of a query (half precision and float32 keep 16 and 24 bits).  A bfloat16 weight is off by up to
    // 2^-8 of itself, the sum that it is divided by is not: over 16,384 tokens the result's error is 1.16 times that of its own
    // rounding (root of the mean square, 5.00e-4 and 4.30e-4), and more where values cancel.  A second part makes half as many products
    // again and takes that away, for 661 us instead of 494; dividing by the sum of the rounded weights leaves 4.95e-4 for 506.
    constexpr int NW = NS;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    // all tiles of a head go to the same XCD where there are 8 heads; the last tiles, which see most, come first
    const int h = blockIdx.x % a.c.heads, at = blockIdx.x / a.c.heads, split = at % a.splits, tile = tiles - 1 - at / a.splits;
    const int lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Piece w = find_piece(a.t.sequences, tile, [&](int b) { return (int)(((int64_t)row_count(a.t, b) * a.group + kRows - 1) / kRows); });
    if (w.sequence < 0) return;
    const int b = w.sequence, all = row_count(a.t, b), length = length_of(a.t, b);
    const int64_t index = (int64_t)w.piece * kRows + wave * 32 + col;
    const bool real = index < (int64_t)all * a.group;
    const int token = (int)(index / a.group), head = h * a.group + (int)(index % a.group);
    const int64_t row = first_row(a.t, b) + (int64_t)token;
    const int place0 = (int)min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all;
    const int sees = !real ? 0 : a.causal ? min(max(place0 + token + 1, 0), length) : length;
    // of all rows of the workgroup: the first and the last see least and most
    const int first_token = (int)((int64_t)w.piece * kRows / a.group);
    const int last_token = min((int)(((int64_t)w.piece * kRows + kRows - 1) / a.group), all - 1);
    const int least = a.causal ? min(max(place0 + first_token + 1, 0), length) : length;
    const int most = a.causal ? min(max(place0 + last_token + 1, 0), length) : length;

    bf16x8 q[NS][D / 16];
    {
        Eight<NS> x[D / 16];
        const E *const at = (const E *)a.queries + (real ? row * a.q_row + head * a.q_head : 0) + hi * 8;
#pragma unroll
        for (int k = 0; k < D / 16; k++) x[k] = load8<NS>(at + k * 16, real);
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                __bf16 s[NS];
                split_into<NS>((float)x[k][i] * a.turn, s);
#pragma unroll
                for (int n = 0; n < NS; n++) q[n][k][i] = s[n];
            }
        }
    }
    f32x16 acc[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0;
    float top = -INFINITY, sum = 0;

    KeyPart<D> kp[PAGES];
    ValuePart<D> vp[PAGES];
    const int id = threadIdx.x & 255;
    const bool brings_keys = WAVES == 4 || wave < 4, brings_values = WAVES == 4 || wave >= 4;
    auto fetch = [&](int k, int page) {
        if (brings_keys) fetch_keys<D>(kp[k], a.c, (int64_t)page * a.c.heads + h, id);
        if (brings_values) fetch_values<D>(vp[k], a.c, (int64_t)page * a.c.heads + h, id);
    };
    auto store = [&](int k, int buffer, int block, bool edge) {
        char *const to = lds + buffer * kBuffer;
        if (brings_keys) store_keys<D>(kp[k], to, id);
        if (brings_values) store_values<D>(vp[k], to, (uint8_t *)to + I::kBytes, id, edge, length - block * kPage);
    };

    const int blocks = (most + kPage - 1) / kPage;
    const int from = (int)((int64_t)blocks * split / a.splits), to = (int)((int64_t)blocks * (split + 1) / a.splits);
    // 64 blocks' pages are looked up at once, a lane each, and handed out as scalars: a lookup of the next page would be waited for
    // at the head of every round
    int pages = -1;
    uint64_t edges = 0;
    auto look_up = [&](int block) {
        block += lane;
        pages = block < to ? (int)page_of(a.t, a.c, b, block) : -1;
        edges = __ballot(pages >= 0 && ((block + 1) * kPage > least || a.c.bound_scales[(int64_t)pages * a.c.heads + h] == kBoundless));
    };
    look_up(from);
    int page[PAGES], next[PAGES];
    uint32_t edge = 0, next_edge = 0;
#pragma unroll
    for (int k = 0; k < PAGES; k++) {
        page[k] = __builtin_amdgcn_readlane(pages, k);
        if (page[k] >= 0) fetch(k, page[k]);
    }
    edge = (uint32_t)edges & ((1u << PAGES) - 1);
#pragma unroll
    for (int k = 0; k < PAGES; k++)
        if (page[k] >= 0) store(k, k, from + k, edge >> k & 1);
    __syncthreads();
    for (int round = from, turn = 0; round < to; round += PAGES, turn ^= 1) {
        const int at = round + PAGES - from & 63;
        if (at == 0) look_up(round + PAGES);
        next_edge = (uint32_t)(edges >> at) & ((1u << PAGES) - 1);
#pragma unroll
        for (int k = 0; k < PAGES; k++) {
            next[k] = __builtin_amdgcn_readlane(pages, at + k);  // -1 behind the last
            if (next[k] >= 0) fetch(k, next[k]);
        }
#pragma unroll
        for (int k = 0; k < PAGES; k++) {
            if (page[k] < 0) continue;
            const int block = round + k;
            const char *const in = lds + (turn * PAGES + k) * kBuffer;
            // of three parts of a query the second and third add to sums of their own, which rounds a score less often
            constexpr int kSums = NS == 3 ? 2 : 1;
            f32x16 sums[kSums][2];
#pragma unroll
            for (int n = 0; n < kSums; n++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) sums[n][t][i] = 0;
#pragma unroll
            for (int c = 0; c < D / 16; c++) {
                // products that add to the same sums do not follow each other: one waits for the other's result
                bf16x8 x[2];
#pragma unroll
                for (int t = 0; t < 2; t++) x[t] = *reinterpret_cast<const bf16x8 *>(in + I::key(t * 32 + col, c * 2 + hi));
#pragma unroll
                for (int n = 0; n < NS; n++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        f32x16 &to = sums[n > 0 ? kSums - 1 : 0][t];
                        to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[t], q[n][c], to, 0, 0, 0);
                    }
            }
            f32x16(&s)[2] = sums[0];
            if constexpr (NS == 3) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[t][i] += sums[1][t][i];
            }
            if (edge >> k & 1) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int place = t * 32 + 8 * (i >> 2) + 4 * hi + (i & 3);
                        if (reinterpret_cast<const uint8_t *>(in)[I::kBytes + place]) s[t][i] = NAN;
                        if (block * kPage + place >= sees) s[t][i] = -INFINITY;
                    }
            }
            float most_here = s[0][0];
#pragma unroll
            for (int i = 1; i < 32; i++) most_here = fmaxf(most_here, s[i >> 4][i & 15]);
            most_here = max_of_halves(most_here) * a.scale;
            // The maximum that weights are measured from may lie up to 8 below the true one: weights up to 256 cost nothing, and
            // the sums are rescaled a few times a row instead of at every new maximum.  Each row's moves when that row passes it, so
            // that no result depends on the rows beside it.
            if (__ballot(most_here > top + 8.0f)) {
                const float now = most_here > top + 8.0f ? most_here : top;
                const float less = now > -INFINITY ? __builtin_amdgcn_exp2f(top - now) : 1.0f;
                top = now;
                sum *= less;
#pragma unroll
                for (int d = 0; d < D / 32; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[d][i] *= less;
            }
            const float minus = top > -INFINITY ? -top : 0.0f;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                float part = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    s[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], a.scale, minus));
                    part += s[t][i];
                }
                sum += part;
            }
#pragma unroll
            for (int step = 0; step < 4; step++) {
                bf16x8 p[NW];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    __bf16 x[NW];
                    split_into<NW>(s[step >> 1][8 * (step & 1) + i], x);
#pragma unroll
                    for (int n = 0; n < NW; n++) p[n][i] = x[n];
                }
                bf16x8 v[D / 32];
#pragma unroll
                for (int d = 0; d < D / 32; d++) v[d] = *reinterpret_cast<const bf16x8 *>(in + I::value(d * 32 + col, step * 2 + hi));
#pragma unroll
                for (int n = 0; n < NW; n++)
#pragma unroll
                    for (int d = 0; d < D / 32; d++) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[d], p[n], acc[d], 0, 0, 0);
            }
        }
#pragma unroll
        for (int k = 0; k < PAGES; k++) {
            if (next[k] >= 0) store(k, (turn ^ 1) * PAGES + k, round + PAGES + k, next_edge >> k & 1);
            page[k] = next[k];
        }
        edge = next_edge;
        __syncthreads();
    }
    sum = sum_of_halves(sum);
    if (!real) return;
    const int64_t out_row = row * a.heads_q + head;
    if (a.splits > 1) {
        float *const to = a.part + (out_row * a.splits + split) * D;
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<f32x4 *>(to + d * 32 + i * 8 + hi * 4) = f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
        if (hi == 0) {
            float *const ends = a.part + (int64_t)a.t.rows * a.heads_q * a.splits * D + (out_row * a.splits + split) * 2;
            ends[0] = top;
            ends[1] = sum;
        }
        return;
    }
    typedef E e4 __attribute__((ext_vector_type(4)));
    const float by = sum == 0 ? 0.0f : 1.0f / sum;
    E *const out = (E *)a.out + out_row * D;
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<e4 *>(out + d * 32 + i * 8 + hi * 4) =
                e4{(E)(acc[d][4 * i] * by), (E)(acc[d][4 * i + 1] * by), (E)(acc[d][4 * i + 2] * by), (E)(acc[d][4 * i + 3] * by)};
    if (hi == 0 && a.lse) a.lse[out_row] = (top + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}
