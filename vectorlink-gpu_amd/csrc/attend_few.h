// Attention of a few rows over many tokens: single tokens of a batch of answers, a handful of proposed tokens, and rows with
// blocks of their own.
//
// What bounds it is the cache's bytes: D + D / 16 a token and head, against 4 D operations for each of the queries that share
// the head.  So a wavefront takes whole pages, 64 tokens at a time, every byte read once in 16-byte pieces, and keeps the
// rest in registers; a maximum and a sum that run along (x -> exp2(x - max), both rescaled where the maximum grows) make one
// pass of it.  Measured: 4 tokens over 131,072, 32 heads on 8 of 128, 570 MB in 100 us (5.7 TB/s; a sum of 2 GiB reads 6.1 to 6.2) and
// 5 us to join; 64 over 4,096 to 8,192 429 MB in 84 to 90 us, where the longest sequences' workgroups are waited for.
//
// S^T = K Q^T: A = 16 tokens x 32 dimensions, B = 32 dimensions x 16 rows (row = lane % 16 = r, quad = lane / 16 = c).  Which
// token stands in which row of A and which dimension at which place of the sum is free, as long as both operands agree:
//   token of tile m, row 4 c' + e of A:  c' * 16 + m * 4 + e,  so the results of a lane are 16 tokens in a row, c * 16 ...
//   dimensions of lane (c, .):           a quarter of a part of 128 (or 64, 32), so that its 16 (8, 4) bytes have one scale.
// out^T = V^T P^T then takes P^T as it lies in the registers: B = 32 tokens x 16 rows, of quad c the tokens c * 16 + 8 s ...,
// and A = 16 dimensions x the same tokens.  A byte of the cache holds two dimensions of a token, so two tokens' bytes turn
// into two dimensions' pairs of tokens by two permutations.  Row i of tile k of a part: dimension 8 i + k (4 i + k, 2 i + k).
//
// Queries enter as NS bfloat16 values that add up to them exactly (bfloat16 1, half 2, float32 3: 24 bits), weights as two that
// hold 16 bits of them (float32: three, 24 bits), keys and values are exact.  Weights of one part would halve the matrix
// instructions of the second product, which are not what bounds this, and their error would be as large as a bfloat16
// result's own rounding.
#pragma once
#include "attend.h"
#include "weigh_scores.h"

template <int D, int BITS = 4>
struct Parts {  // D = parts of 128, then 64, then 32
    static constexpr int k128 = D / 128, k64 = D % 128 / 64, k32 = D % 64 / 32, kCount = k128 + k64 + k32;
    static constexpr int width(int p) { return p < k128 ? 128 : p == k128 && k64 ? 64 : 32; }
    static constexpr int base(int p) { return p <= k128 ? 128 * p : 128 * k128 + 64; }
};
template <int D>
struct Parts<D, 8> {  // D = parts of 64, then 32: 16 bytes are half as many dimensions
    static constexpr int k64 = D / 64, k32 = D % 64 / 32, kCount = k64 + k32;
    static constexpr int width(int p) { return p < k64 ? 64 : 32; }
    static constexpr int base(int p) { return 64 * p; }
};

// one page of a head, as a lane holds it
template <int D, int BITS = 4>
struct PageRegs {
    static constexpr int P = Parts<D>::kCount;
    uint32_t k[P][4][4];  // [part][tile m][word]
    u32x4 ks[P];          // scales of tiles 0 .. 3: byte r % 4 of word m
    u32x4 v[P][4];        // [part][4 tokens m], a word a token
    u32x4 vs[P];          // scales of tokens c * 16 + 4 m + byte
};

template <int D, int USE>
__device__ inline void load_page(PageRegs<D> &g, const CacheView &c, int64_t page, int h) {
    typedef Parts<D> PT;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    const int64_t unit = page * c.heads + h;
    const uint8_t *const kc = c.keys + unit * (kPage * D / 2), *const vc = c.values + unit * (kPage * D / 2);
    const uint8_t *const ks = c.key_scales + unit * (kPage * D / 32), *const vs = c.value_scales + unit * (kPage * D / 32);
    const int token = (r >> 2) * 16 + (r & 3);
#pragma unroll
    for (int p = 0; p < PT::kCount; p++) {
        const int W = PT::width(p), base = PT::base(p);
#pragma unroll
        for (int m = 0; m < 4; m++) {
            const uint8_t *const at = kc + (token + m * 4) * (D / 2) + base / 2 + q * (W / 8);
            if (W == 128) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(at);
                g.k[p][m][0] = x[0], g.k[p][m][1] = x[1], g.k[p][m][2] = x[2], g.k[p][m][3] = x[3];
            } else if (W == 64) {
                const u32x2 x = *reinterpret_cast<const u32x2 *>(at);
                g.k[p][m][0] = x[0], g.k[p][m][1] = x[1];
            } else {
                g.k[p][m][0] = *reinterpret_cast<const uint32_t *>(at);
            }
        }
        g.ks[p] = *reinterpret_cast<const u32x4 *>(ks + (base / 32 + q * W / 128) * kPage + (r >> 2) * 16);
    }
#pragma unroll
    for (int p = 0; p < PT::kCount; p++) {
        const int W = PT::width(p), base = PT::base(p);
        const int seg = base / 8 + r * W / 128;
#pragma unroll
        for (int m = 0; m < 4; m++) g.v[p][m] = *reinterpret_cast<const u32x4 *>(vc + ((q * 4 + m) * (D / 8) + seg) * 16);
        g.vs[p] = *reinterpret_cast<const u32x4 *>(vs + (seg >> 2) * kPage + q * 16);
    }
}

// A page in 8 bits: the same tokens and dimensions of parts of 64 (32).  A word of values is a dimension's codes of four tokens, so
// two halves of it turn into the pairs of tokens that the second product takes, without permutations.
template <int D>
struct PageRegs<D, 8> {
    static constexpr int P = Parts<D, 8>::kCount;
    u32x4 k[P][4];          // [part][tile m]: of 64 dimensions the 16 from q * 16 on
    u32x4 v[P][4];          // [part][4 tokens m], a word a dimension: 4 r + j, or 2 r + j
    float key_scale, value_scale;
};
// What a call over a cache in 8 bits uses a page for.  One that a single wavefront reads - a token's queries are one tile - is asked for
// without leaving a place in the caches to it: 4 tokens over 131,072 186 us with a place and 165 (6.5 TB/s) without, 64 over 4,096 to
// 8,192 149 and 145.  Where several tiles share the pages the caches are what they share them by: 16 sequences of 5 tokens over 8,000
// to 16,384 184 us with and 228 without.
enum PageUse { kShared, kOnce, kOnceAndScores };
template <int USE, class T>
__device__ inline T load_of_page(const uint8_t *at) {
    if constexpr (USE == kShared) return *reinterpret_cast<const T *>(at);
    else return __builtin_nontemporal_load(reinterpret_cast<const T *>(at));
}
template <int USE>
__device__ inline void load_codes(u32x4 &to, const uint8_t *at, int width) {  // of 64 dimensions, or 32
    if (width == 64) {
        to = load_of_page<USE, u32x4>(at);
    } else {
        const u32x2 x = load_of_page<USE, u32x2>(at);
        to[0] = x[0], to[1] = x[1];
    }
}
template <int D, int USE>
__device__ inline void load_page_keys(PageRegs<D, 8> &g, const CacheView &c, int64_t page, int h) {
    typedef Parts<D, 8> PT;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    const uint8_t *const kc = c.keys + (page * c.heads + h) * (kPage * D);
    const int token = (r >> 2) * 16 + (r & 3);
#pragma unroll
    for (int m = 0; m < 4; m++)
#pragma unroll
        for (int p = 0; p < PT::kCount; p++) load_codes<USE>(g.k[p][m], kc + (token + m * 4) * D + PT::base(p) + q * (PT::width(p) / 4), PT::width(p));
}
template <int D, int USE>
__device__ inline void load_page_values(PageRegs<D, 8> &g, const CacheView &c, int64_t page, int h) {
    typedef Parts<D, 8> PT;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    const uint8_t *const vc = c.values + (page * c.heads + h) * (kPage * D);
#pragma unroll
    for (int m = 0; m < 4; m++)
#pragma unroll
        for (int p = 0; p < PT::kCount; p++) load_codes<USE>(g.v[p][m], vc + ((q * 4 + m) * D + PT::base(p) + r * (PT::width(p) / 16)) * 4, PT::width(p));
}
template <int D, int USE>
__device__ inline void load_page(PageRegs<D, 8> &g, const CacheView &c, int64_t page, int h) {
    load_page_keys<D, USE>(g, c, page, h);
    load_page_values<D, USE>(g, c, page, h);
}

// NS bfloat16 values that add up to x (to 8 NS bits of it): the first NS - 1 cut off, so that what is left is exact.
template <int NS>
__device__ inline void split_into(float x, __bf16 (&out)[NS]) {
#pragma unroll
    for (int n = 0; n < NS; n++) {
        if (n == NS - 1) {
            out[n] = (__bf16)x;
        } else {
            const float cut = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xFFFF0000u);
            out[n] = (__bf16)cut;
            x -= cut;
        }
    }
}

// The state of 16 rows: lane (q, r) holds row r, of every part of W dimensions the W / 4 from q * W / 4 on, as [place e][tile k]:
// dimension base + (W / 16) * (4 q + e) + k.
template <int D>
struct RowState {
    f32x4 acc[D / 16];  // tiles of all parts, one after the other
    float top, sum;     // maximum so far (of all lanes of the row), sum of this lane's weights
};

// The queries of lane (q, r): those of row r, the dimensions as the keys' words hold them.
template <int D, int NS>
struct QueryRegs {
    bf16x8 x[NS][D / 32];
};

template <int D, int NS>
struct QueryLoads {
    Eight<NS> x[D / 32];
};
template <int D, int NS, int BITS = 4>
__device__ inline void load_queries(QueryLoads<D, NS> &l, const AttendArgs &a, bool real, int64_t row, int head) {
    typedef Parts<D, BITS> PT;
    typedef typename ElementOf<NS>::type E;
    const int q = (threadIdx.x & 63) >> 4;
    const E *const at = (const E *)a.queries + (real ? row * a.q_row + head * a.q_head : 0);
#pragma unroll
    for (int p = 0; p < PT::kCount; p++) {
        const int W = PT::width(p), base = PT::base(p);
#pragma unroll
        for (int j = 0; j < W / 32; j++) l.x[base / 32 + j] = load8<NS>(at + base + q * (W / 4) + j * 8);
    }
}
template <int D, int NS>
__device__ inline void take_queries(QueryRegs<D, NS> &f, const QueryLoads<D, NS> &l, bool real, float turn) {
    typedef typename ElementOf<NS>::type E;
#pragma unroll
    for (int k = 0; k < D / 32; k++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            __bf16 s[NS];
            split_into<NS>((float)(real ? l.x[k][i] : (E)0.0f) * turn, s);
#pragma unroll
            for (int n = 0; n < NS; n++) f.x[n][k][i] = s[n];
        }
    }
}

// Where a tile has at most C = 4 or 8 rows, three quarters or half of the lanes of S^T hold nothing, and the softmax of it would
// cost as much as that of 16.  Scores then move to where they fill the lanes: of lane (q, r) row r % C, and of its 16 tokens the
// tiles m = (C / 4) (r / C) + k.  Exponentials and all that is around them are C / 16 of the work, for 12 (C = 4) or 8 moves of a
// register there and 12 or 8 back: of 466 vector instructions a page of 128 dimensions 387 are left with C = 4.
template <int C>
__device__ inline void spread_scores(const f32x4 (&s)[4], float (&t)[C / 4][4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        auto moved = [](float to, float from, auto control, auto banks) {
            return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, to), __builtin_bit_cast(int, from),
                                                                         decltype(control)::value, 0xF, decltype(banks)::value, false));
        };
        const float x0 = s[0][e], x1 = s[1][e], x2 = s[2][e], x3 = s[3][e];
        if constexpr (C == 4) {  // row_shr: 4, 8, 12 into the second, third and fourth 4 lanes of a row
            t[0][e] = moved(x0, x1, std::integral_constant<int, 0x114>(), std::integral_constant<int, 2>());
            t[0][e] = moved(t[0][e], x2, std::integral_constant<int, 0x118>(), std::integral_constant<int, 4>());
            t[0][e] = moved(t[0][e], x3, std::integral_constant<int, 0x11C>(), std::integral_constant<int, 8>());
        } else if constexpr (C == 8) {
            t[0][e] = moved(x0, x2, std::integral_constant<int, 0x118>(), std::integral_constant<int, 12>());
            t[1][e] = moved(x1, x3, std::integral_constant<int, 0x118>(), std::integral_constant<int, 12>());
        } else {
            t[0][e] = x0, t[1][e] = x1, t[2][e] = x2, t[3][e] = x3;
        }
    }
}
// The way back, for the word that tile m = (C / 4) (r / C) + k has of a row: lane (q, r < C) gets those of all four tiles.
template <int C>
__device__ inline void gather_words(const uint32_t (&u)[C / 4], uint32_t (&w)[4]) {
    if constexpr (C == 4) {  // row_shl: 4, 8, 12
        w[0] = u[0];
        w[1] = __builtin_amdgcn_update_dpp(0, (int)u[0], 0x104, 0xF, 0xF, false);
        w[2] = __builtin_amdgcn_update_dpp(0, (int)u[0], 0x108, 0xF, 0xF, false);
        w[3] = __builtin_amdgcn_update_dpp(0, (int)u[0], 0x10C, 0xF, 0xF, false);
    } else if constexpr (C == 8) {
        w[0] = u[0], w[1] = u[1];
        w[2] = __builtin_amdgcn_update_dpp(0, (int)u[0], 0x108, 0xF, 0xF, false);
        w[3] = __builtin_amdgcn_update_dpp(0, (int)u[1], 0x108, 0xF, 0xF, false);
    } else {
        w[0] = u[0], w[1] = u[1], w[2] = u[2], w[3] = u[3];
    }
}
// f over the lanes of a row of 16 that hold the same row of the tile
template <int C, class F>
__device__ inline float over_copies(float x, F f) {
    auto turned = [](float x, auto control) {  // row_ror
        const int u = __builtin_bit_cast(int, x);
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, decltype(control)::value, 0xF, 0xF, false));
    };
    if constexpr (C <= 8) x = f(x, turned(x, std::integral_constant<int, 0x128>()));
    if constexpr (C == 4) x = f(x, turned(x, std::integral_constant<int, 0x124>()));
    return x;
}

// Where the scores of single tokens go: a buffer of its own for a token and head, the byte of it that this lane's row of the page has -
// of a lane without a row past its end, where a store is dropped.  A branch around the store would leave the compiler to guess
// how many stores are on their way, and loads would wait for them.
struct ScoresAt {
    __amdgpu_buffer_rsrc_t buffer;
    int lane, page;
};

// A page's 64 tokens: this lane's row (r % C) sees the first `sees` of them, `written` hold something; edge: some row does not see
// some token, or some token may not be finite.  Spoilt tokens (scale 255, of 8 bits codes of NaN) turn the rows that see them into NaN, and
// no others.  put: where scores go, of a call that keeps them.  between(): what is done once the keys have been used and before the
// values are.
template <int D, int NS, int C, int BITS, int USE, class F>
__device__ inline void take_page(RowState<D> &st, PageRegs<D, BITS> &g, const QueryRegs<D, NS> &f, float scale, bool edge, int sees,
                                 int written, const ScoresAt &put, F between) {
    typedef Parts<D, BITS> PT;
    constexpr int NW = NS < 2 ? 2 : NS;  // parts of a weight
    constexpr int M = C / 4;             // tiles of 4 tokens of this lane
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    f32x4 s[4];
    const int turn = (8 * (r & 3) + 9) & 31;
    // products that add to the same sums lie four apart: one waits for the other's result.  Of three parts the second and third add
    // to sums of their own, so that a score is rounded once for 32 dimensions, not three times.
    f32x4 small[4];
#pragma unroll
    for (int m = 0; m < 4; m++) s[m] = small[m] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < PT::kCount; p++) {
        float ks[4];
        if constexpr (BITS == 4) {
#pragma unroll
            for (int m = 0; m < 4; m++) ks[m] = __builtin_bit_cast(float, __builtin_amdgcn_alignbit(g.ks[p][m], g.ks[p][m], turn));
        }
#pragma unroll
        for (int j = 0; j < PT::width(p) / 32; j++) {
            bf16x8 k[4];
#pragma unroll
            for (int m = 0; m < 4; m++) {
                if constexpr (BITS == 4) k[m] = eight_values(g.k[p][m][j], ks[m]);
                else k[m] = eight_of_bytes(g.k[p][m][2 * j], g.k[p][m][2 * j + 1], g.key_scale);
            }
#pragma unroll
            for (int n = 0; n < NS; n++)
#pragma unroll
                for (int m = 0; m < 4; m++) {
                    f32x4 &to = NS == 3 && n > 0 ? small[m] : s[m];
                    to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[m], f.x[n][PT::base(p) / 32 + j], to, 0, 0, 0);
                }
        }
    }
    if constexpr (NS == 3) {
#pragma unroll
        for (int m = 0; m < 4; m++) s[m] += small[m];
    }
    between();
    float t[M][4];
    spread_scores<C>(s, t);
    if (edge) {
        const int m0 = M * (r / C);
        // of 4 tokens m a word whose bytes tell which are spoilt
        auto marks = [&](int m) {
            if constexpr (BITS == 4) return (uint32_t)g.vs[0][m];
            else return g.v[0][m][0];
        };
        auto is_spoilt = [](uint32_t word, int e) {
            if constexpr (BITS == 4) return (word >> (8 * e) & 255) == kNotFinite;
            else return (word >> (8 * e) & 127) == kByteNaN;
        };
#pragma unroll
        for (int k = 0; k < M; k++) {
            uint32_t word = marks(k);
            if constexpr (C == 4) word = r < 4 ? marks(0) : r < 8 ? marks(1) : r < 12 ? marks(2) : marks(3);
            if constexpr (C == 8) word = r < 8 ? marks(k) : marks(2 + k);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (is_spoilt(word, e)) t[k][e] = NAN;
                if (q * 16 + (m0 + k) * 4 + e >= sees) t[k][e] = -INFINITY;
            }
        }
        // values of a token that is spoilt or not there: its weight is 0 or NaN whatever it holds, so any finite value will do
#pragma unroll
        for (int m = 0; m < 4; m++) {
            if constexpr (BITS == 4) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (is_spoilt(marks(m), e) || q * 16 + m * 4 + e >= written) {
#pragma unroll
                        for (int p = 0; p < PT::kCount; p++) g.vs[p][m] = (g.vs[p][m] & ~(255u << (8 * e))) | (127u << (8 * e));
                    }
            } else {
                uint32_t keep = ~0u;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (is_spoilt(marks(m), e) || q * 16 + m * 4 + e >= written) keep &= ~(255u << (8 * e));
#pragma unroll
                for (int p = 0; p < PT::kCount; p++)
#pragma unroll
                    for (int j = 0; j < PT::width(p) / 16; j++) g.v[p][m][j] &= keep;
            }
        }
    }
    if constexpr (USE == kOnceAndScores) {
#pragma unroll
        for (int k = 0; k < M; k++)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{t[k][0], t[k][1], t[k][2], t[k][3]}), put.buffer, put.lane + k * 16, put.page, 0);
    }
    float top = t[0][0];
#pragma unroll
    for (int i = 1; i < 4 * M; i++) top = fmaxf(top, t[i >> 2][i & 3]);
    top = over_copies<C>(top, [](float a, float b) { return fmaxf(a, b); });
    top = fmaxf(max_over_quads(top) * scale, st.top);
    if (__ballot(top > st.top)) {
        const float less = top > -INFINITY ? __builtin_amdgcn_exp2f(st.top - top) : 1.0f;
        st.top = top;
        st.sum *= less;
#pragma unroll
        for (int k = 0; k < D / 16; k++) st.acc[k] *= less;
    }
    // scale s - top with one rounding: a product rounded on its own would be off by a share of the score, not of the difference
    const float minus = st.top > -INFINITY ? -st.top : 0.0f;  // a row that has seen nothing yet: all weights 0
    float by = scale;
    if (const bool far = is_far(minus); __ballot(far)) {
#pragma unroll
        for (int i = 0; i < 4 * M; i++) t[i >> 2][i & 3] = far ? t[i >> 2][i & 3] * scale : t[i >> 2][i & 3];
        by = far ? 1.0f : scale;
    }
    uint32_t weight[NW][2][4];  // [part][two tokens][tile]
    {
        uint32_t pair[NW][2][M];
#pragma unroll
        for (int k = 0; k < M; k++) {
#pragma unroll
            for (int e = 0; e < 4; e++) t[k][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(t[k][e], by, minus));
            st.sum += (t[k][0] + t[k][1]) + (t[k][2] + t[k][3]);
#pragma unroll
            for (int two = 0; two < 2; two++) {
                __bf16 a[NW], b[NW];
                split_into<NW>(t[k][2 * two], a);
                split_into<NW>(t[k][2 * two + 1], b);
#pragma unroll
                for (int n = 0; n < NW; n++) pair[n][two][k] = __builtin_bit_cast(uint32_t, bf16x2{a[n], b[n]});
            }
        }
#pragma unroll
        for (int n = 0; n < NW; n++)
#pragma unroll
            for (int two = 0; two < 2; two++) gather_words<C>(pair[n][two], weight[n][two]);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {  // 32 tokens a step: of every quad 8
        bf16x8 w[NW];
#pragma unroll
        for (int n = 0; n < NW; n++)
            w[n] = __builtin_bit_cast(bf16x8, u32x4{weight[n][0][2 * h], weight[n][1][2 * h], weight[n][0][2 * h + 1], weight[n][1][2 * h + 1]});
#pragma unroll
        for (int p = 0; p < PT::kCount; p++) {
            const int W = PT::width(p), t0 = PT::base(p) / 16;
            if constexpr (BITS == 8) {
                bf16x8 a[4];
#pragma unroll
                for (int j = 0; j < W / 16; j++) a[j] = eight_of_bytes(g.v[p][2 * h][j], g.v[p][2 * h + 1][j], g.value_scale);
#pragma unroll
                for (int n = 0; n < NW; n++)
#pragma unroll
                    for (int j = 0; j < W / 16; j++) st.acc[t0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j], w[n], st.acc[t0 + j], 0, 0, 0);
                continue;
            }
            if constexpr (BITS == 4) {
                uint32_t word[8];
                float vs[8];
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const int m = 2 * h + (u >> 2);
                    word[u] = g.v[p][m][u & 3];
                    if (W == 64) word[u] >>= 16 * (r & 1);
                    if (W == 32) word[u] >>= 8 * (r & 3);
                    vs[u] = scale_at(g.vs[p][m], u & 3);
                }
                // byte B of the words: dimensions of tiles 2 B and 2 B + 1
                auto two_tiles = [&](auto byte, u32x4(&a)[2]) {
                    constexpr int B = decltype(byte)::value;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t x = two_values<B>(word[2 * i], vs[2 * i]), y = two_values<B>(word[2 * i + 1], vs[2 * i + 1]);
                        a[0][i] = __builtin_amdgcn_perm(y, x, 0x05040100);
                        a[1][i] = __builtin_amdgcn_perm(y, x, 0x07060302);
                    }
                };
                auto products = [&](int tile, const u32x4(&a)[2][2], int tiles) {
#pragma unroll
                    for (int n = 0; n < NW; n++)
#pragma unroll
                        for (int k = 0; k < tiles; k++)
                            st.acc[tile + k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[k >> 1][k & 1]), w[n], st.acc[tile + k], 0, 0, 0);
                };
                u32x4 a[2][2];
                two_tiles(std::integral_constant<int, 0>(), a[0]);
                if (W >= 64) two_tiles(std::integral_constant<int, 1>(), a[1]);
                products(t0, a, W >= 64 ? 4 : 2);
                if (W >= 128) {
                    two_tiles(std::integral_constant<int, 2>(), a[0]);
                    two_tiles(std::integral_constant<int, 3>(), a[1]);
                    products(t0 + 4, a, 4);
                }
            }
        }
    }
}

// The blocks i = from, from + step, ... < to of a wavefront, as entries of a list or themselves; pages that do not exist and
// blocks behind the last place that a row sees are passed over.
struct Blocks {
    const int32_t *list;
    int from, step, to;
};

// All of a wavefront's blocks.  64 blocks' pages are looked up at once, a lane each, and handed out as scalars: a lookup in the
// loop would wait, in order, for the page's bytes that were asked for before it.  Where two pages fit the registers of two
// wavefronts a SIMD, the next page's bytes are loaded before a page is worked on (64 dimensions: 61 us with one, 54 with two, 64
// tokens over 4,096 to 8,192 and 8 heads; 128: 94 and 92; 96, and 128 of float32, spill); behind the last one the same page is loaded once more instead
// of a branch, over which the compiler would have to wait for all loads.  The queries' loads are waited for with the first
// page's.
template <int D, int NS, int C, int BITS = 4, int USE = kShared>
__device__ inline void take_blocks(RowState<D> &st, const AttendArgs &a, const QueryLoads<D, NS> &queries, bool real, Blocks l, int b,
                                   int h, int sees, int least, int most, int length, ScoresAt scores = {}) {
    const int lane = threadIdx.x & 63;
    QueryRegs<D, NS> f;
    bool first = true;
    for (int i0 = l.from; i0 < l.to; i0 += 64 * l.step) {
        const int i = i0 + lane * l.step;
        int block = 0, page = -1;
        if (i < l.to) {
            block = l.list ? l.list[i] : i;
            page = (int)page_of(a.t, a.c, b, block);
            if (page >= 0 && block * kPage >= most) page = -1;
        }
        uint64_t left = __ballot(page >= 0), edges = 0;
        if (!left) continue;
        const int64_t unit = (int64_t)max(page, 0) * a.c.heads + h;  // there is a page
        int bound = 0;
        uint32_t scales = 0;
        if constexpr (BITS == 4) bound = a.c.bound_scales[unit];
        else scales = a.c.scales[unit];
        int at = 0;
        auto next = [&](PageRegs<D, BITS> &g) {  // the next page's loads
            if (left) {
                at = __builtin_ctzll(left);
                left &= left - 1;
            }
            load_page<D, USE>(g, a.c, __builtin_amdgcn_readlane(page, at), h);
        };
        auto take = [&](PageRegs<D, BITS> &g, int at, auto between) {
            const int first = __builtin_amdgcn_readlane(block, at) * kPage;
            if constexpr (BITS == 8) {
                const uint32_t word = __builtin_amdgcn_readlane(scales, at);
                g.key_scale = scale_of_keys(word);
                g.value_scale = scale_of_values(word);
            }
            if constexpr (USE == kOnceAndScores) scores.page = first * a.group * 4;
            take_page<D, NS, C, BITS, USE>(st, g, f, a.scale, edges >> at & 1, sees - first, length - first, scores, between);
        };
        auto look = [&] {  // after the first page's loads
            edges = __ballot(page >= 0 && ((block + 1) * kPage > least || (BITS == 4 ? bound == kBoundless : is_marked(scales))));
            if (first) take_queries<D, NS>(f, queries, real, a.turn);
            first = false;
        };
        auto nothing = [] {};
        PageRegs<D, BITS> x;
        next(x);
        look();
        if constexpr (BITS == 8 && D > 64) {
            // one page's registers: the next page's keys are asked for once this one's have been used, its values likewise
            while (left) {
                const int here = at;
                at = __builtin_ctzll(left);
                left &= left - 1;
                const int64_t ahead = __builtin_amdgcn_readlane(page, at);
                take(x, here, [&] { load_page_keys<D, USE>(x, a.c, ahead, h); });
                load_page_values<D, USE>(x, a.c, ahead, h);
            }
            take(x, at, nothing);
        } else if constexpr (BITS == 8 || D == 64 || (D == 128 && NS < 3)) {
            PageRegs<D, BITS> y;
            for (;;) {
                int here = at;
                bool last = !left;
                next(y);
                take(x, here, nothing);
                if (last) break;
                here = at;
                last = !left;
                next(x);
                take(y, here, nothing);
                if (last) break;
            }
        } else {
            for (;;) {
                take(x, at, nothing);
                if (!left) break;
                next(x);
            }
        }
    }
}

template <int C>
__device__ inline float sum_of_row(float x) {
    return sum_over_quads(over_copies<C>(x, [](float a, float b) { return a + b; }));
}

template <int D>
__device__ inline void start_rows(RowState<D> &st) {
#pragma unroll
    for (int k = 0; k < D / 16; k++) st.acc[k] = f32x4{0, 0, 0, 0};
    st.top = -INFINITY;
    st.sum = 0;
}

// Result of a row and head: sums x of dimensions d ..., the maximum and the sum of weights, either whole or one split's.
template <int NS>
__device__ inline void put8(const AttendArgs &a, int64_t out_row, int split, int D, int d, float (&x)[8], float total) {
    typedef typename ElementOf<NS>::type E;
    if (a.splits > 1) {
        float *const to = a.part + (out_row * a.splits + split) * D + d;
        *reinterpret_cast<f32x4 *>(to) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4 *>(to + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        const float by = total == 0 ? 0.0f : 1.0f / total;
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] *= by;
        store8<NS>((E *)a.out + out_row * D + d, x);
    }
}
__device__ inline void put_sums(const AttendArgs &a, int64_t out_row, int split, int D, float top, float total) {
    if (a.splits > 1) {
        float *const to = a.part + (int64_t)a.t.rows * a.heads_q * a.splits * D + (out_row * a.splits + split) * 2;
        to[0] = top;
        to[1] = total;
    } else {
        if (a.lse) a.lse[out_row] = (top + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
        if (a.ends) *reinterpret_cast<f32x2 *>(a.ends + out_row * 2) = f32x2{top, total};
    }
}

// Joins what WAVES wavefronts have of the same 16 rows, 128 dimensions at a time: thread t the 8 dimensions 8 (t % 16) of row
// t / 16.  out_row(r): where row r belongs, negative if it is none.
constexpr int kJoinPad = 132;  // a row of 128 sums in LDS: 16 lanes x 4 words of a store lie in 64 banks
template <int WAVES>
struct JoinLds {
    float sum[WAVES][16 * kJoinPad];
    float top[WAVES][16], all[WAVES][16];
};
template <int D, int NS, int WAVES, int C, int BITS = 4, class F>
__device__ inline void join_waves(const RowState<D> &st, JoinLds<WAVES> &s, const AttendArgs &a, int split, F out_row) {
    typedef Parts<D, BITS> PT;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15, wave = threadIdx.x >> 6;
    const float sum = sum_of_row<C>(st.sum);
    if (q == 0) {
        s.top[wave][r] = st.top;
        s.all[wave][r] = sum;
    }
    __syncthreads();
    const int jr = threadIdx.x >> 4 & 15, js = threadIdx.x & 15;
    float top = s.top[0][jr], weight[WAVES], total = 0;
#pragma unroll
    for (int i = 1; i < WAVES; i++) top = fmaxf(top, s.top[i][jr]);
    const float base = top > -INFINITY ? top : 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        weight[i] = __builtin_amdgcn_exp2f(s.top[i][jr] - base);
        total += weight[i] * s.all[i][jr];
    }
    const int64_t to = threadIdx.x < 256 ? out_row(jr) : -1;
#pragma unroll
    for (int p = 0; p < PT::kCount; p++) {
        const int W = PT::width(p), t0 = PT::base(p) / 16;
        if (p) __syncthreads();
        // lane (q, r) has dimensions q * W / 4 + e * W / 16 + k
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int k = 0; k < W / 16; k += 2)
                *reinterpret_cast<f32x2 *>(&s.sum[wave][r * kJoinPad + q * (W / 4) + e * (W / 16) + k]) = f32x2{st.acc[t0 + k][e], st.acc[t0 + k + 1][e]};
        __syncthreads();
        if (js * 8 < W && to >= 0) {
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < WAVES; i++)
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] += weight[i] * s.sum[i][jr * kJoinPad + js * 8 + k];
            put8<NS>(a, to, split, D, PT::base(p) + js * 8, x, total);
        }
    }
    if (js == 0 && to >= 0) put_sums(a, to, split, D, top, total);
    if constexpr (BITS == 8) {  // for those who come after: what the rows end with
        if (js == 0 && threadIdx.x < 256) {
            s.top[0][jr] = top;
            s.all[0][jr] = total;
        }
    }
}

// A tile is 16 rows of one head: of the queries of one token where there is a list, of all tokens of a sequence otherwise.
// The WAVES wavefronts of a workgroup share a tile's blocks and are joined; 1: each of four has a tile of its own.  C: the most
// rows that a tile has, 16 unless its rows are one token's, which see the same.
template <int D, int NS, int WAVES, int C, int BITS = 4, int USE = kShared>
__global__ __launch_bounds__(WAVES == 8 ? 512 : 256, WAVES != 8 && D <= 128 ? 2 : 1) void attend_few_kernel(AttendArgs a, int tiles) {
    typedef Parts<D, BITS> PT;
    constexpr bool JOIN = WAVES > 1;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.y, split = JOIN ? blockIdx.x % a.splits : 0, tile = JOIN ? blockIdx.x / a.splits : blockIdx.x * 4 + wave;
    if (tile >= tiles) return;
    Piece w;
    int token0 = 0, tokens = 1;
    const int per = (a.group + 15) / 16;
    if (a.list) {
        w = {__builtin_amdgcn_readfirstlane(sequence_of(a.t, tile / per)), tile % per};
        token0 = tile / per - first_row(a.t, w.sequence);
        if (!__builtin_amdgcn_readfirstlane(is_row_of(a.t, w.sequence, tile / per))) return;
    } else if (!a.t.offsets) {
        w = {tile / per, tile % per};
    } else {
        w = find_piece(a.t.sequences, tile, [&](int b) { return (int)(((int64_t)row_count(a.t, b) * a.group + 15) / 16); });
        if (w.sequence < 0) return;
        tokens = row_count(a.t, w.sequence);
    }
    const int b = w.sequence, length = length_of(a.t, b), all = row_count(a.t, b);
    const int row0 = first_row(a.t, b);
    const int index = w.piece * 16 + r;
    const bool real = index < tokens * a.group;
    const int token = token0 + index / a.group, head = h * a.group + index % a.group;
    // tokens that the row sees, and the least and the most that any of the tile does
    const bool causal = a.causal || a.list;
    int sees = causal ? min(max((int)min((int64_t)a.t.lengths[b], (int64_t)1 << 30) - all + token + 1, 0), length) : length;
    if (!real) sees = 0;
    int most = sees, least = real ? sees : length;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        most = max(most, __shfl_xor(most, d));
        least = min(least, __shfl_xor(least, d));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);

    QueryLoads<D, NS> f;
    load_queries<D, NS, BITS>(f, a, real, row0 + (int64_t)token, head);
    RowState<D> st;
    start_rows<D>(st);
    const int entries = a.list ? a.count : (most + kPage - 1) / kPage;
    const int from = (int)((int64_t)entries * split / a.splits), to = (int)((int64_t)entries * (split + 1) / a.splits);
    const int32_t *const list = a.list ? a.list + ((row0 + (int64_t)token0) * a.c.heads + h) * a.count : nullptr;
    ScoresAt scores = {};
    if constexpr (USE == kOnceAndScores) {  // of one token's queries, all in one tile
        const int64_t wide = (int64_t)a.t.blocks * a.group * kPage * 4;  // bytes of a token and head
        scores.buffer = __builtin_amdgcn_make_buffer_rsrc((char *)a.scores + ((int64_t)row0 * a.c.heads + h) * wide, 0, (int)wide, 0x00020000);
        scores.lane = r % C < a.group ? (r % C * kPage + q * 16 + C / 4 * (r / C) * 4) * 4 : INT32_MIN;
    }
    take_blocks<D, NS, C, BITS, USE>(st, a, f, real, {list, JOIN ? from + wave : from, WAVES, to}, b, h, C < 16 ? most : sees, least, most, length, scores);

    auto out_row = [&](int r) {
        const int i = w.piece * 16 + r;
        return i < tokens * a.group ? (row0 + (int64_t)(token0 + i / a.group)) * a.heads_q + h * a.group + i % a.group : -1;
    };
    if constexpr (JOIN) {
        extern __shared__ __attribute__((aligned(16))) char lds[];  // a JoinLds<WAVES>
        JoinLds<WAVES> &s = *reinterpret_cast<JoinLds<WAVES> *>(lds);
        join_waves<D, NS, WAVES, C, BITS>(st, s, a, split, out_row);
        if constexpr (USE == kOnceAndScores) {
            if (a.splits > 1) return;
            __syncthreads();
            weigh_places<C, 1024>(a, b, h, threadIdx.x * 4, length, [&](int g) { return row_ends(s.top[0][g], s.all[0][g]); });
        }
    } else {
        const float total = sum_of_row<C>(st.sum);
        const int64_t to = out_row(r);
        if constexpr (USE == kOnceAndScores) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // the scores are other lanes' stores
            weigh_places<C, 256>(a, b, h, lane * 4, length, [&](int g) {
                const int top = __builtin_amdgcn_readlane(__builtin_bit_cast(int, st.top), g), all = __builtin_amdgcn_readlane(__builtin_bit_cast(int, total), g);
                return row_ends(__builtin_bit_cast(float, top), __builtin_bit_cast(float, all));
            });
        }
        if (to < 0) return;
#pragma unroll
        for (int p = 0; p < PT::kCount; p++) {
            const int W = PT::width(p), t0 = PT::base(p) / 16;
#pragma unroll
            for (int d = 0; d < W / 4; d += 8) {
                float x[8];
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = st.acc[t0 + (d + k) % (W / 16)][(d + k) / (W / 16)];
                put8<NS>(a, to, 0, D, PT::base(p) + q * (W / 4) + d, x, total);
            }
        }
        if (q == 0) put_sums(a, to, 0, D, st.top, total);
    }
}

// A wavefront joins the splits of one row and head: at most 64, a lane for each one's maximum and sum.
template <int D, int NS>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a) {
    typedef typename ElementOf<NS>::type E;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= (int64_t)a.t.rows * a.heads_q) return;
    // rows that are no sequence's have no parts and are not written
    const int token = (int)(row / a.heads_q);
    const bool real = !a.t.offsets || (token >= a.t.offsets[0] && token < a.t.offsets[a.t.sequences]);
    const float *const ends = a.part + (int64_t)a.t.rows * a.heads_q * a.splits * D + row * a.splits * 2;
    float top = lane < a.splits ? ends[lane * 2] : -INFINITY;
    float sum = lane < a.splits ? ends[lane * 2 + 1] : 0;
    float most = top;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    const float weight = __builtin_amdgcn_exp2f(top - (most > -INFINITY ? most : 0.0f));
    float total = sum * weight;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
    constexpr int kEach = D >= 128 ? D / 64 : 2;  // elements of a lane: 2, 3 or 4
    const int at = lane * kEach;
    float x[kEach];
#pragma unroll
    for (int k = 0; k < kEach; k++) x[k] = 0;
    for (int s0 = 0; s0 < a.splits; s0 += 8) {  // 8 parts on their way at once
        float part[8][kEach];
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int k = 0; k < kEach; k++) part[i][k] = a.part[(row * a.splits + min(s0 + i, a.splits - 1)) * D + min(at, D - kEach) + k];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int w = __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), min(s0 + i, kMaxSplits - 1));
            const float by = s0 + i < a.splits ? __builtin_bit_cast(float, w) : 0.0f;
#pragma unroll
            for (int k = 0; k < kEach; k++) x[k] += by * part[i][k];
        }
    }
    const float by = total == 0 ? 0.0f : 1.0f / total;
    if (!real) return;
    if (at < D) {
#pragma unroll
        for (int k = 0; k < kEach; k++) ((E *)a.out)[row * D + at + k] = (E)(x[k] * by);
    }
    if (lane == 0 && a.lse) a.lse[row] = (most + __builtin_amdgcn_logf(total)) * 0.6931471805599453f;
    if (lane == 0 && a.ends) *reinterpret_cast<f32x2 *>(a.ends + row * 2) = f32x2{most, total};
}
