// The choice of blocks, on the device: scores of a row's blocks, and the best of them.
#pragma once
#include "select.h"

constexpr uint32_t kOwnKey = 0xFFFFFFFFu;        // the row's own block
constexpr uint32_t kBoundlessKey = 0xFFFFFFFEu;  // a block without bounds; every other score is lower

// score 2^power in an order that unsigned numbers have.  As a float32 it would pass the largest one (scores lie below 2^22, powers go
// up to 121), so the powers of two are added: the bits of |score| without two of mantissa, which are 0, on 2^21 for a binade.
__device__ inline uint32_t score_key(int score, int power) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, (float)abs(score)) >> 2;
    const uint32_t size = score ? bits + ((uint32_t)(power + 127) << 21) : 0;  // below 2^30
    return score < 0 ? (1u << 30) - size : (1u << 30) + size;
}

// Tokens of a sequence that can share a tile of 16 queries
__device__ __host__ inline int tokens_a_tile(int group) { return group >= 16 ? 1 : 16 / group; }

// What the wavefronts of a workgroup need of LDS to score
template <int WAVES>
struct ScoreLds {
    float top[WAVES][16];
    int score[WAVES][16][17];
};

// LDS of one wavefront is written and read in order; this keeps the compiler to it.
__device__ inline void wave_lds() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

__device__ inline int max_of_row16(int x) {  // over the 16 lanes of a row
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x128, 0xF, 0xF, false));  // row_ror: 8, 4, 2, 1
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x124, 0xF, 0xF, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x122, 0xF, 0xF, false));
    return max(x, __builtin_amdgcn_update_dpp(x, x, 0x121, 0xF, 0xF, false));
}

// Tokens [token0, token0 + tokens) of sequence b and one head; place0: the place of its row 0.
struct Scored {
    int b, h, token0, tokens, place0, length;
    int64_t row0;
};

// keys[token * stride + block] of blocks [from, to), as far as a token's own block: scores in an order that unsigned numbers have,
// 0 for a block that is none.
//
// score = max over the queries of sum_j max(u_j, 0) hi_j + min(u_j, 0) lo_j: one sum over 2 D channels of 8-bit products, which
// the matrix cores make of 16 blocks x 16 (token, query) pairs at once; it is a whole number below 2^22 and is compared with others
// exactly, whatever the blocks' powers of two.  What bounds it is the bounds' bytes, 2 D a block, and how many of them are on
// their way: a wavefront asks for those of several tiles of 16 blocks before it works on the first.  WHOLE: more than 16 queries,
// which fill several tiles.
template <int D, int NS, int WAVES, bool WHOLE>
__device__ inline void score_blocks(const SelectArgs &a, const Scored &s, int from, int to, uint32_t *keys, int64_t stride,
                                    ScoreLds<WAVES> &lds) {
    typedef typename ElementOf<NS>::type E;
    constexpr int kSteps = 2 * D / 64, U = D <= 64 ? 8 : D <= 128 ? 4 : 2;
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ways = WHOLE ? (a.group + 15) / 16 : 1;
    const int token = WHOLE ? 0 : r / a.group;

    // the 16 dimensions of a step: D is a multiple of 32, so they are all of the upper or all of the lower bounds
    constexpr int kOwn = D % 64 ? kSteps : D / 64;  // steps with dimensions of their own
    Eight<NS> x[2 * kOwn];
    auto query = [&](int way) {
        const int g = WHOLE ? way * 16 + r : r % a.group;
        const bool real = token < s.tokens && g < a.group;
        const E *const at = (const E *)a.queries + (real ? (s.row0 + s.token0 + token) * a.q_row + (s.h * a.group + g) * a.q_head : 0);
#pragma unroll
        for (int n = 0; n < 2 * kOwn; n++) x[n] = load8<NS>(at + ((n >> 1) * 64 + q * 16) % D + (n & 1) * 8, real);
    };
    // the largest magnitude of a token's queries; its exponent becomes 6.  Queries that are not finite count as zeros.
    float top = 0;
    bool finite = true;
    auto look_at = [&] {
#pragma unroll
        for (int n = 0; n < 2 * kOwn; n++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = (float)x[n][i];
                finite &= (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) != 0x7F800000u;
                top = fmaxf(top, fabsf(v));
            }
    };
    for (int way = ways - 1; way > 0; way--) {
        query(way);
        look_at();
    }
    query(0);
    look_at();
    if (!finite) top = INFINITY;
    top = max_over_quads(top);
    if (q == 0) lds.top[wave][r] = top;
    wave_lds();
    const int first_column = WHOLE ? 0 : token * a.group, columns = WHOLE ? 16 : a.group;
    for (int i = first_column; i < min(first_column + columns, 16); i++) top = fmaxf(top, lds.top[wave][i]);
    const int e = max((int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127 - 6, -100);
    const float unit = top < INFINITY ? __builtin_bit_cast(float, (uint32_t)(127 - e) << 23 | (uint32_t)a.turned << 31) : 0.0f;
    i32x4 u[kSteps];
    auto ask = [&] {  // the queries in x as the products' operand
#pragma unroll
        for (int step = 0; step < kSteps; step++) {
            const bool upper = step * 64 + q * 16 < D;
            u[step] = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float y = unit != 0.0f ? (float)x[2 * (step % kOwn) + (i >> 3)][i & 7] : 0.0f;
                // cut to 127, and to the sign that these bounds are for
                const int v = (int)__builtin_amdgcn_fmed3f(__builtin_rintf(y * unit), upper ? 0.0f : -127.0f, upper ? 127.0f : 0.0f);
                u[step][i >> 2] |= (v & 255) << (8 * (i & 3));
            }
        }
    };
    ask();

    int page[U], next[U];
    auto look_up = [&](int first0, int(&p)[U]) {
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int block = first0 + k * WAVES * 16 + r;
            p[k] = a.t.table[s.b * a.t.table_stride + min(block, a.t.blocks - 1)];
        }
    };
    if (from >= to) return;
    if (a.c.pages == 0) {  // no bounds to read: a token's own block is all there is to choose
        for (int i = threadIdx.x; i < s.tokens * (to - from); i += WAVES * 64) {
            const int token = i / (to - from), block = from + i % (to - from);
            keys[token * stride + block] = block == min(s.place0 + s.token0 + token, s.length - 1) / kPage ? kOwnKey : 0;
        }
        return;
    }
    look_up(from + wave * 16, next);
    for (int first0 = from + wave * 16; first0 < to; first0 += WAVES * 16 * U) {
        i32x4 edges[U][kSteps];
        int power[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            page[k] = first0 + k * WAVES * 16 + r < to && next[k] < a.c.pages ? next[k] : -1;
            // a block without a page is loaded from page 0 and not looked at: loads behind a branch would wait for each other
            const int64_t at = (int64_t)max(page[k], 0) * a.c.heads + s.h;
            power[k] = a.c.bound_scales[at];
#pragma unroll
            for (int step = 0; step < kSteps; step++)
                edges[k][step] = *reinterpret_cast<const i32x4 *>(a.c.bounds + at * (2 * D) + q * 16 + step * 64);
        }
        look_up(first0 + WAVES * 16 * U, next);
        __builtin_amdgcn_sched_barrier(0);  // all of these are asked for before the first is worked on
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int first = first0 + k * WAVES * 16;
            if (first >= to) break;
            i32x4 best = {INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN};
            for (int way = 0; way < ways; way++) {
                if (WHOLE) {
                    query(way);
                    ask();
                }
                i32x4 sum = {0, 0, 0, 0};
#pragma unroll
                for (int step = 0; step < kSteps; step++) sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(edges[k][step], u[step], sum, 0, 0, 0);
                // columns that are no query of the first token: their zeros are no score
                const bool none = WHOLE ? way * 16 + r >= a.group : s.tokens == 1 && r >= a.group;
#pragma unroll
                for (int i = 0; i < 4; i++) best[i] = max(best[i], none ? INT32_MIN : sum[i]);
            }
            auto key_of = [&](int score, int block, int token, int page, int power) {
                // a place below 0 has no own block and makes no choice
                const int own = min(s.place0 + s.token0 + token, s.length - 1) / kPage;
                if (block >= to || block > own) return;
                uint32_t key = 0;
                if (page >= 0) key = power == kBoundless ? kBoundlessKey : score_key(score, power);
                if (block == own) key = kOwnKey;
                keys[token * stride + block] = key;
            };
            if (WHOLE || s.tokens == 1) {
#pragma unroll
                for (int i = 0; i < 4; i++) best[i] = max_of_row16(best[i]);
                // lane (q, r < 4) has block 4 q + r, whose page lane r' = 4 q + r looked up
                const int score = r == 0 ? best[0] : r == 1 ? best[1] : r == 2 ? best[2] : best[3], from_lane = (q * 4 + (r & 3));
                const int p = __shfl(page[k], from_lane), w = __shfl(power[k], from_lane);
                if (r < 4) key_of(score, first + from_lane, 0, p, w);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) lds.score[wave][q * 4 + i][r] = best[i];
                wave_lds();
                for (int i0 = 0; i0 < s.tokens * 16; i0 += 64) {
                    const int i = i0 + lane, token = i >> 4;
                    const int p = __shfl(page[k], i & 15), w = __shfl(power[k], i & 15);
                    if (token < s.tokens) {
                        int score = INT32_MIN;
                        for (int g = 0; g < a.group; g++) score = max(score, lds.score[wave][i & 15][token * a.group + g]);
                        key_of(score, first + (i & 15), token, p, w);
                    }
                }
                wave_lds();
            }
        }
    }
}

template <int WAVES>
struct ChooseLds {
    alignas(16) int count[4][256];  // read four at a time
    uint32_t differ;
    int more[WAVES], equal[WAVES];
};

__device__ inline int sum_up_to_lane(int x) {  // over lanes 0 .. own
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr: 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast: 15 into rows 1 and 3, 31 into rows 2 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}

__device__ inline uint32_t or_of_wave(uint32_t x) {
    x |= __builtin_amdgcn_update_dpp(x, x, 0x128, 0xF, 0xF, false);
    x |= __builtin_amdgcn_update_dpp(x, x, 0x124, 0xF, 0xF, false);
    x |= __builtin_amdgcn_update_dpp(x, x, 0x122, 0xF, 0xF, false);
    x |= __builtin_amdgcn_update_dpp(x, x, 0x121, 0xF, 0xF, false);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = a[0] | a[1];
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return b[0] | b[1];
}

// The last key, which is a row's own block's, and the largest others of n keys up to `count` in all, 0 excepted, ties to the lower
// one, by WAVES wavefronts together: counts of 8 bits at a time, from the highest in which keys differ, give the last key that
// is taken, then put(place, index) in ascending order.  Returns how many there are.
template <int WAVES, class F>
__device__ inline int choose(const uint32_t *keys, int n, int count, ChooseLds<WAVES> &s, F put) {
    const int lane = threadIdx.x & 63, tid = threadIdx.x % (64 * WAVES), wave = tid >> 6;
    constexpr int kThreads = 64 * WAVES;
    if (n == 0) return 0;
    auto sync = [] {
        if constexpr (WAVES == 1) wave_lds();
        else __syncthreads();
    };
    // up to 8 keys a thread are held in registers
    constexpr int kHeld = 8;
    const bool held = n <= kHeld * kThreads;
    uint32_t mine[kHeld];
    if (held) {
#pragma unroll
        for (int k = 0; k < kHeld; k++) mine[k] = keys[min(tid + k * kThreads, n - 1)];
    }
    auto each = [&](int n, auto f) {  // of keys [0, n)
        if (held) {
#pragma unroll
            for (int k = 0; k < kHeld; k++)
                if (tid + k * kThreads < n) f(mine[k]);
        } else {
            for (int i = tid; i < n; i += kThreads) f(keys[i]);
        }
    };
    uint32_t least = 0;  // keys above are taken
    int ties = 0;        // and so many of those equal to it
    if (n > count) {
        const int others = n - 1;
        int need = count - 1;
        for (int i = tid; i < 1024; i += kThreads) s.count[0][i] = 0;
        if (tid == 0) s.differ = 0;
        sync();
        const uint32_t any = keys[0];
        uint32_t differ = 0;
        each(others, [&](uint32_t key) { differ |= key ^ any; });
        differ = or_of_wave(differ);
        if (lane == 0) atomicOr(&s.differ, differ);
        sync();
        differ = s.differ;
        const int bits = differ ? 32 - __builtin_clz(differ) : 0;  // of a key that may differ, the lowest
        int shift = bits;
        uint32_t prefix = bits < 32 ? any >> bits : 0;  // of the keys from bit `shift` on
        for (int pass = 0; shift > 0 && need > 0; pass++) {
            const int low = shift > 8 ? shift - 8 : 0;
            const uint32_t mask = (1u << (shift - low)) - 1;
            each(others, [&](uint32_t key) {
                if (shift >= 32 || key >> shift == prefix) atomicAdd(&s.count[pass][key >> low & mask], 1);
            });
            sync();
            // lane l has the value 255 - 4 l and the three below it
            const i32x4 c = *reinterpret_cast<const i32x4 *>(&s.count[pass][252 - 4 * lane]);
            const int sum = c[0] + c[1] + c[2] + c[3], upto = sum_up_to_lane(sum);
            int above = upto - sum, value = 0, left = 0;
            const uint64_t here = __ballot(above < need && upto >= need);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (above < need && above + c[3 - i] >= need) {
                    value = 255 - 4 * lane - i;
                    left = need - above;
                }
                above += c[3 - i];
            }
            const int at = __builtin_ctzll(here);  // there are more keys than are needed
            prefix = prefix << (shift - low) | (uint32_t)__builtin_amdgcn_readlane(value, at);
            need = __builtin_amdgcn_readlane(left, at);
            shift = low;
        }
        // all of a key is in prefix now, unless none is needed
        least = need > 0 ? prefix : 0xFFFFFFFEu;
        ties = need;
        if (least == 0) ties = 0;  // fewer keys than are asked for: all of them
    }
    int more = 0, equal = 0;  // larger and equal ones so far
    auto place = [&](int i0, uint32_t key) {  // keys i0 + tid: all threads together
        const int i = i0 + tid;
        const bool own = i == n - 1, gt = i < n && (key > least || own), eq = key == least && i < n - 1;
        const uint64_t gts = __ballot(gt), eqs = __ballot(eq), before = (1ull << lane) - 1;
        int m = more + __popcll(gts & before), e = equal + __popcll(eqs & before);
        if constexpr (WAVES == 1) {
            more += __popcll(gts);
            equal += __popcll(eqs);
        } else {
            __syncthreads();
            if (lane == 0) {
                s.more[wave] = __popcll(gts);
                s.equal[wave] = __popcll(eqs);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < WAVES; k++) {
                if (k < wave) {
                    m += s.more[k];
                    e += s.equal[k];
                }
                more += s.more[k];
                equal += s.equal[k];
            }
        }
        if (gt || (eq && e < ties)) put(m + min(e, ties), i);
    };
    if (held) {
#pragma unroll
        for (int k = 0; k < kHeld; k++)
            if (k * kThreads < n) place(k * kThreads, mine[k]);
    } else {
        for (int i0 = 0; i0 < n; i0 += kThreads) place(i0, i0 + tid < n ? keys[i0 + tid] : 0);
    }
    return more + min(equal, ties);
}

// Where a row stands in its sequence, and of how many blocks it chooses; not real: the row is no sequence's
struct Standing {
    int b, token, place0, length, blocks;
    bool real;
};
__device__ inline Standing standing_of(const Tokens &t, int row) {
    Standing s;
    s.b = sequence_of(t, row);
    s.token = row - first_row(t, s.b);
    s.length = length_of(t, s.b);
    s.place0 = (int)min((int64_t)t.lengths[s.b], (int64_t)1 << 30) - row_count(t, s.b);
    const int place = min(s.place0 + s.token, s.length - 1);
    s.blocks = place < 0 ? 0 : place / kPage + 1;
    s.real = __builtin_amdgcn_readfirstlane(is_row_of(t, s.b, row));
    return s;
}
