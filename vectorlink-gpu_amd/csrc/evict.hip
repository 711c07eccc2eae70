// Eviction from a cache in 8 bits: of every sequence and head the tokens that count most stay.
//
// What stays behind the new length moves into places before it that got free, so a step that gives up 64 tokens moves at most 64
// a head, where closing the gaps in order would move nearly all of them; sources (behind the new length) and destinations
// (before it) are apart, so pages are made in any order.  A workgroup for a sequence and head, or several in
// six launches for a long one, ranks its tokens and lists free places and what moves there; a launch over pages and heads moves.
#include "cache8.h"

namespace {

struct EvictArgs {
    CacheView c;
    Tokens t;
    int keep, recent;
    int most;           // entries of a list: pairs of a sequence and head, at most
    int pages;          // of keep tokens
    int chunks;         // workgroups that share a sequence and head
    int together;       // pages of a workgroup of evict_move_kernel
    int32_t *lengths;   // new ones
    // per sequence and head:
    int64_t *holes, *movers;  // [most] free places and the places whose tokens move there, both ascending, as the token's place in the
                              // cache: (page * heads + head) * 64 + token, negative: on no page
    int32_t *starts;          // [pages + 1] the first hole of every block
    int64_t *border;          // [2] page and head that the new length lies in, and its scales before any change
    // where workgroups share one, per sequence and head:
    int32_t *latest;          // [chunks, 2] the latest position, tokens on pages
    uint32_t *bins;           // [kBinWords]: [3, kBins], and what was found with each of the three: prefix and need
    int32_t *counts;          // [chunks * kSharedWaves, 4]
};

constexpr int kDigit = 11;  // bits of a key that one pass over the weights tells apart
constexpr int kBins = 1 << kDigit, kBinWords = 3 * kBins + 8;
// wavefronts of a workgroup and blocks of a wavefront: where one workgroup has all of a short or a long sequence and head, and where several share
constexpr int kShortWaves = 8, kShortBlocks = 16, kLongWaves = 16, kLongBlocks = 32, kSharedWaves = 16, kSharedBlocks = 8;
constexpr int kChunkBlocks = kSharedWaves * kSharedBlocks;

// Larger stays first; NaN is last.  vl_float_key puts +NaN above all.
__device__ inline uint32_t rank_key(float weight, bool late) { return late ? ~0u : weight != weight ? 0u : vl_float_key(weight); }

// What a launch does of the ranking.  All of it where a workgroup can hold the weights of a sequence and head; else several share them
// and every step that needs what others found is a launch of its own, which reads its part of the weights again.
enum Stage { kWhole, kLatest, kFirstDigit, kSecondDigit, kLastDigit, kCount, kList };

// The digit, from the highest down, at which `need` keys have been passed: need becomes how many of that digit are wanted.  All of a
// workgroup of W wavefronts take part, each thread with its share of the bins, which may be changed once it returns.
template <int W>
struct DigitLds {
    int sum[W];
    int digit, need;
};
template <int W>
__device__ inline uint32_t digit_of(const uint32_t *bins, int &need, DigitLds<W> &s) {
    constexpr int kEach = kBins / (W * kWave);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, top = kBins - 1 - kEach * threadIdx.x;
    int n[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        n[i] = bins[top - i];
        sum += n[i];
    }
    int upto = sum;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int other = __shfl_up(upto, d);
        if (lane >= d) upto += other;
    }
    if (lane == kWave - 1) s.sum[wave] = upto;
    if (threadIdx.x == 0) s.digit = s.need = 0;
    __syncthreads();
    for (int i = 0; i < wave; i++) upto += s.sum[i];
    int above = upto - sum;
    if (above < need && upto >= need) {  // one thread's
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            if (above < need && above + n[i] >= need) {
                s.digit = top - i;
                s.need = need - above;
            }
            above += n[i];
        }
    }
    __syncthreads();
    need = s.need;
    const int digit = s.digit;
    __syncthreads();
    return digit;
}

// A wavefront has K blocks at most, one after the other, the weights and positions of a block a lane each: what bounds this are the loads,
// all of them on their way at once, and 3 rounds over 2,048 bins in LDS.  64 sequences of 4,160 tokens with 8 heads:
// 21 us in one launch (27 with 4 wavefronts or 16 of as many blocks more or less); one of 131,072 in six, 49 us (56 where every launch
// finds all digits from the bins).
template <int STAGE, int W, int K>
__global__ __launch_bounds__(W * 64) void evict_choose_kernel(EvictArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t s_bin[kBins];
    __shared__ int s_latest[W][2], s_count[W][4];
    __shared__ DigitLds<W> s_digit;
    constexpr int kThreads = W * 64;
    constexpr bool whole = STAGE == kWhole;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t list = whole ? blockIdx.x : blockIdx.x / a.chunks;
    const int chunk = whole ? 0 : (int)(blockIdx.x % a.chunks);
    const int h = (int)(list % a.c.heads), b = (int)(list / a.c.heads);
    const int length = length_of(a.t, b);
    int32_t *const starts = a.starts + list * (a.pages + 1);
    uint32_t *const bins = a.bins + list * kBinWords;
    const bool last_stage = whole || STAGE == kList;
    if (length <= a.keep) {
        if (last_stage && chunk == 0) {
            for (int i = threadIdx.x; i <= a.pages; i += kThreads) starts[i] = 0;
            if (h == 0 && threadIdx.x == 0) a.lengths[b] = length;
        }
        return;
    }
    if (a.c.pages == 0) {  // nothing to look at
        if (last_stage && chunk == 0) {
            for (int i = threadIdx.x; i <= a.pages; i += kThreads) starts[i] = 0;
            if (h == 0 && threadIdx.x == 0) a.lengths[b] = 0;
        }
        return;
    }
    const int blocks = (length + kPage - 1) / kPage, first = whole ? 0 : chunk * kChunkBlocks;
    if (first >= blocks) return;
    const int here = whole ? blocks : min(blocks - first, kChunkBlocks), each = (here + W - 1) / W;
    const int from = first + min(wave * each, here), n = min(each, first + here - from);  // this wavefront's blocks
    // lane k has the page of block k
    const int64_t my_page = lane < n ? page_of(a.t, a.c, b, from + lane) : -1;
    const uint64_t paged = __ballot(my_page >= 0);
    float weight[K];
    int position[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        if (k >= n) continue;
        // of a block without a page, and behind the length: whatever is there, and nothing is made of it
        const int64_t at = ((int64_t)max(__builtin_amdgcn_readlane((int)my_page, k), 0) * a.c.heads + h) * kPage + lane;
        if (STAGE != kLatest) weight[k] = a.c.weights[at];
        position[k] = a.c.positions[at];
    }
    auto there = [&](int k) { return (paged >> k & 1) && (from + k) * kPage + lane < length; };

    int newest = INT32_MIN, real = 0;
    if constexpr (whole || STAGE == kLatest) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (k >= n || !there(k)) continue;
            newest = max(newest, position[k]);
            real++;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            newest = max(newest, __shfl_xor(newest, d));
            real += __shfl_xor(real, d);
        }
        if (lane == 0) {
            s_latest[wave][0] = newest;
            s_latest[wave][1] = real;
        }
        if constexpr (STAGE == kLatest) {
            if (chunk == 0)
                for (int i = threadIdx.x; i < 3 * kBins; i += kThreads) bins[i] = 0;
        }
        __syncthreads();
        newest = INT32_MIN, real = 0;
#pragma unroll
        for (int i = 0; i < W; i++) {
            newest = max(newest, s_latest[i][0]);
            real += s_latest[i][1];
        }
        if constexpr (STAGE == kLatest) {
            if (threadIdx.x == 0) {
                a.latest[(list * a.chunks + chunk) * 2] = newest;
                a.latest[(list * a.chunks + chunk) * 2 + 1] = real;
            }
            return;
        }
    } else {
        const int chunks = (blocks + kChunkBlocks - 1) / kChunkBlocks;
        for (int i = lane; i < chunks; i += 64) {
            newest = max(newest, a.latest[(list * a.chunks + i) * 2]);
            real += a.latest[(list * a.chunks + i) * 2 + 1];
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            newest = max(newest, __shfl_xor(newest, d));
            real += __shfl_xor(real, d);
        }
    }
    const int kept = min(a.keep, real);
    if (last_stage && h == 0 && chunk == 0 && threadIdx.x == 0) a.lengths[b] = kept;
    if (kept == 0) {
        if (last_stage && chunk == 0)
            for (int i = threadIdx.x; i <= a.pages; i += kThreads) starts[i] = 0;
        return;
    }
    uint32_t key[K];
#pragma unroll
    for (int k = 0; k < K; k++)
        if (k < n) key[k] = rank_key(weight[k], (int64_t)position[k] > (int64_t)newest - a.recent);

    // the key of the last that stays, 11, 11 and 10 bits at a time, and how many with that key do
    constexpr int kDigits = whole || STAGE > kLastDigit ? 3 : STAGE - kFirstDigit;  // that are known, or are found here
    int need = kept;
    uint32_t prefix = 0;
    constexpr int kBitsOf[3] = {kDigit, kDigit, 32 - 2 * kDigit};
    if constexpr (!whole && kDigits > 0) {
        constexpr int told = STAGE == kList ? kDigits : kDigits - 1;  // by the launches before this one
        if constexpr (told > 0) {
            prefix = bins[3 * kBins + 2 * told - 2];
            need = (int)bins[3 * kBins + 2 * told - 1];
        }
        if constexpr (told < kDigits) {
            prefix = prefix << kBitsOf[told] | digit_of(bins + told * kBins, need, s_digit);
            if (chunk == 0 && threadIdx.x == 0) {
                bins[3 * kBins + 2 * kDigits - 2] = prefix;
                bins[3 * kBins + 2 * kDigits - 1] = (uint32_t)need;
            }
        }
    }
    auto count_digit = [&](int d) {  // into the bins in LDS, which are 0
        const int bits = kBitsOf[d], low = d < 2 ? 32 - (d + 1) * kDigit : 0;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (k >= n || !there(k)) continue;
            if (d == 0 || key[k] >> (low + bits) == prefix) atomicAdd(&s_bin[key[k] >> low & ((1u << bits) - 1)], 1u);
        }
    };
    auto clear = [&] {
        for (int i = threadIdx.x; i < kBins; i += kThreads) s_bin[i] = 0;
    };
    if constexpr (whole) {
#pragma unroll
        for (int d = 0; d < 3; d++) {
            clear();
            __syncthreads();
            count_digit(d);
            __syncthreads();
            prefix = prefix << kBitsOf[d] | digit_of(s_bin, need, s_digit);
        }
    } else if constexpr (STAGE <= kLastDigit) {
        clear();
        __syncthreads();
        count_digit(kDigits);
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads)
            if (s_bin[i]) atomicAdd(&bins[kDigits * kBins + i], s_bin[i]);
        return;
    }
    // keys above `prefix` stay, and the first `need` of those equal to it: how many of both there are, before and behind the new length.
    // Asked of the keys both times: masks of 32 blocks held from the counts to the lists spill vector registers too (one sequence of 9,000
    // 40 us with both launches, 28 without them; with 16 blocks 1 us more).  As it is none spills, but the blocks' pages and ends are scalars of
    // unrolled loops, of which the compiler keeps 216 (with 16 blocks 88) in lanes of vector registers.
    auto more_of = [&](int k) { return __ballot(there(k) && key[k] > prefix); };
    auto equal_of = [&](int k) { return __ballot(there(k) && key[k] == prefix); };
    auto front = [&](int block) {  // the places of a block before the new length
        const int before = min(max(kept - block * kPage, 0), kPage);
        return before == kPage ? ~0ull : (1ull << before) - 1;
    };
    int count[4] = {0, 0, 0, 0};
    if constexpr (whole || STAGE == kCount) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (k >= n) continue;
            const uint64_t f = front(from + k), more = more_of(k), equal = equal_of(k);
            count[0] += __popcll(more & f);
            count[1] += __popcll(more & ~f);
            count[2] += __popcll(equal & f);
            count[3] += __popcll(equal & ~f);
        }
        int32_t *const to = whole ? s_count[wave] : a.counts + ((list * a.chunks + chunk) * W + wave) * 4;
        if (lane < 4) to[lane] = lane == 0 ? count[0] : lane == 1 ? count[1] : lane == 2 ? count[2] : count[3];
        if constexpr (STAGE == kCount) return;
        __syncthreads();
    }
    // of the wavefronts before this one
    count[0] = count[1] = count[2] = count[3] = 0;
    if constexpr (whole) {
        for (int i = 0; i < wave; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) count[k] += s_count[i][k];
    } else {
        const int32_t *const all = a.counts + list * a.chunks * (W * 4);
        for (int i = lane; i < chunk * W + wave; i += 64)
#pragma unroll
            for (int k = 0; k < 4; k++) count[k] += all[i * 4 + k];
#pragma unroll
        for (int d = 1; d < 64; d <<= 1)
#pragma unroll
            for (int k = 0; k < 4; k++) count[k] += __shfl_xor(count[k], d);
    }
    int tie = count[2] + count[3];
    int free = min(from * kPage, kept) - count[0] - min(need, count[2]);
    int moves = count[1] + min(need, tie) - min(need, count[2]);
    int64_t *const holes = a.holes + list * a.most, *const movers = a.movers + list * a.most;
    const uint64_t before = (1ull << lane) - 1;
#pragma unroll
    for (int k = 0; k < K; k++) {
        if (k >= n) continue;
        const uint64_t more = more_of(k), equal = equal_of(k);
        const int block = from + k, ties = __popcll(equal);
        uint64_t in = more | equal;
        if (tie + ties > need) in = more | __ballot((equal >> lane & 1) && tie + __popcll(equal & before) < need);
        tie += ties;
        const uint64_t f = front(block), hole = ~in & f, moving = in & ~f;
        if (lane == 0 && block < a.pages) starts[block] = free;
        if (hole | moving) {
            const int page = __builtin_amdgcn_readlane((int)my_page, k);
            const int64_t token = page < 0 ? -1 : ((int64_t)page * a.c.heads + h) * kPage + lane;
            // within the lists whatever the launches before found: weights that another stream changes meanwhile end in a wrong choice only
            const int hole_at = free + __popcll(hole & before), mover_at = moves + __popcll(moving & before);
            if ((hole >> lane & 1) && (uint32_t)hole_at < (uint32_t)a.most) holes[hole_at] = token;
            if ((moving >> lane & 1) && (uint32_t)mover_at < (uint32_t)a.most) movers[mover_at] = token;
            free += __popcll(hole);
            moves += __popcll(moving);
        }
    }
    // the block that the new length ends: of the pages behind it, none has a hole
    const int ended = (kept - 1) / kPage;
    if (ended >= from && ended < from + n)
        for (int i = ended + 1 + lane; i <= a.pages; i += 64) starts[i] = free;
    if (kept / kPage == from + lane && lane < n) {
        const int64_t unit = my_page * a.c.heads + h;
        a.border[list * 2] = my_page < 0 ? -1 : unit;
        a.border[list * 2 + 1] = my_page < 0 ? 0 : a.c.scales[unit];
    }
}

// A workgroup fills the free places of `together` pages of one head, as many whole pages at a time as have at most 64 of them.  A thread
// takes 16 dimensions of a moving token's key, 16 bytes, and 4 of its value, a byte of each of 4 words: neighbours' words lie side by side,
// so that a line is written a few times and not once a byte (64 sequences of 4,160 tokens with 8 heads, 64 moves each: 68 us with 16
// dimensions of a value a thread, 42 with 4).
constexpr int kMostTogether = 64;
template <int D>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    constexpr int kKeys = D / 16, kValues = D / 4;  // threads of a token
    constexpr int kKeyTurns = (kKeys * kPage + 255) / 256, kValueTurns = (kValues * kPage + 255) / 256;
    __shared__ int s_starts[kMostTogether + 1];
    __shared__ int64_t s_page[kMostTogether];  // of the pages: page and head, -1: none or nothing to fill
    __shared__ uint32_t s_was[kMostTogether], s_top[kMostTogether][2], s_now[kMostTogether][2], s_steps[kMostTogether][2], s_spoilt[kMostTogether];
    __shared__ int s_grown;
    __shared__ int s_at[kPage];                // of the moving tokens: which page they go to
    __shared__ int64_t s_to[kPage], s_source[kPage];  // and their places in the cache
    __shared__ uint32_t s_scales[kPage];
    const int groups = (a.pages + a.together - 1) / a.together;
    const int h = blockIdx.x % a.c.heads, group = blockIdx.x / a.c.heads % groups, b = blockIdx.x / a.c.heads / groups;
    const int64_t list = (int64_t)b * a.c.heads + h;
    const int block0 = group * a.together, pages = min(a.together, a.pages - block0);
    const int kept = a.lengths[b];
    if (threadIdx.x <= pages) s_starts[threadIdx.x] = min(max(a.starts[list * (a.pages + 1) + block0 + threadIdx.x], 0), a.most);
    __syncthreads();
    for (int p0 = 0, p1 = 0; p0 < pages; p0 = p1) {
        const int first = s_starts[p0];
        for (p1 = p0 + 1; p1 < pages && s_starts[p1 + 1] - first <= kPage;) p1++;
        const int n = min(s_starts[p1] - first, kPage);
        if (n <= 0) continue;
        if (threadIdx.x < kMostTogether) {
            s_top[threadIdx.x][0] = s_top[threadIdx.x][1] = 0;
            s_page[threadIdx.x] = -1;
            s_spoilt[threadIdx.x] = 0;
        }
        if (threadIdx.x == 0) s_grown = 0;
        __syncthreads();
        int64_t to = -1, source = 0;
        if (threadIdx.x < n) {
            const int i = threadIdx.x;
            to = a.holes[list * a.most + first + i];
            source = max(a.movers[list * a.most + first + i], (int64_t)0);  // it is on a page
            int p = p0;
            while (p + 1 < p1 && s_starts[p + 1] <= first + i) p++;
            s_at[i] = p;
            s_to[i] = to;
            s_source[i] = source;
            if (to >= 0) s_page[p] = to / kPage;  // the same for all of a page's
        }
        __syncthreads();
        // what moves, as codes
        u32x4 key[kKeyTurns], words[kValueTurns];
        uint32_t value[kValueTurns];
#pragma unroll
        for (int k = 0; k < kKeyTurns; k++) {  // behind the last token once more its bytes: no branch of a thread's own between loads
            const int u = k * 256 + threadIdx.x, i = min(u / kKeys, n - 1);
            if (k * 256 / kKeys < n) key[k] = *reinterpret_cast<const u32x4 *>(a.c.keys + s_source[i] * D + u % kKeys * 16);
        }
#pragma unroll
        for (int k = 0; k < kValueTurns; k++) {
            const int u = k * 256 + threadIdx.x, i = min(u / kValues, n - 1);
            if (k * 256 / kValues < n) words[k] = *reinterpret_cast<const u32x4 *>(a.c.values + ((s_source[i] >> 2) * D + u % kValues * 4) * 4);
        }
        if (threadIdx.x < n) {
            const int64_t unit = source / kPage;
            // the page of the border may be given another power while this one is made; its tokens behind the border are as they were
            s_scales[threadIdx.x] = unit == a.border[list * 2] ? (uint32_t)a.border[list * 2 + 1] : a.c.scales[unit];
            if (to >= 0) {
                a.c.weights[to] = a.c.weights[source];
                a.c.positions[to] = a.c.positions[source];
            }
        }
        if (threadIdx.x < p1 - p0) {
            const int64_t unit = s_page[p0 + threadIdx.x];
            s_was[p0 + threadIdx.x] = unit < 0 ? 0 : a.c.scales[unit];
        }
        __syncthreads();
        // the largest of every page, by the codes' magnitudes, whose order is that of their numbers
        auto largest = [](uint32_t word) {
            word &= 0x7F7F7F7Fu;
            return max(max(word & 255, word >> 8 & 255), max(word >> 16 & 255, word >> 24));
        };
        auto told = [&](int i, int which, uint32_t code) {
            if (code == kByteNaN) {
                s_spoilt[s_at[i]] = 1;
            } else {
                const float scale = which ? scale_of_values(s_scales[i]) : scale_of_keys(s_scales[i]);
                atomicMax(&s_top[s_at[i]][which], __builtin_bit_cast(uint32_t, four_numbers(code)[0] * scale));
            }
        };
#pragma unroll
        for (int k = 0; k < kKeyTurns; k++) {
            const int i = (k * 256 + threadIdx.x) / kKeys;
            if (i < n) told(i, 0, max(max(largest(key[k][0]), largest(key[k][1])), max(largest(key[k][2]), largest(key[k][3]))));
        }
#pragma unroll
        for (int k = 0; k < kValueTurns; k++) {  // 8 threads in a row are one token's
            const int i = (k * 256 + threadIdx.x) / kValues;
            if (k * 256 / kValues >= n) continue;
            const u32x4 v = words[k];
            const int turn = 8 * ((int)s_source[min(i, n - 1)] & 3);
            value[k] = (v[0] >> turn & 255) | (v[1] >> turn & 255) << 8 | (v[2] >> turn & 255) << 16 | (v[3] >> turn & 255) << 24;
            uint32_t top = i < n ? largest(value[k]) : 0;
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
            if (i < n && (threadIdx.x & 7) == 0) told(i, 1, top);
        }
        __syncthreads();
        if (threadIdx.x < 2 * kMostTogether) {
            const int p = threadIdx.x >> 1, which = threadIdx.x & 1;
            const uint32_t old = which ? byte_of_values(s_was[p]) : byte_of_keys(s_was[p]), now = max(old, fitting_byte(s_top[p][which]));
            s_now[p][which] = now;
            s_steps[p][which] = now - old;
            if (p >= p0 && p < p1 && s_page[p] >= 0) {
                if (now != old) s_grown = 1;
                uint8_t *const at = reinterpret_cast<uint8_t *>(a.c.scales + s_page[p]);
                at[which] = (uint8_t)now;
                if (which) at[2] = (uint8_t)(is_marked(s_was[p]) || s_spoilt[p]);
            }
        }
        __syncthreads();
        // what a page whose power grows holds already, up to the new length: places that are filled are overwritten below
        if (s_grown) {
            for (int p = p0; p < p1; p++) {
                const int64_t unit = s_page[p];
                if (unit < 0) continue;
                const int holds = min(kept - (block0 + p) * kPage, kPage);
                if (s_steps[p][0]) {
                    uint32_t *const at = reinterpret_cast<uint32_t *>(a.c.keys + unit * (kPage * D));
                    for (int i = threadIdx.x; i < holds * D / 4; i += 256) at[i] = four_codes(four_numbers(at[i]) * power_below(s_steps[p][0]));
                }
                if (s_steps[p][1]) {
                    uint32_t *const at = reinterpret_cast<uint32_t *>(a.c.values + unit * (kPage * D));
                    for (int i = threadIdx.x; i < (holds + 3) / 4 * D; i += 256) {
                        const int there = holds - i / D * 4;  // of the word's tokens
                        const uint32_t keep = there >= 4 ? 0 : ~0u << (8 * there), word = at[i];
                        at[i] = (four_codes(four_numbers(word) * power_below(s_steps[p][1])) & ~keep) | (word & keep);
                    }
                }
            }
            __syncthreads();
        }
        // powers are up to 2^237 apart: codes go by the difference in two steps, of which the second alone rounds or neither does
        auto again = [](uint32_t word, uint32_t from, uint32_t now) {
            const int up = (int)from - (int)now, half = up / 2;
            return four_codes(four_numbers(word) * power_of_byte((uint32_t)(127 + half)) * power_of_byte((uint32_t)(127 + up - half)));
        };
#pragma unroll
        for (int k = 0; k < kKeyTurns; k++) {
            const int u = k * 256 + threadIdx.x, i = u / kKeys;
            if (i >= n || s_to[i] < 0) continue;
            const uint32_t from = byte_of_keys(s_scales[i]), now = s_now[s_at[i]][0];
            if (from != now) {
#pragma unroll
                for (int w = 0; w < 4; w++) key[k][w] = again(key[k][w], from, now);
            }
            *reinterpret_cast<u32x4 *>(a.c.keys + s_to[i] * D + u % kKeys * 16) = key[k];
        }
#pragma unroll
        for (int k = 0; k < kValueTurns; k++) {
            const int u = k * 256 + threadIdx.x, i = u / kValues;
            if (i >= n || s_to[i] < 0) continue;
            const uint32_t from = byte_of_values(s_scales[i]), now = s_now[s_at[i]][1];
            if (from != now) value[k] = again(value[k], from, now);
            uint8_t *const at = a.c.values + ((s_to[i] >> 2) * D + u % kValues * 4) * 4 + (s_to[i] & 3);
#pragma unroll
            for (int e = 0; e < 4; e++) at[e * 4] = (uint8_t)(value[k] >> (8 * e));
        }
        __syncthreads();
    }
}

struct Layout {
    int64_t holes, movers, starts, border, latest, bins, counts, bytes;
    int64_t groups;
    int most, pages, chunks;
};
// Half of a sequence's places can be free or moving, and no more than stay.
Layout layout_of(const CacheView &c, const Tokens &t, int64_t keep) {
    Layout l;
    const int64_t lists = (int64_t)t.sequences * c.heads, half = (int64_t)t.blocks * kPage / 2;
    l.most = (int)(keep < half ? keep : half);
    const int64_t kept = keep < (int64_t)t.blocks * kPage ? keep : (int64_t)t.blocks * kPage;
    l.pages = (int)((kept + kPage - 1) / kPage);
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    l.holes = 0;
    l.movers = l.holes + up(lists * l.most * 8);
    l.starts = l.movers + up(lists * l.most * 8);
    l.border = l.starts + up(lists * (l.pages + 1) * 4);
    l.latest = l.border + up(lists * 16);
    l.chunks = t.blocks <= kLongWaves * kLongBlocks ? 1 : (t.blocks + kChunkBlocks - 1) / kChunkBlocks;
    const int64_t shared = l.chunks > 1 ? lists : 0;
    l.bins = l.latest + up(shared * l.chunks * 8);
    l.counts = l.bins + up(shared * kBinWords * 4);
    l.bytes = l.counts + up(shared * l.chunks * kSharedWaves * 16);
    return l;
}

int evict_args(const vl_cache8 *cache, const vl_tokens *tokens, int64_t keep, EvictArgs *a, Layout *l) {
    int rc = vl_cache8_of(cache, &a->c);
    if (rc == VL_OK) rc = vl_tokens_of(tokens, &a->t);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(a->t.offsets == nullptr, "an eviction has no rows: offsets must be null");
    VL_REQUIRE(keep >= 0 && keep < (1ll << 31), "keep: %lld", (long long)keep);
    *l = layout_of(a->c, a->t, keep);
    const int64_t lists = (int64_t)a->t.sequences * a->c.heads;
    VL_REQUIRE(lists <= kMaxBlocks && lists * l->chunks <= kMaxBlocks, "more sequences than one call takes: %d of %d blocks", a->t.sequences, a->t.blocks);
    // Pages that have about 64 free places together, if all that the table has room for were to be filled, but two workgroups for every
    // compute unit.  64 sequences of 4,160 that keep 4,096: 34 us with 16 pages together, 24 with 64.
    const int64_t places = (int64_t)a->t.blocks * kPage, free = keep < places - keep ? keep : places - keep;
    int64_t together = free > 0 ? l->pages * (int64_t)kPage / free : kMostTogether;
    const int64_t few = lists * l->pages / (2 * kComputeUnits);
    together = together < few ? together : few;
    a->together = (int)(together < 1 ? 1 : together > kMostTogether ? kMostTogether : together);
    l->groups = lists * ((l->pages + a->together - 1) / a->together);
    VL_REQUIRE(l->groups <= 4 * kMaxBlocks, "more pages than one call takes: %d sequences of %d", a->t.sequences, l->pages);
    a->keep = (int)keep;
    a->most = l->most;
    a->pages = l->pages;
    a->chunks = l->chunks;
    return VL_OK;
}

}  // namespace

VL_EXPORT int64_t vl_cache8_evict_workspace_bytes(const vl_cache8 *cache, const vl_tokens *tokens, int64_t keep) {
    EvictArgs a = {};
    Layout l;
    const int rc = evict_args(cache, tokens, keep, &a, &l);
    return rc != VL_OK ? rc : l.bytes;
}

VL_EXPORT int vl_cache8_evict(const vl_cache8 *cache, const vl_tokens *tokens, int64_t keep, int64_t recent, int32_t *new_lengths,
                              void *workspace, int64_t workspace_bytes, void *stream) {
    EvictArgs a = {};
    Layout l;
    const int rc = evict_args(cache, tokens, keep, &a, &l);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(recent >= 0 && recent <= keep, "recent: %lld of %lld that stay", (long long)recent, (long long)keep);
    if (a.t.sequences == 0) return VL_OK;
    VL_REQUIRE(new_lengths != nullptr, "new_lengths is null");
    VL_REQUIRE(a.c.weights != nullptr || a.c.pages == 0, "the cache has no weights");
    if (l.bytes > workspace_bytes || !workspace) {
        vl_set_error("workspace too small: %lld bytes needed, %lld given", (long long)l.bytes, (long long)workspace_bytes);
        return VL_ERR_WORKSPACE;
    }
    VL_REQUIRE(((uintptr_t)workspace & 15) == 0, "workspace not on a 16-byte boundary");
    // workgroups of other heads still read the old ones
    VL_REQUIRE(new_lengths + a.t.sequences <= a.t.lengths || a.t.lengths + a.t.sequences <= new_lengths, "new_lengths overlap lengths");
    uint8_t *const ws = (uint8_t *)workspace;
    a.recent = (int)recent;
    a.lengths = new_lengths;
    a.holes = (int64_t *)(ws + l.holes);
    a.movers = (int64_t *)(ws + l.movers);
    a.starts = (int32_t *)(ws + l.starts);
    a.border = (int64_t *)(ws + l.border);
    a.latest = (int32_t *)(ws + l.latest);
    a.bins = (uint32_t *)(ws + l.bins);
    a.counts = (int32_t *)(ws + l.counts);
    const hipStream_t s = (hipStream_t)stream;
    const int64_t lists = a.t.sequences * (int64_t)a.c.heads;
    if (l.chunks > 1) {
        const unsigned groups = (unsigned)(lists * l.chunks);
        evict_choose_kernel<kLatest, kSharedWaves, kSharedBlocks><<<groups, kSharedWaves * 64, 0, s>>>(a);
        evict_choose_kernel<kFirstDigit, kSharedWaves, kSharedBlocks><<<groups, kSharedWaves * 64, 0, s>>>(a);
        evict_choose_kernel<kSecondDigit, kSharedWaves, kSharedBlocks><<<groups, kSharedWaves * 64, 0, s>>>(a);
        evict_choose_kernel<kLastDigit, kSharedWaves, kSharedBlocks><<<groups, kSharedWaves * 64, 0, s>>>(a);
        evict_choose_kernel<kCount, kSharedWaves, kSharedBlocks><<<groups, kSharedWaves * 64, 0, s>>>(a);
        evict_choose_kernel<kList, kSharedWaves, kSharedBlocks><<<groups, kSharedWaves * 64, 0, s>>>(a);
    } else if (a.t.blocks > kShortWaves * kShortBlocks) {
        evict_choose_kernel<kWhole, kLongWaves, kLongBlocks><<<(unsigned)lists, kLongWaves * 64, 0, s>>>(a);
    } else {
        evict_choose_kernel<kWhole, kShortWaves, kShortBlocks><<<(unsigned)lists, kShortWaves * 64, 0, s>>>(a);
    }
    VL_LAUNCH_CHECK("evict_choose_kernel");
    if (l.pages == 0) return VL_OK;
    for_dim(a.c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        evict_move_kernel<D><<<(unsigned)l.groups, 256, 0, s>>>(a);
    });
    VL_LAUNCH_CHECK("evict_move_kernel");
    return VL_OK;
}
