// Eviction from a cache in 8 bits: of every sequence and head the tokens that count most stay.
//
// What stays behind the new length moves into places before it that got free, so a step that gives up 64 tokens moves at most 64
// a head, where closing the gaps in order would move nearly all of them; sources (behind the new length) and destinations
// (before it) are apart, so pages are made in any order.  Two launches: one workgroup a sequence and head ranks its tokens and lists
// free places and what moves there; one a page and head moves.
#include "cache8.h"

namespace {

struct EvictArgs {
    CacheView c;
    Tokens t;
    int keep, recent;
    int most;           // entries of a list: pairs of a sequence and head, at most
    int pages;          // of keep tokens
    int32_t *lengths;   // new ones
    // per sequence and head:
    int32_t *holes, *movers;  // [most] free places and the places whose tokens move there, both ascending
    int32_t *starts;          // [pages + 1] the first hole of every block
    uint32_t *border;         // scales of the page that the new length lies in, before any change
};

constexpr int kDigit = 11;  // bits of a key that one pass over the weights tells apart
constexpr int kBins = 1 << kDigit;
constexpr int kChooseWaves = 16;

// Larger stays first; NaN is last.  vl_float_key puts +NaN above all.
__device__ inline uint32_t rank_key(float weight, bool late) { return late ? ~0u : weight != weight ? 0u : vl_float_key(weight); }

__global__ __launch_bounds__(kChooseWaves * 64) void evict_choose_kernel(EvictArgs a) {
    __shared__ uint32_t s_bin[kBins];
    __shared__ int s_newest[kChooseWaves], s_real[kChooseWaves];
    __shared__ int s_above[kChooseWaves][2], s_ties[kChooseWaves][2];  // before and behind the new length
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % a.c.heads, b = blockIdx.x / a.c.heads;
    const int length = length_of(a.t, b);
    int32_t *const starts = a.starts + (int64_t)blockIdx.x * (a.pages + 1);
    if (length <= a.keep) {
        for (int i = threadIdx.x; i <= a.pages; i += kChooseWaves * 64) starts[i] = 0;
        if (h == 0 && threadIdx.x == 0) a.lengths[b] = length;
        return;
    }
    // every wavefront has blocks of its own, one after the other
    const int blocks = (length + kPage - 1) / kPage, each = (blocks + kChooseWaves - 1) / kChooseWaves;
    const int from = min(wave * each, blocks), to = min(from + each, blocks);
    auto page_at = [&](int block) { return page_of(a.t, a.c, b, block); };
    auto weight_at = [&](int64_t page) { return (page * a.c.heads + h) * kPage + lane; };
    // the latest position, and how many tokens there are on pages
    int newest = INT32_MIN, real = 0;
    for (int block = from; block < to; block++) {
        const int64_t page = page_at(block);
        if (page < 0 || block * kPage + lane >= length) continue;
        newest = max(newest, a.c.positions[weight_at(page)]);
        real++;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        newest = max(newest, __shfl_xor(newest, d));
        real += __shfl_xor(real, d);
    }
    if (lane == 0) {
        s_newest[wave] = newest;
        s_real[wave] = real;
    }
    for (int i = threadIdx.x; i < kBins; i += kChooseWaves * 64) s_bin[i] = 0;
    if (threadIdx.x == 0) s_prefix = 0;
    __syncthreads();
    real = 0;
#pragma unroll
    for (int i = 0; i < kChooseWaves; i++) {
        newest = max(newest, s_newest[i]);
        real += s_real[i];
    }
    const int kept = min(a.keep, real);
    if (h == 0 && threadIdx.x == 0) a.lengths[b] = kept;
    if (kept == 0) {
        for (int i = threadIdx.x; i <= a.pages; i += kChooseWaves * 64) starts[i] = 0;
        return;
    }
    auto key_at = [&](int64_t page) {
        const int64_t at = weight_at(page);
        return rank_key(a.c.weights[at], (int64_t)a.c.positions[at] > (int64_t)newest - a.recent);
    };
    // the key of the last that stays, 11, 11 and 10 bits at a time, and how many with that key do
    int need = kept;
    uint32_t prefix = 0;
    for (int shift = 32 - kDigit;; shift -= kDigit) {
        const int low = max(shift, 0), bits = shift >= 0 ? kDigit : kDigit + shift;
        for (int block = from; block < to; block++) {
            const int64_t page = page_at(block);
            if (page < 0 || block * kPage + lane >= length) continue;
            const uint32_t key = key_at(page);
            if (low + bits == 32 || key >> (low + bits) == prefix) atomicAdd(&s_bin[key >> low & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        if (wave == 0) {  // lane l has the bins of the l-th highest 32nd
            constexpr int kEach = kBins / 64;
            const int top = kBins - 1 - lane * kEach;
            int sum = 0;
            for (int i = 0; i < kEach; i++) sum += s_bin[top - i];
            int upto = sum;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int other = __shfl_up(upto, d);
                if (lane >= d) upto += other;
            }
            int above = upto - sum;
            if (above < need && upto >= need) {
                int i = 0;
                for (; above + (int)s_bin[top - i] < need; i++) above += s_bin[top - i];
                s_prefix = prefix << bits | (uint32_t)(top - i);
                s_need = need - above;
            }
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
        if (shift <= 0) break;
        for (int i = threadIdx.x; i < kBins; i += kChooseWaves * 64) s_bin[i] = 0;
        __syncthreads();
    }
    // keys above `prefix` stay, and the first `need` of those equal to it
    int above[2] = {0, 0}, ties[2] = {0, 0};
    for (int block = from; block < to; block++) {
        const int64_t page = page_at(block);
        const int place = block * kPage + lane;
        const bool there = page >= 0 && place < length;
        const uint32_t key = there ? key_at(page) : 0;
        const bool more = there && key > prefix, equal = there && key == prefix, behind = place >= kept;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            above[i] += __popcll(__ballot(more && behind == (i == 1)));
            ties[i] += __popcll(__ballot(equal && behind == (i == 1)));
        }
    }
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            s_above[wave][i] = above[i];
            s_ties[wave][i] = ties[i];
        }
    }
    __syncthreads();
    int tie = 0, stays = 0, moves = 0;  // of the wavefronts before this one
    for (int i = 0; i < wave; i++) {
        const int t0 = min(max(need - tie, 0), s_ties[i][0]);
        stays += s_above[i][0] + t0;
        tie += s_ties[i][0];
        moves += s_above[i][1] + min(max(need - tie, 0), s_ties[i][1]);
        tie += s_ties[i][1];
    }
    int free = min(from * kPage, kept) - stays;  // free places before
    int32_t *const holes = a.holes + (int64_t)blockIdx.x * a.most, *const movers = a.movers + (int64_t)blockIdx.x * a.most;
    const uint64_t before = (1ull << lane) - 1;
    for (int block = from; block < to; block++) {
        const int64_t page = page_at(block);
        const int place = block * kPage + lane;
        const bool there = page >= 0 && place < length;
        const uint32_t key = there ? key_at(page) : 0;
        const uint64_t equal = __ballot(there && key == prefix);
        const bool in = there && (key > prefix || (key == prefix && tie + __popcll(equal & before) < need));
        tie += __popcll(equal);
        const uint64_t hole = __ballot(place < kept && !in), moving = __ballot(place >= kept && in);
        if (lane == 0 && block < a.pages) starts[block] = free;
        if (hole >> lane & 1) holes[free + __popcll(hole & before)] = place;
        if (moving >> lane & 1) movers[moves + __popcll(moving & before)] = place;
        free += __popcll(hole);
        moves += __popcll(moving);
        if (lane == 0 && block == (kept - 1) / kPage)
            for (int i = block + 1; i <= a.pages; i++) starts[i] = free;
        if (block == kept / kPage && lane == 0) a.border[blockIdx.x] = page >= 0 ? a.c.scales[page * a.c.heads + h] : 0;
    }
}

// A workgroup fills the free places of one page of one head.  A unit is 16 dimensions of a moving token: 16 bytes of its key, or one byte
// of each of 16 words of the values.
template <int D>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    constexpr int kSegs = D / 16, kUnits = (2 * kSegs * kPage + 255) / 256;
    __shared__ int s_to[kPage], s_source[kPage];  // places
    __shared__ int64_t s_unit[kPage];             // page and head that it comes from
    __shared__ uint32_t s_scales[kPage], s_top[2];
    __shared__ int s_spoilt;
    const int h = blockIdx.x % a.c.heads, block = blockIdx.x / a.c.heads % a.pages, b = blockIdx.x / a.c.heads / a.pages;
    const int64_t list = (int64_t)b * a.c.heads + h;
    const int32_t *const starts = a.starts + list * (a.pages + 1) + block;
    const int first = starts[0], n = starts[1] - first;
    if (n <= 0) return;
    const int64_t page = page_of(a.t, a.c, b, block);
    if (page < 0) return;
    const int64_t unit = page * a.c.heads + h;
    const int kept = a.lengths[b];
    const uint32_t was = a.c.scales[unit];
    if (threadIdx.x < kPage && threadIdx.x < n) {
        const int i = threadIdx.x, source = a.movers[list * a.most + first + i];
        const int64_t from = page_of(a.t, a.c, b, source / kPage) * a.c.heads + h;  // it is on a page
        s_to[i] = a.holes[list * a.most + first + i] % kPage;
        s_source[i] = source % kPage;
        s_unit[i] = from;
        // the page of the border may be given another power while this one is made; its tokens behind the border are as they were
        s_scales[i] = source / kPage == kept / kPage ? a.border[list] : a.c.scales[from];
        a.c.weights[unit * kPage + s_to[i]] = a.c.weights[from * kPage + s_source[i]];
        a.c.positions[unit * kPage + s_to[i]] = a.c.positions[from * kPage + s_source[i]];
    }
    if (threadIdx.x < 2) s_top[threadIdx.x] = 0;
    if (threadIdx.x == 2) s_spoilt = 0;
    __syncthreads();
    const int units = 2 * kSegs * n;
    u32x4 x[kUnits];
    uint32_t top[2] = {0, 0};
    bool spoilt = false;
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const int u = k * 256 + threadIdx.x;
        if (u >= units) continue;
        const int seg = u % kSegs, i = u / kSegs % n, which = u / kSegs / n;
        const int64_t from = s_unit[i];
        const int token = s_source[i];
        if (which == 0) {
            x[k] = *reinterpret_cast<const u32x4 *>(a.c.keys + from * (kPage * D) + token * D + seg * 16);
        } else {
            const u32x4 *const at = reinterpret_cast<const u32x4 *>(a.c.values + from * (kPage * D) + ((token >> 2) * D + seg * 16) * 4);
            const int turn = 8 * (token & 3);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const u32x4 v = at[w];
                x[k][w] = (v[0] >> turn & 255) | (v[1] >> turn & 255) << 8 | (v[2] >> turn & 255) << 16 | (v[3] >> turn & 255) << 24;
            }
        }
        const float scale = which ? scale_of_values(s_scales[i]) : scale_of_keys(s_scales[i]);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const f32x4 v = four_numbers(x[k][w] & 0x7F7F7F7Fu) * scale;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t bits = __builtin_bit_cast(uint32_t, (float)v[e]);
                if (bits >= 0x7F800000u) spoilt = true;
                else top[which] = max(top[which], bits);
            }
        }
    }
#pragma unroll
    for (int which = 0; which < 2; which++) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top[which] = max(top[which], (uint32_t)__shfl_xor((int)top[which], d));
        if ((threadIdx.x & 63) == 0) atomicMax(&s_top[which], top[which]);
    }
    if (spoilt) s_spoilt = 1;
    __syncthreads();
    const uint32_t old[2] = {byte_of_keys(was), byte_of_values(was)};
    const uint32_t byte[2] = {max(old[0], fitting_byte(s_top[0])), max(old[1], fitting_byte(s_top[1]))};
    // tokens that the page holds already, up to the new length: places that are filled are overwritten below
    const int holds = min(kept - block * kPage, kPage);
    if (byte[0] != old[0]) {
        const float by = power_below(byte[0] - old[0]);
        uint32_t *const at = reinterpret_cast<uint32_t *>(a.c.keys + unit * (kPage * D));
        for (int i = threadIdx.x; i < holds * D / 4; i += 256) at[i] = four_codes(four_numbers(at[i]) * by);
    }
    if (byte[1] != old[1]) {
        const float by = power_below(byte[1] - old[1]);
        uint32_t *const at = reinterpret_cast<uint32_t *>(a.c.values + unit * (kPage * D));
        for (int i = threadIdx.x; i < (holds + 3) / 4 * D; i += 256) {
            const int there = holds - i / D * 4;  // of the word's tokens
            const uint32_t keep = there >= 4 ? 0 : ~0u << (8 * there), word = at[i];
            at[i] = (four_codes(four_numbers(word) * by) & ~keep) | (word & keep);
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const int u = k * 256 + threadIdx.x;
        if (u >= units) continue;
        const int seg = u % kSegs, i = u / kSegs % n, which = u / kSegs / n, token = s_to[i];
        const uint32_t from = which ? byte_of_values(s_scales[i]) : byte_of_keys(s_scales[i]), now = which ? byte[1] : byte[0];
        if (from != now) {
            // powers are up to 2^237 apart: by the difference in two steps, of which the second alone rounds or neither does
            const int up = (int)from - (int)now, half = up / 2;
            const float by0 = power_of_byte((uint32_t)(127 + half)), by1 = power_of_byte((uint32_t)(127 + up - half));
#pragma unroll
            for (int w = 0; w < 4; w++) x[k][w] = four_codes(four_numbers(x[k][w]) * by0 * by1);
        }
        if (which == 0) {
            *reinterpret_cast<u32x4 *>(a.c.keys + unit * (kPage * D) + token * D + seg * 16) = x[k];
        } else {
            uint8_t *const at = a.c.values + unit * (kPage * D) + ((token >> 2) * D + seg * 16) * 4 + (token & 3);
#pragma unroll
            for (int e = 0; e < 16; e++) at[e * 4] = (uint8_t)(x[k][e >> 2] >> (8 * (e & 3)));
        }
    }
    if (threadIdx.x == 0) a.c.scales[unit] = byte[0] | byte[1] << 8 | (is_marked(was) || s_spoilt ? 1u << 16 : 0);
}

struct Layout {
    int64_t holes, movers, starts, border, bytes;
    int most, pages;
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
    l.movers = l.holes + up(lists * l.most * 4);
    l.starts = l.movers + up(lists * l.most * 4);
    l.border = l.starts + up(lists * (l.pages + 1) * 4);
    l.bytes = l.border + up(lists * 4);
    return l;
}

int evict_args(const vl_cache8 *cache, const vl_tokens *tokens, int64_t keep, EvictArgs *a, Layout *l) {
    int rc = vl_cache8_of(cache, &a->c);
    if (rc == VL_OK) rc = vl_tokens_of(tokens, &a->t);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(a->t.offsets == nullptr, "an eviction has no rows: offsets must be null");
    VL_REQUIRE(keep >= 0 && keep < (1ll << 31), "keep: %lld", (long long)keep);
    VL_REQUIRE((int64_t)a->t.sequences * a->c.heads <= 4 * kMaxBlocks, "more sequences than one call takes: %d", a->t.sequences);
    *l = layout_of(a->c, a->t, keep);
    VL_REQUIRE((int64_t)a->t.sequences * a->c.heads * l->pages < (1ll << 31), "more pages than one call takes: %d sequences of %d", a->t.sequences, l->pages);
    a->keep = (int)keep;
    a->most = l->most;
    a->pages = l->pages;
    return VL_OK;
}

}  // namespace

VL_EXPORT int64_t vl_cache8_evict_workspace_bytes(const vl_cache8 *cache, const vl_tokens *tokens, int64_t keep) {
    EvictArgs a;
    Layout l;
    const int rc = evict_args(cache, tokens, keep, &a, &l);
    return rc != VL_OK ? rc : l.bytes;
}

VL_EXPORT int vl_cache8_evict(const vl_cache8 *cache, const vl_tokens *tokens, int64_t keep, int64_t recent, int32_t *new_lengths,
                              void *workspace, int64_t workspace_bytes, void *stream) {
    EvictArgs a;
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
    uint8_t *const ws = (uint8_t *)workspace;
    a.recent = (int)recent;
    a.lengths = new_lengths;
    a.holes = (int32_t *)(ws + l.holes);
    a.movers = (int32_t *)(ws + l.movers);
    a.starts = (int32_t *)(ws + l.starts);
    a.border = (uint32_t *)(ws + l.border);
    const hipStream_t s = (hipStream_t)stream;
    const unsigned lists = (unsigned)(a.t.sequences * (int64_t)a.c.heads);
    evict_choose_kernel<<<lists, kChooseWaves * 64, 0, s>>>(a);
    VL_LAUNCH_CHECK("evict_choose_kernel");
    if (l.pages == 0) return VL_OK;
    for_dim(a.c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        evict_move_kernel<D><<<lists * (unsigned)l.pages, 256, 0, s>>>(a);
    });
    VL_LAUNCH_CHECK("evict_move_kernel");
    return VL_OK;
}
