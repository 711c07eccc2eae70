// Writing keys and values into the cache in 8 bits, and reading them back.
#include "cache8.h"

int vl_cache8_of(const vl_cache8 *c, CacheView *out) {
    VL_REQUIRE(c != nullptr, "cache is null");
    VL_REQUIRE(c->pages >= 0 && c->pages <= (1ll << 31) - 2, "pages: %lld", (long long)c->pages);
    VL_REQUIRE(c->heads >= 1 && c->heads <= 65535, "heads: 1 to 65535, got %lld", (long long)c->heads);
    VL_REQUIRE(c->dim == 32 || c->dim == 64 || c->dim == 96 || c->dim == 128 || c->dim == 192 || c->dim == 256,
               "dim: 32, 64, 96, 128, 192 or 256, got %lld", (long long)c->dim);
    VL_REQUIRE((c->keys && c->values && c->scales) || c->pages == 0, "a part of the cache is null");
    VL_REQUIRE((c->weights != nullptr) == (c->positions != nullptr) || c->pages == 0, "weights without positions, or positions without weights");
    const void *parts[] = {c->keys, c->values, c->scales, c->weights, c->positions};
    for (const void *p : parts) VL_REQUIRE(((uintptr_t)p & 15) == 0, "a part of the cache is not on a 16-byte boundary");
    *out = {};
    out->pages = c->pages;
    out->heads = (int)c->heads;
    out->dim = (int)c->dim;
    out->keys = c->keys;
    out->values = c->values;
    out->scales = (uint32_t *)c->scales;
    out->weights = c->weights;
    out->positions = c->positions;
    return VL_OK;
}

namespace {

struct Rows8 {  // [rows, heads, dim] of a call
    const void *at;
    int64_t row, head;
};

// One workgroup makes one block of one head.  A unit is 8 dimensions of 4 tokens of the keys or of the values: 8 bytes of each of four
// rows, or 32 bytes of the values' image.  The page's power depends on all new elements of the block, so a thread holds its units'
// elements in registers from the loads, over the largest magnitude of all, to the codes: one pass over the rows.  Old codes of the
// block are read where they share words with new ones, and all of them where the power has grown.
template <int D, int NS>
__global__ __launch_bounds__(256) void cache8_write_kernel(CacheView c, Tokens t, Rows8 keys, Rows8 values, const int32_t *positions) {
    constexpr int kSegs = D / 8, kUnits = (2 * kSegs * 16 + 255) / 256;  // of a thread; a wavefront's are all keys or all values
    typedef typename ElementOf<NS>::type E;
    __shared__ uint32_t s_top[2], s_bad[2][2];  // largest magnitude's bits; a bit for a spoilt token
    const int h = blockIdx.x % c.heads;
    Piece w = {(int)blockIdx.x / c.heads, 0};
    if (t.offsets)
        w = find_piece(t.sequences, blockIdx.x / c.heads, [&](int b) {
            const int n = row_count(t, b), start = length_of(t, b);
            return n ? (int)((start + (int64_t)n - 1) / kPage) - start / kPage + 1 : 0;
        });
    if (w.sequence < 0) return;
    const int b = w.sequence, start = length_of(t, b);
    const int block = start / kPage + w.piece;
    const int64_t page = page_of(t, c, b, block);
    if (page < 0) return;
    const int row0 = first_row(t, b);
    const int64_t end = start + (int64_t)row_count(t, b);
    const int first = max(start - block * kPage, 0);                       // places in the block
    const int last = (int)min((int64_t)kPage, end - (int64_t)block * kPage);
    const int64_t unit = page * c.heads + h, row_at = row0 + ((int64_t)block * kPage - start);  // row of place 0
    uint8_t *const kc = c.keys + unit * (kPage * D), *const vc = c.values + unit * (kPage * D);
    const uint32_t was = c.scales[unit];
    if (threadIdx.x < 2) s_top[threadIdx.x] = 0;
    if (threadIdx.x < 4) s_bad[threadIdx.x >> 1][threadIdx.x & 1] = 0;

    Eight<NS> x[kUnits][4];
    auto place_of = [&](int k, int &which, int &four, int &seg) {
        const int u = k * 256 + threadIdx.x;
        which = __builtin_amdgcn_readfirstlane(u / (kSegs * 16));
        seg = u % kSegs;
        four = u / kSegs & 15;
    };
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        int which, four, seg;
        place_of(k, which, four, seg);
        const Rows8 &from = which ? values : keys;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int j = four * 4 + i;
            const bool real = which < 2 && j >= first && j < last;
            x[k][i] = load8<NS>((const E *)from.at + (real ? (row_at + j) * from.row + h * from.head + seg * 8 : 0), real);
        }
    }
    __syncthreads();
    uint32_t top[kUnits][4];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        int which, four, seg;
        place_of(k, which, four, seg);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            top[k][i] = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) top[k][i] = max(top[k][i], __builtin_bit_cast(uint32_t, (float)x[k][i][e]) & 0x7FFFFFFFu);
            if (top[k][i] >= 0x7F800000u) atomicOr(&s_bad[which][four >> 3], 1u << ((four & 7) * 4 + i));
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        int which, four, seg;
        place_of(k, which, four, seg);
        if (which > 1) continue;
        const uint32_t bad = s_bad[which][four >> 3] >> ((four & 7) * 4);
        uint32_t all = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) all = max(all, bad >> i & 1 ? 0 : top[k][i]);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) all = max(all, (uint32_t)__shfl_xor((int)all, d));
        if ((threadIdx.x & 63) == 0) atomicMax(&s_top[which], all);
    }
    __syncthreads();
    uint32_t byte[2] = {fitting_byte(s_top[0]), fitting_byte(s_top[1])}, old[2] = {byte_of_keys(was), byte_of_values(was)};
    bool grown[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (first > 0) byte[i] = max(byte[i], old[i]);
        grown[i] = first > 0 && byte[i] != old[i];
    }
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        int which, four, seg;
        place_of(k, which, four, seg);
        if (which > 1 || four * 4 >= last) continue;
        const bool has_new = four * 4 + 3 >= first, has_others = four * 4 < first || four * 4 + 4 > last;
        const bool again = which ? grown[1] : grown[0];
        if (!has_new && !again) continue;
        const uint32_t b = which ? byte[1] : byte[0];
        const float by = power_of_byte(254 - b);  // 1 / the power
        const float again_by = power_below(b - (which ? old[1] : old[0]));
        auto coded_again = [&](uint32_t word) {
            const f32x4 v = four_numbers(word) * again_by;
            return four_codes(v);
        };
        const uint32_t bad = s_bad[which][four >> 3] >> ((four & 7) * 4);
        u32x2 code[4];  // of a token
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x4 lo = {(float)x[k][i][0], (float)x[k][i][1], (float)x[k][i][2], (float)x[k][i][3]};
            const f32x4 hi = {(float)x[k][i][4], (float)x[k][i][5], (float)x[k][i][6], (float)x[k][i][7]};
            code[i] = u32x2{four_codes(within(lo * by)), four_codes(within(hi * by))};
            if (bad >> i & 1) code[i] = u32x2{0x7F7F7F7Fu, 0x7F7F7F7Fu};
        }
        if (which == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = four * 4 + i;
                u32x2 *const at = reinterpret_cast<u32x2 *>(kc + j * D + seg * 8);
                if (j >= first && j < last) {
                    *at = code[i];
                } else if (j < first && again) {
                    const u32x2 o = *at;
                    *at = u32x2{coded_again(o[0]), coded_again(o[1])};
                }
            }
        } else {
            u32x4 *const at = reinterpret_cast<u32x4 *>(vc + (four * D + seg * 8) * 4);
            u32x4 o[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            if (has_others) o[0] = at[0], o[1] = at[1];
            uint32_t before = 0, fresh = 0;  // bytes of old tokens and of new ones; those behind them are left as they are
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = four * 4 + i;
                if (j < first) before |= 255u << (8 * i);
                else if (j < last) fresh |= 255u << (8 * i);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                uint32_t word = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) word |= (code[i][e >> 2] >> (8 * (e & 3)) & 255) << (8 * i);
                const uint32_t was = o[e >> 2][e & 3];
                word = (word & fresh) | (was & ~fresh);
                if (again && before) word = (coded_again(was) & before) | (word & ~before);
                o[e >> 2][e & 3] = word;
            }
            at[0] = o[0];
            at[1] = o[1];
        }
    }
    if (threadIdx.x == 0) {
        const bool marked = (first > 0 && is_marked(was)) || (s_bad[0][0] | s_bad[0][1] | s_bad[1][0] | s_bad[1][1]);
        c.scales[unit] = byte[0] | byte[1] << 8 | (marked ? 1u << 16 : 0);
    }
    if (c.weights && threadIdx.x >= first && threadIdx.x < last) {
        c.weights[unit * kPage + threadIdx.x] = 0;
        c.positions[unit * kPage + threadIdx.x] = positions ? positions[row_at + threadIdx.x] : block * kPage + (int)threadIdx.x;
    }
}

// 8 dimensions of one row and head a thread
template <int D, int NS>
__global__ __launch_bounds__(256) void cache8_read_kernel(CacheView c, Tokens t, typename ElementOf<NS>::type *keys,
                                                          typename ElementOf<NS>::type *values) {
    constexpr int kSegs = D / 8;
    const int64_t n = (int64_t)t.rows * c.heads * kSegs;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int seg = (int)(i % kSegs), h = (int)(i / kSegs % c.heads), row = (int)(i / kSegs / c.heads);
        const int b = sequence_of(t, row), first = first_row(t, b);
        const int64_t place = (int64_t)length_of(t, b) + row - first;
        const int64_t page = row >= first && row < first + row_count(t, b) ? page_of(t, c, b, (int)min(place / kPage, (int64_t)t.blocks)) : -1;
        float k[8] = {0, 0, 0, 0, 0, 0, 0, 0}, v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (page >= 0) {
            const int j = (int)(place % kPage);
            const int64_t unit = page * c.heads + h;
            const u32x2 kw = *reinterpret_cast<const u32x2 *>(c.keys + unit * (kPage * D) + j * D + seg * 8);
            const u32x4 *const at = reinterpret_cast<const u32x4 *>(c.values + unit * (kPage * D) + ((j >> 2) * D + seg * 8) * 4);
            const u32x4 vw[2] = {at[0], at[1]};
            const uint32_t scales = c.scales[unit];
            const float ks = scale_of_keys(scales), vs = scale_of_values(scales);
            const int turn = 8 * (j & 3);
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const u32x4 x = vw[half];
                const uint32_t word = (x[0] >> turn & 255) | (x[1] >> turn & 255) << 8 | (x[2] >> turn & 255) << 16 | (x[3] >> turn & 255) << 24;
                const f32x4 a = four_numbers(kw[half]), b = four_numbers(word);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    k[half * 4 + e] = a[e] * ks;
                    v[half * 4 + e] = b[e] * vs;
                }
            }
        }
        store8<NS>(keys + i * 8, k);
        store8<NS>(values + i * 8, v);
    }
}

template <int NS>
int write_rows(const CacheView &c, const Tokens &t, Rows8 k, Rows8 v, const int32_t *positions, hipStream_t stream) {
    // a sequence's n rows lie in at most n / 64 + 2 blocks, one row in one
    const int64_t tiles = t.offsets ? (int64_t)t.rows / kPage + 2 * sequences_with_rows(t) : t.rows;
    VL_REQUIRE(tiles * c.heads <= 4 * kMaxBlocks, "more sequences and rows than one call takes: %lld blocks", (long long)tiles);
    for_dim(c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        cache8_write_kernel<D, NS><<<(unsigned)(tiles * c.heads), 256, 0, stream>>>(c, t, k, v, positions);
    });
    VL_LAUNCH_CHECK("cache8_write_kernel");
    return VL_OK;
}

template <int NS>
int read_rows(const CacheView &c, const Tokens &t, void *keys, void *values, hipStream_t stream) {
    typedef typename ElementOf<NS>::type E;
    for_dim(c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        cache8_read_kernel<D, NS><<<vl_grid_for((int64_t)t.rows * c.heads * (D / 8), 256), 256, 0, stream>>>(c, t, (E *)keys, (E *)values);
    });
    VL_LAUNCH_CHECK("cache8_read_kernel");
    return VL_OK;
}

}  // namespace

VL_EXPORT int vl_cache8_write(const vl_cache8 *cache, const vl_tokens *tokens, int type, const void *keys, int64_t key_row,
                              int64_t key_head, const void *values, int64_t value_row, int64_t value_head,
                              const int32_t *positions, void *stream) {
    CacheView c;
    Tokens t;
    int rc = vl_cache8_of(cache, &c);
    if (rc == VL_OK) rc = vl_tokens_of(tokens, &t);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(type >= VL_BF16 && type <= VL_F32, "type: %d", type);
    if (t.rows == 0 || c.pages == 0) return VL_OK;
    VL_REQUIRE(keys && values, "keys or values is null");
    const int size = type == VL_F32 ? 4 : 2;
    VL_REQUIRE(((uintptr_t)keys | (uintptr_t)values) % size == 0, "keys or values not aligned to their type");
    VL_REQUIRE(((uintptr_t)positions & 3) == 0, "positions not aligned to their type");
    const Rows8 k = {keys, key_row, key_head}, v = {values, value_row, value_head};
    const hipStream_t s = (hipStream_t)stream;
    return type == VL_BF16 ? write_rows<1>(c, t, k, v, positions, s) : type == VL_F16 ? write_rows<2>(c, t, k, v, positions, s) : write_rows<3>(c, t, k, v, positions, s);
}

VL_EXPORT int vl_cache8_read(const vl_cache8 *cache, const vl_tokens *tokens, int type, void *keys, void *values, void *stream) {
    CacheView c;
    Tokens t;
    int rc = vl_cache8_of(cache, &c);
    if (rc == VL_OK) rc = vl_tokens_of(tokens, &t);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(type >= VL_BF16 && type <= VL_F32, "type: %d", type);
    if (t.rows == 0) return VL_OK;
    VL_REQUIRE(keys && values, "keys or values is null");
    VL_REQUIRE((((uintptr_t)keys | (uintptr_t)values) & 15) == 0, "keys or values not on a 16-byte boundary");
    const hipStream_t s = (hipStream_t)stream;
    return type == VL_BF16 ? read_rows<1>(c, t, keys, values, s) : type == VL_F16 ? read_rows<2>(c, t, keys, values, s) : read_rows<3>(c, t, keys, values, s);
}
