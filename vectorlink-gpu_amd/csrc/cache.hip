// Writing keys and values into the cache in 4 bits, and reading them back.
#include "cache.h"

int vl_cache_of(const vl_cache *c, CacheView *out) {
    VL_REQUIRE(c != nullptr, "cache is null");
    VL_REQUIRE(c->pages >= 0 && c->pages <= (1ll << 31) - 2, "pages: %lld", (long long)c->pages);
    VL_REQUIRE(c->heads >= 1 && c->heads <= 65535, "heads: 1 to 65535, got %lld", (long long)c->heads);
    VL_REQUIRE(c->dim == 32 || c->dim == 64 || c->dim == 96 || c->dim == 128 || c->dim == 192 || c->dim == 256,
               "dim: 32, 64, 96, 128, 192 or 256, got %lld", (long long)c->dim);
    const void *parts[] = {c->keys, c->key_scales, c->values, c->value_scales, c->bounds, c->bound_scales};
    for (const void *p : parts) {
        VL_REQUIRE(p != nullptr || c->pages == 0, "a part of the cache is null");
        VL_REQUIRE(((uintptr_t)p & 15) == 0, "a part of the cache is not on a 16-byte boundary");
    }
    *out = {c->pages, (int)c->heads, (int)c->dim, c->keys, c->key_scales, c->values, c->value_scales, c->bounds, c->bound_scales};
    return VL_OK;
}

int vl_tokens_of(const vl_tokens *t, Tokens *out) {
    VL_REQUIRE(t != nullptr, "tokens is null");
    VL_REQUIRE(t->rows >= 0 && t->rows < (1ll << 30), "rows: %lld", (long long)t->rows);
    VL_REQUIRE(t->sequences >= 0 && t->sequences < (1ll << 24), "sequences: %lld", (long long)t->sequences);
    VL_REQUIRE(t->blocks >= 0 && t->blocks < (1ll << 24), "blocks: %lld", (long long)t->blocks);
    VL_REQUIRE(t->blocks <= t->table_stride || t->sequences <= 1, "rows of the table overlap: %lld blocks, stride %lld",
               (long long)t->blocks, (long long)t->table_stride);
    VL_REQUIRE(t->offsets != nullptr || t->rows == t->sequences, "without offsets every sequence has one row: %lld rows, %lld sequences",
               (long long)t->rows, (long long)t->sequences);
    VL_REQUIRE(t->rows == 0 || t->sequences > 0, "%lld rows and no sequences", (long long)t->rows);
    VL_REQUIRE(t->lengths != nullptr || t->sequences == 0, "lengths is null");
    VL_REQUIRE(t->table != nullptr || t->sequences == 0 || t->blocks == 0, "table is null");
    *out = {t->table, t->lengths, t->offsets, t->table_stride, (int)t->rows, (int)t->sequences, (int)t->blocks};
    return VL_OK;
}

namespace {

struct Rows {  // [rows, heads, dim] of a call
    const void *at;
    int64_t row, head;
};

__device__ inline uint32_t max_of_four_lanes(uint32_t x) {  // lanes 4 n ... 4 n + 3
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));  // quad_perm: [1, 0, 3, 2]
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));  // [2, 3, 0, 1]
}

// The largest magnitude of a group, 8 elements of each of four lanes, as the bits of a float32: a NaN above an infinity above all
// others.  Magnitudes of 16 bits are compared two at a time as whole numbers, which have the same order.
template <int NS>
__device__ inline uint32_t top_of_group(const Eight<NS> &v) {
    if constexpr (NS == 3) {
        const u32x4 a = {__builtin_bit_cast(uint32_t, (float)v[0]), __builtin_bit_cast(uint32_t, (float)v[1]),
                         __builtin_bit_cast(uint32_t, (float)v[2]), __builtin_bit_cast(uint32_t, (float)v[3])};
        const u32x4 b = {__builtin_bit_cast(uint32_t, (float)v[4]), __builtin_bit_cast(uint32_t, (float)v[5]),
                         __builtin_bit_cast(uint32_t, (float)v[6]), __builtin_bit_cast(uint32_t, (float)v[7])};
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) top = max(top, max(a[i] & 0x7FFFFFFFu, b[i] & 0x7FFFFFFFu));
        return max_of_four_lanes(top);
    } else {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        const u32x4 w = __builtin_bit_cast(u32x4, v) & 0x7FFF7FFFu;
        const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3];
        const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(__builtin_bit_cast(u16x2, w0), __builtin_bit_cast(u16x2, w1)),
                                                  __builtin_elementwise_max(__builtin_bit_cast(u16x2, w2), __builtin_bit_cast(u16x2, w3)));
        const uint32_t top = max_of_four_lanes(max((uint32_t)m[0], (uint32_t)m[1]));
        if constexpr (NS == 1) return top << 16;
        if (top >= 0x7C00u) return 0x7F800000u;
        return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)top));
    }
}

// The codes of 8 elements of a token, four lanes of a group together: the scale's byte, and whether the elements are finite.
template <int NS>
__device__ inline uint32_t quantise8(const Eight<NS> &v, int *byte, bool *finite) {
    const uint32_t bits = top_of_group<NS>(v);
    *finite = bits < 0x7F800000u;
    // the exponent of a number below 2^-126 reads as -127, and both are far below the least
    const int e = max((int)(bits >> 23) - 127 - 2, kLeastExponent);
    *byte = e + 127;
    const float scale = __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
    uint32_t code = 0;  // rounds to nearest, ties to the even code, magnitudes over 6 to 6
    if constexpr (NS == 1) {
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, v.s01, scale, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, v.s23, scale, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, v.s45, scale, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, v.s67, scale, 3);
    } else {
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, (float)v[0], (float)v[1], scale, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, (float)v[2], (float)v[3], scale, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, (float)v[4], (float)v[5], scale, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, (float)v[6], (float)v[7], scale, 3);
    }
    return code;
}

// The upper value of a word stays in it with the lower one's bits behind its own: they change no comparison of two values that
// differ, and are cut off at the end.
__device__ inline void widen(float (&hi)[8], float (&lo)[8], uint32_t code, float scale) {
    const uint32_t w[4] = {two_values<0>(code, scale), two_values<1>(code, scale), two_values<2>(code, scale),
                           two_values<3>(code, scale)};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t u = i & 1 ? w[i >> 1] : w[i >> 1] << 16;
        const float v = __builtin_bit_cast(float, u);
        hi[i] = fmaxf(hi[i], v);
        lo[i] = fminf(lo[i], v);
    }
}
__device__ inline float cut_off(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xFFFF0000u); }

// One workgroup makes one block of one head: T = 2^n >= D / 8 lanes take a token, 8 dimensions each, 256 / T tokens at a time.
// New tokens are quantised and stored, older ones of the block are read back, and both go into the bounds.  What bounds it is the
// bytes: rows are asked for kAhead at a time, and scales, a byte for each 32 elements, are collected in LDS.
template <int D, int NS>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheView c, Tokens t, Rows keys, Rows values) {
    constexpr int kSegs = D / 8;
    constexpr int T = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;
    constexpr int kAtOnce = 256 / T, kAhead = kPage / kAtOnce < 4 ? kPage / kAtOnce : 4;
    typedef typename ElementOf<NS>::type E;
    __shared__ float s_hi[kAtOnce][D], s_lo[kAtOnce][D];
    __shared__ float s_top[4];
    __shared__ int s_bad;
    __shared__ __attribute__((aligned(4))) uint8_t s_scale[2][D / 32][kPage];

    // the heads of a block come one after the other: a token's rows lie side by side (written and read back, 32,768 tokens of 8 heads:
    // 90 us, and 97 with each head's blocks together)
    const int h = blockIdx.x % c.heads;
    Piece w = {(int)blockIdx.x / c.heads, 0};  // without offsets every sequence has one row, in one block
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
    const int64_t unit = page * c.heads + h;
    uint8_t *const kc = c.keys + unit * (kPage * D / 2), *const vc = c.values + unit * (kPage * D / 2);
    uint8_t *const ks = c.key_scales + unit * (kPage * D / 32), *const vs = c.value_scales + unit * (kPage * D / 32);

    const int seg = threadIdx.x % T, at = threadIdx.x / T;
    const uint64_t mine = ((1ull << T) - 1) << ((threadIdx.x & 63) / T * T);  // lanes of my token
    float hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        hi[i] = -INFINITY;
        lo[i] = INFINITY;
    }
    if (threadIdx.x == 0) s_bad = 0;
    for (int i = threadIdx.x; i < 2 * D / 32 * kPage / 4; i += 256) reinterpret_cast<uint32_t *>(s_scale)[i] = 0;
    __syncthreads();
    bool bad = false;
    for (int j0 = 0; j0 < last; j0 += kAtOnce * kAhead) {
        Eight<NS> x[kAhead], y[kAhead];
        uint32_t oldk[kAhead];
        int oldkb[kAhead], oldvb[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int j = j0 + k * kAtOnce + at;
            const bool real = j >= first && j < last && seg < kSegs;
            const int64_t row = row0 + ((int64_t)block * kPage + j - start);
            x[k] = load8<NS>((const E *)keys.at + (real ? row * keys.row + h * keys.head + seg * 8 : 0), real);
            y[k] = load8<NS>((const E *)values.at + (real ? row * values.row + h * values.head + seg * 8 : 0), real);
        }
        if (first > 0) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int j = min(j0 + k * kAtOnce + at, kPage - 1), g = min(seg, kSegs - 1);
                oldk[k] = *reinterpret_cast<const uint32_t *>(kc + j * (D / 2) + g * 4);
                oldkb[k] = ks[(g >> 2) * kPage + j];
                oldvb[k] = vs[(g >> 2) * kPage + j];
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int j = j0 + k * kAtOnce + at;
            const bool fresh = j >= first && j < last, old = j < first;
            int kb, vb;
            bool kf, vf;
            uint32_t kcode = quantise8<NS>(x[k], &kb, &kf), vcode = quantise8<NS>(y[k], &vb, &vf);
            kf = !(__ballot(!kf) & mine);  // one element that is not finite spoils the token
            vf = !(__ballot(!vf) & mine);
            if (!kf) kcode = 0, kb = kNotFinite;
            if (!vf) vcode = 0, vb = kNotFinite;
            if (old) kcode = oldk[k], kb = oldkb[k], vb = oldvb[k];
            if (seg < kSegs && (fresh || old)) {
                if (fresh) {
                    *reinterpret_cast<uint32_t *>(kc + j * (D / 2) + seg * 4) = kcode;
                    *reinterpret_cast<uint32_t *>(vc + ((j >> 2) * kSegs + seg) * 16 + (j & 3) * 4) = vcode;
                }
                if ((seg & 3) == 0) {
                    s_scale[0][seg >> 2][j] = (uint8_t)kb;
                    s_scale[1][seg >> 2][j] = (uint8_t)vb;
                }
                bad |= kb == kNotFinite || vb == kNotFinite;
                if (kb != kNotFinite) widen(hi, lo, kcode, __builtin_bit_cast(float, (uint32_t)kb << 23));
            }
        }
    }
    if (seg < kSegs) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            s_hi[at][seg * 8 + i] = cut_off(hi[i]);
            s_lo[at][seg * 8 + i] = cut_off(lo[i]);
        }
    }
    if (bad) s_bad = 1;
    __syncthreads();
    // scales four tokens at a time; behind the last token a word is filled up with zeros
    for (int i = threadIdx.x; i < 2 * D / 32 * kPage / 4; i += 256) {
        const int word = i % (kPage / 4), g = i / (kPage / 4) % (D / 32), which = i / (kPage / 4) / (D / 32);
        if (word >= first >> 2 && word * 4 < last)
            reinterpret_cast<uint32_t *>(which ? vs : ks)[g * (kPage / 4) + word] = *reinterpret_cast<const uint32_t *>(&s_scale[which][g][word * 4]);
    }
    // D <= 256: a thread for each dimension
    const int d = threadIdx.x;
    float top = 0, dh = 0, dl = 0;
    if (d < D) {
        dh = s_hi[0][d];
        dl = s_lo[0][d];
        for (int i = 1; i < kAtOnce; i++) {
            dh = fmaxf(dh, s_hi[i][d]);
            dl = fminf(dl, s_lo[i][d]);
        }
        top = fmaxf(fabsf(dh), fabsf(dl));
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
    __syncthreads();
    if (d >= D) return;
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    const bool none = s_bad != 0;
    // values are at least 2^-125 or zero, so the exponent's bits are those of a normal number or all zero
    const int e = max((int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127 - 6, -126);
    const float scale = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
    int8_t *const out = c.bounds + unit * (2 * D);
    out[d] = none ? 0 : (int8_t)ceilf(dh * scale);
    out[D + d] = none ? 0 : (int8_t)floorf(dl * scale);
    if (d == 0) c.bound_scales[unit] = none ? kBoundless : (int8_t)e;
}

// 8 dimensions of one row and head a thread
template <int D, int NS>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheView c, Tokens t, typename ElementOf<NS>::type *keys,
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
            const uint32_t kw = *reinterpret_cast<const uint32_t *>(c.keys + unit * (kPage * D / 2) + j * (D / 2) + seg * 4);
            const uint32_t vw = *reinterpret_cast<const uint32_t *>(c.values + unit * (kPage * D / 2) + ((j >> 2) * kSegs + seg) * 16 + (j & 3) * 4);
            const int64_t s = unit * (kPage * D / 32) + (seg >> 2) * kPage + j;
            const float ks = __builtin_bit_cast(float, (uint32_t)c.key_scales[s] << 23);
            const float vs = __builtin_bit_cast(float, (uint32_t)c.value_scales[s] << 23);
            const bf16x8 kx = eight_values(kw, ks), vx = eight_values(vw, vs);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                k[e] = (float)kx[e];
                v[e] = (float)vx[e];
            }
        }
        store8<NS>(keys + i * 8, k);
        store8<NS>(values + i * 8, v);
    }
}

__global__ __launch_bounds__(256) void cache_bounds_kernel(CacheView c, const int32_t *pages, int64_t n, float *out) {
    const int per = 2 * c.dim;
    const int64_t all = n * c.heads * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t unit = i / per;
        const int h = (int)(unit % c.heads), d = (int)(i % per);
        const int64_t page = pages[unit / c.heads];
        float v = 0;
        if (page >= 0 && page < c.pages) {
            const int64_t u = page * c.heads + h;
            const int e = c.bound_scales[u];
            v = e == kBoundless ? (d < c.dim ? INFINITY : -INFINITY)
                                : (float)c.bounds[u * per + d] * __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
        }
        out[i] = v;
    }
}

template <int NS>
int write_rows(const CacheView &c, const Tokens &t, Rows k, Rows v, hipStream_t stream) {
    // a sequence's n rows lie in at most n / 64 + 2 blocks, one row in one
    const int64_t tiles = t.offsets ? (int64_t)t.rows / kPage + 2 * sequences_with_rows(t) : t.rows;
    VL_REQUIRE(tiles * c.heads <= 4 * kMaxBlocks, "more sequences and rows than one call takes: %lld blocks", (long long)tiles);
    for_dim(c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        cache_write_kernel<D, NS><<<(unsigned)(tiles * c.heads), 256, 0, stream>>>(c, t, k, v);
    });
    VL_LAUNCH_CHECK("cache_write_kernel");
    return VL_OK;
}

template <int NS>
int read_rows(const CacheView &c, const Tokens &t, void *keys, void *values, hipStream_t stream) {
    typedef typename ElementOf<NS>::type E;
    for_dim(c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        cache_read_kernel<D, NS><<<vl_grid_for((int64_t)t.rows * c.heads * (D / 8), 256), 256, 0, stream>>>(c, t, (E *)keys, (E *)values);
    });
    VL_LAUNCH_CHECK("cache_read_kernel");
    return VL_OK;
}

}  // namespace

VL_EXPORT int vl_cache_write(const vl_cache *cache, const vl_tokens *tokens, int type, const void *keys, int64_t key_row,
                             int64_t key_head, const void *values, int64_t value_row, int64_t value_head, void *stream) {
    CacheView c;
    Tokens t;
    int rc = vl_cache_of(cache, &c);
    if (rc == VL_OK) rc = vl_tokens_of(tokens, &t);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(type >= VL_BF16 && type <= VL_F32, "type: %d", type);
    if (t.rows == 0 || c.pages == 0) return VL_OK;
    VL_REQUIRE(keys && values, "keys or values is null");
    const int size = type == VL_F32 ? 4 : 2;
    VL_REQUIRE(((uintptr_t)keys | (uintptr_t)values) % size == 0, "keys or values not aligned to their type");
    const Rows k = {keys, key_row, key_head}, v = {values, value_row, value_head};
    const hipStream_t s = (hipStream_t)stream;
    return type == VL_BF16 ? write_rows<1>(c, t, k, v, s) : type == VL_F16 ? write_rows<2>(c, t, k, v, s) : write_rows<3>(c, t, k, v, s);
}

VL_EXPORT int vl_cache_read(const vl_cache *cache, const vl_tokens *tokens, int type, void *keys, void *values, void *stream) {
    CacheView c;
    Tokens t;
    int rc = vl_cache_of(cache, &c);
    if (rc == VL_OK) rc = vl_tokens_of(tokens, &t);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(type >= VL_BF16 && type <= VL_F32, "type: %d", type);
    if (t.rows == 0) return VL_OK;
    VL_REQUIRE(keys && values, "keys or values is null");
    VL_REQUIRE((((uintptr_t)keys | (uintptr_t)values) & 15) == 0, "keys or values not on a 16-byte boundary");
    const hipStream_t s = (hipStream_t)stream;
    return type == VL_BF16 ? read_rows<1>(c, t, keys, values, s) : type == VL_F16 ? read_rows<2>(c, t, keys, values, s) : read_rows<3>(c, t, keys, values, s);
}

VL_EXPORT int vl_cache_read_bounds(const vl_cache *cache, const int32_t *pages, int64_t n, float *out, void *stream) {
    CacheView c;
    const int rc = vl_cache_of(cache, &c);
    if (rc != VL_OK) return rc;
    VL_REQUIRE(n >= 0 && n < (1ll << 40), "n: %lld", (long long)n);
    if (n == 0) return VL_OK;
    VL_REQUIRE(pages && out, "pages or out is null");
    cache_bounds_kernel<<<vl_grid_for(n * c.heads * 2 * c.dim, 256), 256, 0, (hipStream_t)stream>>>(c, pages, n, out);
    VL_LAUNCH_CHECK("cache_bounds_kernel");
    return VL_OK;
}
