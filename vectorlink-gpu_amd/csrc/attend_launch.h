// Launchers of the kernels of one type of queries.
#pragma once
#include "attend_few.h"
#include "attend_many.h"
#include "attend_step.h"

// f(std::integral_constant<int, C>) for tiles of at most `rows` rows
template <class F>
void for_rows(int rows, F f) {
    if (rows <= 4) f(std::integral_constant<int, 4>());
    else if (rows <= 8) f(std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 16>());
}

template <int D, int NS>
void launch_join(const AttendArgs &a, hipStream_t stream) {
    if (a.splits > 1) attend_join_kernel<D, NS><<<(unsigned)(((int64_t)a.t.rows * a.heads_q + 3) / 4), 256, 0, stream>>>(a);
}

template <int NS, int BITS>
int launch_attend_few(const AttendArgs &a, int64_t tiles, hipStream_t stream) {
    VL_REQUIRE(tiles * a.splits <= 4 * kMaxBlocks, "more rows than one call takes: %lld tiles", (long long)tiles);
    hipError_t e = hipSuccess;
    for_dim(a.c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        const unsigned groups = (unsigned)(tiles * a.splits), heads = (unsigned)a.c.heads;
        for_rows(a.list || !a.t.offsets ? a.group : 16, [&](auto c) {
            constexpr int C = decltype(c)::value;
            auto launch = [&](auto use) {
                constexpr int S = decltype(use)::value;
                if (a.waves == 1) {
                    attend_few_kernel<D, NS, 1, C, BITS, S><<<dim3((unsigned)((tiles + 3) / 4), heads), 256, 0, stream>>>(a, (int)tiles);
                } else if (a.waves == 8) {
                    if constexpr (BITS == 4 && D <= 128) {
                        e = vl_allow_lds(attend_few_kernel<D, NS, 8, C, BITS, S>, sizeof(JoinLds<8>));
                        if (e == hipSuccess) attend_few_kernel<D, NS, 8, C, BITS, S><<<dim3(groups, heads), 512, sizeof(JoinLds<8>), stream>>>(a, (int)tiles);
                    }
                } else {
                    attend_few_kernel<D, NS, 4, C, BITS, S><<<dim3(groups, heads), 256, sizeof(JoinLds<4>), stream>>>(a, (int)tiles);
                }
            };
            if constexpr (BITS == 8) {
                if (a.scores) return launch(std::integral_constant<int, kOnceAndScores>());
                if (C < 16 || (!a.t.offsets && a.group <= 16)) return launch(std::integral_constant<int, kOnce>());
            }
            if constexpr (BITS == 4 || C == 16) launch(std::integral_constant<int, kShared>());
        });
        if (e == hipSuccess) launch_join<D, NS>(a, stream);
    });
    VL_HIP(e);
    VL_LAUNCH_CHECK("attend_few_kernel");
    return VL_OK;
}

template <int NS, int BITS>
int launch_attend_many(const AttendArgs &a, int64_t tiles, hipStream_t stream) {
    const int64_t groups = tiles * a.splits * a.c.heads;
    VL_REQUIRE(groups <= 2 * kMaxBlocks, "more rows than one call takes: %lld tiles", (long long)groups);
    hipError_t e = hipSuccess;
    for_dim(a.c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value, W = many_waves(D), P = many_pages(D);
        if constexpr (many_built(D, NS)) {
            constexpr size_t lds = 2 * P * (Images<D>::kBytes + kPage);
            e = vl_allow_lds(attend_many_kernel<D, NS, W, P, BITS>, lds);
            if (e != hipSuccess) return;
            attend_many_kernel<D, NS, W, P, BITS><<<(unsigned)groups, W * 64, lds, stream>>>(a, (int)tiles);
            launch_join<D, NS>(a, stream);
        }
    });
    VL_HIP(e);
    VL_LAUNCH_CHECK("attend_many_kernel");
    return VL_OK;
}

template <int NS>
int launch_attend_step(const AttendArgs &a, const SelectArgs &s, hipStream_t stream) {
    hipError_t e = hipSuccess;
    const size_t keys = ((size_t)a.t.blocks * 4 + 15) / 16 * 16, join = sizeof(JoinLds<kStepWaves>);
    const size_t lds = (keys > join ? keys : join) + (size_t)s.count * 4;
    for_dim(a.c.dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        if constexpr (step_built(D, NS)) {
            for_rows(a.group, [&](auto c) {
                constexpr int C = decltype(c)::value;
                e = vl_allow_lds(attend_step_kernel<D, NS, C>, lds);
                if (e == hipSuccess) attend_step_kernel<D, NS, C><<<(unsigned)(a.t.rows * (int64_t)a.c.heads), 512, lds, stream>>>(a, s);
            });
        }
    });
    VL_HIP(e);
    VL_LAUNCH_CHECK("attend_step_kernel");
    return VL_OK;
}
