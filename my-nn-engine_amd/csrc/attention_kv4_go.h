// Launches of the forms of attention over 4-bit caches, for the translation unit of a type.
#pragma once
#include "attention_kv4_stream.h"
#include "attention_kv4_tile.h"

namespace mynn {

template <int N> using Int = std::integral_constant<int, N>;
template <typename F> inline int kv4_shape(int D, int group, F &&go) {
    if (D == 64) return group == 64 ? go(Int<64>{}, Int<1>{}) : go(Int<64>{}, Int<2>{});
    return group == 128 ? go(Int<128>{}, Int<1>{}) : group == 64 ? go(Int<128>{}, Int<2>{}) : go(Int<128>{}, Int<4>{});
}

template <typename T, int D, int NG, int FOLD, int W> int kv4_stream_launch(const Kv4Args &a, hipStream_t s) {
    const int R = a.Hq / a.c.Hkv * a.Sq, tile = kKv4TileBytes<D, FOLD>, wave = tile > R * D * 4 ? tile : R * D * 4;
    const int lds = W * (wave + 128) + 16, join = 64 * R * 8;
    MYNN_LAUNCH((attn_kv4_stream_kernel<T, D, NG, FOLD, W>), dim3(a.grid), dim3(W * 64), lds > join + 16 ? lds : join + 16, s, a);
    if (const int rc = launch_status("attn_kv4_stream_kernel")) return rc;
    if (a.counters || a.c.pages_per_seq << a.c.page_shift <= W * kKv4Keys<FOLD>) return 0;  // (a unit each: nothing is shared)
    MYNN_LAUNCH((attn_kv4_join_kernel<T, D, FOLD, W>), dim3(a.B * a.c.Hkv), dim3(256), 0, s, a);
    return launch_status("attn_kv4_join_kernel");
}
template <typename T> int kv4_stream_go(const Kv4Args &a, int D, int group, int fold, int waves, hipStream_t s) {
    return kv4_shape(D, group, [&](auto d, auto n) {
        constexpr int DD = decltype(d)::value, NG = decltype(n)::value;
        if constexpr (NG < 4) {
            if (fold == 4) return waves == 1 ? kv4_stream_launch<T, DD, NG, 4, 1>(a, s) : kv4_stream_launch<T, DD, NG, 4, 4>(a, s);
        }
        if (fold == 2) return waves == 1 ? kv4_stream_launch<T, DD, NG, 2, 1>(a, s) : kv4_stream_launch<T, DD, NG, 2, 4>(a, s);
        return kv4_stream_launch<T, DD, NG, 1, 4>(a, s);
    });
}

template <typename T, int D, int NG, int QW, int KW, int KEYS> static int kv4_tile_launch(const Kv4Args &a, const Kv4TilePlan &p, hipStream_t s) {
    using Block = Kv4Block<D, NG, QW, KW, KEYS>;
    static bool set = false;
    if (!set && Block::LDS > 64 * 1024) {
        MYNN_HIP(hipFuncSetAttribute((const void *)attn_kv4_tile_kernel<T, D, NG, QW, KW, KEYS>, hipFuncAttributeMaxDynamicSharedMemorySize, Block::LDS));
        set = true;
    }
    MYNN_LAUNCH((attn_kv4_tile_kernel<T, D, NG, QW, KW, KEYS>), dim3((unsigned)(a.B * a.c.Hkv * p.blocks * p.ranges)), dim3(Block::THREADS), Block::LDS, s, a);
    return launch_status("attn_kv4_tile_kernel");
}
template <typename T> int kv4_tile_go(const Kv4Args &a, int D, int group, const Kv4TilePlan &p, hipStream_t s) {
    return kv4_shape(D, group, [&](auto d, auto n) {
        constexpr int DD = decltype(d)::value, NG = decltype(n)::value;
        const int rc = p.rows == 32 ? kv4_tile_launch<T, DD, NG, 1, 4, 128>(a, p, s) : p.rows == 64 ? kv4_tile_launch<T, DD, NG, 2, 2, 64>(a, p, s) : kv4_tile_launch<T, DD, NG, 4, 1, 64>(a, p, s);
        if (rc || p.ranges == 1) return rc;
        const size_t threads = (size_t)a.B * a.Hq * a.Sq * (DD / 4);
        MYNN_LAUNCH((attn_kv4_ranges_kernel<T, DD>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, a, p.rows, p.rows == 32 ? 128 : 64);
        return launch_status("attn_kv4_ranges_kernel");
    });
}

}  // namespace mynn
