// Products with 4-bit weights.  A matrix [N, K] is N rows of K / 2 bytes, the even column of a byte in its low four bits, in groups of
// `group` columns with a scale and a zero point each: w[n, k] = scale[n, k / group] * (code[n, k] - zero[n, k / group]), zero 8 where
// none are given.  The sum of a group runs over the bare differences (small integers, exact in every type) and meets its scale once:
//   out[m, n] = T( sum over groups of scale[n, g] * sum over k in g of act[m, k] * (code[n, k] - zero[n, g]) )
// in 32 bits, rounded at the store; with int8 activations the inner sum is exact in int32 and the row's scale is applied last.
#include <algorithm>

#include "int4_stream.h"
#include "int4_tile.h"

namespace mynn {

constexpr int kCus = 256;

// Up to 64 rows.  Two weight tiles a wave from 17 rows on: the activations, read from L2 by every workgroup, are then most of what a wave
// loads.  Waves: as many as give each compute unit about 16, no more than there are pieces.
template <typename T, bool I8, int FL> static int int4_rows(const Int4Args &a, hipStream_t s) {
    auto go = [&](auto mt_, auto r_, auto nt_) {
        constexpr int MT = decltype(mt_)::value, R = decltype(r_)::value, NT = decltype(nt_)::value;
        const int blocks = (a.N + 16 * NT - 1) / (16 * NT) * ((a.M + 63) / 64), pieces = (a.K + 127) / 128;
        const int most = MT == 1 ? 16 : 8, share = MT == 1 ? 2 : 1;
        int waves = 1;
        while (waves < most && blocks * waves < kCus * 16 && waves * 2 * share <= pieces) waves *= 2;
        const size_t lds = (size_t)waves * MT * R * NT * 64 * sizeof(float);
        MYNN_LAUNCH((int4_rows_kernel<T, I8, FL, MT, R, NT>), dim3((a.N + 16 * NT - 1) / (16 * NT), (a.M + 63) / 64), dim3(64 * waves), lds, s, a);
        return launch_status("int4_rows_kernel");
    };
    using std::integral_constant;
    if (a.M <= 4) return go(integral_constant<int, 1>{}, integral_constant<int, 1>{}, integral_constant<int, 1>{});
    if (a.M <= 8) return go(integral_constant<int, 1>{}, integral_constant<int, 2>{}, integral_constant<int, 1>{});
    if (a.M <= 16) return go(integral_constant<int, 1>{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
    if (a.M <= 32) return go(integral_constant<int, 2>{}, integral_constant<int, 4>{}, integral_constant<int, 2>{});
    if (a.M <= 48) return go(integral_constant<int, 3>{}, integral_constant<int, 4>{}, integral_constant<int, 2>{});
    return go(integral_constant<int, 4>{}, integral_constant<int, 4>{}, integral_constant<int, 2>{});
}

// Up to 8 rows.  Rows of whole slices, at least a tile of them.
static bool int4_streams(const Int4Args &a) { return a.M <= 8 && a.K % 128 == 0 && a.N >= 8 && (size_t)8 * a.K < 1u << 31; }

template <typename T, bool I8, int FL> static int int4_stream(const Int4Args &a, hipStream_t s) {
    auto go = [&](auto mp_, auto p_, auto d_) {
        constexpr int MP = decltype(mp_)::value, P = decltype(p_)::value, D = decltype(d_)::value;
        const int units = (a.K / 128 + 16 / MP * P - 1) / (16 / MP * P), tiles = (a.N + MP - 1) / MP;
        Int4Stream plan;
        plan.slabs = (units + 7) / 8;
        plan.over_k = (units + plan.slabs - 1) / plan.slabs;
        // eight waves a compute unit: each loads its activations once (twelve, 28672 x 4096, one row: 14.1 -> 15.6 us; six: 16.4)
        const int turns = std::max(1, 4 / plan.over_k), slots = kCus * 8 / plan.over_k;
        const int most = std::max(1, 32768 / (plan.over_k * MP * MP * (int)sizeof(float)) / turns);
        plan.per_wave = std::min(std::min(most, 64), (tiles + slots - 1) / slots);
        plan.tiles = turns * plan.per_wave;
        const size_t lds = (size_t)plan.tiles * plan.over_k * MP * MP * sizeof(float);
        MYNN_LAUNCH((int4_stream_kernel<T, I8, FL, MP, P, D>), dim3((tiles + plan.tiles - 1) / plan.tiles), dim3(64 * turns * plan.over_k), lds, s, a, plan);
        return launch_status("int4_stream_kernel");
    };
    using std::integral_constant;
    // (P, D): units of 128 S columns of a wave's share, tiles in flight.  Larger shares where eight waves do not cover K otherwise (4096 x 14336, us,
    // four rows: 14.4 -> 12.5, eight 19.7 -> 18.1; elsewhere slower: 28672 x 4096, one row 14.1 -> 20.6).
    auto shares = [&](auto mp) {
        constexpr int MP = decltype(mp)::value;
        if constexpr (FL > 1) {
            if (a.K > 128 * (16 / MP) * 2 * 8) return go(mp, integral_constant<int, 4>{}, integral_constant<int, 2>{});
        }
        if (MP == 1 && a.K <= 2048) return go(mp, integral_constant<int, 1>{}, integral_constant<int, 4>{});
        return go(mp, integral_constant<int, 2>{}, integral_constant<int, 3>{});
    };
    if (a.M == 1) return shares(integral_constant<int, 1>{});
    if (a.M == 2) return shares(integral_constant<int, 2>{});
    if (a.M <= 4) return shares(integral_constant<int, 4>{});
    return shares(integral_constant<int, 8>{});
}

template <typename T, bool I8> static int int4_few(const Int4Args &a, hipStream_t s) {
    if (int4_streams(a)) return a.group == 32 ? int4_stream<T, I8, 1>(a, s) : a.group == 64 ? int4_stream<T, I8, 2>(a, s) : int4_stream<T, I8, 4>(a, s);
    if (a.group == 32) return int4_rows<T, I8, 1>(a, s);
    if (a.group == 64) return int4_rows<T, I8, 2>(a, s);
    return int4_rows<T, I8, 4>(a, s);
}

// Heights of the row tiles, in blocks of 32 rows: four as often as they go and the rest in a short tile, or all (but for one block) alike, by
// how long the last compute unit is busy.  A tile of h blocks takes h + 1.5 units, of int8 h + 2.2 (one round of K = 4096, us: 46, 58,
// 80, 104 for one to four blocks of fp16, 40, 48, 60, 75 of int8).
static Int4Rows int4_row_tiles(int M, int columns, double fixed) {
    const int blocks = (M + 31) / 32;
    auto busy = [&](const Int4Rows &r) {
        const double high = r.high + fixed, low = r.low ? r.low + fixed : 0.0;
        const long long tall = (long long)r.tall * columns, others = (long long)(r.tiles - r.tall) * columns, over = tall % kCus;
        // (the short tiles go beside the tall ones of the last round, and on from there)
        const long long beside = over && others ? (kCus - over) * (long long)(high / low) : 0;
        return (double)((tall + kCus - 1) / kCus) * high + (others > beside ? (double)((others - beside + kCus - 1) / kCus) * low : 0.0);
    };
    Int4Rows best{blocks / 4, 4, blocks % 4, (blocks + 3) / 4};
    if (!best.tall) best = {1, blocks, 0, 1};
    for (int tiles = (blocks + 3) / 4; tiles <= blocks; tiles++) {
        const int low = blocks / tiles, over = blocks % tiles;
        const Int4Rows even = over ? Int4Rows{over, low + 1, low, tiles} : Int4Rows{tiles, low, 0, tiles};
        if (busy(even) < busy(best)) best = even;
        if (low == 1) break;
    }
    return best;
}

template <typename T, bool I8, int FL> static int int4_tiles(const Int4Args &a, hipStream_t s) {
    using G = Int4Tile<I8, FL>;
    const int columns = (a.N + G::BN - 1) / G::BN;
    const Int4Rows rows = int4_row_tiles(a.M, columns, I8 ? 2.2 : 1.5);
    MYNN_REQUIRE((long long)rows.tiles * columns < 1 << 30, MYNN_ERR_UNSUPPORTED, "4-bit product: M=%d N=%d", a.M, a.N);
    constexpr int lds = G::NS * G::STAGE;
    static bool lds_set = false;
    if (!lds_set) {
        MYNN_HIP(hipFuncSetAttribute((const void *)int4_tile_kernel<T, I8, FL>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        lds_set = true;
    }
    MYNN_LAUNCH((int4_tile_kernel<T, I8, FL>), dim3(rows.tiles * columns), dim3(512), lds, s, a, rows);
    return launch_status("int4_tile_kernel");
}
template <typename T, bool I8> static int int4_many(const Int4Args &a, hipStream_t s) {
    if (a.group == 32) return int4_tiles<T, I8, 1>(a, s);
    if (a.group == 64) return int4_tiles<T, I8, 2>(a, s);
    return int4_tiles<T, I8, 4>(a, s);
}

// c / (pieces of a group) as the upper half of a product: exact while (pieces of a row) * (pieces of a group) < 2^32
static uint32_t pieces_magic(int group) { return group <= 128 ? 0u : (uint32_t)((((uint64_t)1 << 32) + group / 128 - 1) / (group / 128)); }

static int check_int4(const char *who, const void *out, const void *act, const void *wq, const void *scale, int M, int N, int K, int group) {
    MYNN_REQUIRE(out && act && wq && scale && M > 0 && N > 0 && K > 0, MYNN_ERR_INVALID, "%s: bad operand (M=%d N=%d K=%d)", who, M, N, K);
    MYNN_REQUIRE(group == 32 || group == 64 || (group > 0 && group % 128 == 0), MYNN_ERR_UNSUPPORTED, "%s: group=%d (32, 64 or a multiple of 128)", who, group);
    MYNN_REQUIRE(K % group == 0, MYNN_ERR_INVALID, "%s: K=%d is no multiple of the group of %d", who, K, group);
    MYNN_REQUIRE(K <= 1 << 22, MYNN_ERR_UNSUPPORTED, "%s: K=%d", who, K);
    MYNN_REQUIRE(aligned16(act) && aligned16(wq), MYNN_ERR_INVALID, "%s: activations and weights have to be 16-byte aligned", who);
    return 0;
}

}  // namespace mynn

using namespace mynn;

extern "C" int mynn_dequant_matmul_int4(void *out, const void *act, const uint8_t *wq, const void *scale, const uint8_t *zero, int M, int N, int K,
                                        int group, int dtype, mynn_stream s) {
    if (int rc = check_int4("dequant_matmul_int4", out, act, wq, scale, M, N, K, group)) return rc;
    const Int4Args args{out, act, nullptr, wq, scale, zero, M, N, K, group, pieces_magic(group)};
    return dispatch_dtype16(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        static const int most_few = getenv("I4FEW") ? atoi(getenv("I4FEW")) : 64;
        return M <= most_few ? int4_few<T, false>(args, as_stream(s)) : int4_many<T, false>(args, as_stream(s));
    });
}

extern "C" int mynn_quantized_matmul_int4(void *out, const int8_t *lhs, const void *lhs_scale, const uint8_t *wq, const void *scale, const uint8_t *zero,
                                          int M, int N, int K, int group, int dtype, mynn_stream s) {
    if (int rc = check_int4("quantized_matmul_int4", out, lhs, wq, scale, M, N, K, group)) return rc;
    MYNN_REQUIRE(lhs_scale, MYNN_ERR_INVALID, "quantized_matmul_int4: lhs_scale is null");
    const Int4Args args{out, lhs, lhs_scale, wq, scale, zero, M, N, K, group, pieces_magic(group)};
    return dispatch_dtype16(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        static const int most_few = getenv("I4FEW") ? atoi(getenv("I4FEW")) : 64;
        return M <= most_few ? int4_few<T, true>(args, as_stream(s)) : int4_many<T, true>(args, as_stream(s));
    });
}
