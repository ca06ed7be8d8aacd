// Products with 4-bit weights.  A matrix [N, K] is N rows of K / 2 bytes, the even column of a byte in its low four bits, in groups of
// `group` columns with a scale and a zero point each: w[n, k] = scale[n, k / group] * (code[n, k] - zero[n, k / group]), zero 8 where
// none are given.  The sum of a group runs over the bare differences (small integers, exact in every type) and meets its scale once:
//   out[m, n] = T( sum over groups of scale[n, g] * sum over k in g of act[m, k] * (code[n, k] - zero[n, g]) )
// in 32 bits, rounded at the store; with int8 activations the inner sum is exact in int32 and the row's scale is applied last.
#include <algorithm>
#include <atomic>

#include "int4_stream.h"
#include "int4_tile.h"
#include "stream_block.h"

namespace mynn {

constexpr int kCus = 256;

// Few rows, of whole slices of 128 columns, for which eight waves hold the activations of all of K: more rows would be read several times over
// (4096 x 14336, 16 rows, us: 40 this way, 17 as tiles).  Up to eight rows are always streamed (8 rows of 4096 x 14336 18).  From nine on it is not the
// faster form everywhere (us, this way and as tiles: fp16, 16 rows of 2560 x 2048 7.1 and 9.1, 11264 x 2048 12.9 and 12.6, 28672 x 4096 27 and 25.6, 4096 x
// 4096 12.6 and 9.8; 24 rows of 2560 x 2048 8.5 and 9.4, 11264 x 2048 11.9 and 13.2; 32 rows of 32000 x 2048 19.6 and 15.1), but the one that
// needs no workspace and one launch, captured too.
static bool int4_streams(const Int4Args &a) {
    const int rows = a.M <= 8 ? 1 : a.M <= 16 ? 4096 : a.M <= 32 ? 2048 : 0;
    return (rows == 1 || a.K <= (a.group == 32 ? rows / 2 : rows)) && a.K % 128 == 0 && a.N >= 16;
}

// room for `bytes` of LDS a workgroup, asked for once a kernel and device (done: the devices' bits)
static int int4_lds(const void *kernel, int bytes, std::atomic<uint64_t> &done) {
    int device = 0;
    MYNN_HIP(hipGetDevice(&device));
    const uint64_t bit = (uint64_t)1 << (device & 63);
    if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return 0;
    MYNN_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

template <typename T, bool I8, int FL> static int int4_stream(const Int4Args &a, hipStream_t s) {
    auto go = [&](auto mp_, auto p_, auto d_, auto mt_) {
        constexpr int MP = decltype(mp_)::value, P = decltype(p_)::value, D = decltype(d_)::value, MT = decltype(mt_)::value;
        constexpr int OUT = MP * MP * MT;
        const int units = (a.K / 128 + 16 / MP * P - 1) / (16 / MP * P), tiles = (a.N + MP - 1) / MP;
        Int4Stream plan;
        plan.slabs = (units + 7) / 8;
        plan.over_k = (units + plan.slabs - 1) / plan.slabs;
        // eight waves a compute unit: each loads its activations once (twelve, 28672 x 4096, one row: 14.1 -> 15.6 us; six: 16.4)
        const int turns = std::max(1, 4 / plan.over_k), slots = kCus * 8 / plan.over_k;
        // (a workgroup's results of all its tiles lie in LDS)
        const int most = std::max(1, (MP < 16 ? 32 : 128) * 1024 / (plan.over_k * OUT * (int)sizeof(float)) / turns);
        plan.per_wave = std::min(std::min(most, 64), (tiles + slots - 1) / slots);
        plan.tiles = turns * plan.per_wave;
        const size_t lds = (size_t)plan.tiles * plan.over_k * OUT * sizeof(float);
        if (MP == 16) {
            static std::atomic<uint64_t> set{0};
            if (const int rc = int4_lds((const void *)int4_stream_kernel<T, I8, FL, MP, P, D, MT>, 128 * 1024, set)) return rc;
        }
        MYNN_LAUNCH((int4_stream_kernel<T, I8, FL, MP, P, D, MT>), dim3((tiles + plan.tiles - 1) / plan.tiles), dim3(64 * turns * plan.over_k), lds, s, a, plan);
        return launch_status("int4_stream_kernel");
    };
    using std::integral_constant;
    // (P, D): units of 128 S columns of a wave's share, tiles in flight.  Larger shares where eight waves do not cover K otherwise (4096 x 14336, us,
    // four rows: 14.4 -> 12.1, eight 19.4 -> 17.6; elsewhere slower: 28672 x 4096, one row 14 -> 21).
    auto shares = [&](auto mp) {
        constexpr int MP = decltype(mp)::value;
        if constexpr (FL > 1) {
            if (a.K > 128 * (16 / MP) * 2 * 8) return go(mp, integral_constant<int, 4>{}, integral_constant<int, 2>{}, integral_constant<int, 1>{});
        }
        if (MP == 1 && a.K <= 2048) return go(mp, integral_constant<int, 1>{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
        return go(mp, integral_constant<int, 2>{}, integral_constant<int, 3>{}, integral_constant<int, 1>{});
    };
    if (a.M == 1) return shares(integral_constant<int, 1>{});
    if (a.M == 2) return shares(integral_constant<int, 2>{});
    if (a.M <= 4) return shares(integral_constant<int, 4>{});
    if (a.M <= 8) return shares(integral_constant<int, 8>{});
    constexpr integral_constant<int, 16> full{};
    if (a.M <= 16) return go(full, integral_constant<int, FL == 1 ? 2 : 4>{}, integral_constant<int, 2>{}, integral_constant<int, 1>{});
    return go(full, integral_constant<int, FL == 1 ? 1 : 2>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
}

// Heights of the row tiles, in blocks of 32 rows: four as often as they go and the rest in a short tile, or all (but for one block) alike, by
// how long the last compute unit is busy.  A tile of h blocks takes some h + 1.5 units, of int8 h + 2.2 (one round of K = 4096, us: 44, 54,
// 69, 90 for one to four blocks of fp16, 42, 51, 61, 68 of int8).
static Int4Rows int4_row_tiles(int M, int columns, double fixed, int most) {
    const int blocks = (M + 31) / 32;
    auto busy = [&](const Int4Rows &r) {
        const double high = r.high + fixed, low = r.low ? r.low + fixed : 0.0;
        const long long tall = (long long)r.tall * columns, others = (long long)(r.tiles - r.tall) * columns, over = tall % kCus;
        // (the short tiles go beside the tall ones of the last round, and on from there)
        const long long beside = over && others ? (kCus - over) * (long long)(high / low) : 0;
        return (double)((tall + kCus - 1) / kCus) * high + (others > beside ? (double)((others - beside + kCus - 1) / kCus) * low : 0.0);
    };
    Int4Rows best{blocks / most, most, blocks % most, (blocks + most - 1) / most};
    if (!best.tall) best = {1, blocks, 0, 1};
    for (int tiles = (blocks + most - 1) / most; tiles <= blocks; tiles++) {
        const int low = blocks / tiles, over = blocks % tiles;
        const Int4Rows even = over ? Int4Rows{over, low + 1, low, tiles} : Int4Rows{tiles, low, 0, tiles};
        if (busy(even) < busy(best)) best = even;
        if (low == 1 || (long long)tiles * columns > 8 * kCus) break;  // (in many rounds the last one matters little)
    }
    return best;
}

// K ranges of a product whose tiles leave compute units idle, by what they take: a piece 0.85 us, the sums that are left and added up 0.8 us a
// megabyte and a launch of 2.5 us (us with 1 / 2 / 4 / 8 / 16 ranges: 48 x 4096 x 4096 23.8 / 17.7 / 12.3 / 12.7 / 14, 48 x 4096 x 14336 87 / 48 / 29 / 25.6 /
// 23.3, 256 x 2048 x 2048 18.5 / 17.1 / 16.8 / 22, 64 x 11264 x 2048 14.3 / 16.7 / 19.9 / 24, 64 x 28672 x 4096 35.1 / 35.2 / 43).
static int int4_ranges(int M, int N, int K) {
    const long long tiles = ((long long)M + 63) / 64 * ((N + 255ll) / 256), pieces = (K + 127ll) / 128;
    const double sums = 0.8e-6 * M * N * sizeof(float);
    int best = 1;
    double least = 0.85 * pieces;
    for (int r = 2; r <= 32 && r <= kCus / tiles && r <= pieces / 2; r++) {
        const double us = 0.85 * ((pieces + r - 1) / r) + sums * r + 2.5;
        if (us < least) {
            least = us;
            best = r;
        }
    }
    return best;
}
static size_t int4_workspace(const Int4Args &a) {
    const int ranges = int4_streams(a) ? 1 : int4_ranges(a.M, a.N, a.K);
    return ranges > 1 ? (size_t)ranges * a.M * a.N * sizeof(float) : 0;
}

static StreamBlocks g_int4_blocks;  // the ranges' sums

// Memory for the ranges' sums: the caller's, the stream's block, or none: a captured call that was given none takes the ranges one after the
// other (the same bits), so that its graph may be replayed anywhere.
struct Int4Memory {
    bool given;
    void *ptr;
    size_t bytes;
};

template <typename T, bool I8, int FL> static int int4_tiles(const Int4Args &a, const Int4Memory &memory, hipStream_t s) {
    Int4Ranges ranges{int4_ranges(a.M, a.N, a.K), nullptr};
    const size_t total = (size_t)a.M * a.N;
    StreamBlocks::Lease block;
    if (ranges.count > 1 && memory.given) ranges.part = (float *)memory.ptr;
    else if (ranges.count > 1 && !stream_capturing(s)) {
        if (const int rc = g_int4_blocks.lease(s, false, int4_workspace(a), 0, "4-bit product", &block)) return rc;
        ranges.part = (float *)block.ptr;
    }
    const int side = ranges.part ? ranges.count : 1;  // ranges side by side
    auto launch = [&](auto nw_, auto wide, const Int4Rows &rows) {
        constexpr int NW = decltype(nw_)::value;
        constexpr bool WIDE = decltype(wide)::value;
        using G = Int4Tile<I8, FL, NW, WIDE>;
        const long long blocks = (long long)rows.tiles * ((a.N + G::BN - 1) / G::BN) * side;
        MYNN_REQUIRE(blocks < (1ll << 32) / (64 * NW), MYNN_ERR_UNSUPPORTED, "4-bit product: M=%d N=%d", a.M, a.N);  // (the threads of a launch)
        static std::atomic<uint64_t> set{0};
        if (const int rc = int4_lds((const void *)int4_tile_kernel<T, I8, FL, NW, WIDE>, G::LDS, set)) return rc;
        MYNN_LAUNCH((int4_tile_kernel<T, I8, FL, NW, WIDE>), dim3((unsigned)blocks), dim3(64 * NW), G::LDS, s, a, rows, ranges);
        return launch_status("int4_tile_kernel");
    };
    auto go = [&](auto nw, const Int4Rows &rows) {
        // (us, without / with: 24 x 4096 x 14336 of int8, groups of 64 and zero points 22.8 / 20, 64 x 28672 x 4096, groups of 32 and zero points 68 / 50, 411 x 4096 x
        // 14336 125 / 104; groups of 64 without zero points, 2048 x 4096 x 4096 bf16 83.5 / 81.5, 64 x 65536 x 4096 of int8 59.6 / 57.3)
        if constexpr (FL < 4) {
            if (a.K % 128 == 0 && ((uintptr_t)a.scale & 3) == 0 && ((uintptr_t)a.zero & (FL == 1 ? 3 : 1)) == 0) return launch(nw, std::true_type{}, rows);
        }
        return launch(nw, std::false_type{}, rows);
    };
    // Tiles of at most 64 rows: two workgroups of four waves a compute unit, one computes while the other meets at its barrier (us, one of eight / two of
    // four: 128 x 4096 x 4096 19.7 / 16.4, 339 x 2560 x 2048 of int8 23 / 18.5, 64 x 28672 x 4096 35.8 / 34.3; taller tiles are the better ones where
    // there are rows for them, 777 x 28672 x 4096 266 / 231, and three of their stages do not fit twice)
    const Int4Rows rows = int4_row_tiles(a.M, (a.N + 255) / 256 * ranges.count, I8 ? 2.2 : 1.5, ranges.count > 1 ? 2 : 4);
    const int rc = rows.high <= 2 ? go(std::integral_constant<int, 4>{}, rows) : go(std::integral_constant<int, 8>{}, rows);
    if (rc || !ranges.part) return rc;
    // (two values a thread where rows are whole pairs)
    auto join = [&](auto v) {
        constexpr int V = decltype(v)::value;
        MYNN_LAUNCH((int4_join_kernel<T, I8, V>), dim3((unsigned)((total / V + 255) / 256)), dim3(256), 0, s, (T *)a.out, (const float *)ranges.part,
                    (const T *)a.act_scale, ranges.count, (uint32_t)a.N, (uint32_t)total);
        return launch_status("int4_join_kernel");
    };
    return a.N % 2 == 0 ? join(std::integral_constant<int, 2>{}) : join(std::integral_constant<int, 1>{});
}

template <typename T, bool I8, int FL> static int int4_product_of(const Int4Args &a, const Int4Memory &memory, hipStream_t s) {
    return int4_streams(a) ? int4_stream<T, I8, FL>(a, s) : int4_tiles<T, I8, FL>(a, memory, s);
}
template <bool I8> static int int4_product(const Int4Args &a, const Int4Memory &memory, int dtype, hipStream_t s) {
    if (memory.given) {
        const size_t need = int4_workspace(a);
        MYNN_REQUIRE(!need || (memory.ptr && memory.bytes >= need && aligned16(memory.ptr)), MYNN_ERR_INVALID,
                     "4-bit product: %zu bytes of workspace, 16-byte aligned, are needed", need);
    }
    return dispatch_dtype16(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return a.group == 32 ? int4_product_of<T, I8, 1>(a, memory, s) : a.group == 64 ? int4_product_of<T, I8, 2>(a, memory, s) : int4_product_of<T, I8, 4>(a, memory, s);
    });
}

// c / (pieces of a group) as the upper half of a product: exact while (pieces of a row) * (pieces of a group) < 2^32
static uint32_t pieces_magic(int group) { return group <= 128 ? 0u : (uint32_t)((((uint64_t)1 << 32) + group / 128 - 1) / (group / 128)); }

static int check_int4(const char *who, const void *out, const void *act, const void *wq, const void *scale, int M, int N, int K, int group) {
    MYNN_REQUIRE(out && act && wq && scale && M > 0 && N > 0 && K > 0, MYNN_ERR_INVALID, "%s: bad operand (M=%d N=%d K=%d)", who, M, N, K);
    MYNN_REQUIRE(group == 32 || group == 64 || (group > 0 && group % 128 == 0), MYNN_ERR_UNSUPPORTED, "%s: group=%d (32, 64 or a multiple of 128)", who, group);
    MYNN_REQUIRE(K % group == 0, MYNN_ERR_INVALID, "%s: K=%d is no multiple of the group of %d", who, K, group);
    MYNN_REQUIRE(K <= 1 << 22 && M <= 1 << 30 && N <= 1 << 30, MYNN_ERR_UNSUPPORTED, "%s: M=%d N=%d K=%d", who, M, N, K);
    MYNN_REQUIRE(aligned16(act) && aligned16(wq), MYNN_ERR_INVALID, "%s: activations and weights have to be 16-byte aligned", who);
    return 0;
}

}  // namespace mynn

using namespace mynn;

static int dequant_matmul_int4(void *out, const void *act, const uint8_t *wq, const void *scale, const uint8_t *zero, int M, int N, int K, int group, int dtype,
                               const Int4Memory &memory, mynn_stream s) {
    if (int rc = check_int4("dequant_matmul_int4", out, act, wq, scale, M, N, K, group)) return rc;
    return int4_product<false>(Int4Args{out, act, nullptr, wq, scale, zero, M, N, K, group, pieces_magic(group)}, memory, dtype, as_stream(s));
}
static int quantized_matmul_int4(void *out, const int8_t *lhs, const void *lhs_scale, const uint8_t *wq, const void *scale, const uint8_t *zero, int M, int N,
                                 int K, int group, int dtype, const Int4Memory &memory, mynn_stream s) {
    if (int rc = check_int4("quantized_matmul_int4", out, lhs, wq, scale, M, N, K, group)) return rc;
    MYNN_REQUIRE(lhs_scale, MYNN_ERR_INVALID, "quantized_matmul_int4: lhs_scale is null");
    return int4_product<true>(Int4Args{out, lhs, lhs_scale, wq, scale, zero, M, N, K, group, pieces_magic(group)}, memory, dtype, as_stream(s));
}

extern "C" size_t mynn_matmul_int4_workspace_bytes(int M, int N, int K, int group) {
    if (M < 1 || N < 1 || K < 1 || group < 1 || M > 1 << 30 || N > 1 << 30 || K > 1 << 22) return 0;
    Int4Args a{};
    a.M = M, a.N = N, a.K = K, a.group = group;
    return int4_workspace(a);
}

extern "C" int mynn_dequant_matmul_int4(void *out, const void *act, const uint8_t *wq, const void *scale, const uint8_t *zero, int M, int N, int K,
                                        int group, int dtype, mynn_stream s) {
    return dequant_matmul_int4(out, act, wq, scale, zero, M, N, K, group, dtype, Int4Memory{}, s);
}
extern "C" int mynn_dequant_matmul_int4_ws(void *out, const void *act, const uint8_t *wq, const void *scale, const uint8_t *zero, int M, int N, int K,
                                           int group, int dtype, void *workspace, size_t workspace_bytes, mynn_stream s) {
    return dequant_matmul_int4(out, act, wq, scale, zero, M, N, K, group, dtype, Int4Memory{true, workspace, workspace_bytes}, s);
}

extern "C" int mynn_quantized_matmul_int4(void *out, const int8_t *lhs, const void *lhs_scale, const uint8_t *wq, const void *scale, const uint8_t *zero,
                                          int M, int N, int K, int group, int dtype, mynn_stream s) {
    return quantized_matmul_int4(out, lhs, lhs_scale, wq, scale, zero, M, N, K, group, dtype, Int4Memory{}, s);
}
extern "C" int mynn_quantized_matmul_int4_ws(void *out, const int8_t *lhs, const void *lhs_scale, const uint8_t *wq, const void *scale, const uint8_t *zero,
                                             int M, int N, int K, int group, int dtype, void *workspace, size_t workspace_bytes, mynn_stream s) {
    return quantized_matmul_int4(out, lhs, lhs_scale, wq, scale, zero, M, N, K, group, dtype, Int4Memory{true, workspace, workspace_bytes}, s);
}
