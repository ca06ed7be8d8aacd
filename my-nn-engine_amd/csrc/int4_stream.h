// Few rows of activations times 4-bit weights: the activations stay in registers and the weights stream past them.
//
// The 16 x 16 x 32 matrix instruction has room for 16 rows; with M <= MP of them (MP = 1, 2, 4, 8) the others are S = 16 / MP slices of K.  Row
// (slice a, m) holds act[m] of slice a, column (weight row w, slice b) the codes of slice b of one of MP weight rows, and of the 16 x 16 sums
// those with a = b are the product's.  A slice is 128 columns, so an instruction's operands cover 128 S columns (with one row 2048: a kilobyte
// of one weight row, 64 bytes a slice, 16 a lane), the wave's activations stay in 16 registers for each 128 S columns of its share of K
// for all the weight rows it takes, and a tile asks for its codes, scales and zero points alone.  (With the activations loaded again for every 16 weight
// rows, four loads for each one of weights, 128256 x 4096 took 92 us for one row; now 48 to 49, 5.6 TB/s, part of
// it from the 256 MB cache.)
//
// From nine rows on MP is 16: one slice, MT tiles of 16 rows, nothing to be summed inside a wave.
//
// A wave keeps D tiles of MP weight rows in flight.  What it leaves of a tile is summed over its slices in registers and over the waves that
// share K in LDS, in their order.
#pragma once
#include "int4_codes.h"

namespace mynn {

// Codes go to the matrix cores as fp16 (Int4Pairs), and bf16 activations with them: to bf16 a code less its zero point is 19 operations for eight, to
// fp16 nine (one row of 128256 x 4096: 67 us, and 48).  A wave holds its share of a row times the power of two that takes the row's largest value to
// 2^14.  What is not below 2^-31 of that value is an fp16 number then, exactly (eight bits, and the subnormal numbers go down to 2^-24).  A wave that
// finds a value below begins again with passes for such rows: zero in the first, they come in the next, by the largest of what is left.  So products
// are those of the bf16 values, and a row's sums do not depend on the other rows.  (The conversion is 0.3 us for 64 values a lane; four and eight rows of
// 4096 x 14336, with twice as many, take 14.8 and 18.4 us, and took 13.8 and 17.6 with sums of codes and zero points apart.)

// the halves of two dwords of 16-bit values
__device__ inline uint32_t int4_lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ inline uint32_t int4_highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// the largest and the smallest magnitude (zeros apart) of bf16 values, as bits
struct Int4Extent {
    typedef unsigned short two_t __attribute__((ext_vector_type(2)));
    two_t most_ = {0, 0}, least_ = {0xFFFF, 0xFFFF};
    __device__ void add(const U4 &v) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const two_t b = __builtin_bit_cast(two_t, v[i] & 0x7FFF7FFFu);
            most_ = __builtin_elementwise_max(most_, b);
            least_ = __builtin_elementwise_min(least_, (two_t)(b - (two_t){1, 1}));
        }
    }
    __device__ uint32_t most() const { return max((uint32_t)most_[0], (uint32_t)most_[1]); }
    __device__ uint32_t least() const { return min((uint32_t)least_[0], (uint32_t)least_[1]) + 1u; }  // (2^16: all are zero)
};
// over the lanes whose column is the same modulo MP
template <int MP> __device__ inline uint32_t int4_same_row_max(uint32_t v) {
    auto ror = [&](auto n) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x120 + decltype(n)::value, 0xF, 0xF, false); };
    if constexpr (MP <= 8) v = max(v, ror(std::integral_constant<int, 8>{}));
    if constexpr (MP <= 4) v = max(v, ror(std::integral_constant<int, 4>{}));
    if constexpr (MP <= 2) v = max(v, ror(std::integral_constant<int, 2>{}));
    if constexpr (MP <= 1) v = max(v, ror(std::integral_constant<int, 1>{}));
    float a = __builtin_bit_cast(float, v), b = a;
    permlane16_swap(a, b);
    v = max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    a = b = __builtin_bit_cast(float, v);
    permlane32_swap(a, b);
    return max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}
// The power of two for a largest magnitude (its bits), the one that takes it back, and the bits of the smallest magnitude that a pass takes.  The smallest
// numbers are multiplied by 2^126, and all are taken.  An infinity or a NaN decides its row alone and stays one; the rest of that row is to stay finite.
struct Int4Scale {
    float to, back;
    uint32_t from;
    __device__ explicit Int4Scale(uint32_t most) {
        const uint32_t exponent = most >> 7, up = min(268u - exponent, 253u);
        to = __builtin_bit_cast(float, up << 23);
        back = __builtin_bit_cast(float, (254u - up) << 23);
        from = exponent == 255u ? 0u : (max(exponent, 31u) - 31u) << 7;
    }
    // eight values in the order of Int4Pairs (rounded nowhere)
    __device__ U4 pairs(const U4 &v) const {
        auto two = [&](uint32_t x, uint32_t y) {
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__builtin_bit_cast(float, x) * to, __builtin_bit_cast(float, y) * to));
        };
        auto high = [](uint32_t x) { return x & 0xFFFF0000u; };
        return U4{two(v[0] << 16, v[2] << 16), two(high(v[0]), high(v[2])), two(v[1] << 16, v[3] << 16), two(high(v[1]), high(v[3]))};
    }
};
// zero in the place of values whose magnitude is not in [from, to)
__device__ inline void int4_keep(U4 &v, uint32_t from, uint32_t to) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t l = v[i] & 0x7FFFu, h = (v[i] >> 16) & 0x7FFFu;
        v[i] &= (l >= from && l < to ? 0xFFFFu : 0u) | (h >= from && h < to ? 0xFFFF0000u : 0u);
    }
}

struct Int4Stream {
    int over_k, slabs, tiles, per_wave;  // waves that share K, rounds of them over K, tiles of a workgroup, tiles of a wave
};

template <typename T, bool I8, int FL, int MP, int P, int D, int MT>
__global__ __launch_bounds__(512) void int4_stream_kernel(Int4Args p, Int4Stream plan) {
    constexpr int S = 16 / MP, AV = I8 ? 2 : 4, EB = I8 ? 1 : 2, PARTS = 4 / FL;
    constexpr int V = MP < 4 ? MP : 4;  // values of a lane that are the product's
    static_assert(MT == 1 || MP == 16, "further tiles of rows behind a full one");
    constexpr int OUT = MP * MP * MT;  // values of a tile
    constexpr bool SCALED = !I8 && std::is_same<T, bf16_t>::value;
    using Acc = std::conditional_t<I8, i4_t, f4_t>;
    extern __shared__ __align__(16) float red[];  // [tile][wave over K][tile of rows][weight row][m]
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int share = wave % plan.over_k, turn = wave / plan.over_k, turns = (blockDim.x >> 6) / plan.over_k;
    const int groups = p.K / p.group, slices = p.K >> 7, half = p.K >> 1;
    const int wrow = col / S, b = col % S;
    const int first = blockIdx.x * plan.tiles, last = min(first + plan.tiles, (p.N + MP - 1) / MP);

    // the one of the four sums (or two, of two rows) that belongs to this lane's slice, and whether it is this lane's at all
    auto pick = [&](const auto &c, float *v) {
        if constexpr (MP == 1) {
            const auto lo = b & 1 ? c[1] : c[0], hi = b & 1 ? c[3] : c[2];
            v[0] = (float)(b & 2 ? hi : lo);
        } else if constexpr (MP == 2) {
#pragma unroll
            for (int m = 0; m < 2; m++) v[m] = (float)(b & 1 ? c[2 + m] : c[m]);
        } else {
#pragma unroll
            for (int m = 0; m < 4; m++) v[m] = (float)c[m];
        }
    };
    const bool mine = MP == 1 ? kg == b >> 2 : MP == 2 ? kg == b >> 1 : MP == 4 ? kg == b : MP == 8 ? kg >> 1 == b : true;

    Int4Pairs conv;
    struct Tile {
        U4 w[P];
        uint2 s[P];
        uint32_t z[P];
    };

    // All of K in a pass a slab; false where rows have values below those of a pass.  WIDE: with further passes for those.
    auto run = [&](auto wide_) -> bool {
        constexpr bool WIDE = decltype(wide_)::value;
        bool more = false;
        uint32_t above[MT];
        for (int slab = 0; slab < plan.slabs; slab += !more) {
            const bool begun = slab || more;
            const int sp0 = (slab * plan.over_k + share) * P;
            // this lane's slices as a column; those behind K repeat the last one and count as zero
            uint32_t woff[P], goff[P];
            bool have[P];
#pragma unroll
            for (int q = 0; q < P; q++) {
                const int slice = (sp0 + q) * S + b, at = min(slice, slices - 1);
                have[q] = slice < slices;
                woff[q] = (uint32_t)(wrow * half + at * 64 + kg * 16);
                goff[q] = (uint32_t)(wrow * groups + (FL == 4 ? (p.pieces_magic ? (int)__umulhi((uint32_t)at, p.pieces_magic) : at) : at * PARTS));
            }
            // ... and as a row: its activations
            U4 a[P][MT][AV];
#pragma unroll
            for (int x = 0; x < P * MT; x++) {
                const int q = x / MT, mt = x % MT;
                const int slice = (sp0 + q) * S + col / MP;
                const size_t m = min(16 * mt + col % MP, p.M - 1);
                const char *src = (const char *)p.act + (m * p.K + (size_t)min(slice, slices - 1) * 128 + (FL == 4 ? 32 : 8) * kg) * EB;
#pragma unroll
                for (int v = 0; v < AV; v++) {
                    if constexpr (FL == 4) a[q][mt][v] = *(const U4 *)(src + 16 * v);
                    else if constexpr (!I8) a[q][mt][v] = *(const U4 *)(src + 64 * v);
                    else {
                        const uint2 lo = *(const uint2 *)(src + 64 * v), hi = *(const uint2 *)(src + 64 * v + 32);
                        a[q][mt][v] = U4{lo.x, lo.y, hi.x, hi.y};
                    }
                    if (slice >= slices) a[q][mt][v] = U4{0u, 0u, 0u, 0u};
                }
            }
            float unit[MT][V];  // (what a sum of the lane is to be multiplied by)
            if constexpr (SCALED) {
                bool low = false;
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    auto each = [&](auto &&f) {
#pragma unroll
                        for (int x = 0; x < P * AV; x++) f(a[x / AV][mt][x % AV]);
                    };
                    if (WIDE && more) each([&](U4 &v) { int4_keep(v, 0u, above[mt]); });
                    Int4Extent extent;
                    each([&](const U4 &v) { extent.add(v); });
                    const Int4Scale scale(int4_same_row_max<MP>(extent.most()));
                    above[mt] = scale.from;
                    const bool some = extent.least() < scale.from;
                    low = low || some;
                    if (WIDE && __any(some)) each([&](U4 &v) { int4_keep(v, scale.from, 0x8000u); });
                    each([&](U4 &v) { v = scale.pairs(v); });
#pragma unroll
                    for (int m = 0; m < V; m++)
                        unit[mt][m] = MP <= 4 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale.back), m))
                                              : __shfl(scale.back, 4 * (MP == 8 ? kg & 1 : kg) + m);
                }
                more = __any(low);
                if (!WIDE && more) return false;
            } else if constexpr (!I8) {
#pragma unroll
                for (int x = 0; x < P * MT * AV; x++) {
                    U4 &v = a[x / (MT * AV)][x / AV % MT][x % AV];
                    v = U4{int4_lows(v[0], v[2]), int4_highs(v[0], v[2]), int4_lows(v[1], v[3]), int4_highs(v[1], v[3])};
                }
            }
            auto load = [&](Tile &t, int tile) {
                const size_t row0 = min(min(tile, last - 1) * MP, p.N - MP);  // (the last tile may take rows of the one before again)
                const uint8_t *w = p.wq + row0 * half;
                const T *s = (const T *)p.scale + row0 * groups;
                const uint8_t *z = p.zero ? p.zero + row0 * groups : nullptr;
#pragma unroll
                for (int q = 0; q < P; q++) {
                    t.w[q] = __builtin_nontemporal_load((const U4 *)(w + woff[q]));
                    if constexpr (FL == 4) t.s[q].x = ((const uint16_t *)s)[goff[q]];
                    else if constexpr (FL == 2) __builtin_memcpy(&t.s[q].x, s + goff[q], 4);
                    else __builtin_memcpy(&t.s[q], s + goff[q], 8);
                    if (z) __builtin_memcpy(&t.z[q], z + goff[q], PARTS);
                }
            };
            auto compute = [&](Tile &t, int tile) {
                float tot[MT][V];
#pragma unroll
                for (int x = 0; x < MT * V; x++) tot[x / V][x % V] = 0.f;
#pragma unroll
                for (int q = 0; q < P; q++) {
                    if constexpr (FL < 4) int4_transpose(t.w[q]);
                    const uint32_t zeros = p.zero ? t.z[q] : 0x08080808u;
#pragma unroll
                    for (int part = 0; part < PARTS; part++) {
                        const uint32_t z = (zeros >> (8 * part)) & 15u;
                        Acc acc[MT];
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) acc[mt] = Acc{0, 0, 0, 0};
                        if constexpr (!I8) conv.at(z);
#pragma unroll
                        for (int i = 0; i < FL; i++) {
                            const int j = part * FL + i;
                            if constexpr (I8) {
                                const uint2 d = int4_to_i8(t.w[q][j], z * 0x01010101u);
#pragma unroll
                                for (int mt = 0; mt < MT; mt++) {
                                    const uint2 x = uint2{a[q][mt][j >> 1][2 * (j & 1)], a[q][mt][j >> 1][2 * (j & 1) + 1]};
                                    acc[mt] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, x), __builtin_bit_cast(long, d), acc[mt], 0, 0, 0);
                                }
                            } else {
                                const U4 d = conv(t.w[q][j]);
#pragma unroll
                                for (int mt = 0; mt < MT; mt++) acc[mt] = mfma16(a[q][mt][j], d, acc[mt]);
                            }
                        }
                        const uint32_t bits = FL == 4 ? t.s[q].x : (part < 2 ? t.s[q].x : t.s[q].y) >> (16 * (part & 1));
                        const uint16_t sbits = (uint16_t)bits;
                        const float s = have[q] ? Elem<T>::ld((const T *)&sbits, 0) : 0.f;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            float v[V];
                            pick(acc[mt], v);
#pragma unroll
                            for (int m = 0; m < V; m++) tot[mt][m] = fmaf(s, SCALED ? v[m] * unit[mt][m] : v[m], tot[mt][m]);
                        }
                    }
                }
                // over the slices: the lane groups, then the columns of a weight row
#pragma unroll
                for (int x = 0; x < MT * V; x++) {
                    float v = tot[x / V][x % V];
                    if constexpr (MP < 16) v = mine ? v : 0.f;
                    if constexpr (MP == 1) v = wave_sum(v);
                    else if constexpr (MP < 16) {
                        v = group_sum<S>(v);
                        if constexpr (MP < 8) v = xor16_sum(v);
                        v = xor32_sum(v);
                    }
                    tot[x / V][x % V] = v;
                }
                if (MP == 16 || (b == 0 && (MP == 8 ? kg < 2 : kg == 0))) {
                    typedef float vec __attribute__((ext_vector_type(V)));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        vec v, *to = (vec *)(red + (((tile - first) * plan.over_k + share) * MT + mt) * MP * MP + wrow * MP + (MP == 16 ? 4 * kg : MP == 8 ? 4 * (kg & 1) : 0));
#pragma unroll
                        for (int m = 0; m < V; m++) v[m] = tot[mt][m];
                        *to = begun ? *to + v : v;
                    }
                }
            };

            Tile ring[D];
            int tile = first + turn;
#pragma unroll
            for (int d = 0; d < D; d++) load(ring[d], tile + d * turns);
            for (; tile < last; tile += D * turns) {
#pragma unroll
                for (int d = 0; d < D; d++) {
                    if (tile + d * turns < last) compute(ring[d], tile + d * turns);
                    load(ring[d], tile + (D + d) * turns);
                }
            }
        }
        return true;
    };
    if (!run(std::false_type{})) {
        if constexpr (SCALED) run(std::true_type{});
    }
    __syncthreads();
    for (int e = threadIdx.x; e < (last - first) * OUT; e += blockDim.x) {
        const int tile = e / OUT, m = e / MP % (MP * MT), w = e % MP;  // (m < MP of each tile of rows)
        const float *from = red + tile * plan.over_k * OUT + m / MP * MP * MP + w * MP + m % MP;
        float sum = from[0];
        for (int k = 1; k < plan.over_k; k++) sum += from[k * OUT];
        const int own = (first + tile) * MP, n = min(own, p.N - MP) + w;
        if (m < p.M && n >= own) {  // (rows of the tile before are that tile's alone: one store to a place)
            if constexpr (I8) sum *= Elem<T>::ld((const T *)p.act_scale, m);
            Elem<T>::st((T *)p.out, (size_t)m * p.N + n, sum);
        }
    }
}

}  // namespace mynn
