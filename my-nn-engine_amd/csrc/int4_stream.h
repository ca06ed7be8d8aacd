// Few rows of activations times 4-bit weights: the activations stay in registers and the weights stream past them.
//
// The 16 x 16 x 32 matrix instruction has room for 16 rows; with M <= MP of them (MP = 1, 2, 4, 8) the others are S = 16 / MP slices of K.  Row
// (slice a, m) holds act[m] of slice a, column (weight row w, slice b) the codes of slice b of one of MP weight rows, and of the 16 x 16 sums
// those with a = b are the product's.  A slice is 128 columns, so an instruction's operands cover 128 S columns (with one row 2048: a kilobyte
// of one weight row, 64 bytes a slice, 16 a lane), the wave's activations stay in 16 registers for each 128 S columns of its share of K
// for all the weight rows it takes, and a load of weights is the only load there is.  (With the activations loaded again for every 16 weight
// rows, four loads for each one of weights, 128256 x 4096 took 92 us for one row; now 50, 5.4 TB/s.)
//
// From nine rows on MP is 16: one slice, MT tiles of 16 rows, nothing to be summed inside a wave.
//
// A wave keeps D tiles of MP weight rows in flight.  What it leaves of a tile is summed over its slices in registers and over the waves that
// share K in LDS, in their order.
#pragma once
#include "int4_codes.h"

namespace mynn {

struct Int4Stream {
    int over_k, slabs, tiles, per_wave;  // waves that share K, rounds of them over K, tiles of a workgroup, tiles of a wave
};

template <typename T, bool I8, int FL, int MP, int P, int D, int MT>
__global__ __launch_bounds__(512) void int4_stream_kernel(Int4Args p, Int4Stream plan) {
    constexpr int S = 16 / MP, AV = I8 ? 2 : 4, EB = I8 ? 1 : 2, PARTS = 4 / FL;
    constexpr int V = MP < 4 ? MP : 4;  // values of a lane that are the product's
    constexpr bool KEEP = FL == 4 && !I8;  // sums of activations kept (otherwise made again: more registers than a product with ones is worth)
    static_assert(MT == 1 || MP == 16, "further tiles of rows behind a full one");
    constexpr int OUT = MP * MP * MT;  // values of a tile
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

    const U4 ones = std::is_same<T, f16_t>::value ? U4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u}
                                                  : U4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
    struct Tile {
        U4 w[P];
        uint2 s[P];
        uint32_t z[P];
    };

    auto run = [&](auto exact_) -> bool {
        constexpr bool EXACT = decltype(exact_)::value;
        float bad = 0.f;
        for (int slab = 0; slab < plan.slabs; slab++) {
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
            float sa[P][MT][V];
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
                        f4_t sums[MT];
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            acc[mt] = Acc{0, 0, 0, 0};
                            sums[mt] = f4_t{0.f, 0.f, 0.f, 0.f};
                        }
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
                                const U4 d = EXACT ? int4_differences<T>(t.w[q][j], (int)z) : int4_codes<T>(t.w[q][j]);
#pragma unroll
                                for (int mt = 0; mt < MT; mt++) {
                                    acc[mt] = mfma16<T>(a[q][mt][j], d, acc[mt]);
                                    if constexpr (!KEEP && !EXACT) sums[mt] = mfma16<T>(a[q][mt][j], ones, sums[mt]);
                                }
                            }
                        }
                        const uint32_t bits = FL == 4 ? t.s[q].x : (part < 2 ? t.s[q].x : t.s[q].y) >> (16 * (part & 1));
                        const uint16_t sbits = (uint16_t)bits;
                        const float s = have[q] ? Elem<T>::ld((const T *)&sbits, 0) : 0.f;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            float v[V], r[V];
                            pick(acc[mt], v);
                            if constexpr (!I8 && !EXACT) {
                                if constexpr (!KEEP) pick(sums[mt], r);
#pragma unroll
                                for (int m = 0; m < V; m++) v[m] = fmaf(-(float)z, KEEP ? sa[q][mt][m] : r[m], v[m]);
                            }
#pragma unroll
                            for (int m = 0; m < V; m++) tot[mt][m] = fmaf(s, v[m], tot[mt][m]);
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
                    if constexpr (!I8 && !EXACT) bad = fmaf(v, 0.f, bad);
                    tot[x / V][x % V] = v;
                }
                if (MP == 16 || (b == 0 && (MP == 8 ? kg < 2 : kg == 0))) {
                    typedef float vec __attribute__((ext_vector_type(V)));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        vec v, *to = (vec *)(red + (((tile - first) * plan.over_k + share) * MT + mt) * MP * MP + wrow * MP + (MP == 16 ? 4 * kg : MP == 8 ? 4 * (kg & 1) : 0));
#pragma unroll
                        for (int m = 0; m < V; m++) v[m] = tot[mt][m];
                        *to = slab ? *to + v : v;
                    }
                }
            };

            Tile ring[D];
            int tile = first + turn;
#pragma unroll
            for (int d = 0; d < D; d++) load(ring[d], tile + d * turns);
            if constexpr (KEEP && !EXACT) {
#pragma unroll
                for (int x = 0; x < P * MT; x++) {
                    f4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < 4; j++) c = mfma16<T>(a[x / MT][x % MT][j], ones, c);
                    pick(c, sa[x / MT][x % MT]);
                }
            }
            for (; tile < last; tile += D * turns) {
#pragma unroll
                for (int d = 0; d < D; d++) {
                    if (tile + d * turns < last) compute(ring[d], tile + d * turns);
                    load(ring[d], tile + (D + d) * turns);
                }
            }
        }
        return bad == 0.f;  // (not so of an infinity or a NaN)
    };
    bool fine = run(std::false_type{});
    if constexpr (!I8) {
        if (__any(!fine)) run(std::true_type{});
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
