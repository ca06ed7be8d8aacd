// Few rows of activations times 4-bit weights, on the matrix cores.
//
// A workgroup owns 16 * NT weight rows; its waves deal out K among themselves in pieces and meet in LDS at the end, so the weights are
// read once, by one launch, with no partial sums in memory and one order of sums.  v_mfma 16x16x32 with the activations as the rows and
// the weights as the columns: a lane holds eight codes of one weight row (a dword), the sum of a lane's column is scaled by one number.
// Up to 16 rows cost what one costs -- the stream of weights bounds them all --, up to 64 in MT tiles.
//
// Pieces of 128 columns are 64 bytes of a row, 16 bytes a lane.  Groups of 128 and more: the lane's own 32 columns are multiplied as they
// lie, four instructions of 8 columns from each quarter of the piece.  Groups of 32 and 64 must not meet inside an instruction:
// the four dwords are transposed over the four lanes of a row (two swaps of half waves, two of rows), after which dword j holds the
// columns 32 j .. of the piece.
//
// Codes to 16 bits, nine vector operations for eight: a nibble as a byte is 2^-9 times its value as an fp8 number (e4m3: below 8
// subnormal, from 8 on the first binade, one line), so v_cvt_scalef32_pk makes two exact values of T from two bytes.  The zero point comes off
// the sums: sum a (q - z) = sum a q - z sum a, the second sum a product with ones on the matrix cores, which wait for the weights anyway.
// Taking it off in 16 bits instead costs four more operations in fp16 and ten in bf16, which has no packed arithmetic.  Both sums may
// overflow, or meet an infinity, where their difference does not: a wave whose result is not finite starts again with the differences themselves.
// Int8: nibbles to bytes, the zero point taken off inside the bytes (7 bits apart, no borrow), sums exact.
#pragma once
#include <type_traits>

#include "mfma.h"
#include "mynn_common.h"

namespace mynn {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef int i4_t __attribute__((ext_vector_type(4)));

template <typename T> __device__ inline f4_t mfma16(const U4 &a, const U4 &b, f4_t c) {
    if constexpr (std::is_same<T, f16_t>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}

// the eight codes of a dword as bytes, in their order
__device__ inline uint2 int4_bytes(uint32_t w) {
    const uint32_t e = w & 0x0F0F0F0Fu, o = (w >> 4) & 0x0F0F0F0Fu;
    return uint2{__builtin_amdgcn_perm(o, e, 0x05010400u), __builtin_amdgcn_perm(o, e, 0x07030602u)};
}
// code - zero of the eight as int8 (zz: the zero point in each byte): 0x80 + code - zero never borrows from its neighbour
__device__ inline uint2 int4_to_i8(uint32_t w, uint32_t zz) {
    const uint32_t e = ((w & 0x0F0F0F0Fu) | 0x80808080u) - zz, o = (((w >> 4) & 0x0F0F0F0Fu) | 0x80808080u) - zz;
    return uint2{__builtin_amdgcn_perm(o, e, 0x05010400u) ^ 0x80808080u, __builtin_amdgcn_perm(o, e, 0x07030602u) ^ 0x80808080u};
}
// the eight codes as T
template <typename T> __device__ inline U4 int4_codes(uint32_t w) {
    const uint2 b = int4_bytes(w);
    if constexpr (std::is_same<T, f16_t>::value)
        return U4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b.x, 512.f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b.x, 512.f, true)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b.y, 512.f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b.y, 512.f, true))};
    else
        return U4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b.x, 512.f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b.x, 512.f, true)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b.y, 512.f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b.y, 512.f, true))};
}
// code - zero of the eight as T
template <typename T> __device__ inline U4 int4_differences(uint32_t w, int z) {
    auto two = [&](int i) { return pack2<T>((float)((int)((w >> (8 * i)) & 15u) - z), (float)((int)((w >> (8 * i + 4)) & 15u) - z)); };
    return U4{two(0), two(1), two(2), two(3)};
}
// dword j of lane group g (16 lanes each) <-> dword g of lane group j
__device__ inline void int4_transpose(U4 &d) {
    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
    const u2_t a = __builtin_bit_cast(u2_t, __builtin_amdgcn_permlane32_swap(d.x, d.z, false, false));
    const u2_t b = __builtin_bit_cast(u2_t, __builtin_amdgcn_permlane32_swap(d.y, d.w, false, false));
    const u2_t c = __builtin_bit_cast(u2_t, __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false));
    const u2_t e = __builtin_bit_cast(u2_t, __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false));
    d = U4{c.x, c.y, e.x, e.y};
}

struct Int4Args {
    void *out;
    const void *act, *act_scale;
    const uint8_t *wq;
    const void *scale;
    const uint8_t *zero;
    int M, N, K, group;
    uint32_t pieces_magic;  // 2^32 / (pieces of a group), rounded up; 0: a piece or less
};

// FL: instructions (of 32 columns) to a scale: 1 and 2 for groups of 32 and 64, 4 for longer ones
// R: of the four rows of a tile that a lane holds, how many there are (MT = 1: rows / 4, rounded up); rows are dealt out so that these
// come first: row 4 i + g of a tile is register i of lane group g
template <typename T, bool I8, int FL, int MT, int R, int NT>
__global__ __launch_bounds__(MT == 1 ? 1024 : 512) void int4_rows_kernel(Int4Args p) {
    constexpr int C = MT == 1 ? 2 : 1;  // pieces in flight at a time
    constexpr int AV = I8 ? 2 : 4;      // 16-byte registers of a piece's activations
    using Acc = std::conditional_t<I8, i4_t, f4_t>;
    extern __shared__ __align__(16) float red[];
    const int lane = threadIdx.x & 63, col = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * 64;
    const int groups = p.K / p.group, full = p.K >> 7;
    constexpr int EB = I8 ? 1 : 2;

    const uint8_t *wrow[NT];
    const T *srow[NT];
    const uint8_t *zrow[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const size_t n = min(n0 + 16 * t + col, p.N - 1);
        wrow[t] = p.wq + n * (size_t)(p.K >> 1) + kg * 16;
        srow[t] = (const T *)p.scale + n * groups;
        zrow[t] = p.zero ? p.zero + n * groups : (const uint8_t *)srow[t];  // (any that may be read: no test around the loads)
    }
    const char *arow[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
        const size_t m = min(m0 + 16 * t + (col & 3) * 4 + (col >> 2), p.M - 1);
        arow[t] = (const char *)p.act + (m * p.K + (FL == 4 ? 32 : 8) * kg) * EB;
    }

    struct Piece {
        U4 w[NT], a[MT][AV];
        uint2 s[NT];
        uint32_t z[NT];
    };
    // what a piece needs, of `steps` (1 .. 4) instructions
    auto load = [&](Piece &q, int c, int steps) {
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const char *a = arow[t] + (size_t)c * 128 * EB;
            if constexpr (FL == 4) {
#pragma unroll
                for (int v = 0; v < AV; v++) q.a[t][v] = *(const U4 *)(a + 16 * v);
            } else if constexpr (!I8) {
#pragma unroll
                for (int j = 0; j < 4; j++) q.a[t][j] = *(const U4 *)(a + 64 * min(j, steps - 1));
            } else {
#pragma unroll
                for (int v = 0; v < 2; v++) {
                    const uint2 lo = *(const uint2 *)(a + 32 * min(2 * v, steps - 1)), hi = *(const uint2 *)(a + 32 * min(2 * v + 1, steps - 1));
                    q.a[t][v] = U4{lo.x, lo.y, hi.x, hi.y};
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if constexpr (FL == 4) {
                const int g = p.pieces_magic ? (int)__umulhi((uint32_t)c, p.pieces_magic) : c;
                q.s[t].x = ((const uint16_t *)srow[t])[g];
                q.z[t] = zrow[t][g];
            } else {
                constexpr int P = 4 / FL;  // groups of a piece
                const int g = c * P, have = FL == 1 ? steps : (steps + 1) / 2;
                uint32_t s[4] = {0, 0, 0, 0}, z = 0;
                if (have == P) {  // (of the wave alike)
                    if constexpr (P == 4) __builtin_memcpy(&q.s[t], srow[t] + g, 8);
                    else __builtin_memcpy(&q.s[t].x, srow[t] + g, 4);
                    __builtin_memcpy(&z, zrow[t] + g, P);
                } else {
                    for (int i = 0; i < P; i++) {
                        const int at = g + min(i, have - 1);
                        s[i] = ((const uint16_t *)srow[t])[at];
                        z |= (uint32_t)zrow[t][at] << (8 * i);
                    }
                    q.s[t] = uint2{s[0] | s[1] << 16, s[2] | s[3] << 16};
                }
                q.z[t] = z;
            }
            // (of a broken piece a lane may lie behind the row: it repeats the first lane's)
            q.w[t] = *(const U4 *)(wrow[t] + (size_t)c * 64 - (kg < steps ? 0 : 16 * kg));
        }
    };

    f4_t tot[NT][MT];
    auto compute = [&](Piece &q, int steps, auto exact_) {
        constexpr bool EXACT = decltype(exact_)::value;
        const U4 ones = std::is_same<T, f16_t>::value ? U4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u}
                                                      : U4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
        if constexpr (FL < 4) {
#pragma unroll
            for (int t = 0; t < NT; t++) int4_transpose(q.w[t]);
        }
        if (!p.zero) {
#pragma unroll
            for (int t = 0; t < NT; t++) q.z[t] = 0x08080808u;
        }
#pragma unroll
        for (int part = 0; part < 4 / FL; part++) {
            if (part * FL >= steps) break;
            Acc acc[NT][MT];
            f4_t sa[MT];
#pragma unroll
            for (int m = 0; m < MT; m++) {
                sa[m] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 0; t < NT; t++) acc[t][m] = Acc{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < FL; i++) {
                const int j = part * FL + i;
                if constexpr (I8) {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const uint2 b = int4_to_i8(q.w[t][j], ((q.z[t] >> (8 * part)) & 15u) * 0x01010101u);
#pragma unroll
                        for (int m = 0; m < MT; m++) {
                            const uint2 a = uint2{q.a[m][j >> 1][2 * (j & 1)], q.a[m][j >> 1][2 * (j & 1) + 1]};
                            acc[t][m] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, a), __builtin_bit_cast(long, b), acc[t][m], 0, 0, 0);
                        }
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const U4 b = EXACT ? int4_differences<T>(q.w[t][j], (int)((q.z[t] >> (8 * part)) & 15u)) : int4_codes<T>(q.w[t][j]);
#pragma unroll
                        for (int m = 0; m < MT; m++) acc[t][m] = mfma16<T>(q.a[m][j], b, acc[t][m]);
                    }
                    if constexpr (!EXACT) {
#pragma unroll
                        for (int m = 0; m < MT; m++) sa[m] = mfma16<T>(q.a[m][j], ones, sa[m]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t bits = FL == 4 ? q.s[t].x : (part < 2 ? q.s[t].x : q.s[t].y) >> (16 * (part & 1));
                const uint16_t half = (uint16_t)bits;
                const float s = Elem<T>::ld((const T *)&half, 0);
                const float z = (float)((q.z[t] >> (8 * part)) & 15u);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int i = 0; i < R; i++) {
                        float v = (float)acc[t][m][i];
                        if constexpr (!I8 && !EXACT) v = fmaf(-z, sa[m][i], v);
                        tot[t][m][i] = fmaf(s, v, tot[t][m][i]);
                    }
            }
        }
    };

    auto run = [&](auto exact) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int m = 0; m < MT; m++) tot[t][m] = f4_t{0.f, 0.f, 0.f, 0.f};
        const int stride = waves * C;
        Piece now[C], next[C];
        int c = wave * C;
        if (c < full) {
#pragma unroll
            for (int u = 0; u < C; u++) load(now[u], min(c + u, full - 1), 4);
        }
        for (; c < full; c += stride) {
            const bool more = c + stride < full;
            if (more) {
#pragma unroll
                for (int u = 0; u < C; u++) load(next[u], min(c + stride + u, full - 1), 4);
            }
#pragma unroll
            for (int u = 0; u < C; u++)
                if (c + u < full) compute(now[u], 4, exact);
            if (more) {
#pragma unroll
                for (int u = 0; u < C; u++) now[u] = next[u];
            }
        }
        if constexpr (FL < 4) {  // (groups of 128 and more: K is whole pieces)
            const int steps = (p.K & 127) >> 5;
            if (steps && wave == (full / C) % waves) {
                load(now[0], full, steps);
                compute(now[0], steps, exact);
            }
        }
    };
    run(std::false_type{});
    if constexpr (!I8) {
        bool finite = true;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int i = 0; i < R; i++) finite = finite && __builtin_isfinite(tot[t][m][i]);
        if (__any(!finite)) run(std::true_type{});
    }

    // the waves' sums, in their order
    constexpr int V = NT * MT * R;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < R; i++) red[(wave * V + (t * MT + m) * R + i) * 64 + lane] = tot[t][m][i];
    __syncthreads();
    for (int v = wave; v < V; v += waves) {
        const int t = v / (MT * R), m = v / R % MT, i = v % R;
        const int row = m0 + 16 * m + 4 * i + kg, n = n0 + 16 * t + col;
        float sum = red[v * 64 + lane];
        for (int w = 1; w < waves; w++) sum += red[(w * V + v) * 64 + lane];
        if (row < p.M && n < p.N) {
            if constexpr (I8) sum *= Elem<T>::ld((const T *)p.act_scale, row);
            Elem<T>::st((T *)p.out, (size_t)row * p.N + n, sum);
        }
    }
}

}  // namespace mynn
