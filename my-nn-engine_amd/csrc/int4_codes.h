// 4-bit codes on their way to the matrix cores, for the kernels of int4_stream.h and int4_tile.h.
//
// A dword holds eight codes, the first in its lowest four bits.  A lane of v_mfma 16x16x32 takes the eight of a dword, one of v_mfma 32x32x16 too,
// one of v_mfma 32x32x32 (int8) those of two.
//
// To 16 bits as they are, nine vector operations for eight: a nibble as a byte is 2^-9 times its value as an fp8 number (e4m3: below 8
// subnormal, from 8 on the first binade, one line), so v_cvt_scalef32_pk makes two exact values of T from two bytes.  The zero point then comes
// off the sums: sum a (q - z) = sum a q - z sum a.  Both sums may overflow, or meet an infinity, where their difference does not: who uses
// them looks at the result and starts again with the differences themselves where it is not finite.
// To int8: nibbles to bytes, the zero point taken off inside the bytes (a bit set above them: no borrow).
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

}  // namespace mynn
