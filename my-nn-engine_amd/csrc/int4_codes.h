// 4-bit codes on their way to the matrix cores, for the kernels of int4_stream.h and int4_tile.h.
//
// A dword holds eight codes, the first in its lowest four bits.  A lane of v_mfma 16x16x32 takes the eight of a dword, one of v_mfma 32x32x16 too,
// one of v_mfma 32x32x32 (int8) those of two.
//
// The zero point comes off each code, exactly, before the code meets an activation.  (Sums of act * code less the zero point times the sum of act took two
// operations fewer for eight codes; but an activation whose code is the zero point, which is to count for nothing, left the rounding of both sums, and an
// infinite one more than that.)
// To int8: nibbles to bytes, the zero point taken off inside the bytes (a bit set above them: no borrow).
// To fp16: a nibble under an exponent that makes it 1024 + n, or, four bits further up, 64 + n; one addition takes 1024 or 64 and the zero point off two.
#pragma once
#include <type_traits>

#include "mfma.h"
#include "mynn_common.h"

namespace mynn {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef int i4_t __attribute__((ext_vector_type(4)));

__device__ inline f4_t mfma16(const U4 &a, const U4 &b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
}

// code - zero of the eight as int8 (zz: the zero point in each byte): 0x80 + code - zero never borrows from its neighbour
__device__ inline uint2 int4_to_i8(uint32_t w, uint32_t zz) {
    const uint32_t e = ((w & 0x0F0F0F0Fu) | 0x80808080u) - zz, o = (((w >> 4) & 0x0F0F0F0Fu) | 0x80808080u) - zz;
    return uint2{__builtin_amdgcn_perm(o, e, 0x05010400u) ^ 0x80808080u, __builtin_amdgcn_perm(o, e, 0x07030602u) ^ 0x80808080u};
}
// code - zero of a dword's eight as fp16, in pairs (0, 4), (1, 5), (2, 6), (3, 7): where the other operand can be in that order too, one shift takes the
// place of the four byte selections, nine operations in all.
struct Int4Pairs {
    h2_t low, high;
    uint32_t nibbles0 = 0x000F000Fu, nibbles1 = 0x00F000F0u;
    // (in vector registers: one instruction takes both, but at most one constant from elsewhere)
    __device__ Int4Pairs() { asm volatile("" : "+v"(nibbles0), "+v"(nibbles1)); }
    __device__ void at(uint32_t z) {
        low = __builtin_bit_cast(h2_t, 0xE400E400u + z * 0x00010001u);
        high = __builtin_bit_cast(h2_t, 0xD400D400u + z * 0x00100010u);
    }
    __device__ U4 operator()(uint32_t w) const {
        auto two = [&](uint32_t v, uint32_t nibbles, uint32_t exponents, h2_t off) {
            const uint32_t n = (v & nibbles) | exponents;
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, n) + off);
        };
        const uint32_t v = w >> 8;
        return U4{two(w, nibbles0, 0x64006400u, low), two(w, nibbles1, 0x54005400u, high), two(v, nibbles0, 0x64006400u, low), two(v, nibbles1, 0x54005400u, high)};
    }
};
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
