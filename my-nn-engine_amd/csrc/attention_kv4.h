// Attention over a paged cache held in 4 bits, for sequences of different lengths: what the forms for few rows (attention_kv4_stream.h) and for many
// (attention_kv4_tile.h) share.
//
// Both keep the codes exact: (code - zero) is a whole number of -15 .. 15, an operand of the matrix cores in either product, whatever T is; a key's scale
// meets its score, a value's scale its weight, in 32 bits.
// Scores: queries enter as fp16 times a power of two of their row (T = bf16 has fewer bits and more range), a key's codes as they lie in their nibble, fp16
// numbers without a leading one: (code - zero) 2^-24 or, four bits further up, 2^-20.  So the sum over a row's columns is below 4, whatever the queries are, and
// its product with a scale of bf16 fits 32 bits.
// Weights: p = 2^(s - M), s the score in units of log2 and M the largest of them so far, enter the second product with the value's scale: w = p * vs.  As fp16, in two
// parts, where the scales of all values that are seen lie within 11 binades (Kv4Band): in units of a power of two that puts these near the upper end of fp16.  Elsewhere --
// a group of zeros has the scale 1 and may lie beside values of 2^-60, one group may be 2^40 of the next, stand for NaN -- in three parts of bf16, all 24 bits of w in the
// range of 32-bit numbers, and the codes as bf16 too.  (One reference for weight and scale, M = max (s + log2 vs), lost such neighbours without a word.)
#pragma once
#include "int4_codes.h"
#include "kv_cache4.h"
#include "mfma.h"

namespace mynn {

struct Kv4Args {
    PagedKv c;
    void *out;
    const void *q;
    float scale;
    int causal, B, Sq, Hq;
    float *part_o, *part_ml;  // parts of rows that several workgroups share
    int32_t *counters;        // one for each workgroup, zero between calls, or null: joined by a second launch
    int grid;                 // workgroups of the form for few rows, those that run at once of the form for many
    int blocks, ranges;       // the form for many rows: blocks of rows of a kv head, the most ranges that their keys come in
    int *length;              // and how long a range is, as the first workgroup found it
};

// Keys: (code - zero) 2^-24 of a dword's eight in pairs (0, 4), (2, 6), 2^-20 in (1, 5), (3, 7): a nibble under no exponent is such a number, and so is its difference to another.
struct Kv4Keys {
    h2_t low, high;
    __device__ void at(uint32_t z) {
        low = __builtin_bit_cast(h2_t, 0x80008000u + z * 0x00010001u);
        high = __builtin_bit_cast(h2_t, 0x80008000u + z * 0x00100010u);
    }
    __device__ U4 operator()(uint32_t w) const {
        auto two = [&](uint32_t n, h2_t off) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, n) + off); };
        const uint32_t v = w >> 8;
        return U4{two(w & 0x000F000Fu, low), two(w & 0x00F000F0u, high), two(v & 0x000F000Fu, low), two(v & 0x00F000F0u, high)};
    }
};
// A row's queries for them: eight times 2^e in the same order, e as large as fp16 takes for a row whose largest is `peak` (2^e of it below 2^15; the odd columns have 2^-4
// of that, which their codes make up for).  Values down to 2^-24 of the largest keep their 11 bits.
__device__ __forceinline__ int kv4_query_exponent(float peak) { return peak > 0.f ? 15 - __builtin_amdgcn_frexp_expf(peak) : 0; }
__device__ __forceinline__ U4 kv4_queries(const float *f, int e) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __builtin_amdgcn_ldexpf(f[i], e - 4 * (i & 1));
    return U4{pack2<f16_t>(x[0], x[4]), pack2<f16_t>(x[1], x[5]), pack2<f16_t>(x[2], x[6]), pack2<f16_t>(x[3], x[7])};
}
// What makes a score, in units of log2, of a sum of theirs: 2^(24 - e) times the call's scale.  For queries past 2^91 (T = bf16) that could leave the 32-bit numbers: the
// scores of the lanes in `far` are multiplied with 2^37 then.
struct Kv4Score {
    float by;
    uint64_t far;
    template <typename T> static __device__ __forceinline__ Kv4Score of(float scale, int e) {
        const bool past = !std::is_same<T, f16_t>::value && 24 - e > 100;
        return {__builtin_amdgcn_ldexpf(scale * 1.4426950408889634f, 24 - e - (past ? 37 : 0)), __builtin_amdgcn_ballot_w64(past)};
    }
    __device__ __forceinline__ float far_by() const { return __builtin_amdgcn_inverse_ballot_w64(far) ? 0x1p37f : 1.f; }
};

// Values: code - zero of a dword's eight, as Int4Pairs has them, each pair with zero points of its own (pairs (0,4), (1,5), (2,6), (3,7): off[0 .. 3])
__device__ __forceinline__ U4 kv4_pairs(uint32_t w, const h2_t *off, uint32_t nibbles0, uint32_t nibbles1) {
    auto two = [&](uint32_t v, uint32_t nibbles, uint32_t exponents, h2_t o) {
        const uint32_t n = (v & nibbles) | exponents;
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, n) + o);
    };
    const uint32_t v = w >> 8;
    return U4{two(w, nibbles0, 0x64006400u, off[0]), two(w, nibbles1, 0x54005400u, off[1]), two(v, nibbles0, 0x64006400u, off[2]), two(v, nibbles1, 0x54005400u, off[3])};
}
// -(1024 + z) and -(64 + z) of two zero points (bytes 0 and 2 of zz)
__device__ __forceinline__ h2_t kv4_low(uint32_t zz) { return __builtin_bit_cast(h2_t, (zz & 0x000F000Fu) | 0xE400E400u); }
__device__ __forceinline__ h2_t kv4_high(uint32_t zz) { return __builtin_bit_cast(h2_t, ((zz << 4) & 0x00F000F0u) | 0xD400D400u); }
__device__ inline f4_t mfma16_bf16(const U4 &a, const U4 &b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}
// whole numbers of fp16 as bf16 (at most 4 bits: the upper half of the 32-bit number)
__device__ __forceinline__ U4 kv4_as_bf16(const U4 &x) {
    auto two = [](uint32_t w) {
        const h2_t h = __builtin_bit_cast(h2_t, w);
        return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, (float)h[1]), __builtin_bit_cast(uint32_t, (float)h[0]), 0x07060302u);
    };
    return U4{two(x.x), two(x.y), two(x.z), two(x.w)};
}

// M may lag 2^4 behind in the form for many rows: moving it moves every sum, and a row meets a new maximum every few keys for long.
constexpr float kKv4Lag = 4.f;

// Where the scales of the values lie that a wave has seen, one answer for all its rows: `unit` is log2 of what p is multiplied with.  Compared are the upper bits of a scale, sign
// off; an exponent of the 32-bit number and T's differ by BIAS.
//   fp16 parts   2^unit puts a scale of the size e at 2^TOP (2^12, or 2^8 where M may lag: scales of 4 e and weights of 2^4 stay below 2^16), the least that is let through,
//                2^-8 e, at 2^4 or 1: a weight is off by 2^-25 of that unit, next to a scale of its own.  e is 1 at first, then the largest of the last tile that did not fit, of
//                2^-40 .. 2^24: sums in one unit are finite in any other.
//   wide         bf16 parts, from the first tile on whose scales do not lie within 9 binades, or lie outside of that, to the end of the keys.  2^unit is 2^40 while all scales are
//                below 2^51, so that small ones are far from the least 32-bit number (and sums over 2^28 keys from the largest), then 2^-8: weights of 2^4 and scales of 2^125 have a
//                finite product with a code.
//                Such calls take up to twice as long: one token of 64 sequences of 8192 keys, bf16, 112 us and 225, of one of 32768 18 and 29, 4 x 2048 rows 234 and 485.
template <typename T, int TOP> struct Kv4Band {
    static constexpr int SHIFT = std::is_same<T, f16_t>::value ? 10 : 7, BIAS = std::is_same<T, f16_t>::value ? 112 : 0, EMAX = std::is_same<T, f16_t>::value ? 31 : 255;
    uint32_t from, last;  // scales whose bits less `from` are above `last` are not let through
    int unit;
    bool wide = false;
    __device__ __forceinline__ Kv4Band() { put(127); }
    __device__ __forceinline__ void put(int e) {
        from = (uint32_t)max(e - 8 - BIAS, 1) << SHIFT;
        last = ((uint32_t)min(e + 3 - BIAS, EMAX) << SHIFT) - from - 1;
        unit = TOP + 127 - e;
    }
    static __device__ __forceinline__ uint32_t bits(uint32_t w, int hi) { return __builtin_amdgcn_ubfe(w, hi ? 16 : 0, 15); }
    __device__ __forceinline__ uint32_t off(uint32_t b) const { return b - from; }
    // the larger of `most` and what off() makes of two scales, in halves
    typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
    __device__ __forceinline__ uint32_t off2(uint32_t most, uint32_t w) const {
        const us2_t x = __builtin_bit_cast(us2_t, w & 0x7FFF7FFFu) - __builtin_bit_cast(us2_t, from * 0x00010001u);
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2_t, most), x));
    }
    // the exponent of a scale that is not zero, as of a 32-bit number, among the least lo and the largest hi; what is no number has none, and is below all others
    static __device__ __forceinline__ void among(float scale, int &lo, int &hi) {
        const int x = (int)(__builtin_bit_cast(uint32_t, scale) >> 23 & 255u), e = x == 255 ? 0 : x;
        lo = scale == 0.f ? lo : min(lo, e), hi = max(hi, e);
    }
    // Scales that are not let through: each lane has the least and the largest exponent of some.
    __device__ __forceinline__ void settle(int lane_lo, int lane_hi) {
        int x = (255 - lane_lo) | lane_hi << 16;
        auto join = [&](int y) { x = __builtin_bit_cast(int, __builtin_elementwise_max(__builtin_bit_cast(us2_t, x), __builtin_bit_cast(us2_t, y))); };
        join(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false));
        join(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false));
        join(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false));
        join(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false));
        join(__builtin_amdgcn_update_dpp(0, x, kDppBcast15, 0xA, 0xF, false));
        join(__builtin_amdgcn_update_dpp(0, x, kDppBcast31, 0xC, 0xF, false));
        const int all = __builtin_amdgcn_readlane(x, 63), lo = 255 - (all & 0xFFFF), hi = all >> 16;
        if (lo > hi) return;  // (zeros)
        const bool high = hi > 127 + 50 || (wide && unit < 0);
        wide = wide || lo < 1 + BIAS || hi - lo > 8 || hi < 127 - 40 || hi > 127 + 24;
        if (!wide) {
            put(hi);
            return;
        }
        from = 0u, last = high || BIAS ? 0x7FFFu : ((127 + 51) << SHIFT) - 1;
        unit = high ? -8 : 40;
    }
};
// what sums in units of 2^unit are multiplied with at the end, so that all parts of a row are in the same one (2^-8: a sum of values at the end of bf16 has room)
__device__ __forceinline__ float kv4_plain(int unit) { return __builtin_amdgcn_ldexpf(1.f, -8 - unit); }
template <typename T> __device__ __forceinline__ float kv4_half(uint32_t w, int hi) {  // one of two packed values of T
    const uint16_t b = (uint16_t)(hi ? w >> 16 : w & 0xFFFFu);
    const T v = __builtin_bit_cast(T, b);
    return Elem<T>::ld(&v, 0);
}

// Two numbers as fp16, and what is left of them: hi + lo of a pair are 22 bits.  `minus` is -1, from kv4_minus: then a rest is one instruction, which reads either half of hi;
// of what it knows to be -1 the compiler makes a conversion and a subtraction.
__device__ __forceinline__ float kv4_minus() {
    float x = -1.f;
    asm volatile("" : "+s"(x));
    return x;
}
__device__ __forceinline__ uint32_t kv4_take(float &x, float &y, float minus) {
    const uint32_t w = cvt2<f16_t>(x, y);
    const h2_t hi = __builtin_bit_cast(h2_t, w);
    x = fmaf((float)hi[0], minus, x);
    y = fmaf((float)hi[1], minus, y);
    return w;
}

// Which of a launch's workgroups have which keys.  The keys of a (sequence, kv head) come in units of UNIT; a sequence has at least one.  All units in a
// row, by sequence, head and place, are dealt out in equal runs, so that workgroups have the same to do whatever the lengths are: lens are read on the
// device, the launch is the same for all of them.  Every wave finds the run for itself (64 sequences at a time, a lane each).
template <int UNIT> struct Kv4Share {
    int quota, total;  // units of a workgroup, units in all
    int first;         // this workgroup's first unit
    int b, before;     // the sequence that has it, and the units of the sequences in front
    int past, fresh, from;  // lengths of the sequences from .. from + 63, a lane each
    __device__ static int share_of(const Kv4Args &a, int total) { return (total + a.grid - 1) / a.grid; }
    __device__ static int units(const PagedSeq &s) { return max(1, (s.len + UNIT - 1) / UNIT); }
    __device__ void lengths(const Kv4Args &a, int b0, int lane) {
        from = b0;
        past = 0, fresh = a.Sq;
        if (b0 + lane < a.B) {
            past = a.c.past[b0 + lane];
            if (a.c.fresh) fresh = a.c.fresh[b0 + lane];
        }
    }
    __device__ PagedSeq seq(const Kv4Args &a, int b, int lane) {
        if (b - from >= 64) lengths(a, b, lane);
        return PagedSeq(a.c, __builtin_amdgcn_readlane(past, b - from), __builtin_amdgcn_readlane(fresh, b - from), a.Sq);
    }
    // inclusive sum over the lanes: inside rows of 16, then over the rows
    __device__ static int running(int v) {
        v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, kDppBcast15, 0xA, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, kDppBcast31, 0xC, 0xF, false);
        return v;
    }
    // ... of the units of the sequences that `lengths` has
    __device__ int run(const Kv4Args &a, int lane) { return running(from + lane < a.B ? units(PagedSeq(a.c, past, fresh, a.Sq)) : 0); }
    __device__ Kv4Share(const Kv4Args &a, int wg, int lane) {
        const int H = a.c.Hkv;
        lengths(a, 0, lane);
        int r = run(a, lane), sum = __builtin_amdgcn_readlane(r, 63);
        if (a.B > 64) {
            // (four lengths of a lane on their way at a time: each of them is a wait for memory)
            int mine = 0;
            for (int b0 = 64 + lane; b0 - lane < a.B; b0 += 256) {
                int p[4], f[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int b = min(b0 + 64 * i, a.B - 1);
                    p[i] = a.c.past[b], f[i] = a.c.fresh ? a.c.fresh[b] : a.Sq;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) mine += b0 + 64 * i < a.B ? units(PagedSeq(a.c, p[i], f[i], a.Sq)) : 0;
            }
            sum += __builtin_amdgcn_readlane(running(mine), 63);
        }
        total = sum * H;
        quota = share_of(a, total);
        first = wg * quota;
        b = before = 0;
        if (first >= total) return;
        int front = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const int here_past = past, here_fresh = fresh;
            if (b0 + 64 < a.B) lengths(a, b0 + 64, lane);  // (on their way meanwhile)
            const uint64_t behind = __builtin_amdgcn_ballot_w64((front + r) * H > first);
            if (behind) {
                const int l = __builtin_ctzll(behind);
                b = b0 + l;
                before = (front + (l ? __builtin_amdgcn_readlane(r, l - 1) : 0)) * H;
                from = b0, past = here_past, fresh = here_fresh;
                return;
            }
            front += __builtin_amdgcn_readlane(r, 63);
            r = run(a, lane);
        }
        first = total;  // (lengths that change under the call, which no program may do: nothing to do, and an end)
    }
};

}  // namespace mynn
