// Attention over a paged cache held in 4 bits, for sequences of different lengths: what the forms for few rows (attention_kv4_stream.h) and for many
// (attention_kv4_tile.h) share.
//
// Both keep the codes exact: (code - zero) is a whole number of -15 .. 15, an fp16 operand of the matrix cores in either product, whatever T is; a key's
// scale meets its score, a value's scale its weight, in 32 bits.  Queries enter as fp16 times a power of two of their row (T = bf16 has fewer bits and more
// range).  Weights enter the second product as fp16 numbers p * vs: the reference M of the online softmax is chosen so that they fit,
//   M = max over the keys of (s + max(e - 14, -100)),   2^e the scale's power of two, s the score in units of log2,
// so that p = 2^(s - M) <= 2^100 and p * vs < 2^14, with the largest near it.  A value row with a large scale and no weight takes nothing from the others then, and
// no unit is left to be taken out: numerator and denominator have the same M.
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
    int32_t *counters;        // [B * Hkv], zero between calls, or null: joined by a second launch
    int grid;                 // workgroups
};

// code - zero of a dword's eight, as Int4Pairs has them, each pair with zero points of its own (pairs (0,4), (1,5), (2,6), (3,7): off[0 .. 3])
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

// the key's share in the reference: max(e - 14, -100)
__device__ __forceinline__ float kv4_lift(float vs) { return fmaxf((float)(__builtin_amdgcn_frexp_expf(vs) - 14), -100.f); }

template <typename T> __device__ __forceinline__ float kv4_half(uint32_t w, int hi) {  // one of two packed values of T
    const uint16_t b = (uint16_t)(hi ? w >> 16 : w & 0xFFFFu);
    const T v = __builtin_bit_cast(T, b);
    return Elem<T>::ld(&v, 0);
}

// Which of a launch's workgroups have which keys.  The keys of a (sequence, kv head) come in units of UNIT; a sequence has at least one.  All units in a
// row, by sequence, head and place, are dealt out in equal runs, so that workgroups have the same to do whatever the lengths are: lens are read on the
// device, the launch is the same for all of them.  Every wave finds the run for itself (64 sequences at a time, a lane each).
template <int UNIT> struct Kv4Share {
    int quota, total;  // units of a workgroup, units in all
    int first;         // this workgroup's first unit
    int b, before;     // the sequence that has it, and the units of the sequences in front
    __device__ static int units(const PagedKv &c, int b, int S) {
        const PagedSeq s(c, b, S);
        return max(1, (s.len + UNIT - 1) / UNIT);
    }
    // inclusive sum over the lanes
    __device__ static int running(int v, int lane) {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(v, d, 64);
            if (lane >= d) v += o;
        }
        return v;
    }
    __device__ Kv4Share(const Kv4Args &a, int wg, int lane) {
        const int H = a.c.Hkv;
        int run = 0, sum = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            run = running(b0 + lane < a.B ? units(a.c, b0 + lane, a.Sq) : 0, lane);
            sum += __builtin_amdgcn_readlane(run, 63);
        }
        total = sum * H;
        quota = (total + a.grid - 1) / a.grid;
        first = wg * quota;
        b = before = 0;
        if (first >= total) return;
        int front = 0;
        for (int b0 = 0;; b0 += 64) {
            if (a.B > 64) run = running(b0 + lane < a.B ? units(a.c, b0 + lane, a.Sq) : 0, lane);
            const uint64_t past = __builtin_amdgcn_ballot_w64((front + run) * H > first);
            if (past) {
                const int l = __builtin_ctzll(past);
                b = b0 + l;
                before = (front + (l ? __builtin_amdgcn_readlane(run, l - 1) : 0)) * H;
                return;
            }
            front += __builtin_amdgcn_readlane(run, 63);
        }
    }
};

}  // namespace mynn
