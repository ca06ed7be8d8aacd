// Paged caches as the operators for sequences of different lengths see them: which rows there are, where a row lies, and the 4-bit
// form of a row (codes, scales and zero points of groups of columns, as the 4-bit weights have them).
#pragma once
#include "mynn_common.h"

namespace mynn {

// The pools of a cache and the page table of B sequences.  A page number outside [0, n_pages) stands for a page that is not there:
// no address is made of it.
struct PagedKv {
    void *k, *v;              // T, int8 or pairs of 4-bit codes: [n_pages, Hkv, P, D]
    void *k_scale, *v_scale;  // T: int8 [n_pages, Hkv, P], 4 bits [n_pages, Hkv, P, D / group]
    uint8_t *k_zero, *v_zero;  // 4 bits: as the scales
    const int32_t *table;     // [B, pages_per_seq]
    const int32_t *past, *fresh;  // [B] rows in the cache before the S new ones, and how many of those there are (null: S)
    int n_pages, pages_per_seq, page_shift, Hkv;
};

// A sequence: rows [0, past) were there before, [past, len) are new.  (An int holds every sum below: a past that no cache could have is cut off.)
struct PagedSeq {
    int past, fresh, len, cap;
    __device__ PagedSeq(const PagedKv &c, int b, int S) : PagedSeq(c, c.past[b], c.fresh ? c.fresh[b] : S, S) {}
    __device__ PagedSeq(const PagedKv &c, int past_len, int new_len, int S) {
        cap = c.pages_per_seq << c.page_shift;
        past = min(max(past_len, -S), cap);
        fresh = min(max(new_len, 0), S);
        len = fresh ? min(max(past + fresh, 0), cap) : 0;
    }
    // keys that query row i sees
    __device__ int bound(int i, bool causal) const { return i >= fresh ? 0 : causal ? min(max(past + i + 1, 0), len) : len; }
};

// the page that row r of sequence b lies in, -1: none
__device__ inline int paged_page(const PagedKv &c, int b, int r) {
    const int page = c.table[(size_t)b * c.pages_per_seq + (r >> c.page_shift)];
    return (unsigned)page < (unsigned)c.n_pages ? page : -1;
}
// ... and the index of its row for kv head h, in rows
__device__ inline size_t paged_row(const PagedKv &c, int page, int h, int r) {
    return (((size_t)page * c.Hkv + h) << c.page_shift) + (size_t)(r & ((1 << c.page_shift) - 1));
}

// The 4-bit form of a group of columns with least value lo <= 0 and largest hi >= 0 (zero among them: a value of zero stays zero):
//   s = T(hi/15 - lo/15), z = round(-lo/s), code = round(x/s) + z in 0 .. 15, which stands for s * (code - z)
// -- mynn_quantize_int4_groups for a row.  A group with a value that is not finite stands for NaN.
// A division of 32 bits for each value is most of the append's work.  x and s are of T, with at most 11 bits, so x/s is a half or 2^-12 and more away from it, and a product with
// 1/s, off by 2^-18 at |x/s| < 32, rounds like the quotient where 2^-15 goes on top of the half: 4 x 2048 tokens, 16 heads of 128 quantised, 42.9 -> 39.0 us.
template <typename T> struct Int4Row {
    float s, z, up, r;  // r = 1 / (s up): up keeps it from overflow where s is one of the least numbers of bf16
    __device__ Int4Row(float lo, float hi, bool finite) {
        s = Elem<T>::rnd(hi / 15.0f - lo / 15.0f);
        if (s == 0.f) s = 1.f;
        z = fminf(roundf(-lo / s), 15.f);
        if (!finite) s = __builtin_nanf(""), z = 0.f;
        up = !std::is_same<T, f16_t>::value && s < 0x1p-64f ? 0x1p64f : 1.f;
        r = 1.0f / (s * up);
    }
    __device__ uint32_t code(float x) const {
        if (!std::is_same<T, f16_t>::value) x *= up;
        const float y = x * r, c = fminf(fmaxf(copysignf(truncf(fabsf(y) + (0.5f + 0x1p-15f)), y) + z, 0.f), 15.f);
        return c == c ? (uint32_t)c : 0u;
    }
};

}  // namespace mynn
