// Position rotation of q and k with the append of k and v to a paged cache of 16, 8 or 4 bits, for sequences of different lengths, and
// the cache's rows as plain rows again.
//
// Rotation: lo' = lo*cos[p,j] - hi*sin[p,j], hi' = hi*cos[p,j+D/2] + lo*sin[p,j+D/2], separate products, one rounding (as
// rope_kv_append).  What goes to the cache is the row that a 16-bit cache would hold: as it is, by the rule of
// quantizing_kvcache_update in 8 bits, by that of Int4Row in 4.
//
// Memory bounds both where there are many rows (4 x 2048 tokens, 32 / 8 heads of 128; in brackets the bytes at a copy's 5.1 TB/s): in 16 bits 36.5 us (39), in 8 38.5 (36), in 4 39.0
// (35), rows read back from 4 bits 11.2 (8.2); a launch and a chain of waits elsewhere (32 tokens into 4 bits 4.4 us, 400 5.8).  A thread with several heads of a token
// keeps its table rows in registers and was no faster (42 us, 43 then), a wave with 8 tokens of a head 42; a thread that reads back 16 columns instead of 8 11.1.
#include "kv_cache4.h"
#include "mfma.h"

namespace mynn {

struct AppendArgs {
    PagedKv c;
    void *q_out;
    const void *x[3];      // q, k, v
    long bs[3], hs[3], rs[3];  // their strides in elements: sequence, head, row
    const void *cos_t, *sin_t;
    const int64_t *position;
    int table_rows, B, S, Hq;
};

template <typename T, bool ALIGNED> __device__ __forceinline__ U4 load8(const T *p) {
    if constexpr (ALIGNED) return *(const U4 *)p;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)__builtin_bit_cast(uint16_t, p[2 * i]) | (uint32_t)__builtin_bit_cast(uint16_t, p[2 * i + 1]) << 16;
    return U4{w[0], w[1], w[2], w[3]};
}
template <typename T> __device__ __forceinline__ U4 pack8(const float *f) {
    return U4{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7])};
}

// A head of a token is LPH = D/16 lanes', neighbours of each other: each has 8 dims of the lower half and the 8 that they are rotated with, so that nothing is exchanged but a
// group's extremes.
template <typename T, int KV, int D, int GROUP, bool ALIGNED> __global__ __launch_bounds__(256) void rope_append_paged_kernel(AppendArgs a) {
    constexpr int LPH = D / 16, HALF = D / 2;
    // (32 bits, as many as there can be threads: dividing 64 took longer than everything else)
    const uint32_t at = blockIdx.x * 256u + threadIdx.x, item = at / LPH, u = at % LPH;
    const uint32_t heads = (a.q_out ? a.Hq : 0) + 2 * a.c.Hkv, token = item / heads;
    if (token >= (uint32_t)(a.B * a.S)) return;  // (whole heads: the lanes of one meet below)
    const int head = (int)(item - token * heads) + (a.q_out ? 0 : a.Hq), b = (int)(token / (uint32_t)a.S), i = (int)(token - (uint32_t)b * a.S);
    const int part = head < a.Hq ? 0 : head < a.Hq + a.c.Hkv ? 1 : 2;
    const int h = part == 0 ? head : part == 1 ? head - a.Hq : head - a.Hq - a.c.Hkv;
    // (on its way before it is known whether the token is there)
    const T *src = (const T *)a.x[part] + (long)b * a.bs[part] + (long)h * a.hs[part] + (long)i * a.rs[part] + 8 * u;
    U4 lo = load8<T, ALIGNED>(src), hi = load8<T, ALIGNED>(src + HALF);
    const PagedSeq seq(a.c, b, a.S);
    const int row = seq.past + i;
    const int64_t pos = a.position ? a.position[token] : (int64_t)row;
    const bool there = i < seq.fresh && row >= 0 && row < seq.cap && pos >= 0 && pos < a.table_rows;
    int page = -1;
    float cl[8], ch[8], sl[8], sh[8];
    if (there) {
        page = paged_page(a.c, b, row);
        const T *ct = (const T *)a.cos_t + (size_t)pos * D + 8 * u, *st = (const T *)a.sin_t + (size_t)pos * D + 8 * u;
        widen8<T>(load8<T, ALIGNED>(ct), cl);
        widen8<T>(load8<T, ALIGNED>(ct + HALF), ch);
        widen8<T>(load8<T, ALIGNED>(st), sl);
        widen8<T>(load8<T, ALIGNED>(st + HALF), sh);
    }
    T *q_row = part == 0 ? (T *)a.q_out + (((size_t)b * a.Hq + h) * a.S + i) * D + 8 * u : nullptr;
    if (!there || (part && page < 0)) {
        if (part == 0) *(U4 *)q_row = *(U4 *)(q_row + HALF) = U4{0u, 0u, 0u, 0u};
        return;
    }
    float xl[8], xh[8];
    if (part < 2) {
        float ol[8], oh[8];
        widen8<T>(lo, xl);
        widen8<T>(hi, xh);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            ol[e] = xl[e] * cl[e] - xh[e] * sl[e];
            oh[e] = xh[e] * ch[e] + xl[e] * sh[e];
        }
        lo = pack8<T>(ol);
        hi = pack8<T>(oh);
    }
    if (part == 0) {
        *(U4 *)q_row = lo;
        *(U4 *)(q_row + HALF) = hi;
        return;
    }
    const size_t r = paged_row(a.c, page, h, row);
    void *pool = part == 1 ? a.c.k : a.c.v, *scales = part == 1 ? a.c.k_scale : a.c.v_scale;
    if constexpr (KV == 16) {
        T *dst = (T *)pool + r * D + 8 * u;
        *(U4 *)dst = lo;
        *(U4 *)(dst + HALF) = hi;
    } else {
        widen8<T>(lo, xl);
        widen8<T>(hi, xh);
        if constexpr (KV == 8) {
            float peak = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) peak = fmaxf(peak, fmaxf(fabsf(xl[e]), fabsf(xh[e])));
            peak = group_max<LPH>(peak);
            const float inv = peak == 0.f ? 0.f : 127.0f / peak;
            auto code = [&](float x) -> uint32_t {
                const float y = x * inv;
                const int q = (int)(y + (y >= 0.f ? 0.5f : -0.5f));
                return (uint32_t)(q < -128 ? -128 : (q > 127 ? 127 : q)) & 0xFFu;
            };
            auto four = [&](const float *x) { return code(x[0]) | code(x[1]) << 8 | code(x[2]) << 16 | code(x[3]) << 24; };
            uint8_t *dst = (uint8_t *)pool + r * D + 8 * u;
            *(uint2 *)dst = uint2{four(xl), four(xl + 4)};
            *(uint2 *)(dst + HALF) = uint2{four(xh), four(xh + 4)};
            if (u == 0) Elem<T>::st((T *)scales, r, peak * (1.0f / 127.0f));
        } else {
            // groups: all of the row (both halves of every lane), a half of it (a half of every lane), a quarter (a half of half the lanes)
            constexpr int GROUPS = D / GROUP;
            float lo0 = 0.f, hi0 = 0.f, lo1 = 0.f, hi1 = 0.f;
            float bad0 = 0.f, bad1 = 0.f;  // 0 * x: NaN where x is not finite
#pragma unroll
            for (int e = 0; e < 8; e++) {
                lo0 = fminf(lo0, xl[e]), hi0 = fmaxf(hi0, xl[e]), bad0 += 0.f * xl[e];
                lo1 = fminf(lo1, xh[e]), hi1 = fmaxf(hi1, xh[e]), bad1 += 0.f * xh[e];
            }
            constexpr int LANES = GROUPS == 4 ? LPH / 2 : LPH;
            lo0 = -group_max<LANES>(-lo0), hi0 = group_max<LANES>(hi0), bad0 = group_sum<LANES>(bad0);
            lo1 = -group_max<LANES>(-lo1), hi1 = group_max<LANES>(hi1), bad1 = group_sum<LANES>(bad1);
            if constexpr (GROUPS == 1) lo0 = lo1 = fminf(lo0, lo1), hi0 = hi1 = fmaxf(hi0, hi1), bad0 = bad1 = bad0 + bad1;
            const Int4Row<T> g0(lo0, hi0, bad0 == 0.f), g1(lo1, hi1, bad1 == 0.f);
            uint32_t w0 = 0, w1 = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) w0 |= g0.code(xl[e]) << (4 * e), w1 |= g1.code(xh[e]) << (4 * e);
            uint8_t *dst = (uint8_t *)pool + r * (D / 2) + 4 * u;
            *(uint32_t *)dst = w0;
            *(uint32_t *)(dst + HALF / 2) = w1;
            if (u % LANES == 0) {
                T *sc = (T *)scales + r * GROUPS;
                uint8_t *zp = (part == 1 ? a.c.k_zero : a.c.v_zero) + r * GROUPS;
                const int g = GROUPS == 4 ? u / LANES : 0;
                Elem<T>::st(sc, g, g0.s);
                zp[g] = (uint8_t)g0.z;
                if constexpr (GROUPS > 1) {
                    Elem<T>::st(sc, GROUPS / 2 + g, g1.s);
                    zp[GROUPS / 2 + g] = (uint8_t)g1.z;
                }
            }
        }
    }
}

// rows first .. first + n - 1 of each sequence as plain rows; a thread has 8 columns of k, of v or of both
template <typename T, int KV> __global__ __launch_bounds__(256) void kv_rows_paged_kernel(PagedKv c, T *k_out, T *v_out, int B, int S, int D, int group) {
    const uint32_t at = blockIdx.x * 256u + threadIdx.x, chunks = D / 8, line = at / chunks, pair = line / (uint32_t)S, b = pair / (uint32_t)c.Hkv;
    if (b >= (uint32_t)B) return;
    const int d = (int)(at - line * chunks) * 8, i = (int)(line - pair * S), h = (int)(pair - b * c.Hkv);
    const PagedSeq seq(c, b, S);
    const int row = seq.past + i;
    const int page = i < seq.fresh && row >= 0 && row < seq.cap ? paged_page(c, b, row) : -1;
    const size_t r = page >= 0 ? paged_row(c, page, h, row) : 0;
    T *const out[2] = {k_out, v_out};
    U4 w[2] = {};
    float s[2], z[2];
#pragma unroll
    for (int n = 0; n < 2; n++) {
        if (!out[n] || page < 0) continue;
        const void *pool = n ? c.v : c.k, *scales = n ? c.v_scale : c.k_scale;
        if constexpr (KV == 16) w[n] = *(const U4 *)((const T *)pool + r * D + d);
        else if constexpr (KV == 8) {
            const uint2 x = *(const uint2 *)((const int8_t *)pool + r * D + d);
            w[n].x = x.x, w[n].y = x.y;
            s[n] = Elem<T>::ld((const T *)scales, r);
        } else {
            const size_t g = r * (D / group) + d / group;
            w[n].x = *(const uint32_t *)((const uint8_t *)pool + (r * D + d) / 2);
            s[n] = Elem<T>::ld((const T *)scales, g);
            z[n] = (float)((n ? c.v_zero : c.k_zero)[g] & 15);
        }
    }
#pragma unroll
    for (int n = 0; n < 2; n++) {
        if (!out[n]) continue;
        U4 y = w[n];
        if (KV < 16 && page >= 0) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e++)
                f[e] = KV == 8 ? (float)(int8_t)((e < 4 ? w[n].x : w[n].y) >> (8 * (e & 3)) & 0xFFu) * s[n] : ((float)(w[n].x >> (4 * e) & 15u) - z[n]) * s[n];
            y = pack8<T>(f);
        }
        *(U4 *)(out[n] + (size_t)line * D + d) = y;
    }
}

// what every call over pools asks of them
int paged_kv_check(const char *who, const PagedKv &c, int page_rows, int kv_bits, int group, int D) {
    MYNN_REQUIRE(c.table && c.past, MYNN_ERR_INVALID, "%s: null page table or lengths", who);
    MYNN_REQUIRE(D == 64 || D == 128, MYNN_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", who, D);
    MYNN_REQUIRE(kv_bits == 16 || kv_bits == 8 || kv_bits == 4, MYNN_ERR_INVALID, "%s: a cache of %d bits (16, 8 or 4)", who, kv_bits);
    MYNN_REQUIRE(kv_bits != 4 || ((group == 32 || group == 64 || group == 128) && group <= D), MYNN_ERR_UNSUPPORTED,
                 "%s: groups of %d columns (32, 64 or 128, at most head_dim)", who, group);
    MYNN_REQUIRE(c.k && c.v && aligned16(c.k) && aligned16(c.v), MYNN_ERR_INVALID, "%s: null or unaligned pool", who);
    MYNN_REQUIRE(kv_bits == 16 || (c.k_scale && c.v_scale && aligned16(c.k_scale) && aligned16(c.v_scale)), MYNN_ERR_INVALID, "%s: null or unaligned scale pool", who);
    MYNN_REQUIRE(kv_bits != 4 || (c.k_zero && c.v_zero && aligned16(c.k_zero) && aligned16(c.v_zero)), MYNN_ERR_INVALID, "%s: null or unaligned zero point pool", who);
    MYNN_REQUIRE(page_rows >= 32 && page_rows <= (1 << 20) && (page_rows & (page_rows - 1)) == 0 && c.n_pages > 0 && c.pages_per_seq > 0, MYNN_ERR_INVALID,
                 "%s: %d pages of %d rows, %d for a sequence (rows per page: a power of two, 32 or more)", who, c.n_pages, page_rows, c.pages_per_seq);
    MYNN_REQUIRE((long)c.pages_per_seq * page_rows <= 1 << 30, MYNN_ERR_UNSUPPORTED, "%s: sequences of %ld rows", who, (long)c.pages_per_seq * page_rows);
    return 0;
}
int paged_shift(int page_rows) {
    int shift = 0;
    while ((1 << shift) < page_rows) shift++;
    return shift;
}

template <typename T, int KV, int D, int GROUP> static int append_go(const AppendArgs &a, bool aligned, unsigned blocks, hipStream_t s) {
    if (aligned) MYNN_LAUNCH((rope_append_paged_kernel<T, KV, D, GROUP, true>), dim3(blocks), dim3(256), 0, s, a);
    else MYNN_LAUNCH((rope_append_paged_kernel<T, KV, D, GROUP, false>), dim3(blocks), dim3(256), 0, s, a);
    return launch_status("rope_append_paged_kernel");
}

}  // namespace mynn

using namespace mynn;

extern "C" int mynn_rope_append_paged(void *q_out, const void *q, const void *k, const void *v, const int64_t *strides, const void *cos_t, const void *sin_t,
                                      int table_rows, const int64_t *position, void *k_pool, void *v_pool, void *k_scale_pool, void *v_scale_pool,
                                      uint8_t *k_zero_pool, uint8_t *v_zero_pool, const int32_t *page_table, int n_pages, int pages_per_seq, int page_rows,
                                      const int32_t *past_lens, const int32_t *new_lens, int B, int S, int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                                      int kv_bits, int group, mynn_stream s) {
    const char *who = "rope_append_paged";
    const int D = head_dim;
    MYNN_REQUIRE((q != nullptr) == (q_out != nullptr) && k && v && strides && cos_t && sin_t, MYNN_ERR_INVALID, "%s: null operand", who);
    MYNN_REQUIRE(B > 0 && S > 0 && num_q_heads > 0 && num_kv_heads > 0 && table_rows > 0, MYNN_ERR_INVALID, "%s: B=%d S=%d heads %d/%d, %d table rows", who, B, S,
                 num_q_heads, num_kv_heads, table_rows);
    AppendArgs a{{k_pool, v_pool, k_scale_pool, v_scale_pool, k_zero_pool, v_zero_pool, page_table, past_lens, new_lens, n_pages, pages_per_seq, 0, num_kv_heads},
                 q_out, {q, k, v}, {}, {}, {}, cos_t, sin_t, position, table_rows, B, S, num_q_heads};
    if (const int rc = paged_kv_check(who, a.c, page_rows, kv_bits, group, D)) return rc;
    a.c.page_shift = paged_shift(page_rows);
    MYNN_REQUIRE(num_q_heads <= 65536 && num_kv_heads <= 65536 && S <= 1 << 30, MYNN_ERR_UNSUPPORTED, "%s: S=%d heads %d/%d", who, S, num_q_heads, num_kv_heads);
    bool aligned = aligned16(cos_t) && aligned16(sin_t);
    for (int i = 0; i < 3; i++) {
        a.bs[i] = strides[3 * i], a.hs[i] = strides[3 * i + 1], a.rs[i] = strides[3 * i + 2];
        if (i > 0 || q) aligned = aligned && aligned16(a.x[i]) && a.bs[i] % 8 == 0 && a.hs[i] % 8 == 0 && a.rs[i] % 8 == 0;
    }
    MYNN_REQUIRE(!q_out || aligned16(q_out), MYNN_ERR_INVALID, "%s: q_out has to be 16-byte aligned", who);
    const int heads = (q ? num_q_heads : 0) + 2 * num_kv_heads;
    const size_t blocks = ((size_t)B * S * heads * (D / 16) + 255) / 256;
    MYNN_REQUIRE(blocks < 1u << 24, MYNN_ERR_UNSUPPORTED, "%s: %d x %d tokens of %d heads", who, B, S, heads);
    return dispatch_dtype16(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        auto go = [&](auto d) {
            constexpr int DD = decltype(d)::value;
            if (kv_bits == 16) return append_go<T, 16, DD, DD>(a, aligned, (unsigned)blocks, as_stream(s));
            if (kv_bits == 8) return append_go<T, 8, DD, DD>(a, aligned, (unsigned)blocks, as_stream(s));
            if (group == DD) return append_go<T, 4, DD, DD>(a, aligned, (unsigned)blocks, as_stream(s));
            if (group == DD / 2) return append_go<T, 4, DD, DD / 2>(a, aligned, (unsigned)blocks, as_stream(s));
            if constexpr (DD == 128) return append_go<T, 4, DD, DD / 4>(a, aligned, (unsigned)blocks, as_stream(s));
            return fail(MYNN_ERR_UNSUPPORTED, "%s: groups of %d columns", who, group);
        };
        return D == 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
    });
}

extern "C" int mynn_kv_rows_paged(void *k_out, void *v_out, const void *k_pool, const void *v_pool, const void *k_scale_pool, const void *v_scale_pool,
                                  const uint8_t *k_zero_pool, const uint8_t *v_zero_pool, const int32_t *page_table, int n_pages, int pages_per_seq, int page_rows,
                                  const int32_t *first_rows, const int32_t *n_rows, int B, int S, int num_kv_heads, int head_dim, int dtype, int kv_bits, int group,
                                  mynn_stream s) {
    const char *who = "kv_rows_paged";
    MYNN_REQUIRE((k_out || v_out) && aligned16(k_out) && aligned16(v_out), MYNN_ERR_INVALID, "%s: null or unaligned output", who);
    MYNN_REQUIRE(B > 0 && S > 0 && num_kv_heads > 0, MYNN_ERR_INVALID, "%s: B=%d S=%d kv heads %d", who, B, S, num_kv_heads);
    PagedKv c{(void *)k_pool, (void *)v_pool, (void *)k_scale_pool, (void *)v_scale_pool, (uint8_t *)k_zero_pool, (uint8_t *)v_zero_pool, page_table, first_rows, n_rows,
              n_pages, pages_per_seq, 0, num_kv_heads};
    if (const int rc = paged_kv_check(who, c, page_rows, kv_bits, group, head_dim)) return rc;
    c.page_shift = paged_shift(page_rows);
    MYNN_REQUIRE(num_kv_heads <= 65536 && S <= 1 << 30, MYNN_ERR_UNSUPPORTED, "%s: S=%d kv heads %d", who, S, num_kv_heads);
    const size_t threads = (size_t)B * num_kv_heads * S * (head_dim / 8), blocks = (threads + 255) / 256;
    MYNN_REQUIRE(blocks < 1u << 24, MYNN_ERR_UNSUPPORTED, "%s: %d x %d rows of %d heads", who, B, S, num_kv_heads);
    return dispatch_dtype16(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const dim3 grid((unsigned)blocks);
        if (kv_bits == 16) MYNN_LAUNCH((kv_rows_paged_kernel<T, 16>), grid, dim3(256), 0, as_stream(s), c, (T *)k_out, (T *)v_out, B, S, head_dim, group);
        else if (kv_bits == 8) MYNN_LAUNCH((kv_rows_paged_kernel<T, 8>), grid, dim3(256), 0, as_stream(s), c, (T *)k_out, (T *)v_out, B, S, head_dim, group);
        else MYNN_LAUNCH((kv_rows_paged_kernel<T, 4>), grid, dim3(256), 0, as_stream(s), c, (T *)k_out, (T *)v_out, B, S, head_dim, group);
        return launch_status("kv_rows_paged_kernel");
    });
}
