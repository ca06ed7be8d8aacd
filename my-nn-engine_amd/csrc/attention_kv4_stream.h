// The form for few rows: up to 16 query rows of a kv head (query heads times new tokens) are the 16 columns of v_mfma_f32_16x16x32_f16.
//
// A workgroup of four waves walks its run of keys, 32 a wave, the next ones' codes, scales and zero points on their way to registers meanwhile.
//   S[keys x rows] = K . Q^T  a lane has a key's 32 columns of 16 bytes; dwords are exchanged between its four lane groups so that each matrix
//                             instruction takes 32 neighbouring columns, of one group of columns
//   softmax                   online; a lane has one row (column of the instruction) and 8 of the 32 keys
//   O^T[columns x rows] += V^T . P   V goes to LDS as codes and comes back transposed (ds_read_b64_tr_b4: of 16 rows that its lanes name, a lane receives
//                             one column); named are a lane group's own 8 keys twice, for 16 columns and the 16 behind them, so that the order of the
//                             keys is the one in which the scores lie in registers.  p * vs in two fp16 values, rounded and rest: 22 bits.
#pragma once
#include "attention_kv4.h"

namespace mynn {

constexpr int kKv4Waves = 4, kKv4Unit = 32 * kKv4Waves;

// one wave's loads of 32 keys
template <int D, int NG> struct Kv4Tile {
    static constexpr int KW = D / 32;  // dwords of codes of a lane and 16 keys
    uint32_t k[2][KW], v[D / 16];
    uint32_t ks[2][2 * NG], vs[2][2 * NG], vz[2][NG];
    uint32_t kz[2];
    bool there;
};

template <typename T, int D, int NG> __global__ __launch_bounds__(kKv4Waves * 64) void attn_kv4_stream_kernel(Kv4Args a) {
    constexpr int NW = kKv4Waves, GROUP = D / NG, KS = D / 32, VROW = D / 2 + 16;  // bytes of a row of V codes in LDS
    constexpr int MPG = GROUP / 32;                                               // matrix instructions of a group
    extern __shared__ __align__(16) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, j = lane >> 4;
    const int G = a.Hq / a.c.Hkv, R = G * a.Sq;
    const int wave_bytes = max(32 * VROW, R * D * 4);
    char *mine = sm + wave * wave_bytes;
    float *m_s = (float *)(sm + NW * wave_bytes), *l_s = m_s + NW * 16;
    auto o_s = [&](int w) { return (float *)(sm + w * wave_bytes); };

    const Kv4Share<kKv4Unit> share(a, blockIdx.x, lane);
    int unit = __builtin_amdgcn_readfirstlane(share.first);
    if (unit >= __builtin_amdgcn_readfirstlane(share.total)) return;
    const int stop = min(unit + __builtin_amdgcn_readfirstlane(share.quota), __builtin_amdgcn_readfirstlane(share.total));
    int b = __builtin_amdgcn_readfirstlane(share.b), h = 0, at = 0;  // at: unit inside the (sequence, head)
    PagedSeq seq(a.c, b, a.Sq);
    int n_units = max(1, (seq.len + kKv4Unit - 1) / kKv4Unit);
    {
        const int r = unit - __builtin_amdgcn_readfirstlane(share.before);
        h = r / n_units;
        at = r - h * n_units;
    }
    Int4Pairs pairs;
    const int psh = a.c.page_shift, pmask = (1 << psh) - 1;

    while (unit < stop) {
        const int end = min(n_units, at + stop - unit);
        const int k0 = at * kKv4Unit, k1 = min(seq.len, end * kKv4Unit);
        // ---- the rows' queries: B operand, columns 32 m + 8 j .. +7 (D = 64: in the order in which the exchange below leaves them) by pairs
        const int row = col < R ? col : 0, qi = row / G, head = h * G + row % G;
        const int bound = col < R ? seq.bound(qi, a.causal) : 0;
        U4 qf[KS];
        float csc;
        {
            const T *q = (const T *)a.q + (((size_t)b * a.Hq + head) * a.Sq + qi) * D;
            float x[KS][8], peak = 0.f;
#pragma unroll
            for (int m = 0; m < KS; m++) {
                const int d = D == 128 ? 32 * m + 8 * j : 32 * m + (j & 1) * 16 + (j >> 1) * 8;
                widen8<T>(*(const U4 *)(q + d), x[m]);
#pragma unroll
                for (int e = 0; e < 8; e++) peak = fmaxf(peak, fabsf(x[m][e]));
            }
            peak = xor32_max(xor16_max(peak));
            // (2^10 at the most: values down to 2^-24 of a row's largest keep their 11 bits, and sums stay far from the largest 32-bit number)
            const int e10 = peak > 0.f ? 10 - __builtin_amdgcn_frexp_expf(peak) : 0;
#pragma unroll
            for (int m = 0; m < KS; m++) {
#pragma unroll
                for (int e = 0; e < 8; e++) x[m][e] = __builtin_amdgcn_ldexpf(x[m][e], e10);
                qf[m] = U4{pack2<f16_t>(x[m][0], x[m][4]), pack2<f16_t>(x[m][1], x[m][5]), pack2<f16_t>(x[m][2], x[m][6]), pack2<f16_t>(x[m][3], x[m][7])};
                if (col >= R) qf[m] = U4{0u, 0u, 0u, 0u};
            }
            csc = __builtin_amdgcn_ldexpf(a.scale * 1.4426950408889634f, -e10);
        }
        f4_t acc[D / 16];
#pragma unroll
        for (int c = 0; c < D / 16; c++) acc[c] = f4_t{0.f, 0.f, 0.f, 0.f};
        float M = -INFINITY, l = 0.f;

        // the entries of 64 pages of the sequence, a lane each
        int pages = -1, pages_at = -(1 << 30);
        auto load = [&](Kv4Tile<D, NG> &t, int key0) {
            const int p = __builtin_amdgcn_readfirstlane(key0 >> psh);
            if (p - pages_at >= 64 || p < pages_at) {
                pages_at = p;
                pages = p + lane < a.c.pages_per_seq ? a.c.table[(size_t)b * a.c.pages_per_seq + p + lane] : -1;
                if ((unsigned)pages >= (unsigned)a.c.n_pages) pages = -1;
            }
            const int page = __builtin_amdgcn_readlane(pages, p - pages_at);
            t.there = page >= 0;
            // (a page that is not there: page 0 is read, and nothing made of it)
            const size_t r0 = (((size_t)max(page, 0) * a.c.Hkv + h) << psh) + (size_t)(key0 & pmask);
            const uint8_t *k = (const uint8_t *)a.c.k + r0 * (D / 2), *v = (const uint8_t *)a.c.v + r0 * (D / 2);
            const T *ks = (const T *)a.c.k_scale + r0 * NG, *vs = (const T *)a.c.v_scale + r0 * NG;
            const uint8_t *kz = a.c.k_zero + r0 * NG, *vz = a.c.v_zero + r0 * NG;
            auto put = [](auto &to, const void *from) { __builtin_memcpy(&to, from, sizeof to); };
#pragma unroll
            for (int s = 0; s < 2; s++) {
                put(t.k[s], __builtin_assume_aligned(k + (16 * s + col) * (D / 2) + j * KS * 4, KS * 4));
                put(t.ks[s], __builtin_assume_aligned(ks + (16 * s + 4 * j) * NG, 8));
                put(t.vs[s], __builtin_assume_aligned(vs + (16 * s + 4 * j) * NG, 8));
                put(t.vz[s], __builtin_assume_aligned(vz + (16 * s + 4 * j) * NG, 4));
                if constexpr (NG == 1) t.kz[s] = kz[16 * s + col];
                else if constexpr (NG == 2) t.kz[s] = *(const uint16_t *)(kz + (16 * s + col) * 2);
                else t.kz[s] = *(const uint32_t *)(kz + (16 * s + col) * 4);
            }
            if constexpr (D == 128) {
#pragma unroll
                for (int s = 0; s < 2; s++) *(U4 *)&t.v[4 * s] = *(const U4 *)(v + (16 * s + lane / 4) * 64 + lane % 4 * 16);
            } else *(U4 *)&t.v[0] = *(const U4 *)(v + lane / 2 * 32 + lane % 2 * 16);
        };

        auto process = [&](Kv4Tile<D, NG> &t, int key0) {
            // ---- V codes to LDS
            if constexpr (D == 128) {
#pragma unroll
                for (int s = 0; s < 2; s++) *(U4 *)(mine + (16 * s + lane / 4) * VROW + lane % 4 * 16) = *(const U4 *)&t.v[4 * s];
            } else *(U4 *)(mine + lane / 2 * VROW + lane % 2 * 16) = *(const U4 *)&t.v[0];
            // ---- scores: lane = row `col`, keys 16 s + 4 j + e
            float sv[2][4], top = -INFINITY;
            const int room = (t.there ? bound : 0) - key0 - 4 * j;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                uint32_t d[KS];
                if constexpr (D == 128) {
                    U4 x = {t.k[s][0], t.k[s][1], t.k[s][2], t.k[s][3]};
                    int4_transpose(x);
                    d[0] = x.x, d[1] = x.y, d[2] = x.z, d[3] = x.w;
                } else {
                    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
                    const u2_t x = __builtin_bit_cast(u2_t, __builtin_amdgcn_permlane32_swap(t.k[s][0], t.k[s][1], false, false));
                    d[0] = x.x, d[1] = x.y;
                }
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    pairs.at(t.kz[s] >> (8 * g) & 15u);
                    f4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int m = 0; m < MPG; m++) x = mfma16(pairs(d[g * MPG + m]), qf[g * MPG + m], x);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int n = e * NG + g;
                        sum[e] = fmaf(x[e], kv4_half<T>(t.ks[s][n / 2], n & 1), sum[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float big = 0.f;
#pragma unroll
                    for (int g = 0; g < NG; g++) big = fmaxf(big, fabsf(kv4_half<T>(t.vs[s][(e * NG + g) / 2], (e * NG + g) & 1)));
                    sv[s][e] = 16 * s + e < room ? sum[e] * csc : -INFINITY;
                    top = fmaxf(top, sv[s][e] + kv4_lift(big));
                }
            }
            top = xor32_max(xor16_max(top));
            const float Mn = fmaxf(M, top), ref = Mn == -INFINITY ? 0.f : Mn;
            const float alpha = __builtin_amdgcn_exp2f(M - ref);
            M = Mn;
            float ps = 0.f;
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    sv[s][e] = __builtin_amdgcn_exp2f(sv[s][e] - ref);
                    ps += sv[s][e];
                }
            l = fmaf(l, alpha, ps);
            if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
                for (int c = 0; c < D / 16; c++) acc[c] *= alpha;
            }
            // ---- O^T += V^T . P
            const int i = lane & 15, n = i & 7, key = 4 * j + ((n & 1) << 1) + (n >> 2) + ((n & 2) << 3);
            const char *from = mine + key * VROW + (i >> 3) * 8;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                U4 p[2];
                {
                    float w[2][4];
#pragma unroll
                    for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int e = 0; e < 4; e++) w[s][e] = 16 * s + e < room ? sv[s][e] * kv4_half<T>(t.vs[s][(e * NG + g) / 2], (e * NG + g) & 1) : 0.f;
#pragma unroll
                    for (int part = 0; part < 2; part++)
                        p[part] = U4{take_part<f16_t>(w[0][0], w[0][1]), take_part<f16_t>(w[0][2], w[0][3]), take_part<f16_t>(w[1][0], w[1][1]), take_part<f16_t>(w[1][2], w[1][3])};
                }
                h2_t off[4];
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    // zero points of keys (4 j, 4 j + 1) and (4 j + 2, 4 j + 3): bytes NG e + g
                    uint32_t z01, z23;
                    if constexpr (NG == 1) {
                        z01 = __builtin_amdgcn_perm(0u, t.vz[s][0], 0x0C010C00u);
                        z23 = __builtin_amdgcn_perm(0u, t.vz[s][0], 0x0C030C02u);
                    } else if constexpr (NG == 2) {
                        z01 = t.vz[s][0] >> (8 * g);
                        z23 = t.vz[s][1] >> (8 * g);
                    } else {
                        z01 = __builtin_amdgcn_perm(t.vz[s][1], t.vz[s][0], g == 0 ? 0x0C040C00u : g == 1 ? 0x0C050C01u : g == 2 ? 0x0C060C02u : 0x0C070C03u);
                        z23 = __builtin_amdgcn_perm(t.vz[s][3], t.vz[s][2], g == 0 ? 0x0C040C00u : g == 1 ? 0x0C050C01u : g == 2 ? 0x0C060C02u : 0x0C070C03u);
                    }
                    off[2 * s] = kv4_low(z01);
                    off[2 * s + 1] = kv4_high(z23);
                }
#pragma unroll
                for (int c2 = g * MPG; c2 < (g + 1) * MPG; c2++) {
                    typedef int i2_t __attribute__((ext_vector_type(2)));
                    const i2_t w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i2_t *)(from + 16 * c2));
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const U4 codes = kv4_pairs((uint32_t)w[x], off, pairs.nibbles0, pairs.nibbles1);
                        acc[2 * c2 + x] = mfma16(codes, p[0], acc[2 * c2 + x]);
                        acc[2 * c2 + x] = mfma16(codes, p[1], acc[2 * c2 + x]);
                    }
                }
            }
        };

        // tiles of this wave: k0 + 32 (wave + 4 n); the loads behind the last one repeat it
        const int nt = k1 > k0 ? (k1 - k0 - 32 * wave + kKv4Unit - 1) / kKv4Unit : 0;
        if (nt > 0) {
            Kv4Tile<D, NG> ta, tb;
            auto tile_at = [&](int n) { return k0 + 32 * wave + kKv4Unit * min(n, nt - 1); };
            load(ta, tile_at(0));
            for (int n = 0;;) {
                load(tb, tile_at(n + 1));
                process(ta, tile_at(n));
                if (++n >= nt) break;
                load(ta, tile_at(n + 1));
                process(tb, tile_at(n));
                if (++n >= nt) break;
            }
        }
        // ---- the waves' results meet in LDS
        l = xor32_sum(xor16_sum(l));
        if (lane < 16) {
            m_s[wave * 16 + lane] = M;
            l_s[wave * 16 + lane] = l;
        }
        if (col < R) {
#pragma unroll
            for (int c = 0; c < D / 16; c++) *(f4_t *)(o_s(wave) + col * D + 16 * c + 4 * j) = acc[c];
        }
        __syncthreads();
        const bool whole = at == 0 && end == n_units;
        const size_t slot = 2 * (size_t)blockIdx.x + (unit != share.first);
        for (int x = tid; x < R * (D / 4); x += NW * 64) {
            const int r = x / (D / 4), d = x % (D / 4) * 4;
            float mt = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; w++) mt = fmaxf(mt, m_s[w * 16 + r]);
            float lt = 0.f;
            f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float c = m_s[w * 16 + r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_s[w * 16 + r] - mt);
                lt = fmaf(l_s[w * 16 + r], c, lt);
                const f4_t ow = *(const f4_t *)(o_s(w) + r * D + d);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = fmaf(ow[e], c, o[e]);
            }
            if (whole) {
                T *out = (T *)a.out + (((size_t)b * a.Hq + h * G + r % G) * a.Sq + r / G) * D + d;
                const float inv = lt == 0.f ? 0.f : 1.0f / lt;
                *(uint2 *)out = uint2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
            } else {
                *(f4_t *)(a.part_o + (slot * R + r) * D + d) = o;
                if (d == 0) *(float2 *)(a.part_ml + (slot * R + r) * 2) = float2{mt, lt};
            }
        }
        unit += end - at;
        if (unit >= stop) break;
        __syncthreads();  // (the next keys' V codes take the place of the results)
        at = 0;
        if (++h == a.c.Hkv) {
            h = 0;
            b++;
            seq = PagedSeq(a.c, b, a.Sq);
            n_units = max(1, (seq.len + kKv4Unit - 1) / kKv4Unit);
        }
    }
}

// Joins the parts of a (sequence, kv head) that several workgroups had: a workgroup for each of them.
template <typename T, int D> __global__ __launch_bounds__(256) void attn_kv4_join_kernel(Kv4Args a) {
    const int lane = threadIdx.x & 63, pair = blockIdx.x, b = pair / a.c.Hkv, h = pair % a.c.Hkv;
    const int G = a.Hq / a.c.Hkv, R = G * a.Sq;
    // the units in front of the pair's, and how many there are in all
    int front = 0, total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int n = b0 + lane < a.B ? Kv4Share<kKv4Unit>::units(a.c, b0 + lane, a.Sq) : 0;
        total += wave_sum_i32(n);
        front += wave_sum_i32(b0 + lane < b ? n : 0);
    }
    const int n_units = Kv4Share<kKv4Unit>::units(a.c, b, a.Sq);
    const int quota = (total * a.c.Hkv + a.grid - 1) / a.grid;
    const int u0 = front * a.c.Hkv + h * n_units, w0 = u0 / quota, w1 = (u0 + n_units - 1) / quota;
    if (w0 == w1) return;
    for (int x = threadIdx.x; x < R * (D / 4); x += 256) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        auto slot = [&](int w) { return (2 * (size_t)w + (w == w0 && u0 != w * quota)) * R + r; };
        float mt = -INFINITY;
        for (int w = w0; w <= w1; w++) mt = fmaxf(mt, a.part_ml[slot(w) * 2]);
        float lt = 0.f;
        f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int w = w0; w <= w1; w++) {
            const float2 ml = *(const float2 *)(a.part_ml + slot(w) * 2);
            const f4_t ow = *(const f4_t *)(a.part_o + slot(w) * D + d);
            const float c = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mt);
            lt = fmaf(ml.y, c, lt);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(ow[e], c, o[e]);
        }
        T *out = (T *)a.out + (((size_t)b * a.Hq + h * G + r % G) * a.Sq + r / G) * D + d;
        const float inv = lt == 0.f ? 0.f : 1.0f / lt;
        *(uint2 *)out = uint2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
    }
}

}  // namespace mynn
