// The form for many rows: blocks of 32 query rows of a kv head (query heads times new tokens, the heads of a token next to each other) as the columns of
// v_mfma_f32_32x32x16_f16.
//
// A workgroup of QW x KW waves has QW blocks of rows and walks their keys in tiles of KEYS, a KW-th of each tile a wave.  Codes travel global -> registers (a tile ahead)
// -> (code - zero) in fp16 -> LDS, once for all rows of the workgroup: two stages, one barrier a tile (tiles of 128 keys: one stage, two barriers).
//   S^T = K . Q^T      per group of columns; a key's scale meets the group's sum
//   softmax            a lane has ONE row and half of the keys of each 32
//   O^T += V^T . P^T   p * vs as two fp16 numbers, or three of bf16 (attention_kv4.h); P stays in registers (the D layout of S^T is the B layout of P^T with the keys in the order 4g+0..3, 8+4g+0..3), V^T
//                      comes from the row-major tile by transposing reads
// Vector operations and matrix instructions bound it together (busy 65 and 42 % of the time at 4 x 2048 rows): 380 of the one for 48 of the other in a wave's 64 keys of 32 rows,
// 100 of them the staging's.  4 prompts of 2048 rows, 32 / 8 heads of 128, groups of 128, bf16: 234 us in a program's calls, 0.59 PFLOP/s (the products alone, at what a large
// matrix product reaches: 112; the second of them is done twice); fp16, 4 x 512 rows behind 3000 200.  Blocks of 256 rows, as eight waves or as four with 64 rows each, share
// a tile's staging between more rows and hold one workgroup a CU: no faster, and 310 us where this took 230.  Raised priorities around the products, and reads of their operands
// ahead in a fixed order, were within 4 % of this, 64 columns and groups of 32 slower.
// Codes leave a dword in the order of kv4_pairs, so columns lie in that order inside every 8: queries are put in the same order when they are read, results back when stored.
#pragma once
#include "attention_kv4.h"

namespace mynn {

template <int D, int NG, int QW, int KW, int KEYS> struct Kv4Block {
    static constexpr int ROWB = D * 2, TILEB = KEYS * ROWB, THREADS = QW * KW * 64, ROWS = QW * 32, NH = KEYS / 32 / KW;
    static constexpr int UNITS = KEYS * 4 / THREADS;  // a thread stages a quarter of a row, of K and of V
    static constexpr int SCALES = 2 * NG * KEYS * 4, FLAGS = KEYS / 16 * 4;
    static constexpr int STAGE = 2 * TILEB + SCALES + FLAGS;
    static constexpr int WORDS = D / 2 + 2;  // of a lane's result: reference, sum, O^T
    static constexpr int MERGE = KW > 1 ? QW * KW * 64 * WORDS * 4 : 0;
    static constexpr int STAGES = KEYS == 64 ? 2 : 1;  // (two workgroups a CU)
    static constexpr int LDS = STAGES * STAGE > MERGE ? STAGES * STAGE : MERGE;
    static_assert(NH >= 1 && UNITS >= 1 && STAGE % 16 == 0, "whole 32s of keys a wave, whole quarter rows a thread");
};

// Keys of a range in tiles: ranges of about the same length in all blocks of the call, so many that the workgroups all run at once.  (The lengths are known on the device alone;
// a wave adds them up, 64 sequences at a time.)
__device__ inline int kv4_range_length(const Kv4Args &a, int rows, int keys, int lane) {
    const int G = a.Hq / a.c.Hkv;
    float sum = 0.f;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        float x = 0.f;
        if (b0 + lane < a.B) {
            const PagedSeq s(a.c, b0 + lane, a.Sq);
            const int middle = s.fresh ? s.bound(s.fresh / 2, a.causal) : 0;
            x = (float)((s.fresh * G + rows - 1) / rows) * (float)((middle + keys - 1) / keys);
        }
        sum += wave_sum(x);
    }
    return __builtin_amdgcn_readfirstlane(max(2, (int)ceilf(sum * (float)a.c.Hkv / (0.875f * (float)a.grid))));
}
__device__ __forceinline__ int kv4_ranges(int tiles, int length, int most) { return min(max((tiles + length - 1) / length, 1), most); }

template <typename T, int D, int NG, int QW, int KW, int KEYS> __global__ __launch_bounds__(QW *KW * 64, 2) void attn_kv4_tile_kernel(Kv4Args a) {
    using B = Kv4Block<D, NG, QW, KW, KEYS>;
    constexpr int KS = D / 16, DT = D / 32, NH = B::NH, DW = D / 32, ROWB = B::ROWB, KPG = KS / NG, TPG = DT / NG;
    // p * vs for the second product in fp16: two numbers of 11 bits.  (One is off by as much as results in fp16 are rounded.  Results in bf16 hide most of that, and 4 x 2048 rows took
    // 196 us for 225; but those of many rows then differed by 10^-3 from what few rows, 22 bits all, and 32-bit operations give, 6 10^-5 with two.)
    constexpr int PARTS = 2;
    extern __shared__ __align__(16) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wave = w % QW, kg = w / QW, col = lane & 31, g = lane >> 5;
    const int G = a.Hq / a.c.Hkv, R = G * a.Sq;
    // kv heads next to each other (XCDs take turns: one works on as few heads as it goes), blocks of rows with the most keys first.
    const int i0 = blockIdx.x, i1 = i0 / a.c.Hkv, h = i0 - i1 * a.c.Hkv;
    int b, block, range = 0;
    if (a.c.fresh || a.ranges > 1) {
        // Then sequences, ranges outermost.  Workgroups go to the shader engines in turn, and those that end at once should not have every other turn: 2 pieces of prompts, 512
        // rows and 79, take 95 us, 108 with the sequences inside the blocks (97 with them taking turns), 8 of up to 1024 rows 170, 245 (175), and 32 x 5 rows over 4000 keys, 2 ranges of 4
        // there, 62, with the ranges inside 104.
        const int i2 = i1 / a.blocks;
        block = i1 - i2 * a.blocks, range = i2 / a.B, b = i2 - range * a.B;
    } else {
        // All blocks have rows: sequences inside the blocks, taking turns, and the heaviest of all go first (4 x 2048 rows, four times as many workgroups as run at once, 233 us;
        // outermost 239).
        block = i1 / a.B, b = (i1 - block * a.B + block / 2) % a.B;
    }
    const int row0 = (a.blocks - 1 - block) * B::ROWS;
    int length = 0;
    if (a.ranges > 1) {
        length = kv4_range_length(a, B::ROWS, KEYS, lane);
        if (i0 == 0 && tid == 0) *a.length = length;
    }
    const PagedSeq seq(a.c, b, a.Sq);
    const int valid = seq.fresh * G;  // rows behind it are zeros
    auto out_row = [&](int r) { return (T *)a.out + (((size_t)b * a.Hq + h * G + r % G) * a.Sq + r / G) * D; };
    if (row0 >= valid) {
        if (range == 0)
            for (int x = tid; x < min(B::ROWS, R - row0) * (D / 8); x += B::THREADS) *(U4 *)(out_row(row0 + x / (D / 8)) + x % (D / 8) * 8) = U4{0u, 0u, 0u, 0u};
        return;
    }
    auto bound_of = [&](int r) { return seq.bound(min(r, valid - 1) / G, a.causal); };
    const int ntiles = (bound_of(row0 + B::ROWS - 1) + KEYS - 1) / KEYS;
    const int nz = a.ranges > 1 ? kv4_ranges(ntiles, length, a.ranges) : 1;
    if (range >= nz) return;
    const int t0 = (int)((long)ntiles * range / nz), t1 = (int)((long)ntiles * (range + 1) / nz);
    const int row = row0 + 32 * wave + col, row_c = min(row, valid - 1);
    const int bound = bound_of(row), wave_last = row0 + 32 * wave < valid ? bound_of(row0 + 32 * wave + 31) : 0;

    // ---- staging
    constexpr int QUARTERS = B::THREADS / 4;
    const int quarter = tid & 3, sg = quarter * NG / 4;
    const int psh = a.c.page_shift, pmask = (1 << psh) - 1;
    int pages = -1, pages_at = -(1 << 30);
    bool all_there = true;
    for (int p = (t0 * KEYS) >> psh; p <= (t1 * KEYS - 1) >> psh; p += 64) {
        int x = 0;
        if (p + lane < a.c.pages_per_seq && (p + lane) << psh < seq.len) x = a.c.table[(size_t)b * a.c.pages_per_seq + p + lane];
        all_there = all_there && __builtin_amdgcn_ballot_w64((unsigned)x >= (unsigned)a.c.n_pages) == 0;
    }
    struct Raw {
        uint32_t codes[DW];
        T scale;
        uint8_t zero;
    } raw[B::UNITS][2];  // keys, values
    int raw_there[B::UNITS];
    auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < B::UNITS; u++) {
            // (a wave's 16 rows lie in one page)
            const int first = t * KEYS + u * QUARTERS + 16 * w, p = first >> psh;
            if (p - pages_at >= 64 || p < pages_at) {
                pages_at = p;
                pages = p + lane < a.c.pages_per_seq ? a.c.table[(size_t)b * a.c.pages_per_seq + p + lane] : -1;
                if ((unsigned)pages >= (unsigned)a.c.n_pages) pages = -1;
            }
            const int page = __builtin_amdgcn_readlane(pages, p - pages_at);
            raw_there[u] = page >= 0;
            const size_t r = (((size_t)max(page, 0) * a.c.Hkv + h) << psh) + (size_t)(first & pmask) + (lane >> 2);
#pragma unroll
            for (int n = 0; n < 2; n++) {
                Raw &x = raw[u][n];
                const bool v = n == 1;
                __builtin_memcpy(&x.codes, __builtin_assume_aligned((const uint8_t *)(v ? a.c.v : a.c.k) + r * (D / 2) + quarter * (D / 8), D / 8), D / 8);
                x.scale = ((const T *)(v ? a.c.v_scale : a.c.k_scale))[r * NG + sg];
                x.zero = (v ? a.c.v_zero : a.c.k_zero)[r * NG + sg];
            }
        }
    };
    auto k_swz = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
    auto v_swz = [](int r) { return D == 128 ? (r & 3) * 5 : (((r >> 1) ^ r) & 1) << 2; };
    const float minus = kv4_minus();
    Int4Pairs pairs;
    Kv4Keys keys;
    Kv4Band<T, 8> band;  // (the same in all waves: each settles it from what lies in LDS)
    auto store = [&](char *stage, int key0) __attribute__((always_inline)) {
        float *scales = (float *)(stage + 2 * B::TILEB);
        int *there = (int *)(scales + 2 * NG * KEYS);
#pragma unroll
        for (int u = 0; u < B::UNITS; u++) {
            const int r = u * QUARTERS + (tid >> 2);
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const Raw &x = raw[u][n];
                const bool v = n == 1;
                if (v) pairs.at(x.zero & 15u);
                else keys.at(x.zero & 15u);
                const int swz = v ? v_swz(r) : k_swz(r);
                char *to = stage + (v ? B::TILEB : 0) + r * ROWB;
#pragma unroll
                for (int i = 0; i < DW; i++) *(U4 *)(to + (((quarter * DW + i) ^ swz) << 4)) = v ? pairs(x.codes[i]) : keys(x.codes[i]);
                // (values that no row sees have the scale 0)
                const bool seen = !v || (raw_there[u] && key0 + r < seq.len);
                if (quarter % (4 / NG) == 0) scales[(v ? NG * KEYS : 0) + sg * KEYS + r] = seen ? Elem<T>::ld(&x.scale, 0) : 0.f;
            }
            const bool seen = raw_there[u] && key0 + r < seq.len;
            const uint64_t off = __builtin_amdgcn_ballot_w64(seen && band.off(band.bits(__builtin_bit_cast(uint16_t, raw[u][1].scale), 0)) > band.last);
            if (lane == 0) there[r >> 4] = raw_there[u] | (off != 0 ? 2 : 0);
        }
    };
    if (t0 < t1) load(t0);

    // ---- Q^T: B operand, columns 16 ks + 8 g .. +7 in the codes' order, as fp16 times a power of two of the row
    U4 qf[KS];
    Kv4Score score;
    {
        const T *q = (const T *)a.q + (((size_t)b * a.Hq + h * G + row_c % G) * a.Sq + row_c / G) * D;
        U4 x[KS];
        float f[8], peak = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            x[ks] = *(const U4 *)(q + 16 * ks + 8 * g);
            widen8<T>(x[ks], f);
#pragma unroll
            for (int e = 0; e < 8; e++) peak = fmaxf(peak, fabsf(f[e]));
        }
        const int exponent = kv4_query_exponent(xor32_max(peak));
        // (a scale below zero turns the queries around: that of the scores is not, and their largest is that of the sums)
        const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            widen8<T>(x[ks], f);
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] *= sign;
            qf[ks] = kv4_queries(f, exponent);
        }
        score = Kv4Score::of<T>(fabsf(a.scale), exponent);
    }
    f16x_t o[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[t][e] = 0.f;
    float M = -INFINITY, l = 0.f;
    int unit_of_sums = band.unit;
    const int krow = col * ROWB + ((g ^ k_swz(col)) << 4);
    int vrow[DT];
    {
        const int i = lane & 15, r = 4 * g + (i >> 2);
#pragma unroll
        for (int t2 = 0; t2 < DT; t2++) vrow[t2] = r * ROWB + (((4 * t2 + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ v_swz(r)) << 4) + 8 * (i & 1);
    }

    auto tile = [&](const char *stage, int key0, auto masked, auto in_parts) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value, WIDE = decltype(in_parts)::value;
        const int off = kg * 32 * NH;  // this wave's keys of the tile
        const char *kt = stage + off * ROWB, *vt = kt + B::TILEB;
        const float *ksc = (const float *)(stage + 2 * B::TILEB) + off, *vsc = ksc + NG * KEYS;
        const int *there = (const int *)(vsc + NG * KEYS - off) + off / 16;
        f16x_t s[NH];
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int hf = 0; hf < NH; hf++) {
                if (NG > 1 && (hf == 0 || NG == 4)) __builtin_amdgcn_sched_barrier(0);  // (operands read ahead for several groups take more registers than there are)
                f16x_t x;
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] = 0.f;
#pragma unroll
                for (int ks = gr * KPG; ks < (gr + 1) * KPG; ks++) x = Mfma<f16_t>::run(*(const U4 *)(kt + (krow ^ (32 * ks)) + 32 * hf * ROWB), qf[ks], x);
#pragma unroll
                for (int e4 = 0; e4 < 4; e4++) {
                    const f4_t f = *(const f4_t *)&ksc[gr * KEYS + 32 * hf + 8 * e4 + 4 * g];
#pragma unroll
                    for (int e = 0; e < 4; e++) s[hf][4 * e4 + e] = gr == 0 ? x[4 * e4 + e] * f[e] : fmaf(x[4 * e4 + e], f[e], s[hf][4 * e4 + e]);
                }
            }
        if (!std::is_same<T, f16_t>::value && __builtin_expect(score.far != 0, 0)) {
            const float f = score.far_by();
#pragma unroll
            for (int hf = 0; hf < NH; hf++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[hf][e] *= f;
        }
        float top = -INFINITY;
        uint32_t seen[NH];  // MASKED: a bit for each of the lane's keys of a 32
#pragma unroll
        for (int hf = 0; hf < NH; hf++) {
            seen[hf] = ~0u;
            if (MASKED) {
                seen[hf] = 0;
                const int room = bound - key0 - 32 * hf - 4 * g;
                const uint32_t pages = (there[2 * hf] & 1 ? 0xFFu : 0u) | (there[2 * hf + 1] & 1 ? 0xFF00u : 0u);
#pragma unroll
                for (int e = 0; e < 16; e++) seen[hf] |= (uint32_t)(8 * (e >> 2) + (e & 3) < room) << e;
                seen[hf] &= pages;
#pragma unroll
                for (int e = 0; e < 16; e++) s[hf][e] = seen[hf] >> e & 1 ? s[hf][e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, s[hf][e]);
        }
        top = xor32_max(top);
        top = top == -INFINITY ? top : top * score.by;
        const bool up = top > M + kKv4Lag;
        if (__builtin_amdgcn_ballot_w64(up) != 0 || band.unit != unit_of_sums) {
            const float mn = up ? top : M, corr = __builtin_amdgcn_exp2f((up ? M - mn : 0.f) + (float)(band.unit - unit_of_sums));
            M = mn;
            unit_of_sums = band.unit;
            l *= corr;
#pragma unroll
            for (int t2 = 0; t2 < DT; t2++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[t2][e] *= corr;
        }
        float by = score.by, ref = M == -INFINITY ? 0.f : M - (float)band.unit;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(fabsf(ref) > 0x1p20f) != 0, 0)) {
            // scores so large that what M's rounding took off it, or the unit next to it, is no small thing (the fused step below has the scores' products whole)
            const float m = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int hf = 0; hf < NH; hf++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float x = s[hf][e] * by;
                    s[hf][e] = x - m;
                }
            by = 1.f, ref = -(float)band.unit;
        }
        float lt = 0.f;
#pragma unroll
        for (int hf = 0; hf < NH; hf++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[hf][e], by, -ref));
                s[hf][e] = MASKED ? (seen[hf] >> e & 1 ? p : 0.f) : p;
                lt += s[hf][e];
            }
        l += lt;
#pragma unroll
        for (int gr = 0; gr < NG; gr++)
#pragma unroll
            for (int st = 0; st < 2 * NH; st++) {
                const int e0 = 8 * (st & 1);
                float p[8];
#pragma unroll
                for (int e4 = 0; e4 < 2; e4++) {
                    const f4_t f = *(const f4_t *)&vsc[gr * KEYS + 16 * st + 8 * e4 + 4 * g];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = s[st >> 1][e0 + 4 * e4 + e];
                        p[4 * e4 + e] = MASKED ? (seen[st >> 1] >> (e0 + 4 * e4 + e) & 1 ? x * f[e] : 0.f) : x * f[e];
                    }
                }
                auto product = [&](int t2, auto &&take) __attribute__((always_inline)) {
                    const char *vr = vt + vrow[t2] + 16 * st * ROWB;
                    const uint2 lo = lds_read_tr16(vr), hi = lds_read_tr16(vr + 8 * ROWB);
                    take(U4{lo.x, lo.y, hi.x, hi.y});
                };
                if constexpr (WIDE) {
#pragma unroll 1
                    for (int part = 0; part < kParts<bf16_t>; part++) {
                        const U4 pf = {take_part<bf16_t>(p[0], p[1]), take_part<bf16_t>(p[2], p[3]), take_part<bf16_t>(p[4], p[5]), take_part<bf16_t>(p[6], p[7])};
#pragma unroll
                        for (int t2 = gr * TPG; t2 < (gr + 1) * TPG; t2++)
                            product(t2, [&](const U4 &codes) __attribute__((always_inline)) { o[t2] = Mfma<bf16_t>::run(kv4_as_bf16(codes), pf, o[t2]); });
                    }
                } else {
                    U4 pf[PARTS];
#pragma unroll
                    for (int part = 0; part < PARTS; part++)
                        pf[part] = U4{kv4_take(p[0], p[1], minus), kv4_take(p[2], p[3], minus), kv4_take(p[4], p[5], minus), kv4_take(p[6], p[7], minus)};
#pragma unroll
                    for (int t2 = gr * TPG; t2 < (gr + 1) * TPG; t2++)
                        product(t2, [&](const U4 &codes) __attribute__((always_inline)) {
#pragma unroll
                            for (int part = 0; part < PARTS; part++) o[t2] = Mfma<f16_t>::run(codes, pf[part], o[t2]);
                        });
                }
            }
    };

    int t = t0, stage = 0;
    auto next = [&]() __attribute__((always_inline)) {
        char *here = sm + stage * B::STAGE;
        if (B::STAGES == 1 && t > t0) __syncthreads();
        store(here, t * KEYS);  // (tile t - 2, which lay here, is behind the last barrier for every wave)
        if (t + 1 < t1) load(t + 1);
        __syncthreads();
        // scales that the band does not let through, in any of the tile's rows
        const float *vsc = (const float *)(here + 2 * B::TILEB) + NG * KEYS;
        int any = 0;
#pragma unroll
        for (int i = 0; i < KEYS / 16; i++) any |= ((const int *)(vsc + NG * KEYS))[i];
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(any) & 2, 0)) {
            int lo = 255, hi = 0;
#pragma unroll
            for (int i = 0; i < NG * KEYS / 64; i++) band.among(vsc[64 * i + lane], lo, hi);
            band.settle(lo, hi);
        }
        if (B::STAGES == 2) stage ^= 1;
        return here;
    };
    // the tiles that all rows of the workgroup see in full, then those with hidden keys; and all from the first on whose scales do not fit fp16.  (Loops of their own: with two
    // kinds of tile in one, the results were copied from where one leaves them to where the other expects them.)
    const int full = min(t1, seq.bound(row0 / G, a.causal) / KEYS);
    const char *here = nullptr;
    auto key_of = [&](int n) { return n * KEYS + kg * 32 * NH; };
    for (; t < full && all_there; t++) {
        here = next();
        if (band.wide) break;
        tile(here, 0, std::false_type{}, std::false_type{});
    }
    for (; t < t1 && !band.wide; t++) {
        here = next();
        if (band.wide) break;
        if (key_of(t) < wave_last) tile(here, key_of(t), std::true_type{}, std::false_type{});
    }
    while (t < t1) {
        if (key_of(t) < wave_last) tile(here, key_of(t), std::true_type{}, std::true_type{});
        if (++t < t1) here = next();
    }

    l = xor32_sum(l);
    if constexpr (KW > 1) {
        if (unit_of_sums != band.unit) {  // (a wave whose rows do not see the last tiles)
            const float f = __builtin_amdgcn_ldexpf(1.f, band.unit - unit_of_sums);
            l *= f;
#pragma unroll
            for (int t2 = 0; t2 < DT; t2++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[t2][e] *= f;
            unit_of_sums = band.unit;
        }
        // the waves that shared a block of rows: the first of them takes the others' results in
        __syncthreads();
        float *to = (float *)sm + (size_t)w * 64 * B::WORDS + lane;
        if (kg > 0) {
            to[0] = M;
            to[64] = l;
#pragma unroll
            for (int t2 = 0; t2 < DT; t2++)
#pragma unroll
                for (int e = 0; e < 16; e++) to[(2 + 16 * t2 + e) * 64] = o[t2][e];
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int k = 1; k < KW; k++) {
            const float *from = (const float *)sm + (size_t)(k * QW + wave) * 64 * B::WORDS + lane;
            const float mo = from[0], mn = fmaxf(M, mo);
            const float ca = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mn), cb = mo == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mo - mn);
            l = l * ca + from[64] * cb;
            M = mn;
#pragma unroll
            for (int t2 = 0; t2 < DT; t2++) {
#pragma unroll
                for (int e = 0; e < 16; e++) o[t2][e] = o[t2][e] * ca + from[(2 + 16 * t2 + e) * 64] * cb;
                asm volatile("" : "+v"(o[t2]));  // (here, and not with the stores: the waves' results of all would have to be kept till then)
            }
        }
    }
    // (The lane's place once more, from the wave: what it is known by at the start would be one register too many over the loops.)
    const int place = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), row_out = row0 + 32 * wave + (place & 31), gr = place >> 5;
    const float plain = kv4_plain(unit_of_sums);
    const float inv = nz > 1 ? plain : row_out >= valid || l == 0.f ? 0.f : 1.0f / l;
    const size_t line = (((size_t)b * a.c.Hkv + h) * R + row_out) * a.ranges + range;
#pragma unroll
    for (int t2 = 0; t2 < DT; t2++)
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++) {
            // columns 0, 4, 1, 5 of an 8 in the lower lanes, 2, 6, 3, 7 in the upper: 0 .. 3 and 4 .. 7
            float x0 = o[t2][4 * e4], x2 = o[t2][4 * e4 + 1], x1 = o[t2][4 * e4 + 2], x3 = o[t2][4 * e4 + 3];
            permlane32_swap(x0, x2);
            permlane32_swap(x1, x3);
            const int d = 32 * t2 + 8 * e4 + 4 * gr;
            if (row_out >= R) continue;
            if (nz > 1) *(f4_t *)(a.part_o + line * D + d) = f4_t{x0 * inv, x1 * inv, x2 * inv, x3 * inv};
            else if (row_out >= valid) *(uint2 *)(out_row(row_out) + d) = uint2{0u, 0u};
            else *(uint2 *)(out_row(row_out) + d) = uint2{pack2<T>(x0 * inv, x1 * inv), pack2<T>(x2 * inv, x3 * inv)};
        }
    if (nz > 1 && gr == 0 && row_out < R) *(float2 *)(a.part_ml + line * 2) = float2{M, l * plain};
}

// Joins the ranges of keys of each row.  Blocks with one range, or none of the sequence's own rows, are done already.
template <typename T, int D> __global__ __launch_bounds__(256) void attn_kv4_ranges_kernel(Kv4Args a, int block_rows, int keys) {
    const int G = a.Hq / a.c.Hkv, R = G * a.Sq;
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x, line = at / (D / 4);
    const int d = (int)(at % (D / 4)) * 4;
    if (line >= (size_t)a.B * a.c.Hkv * R) return;
    const int most = a.ranges, pair = (int)(line / R), r = (int)(line % R), b = pair / a.c.Hkv, h = pair % a.c.Hkv;
    const PagedSeq seq(a.c, b, a.Sq);
    const int valid = seq.fresh * G, row0 = r / block_rows * block_rows;
    if (row0 >= valid) return;
    const int nz = kv4_ranges((seq.bound((min(row0 + block_rows, valid) - 1) / G, a.causal) + keys - 1) / keys, *a.length, most);
    if (nz == 1) return;
    const uint64_t *ml = (const uint64_t *)a.part_ml + line * most;
    const float *po = a.part_o + line * most * D + d;
    auto lo = [](uint64_t w) { return __builtin_bit_cast(float, (uint32_t)w); };
    float mt = -INFINITY, lt = 0.f;
    f4_t o = {0.f, 0.f, 0.f, 0.f};
    // four ranges at a time, with a reference of their own
    for (int z0 = 0; z0 < nz; z0 += 4) {
        uint64_t w[4];
        f4_t x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int z = min(z0 + i, nz - 1);
            w[i] = ml[z];
            x[i] = *(const f4_t *)(po + (size_t)z * D);
        }
        float mn = mt;
#pragma unroll
        for (int i = 0; i < 4; i++) mn = fmaxf(mn, lo(w[i]));
        const float c0 = mt == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mt - mn);
        mt = mn;
        lt *= c0;
        o *= c0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float c = lo(w[i]) == -INFINITY || z0 + i >= nz ? 0.f : __builtin_amdgcn_exp2f(lo(w[i]) - mt);
            lt = fmaf(lo(w[i] >> 32), c, lt);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(x[i][e], c, o[e]);
        }
    }
    const float inv = 1.0f / lt;
    uint2 x = uint2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
    if (r >= valid || lt == 0.f) x = uint2{0u, 0u};
    *(uint2 *)((T *)a.out + (((size_t)b * a.Hq + h * G + r % G) * a.Sq + r / G) * D + d) = x;
}

// Rows of a workgroup, blocks of rows of a kv head, and the ranges that their keys come in.
struct Kv4TilePlan {
    int rows, blocks, ranges;
};
// by type, a translation unit each (attention_kv4_go.h)
template <typename T> int kv4_tile_go(const Kv4Args &a, int D, int group, const Kv4TilePlan &p, hipStream_t s);

}  // namespace mynn
