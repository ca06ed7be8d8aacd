// The form for few rows: up to 16 query rows of a kv head (query heads times new tokens) are the 16 columns of v_mfma_f32_16x16x32_f16.
//
// A workgroup of four waves walks its run of keys, a tile a wave, the next one's codes, scales and zero points on their way to registers meanwhile.
//   S[keys x rows] = K . Q^T  per 16 keys; a lane has a key's 32 columns of 16 bytes; dwords are exchanged between its four lane groups so that each matrix
//                             instruction takes 32 neighbouring columns, of one group of columns
//   softmax                   online; a lane has one row (column of the instruction) and 4 keys of each 16
//   O^T[columns x rows] += V^T . P   V goes to LDS as codes and comes back transposed (ds_read_b64_tr_b4: of 16 rows that its lanes name, a lane receives
//                             one column); named are a lane group's own 8 keys twice, for 16 columns and the 16 behind them, so that the order of the
//                             keys is the one in which the scores lie in registers.  p * vs in two fp16 values, rounded and rest: 22 bits (or three of bf16, attention_kv4.h).
// The vector operations bound it (one pass of 32 keys, D = 128: 144 to turn codes into operands, the softmax and the look at the value scales 230 where every lane has 8 scores).  So where 8 rows or 4 are
// all there are (FOLD 2, 4), they are the columns twice or four times, and each of these takes the scores of its own 16 keys of 32 or 64: 4 for a lane.  Weights go back with
// lane rotations.
//
// Measured (kernel times; bytes at what a copy reaches, 5.1 TB/s, in brackets): one token of 64 sequences of 8192 keys, 32 / 8 heads of 128, groups of 128 104 us (110: some of
// it is from the last cache), of 64 123 (115), of 32 170 (125), 2 tokens 122 (110), 4 tokens 138 (111); 128 sequences, 32 / 4 heads of 64 85 (58), groups of 32 100 (62).  Where
// the bracket is far the vector operations are busy 80 % of the time and more.  Short calls are a chain of waits -- lengths, page table, codes, a step of 0.65 us or more for each 128 or
// 256 keys, the join's 7 us --: one sequence of 32768 keys 18.5 us, 32 of up to 4096 32, 8 x 4 tokens of up to 2000 keys 22.5.
// Units of a workgroup's run are whole steps: smaller ones dealt out better and split more steps, and took longer.  The join inside the launch or in one of its own: 32 sequences of up to
// 4096 keys 31 us and 27.3 + 4.8, one of 32768 18.5 and 15 + 6.4, 8 x 4 tokens 22 and 14.5 + 6.4, the second launch's start not counted.
#pragma once
#include "attention_kv4.h"

namespace mynn {

template <int FOLD> constexpr int kKv4Keys = FOLD == 4 ? 64 : 32;              // of a wave's tile
template <int FOLD, int W> using Kv4Run = Kv4Share<W * kKv4Keys<FOLD>>;         // a workgroup's step: W waves
template <int D, int FOLD> constexpr int kKv4TileBytes = kKv4Keys<FOLD> * (D / 2 + 16);  // of V codes in LDS

// one wave's loads of a tile, all but the codes of the values
template <int D, int NG, int FOLD> struct Kv4Tile {
    static constexpr int KW = D / 32, SUBS = kKv4Keys<FOLD> / 16, OWN = SUBS / FOLD;  // dwords of codes of a lane and 16 keys, 16s of keys, those whose scores a lane has
    uint32_t k[SUBS][KW];
    size_t row[SUBS / 2];  // of each 32 keys
    uint32_t ks[OWN][2 * NG], vs[OWN][2 * NG], vz[SUBS][NG];
    uint32_t kz[SUBS];
    int there[SUBS / 2];
};

// A (sequence, kv head) whose keys several workgroups had: w0 .. w1, the first of them in its second part where `second`.
struct Kv4Parts {
    int b, h, fresh, w0, w1, second;
};
// Joins them in their order, all THREADS of a workgroup, `ml` 64 x 16 pairs in LDS.  AGENT: past this XCD's L2.  Parts are a wait for memory each if they are asked for
// one by one: references and sums of 64 go through LDS, results come in batches, the first of them with the references.
template <typename T, int D, int ROWS, int THREADS, bool AGENT> __device__ __forceinline__ void kv4_join(const Kv4Args &a, const Kv4Parts &p, uint64_t *ml, int tid) {
    constexpr int N = (ROWS * D / 2 + THREADS - 1) / THREADS, AH = 32 / N;  // pairs of columns of a thread, parts in flight
    const int G = a.Hq / a.c.Hkv, R = G * a.Sq, n = p.w1 - p.w0 + 1;
    auto get = [](const uint64_t *x) { return AGENT ? __hip_atomic_load(x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *x; };
    auto lo = [](uint64_t w) { return __builtin_bit_cast(float, (uint32_t)w); };
    auto hi = [](uint64_t w) { return __builtin_bit_cast(float, (uint32_t)(w >> 32)); };
    auto slot = [&](int i) { return (2 * (size_t)(p.w0 + i) + (i == 0 && p.second)) * R; };
    float M[N], l[N], o0[N], o1[N];
    int r[N], d[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int x = min(tid + THREADS * k, R * (D / 2) - 1);
        r[k] = x / (D / 2), d[k] = x % (D / 2) * 2;
        M[k] = -INFINITY, l[k] = o0[k] = o1[k] = 0.f;
    }
    for (int c0 = 0; c0 < n; c0 += 64) {
        const int m = min(64, n - c0);
        uint64_t o[N][AH];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int i1 = 0; i1 < AH; i1 += AH / 4) {
                if (i0 + i1 >= m) break;
#pragma unroll
                for (int k = 0; k < N; k++)
#pragma unroll
                    for (int i = i1; i < i1 + AH / 4; i++) o[k][i] = get((const uint64_t *)(a.part_o + (slot(c0 + min(i0 + i, m - 1)) + r[k]) * D + d[k]));
            }
        };
        fetch(0);
        __syncthreads();  // (of the 64 before)
        for (int x = tid; x < m * R; x += THREADS) ml[x] = get((const uint64_t *)a.part_ml + slot(c0 + x / R) + x % R);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; k++) {
            float top = M[k];
#pragma unroll 8
            for (int i = 0; i < m; i++) top = fmaxf(top, lo(ml[i * R + r[k]]));
            const float c = M[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M[k] - top);
            M[k] = top;
            l[k] *= c, o0[k] *= c, o1[k] *= c;
        }
        for (int i0 = 0; i0 < m; i0 += AH) {
            if (i0) fetch(i0);
#pragma unroll
            for (int k = 0; k < N; k++)
#pragma unroll
                for (int i = 0; i < AH; i++) {
                    if (i0 + i >= m) break;
                    const uint64_t w = ml[(i0 + i) * R + r[k]];
                    const float c = lo(w) == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lo(w) - M[k]);
                    l[k] = fmaf(hi(w), c, l[k]);
                    o0[k] = fmaf(lo(o[k][i]), c, o0[k]);
                    o1[k] = fmaf(hi(o[k][i]), c, o1[k]);
                }
        }
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        if (tid + THREADS * k >= R * (D / 2)) break;
        T *out = (T *)a.out + (((size_t)p.b * a.Hq + p.h * G + r[k] % G) * a.Sq + r[k] / G) * D + d[k];
        const float inv = 1.0f / l[k];
        *(uint32_t *)out = l[k] == 0.f || r[k] / G >= p.fresh ? 0u : pack2<T>(o0[k] * inv, o1[k] * inv);
    }
}

constexpr int kDppRor4 = 0x124, kDppRor12 = 0x12C;  // lane i <- i - 4, i + 4, inside each row of 16
template <int CTRL> __device__ __forceinline__ uint32_t dpp_word(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false); }

template <typename T, int D, int NG, int FOLD, int NW> __global__ __launch_bounds__(NW * 64, 2) void attn_kv4_stream_kernel(Kv4Args a) {
    using Tile = Kv4Tile<D, NG, FOLD>;
    constexpr int GROUP = D / NG, KS = D / 32, VROW = D / 2 + 16;  // bytes of a row of V codes in LDS
    constexpr int MPG = GROUP / 32;                                               // matrix instructions of a group
    constexpr int KEYS = kKv4Keys<FOLD>, UNIT = NW * KEYS, SUBS = Tile::SUBS, OWN = Tile::OWN, COLS = 16 / FOLD;
    extern __shared__ __align__(16) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, j = lane >> 4;
    const int G = a.Hq / a.c.Hkv, R = G * a.Sq;
    const int wave_bytes = max(kKv4TileBytes<D, FOLD>, R * D * 4);
    char *mine = sm + wave * wave_bytes;
    float *m_s = (float *)(sm + NW * wave_bytes), *l_s = m_s + NW * 16;
    int *flag = (int *)(l_s + NW * 16);
    auto o_s = [&](int w) { return (float *)(sm + w * wave_bytes); };

    Kv4Run<FOLD, NW> share(a, blockIdx.x, lane);
    const int first = __builtin_amdgcn_readfirstlane(share.first), total = __builtin_amdgcn_readfirstlane(share.total), quota = __builtin_amdgcn_readfirstlane(share.quota);
    int unit = first;
    if (unit >= total) return;
    const int stop = min(unit + quota, total);
    Kv4Parts front{0, 0, 0, 0, -1, 0}, tail{0, 0, 0, 0, -1, 0};  // what this workgroup has parts of
    Int4Pairs pairs;
    Kv4Keys keys;
    const float minus = kv4_minus();
    const int psh = a.c.page_shift, pmask = (1 << psh) - 1;
    const int fold = col / COLS, row = col % COLS < R ? col % COLS : 0;  // this lane's row, and which of the folds has it

    // What is needed once for a (sequence, kv head) is computed each time: kept over the walk over the keys, it took the registers of the tiles.
    auto again = [](int x) __attribute__((always_inline)) {
        asm volatile("" : "+v"(x));
        return x;
    };
    // the (sequence, kv head) whose keys are next, and the units of it that are this workgroup's
    int b = __builtin_amdgcn_readfirstlane(share.b), h, at;
    PagedSeq seq = share.seq(a, b, lane);
    int n_units = share.units(seq);
    {
        const int r = unit - __builtin_amdgcn_readfirstlane(share.before);
        h = r / n_units;
        at = r - h * n_units;
    }
    // the entries of 64 pages of the sequence, a lane each; and of the first 64 of the (sequence, kv head) behind it, which are asked for as soon as this one's walk begins
    int pages, pages_at, pages_next = -1;
    auto entries = [&](int seq_b, int p) __attribute__((always_inline)) {
        int x = -1;
        if (p + lane < a.c.pages_per_seq) x = a.c.table[(size_t)seq_b * a.c.pages_per_seq + p + lane];
        return x;
    };
    auto look_up = [&](int p) __attribute__((always_inline)) {
        pages_at = p;
        pages = entries(b, p);
    };
    auto load = [&](Tile &t, int key0) __attribute__((always_inline)) {
        auto put = [](auto &to, const void *from) { __builtin_memcpy(&to, from, sizeof to); };
        size_t *r0 = t.row;
#pragma unroll
        for (int x = 0; x < SUBS / 2; x++) {  // (32 keys lie in one page; behind the sequence's last page there is none)
            const int key = key0 + 32 * x, p = key >> psh;
            if (p - pages_at >= 64) look_up(p);
            const int page = __builtin_amdgcn_readlane(pages, p - pages_at);
            t.there[x] = (unsigned)page < (unsigned)a.c.n_pages;
            // (a page that is not there: page 0 is read, and nothing made of it)
            r0[x] = (((size_t)(t.there[x] ? page : 0) * a.c.Hkv + h) << psh) + (size_t)(key & pmask);
        }
#pragma unroll
        for (int s = 0; s < SUBS; s++) {
            const size_t r = r0[s / 2] + 16 * (s & 1);
            put(t.k[s], __builtin_assume_aligned((const uint8_t *)a.c.k + r * (D / 2) + (col * (D / 2) + j * KS * 4), KS * 4));
            put(t.vz[s], __builtin_assume_aligned(a.c.v_zero + r * NG + 4 * j * NG, 4));
            const uint8_t *kz = a.c.k_zero + r * NG + col * NG;
            if constexpr (NG == 1) t.kz[s] = *kz;
            else if constexpr (NG == 2) t.kz[s] = *(const uint16_t *)kz;
            else t.kz[s] = *(const uint32_t *)kz;
        }
#pragma unroll
        for (int s = 0; s < OWN; s++) {
            // (the lane's own 16s of keys: all, or the fold's)
            const size_t r = FOLD == 1 ? r0[0] + 16 * s + 4 * j : FOLD == 2 ? r0[0] + 16 * fold + 4 * j : (fold & 2 ? r0[SUBS / 2 - 1] : r0[0]) + 16 * (fold & 1) + 4 * j;
            put(t.ks[s], __builtin_assume_aligned((const T *)a.c.k_scale + r * NG, 8));
            put(t.vs[s], __builtin_assume_aligned((const T *)a.c.v_scale + r * NG, 8));
        }
    };
    // The codes of a tile's values: asked for when those of the tile before have gone to LDS, into the same registers (two sets of them, in flight with everything
    // else of their tiles, went past 256).
    uint32_t v[SUBS * D / 32];
    auto load_values = [&](const Tile &t) __attribute__((always_inline)) {
        if constexpr (D == 128) {
#pragma unroll
            for (int s = 0; s < SUBS; s++)
                *(U4 *)&v[4 * s] = *(const U4 *)((const uint8_t *)a.c.v + (t.row[s / 2] + 16 * (s & 1)) * 64 + (lane / 4 * 64 + lane % 4 * 16));
        } else {
#pragma unroll
            for (int s = 0; s < SUBS / 2; s++) *(U4 *)&v[4 * s] = *(const U4 *)((const uint8_t *)a.c.v + t.row[s] * 32 + (lane / 2 * 32 + lane % 2 * 16));
        }
    };
    auto park_values = [&]() __attribute__((always_inline)) {
        if constexpr (D == 128) {
#pragma unroll
            for (int s = 0; s < SUBS; s++) *(U4 *)(mine + (16 * s + lane / 4) * VROW + lane % 4 * 16) = *(const U4 *)&v[4 * s];
        } else {
#pragma unroll
            for (int s = 0; s < SUBS / 2; s++) *(U4 *)(mine + (32 * s + lane / 2) * VROW + lane % 2 * 16) = *(const U4 *)&v[4 * s];
        }
    };

    // what the walk over its keys begins with, in the order in which it is waited for: page table, queries, the first tile
    Tile ta, tb;
    U4 qraw[KS];
    int k0, k1, nt;
    auto tile_at = [&](int n) __attribute__((always_inline)) { return k0 + KEYS * wave + UNIT * max(min(n, nt - 1), 0); };  // (the loads behind the last tile repeat it; without any, they are made for nothing)
    auto begin = [&]() __attribute__((always_inline)) {
        const int end = min(n_units, at + stop - unit);
        k0 = at * UNIT, k1 = min(seq.len, end * UNIT);
        nt = k1 > k0 ? (k1 - k0 - KEYS * wave + UNIT - 1) / UNIT : 0;
        const int r = again(row);
        const T *q = (const T *)a.q + (((size_t)b * a.Hq + h * G + r % G) * a.Sq + r / G) * D;
#pragma unroll
        for (int m = 0; m < KS; m++) qraw[m] = *(const U4 *)(q + (D == 128 ? 32 * m + 8 * j : 32 * m + (j & 1) * 16 + (j >> 1) * 8));
        load(ta, tile_at(0));
        load_values(ta);
        pages_next = entries(h + 1 < a.c.Hkv ? b : min(b + 1, a.B - 1), 0);
    };
    look_up((at * UNIT) >> psh);
    begin();
    while (true) {
        // ---- the rows' queries: B operand, columns 32 m + 8 j .. +7 (D = 64: in the order in which the exchange below leaves them) by pairs
        const int bound = col % COLS < R ? seq.bound(again(row) / G, a.causal) : 0;
        U4 qf[KS];
        Kv4Score score;
        {
            float x[KS][8], peak = 0.f;
#pragma unroll
            for (int m = 0; m < KS; m++) {
                widen8<T>(qraw[m], x[m]);
#pragma unroll
                for (int e = 0; e < 8; e++) peak = fmaxf(peak, fabsf(x[m][e]));
            }
            const int exponent = kv4_query_exponent(xor32_max(xor16_max(peak)));
#pragma unroll
            for (int m = 0; m < KS; m++) qf[m] = col % COLS >= R ? U4{0u, 0u, 0u, 0u} : kv4_queries(x[m], exponent);
            score = Kv4Score::of<T>(a.scale, exponent);
        }
        Kv4Band<T, 12> band;
        int unit_of_sums = band.unit;
        f4_t acc[D / 16];
#pragma unroll
        for (int c = 0; c < D / 16; c++) acc[c] = f4_t{0.f, 0.f, 0.f, 0.f};
        float M = -INFINITY, l = 0.f;

        // Tiles up to the first whose scales do not fit fp16; that one, and what follows, in a loop of its own: with both ways in one, the sums were copied from where one leaves them
        // to where the other expects them, and a way out of the middle of a tile took 25 registers more than that tile with all its keys hidden does.
        int fitting = nt;
        auto room_of = [&](const Tile &t, int key0, int limit, int s) __attribute__((always_inline)) {
            const int there = FOLD == 4 && fold >= 2 ? t.there[SUBS / 2 - 1] : t.there[0];
            return (there ? limit : 0) - key0 - 16 * (FOLD == 1 ? s : fold) - 4 * j;
        };
        auto value_scale = [&](const Tile &t, int room, int s, int e, int g) __attribute__((always_inline)) {
            uint32_t w = t.vs[s][(e * NG + g) / 2];
            if (NG == 4 && FOLD == 1) asm("" : "+v"(w));  // (made again where they are needed: 32 of them kept from the first look at them on took the registers of other things)
            return e < room ? kv4_half<T>(w, (e * NG + g) & 1) : 0.f;
        };
        auto check = [&](Tile &t, int turn, auto in_parts) __attribute__((always_inline)) {
            constexpr bool WIDE = decltype(in_parts)::value;
            const int key0 = tile_at(turn);
            int limit = bound;
            // ---- the scales of the values that the row sees
            {
                uint32_t off = 0;
                if (__builtin_amdgcn_ballot_w64(col % COLS < R && room_of(t, key0, limit, OWN - 1) < 4) == 0) {  // (all keys: two scales at a time)
                    uint32_t most = 0;
#pragma unroll
                    for (int s = 0; s < OWN; s++)
#pragma unroll
                        for (int n = 0; n < 2 * NG; n++) most = band.off2(most, t.vs[s][n]);
                    off = max(most & 0xFFFFu, most >> 16);
                } else {
#pragma unroll
                    for (int s = 0; s < OWN; s++)
#pragma unroll
                        for (int n = 0; n < 4 * NG; n++) off = max(off, n / NG < room_of(t, key0, limit, s) ? band.off(band.bits(t.vs[s][n / 2], n & 1)) : 0u);
                }
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(off > band.last) != 0, 0)) {
                    int lo = 255, hi = 0;
#pragma unroll
                    for (int s = 0; s < OWN; s++)
#pragma unroll
                        for (int n = 0; n < 4 * NG; n++) band.among(value_scale(t, room_of(t, key0, limit, s), s, n / NG, n % NG), lo, hi);
                    band.settle(lo, hi);
                    if (!WIDE && band.wide) limit = 0, fitting = turn;
                }
            }
            return limit;
        };
        auto process = [&](Tile &t, int turn, int limit, auto in_parts) __attribute__((always_inline)) {
            constexpr bool WIDE = decltype(in_parts)::value;
            const int key0 = tile_at(turn);
            // ---- scores: lane = row, keys 16 s + 4 j + e of its own 16s
            float x[NG][4], sv[OWN][4];
            auto scaled = [&](const float *y, int s, int g, int e) __attribute__((always_inline)) {
                const float f = kv4_half<T>(t.ks[s][(e * NG + g) / 2], (e * NG + g) & 1);
                sv[s][e] = g == 0 ? y[e] * f : fmaf(y[e], f, sv[s][e]);
            };
#pragma unroll
            for (int s = 0; s < SUBS; s++) {
                uint32_t d[KS];
                if constexpr (D == 128) {
                    U4 w = {t.k[s][0], t.k[s][1], t.k[s][2], t.k[s][3]};
                    int4_transpose(w);
                    d[0] = w.x, d[1] = w.y, d[2] = w.z, d[3] = w.w;
                } else {
                    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
                    const u2_t w = __builtin_bit_cast(u2_t, __builtin_amdgcn_permlane32_swap(t.k[s][0], t.k[s][1], false, false));
                    d[0] = w.x, d[1] = w.y;
                }
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    keys.at(t.kz[s] >> (8 * g) & 15u);
                    f4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int m = 0; m < MPG; m++) y = mfma16(keys(d[g * MPG + m]), qf[g * MPG + m], y);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[g][e] = FOLD == 1 || s == 0 || fold == s ? y[e] : x[g][e];
                        if (FOLD == 1) scaled(x[g], s, g, e);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);  // (operands made for all 16s of keys ahead of their products, and for all columns below, take more registers than there are)
            }
            // keys that the row does not see have no weight, and what lies in their scales does not count.  (Tiles that every row sees in full go the same way: a
            // path of their own would save 3 selections a score, 12 of 480 operations in a tile of 64 keys, and holds half as much code again.)
            float top = -INFINITY;
#pragma unroll
            for (int s = 0; s < OWN; s++) {
                const int room = room_of(t, key0, limit, s);
#pragma unroll
                for (int e = 0; e < 4; e++) {
#pragma unroll
                    for (int g = 0; g < NG; g++)
                        if (FOLD > 1) scaled(x[g], s, g, e);
                    sv[s][e] = e < room ? sv[s][e] * score.by : -INFINITY;
                    top = fmaxf(top, sv[s][e]);
                }
            }
            if (!std::is_same<T, f16_t>::value && __builtin_expect(score.far != 0, 0)) {
                const float f = score.far_by();
                top *= f;
#pragma unroll
                for (int s = 0; s < OWN; s++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sv[s][e] *= f;
            }
            top = xor32_max(xor16_max(top));
            if constexpr (FOLD >= 2) top = fmaxf(top, dpp_get<kDppRor8>(top));
            if constexpr (FOLD == 4) top = fmaxf(top, dpp_get<kDppRor4>(top));
            const float Mn = fmaxf(M, top), unit = (float)band.unit;
            float ref = Mn == -INFINITY ? 0.f : Mn - unit;
            const float alpha = Mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - Mn + (float)(band.unit - unit_of_sums));
            M = Mn;
            unit_of_sums = band.unit;
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(fabsf(ref) > 0x1p20f) != 0, 0)) {  // (scores so large that the unit is a small thing next to them: one after the other)
#pragma unroll
                for (int s = 0; s < OWN; s++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sv[s][e] -= Mn == -INFINITY ? 0.f : Mn;
                ref = -unit;
            }
            float ps = 0.f;
#pragma unroll
            for (int s = 0; s < OWN; s++)
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
            __builtin_amdgcn_sched_barrier(0);
            // ---- O^T += V^T . P
            const int i = lane & 15, n = i & 7, key = 4 * j + ((n & 1) << 1) + (n >> 2) + ((n & 2) << 3);
            const char *from = mine + key * VROW + (i >> 3) * 8;
            // a part of the weights of OWN 16s of keys as the operand: of FOLD columns that are one row, each has keys of its own
            auto operand = [&](const uint32_t (*w)[2], U4 *p) __attribute__((always_inline)) {
                const uint32_t *w0 = w[0];
                if constexpr (FOLD == 1) p[0] = U4{w0[0], w0[1], w[OWN - 1][0], w[OWN - 1][1]};
                else if constexpr (FOLD == 2) p[0] = U4{w0[0], w0[1], dpp_word<kDppRor8>(w0[0]), dpp_word<kDppRor8>(w0[1])};
                else {
                    // (columns 0 .. 3 are the ones whose results count: they take the weights of the folds behind them, 4, 8 and 12 lanes up)
                    p[0] = U4{w0[0], w0[1], dpp_word<kDppRor12>(w0[0]), dpp_word<kDppRor12>(w0[1])};
                    p[SUBS / 2 - 1] = U4{dpp_word<kDppRor8>(w0[0]), dpp_word<kDppRor8>(w0[1]), dpp_word<kDppRor4>(w0[0]), dpp_word<kDppRor4>(w0[1])};
                }
            };
#pragma unroll
            for (int g = 0; g < NG; g++) {
                float y[OWN][4];
#pragma unroll
                for (int s = 0; s < OWN; s++)
#pragma unroll
                    for (int e = 0; e < 4; e++) y[s][e] = sv[s][e] * value_scale(t, room_of(t, key0, limit, s), s, e, g);
                // fp16: rounded, and the rest, side by side.  bf16: one part after the other.
                constexpr int PARTS = WIDE ? 1 : 2, TURNS = WIDE ? kParts<bf16_t> : 1;
#pragma unroll 1
                for (int part0 = 0; part0 < TURNS; part0++) {
                    U4 p[PARTS][SUBS / 2];
                    {
                        uint32_t w[PARTS][OWN][2];
#pragma unroll
                        for (int s = 0; s < OWN; s++)
#pragma unroll
                            for (int part = 0; part < PARTS; part++)
#pragma unroll
                                for (int e = 0; e < 2; e++) w[part][s][e] = WIDE ? take_part<bf16_t>(y[s][2 * e], y[s][2 * e + 1]) : kv4_take(y[s][2 * e], y[s][2 * e + 1], minus);
#pragma unroll
                        for (int part = 0; part < PARTS; part++) operand(w[part], p[part]);
                    }
#pragma unroll
                    for (int sp = 0; sp < SUBS / 2; sp++) {
                        h2_t off[4];
#pragma unroll
                        for (int s = 0; s < 2; s++) {
                            // zero points of keys (4 j, 4 j + 1) and (4 j + 2, 4 j + 3): bytes NG e + g
                            const uint32_t *z = t.vz[2 * sp + s];
                            uint32_t z01, z23;
                            if constexpr (NG == 1) {
                                z01 = __builtin_amdgcn_perm(0u, z[0], 0x0C010C00u);
                                z23 = __builtin_amdgcn_perm(0u, z[0], 0x0C030C02u);
                            } else if constexpr (NG == 2) {
                                z01 = z[0] >> (8 * g);
                                z23 = z[1] >> (8 * g);
                            } else {
                                const uint32_t sel = 0x0C040C00u + 0x00010001u * g;
                                z01 = __builtin_amdgcn_perm(z[1], z[0], sel);
                                z23 = __builtin_amdgcn_perm(z[NG - 1], z[NG - 2], sel);
                            }
                            off[2 * s] = kv4_low(z01);
                            off[2 * s + 1] = kv4_high(z23);
                        }
#pragma unroll
                        for (int c2 = g * MPG; c2 < (g + 1) * MPG; c2++) {
                            typedef int i2_t __attribute__((ext_vector_type(2)));
                            const i2_t w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i2_t *)(from + 32 * sp * VROW + 16 * c2));
#pragma unroll
                            for (int y = 0; y < 2; y++) {
                                const U4 codes = kv4_pairs((uint32_t)w[y], off, pairs.nibbles0, pairs.nibbles1);
#pragma unroll
                                for (int part = 0; part < PARTS; part++)
                                    acc[2 * c2 + y] = WIDE ? mfma16_bf16(kv4_as_bf16(codes), p[part][sp], acc[2 * c2 + y]) : mfma16(codes, p[part][sp], acc[2 * c2 + y]);
                            }
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        };
        for (int n = 0; n < fitting; n++) {
            // (the next tile's loads have all of this one's work to arrive.  Two sets that take turns, without the copies, left the registers of the sums no
            // place to stay: up to 256 of them and scratch memory for 156 that are alive)
            load(tb, tile_at(n + 1));
            park_values();
            load_values(tb);
            process(ta, n, check(ta, n, std::false_type{}), std::false_type{});
            ta = tb;
        }
        for (int n = fitting; n < nt; n++) {  // (rare: from memory again, a tile at a time)
            look_up(tile_at(n) >> psh);
            load(ta, tile_at(n));
            load_values(ta);
            park_values();
            process(ta, n, check(ta, n, std::true_type{}), std::true_type{});
        }
        // ---- the next (sequence, kv head)'s loads before this one's results are put together
        const int done_b = b, done_h = h, done_fresh = seq.fresh, u0 = unit - at, units = n_units, end = min(n_units, at + stop - unit);
        const bool whole = at == 0 && end == n_units, second = unit != first;  // (a workgroup has two parts at the most: in its first place and in another)
        unit += end - at;
        if (h + 1 == a.c.Hkv && b + 1 == a.B) unit = max(unit, stop);  // (the last there is, whatever the lengths were when they were added up)
        if (unit < stop) {
            at = 0;
            if (++h == a.c.Hkv) {
                h = 0;
                seq = share.seq(a, ++b, lane);
                n_units = share.units(seq);
            }
            pages_at = 0;
            pages = pages_next;
            begin();
        }
        // ---- the waves' results meet in LDS
        const int me = again(lane);
        l = xor32_sum(xor16_sum(l));
        if constexpr (FOLD >= 2) l += dpp_get<kDppRor8>(l);
        if constexpr (FOLD == 4) l += dpp_get<kDppRor4>(l);
        const float plain = kv4_plain(unit_of_sums);
        l *= plain;
        if (me < 16) {
            m_s[wave * 16 + me] = M;
            l_s[wave * 16 + me] = l;
        }
        if ((me & 15) < R) {
#pragma unroll
            for (int c = 0; c < D / 16; c++) *(f4_t *)(o_s(wave) + (me & 15) * D + 16 * c + 4 * (me >> 4)) = acc[c] * plain;
        }
        __syncthreads();
        const size_t slot = 2 * (size_t)blockIdx.x + second;
        for (int x = again(tid); x < R * (D / 4); x += NW * 64) {
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
                T *out = (T *)a.out + (((size_t)done_b * a.Hq + done_h * G + r % G) * a.Sq + r / G) * D + d;
                const float inv = 1.0f / lt;
                *(uint2 *)out = lt == 0.f || r / G >= done_fresh ? uint2{0u, 0u} : uint2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
            } else {
                uint64_t *po = (uint64_t *)(a.part_o + (slot * R + r) * D + d), *ml = (uint64_t *)a.part_ml + slot * R + r;
                auto word = [](float lo, float hi) { return (uint64_t)__builtin_bit_cast(uint32_t, lo) | ((uint64_t)__builtin_bit_cast(uint32_t, hi) << 32); };
                if (a.counters) {  // (past this XCD's L2: whoever arrives last reads them)
                    __hip_atomic_store(po, word(o[0], o[1]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    __hip_atomic_store(po + 1, word(o[2], o[3]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    if (d == 0) __hip_atomic_store(ml, word(mt, lt), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                } else {
                    po[0] = word(o[0], o[1]);
                    po[1] = word(o[2], o[3]);
                    if (d == 0) *ml = word(mt, lt);
                }
            }
        }
        if (!whole) {  // the first of this workgroup's (sequence, kv head)s, or the last
            const int w0 = u0 / quota;
            const Kv4Parts p{done_b, done_h, done_fresh, w0, (u0 + units - 1) / quota, u0 != w0 * quota};
            // (each member for itself: as structures, the choice is one of addresses, and both go to scratch memory)
            auto take = [&](int Kv4Parts::*m) __attribute__((always_inline)) {
                tail.*m = second ? p.*m : tail.*m;
                front.*m = second ? front.*m : p.*m;
            };
            take(&Kv4Parts::b), take(&Kv4Parts::h), take(&Kv4Parts::fresh), take(&Kv4Parts::w0), take(&Kv4Parts::w1), take(&Kv4Parts::second);
        }
        __syncthreads();  // (the next keys' V codes take the place of the results)
        if (unit >= stop) break;
    }
    // ---- the last workgroup to arrive with a part of a (sequence, kv head) joins them all.  Both of a workgroup's parts are counted at its end: a wait in its middle is one that
    // nothing else of its own fills.
    if (!a.counters || (front.w1 < 0 && tail.w1 < 0)) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the parts are written through before they are counted
    __syncthreads();
    if (tid < 2) {
        const int w1 = tid ? tail.w1 : front.w1, n = w1 - (tid ? tail.w0 : front.w0);
        int before = -1;
        if (w1 >= 0) {
            // (the one of the first workgroup that has a part: no other (sequence, kv head) that is shared begins there, for this one goes on behind it)
            int32_t *counter = a.counters + (tid ? tail.w0 : front.w0);
            before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (before == n) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // ready for the next call
        }
        flag[tid] = before;
    }
    __syncthreads();
    const int n_front = flag[0], n_tail = flag[1];
    if (n_front >= 0 && n_front == front.w1 - front.w0) kv4_join<T, D, COLS, NW * 64, true>(a, front, (uint64_t *)sm, tid);
    if (n_tail >= 0 && n_tail == tail.w1 - tail.w0) kv4_join<T, D, COLS, NW * 64, true>(a, tail, (uint64_t *)sm, tid);
}

// The same by a launch of its own, a workgroup for each pair of sequence and kv head.
template <typename T, int D, int FOLD, int W> __global__ __launch_bounds__(256) void attn_kv4_join_kernel(Kv4Args a) {
    __shared__ uint64_t ml[64 * 16 / FOLD];
    const int lane = threadIdx.x & 63, b = blockIdx.x / a.c.Hkv, h = blockIdx.x % a.c.Hkv;
    // the units in front of the pair's, and how many there are in all
    int front = 0, total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int n = b0 + lane < a.B ? Kv4Run<FOLD, W>::units(PagedSeq(a.c, b0 + lane, a.Sq)) : 0;
        total += wave_sum_i32(n);
        front += wave_sum_i32(b0 + lane < b ? n : 0);
    }
    const PagedSeq seq(a.c, b, a.Sq);
    const int n_units = Kv4Run<FOLD, W>::units(seq);
    const int quota = Kv4Run<FOLD, W>::share_of(a, total * a.c.Hkv);
    const int u0 = front * a.c.Hkv + h * n_units, w0 = u0 / quota;
    const Kv4Parts p{b, h, seq.fresh, w0, (u0 + n_units - 1) / quota, u0 != w0 * quota};
    if (p.w1 > w0) kv4_join<T, D, 16 / FOLD, 256, false>(a, p, ml, threadIdx.x);
}

// by type, a translation unit each (attention_kv4_go.h): fold: how often the rows are put side by side
template <typename T> int kv4_stream_go(const Kv4Args &a, int D, int group, int fold, int waves, hipStream_t s);

}  // namespace mynn
