// Many rows of activations times 4-bit weights: tiles of 32 TI rows (TI = 1 .. 4), a wave 32 TI x 32; eight waves side by side where tiles are tall, two
// workgroups of four a compute unit where they are not.
//
// Activations, codes, scales and zero points go from memory to LDS without passing registers (global_load_lds), a piece of 128 columns
// a stage, so that a piece is asked for two to five pieces ahead.  (Weights and scales loaded into registers were waited for at every piece, with all
// that had been asked for since: 777 x 28672 x 4096 fp16 304 us, 231 with those loads left out.)  Each wave converts the codes of its columns in
// registers, once for all rows of the tile; taller waves were better than wider ones (128 x 32 against 64 x 64: 275 against 282 us).
// v_mfma 32x32 with the activations as the rows, so that a lane's 16 sums belong to one weight row and meet one scale.  A group's sum
// starts from zero in registers of its own and is added, scaled, to the total: the codes' differences are exact in every type, so nothing
// is rounded before the store, where weights dequantised to 16 bits would be rounded once each.
//
// What bounds it.  Tall tiles: of a piece (128 rows x 256 columns, 2.2 us in rounds that fill the device) the MFMAs alone are 1.6; the rest is what the
// vector operations (12 for eight codes in fp16, 19 in bf16, 9 to int8; 64 sums to scale; a wave's seven loads) do not hide behind them.  2048 x 28672 x
// 4096 fp16 501 - 514 us, 0.95 PFLOP/s; 128 x 65536 x 4096 of int8 66 - 68 us, 1.02 POP/s.  Short ones: the steps of a piece one after the other, 0.65 us
// with 32 rows, 0.85 with 64 (its barrier and its reads from LDS are half of that; read a piece ahead they cost as much elsewhere).
#pragma once
#include "int4_codes.h"

namespace mynn {

typedef int i16v_t __attribute__((ext_vector_type(16)));

// code - zero of eight codes as T, exactly.  fp16: a byte's two nibbles under exponents that make them 1024 + n and 64 + n; `off` takes both
// off.  bf16: through signed bytes, the upper halves of their f32 forms (at most four significant bits).
template <typename T> struct Int4Zero;
template <> struct Int4Zero<f16_t> {
    h2_t off;
    uint32_t nibbles = 0x00F0000Fu, exponents = 0x54006400u;
    __device__ explicit Int4Zero(uint32_t z) : off{(_Float16)(-1024.f - (float)z), (_Float16)(-64.f - (float)z)} {
        // (in vector registers: one instruction takes both, but at most one constant from elsewhere)
        asm volatile("" : "+v"(nibbles), "+v"(exponents));
    }
    __device__ U4 operator()(uint32_t w) const {
        auto two = [&](uint32_t sel) {
            const uint32_t n = (__builtin_amdgcn_perm(0u, w, sel) & nibbles) | exponents;
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2_t, n) + off);
        };
        return U4{two(0x0C000C00u), two(0x0C010C01u), two(0x0C020C02u), two(0x0C030C03u)};
    }
};
template <> struct Int4Zero<bf16_t> {
    uint32_t zz;
    __device__ explicit Int4Zero(uint32_t z) : zz(z * 0x01010101u) {}
    __device__ U4 operator()(uint32_t w) const {
        const uint32_t e = (((w & 0x0F0F0F0Fu) | 0x80808080u) - zz) ^ 0x80808080u, o = ((((w >> 4) & 0x0F0F0F0Fu) | 0x80808080u) - zz) ^ 0x80808080u;
        auto two = [&](int sh) {
            const float a = (float)(int8_t)((e >> sh) & 0xFF), b = (float)(int8_t)((o >> sh) & 0xFF);
            return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
        };
        return U4{two(0), two(8), two(16), two(24)};
    }
};
struct Int4ZeroI8 {
    uint32_t zz;
    __device__ explicit Int4ZeroI8(uint32_t z) : zz(z * 0x01010101u) {}
    __device__ U4 operator()(uint32_t w0, uint32_t w1) const {
        const uint2 a = int4_to_i8(w0, zz), b = int4_to_i8(w1, zz);
        return U4{a.x, a.y, b.x, b.y};
    }
};

// LDS of a stage: codes, then a dword for each column's scale and one for its zero point, for each group of a piece, then activations of
// 32 TI rows; as many stages as there is room for, up to six: short tiles wait for memory, not for the matrix cores.
// WIDE (groups of 32 and 64): a piece's scales of a column as one dword or two and its zero points as one, where rows are whole pieces and addresses
// allow it, instead of a load for each, every one of which asks for a line of its own.
template <bool I8, int FL, int NW, bool WIDE> struct Int4Tile {
    static constexpr int LDS = NW * 20 * 1024;  // (a compute unit has 160 KB and takes eight waves)
    static constexpr int BN = 32 * NW, PARTS = 4 / FL;
    static constexpr int ROW = I8 ? 128 : 256;  // bytes of a piece of an activation row
    static constexpr int W = BN * 64, S = BN * 4 * PARTS, HEAD = W + 2 * S;
    static constexpr int LW = 2, LS = !WIDE ? PARTS : FL == 1 ? 2 : 1;  // load instructions of a wave and stage, codes and scales
    static constexpr int loads(int ti) { return (32 * ti * ROW + 1024 * NW - 1) / (1024 * NW); }
    static constexpr int stage(int ti) { return HEAD + 1024 * NW * loads(ti); }
    static constexpr int stages(int ti) { return LDS / stage(ti) < 6 ? LDS / stage(ti) : 6; }
};

// 4 bytes, 2 or one a lane to LDS dword lds + 4 * lane, from base + off (base wave-uniform)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int BYTES> __device__ inline void load_small_to_lds(const char *base, uint32_t off, uint32_t lds) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    base = scalar_pointer(base);
    if constexpr (BYTES == 4) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
    else if constexpr (BYTES == 2) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
    else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

// The row tiles of a column: `tall` of `high` blocks of 32 rows, then short ones of `low`.
struct Int4Rows {
    int tall, high, low, tiles;
};
// K in ranges whose sums are added up in their order: by workgroups of their own that leave them in `part` ([range][M][N], for
// int4_join_kernel), or without it one after the other in one workgroup -- the same bits.
struct Int4Ranges {
    int count;
    float *part;
};

// the waiting part of a step: all but the `ahead` youngest stages of LOADS instructions have arrived
template <int LOADS, int MOST> __device__ inline void wait_stages(int ahead) {
    static_assert(LOADS * MOST < 64, "the counter has six bits");
    if constexpr (MOST > 0) {
        if (ahead >= MOST) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS * MOST) : "memory");
        else wait_stages<LOADS, MOST - 1>(ahead);
    } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <typename T, bool I8, int FL, int NW, bool WIDE>
__global__ __launch_bounds__(64 * NW, 2) void int4_tile_kernel(Int4Args p, Int4Rows rows, Int4Ranges ranges) {
    using G = Int4Tile<I8, FL, NW, WIDE>;
    constexpr int EB = I8 ? 1 : 2, ROW = G::ROW, PARTS = G::PARTS;
    constexpr int SP = (I8 ? 1 : 2) * FL;  // instructions to a scale
    constexpr int CPR = ROW / 16;          // 16-byte chunks of a row
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Consecutive workgroups go round-robin over the 8 XCDs: an id becomes an index that is contiguous inside an XCD, where the row
    // tiles that share weights follow one another.  All tall tiles come before the short ones, which fill the gaps of the last round.
    int tm, tn;
    {
        const int x = blockIdx.x & 7, i = blockIdx.x >> 3;
        const int columns = (p.N + G::BN - 1) / G::BN * (ranges.part ? ranges.count : 1), tall = rows.tall * columns, others = rows.tiles - rows.tall, low = others * columns;
        const int mine = (tall >> 3) + (x < (tall & 7)), y = (x - tall) & 7;  // (the XCDs that got one tall tile less come first for the short ones)
        if (i < mine) {
            const int l = x * (tall >> 3) + min(x, tall & 7) + i;
            tn = l / rows.tall;
            tm = l - tn * rows.tall;
        } else {
            const int l = y * (low >> 3) + min(y, low & 7) + i - mine;
            tn = l / others;
            tm = rows.tall + l - tn * others;
        }
    }
    // (ranges of their own: the column tile's, side by side)
    int z0 = 0, z1 = ranges.count;
    if (ranges.part) {
        z0 = tn % ranges.count;
        z1 = z0 + 1;
        tn /= ranges.count;
    }
    const bool is_tall = tm < rows.tall;
    const int height = __builtin_amdgcn_readfirstlane(is_tall ? rows.high : rows.low);
    const int m0 = 32 * __builtin_amdgcn_readfirstlane(is_tall ? tm * rows.high : rows.tall * rows.high + (tm - rows.tall) * rows.low), n0 = __builtin_amdgcn_readfirstlane(tn * G::BN);
    const int groups = p.K / p.group, pieces = (p.K + 127) >> 7;
    const int c32 = lane & 31, kh = lane >> 5;

    // Staging: an instruction fills a kilobyte of whole rows.  The chunk at position q of row r is q ^ key(r), so that the reads of
    // neighbouring rows fall into different banks.
    auto akey = [](int r) { return I8 ? (r >> 1) & 7 : r & 15; };
    auto wkey = [](int r) { return (r >> 2) & 3; };
    const char *abase = (const char *)p.act + (size_t)m0 * p.K * EB, *wbase = (const char *)p.wq + (size_t)n0 * (p.K >> 1);
    const uint32_t at0 = lds_offset(lds);
    auto run = [&](auto ti_) {
        constexpr int TI = decltype(ti_)::value;
        constexpr int LA = G::loads(TI), STAGE = G::stage(TI), NS = G::stages(TI), INFLIGHT = LA + G::LW + G::LS;
        // This wave's loads of a stage, one instruction each: LA of activations, LW of codes, LS of scales (the first half of the waves) or zero
        // points (the second; one scale for all its lanes where there are none: all waves have the same number in flight).
        uint32_t aoff[LA], woff[G::LW], soff[G::LS];
#pragma unroll
        for (int i = 0; i < LA; i++) {
            const int at = (wave * LA + i) * 64 + lane, r = at / CPR;
            aoff[i] = (uint32_t)min(r, p.M - 1 - m0) * (uint32_t)(p.K * EB) + 16u * (uint32_t)((at % CPR) ^ akey(r));
        }
#pragma unroll
        for (int i = 0; i < G::LW; i++) {
            const int at = (wave * G::LW + i) * 64 + lane, r = at / 4;
            woff[i] = (uint32_t)min(r, p.N - 1 - n0) * (uint32_t)(p.K >> 1) + 16u * (uint32_t)((at % 4) ^ wkey(r));
        }
#pragma unroll
        for (int i = 0; i < G::LS; i++) {
            const int v = wave * G::LS + i, row = min(64 * (v % (NW / 2)) + lane, p.N - 1 - n0);
            if constexpr (WIDE) soff[i] = (uint32_t)row * (uint32_t)groups * (v < NW / (3 - G::LS) ? 2u : p.zero && v < NW / (3 - G::LS) + NW / 2 ? 1u : 0u);
            else soff[i] = (uint32_t)row * (uint32_t)groups * (v < NW / 2 * PARTS ? 2u : p.zero ? 1u : 0u);
        }
        auto load = [&](int i, int c, int slot) {
            const uint32_t to = at0 + slot * STAGE;
            // (of a broken piece: chunks behind the row are not multiplied, its last one in their place)
            const bool broken = FL < 4 && !WIDE && 128 * c + 128 > p.K;
            if (i < LA) {
                uint32_t off = aoff[i];
                if (broken) {
                    const int at = (wave * LA + i) * 64 + lane;
                    off -= 16u * (uint32_t)max(((at % CPR) ^ akey(at / CPR)) - ((p.K - 128 * c) * EB / 16 - 1), 0);
                }
                load_to_lds(abase + (size_t)c * ROW, off, to + G::HEAD + (wave * LA + i) * 1024);
            } else if (i < LA + G::LW) {
                i -= LA;
                uint32_t off = woff[i];
                if (broken) {
                    const int at = (wave * G::LW + i) * 64 + lane;
                    off -= 16u * (uint32_t)max(((at % 4) ^ wkey(at / 4)) - ((p.K - 128 * c) / 32 - 1), 0);
                }
                load_to_lds(wbase + (size_t)c * 64, off, to + (wave * G::LW + i) * 1024);
            } else {
                i -= LA + G::LW;
                if constexpr (WIDE) {
                    // dword `which` of the scales, then the zero points, then (groups of 32) nothing: one scale for all lanes
                    constexpr int scales = NW / (3 - G::LS);
                    const int v = wave * G::LS + i, which = v / (NW / 2);
                    const size_t first = (size_t)n0 * groups + c * PARTS;
                    const uint32_t where = to + G::W + (v < scales ? v * 256 : G::S + (v - scales) * 256);
                    if (v >= scales && v < scales + NW / 2 && p.zero) load_small_to_lds<FL == 1 ? 4 : 2>((const char *)p.zero + first, soff[i], where);
                    else load_small_to_lds<4>((const char *)p.scale + (v < scales ? first * 2 + 4 * which : 0), soff[i], where);
                    return;
                }
                const int v = wave * G::LS + i, part = v / (NW / 2) % PARTS;  // (of the wave alike)
                const int g = FL == 4 ? (p.pieces_magic ? (int)__umulhi((uint32_t)c, p.pieces_magic) : c) : min(c * PARTS + part, groups - 1);
                const size_t first = (size_t)n0 * groups + g;
                if (v >= NW / 2 * PARTS && p.zero) load_small_to_lds<1>((const char *)p.zero + first, soff[i], to + G::W + v * 256);
                else load_small_to_lds<2>((const char *)p.scale + first * 2, soff[i], to + G::W + v * 256);
            }
        };
        auto stage = [&](int c, int slot) {
#pragma unroll
            for (int i = 0; i < INFLIGHT; i++) load(i, c, slot);
        };
        constexpr bool SEQ = TI <= 2;  // (K is in ranges for short tiles only)
        f16x_t tot[TI], sum[SEQ ? TI : 1];
        for (int z = z0; z < z1; z++) {
            const int c0 = (int)((unsigned)(pieces * z) / (unsigned)ranges.count), c1 = (int)((unsigned)(pieces * (z + 1)) / (unsigned)ranges.count);
            if (z > z0) __syncthreads();
#pragma unroll
            for (int i = 0; i < TI; i++)
#pragma unroll
                for (int e = 0; e < 16; e++) tot[i][e] = 0.f;
#pragma unroll
            for (int i = 0; i < NS - 1; i++)
                if (c0 + i < c1) stage(c0 + i, i);
            int slot = 0;
            for (int c = c0; c < c1; c++) {
                // this piece has arrived (later ones may be on their way), and nobody reads the stage that is filled next any more
                wait_stages<INFLIGHT, NS - 2>(c1 - 1 - c);
                __syncthreads();
                const int to = slot == 0 ? NS - 1 : slot - 1;
                const char *at = lds + slot * STAGE;
                slot = slot == NS - 1 ? 0 : slot + 1;

                uint32_t w[8];
                {
                    const int r = 32 * wave + c32;
                    const char *row = at + r * 64;
                    if constexpr (FL == 1) {
#pragma unroll
                        for (int h = 0; h < 4; h++) {
                            const uint2 v = *(const uint2 *)(row + (h ^ wkey(r)) * 16 + 8 * kh);
                            w[2 * h] = v.x;
                            w[2 * h + 1] = v.y;
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const U4 v = *(const U4 *)(row + ((2 * h + kh) ^ wkey(r)) * 16);
#pragma unroll
                            for (int j = 0; j < 4; j++) w[4 * h + j] = v[j];
                        }
                    }
                }
                // WIDE has whole pieces alone: a column's scales and zero points are read at once, and a piece's groups are one block of code (365 x 2560 x
                // 2048 of int8 in groups of 32 31.5 -> 26.4 us, 411 x 4096 x 14336 114 -> 103).  Not in the tallest tiles (nor the next in fp16,
                // whose conversion holds constants), which have no registers for two groups' sums: the branch keeps their groups apart.
                constexpr bool AT_ONCE = WIDE && TI <= (std::is_same<T, f16_t>::value && !I8 && FL == 1 ? 2 : 3);
                const char *column = at + G::W + (32 * wave + c32) * 4;
                uint32_t sw[2] = {}, zw = 0x08080808u;
                if constexpr (AT_ONCE) {
                    sw[0] = *(const uint32_t *)column;
                    if constexpr (FL == 1) sw[1] = *(const uint32_t *)(column + G::BN * 4);
                    if (p.zero) zw = *(const uint32_t *)(column + G::S);
                }
                // Fragments are read an instruction ahead, in short tiles, whose products do not cover the way to LDS, all of a piece at once; the
                // loads of a later piece are asked for between the products, one here and there: the eight waves' together keep the memory pipe busy for
                // most of a piece, and a wave that waits to hand it the next one does nothing else.
                constexpr int STEPS = PARTS * SP, KEPT = TI <= 2 ? STEPS : 2;
                U4 a[KEPT][TI];
                auto fragments = [&](int st) {
                    int chunk;
                    if constexpr (I8) chunk = FL == 1 ? 2 * st + kh : 4 * (st >> 1) + 2 * kh + (st & 1);
                    else chunk = FL == 1 ? 4 * (st >> 1) + 2 * kh + (st & 1) : 8 * (st >> 2) + 4 * kh + (st & 3);
#pragma unroll
                    for (int i = 0; i < TI; i++) {
                        const int r = 32 * i + c32;
                        a[st % KEPT][i] = *(const U4 *)(at + G::HEAD + r * ROW + (chunk ^ akey(r)) * 16);
                    }
                };
#pragma unroll
                for (int st = 0; st < KEPT - 1; st++) fragments(st);
                const bool more = c + NS - 1 < c1;
#pragma unroll
                for (int part = 0; part < PARTS; part++) {
                    if (FL < 4 && !AT_ONCE && 128 * c + 32 * FL * part >= p.K) break;
                    const char *sz = column + (WIDE ? part >> 1 : part) * G::BN * 4;
                    const uint16_t half = AT_ONCE ? (uint16_t)(sw[part >> 1] >> (16 * (part & 1))) : *(const uint16_t *)(sz + (WIDE ? 2 * (part & 1) : 0));
                    const float s = Elem<T>::ld((const T *)&half, 0);
                    const uint32_t zero = AT_ONCE ? (zw >> (8 * part)) & 15u : p.zero ? *(const uint8_t *)(WIDE ? column + G::S + part : sz + G::S) & 15u : 8u;
                    const std::conditional_t<I8, Int4ZeroI8, Int4Zero<T>> conv(zero);
                    std::conditional_t<I8, i16v_t, f16x_t> acc[TI] = {};
#pragma unroll
                    for (int k = 0; k < SP; k++) {
                        const int st = part * SP + k;  // instruction of the piece
                        if (st + KEPT - 1 < STEPS) fragments(st + KEPT - 1);
                        if (more) {
#pragma unroll
                            for (int i = 0; i < INFLIGHT; i++)
                                if (i * STEPS / INFLIGHT == st) load(i, c + NS - 1, to);
                        }
                        U4 b;
                        if constexpr (I8) b = conv(w[2 * st], w[2 * st + 1]);
                        else b = conv(w[st]);
#pragma unroll
                        for (int i = 0; i < TI; i++) {
                            if constexpr (I8) acc[i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i4_t, a[st % KEPT][i]), __builtin_bit_cast(i4_t, b), acc[i], 0, 0, 0);
                            else acc[i] = Mfma<T>::run(a[st % KEPT][i], b, acc[i]);
                        }
                        if constexpr (KEPT < STEPS) __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
                    for (int i = 0; i < TI; i++)
#pragma unroll
                        for (int e = 0; e < 16; e++) tot[i][e] = fmaf(s, (float)acc[i][e], tot[i][e]);
                }
            }
            if constexpr (SEQ) {
#pragma unroll
                for (int i = 0; i < TI; i++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sum[i][e] = z == z0 ? tot[i][e] : sum[i][e] + tot[i][e];
            }
        }

        const int n = n0 + 32 * wave + c32;
#pragma unroll
        for (int i = 0; i < TI; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int row = m0 + 32 * i + 8 * (e >> 2) + 4 * kh + (e & 3);
                if (row >= p.M || n >= p.N) continue;
                const float v = SEQ ? sum[SEQ ? i : 0][e] : tot[i][e];
                if (SEQ && ranges.part) ranges.part[((size_t)z0 * p.M + row) * p.N + n] = v;
                else Elem<T>::st((T *)p.out, (size_t)row * p.N + n, I8 ? v * Elem<T>::ld((const T *)p.act_scale, row) : v);
            }
    };
    // (a loop for each height: the sums and fragments are registers)
    if constexpr (NW == 8) {
        if (height >= 3) {
            if (height == 4) run(std::integral_constant<int, 4>{});
            else run(std::integral_constant<int, 3>{});
            return;
        }
    }
    if (height == 2) run(std::integral_constant<int, 2>{});
    else run(std::integral_constant<int, 1>{});
}

// the ranges' sums added up in their order, V values a thread
template <typename T, bool I8, int V>
__global__ __launch_bounds__(256) void int4_join_kernel(T *out, const float *part, const T *act_scale, int ranges, uint32_t N, uint32_t total) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const uint32_t i = (blockIdx.x * 256u + threadIdx.x) * V;
    if (i >= total) return;
    vec sum = *(const vec *)(part + i);
#pragma unroll 8
    for (int z = 1; z < ranges; z++) sum += *(const vec *)(part + (size_t)z * total + i);
    if constexpr (I8) sum *= Elem<T>::ld(act_scale, i / N);
#pragma unroll
    for (int v = 0; v < V; v++) Elem<T>::st(out, i + v, sum[v]);
}

}  // namespace mynn
