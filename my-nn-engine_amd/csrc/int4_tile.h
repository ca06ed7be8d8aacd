// Many rows of activations times 4-bit weights: eight waves of 64 x 64, as 128 rows x 256 columns or 64 x 512.
//
// Activations, codes, scales and zero points go from memory to LDS without passing registers (global_load_lds), a piece of 128 columns
// a stage, three stages where they fit: a piece is asked for two pieces ahead, because a weight tile's first reader waits for HBM.
// (Weights and scales loaded into registers instead were waited for at every piece, with all that had been asked for since: 304 us
// for 777 x 28672 x 4096, 231 with those loads left out.)  The codes are converted in registers, by each wave for its columns.
// v_mfma 32x32 with the activations as the rows, so that a lane's 16 sums belong to one weight row and meet one scale.  A group's sum
// starts from zero in registers of its own and is added, scaled, to the total: the codes' differences are exact in every type, so nothing
// is rounded before the store, where weights dequantised to 16 bits would be rounded once each.
//
// What bounds it: MFMAs against the vector operations of two waves a SIMD -- for 32 MFMAs (int8: 16) of a wave and piece, 16 dwords of codes
// (12 operations each in fp16, 19 in bf16, 9 to int8) and 64 sums to scale (int8: a conversion more).
#pragma once
#include "int4_rows.h"

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

// LDS of a stage: activations, codes, then a dword for each column's scale and one for its zero point, for each group of a piece
template <bool I8, int FL, int WM, int WN> struct Int4Tile {
    static constexpr int BM = 64 * WM, BN = 64 * WN, PARTS = 4 / FL;
    static constexpr int ROW = I8 ? 128 : 256;  // bytes of a piece of an activation row
    static constexpr int A = BM * ROW, W = BN * 64, S = BN * 4 * PARTS;
    static constexpr int STAGE = A + W + 2 * S;
    static constexpr int NS = 3 * STAGE <= 160 * 1024 ? 3 : 2;
    static constexpr int LA = A / 8192, LW = W / 8192, LS = PARTS * WN * 2 / 8;  // load instructions of a wave and stage
    static_assert(WM * WN == 8 && NS * STAGE <= 160 * 1024, "");
};

// 4 or 1 or 2 bytes a lane to LDS dword lds + 4 * lane
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void load_u16_to_lds(const void *p, uint32_t lds) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
__device__ inline void load_u8_to_lds(const void *p, uint32_t lds) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
#pragma clang diagnostic pop

template <typename T, bool I8, int FL, int WM, int WN>
__global__ __launch_bounds__(512, 2) void int4_tile_kernel(Int4Args p) {
    using G = Int4Tile<I8, FL, WM, WN>;
    constexpr int EB = I8 ? 1 : 2, ROW = G::ROW, PARTS = G::PARTS, NS = G::NS;
    constexpr int SP = (I8 ? 1 : 2) * FL;  // instructions to a scale
    constexpr int CPR = ROW / 16;          // 16-byte chunks of a row
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int tiles_m = (p.M + G::BM - 1) / G::BM;
    // Consecutive workgroups go round-robin over the 8 XCDs: an id becomes an index that is contiguous inside an XCD, where the row
    // tiles that share weights follow one another.
    int tm, tn;
    {
        const int nb = gridDim.x, x = blockIdx.x & 7, per = nb >> 3, rem = nb & 7;
        const int l = x * per + min(x, rem) + (blockIdx.x >> 3);
        tn = l / tiles_m;
        tm = l - tn * tiles_m;
    }
    const int m0 = __builtin_amdgcn_readfirstlane(tm * G::BM), n0 = __builtin_amdgcn_readfirstlane(tn * G::BN);
    const int groups = p.K / p.group, pieces = (p.K + 127) >> 7;
    const int c32 = lane & 31, kh = lane >> 5;

    // Staging: an instruction fills a kilobyte of whole rows.  The chunk at position q of row r is q ^ key(r), so that the reads of
    // neighbouring rows fall into different banks.  Offsets are from 4096 bytes in front of the tile's first row, less what load_group_to_lds adds.
    auto akey = [](int r) { return I8 ? (r >> 1) & 7 : r & 15; };
    auto wkey = [](int r) { return (r >> 2) & 3; };
    uint32_t aoff[G::LA], woff[G::LW];
#pragma unroll
    for (int i = 0; i < G::LA; i++) {
        const int at = (wave * G::LA + i) * 64 + lane, r = at / CPR;
        aoff[i] = (uint32_t)min(r, p.M - 1 - m0) * (uint32_t)(p.K * EB) + 16u * (uint32_t)((at % CPR) ^ akey(r)) + 4096u - 1024u * (i % 4);
    }
#pragma unroll
    for (int i = 0; i < G::LW; i++) {
        const int at = (wave * G::LW + i) * 64 + lane, r = at / 4;
        woff[i] = (uint32_t)min(r, p.N - 1 - n0) * (uint32_t)(p.K >> 1) + 16u * (uint32_t)((at % 4) ^ wkey(r)) + 4096u - 1024u * (i % 4);
    }
    const char *abase = (const char *)p.act + (size_t)m0 * p.K * EB - 4096;
    const char *wbase = (const char *)p.wq + (size_t)n0 * (p.K >> 1) - 4096;
    // scales by the first half of the loads of this kind, zero points by the second (scales again where there are none: all waves have the
    // same number in flight)
    const uint32_t at0 = lds_offset(lds);
    auto stage = [&](int c, int slot) {
        const uint32_t to = at0 + slot * G::STAGE;
        uint32_t ao[G::LA], wo[G::LW];
#pragma unroll
        for (int i = 0; i < G::LA; i++) ao[i] = aoff[i];
#pragma unroll
        for (int i = 0; i < G::LW; i++) wo[i] = woff[i];
        if (FL < 4 && 128 * c + 128 > p.K) {  // (chunks behind the row are not multiplied: its last one in their place)
            const int alast = (p.K - 128 * c) * EB / 16 - 1, wlast = (p.K - 128 * c) / 32 - 1;
#pragma unroll
            for (int i = 0; i < G::LA; i++) {
                const int at = (wave * G::LA + i) * 64 + lane;
                ao[i] -= 16u * (uint32_t)max(((at % CPR) ^ akey(at / CPR)) - alast, 0);
            }
#pragma unroll
            for (int i = 0; i < G::LW; i++) {
                const int at = (wave * G::LW + i) * 64 + lane;
                wo[i] -= 16u * (uint32_t)max(((at % 4) ^ wkey(at / 4)) - wlast, 0);
            }
        }
        const char *a = abase + (size_t)c * ROW, *w = wbase + (size_t)c * 64;
#pragma unroll
        for (int i = 0; i + 4 <= G::LA; i += 4) load_group_to_lds<4>(a, ao + i, to + (wave * G::LA + i) * 1024);
        if constexpr (G::LA % 4) load_group_to_lds<G::LA % 4>(a, ao + G::LA / 4 * 4, to + (wave * G::LA + G::LA / 4 * 4) * 1024);
        load_group_to_lds<G::LW>(w, wo, to + G::A + wave * G::LW * 1024);
#pragma unroll
        for (int i = 0; i < G::LS; i++) {
            const int v = wave * G::LS + i, half = PARTS * WN;          // (of the wave alike)
            const bool zeros = v >= half;
            const int u = zeros ? v - half : v, part = u / WN, block = u % WN;
            const size_t n = min(n0 + 64 * block + lane, p.N - 1);
            const int g = FL == 4 ? (p.pieces_magic ? (int)__umulhi((uint32_t)c, p.pieces_magic) : c) : min(c * PARTS + part, groups - 1);
            const uint32_t slot_at = to + G::A + G::W + v * 256;
            if (zeros && p.zero) load_u8_to_lds(p.zero + n * groups + g, slot_at);
            else load_u16_to_lds((const uint16_t *)p.scale + n * groups + g, slot_at);
        }
    };
    constexpr int INFLIGHT = G::LA + G::LW + G::LS;

    f16x_t tot[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) tot[i][t][e] = 0.f;

    stage(0, 0);
    if (NS == 3 && pieces > 1) stage(1, 1);
    int slot = 0;
    for (int c = 0; c < pieces; c++) {
        // this piece has arrived (the next one may be on its way), and nobody reads the stage that is filled next any more
        if (NS == 3 && c + 1 < pieces) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(INFLIGHT) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (c + NS - 1 < pieces) stage(c + NS - 1, slot == 0 ? NS - 1 : slot - 1);
        const char *at = lds + slot * G::STAGE;
        slot = slot == NS - 1 ? 0 : slot + 1;

        uint32_t w[2][8];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int r = 64 * wn + 32 * t + c32;
            const char *row = at + G::A + r * 64;
            if constexpr (FL == 1) {
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    const uint2 v = *(const uint2 *)(row + (h ^ wkey(r)) * 16 + 8 * kh);
                    w[t][2 * h] = v.x;
                    w[t][2 * h + 1] = v.y;
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const U4 v = *(const U4 *)(row + ((2 * h + kh) ^ wkey(r)) * 16);
#pragma unroll
                    for (int j = 0; j < 4; j++) w[t][4 * h + j] = v[j];
                }
            }
        }
#pragma unroll
        for (int part = 0; part < PARTS; part++) {
            if (FL < 4 && 128 * c + 32 * FL * part >= p.K) break;
            float s[2];
            uint32_t z[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const char *sz = at + G::A + G::W + ((part * WN + wn) * 64 + 32 * t + c32) * 4;
                const uint16_t half = *(const uint16_t *)sz;
                s[t] = Elem<T>::ld((const T *)&half, 0);
                z[t] = p.zero ? *(const uint32_t *)(sz + G::S) & 15u : 8u;
            }
            std::conditional_t<I8, i16v_t, f16x_t> acc[2][2] = {{{}, {}}, {{}, {}}};
            const std::conditional_t<I8, Int4ZeroI8, Int4Zero<T>> conv[2] = {std::conditional_t<I8, Int4ZeroI8, Int4Zero<T>>(z[0]), std::conditional_t<I8, Int4ZeroI8, Int4Zero<T>>(z[1])};
#pragma unroll
            for (int k = 0; k < SP; k++) {
                const int st = part * SP + k;  // instruction of the piece
                int chunk;
                if constexpr (I8) chunk = FL == 1 ? 2 * st + kh : 4 * (st >> 1) + 2 * kh + (st & 1);
                else chunk = FL == 1 ? 4 * (st >> 1) + 2 * kh + (st & 1) : 8 * (st >> 2) + 4 * kh + (st & 3);
                U4 a[2], b[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int r = 64 * wm + 32 * i + c32;
                    a[i] = *(const U4 *)(at + r * ROW + (chunk ^ akey(r)) * 16);
                }
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if constexpr (I8) b[t] = conv[t](w[t][2 * st], w[t][2 * st + 1]);
                    else b[t] = conv[t](w[t][st]);
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        if constexpr (I8)
                            acc[i][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i4_t, a[i]), __builtin_bit_cast(i4_t, b[t]), acc[i][t], 0, 0, 0);
                        else acc[i][t] = Mfma<T>::run(a[i], b[t], acc[i][t]);
                    }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) tot[i][t][e] = fmaf(s[t], (float)acc[i][t][e], tot[i][t][e]);
        }
    }

#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int row = m0 + 64 * wm + 32 * i + 8 * (e >> 2) + 4 * kh + (e & 3);
            if (row >= p.M) continue;
            const float as = I8 ? Elem<T>::ld((const T *)p.act_scale, row) : 1.f;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int n = n0 + 64 * wn + 32 * t + c32;
                if (n < p.N) Elem<T>::st((T *)p.out, (size_t)row * p.N + n, I8 ? tot[i][t][e] * as : tot[i][t][e]);
            }
        }
}

}  // namespace mynn
