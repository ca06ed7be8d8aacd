// The residual's addition with the RMSNorm behind it: sum = T(x + residual) is stored and normalised in one pass over the row,
//   y = sum * 1/sqrt(mean(sum^2) + eps) * w,
// to the storage type or, per row, to 8 bits: step = max|y| / 127 (1 for a row of zeros), code = y / step rounded half away from zero.
// Statistics and y are held in 32 bits; y goes to 8 bits without a rounding to T in between.  A row whose y is not all finite
// gets the step NaN and codes of zero, so that a product of it is NaN and not some number.
#include <algorithm>
#include <type_traits>

#include "mfma.h"
#include "mynn_common.h"

namespace mynn {

constexpr int kAnThreads = 256;

__device__ inline float an_sum(float v, float *red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
// the largest of magnitudes, as bits: infinity is above every number and NaN above that, where fmaxf would pass it over
__device__ inline uint32_t an_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }
__device__ inline float an_max(uint32_t v, uint32_t *red) {
    for (int i = 32; i; i >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, i));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return __builtin_bit_cast(float, max(max(red[0], red[1]), max(red[2], red[3])));
}
// A row's step and the codes by it.  Below 2^-120 a row counts as zeros: the reciprocal of a step below 2^-128 is no number.
// A code is the 32-bit quotient y / step, rounded: the product with the reciprocal alone is a unit off it now and then, and with bf16 rows, of which
// 4 values in 100000 are ties, that is the other side of one (3 codes of a million).  Quotient and remainder from the rounded reciprocal as Markstein has
// it (IBM Journal of Research and Development 34, 1990): q = y * per, then q + (y - q * step) * per is the quotient rounded to nearest.
struct AnStep {
    float step, per;
    __device__ explicit AnStep(float amax) {
        const bool finite = amax < INFINITY, some = amax >= 0x1p-120f;
        step = !finite ? NAN : some ? amax / 127.0f : 1.0f;
        per = finite && some ? 1.0f / step : 0.f;
    }
    __device__ float code(float y) const {
        const float first = y * per, quotient = fmaf(fmaf(-first, step, y), per, first);
        const float q = fminf(fmaxf(roundf(quotient), -127.f), 127.f);  // half away from zero
        return per == 0.f ? 0.f : q;
    }
};

// A row whose squares have no 32-bit sum (values of 1e19 and more), or whose mean square and eps are so small that squares get lost (eps 0), is summed
// again, each value times this: the sum then lies between 2^-64 and 2^126.  0: neither (and what is not a number stays so).
__device__ inline float an_unit(float ss, int dim, float eps) { return ss == INFINITY ? 0x1p-96f : ss / (float)dim + eps < 0x1p-100f ? 0x1p96f : 0.f; }
// y = (h * first) * inv * w of such a row; large ones in two factors, because their product may be below the normal numbers
struct AnRange {
    float first, inv;
    __device__ AnRange(float unit, float ss, int dim, float eps) {
        const bool large = unit < 1.0f;
        first = large ? 0x1p-32f : unit;
        inv = (large ? 0x1p-64f : 1.0f) / sqrtf(ss / (float)dim + eps * unit * unit);
    }
};

// Rows of any length, at any address, of any type: a workgroup per row, an element a thread and step.  What a thread wrote of `sum`
// it reads again itself, so `sum` may be x or the residual, and so may `out` where no sum is asked for.  Two or three passes of which only the first reads
// from memory: rows of the others' kind are faster there (us, to T and to 8 bits: f32, one row of 4096 8.7 and 11.5, 8192 x 4096 151 and 153; bf16, 8192 x
// 4097 136 and 166 against 46 and 44 of 8192 x 4096, 500 x 1001 5.5 and 6.8).
template <typename T, bool Q8>
__global__ __launch_bounds__(kAnThreads) void add_norm_kernel(void *out_, T *y_scale, T *sum, const T *x, const T *residual, const T *w, int dim, float eps) {
    __shared__ float red[4];
    const size_t base = (size_t)blockIdx.x * dim;
    auto stored = [&](int i) {
        float v = Elem<T>::ld(x, base + i);
        return residual ? Elem<T>::rnd(v + Elem<T>::ld(residual, base + i)) : v;
    };
    auto again = [&](int i) { return sum ? Elem<T>::ld(sum, base + i) : stored(i); };
    float ss = 0.f;
    for (int i = threadIdx.x; i < dim; i += kAnThreads) {
        const float h = stored(i);
        if (sum) Elem<T>::st(sum, base + i, h);
        ss += h * h;
    }
    ss = an_sum(ss, red);
    float first = 1.0f, inv = 1.0f / sqrtf(ss / (float)dim + eps);
    if (const float unit = an_unit(ss, dim, eps); unit != 0.f) {  // (all threads alike)
        ss = 0.f;
        for (int i = threadIdx.x; i < dim; i += kAnThreads) {
            const float h = again(i) * unit;
            ss += h * h;
        }
        const AnRange range(unit, an_sum(ss, red), dim, eps);
        first = range.first;
        inv = range.inv;
    }
    auto y = [&](int i) { return ((again(i) * first) * inv) * Elem<T>::ld(w, i); };
    if constexpr (!Q8) {
        for (int i = threadIdx.x; i < dim; i += kAnThreads) Elem<T>::st((T *)out_, base + i, y(i));
    } else {
        __shared__ uint32_t peak[4];
        uint32_t amax = 0;
        for (int i = threadIdx.x; i < dim; i += kAnThreads) amax = max(amax, an_bits(y(i)));
        const AnStep step(an_max(amax, peak));
        for (int i = threadIdx.x; i < dim; i += kAnThreads) ((int8_t *)out_)[base + i] = (int8_t)step.code(y(i));
        if (threadIdx.x == 0) Elem<T>::st(y_scale, blockIdx.x, step.step);
    }
}

// sum / largest bits over the W waves of a row, in every thread
template <int W> __device__ inline float an_row_sum(float v, float *red) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < W; i++) v += red[i];
    return v;
}
template <int W> __device__ inline float an_row_max(uint32_t v, uint32_t *red) {
    auto dpp = [](uint32_t x, auto ctrl, auto rows) {
        return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    };
    using std::integral_constant;
    v = max(v, dpp(v, integral_constant<int, kDppXor1>{}, integral_constant<int, 0xF>{}));
    v = max(v, dpp(v, integral_constant<int, kDppXor2>{}, integral_constant<int, 0xF>{}));
    v = max(v, dpp(v, integral_constant<int, kDppHalfMirror>{}, integral_constant<int, 0xF>{}));
    v = max(v, dpp(v, integral_constant<int, kDppMirror>{}, integral_constant<int, 0xF>{}));
    v = max(v, dpp(v, integral_constant<int, kDppBcast15>{}, integral_constant<int, 0xA>{}));
    v = max(v, dpp(v, integral_constant<int, kDppBcast31>{}, integral_constant<int, 0xC>{}));
    v = (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; i++) v = max(v, red[i]);
    return __builtin_bit_cast(float, v);
}

// Rows of 16-bit values, whole 16-byte pieces: read once, 128 bits a load, and kept in registers; a workgroup of W waves a row, NCH pieces a
// thread.  Bound by memory (8192 x 4096 bf16 to 16 bits 46 us, to 8 bits 44: 5.8 TB/s and, the inputs partly in the caches, 6.9), few rows by
// one round trip (one row of 4096 2.3 us; in four waves 2.5).  A wave a row was slower everywhere (8192 x 4096 83 and 48 us, 300 x 2048 4.6 against 3.4).  All
// loads, the weights' too, are asked for first and without a test around them (pieces past the row repeat its last one and count as zero): the
// launch is one round trip to memory, a reduction (for 8 bits two) and the stores.  The sum's 32-bit values are packed to the storage type
// at once, which is what is stored, normalised and kept.
template <typename T, bool Q8, int NCH, int W>
__global__ __launch_bounds__(64 * W) void add_norm_vec_kernel(void *out_, const T *x, const T *residual, const T *w, T *sum, int dim, float eps, T *y_scale) {
    __shared__ float red[W];
    __shared__ uint32_t peak[W];
    const int lane = threadIdx.x, row = blockIdx.x;
    const size_t base = (size_t)row * dim;
    const int chunks = dim >> 3;
    U4 v[NCH], r[NCH], nw[NCH];
#pragma unroll
    for (int q = 0; q < NCH; q++) {
        const size_t c = base + (size_t)min(lane + q * 64 * W, chunks - 1) * 8;
        v[q] = *(const U4 *)(x + c);
        if (residual) r[q] = *(const U4 *)(residual + c);
    }
#pragma unroll
    for (int q = 0; q < NCH; q++) nw[q] = *(const U4 *)(w + (size_t)min(lane + q * 64 * W, chunks - 1) * 8);
    float ss = 0.f;
#pragma unroll
    for (int q = 0; q < NCH; q++) {
        const int c = lane + q * 64 * W;
        float f[8];
        widen8<T>(v[q], f);
        if (residual) {
            float g[8];
            widen8<T>(r[q], g);
            v[q] = U4{pack2<T>(f[0] + g[0], f[1] + g[1]), pack2<T>(f[2] + g[2], f[3] + g[3]), pack2<T>(f[4] + g[4], f[5] + g[5]), pack2<T>(f[6] + g[6], f[7] + g[7])};
        }
        if (c >= chunks) v[q] = U4{0u, 0u, 0u, 0u};
        else if (sum) *(U4 *)(sum + base + (size_t)c * 8) = v[q];
        widen8<T>(v[q], f);
#pragma unroll
        for (int i = 0; i < 8; i++) ss += f[i] * f[i];
    }
    ss = an_row_sum<W>(ss, red);
    float inv = 1.0f / sqrtf(ss / (float)dim + eps);
    if constexpr (std::is_same<T, bf16_t>::value) {  // (fp16 values have squares between)
        if (const float unit = an_unit(ss, dim, eps); unit != 0.f) {  // (all threads alike)
            auto times = [&](float by, bool keep) {
                float sum_ = 0.f;
#pragma unroll
                for (int q = 0; q < NCH; q++) {
                    float f[8];
                    widen8<T>(v[q], f);
#pragma unroll
                    for (int i = 0; i < 8; i++) sum_ += (f[i] *= by) * f[i];
                    if (keep) v[q] = U4{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7])};
                }
                return sum_;
            };
            __syncthreads();
            const AnRange range(unit, an_row_sum<W>(times(unit, false), red), dim, eps);
            times(range.first, true);  // (a power of two; of a large row, what has no bf16 number is nothing beside the rest)
            inv = range.inv;
        }
    }
    if constexpr (!Q8) {
#pragma unroll
        for (int q = 0; q < NCH; q++) {
            const int c = lane + q * 64 * W;
            float f[8], g[8];
            widen8<T>(v[q], f);
            widen8<T>(nw[q], g);
            const U4 o = U4{pack2<T>((f[0] * inv) * g[0], (f[1] * inv) * g[1]), pack2<T>((f[2] * inv) * g[2], (f[3] * inv) * g[3]),
                            pack2<T>((f[4] * inv) * g[4], (f[5] * inv) * g[5]), pack2<T>((f[6] * inv) * g[6], (f[7] * inv) * g[7])};
            if (c < chunks) *(U4 *)((T *)out_ + base + (size_t)c * 8) = o;
        }
    } else {
        // (the normalised values are made twice rather than kept: 16 registers a piece)
        uint32_t amax = 0;
#pragma unroll
        for (int q = 0; q < NCH; q++) {
            float f[8], g[8];
            widen8<T>(v[q], f);
            widen8<T>(nw[q], g);
#pragma unroll
            for (int i = 0; i < 8; i++) amax = max(amax, lane + q * 64 * W < chunks ? an_bits((f[i] * inv) * g[i]) : 0u);
        }
        const AnStep step(an_row_max<W>(amax, peak));
#pragma unroll
        for (int q = 0; q < NCH; q++) {
            const int c = lane + q * 64 * W;
            float f[8], g[8];
            widen8<T>(v[q], f);
            widen8<T>(nw[q], g);
            uint32_t b[2] = {0u, 0u};
#pragma unroll
            for (int i = 0; i < 8; i++) b[i >> 2] |= ((uint32_t)(int)step.code((f[i] * inv) * g[i]) & 0xFFu) << (8 * (i & 3));
            if (c < chunks) *(uint2 *)((int8_t *)out_ + base + (size_t)c * 8) = uint2{b[0], b[1]};
        }
        if (lane == 0) Elem<T>::st(y_scale, row, step.step);
    }
}

constexpr int kAnRows = 1 << 21;  // rows of a launch: with 1024 threads each it stays below the 2^32 that one may have

template <bool Q8>
static int add_norm(void *out, void *y_scale, void *sum, const void *x, const void *residual, const void *w, int rows, int dim, float eps, int dtype,
                    hipStream_t s) {
    if (rows > kAnRows) {
        const size_t bytes = dtype == MYNN_F32 ? 4 : 2, step = (size_t)kAnRows * dim;
        for (int r = 0; r < rows; r += std::min(kAnRows, rows - r)) {
            const size_t i = r / kAnRows;
            auto at = [&](const void *p) { return p ? (char *)p + i * step * bytes : nullptr; };
            if (const int rc = add_norm<Q8>((char *)out + i * step * (Q8 ? 1 : bytes), Q8 ? (char *)y_scale + i * kAnRows * bytes : nullptr, at(sum), at(x), at(residual),
                                            w, std::min(kAnRows, rows - r), dim, eps, dtype, s))
                return rc;
        }
        return 0;
    }
    return dispatch_dtype(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if constexpr (sizeof(T) == 2) {
            const bool whole = dim % 8 == 0 && aligned16(x) && aligned16(w) && (!residual || aligned16(residual)) && (!sum || aligned16(sum)) &&
                               ((uintptr_t)out & (Q8 ? 7 : 15)) == 0;
            auto go = [&](auto nch, auto w_) {
                constexpr int NCH = decltype(nch)::value, W = decltype(w_)::value;
                MYNN_LAUNCH((add_norm_vec_kernel<T, Q8, NCH, W>), dim3(rows), dim3(64 * W), 0, s, out, (const T *)x, (const T *)residual, (const T *)w,
                            (T *)sum, dim, eps, (T *)y_scale);
                return launch_status("add_norm_vec_kernel");
            };
            using std::integral_constant;
            const int chunks = dim / 8;
            if (whole) {
                if (chunks <= 256) return go(integral_constant<int, 1>{}, integral_constant<int, 4>{});
                if (chunks <= 512 && rows >= 256) return go(integral_constant<int, 2>{}, integral_constant<int, 4>{});
                if (chunks <= 512) return go(integral_constant<int, 1>{}, integral_constant<int, 8>{});
                if (chunks <= 1024) return go(integral_constant<int, 2>{}, integral_constant<int, 8>{});
                if (chunks <= 2048) return go(integral_constant<int, 2>{}, integral_constant<int, 16>{});
                if (chunks <= 4096) return go(integral_constant<int, 4>{}, integral_constant<int, 16>{});
            }
        }
        MYNN_LAUNCH((add_norm_kernel<T, Q8>), dim3(rows), dim3(kAnThreads), 0, s, out, (T *)y_scale, (T *)sum, (const T *)x, (const T *)residual,
                    (const T *)w, dim, eps);
        return launch_status("add_norm_kernel");
    });
}

}  // namespace mynn

using namespace mynn;

extern "C" int mynn_add_rms_norm(void *out, void *sum, const void *x, const void *residual, const void *w, int rows, int dim, float eps, int dtype,
                                 mynn_stream s) {
    MYNN_REQUIRE(out && x && w && rows > 0 && dim > 0, MYNN_ERR_INVALID, "add_rms_norm: bad operand (rows=%d dim=%d)", rows, dim);
    MYNN_REQUIRE(out != sum, MYNN_ERR_INVALID, "add_rms_norm: out and sum are the same memory");
    return add_norm<false>(out, nullptr, sum, x, residual, w, rows, dim, eps, dtype, as_stream(s));
}

extern "C" int mynn_add_rms_norm_quantize(int8_t *y, void *y_scale, void *sum, const void *x, const void *residual, const void *w, int rows, int dim,
                                          float eps, int dtype, mynn_stream s) {
    MYNN_REQUIRE(y && y_scale && x && w && rows > 0 && dim > 0, MYNN_ERR_INVALID, "add_rms_norm_quantize: bad operand (rows=%d dim=%d)", rows, dim);
    return add_norm<true>(y, y_scale, sum, x, residual, w, rows, dim, eps, dtype, as_stream(s));
}
