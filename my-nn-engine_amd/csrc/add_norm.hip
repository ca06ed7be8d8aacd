// The residual's addition with the RMSNorm behind it: sum = T(x + residual) is stored and normalised in one pass over the row,
//   y = sum * 1/sqrt(mean(sum^2) + eps) * w,
// to the storage type or, per row, to 8 bits: step = max|y| / 127 (1 for a row of zeros), code = y / step rounded half away from zero.
// Statistics and y are held in 32 bits; y goes to 8 bits without a rounding to T in between.  A row whose y is not all finite
// gets the step NaN and codes of zero, so that a product of it is NaN and not some number.
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
// A row's step and what its values are multiplied by.  Below 2^-120 (no bf16 or fp16 scale says it) a row counts as zeros: 127 / amax
// would overflow.
struct AnStep {
    float step, per;
    __device__ explicit AnStep(float amax) {
        const bool finite = amax < INFINITY, some = amax >= 0x1p-120f;
        step = !finite ? NAN : some ? amax / 127.0f : 1.0f;
        per = finite && some ? 1.0f / step : 0.f;
    }
    __device__ float code(float y) const {
        const float q = fminf(fmaxf(roundf(y * per), -127.f), 127.f);  // half away from zero
        return per == 0.f ? 0.f : q;
    }
};

// Rows of any length, at any address, of any type: a workgroup per row, an element a thread and step.  What a thread wrote of `sum`
// it reads again itself, so `sum` may be x or the residual, and so may `out` where no sum is asked for.
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
    const float inv = 1.0f / sqrtf(an_sum(ss, red) / (float)dim + eps);
    if constexpr (!Q8) {
        for (int i = threadIdx.x; i < dim; i += kAnThreads) Elem<T>::st((T *)out_, base + i, (again(i) * inv) * Elem<T>::ld(w, i));
    } else {
        __shared__ uint32_t peak[4];
        uint32_t amax = 0;
        for (int i = threadIdx.x; i < dim; i += kAnThreads) amax = max(amax, an_bits((again(i) * inv) * Elem<T>::ld(w, i)));
        const AnStep step(an_max(amax, peak));
        for (int i = threadIdx.x; i < dim; i += kAnThreads) ((int8_t *)out_)[base + i] = (int8_t)step.code((again(i) * inv) * Elem<T>::ld(w, i));
        if (threadIdx.x == 0) Elem<T>::st(y_scale, blockIdx.x, step.step);
    }
}

template <bool Q8>
static int add_norm(void *out, void *y_scale, void *sum, const void *x, const void *residual, const void *w, int rows, int dim, float eps, int dtype,
                    hipStream_t s) {
    return dispatch_dtype(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
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
