// RMS norm of a residual sum, forward (also with an output in 8 bits) and backward, and the 8-bit form of a tensor's rows.
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = w h r
//   q = rint(w h * 127 / max|w h|),  scale = r max|w h| / 127        (r > 0 leaves the rounding: it only scales the row)
//   dx = dsum + r (g - h r^2 mean(g h)),  g = w dy;   dw = sum over the rows of dy h r
#include "tl_kernels.h"
#include "tl_reduce.cuh"

namespace tl {

enum { NORM_PLAIN = 0, NORM_INT8 = 1, QUANT_ROWS = 2 };

// maximum of magnitudes over the CTA (fmaxf passes over NaN: the row's scale carries it)
__device__ __forceinline__ float2 block_sum_max(float s, float m, float *red)
{
    s = block_sum(s, red);
    m = block_max(m, red);
    return make_float2(s, m);
}
// 127 / m and what a value is multiplied by first, so that the quotient stays finite for rows of tiny values; a row of zeros gives zeros
__device__ __forceinline__ float2 quant_factor(float m)
{
    const float up = m < 0x1p-100f ? 0x1p100f : 1.f;
    return make_float2(up, m > 0.f ? __fdiv_rn(127.f, m * up) : 0.f);
}
__device__ __forceinline__ signed char quant(float v, float2 f)
{
    v *= f.x;
    v *= f.y;
    return (signed char)__float2int_rn(fminf(fmaxf(v == v ? v : 0.f, -127.f), 127.f));
}

// A CTA per row, any width and alignment: one pass for the row's sum of squares and largest magnitude, a second one for the results.
template <class T, int MODE>
__global__ void __launch_bounds__(256) rmsnorm_fw_kernel(const T *x, const T *res, const T *__restrict__ w, T *sum, T *y, signed char *__restrict__ q,
                                                         float *__restrict__ scale, int size, float eps)
{
    pdl_wait();
    __shared__ float red[33];
    const size_t at = (size_t)blockIdx.x * size;
    float s = 0.f, m = 0.f;
    for (int j = threadIdx.x; j < size; j += 256) {
        const float h = ld(x + at + j) + (res ? ld(res + at + j) : 0.f);
        s = MODE == QUANT_ROWS ? fmaf(h, 0.f, s) : fmaf(h, h, s);             // (quantised alone, the sum tells only whether every value is finite)
        if (MODE != NORM_PLAIN) m = fmaxf(m, fabsf(MODE == NORM_INT8 ? h * ld(w + j) : h));
    }
    const float2 t = block_sum_max(s, m, red);
    const float r = MODE == QUANT_ROWS ? 1.f : 1.f / sqrtf(t.x / (float)size + eps);
    const float2 f = quant_factor(t.y);
    for (int j = threadIdx.x; j < size; j += 256) {
        const float h = ld(x + at + j) + (res ? ld(res + at + j) : 0.f);
        if (MODE != QUANT_ROWS && sum) st(sum + at + j, h);
        if (MODE == NORM_PLAIN) st(y + at + j, h * r * ld(w + j));
        else q[at + j] = quant(MODE == NORM_INT8 ? h * ld(w + j) : h, f);
    }
    if (MODE != NORM_PLAIN && threadIdx.x == 0) scale[blockIdx.x] = t.x - t.x == 0.f ? r * (t.y / 127.f) : t.x * 0.f;
}

// backward: the row's r and r^3 mean(g h)
template <class T>
__global__ void __launch_bounds__(256) rmsnorm_bw_stats_kernel(const T *__restrict__ h, const T *__restrict__ w, const T *__restrict__ dy, float2 *__restrict__ stats, int size, float eps)
{
    pdl_wait();
    __shared__ float red[33];
    const size_t at = (size_t)blockIdx.x * size;
    float s = 0.f, c = 0.f;
    for (int j = threadIdx.x; j < size; j += 256) {
        const float v = ld(h + at + j);
        s = fmaf(v, v, s);
        c = fmaf(v, ld(dy + at + j) * ld(w + j), c);
    }
    s = block_sum(s, red);
    c = block_sum(c, red);
    const float r = 1.f / sqrtf(s / (float)size + eps);
    if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(r, c / (float)size * r * r);
}
// column sums of dy h r over a group of rows
template <class T>
__global__ void __launch_bounds__(128) rmsnorm_bw_cols_kernel(const T *__restrict__ h, const T *__restrict__ dy, const float2 *__restrict__ stats, float *__restrict__ part,
                                                              int rows, int size, int rows_per)
{
    pdl_wait();
    const int j = blockIdx.x * 128 + threadIdx.x, r0 = blockIdx.y * rows_per, r1 = min(rows, r0 + rows_per);
    if (j >= size) return;
    float t = 0.f;
    for (int r = r0; r < r1; r++) t = fmaf(ld(dy + (size_t)r * size + j) * ld(h + (size_t)r * size + j), stats[r].x, t);
    part[(size_t)blockIdx.y * size + j] = t;
}
template <class T> __global__ void __launch_bounds__(128) rmsnorm_bw_cols_sum_kernel(const float *__restrict__ part, T *__restrict__ dw, int size, int groups)
{
    pdl_wait();
    const int j = blockIdx.x * 128 + threadIdx.x;
    if (j >= size) return;
    float t = 0.f;
    for (int g = 0; g < groups; g++) t += part[(size_t)g * size + j];
    st(dw + j, t);
}
template <class T>
__global__ void __launch_bounds__(256) rmsnorm_bw_dx_kernel(const T *h, const T *__restrict__ w, const T *dy, const T *dsum, T *dx, const float2 *__restrict__ stats, int size)
{
    pdl_wait();
    const size_t at = (size_t)blockIdx.x * size;
    const float2 t = stats[blockIdx.x];
    for (int j = threadIdx.x; j < size; j += 256) {
        const float g = ld(dy + at + j) * ld(w + j), v = ld(h + at + j);
        st(dx + at + j, (dsum ? ld(dsum + at + j) : 0.f) + t.x * (g - v * t.y));
    }
}

template <class T> void rmsnorm_fw(const T *x, const T *res, const T *w, T *sum, T *y, int rows, int size, float eps)
{
    TL_LAUNCH((rmsnorm_fw_kernel<T, NORM_PLAIN>), rows, 256, 0, x, res, w, sum, y, (signed char *)nullptr, (float *)nullptr, size, eps);
}
template <class T> void rmsnorm_int8_fw(const T *x, const T *res, const T *w, T *sum, signed char *q, float *scale, int rows, int size, float eps)
{
    TL_LAUNCH((rmsnorm_fw_kernel<T, NORM_INT8>), rows, 256, 0, x, res, w, sum, (T *)nullptr, q, scale, size, eps);
}
template <class T> void quantize_rows(const T *x, signed char *q, float *scale, int rows, int size)
{
    TL_LAUNCH((rmsnorm_fw_kernel<T, QUANT_ROWS>), rows, 256, 0, x, (const T *)nullptr, (const T *)nullptr, (T *)nullptr, (T *)nullptr, q, scale, size, 0.f);
}
template <class T> void rmsnorm_bw(Scope &sc, const T *h, const T *w, const T *dy, const T *dsum, T *dx, T *dw, int rows, int size, float eps)
{
    const int rows_per = std::max(16, ceil_div(rows, 64)), groups = ceil_div(rows, rows_per);
    float2 *stats = sc.scratch<float2>((size_t)rows);
    float *part = dw ? sc.scratch<float>((size_t)groups * size) : nullptr;
    if (!stats || (dw && !part)) return;
    TL_LAUNCH((rmsnorm_bw_stats_kernel<T>), rows, 256, 0, h, w, dy, stats, size, eps);
    if (dw) {
        TL_LAUNCH((rmsnorm_bw_cols_kernel<T>), dim3(ceil_div(size, 128), groups), 128, 0, h, dy, stats, part, rows, size, rows_per);
        TL_LAUNCH((rmsnorm_bw_cols_sum_kernel<T>), ceil_div(size, 128), 128, 0, part, dw, size, groups);
    }
    if (dx) TL_LAUNCH((rmsnorm_bw_dx_kernel<T>), rows, 256, 0, h, w, dy, dsum, dx, stats, size);
}

#define INST(T)                                                                                                    \
    template void rmsnorm_fw<T>(const T *, const T *, const T *, T *, T *, int, int, float);                       \
    template void rmsnorm_int8_fw<T>(const T *, const T *, const T *, T *, signed char *, float *, int, int, float); \
    template void quantize_rows<T>(const T *, signed char *, float *, int, int);                                   \
    template void rmsnorm_bw<T>(Scope &, const T *, const T *, const T *, const T *, T *, T *, int, int, float);
INST(float)
INST(__half)

} // namespace tl
