// Linear layer in 8-bit integers: y[r][o] = xs[r] ws[o] sum_i x[r][i] w[o][i] (+ b[o]).  The sums are exact in 32 bits (|product| <= 2^14, in <= 131071).
#include "tl_kernels.h"

namespace tl {

// 64 x 64 tiles on CUDA cores, any width and alignment
template <class T>
__global__ void __launch_bounds__(256) linear_int8_kernel(const signed char *__restrict__ x, const float *__restrict__ xs, const signed char *__restrict__ w,
                                                          const float *__restrict__ ws, const T *__restrict__ bias, T *__restrict__ y, int rows, int in, int out)
{
    pdl_wait();
    __shared__ signed char As[64][36], Bs[64][36];
    const int row0 = blockIdx.y * 64, col0 = blockIdx.x * 64, tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < in; k0 += 32) {
        for (int e = threadIdx.x; e < 2048; e += 256) {
            const int i = e / 32, k = e % 32;
            As[i][k] = row0 + i < rows && k0 + k < in ? x[(size_t)(row0 + i) * in + k0 + k] : 0;
            Bs[i][k] = col0 + i < out && k0 + k < in ? w[(size_t)(col0 + i) * in + k0 + k] : 0;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
            int a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) { a[i] = *reinterpret_cast<const int *>(&As[tr + 16 * i][k]); b[i] = *reinterpret_cast<const int *>(&Bs[tc + 16 * i][k]); }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = row0 + tr + 16 * i, col = col0 + tc + 16 * j;
            if (row < rows && col < out) st(y + (size_t)row * out + col, (float)acc[i][j] * xs[row] * ws[col] + (bias ? ld(bias + col) : 0.f));
        }
}
template <class T> void linear_int8(Scope &, const signed char *x, const float *xs, const signed char *w, const float *ws, const T *bias, T *y, int rows, int in, int out)
{
    TL_LAUNCH((linear_int8_kernel<T>), dim3(ceil_div(out, 64), ceil_div(rows, 64)), 256, 0, x, xs, w, ws, bias, y, rows, in, out);
}
template void linear_int8<float>(Scope &, const signed char *, const float *, const signed char *, const float *, const float *, float *, int, int, int);
template void linear_int8<__half>(Scope &, const signed char *, const float *, const signed char *, const float *, const __half *, __half *, int, int, int);

} // namespace tl
