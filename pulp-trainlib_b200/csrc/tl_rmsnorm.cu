// RMS norm of a residual sum, forward (also with an output in 8 bits) and backward, and the 8-bit form of a tensor's rows.
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = w h r
//   q = rint(w h * 127 / max|w h|),  scale = r max|w h| / 127        (r > 0 leaves the rounding: it only scales the row)
//   dx = dsum + r (g - h r^2 mean(g h)),  g = w dy;   dw = sum over the rows of dy h r
// All of it is bound by its tensors' bytes: a row is read once into registers, by a warp or by a CTA, and everything that depends on it leaves
// from there.  Rows that no CTA's registers hold (above 32768 elements forward, 16384 backward) are read twice.
#include "tl_kernels.h"
#include "tl_reduce.cuh"

namespace tl {

enum { NORM_PLAIN = 0, NORM_INT8 = 1, QUANT_ROWS = 2 };

// ---------------------------------------------------------------- 8 bits
// What a value is multiplied by: 127 / m behind a power of two that keeps the quotient finite for rows of tiny values; a row of zeros gives zeros.
__device__ __forceinline__ float2 quant_factor(float m)
{
    const float up = m < 0x1p-100f ? 0x1p100f : 1.f;
    return make_float2(up, m > 0.f ? __fdiv_rn(127.f, m * up) : 0.f);
}
// v / (m / 127) to the nearest whole number.  The quotient in 32 bits is off by three roundings, 127 * 3 * 2^-24 at most; beside the border of two steps
// (one value in ten thousand, and every exact tie) 64 bits decide.
__device__ __forceinline__ int quant(float v, float2 f, float m)
{
    float t = v * f.x;
    t *= f.y;
    float n = rintf(t);
    if (fabsf(fabsf(t - n) - 0.5f) < 3e-5f) n = (float)rint((double)v / ((double)m / 127.0));
    return __float2int_rn(fminf(fmaxf(n == n ? n : 0.f, -127.f), 127.f));
}
// a row's scale from r, its largest magnitude and a sum that is finite if all of it is
__device__ __forceinline__ float quant_scale(float r, float m, float sum) { return sum - sum == 0.f ? r * __fdiv_rn(m, 127.f) : sum * 0.f; }

// ---------------------------------------------------------------- V neighbouring elements
template <class T, int V> struct alignas(sizeof(T) * V) Pack { T e[V]; };
template <class T, int V> __device__ __forceinline__ Pack<T, V> ldv(const T *p) { return *reinterpret_cast<const Pack<T, V> *>(p); }
template <class T, int V> __device__ __forceinline__ void stv(T *p, const Pack<T, V> &v) { *reinterpret_cast<Pack<T, V> *>(p) = v; }
__device__ __forceinline__ float tof(float v) { return v; }
__device__ __forceinline__ float tof(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T fromf(float v) { if constexpr (sizeof(T) == 2) return __float2half_rn(v); else return v; }
template <class T, int V> __device__ __forceinline__ Pack<T, V> zerov()
{
    Pack<T, V> z;
#pragma unroll
    for (int i = 0; i < V; i++) z.e[i] = fromf<T>(0.f);
    return z;
}

// Two values over the G threads of a row (sum and sum, or sum and maximum), the same for all of them.  Every thread of the block takes part.
template <int G, bool MAX> __device__ __forceinline__ float2 row_reduce(float a, float b, float2 *red)
{
    a = warp_sum(a);
    b = MAX ? warp_max(b) : warp_sum(b);
    if constexpr (G == 32) return make_float2(a, b);
    const int lane = threadIdx.x & 31, w0 = threadIdx.x / G * (G / 32);
    if (lane == 0) red[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    const float2 v = lane < G / 32 ? red[w0 + lane] : make_float2(0.f, 0.f);
    return make_float2(warp_sum(v.x), MAX ? warp_max(v.y) : warp_sum(v.y));
}

// ---------------------------------------------------------------- forward
// G threads per row, a block's rows side by side, NV packs of V elements per thread.
template <class T, int MODE, int G, int NV, int V>
__global__ void __launch_bounds__(G < 256 ? 256 : G) rmsnorm_fw_kernel(const T *x, const T *res, const T *__restrict__ w, T *sum, T *y, signed char *__restrict__ q,
                                                                       float *__restrict__ scale, int rows, int size, float eps)
{
    pdl_wait();
    constexpr int TPB = G < 256 ? 256 : G;
    __shared__ float2 red[TPB / 32];
    const int row = blockIdx.x * (TPB / G) + threadIdx.x / G, t = threadIdx.x % G;
    const size_t at = (size_t)row * size;
    Pack<T, V> a[NV], b[NV], wv[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = (k * G + t) * V;
        const bool in = row < rows && j < size;
        a[k] = b[k] = wv[k] = zerov<T, V>();
        if (in) a[k] = ldv<T, V>(x + at + j);
        if (in && res) b[k] = ldv<T, V>(res + at + j);
        if (MODE != QUANT_ROWS && in) wv[k] = ldv<T, V>(w + j);
    }
    float s = 0.f, m = 0.f, h[NV][V];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            h[k][i] = tof(a[k].e[i]) + tof(b[k].e[i]);
            s = MODE == QUANT_ROWS ? fmaf(h[k][i], 0.f, s) : fmaf(h[k][i], h[k][i], s);                  // (quantised alone, the sum tells only whether every value is finite)
            if (MODE != NORM_PLAIN) m = fmaxf(m, fabsf(MODE == NORM_INT8 ? h[k][i] * tof(wv[k].e[i]) : h[k][i]));       // (passes over NaN: the scale carries it)
        }
    const float2 tot = row_reduce<G, true>(s, m, red);
    if (row >= rows) return;
    const float r = MODE == QUANT_ROWS ? 1.f : 1.f / sqrtf(tot.x / (float)size + eps);
    const float2 f = MODE == NORM_PLAIN ? make_float2(0.f, 0.f) : quant_factor(tot.y);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = (k * G + t) * V;
        if (j >= size) continue;
        if (MODE != QUANT_ROWS && sum) {
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; i++) o.e[i] = fromf<T>(h[k][i]);
            stv<T, V>(sum + at + j, o);
        }
        if constexpr (MODE == NORM_PLAIN) {
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; i++) o.e[i] = fromf<T>(h[k][i] * r * tof(wv[k].e[i]));
            stv<T, V>(y + at + j, o);
        } else {
            Pack<signed char, V> o;
#pragma unroll
            for (int i = 0; i < V; i++) o.e[i] = (signed char)quant(MODE == NORM_INT8 ? h[k][i] * tof(wv[k].e[i]) : h[k][i], f, tot.y);
            stv<signed char, V>(q + at + j, o);
        }
    }
    if (MODE != NORM_PLAIN && t == 0) scale[row] = quant_scale(r, tot.y, tot.x);
}
// A CTA per row, any width: a pass for the row's sum of squares and largest magnitude, a second one for the results.
template <class T, int MODE>
__global__ void __launch_bounds__(1024) rmsnorm_fw_wide_kernel(const T *x, const T *res, const T *__restrict__ w, T *sum, T *y, signed char *__restrict__ q,
                                                               float *__restrict__ scale, int size, float eps)
{
    pdl_wait();
    __shared__ float2 red[32];
    const size_t at = (size_t)blockIdx.x * size;
    float s = 0.f, m = 0.f;
#pragma unroll 4
    for (int j = threadIdx.x; j < size; j += 1024) {
        const float h = ld(x + at + j) + (res ? ld(res + at + j) : 0.f);
        s = MODE == QUANT_ROWS ? fmaf(h, 0.f, s) : fmaf(h, h, s);
        if (MODE != NORM_PLAIN) m = fmaxf(m, fabsf(MODE == NORM_INT8 ? h * ld(w + j) : h));
    }
    const float2 tot = row_reduce<1024, true>(s, m, red);
    const float r = MODE == QUANT_ROWS ? 1.f : 1.f / sqrtf(tot.x / (float)size + eps);
    const float2 f = quant_factor(tot.y);
    for (int j = threadIdx.x; j < size; j += 1024) {
        const float h = ld(x + at + j) + (res ? ld(res + at + j) : 0.f);
        if (MODE != QUANT_ROWS && sum) st(sum + at + j, h);
        if (MODE == NORM_PLAIN) st(y + at + j, h * r * ld(w + j));
        else q[at + j] = (signed char)quant(MODE == NORM_INT8 ? h * ld(w + j) : h, f, tot.y);
    }
    if (MODE != NORM_PLAIN && threadIdx.x == 0) scale[blockIdx.x] = quant_scale(r, tot.y, tot.x);
}

template <class T, int MODE>
static void norm_forward(const T *x, const T *res, const T *w, T *sum, T *y, signed char *q, float *scale, int rows, int size, float eps)
{
    constexpr int V16 = 16 / (int)sizeof(T);
    // packs of 16 bytes where every row of every tensor starts on such a boundary (the 8-bit one on V16 bytes)
    const uintptr_t at = (uintptr_t)x | (uintptr_t)res | (uintptr_t)w | (uintptr_t)sum | (uintptr_t)y;
    const bool wide = size % V16 == 0 && at % 16 == 0 && (uintptr_t)q % V16 == 0;
    const int packs = wide ? size / V16 : size;
#define TL_NORM(G, NV, V) TL_LAUNCH((rmsnorm_fw_kernel<T, MODE, G, NV, V>), ceil_div(rows, (G < 256 ? 256 : G) / G), G < 256 ? 256 : G, 0, x, res, w, sum, y, q, scale, rows, size, eps)
#define TL_NORM_V(V)                                                                                  \
    do {                                                                                              \
        if (packs <= 32) TL_NORM(32, 1, V);                                                           \
        else if (packs <= 64) TL_NORM(32, 2, V);                                                      \
        else if (packs <= 128 && rows > 4 * sm_count()) TL_NORM(32, 4, V);                            \
        else if (packs <= 256) TL_NORM(128, 2, V);                                                    \
        else if (packs <= 512) TL_NORM(256, 2, V);                                                    \
        else if (packs <= 1024) TL_NORM(512, 2, V);                                                   \
        else if (packs <= 2048) TL_NORM(1024, 2, V);                                                  \
        else TL_NORM(1024, 4, V);                                                                     \
    } while (0)
    if (packs > 4096) TL_LAUNCH((rmsnorm_fw_wide_kernel<T, MODE>), rows, 1024, 0, x, res, w, sum, y, q, scale, size, eps);
    else if (wide) TL_NORM_V(V16);
    else TL_NORM_V(1);
#undef TL_NORM_V
#undef TL_NORM
}
template <class T> void rmsnorm_fw(const T *x, const T *res, const T *w, T *sum, T *y, int rows, int size, float eps)
{
    norm_forward<T, NORM_PLAIN>(x, res, w, sum, y, nullptr, nullptr, rows, size, eps);
}
template <class T> void rmsnorm_int8_fw(const T *x, const T *res, const T *w, T *sum, signed char *q, float *scale, int rows, int size, float eps)
{
    norm_forward<T, NORM_INT8>(x, res, w, sum, nullptr, q, scale, rows, size, eps);
}
template <class T> void quantize_rows(const T *x, signed char *q, float *scale, int rows, int size)
{
    norm_forward<T, QUANT_ROWS>(x, nullptr, nullptr, nullptr, nullptr, q, scale, rows, size, 0.f);
}

// ---------------------------------------------------------------- backward
// A block walks rows, G threads per row and TPB / G rows at a time; a thread keeps its columns' sums of dy h r in registers from row to row, so that dx and
// dw come from one read.  The rows of a block meet in shared memory at the end, in order, and leave one partial sum per block.
static constexpr int NB_TPB = 512;
template <class T, int G, int NV, int V, bool PRE>
__global__ void __launch_bounds__(G < NB_TPB ? NB_TPB : G) rmsnorm_bw_kernel(const T *h, const T *__restrict__ w, const T *dy, const T *dsum, T *dx, float *__restrict__ part,
                                                                            int rows, int size, float eps)
{
    pdl_wait();
    constexpr int TPB = G < NB_TPB ? NB_TPB : G, RG = TPB / G;
    __shared__ float2 red[2][TPB / 32];
    extern __shared__ float cols[];                      // [size], where RG > 1
    const int t = threadIdx.x % G, mine = threadIdx.x / G;
    Pack<T, V> hv[NV], gv[NV];
    float acc[NV][V];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < V; i++) acc[k][i] = 0.f;
    auto weight = [&](int k) { const int j = (k * G + t) * V; return j < size ? ldv<T, V>(w + j) : zerov<T, V>(); };       // (from L1: registers go to the rows)
    auto fetch = [&](int row) {
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int j = (k * G + t) * V;
            const bool in = row < rows && j < size;
            hv[k] = gv[k] = zerov<T, V>();
            if (in) { hv[k] = ldv<T, V>(h + (size_t)row * size + j); gv[k] = ldv<T, V>(dy + (size_t)row * size + j); }
        }
    };
    int turn = 0;
    if (PRE) fetch(blockIdx.x * RG + mine);
    for (int base = blockIdx.x * RG; base < rows; base += gridDim.x * RG, turn ^= 1) {
        const int row = base + mine;
        const size_t at = (size_t)row * size;
        Pack<T, V> dv[NV], hc[NV], gc[NV];
        auto residual = [&]() {
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int j = (k * G + t) * V;
                dv[k] = zerov<T, V>();
                if (dx && dsum && row < rows && j < size) dv[k] = ldv<T, V>(dsum + at + j);
            }
        };
        if (PRE) residual(); else fetch(row);
#pragma unroll
        for (int k = 0; k < NV; k++) { hc[k] = hv[k]; gc[k] = gv[k]; }
        float s = 0.f, c = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const Pack<T, V> wk = weight(k);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float v = tof(hc[k].e[i]);
                s = fmaf(v, v, s);
                c = fmaf(v, tof(gc[k].e[i]) * tof(wk.e[i]), c);
            }
        }
        if (PRE) fetch(row + (int)gridDim.x * RG);       // under way while the row's sums meet (dx may be one of the inputs: of this row, which is in registers)
        const float2 tot = row_reduce<G, false>(s, c, red[turn]);
        if (!PRE) residual();
        const float r = 1.f / sqrtf(tot.x / (float)size + eps), cr = tot.y / (float)size * r * r;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int j = (k * G + t) * V;
            const Pack<T, V> wk = weight(k);
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float v = tof(hc[k].e[i]), g = tof(gc[k].e[i]);
                if (row < rows) acc[k][i] = fmaf(g * v, r, acc[k][i]);
                o.e[i] = fromf<T>(tof(dv[k].e[i]) + r * (g * tof(wk.e[i]) - v * cr));
            }
            if (dx && row < rows && j < size) stv<T, V>(dx + at + j, o);
        }
    }
    if (!part) return;
    float *out = part + (size_t)blockIdx.x * size;
    if constexpr (RG == 1) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < V; i++) { const int j = (k * G + t) * V + i; if (j < size) out[j] = acc[k][i]; }
    } else {
        for (int g = 0; g < RG; g++) {
            __syncthreads();
            if (mine != g) continue;
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int i = 0; i < V; i++) { const int j = (k * G + t) * V + i; if (j < size) cols[j] = g ? cols[j] + acc[k][i] : acc[k][i]; }
        }
        __syncthreads();
        for (int j = threadIdx.x; j < size; j += TPB) out[j] = cols[j];
    }
}
// dw from the blocks' partial sums: 32 columns by 32 slices of the blocks, each slice in order, the slices in order
template <class T> __global__ void __launch_bounds__(1024) rmsnorm_bw_sum_kernel(const float *__restrict__ part, T *__restrict__ dw, int size, int blocks)
{
    pdl_wait();
    __shared__ float sm[32][33];
    const int c = threadIdx.x & 31, sl = threadIdx.x >> 5, j = blockIdx.x * 32 + c;
    float t = 0.f;
    if (j < size)
#pragma unroll 4
        for (int b = sl; b < blocks; b += 32) t += part[(size_t)b * size + j];
    sm[sl][c] = t;
    __syncthreads();
    if (sl > 0 || j >= size) return;
#pragma unroll
    for (int k = 1; k < 32; k++) t += sm[k][c];
    st(dw + j, t);
}
// Wider rows: r and r^2 mean(g h) of each row, then the columns, then dx
template <class T>
__global__ void __launch_bounds__(1024) rmsnorm_bw_stats_kernel(const T *__restrict__ h, const T *__restrict__ w, const T *__restrict__ dy, float2 *__restrict__ stats, int size, float eps)
{
    pdl_wait();
    __shared__ float2 red[32];
    const size_t at = (size_t)blockIdx.x * size;
    float s = 0.f, c = 0.f;
#pragma unroll 4
    for (int j = threadIdx.x; j < size; j += 1024) {
        const float v = ld(h + at + j);
        s = fmaf(v, v, s);
        c = fmaf(v, ld(dy + at + j) * ld(w + j), c);
    }
    const float2 tot = row_reduce<1024, false>(s, c, red);
    const float r = 1.f / sqrtf(tot.x / (float)size + eps);
    if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(r, tot.y / (float)size * r * r);
}
template <class T>
__global__ void __launch_bounds__(128) rmsnorm_bw_cols_kernel(const T *__restrict__ h, const T *__restrict__ dy, const float2 *__restrict__ stats, float *__restrict__ part,
                                                              int rows, int size, int rows_per)
{
    pdl_wait();
    const int j = blockIdx.x * 128 + threadIdx.x, r0 = blockIdx.y * rows_per, r1 = min(rows, r0 + rows_per);
    if (j >= size) return;
    float t = 0.f;
#pragma unroll 4
    for (int r = r0; r < r1; r++) t = fmaf(ld(dy + (size_t)r * size + j) * ld(h + (size_t)r * size + j), stats[r].x, t);
    part[(size_t)blockIdx.y * size + j] = t;
}
template <class T>
__global__ void __launch_bounds__(1024) rmsnorm_bw_dx_kernel(const T *h, const T *__restrict__ w, const T *dy, const T *dsum, T *dx, const float2 *__restrict__ stats, int size)
{
    pdl_wait();
    const size_t at = (size_t)blockIdx.x * size;
    const float2 t = stats[blockIdx.x];
    for (int j = threadIdx.x; j < size; j += 1024) {
        const float g = ld(dy + at + j) * ld(w + j), v = ld(h + at + j);
        st(dx + at + j, (dsum ? ld(dsum + at + j) : 0.f) + t.x * (g - v * t.y));
    }
}
template <class T> static void norm_columns(const float *part, T *dw, int size, int blocks) { TL_LAUNCH((rmsnorm_bw_sum_kernel<T>), ceil_div(size, 32), 1024, 0, part, dw, size, blocks); }

template <class T> void rmsnorm_bw(Scope &sc, const T *h, const T *w, const T *dy, const T *dsum, T *dx, T *dw, int rows, int size, float eps)
{
    // elements per thread: their columns' sums and those of two rows (of one, in blocks of 1024 threads) fit its registers
    constexpr int V16 = 16 / (int)sizeof(T), MOST = 16 * 1024;
    const uintptr_t at = (uintptr_t)h | (uintptr_t)w | (uintptr_t)dy | (uintptr_t)dsum | (uintptr_t)dx;
    const bool wide = size % V16 == 0 && at % 16 == 0;
    if (size > MOST) {
        const int rows_per = std::max(16, ceil_div(rows, 64)), groups = ceil_div(rows, rows_per);
        float2 *stats = sc.scratch<float2>((size_t)rows);
        float *part = dw ? sc.scratch<float>((size_t)groups * size) : nullptr;
        if (!stats || (dw && !part)) return;
        TL_LAUNCH((rmsnorm_bw_stats_kernel<T>), rows, 1024, 0, h, w, dy, stats, size, eps);
        if (dw) {
            TL_LAUNCH((rmsnorm_bw_cols_kernel<T>), dim3(ceil_div(size, 128), groups), 128, 0, h, dy, stats, part, rows, size, rows_per);
            norm_columns<T>(part, dw, size, groups);
        }
        if (dx) TL_LAUNCH((rmsnorm_bw_dx_kernel<T>), rows, 1024, 0, h, w, dy, dsum, dx, stats, size);
        return;
    }
#define TL_NORM_BW(G, NV, V, PRE)                                                                                                                             \
    do {                                                                                                                                                      \
        constexpr int TPB = G < NB_TPB ? NB_TPB : G, RG = TPB / G;                                                                                            \
        const int blocks = std::min(ceil_div(rows, RG), (TPB == 1024 ? 1 : 2) * sm_count());                                                                  \
        float *part = dw ? sc.scratch<float>((size_t)blocks * size) : nullptr;                                                                                \
        if (dw && !part) return;                                                                                                                              \
        TL_LAUNCH((rmsnorm_bw_kernel<T, G, NV, V, PRE>), blocks, TPB, RG > 1 ? size * sizeof(float) : 0, h, w, dy, dsum, dx, part, rows, size, eps);          \
        if (dw) norm_columns<T>(part, dw, size, blocks);                                                                                                      \
    } while (0)
#define TL_NORM_BW_V(V, E)                                                     \
    do {                                                                       \
        if (size <= 32 * V) TL_NORM_BW(32, 1, V, true);                        \
        else if (size <= 32 * E) TL_NORM_BW(32, E / V, V, true);               \
        else if (size <= 128 * E) TL_NORM_BW(128, E / V, V, true);             \
        else if (size <= 256 * E) TL_NORM_BW(256, E / V, V, true);             \
        else if (size <= 512 * E) TL_NORM_BW(512, E / V, V, true);             \
        else if (size <= 1024 * 8) TL_NORM_BW(1024, 8 / V, V, false);          \
        else TL_NORM_BW(1024, 16 / V, V, false);                               \
    } while (0)
    if (wide) TL_NORM_BW_V(V16, 2 * V16);
    else TL_NORM_BW_V(1, 8);
#undef TL_NORM_BW_V
#undef TL_NORM_BW
}

#define INST(T)                                                                                                    \
    template void rmsnorm_fw<T>(const T *, const T *, const T *, T *, T *, int, int, float);                       \
    template void rmsnorm_int8_fw<T>(const T *, const T *, const T *, T *, signed char *, float *, int, int, float); \
    template void quantize_rows<T>(const T *, signed char *, float *, int, int);                                   \
    template void rmsnorm_bw<T>(Scope &, const T *, const T *, const T *, const T *, T *, T *, int, int, float);
INST(float)
INST(__half)

} // namespace tl
