// RMS norm of a residual sum, forward (also with an output in 8 bits) and backward, and the 8-bit form of a tensor's rows.
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = w h r
//   q = rint(w h * 127 / max|w h|),  scale = r max|w h| / 127        (r > 0 leaves the rounding: it only scales the row)
//   dx = dsum + r (g - h r^2 mean(g h)),  g = w dy;   dw = sum over the rows of dy h r
// All of it is bound by its tensors' bytes: a row is read once into registers, by a warp or by a CTA, and everything that depends on it leaves
// from there.  Rows that no CTA's registers hold are read twice: forward above 4096 packs of 16 bytes (32768 halves, 16384 floats; of rows that do not start
// on 16 bytes, 4096 single elements or pairs of halves), backward above 16384 elements.
#include "tl_kernels.h"
#include "tl_reduce.cuh"
#include "tl_tc.cuh"

namespace tl {

int *tc_status_word();          // tl_conv_tc.cu

enum { NORM_PLAIN = 0, NORM_INT8 = 1, QUANT_ROWS = 2 };

// ---------------------------------------------------------------- 8 bits
// What a value is multiplied by: 127 / m behind a power of two that keeps the quotient finite for rows of tiny values; a row of zeros gives zeros.
__device__ __forceinline__ float2 quant_factor(float m)
{
    const float up = m < 0x1p-100f ? 0x1p100f : 1.f;
    return make_float2(up, m > 0.f ? __fdiv_rn(127.f, m * up) : 0.f);
}
// v / (m / 127) to the nearest whole number, V values at a time into bytes.  Adding 1.5 * 2^23 leaves the nearest whole number (ties to even) in the low bits.
// The quotient in 32 bits is off by three roundings, 127 * 3 * 2^-24 at most: where one of the values lies that near the border of two steps (a few
// in a hundred thousand, and every exact tie), and in rows that are not finite, 64 bits decide: 127 v is exact there (31 bits), so the one rounding of the
// quotient leaves a tie a tie.  (A rounded m / 127 as the divisor put half of a row's largest magnitude, 63.5 steps, at 63 for an eighth of all m.)
__device__ __noinline__ int quant_exact(float v, float m)
{
    const double n = rint((double)v * 127.0 / (double)m);
    return m > 0.f && n == n ? (int)fmin(fmax(n, -127.0), 127.0) : 0;
}
template <int V> __device__ __forceinline__ void quant(const float (&v)[V], float2 f, float m, bool finite, signed char (&q)[V])
{
    float off = 0.f;
    uint32_t u[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float t = v[i] * f.x * f.y, s = __fadd_rn(t, 12582912.f), d = fabsf(__fsub_rn(t, __fsub_rn(s, 12582912.f)));
        off = fmaxf(off, d);
        u[i] = __float_as_uint(s);
    }
    if (off > 0.5f - 3e-5f || !finite) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float t = v[i] * f.x * f.y;
            if (!finite || fabsf(__fsub_rn(t, __fsub_rn(__uint_as_float(u[i]), 12582912.f))) > 0.5f - 3e-5f) u[i] = (uint32_t)quant_exact(v[i], m);
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++) q[i] = (signed char)(u[i] & 255u);
}
// a row's scale from r, its largest magnitude and a sum that is finite if all of it is (of h^2 and, for the norm, 0 * w h: NaN where w h is no finite number)
__device__ __forceinline__ float quant_scale(float r, float m, float sum) { return sum - sum == 0.f ? r * __fdiv_rn(m, 127.f) : sum * 0.f; }

// 1 / sqrt(v): the hardware's value (off by 2^-22.9) and one step of Newton's method; v = inf gives 0
__device__ __forceinline__ float norm_factor(float v)
{
    const float r = rsqrtf(v);
    return v < INFINITY ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}

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

// Pairs of single-precision values: one instruction for two products or sums, rounded as two.  What bounds these kernels beside the bytes is the number of
// instructions per element: 31 of them, one by one and with every load under a condition of its own, held the half-precision backward pass at 4 TB/s, and the
// half-precision forward pass at 8192 columns took 57 us value by value, 41 us in pairs.
__device__ __forceinline__ uint64_t pair_bits(float2 v) { return *reinterpret_cast<const uint64_t *>(&v); }
__device__ __forceinline__ float2 pair(uint64_t v) { return *reinterpret_cast<const float2 *>(&v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
    return pair(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
    return pair(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
    return pair(d);
}
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }
template <int V> __device__ __forceinline__ void unpack(const Pack<float, V> &p, float2 (&f)[V / 2])
{
#pragma unroll
    for (int i = 0; i < V / 2; i++) f[i] = make_float2(p.e[2 * i], p.e[2 * i + 1]);
}
template <int V> __device__ __forceinline__ void unpack(const Pack<__half, V> &p, float2 (&f)[V / 2])
{
#pragma unroll
    for (int i = 0; i < V / 2; i++) f[i] = __half22float2(*reinterpret_cast<const __half2 *>(&p.e[2 * i]));
}
template <int V> __device__ __forceinline__ Pack<float, V> repack(const float2 (&f)[V / 2], float *)
{
    Pack<float, V> p;
#pragma unroll
    for (int i = 0; i < V / 2; i++) { p.e[2 * i] = f[i].x; p.e[2 * i + 1] = f[i].y; }
    return p;
}
template <int V> __device__ __forceinline__ Pack<__half, V> repack(const float2 (&f)[V / 2], __half *)
{
    Pack<__half, V> p;
#pragma unroll
    for (int i = 0; i < V / 2; i++) *reinterpret_cast<__half2 *>(&p.e[2 * i]) = __float22half2_rn(f[i]);
    return p;
}

// Two values over a warp, a sum and a sum or maximum, in five exchanges: after the first one the lower half has the first value and the upper half the second.
template <bool MAX> __device__ __forceinline__ float warp_two(float a, float b)
{
    const bool low = (threadIdx.x & 16) == 0;
    float v = low ? a : b;
    const float u = __shfl_xor_sync(0xffffffffu, low ? b : a, 16);
    v = MAX && !low ? fmaxf(v, u) : v + u;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        const float x = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX && !low ? fmaxf(v, x) : v + x;
    }
    return v;
}
// The same over the G threads of a row, for all of them; red: [warps of the block].  SYNC: the barrier between the warps' results and their sum.
template <int G, bool MAX, class SYNC> __device__ __forceinline__ float2 two_reduce(float a, float b, float2 *red, SYNC sync)
{
    const float v = warp_two<MAX>(a, b);
    if constexpr (G == 32) { sync(); return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16)); }
    if ((threadIdx.x & 15) == 0) reinterpret_cast<float *>(&red[threadIdx.x >> 5])[threadIdx.x >> 4 & 1] = v;
    sync();
    const float2 *of = red + threadIdx.x / G * (G / 32);
    float2 t = of[0];
#pragma unroll
    for (int k = 1; k < G / 32; k++) { const float2 x = of[k]; t.x += x.x; t.y = MAX ? fmaxf(t.y, x.y) : t.y + x.y; }
    return t;
}
template <int G, bool MAX> __device__ __forceinline__ float2 row_reduce(float a, float b, float2 *red)        // every thread of the block takes part
{
    return two_reduce<G, MAX>(a, b, red, [] { if (G > 32) __syncthreads(); });
}

// W results of a row: h (the unrounded sum) and the weights of V neighbouring columns
template <class T, int MODE, int V>
__device__ __forceinline__ void norm_leave(float (&h)[V], const Pack<T, V> &wv, float r, float2 f, float2 tot, T *sum, T *y, signed char *q, size_t at)
{
    if (MODE != QUANT_ROWS && sum) {
        Pack<T, V> o;
#pragma unroll
        for (int i = 0; i < V; i++) o.e[i] = fromf<T>(h[i]);
        stv<T, V>(sum + at, o);
    }
    if constexpr (MODE == NORM_PLAIN) {
        Pack<T, V> o;
#pragma unroll
        for (int i = 0; i < V; i++) o.e[i] = fromf<T>(h[i] * r * tof(wv.e[i]));
        stv<T, V>(y + at, o);
    } else {
        Pack<signed char, V> o;
        if (MODE == NORM_INT8) {
#pragma unroll
            for (int i = 0; i < V; i++) h[i] *= tof(wv.e[i]);
        }
        quant<V>(h, f, tot.y, tot.x - tot.x == 0.f, o.e);
        stv<signed char, V>(q + at, o);
    }
}
// dw's partial sum of a block from its RG groups of rows, the groups in order; cols: [RG, size]
template <class T, int G, int NV, int V, int RG, int TPB>
__device__ __forceinline__ void block_columns(const float (&acc)[NV][V], float *out, float *cols, int size, int t, int mine)
{
    if constexpr (RG > 1) __syncthreads();                   // (the ring's memory is read no more)
    float *to = RG > 1 ? cols + mine * size : out;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = (k * G + t) * V;
        constexpr int U = V < 4 ? V : 4;
        if (j >= size) continue;
#pragma unroll
        for (int i = 0; i < V; i += U) {
            Pack<float, U> o;
#pragma unroll
            for (int e = 0; e < U; e++) o.e[e] = acc[k][i + e];
            stv<float, U>(to + j + i, o);
        }
    }
    if constexpr (RG > 1) {
        __syncthreads();
        for (int j = threadIdx.x; j < size; j += TPB) {
            float v = cols[j];
#pragma unroll
            for (int g = 1; g < RG; g++) v += cols[g * size + j];
            out[j] = v;
        }
    }
}

// ---------------------------------------------------------------- rows through a ring in shared memory
// The backward pass holds its columns' sums of dy h r in registers from row to row, so one CTA per SM walks many rows, and what its registers leave free does not
// cover the memory's latency.  So the rows arrive by bulk copies in a ring of stages (IN tensors' rows each), some 200 KB under way per SM; a group of G threads
// walks rows of its own and waits for nobody but itself.  A stage is fetched anew as soon as the group's sums have met: by then all of it is in registers.
static constexpr int RING_TPB = 512, RING_BYTES = 200 * 1024, RING_MOST = 8;
template <int G> __device__ __forceinline__ void group_sync()
{
    if constexpr (G == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / G), "n"(G) : "memory");
}
template <int G, bool MAX> __device__ __forceinline__ float2 group_reduce(float a, float b, float2 *red) { return two_reduce<G, MAX>(a, b, red, [] { group_sync<G>(); }); }
template <class T, int G, int IN> struct Ring {
    const T *src[IN];
    unsigned char *base;
    uint64_t *full;
    volatile int *failed;
    int *status;
    int stages, size, rows, row0, step, count;           // of this group: first row, rows between two of its rows, how many
    int issued;                                          // (of the thread that fetches)
    __device__ __forceinline__ T *stage(int s, int in) const { return reinterpret_cast<T *>(base) + ((size_t)s * IN + in) * size; }
    __device__ __forceinline__ void issue(int i)
    {
        const int s = i % stages;
        issued = i + 1;
        const size_t at = (size_t)(row0 + (long long)i * step) * size;
        int n = 0;
#pragma unroll
        for (int k = 0; k < IN; k++) n += src[k] != nullptr;
        tc::mbar_arrive_expect_tx(&full[s], (uint32_t)(n * size * (int)sizeof(T)));
#pragma unroll
        for (int k = 0; k < IN; k++) if (src[k]) tc::bulk_load(stage(s, k), src[k] + at, (uint32_t)(size * sizeof(T)), &full[s]);
    }
    // Bounded: after about a second the CTA's flag is up, nothing is fetched any more and the other waits end at once (all threads keep walking, so that no
    // barrier is short of one); the status word tells.
    __device__ __forceinline__ void wait(int i)
    {
        uint64_t *bar = &full[i % stages];
        const uint32_t parity = (uint32_t)(i / stages) & 1u;
        for (uint32_t k = 0; k < 8000000u; k++) {
            if (tc::mbar_try_wait(bar, parity)) return;
            if ((k & 63u) == 63u && *failed) return;
        }
        *failed = 1;
        atomicCAS(status, 0, 10);
    }
    __device__ __forceinline__ void start(int t) { if (t == 0) for (int i = 0; i < min(stages, count); i++) issue(i); }
    __device__ __forceinline__ void refill(int i, int t) { if (t == 0 && i + stages < count && !*failed) issue(i + stages); }
    // given up: what is under way lands before the shared memory is left
    __device__ __forceinline__ void settle(int t)
    {
        if (t != 0 || !*failed) return;
        for (int i = max(0, issued - stages); i < issued; i++)
            for (int k = 0; k < 100000 && !tc::mbar_try_wait(&full[i % stages], (uint32_t)(i / stages) & 1u); k++) __nanosleep(100);
    }
};
template <class T, int G, int IN> __device__ __forceinline__ Ring<T, G, IN> make_ring(unsigned char *mem, uint64_t (*full)[RING_MOST], int *failed, int *status, int stages, int size, int rows)
{
    constexpr int RG = RING_TPB / G;
    const int mine = threadIdx.x / G;
    Ring<T, G, IN> r;
    r.base = mem + (size_t)mine * stages * IN * size * sizeof(T);
    r.full = full[mine]; r.failed = failed; r.status = status;
    r.stages = stages; r.size = size; r.rows = rows;
    r.row0 = blockIdx.x * RG + mine; r.step = gridDim.x * RG;
    r.count = r.row0 < rows ? (rows - 1 - r.row0) / r.step + 1 : 0;
    r.issued = 0;
    if (threadIdx.x < RG) for (int s = 0; s < stages; s++) tc::mbar_init(&full[threadIdx.x][s], 1);
    if (threadIdx.x == 0) *failed = 0;
    tc::fence_barrier_init();
    __syncthreads();
    return r;
}

// the 8-bit form of V values, as quant(); SCALED: a row's magnitudes may be so small that 127 / m is not finite (half precision has none such)
template <int V, bool SCALED> __device__ __forceinline__ Pack<signed char, V> quant_pairs(const float2 (&v)[V / 2], float2 f, float m, bool finite)
{
    uint32_t u[V];
    float off = 0.f;
    const float2 fx = twice(f.x), fy = twice(f.y), big = twice(12582912.f), less = twice(-12582912.f);
#pragma unroll
    for (int i = 0; i < V / 2; i++) {
        const float2 t = SCALED ? mul2(mul2(v[i], fx), fy) : mul2(v[i], fy), r = add2(t, big), n = add2(r, less), d = fma2(n, twice(-1.f), t);
        off = fmaxf(off, fmaxf(fabsf(d.x), fabsf(d.y)));
        u[2 * i] = __float_as_uint(r.x); u[2 * i + 1] = __float_as_uint(r.y);
    }
    if (off > 0.5f - 3e-5f || !finite) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float x = i & 1 ? v[i / 2].y : v[i / 2].x, t = x * f.x * f.y;
            if (!finite || fabsf(__fsub_rn(t, __fsub_rn(__uint_as_float(u[i]), 12582912.f))) > 0.5f - 3e-5f) u[i] = (uint32_t)quant_exact(x, m);
        }
    }
    Pack<signed char, V> q;
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<uint32_t *>(&q.e[i]) = __byte_perm(__byte_perm(u[i], u[i + 1], 0x0040), __byte_perm(u[i + 2], u[i + 3], 0x0040), 0x5410);
    return q;
}

// backward: as rmsnorm_bw_kernel, below.  2^25 elements of each of four tensors with the sum of dw's parts behind it: halves 46 us at 1000, 2048 and 8192 columns, 73 at 256
// (a warp's fixed cost per row), floats 81 to 86 (41 and 82 at the rate of a plain copy).
template <class T, int G, int NV, int V>
__global__ void __launch_bounds__(RING_TPB) rmsnorm_bw_ring_kernel(const T *h, const T *__restrict__ w, const T *dy, const T *dsum, T *dx, float *__restrict__ part,
                                                                   int rows, int size, int stages, float eps, int *status)
{
    pdl_wait();
    const float per = 1.f / (float)size;
    constexpr int RG = RING_TPB / G, P = V / 2;
    extern __shared__ __align__(128) unsigned char ring_mem[];
    __shared__ uint64_t full[RG][RING_MOST];
    __shared__ float2 red[2][RING_TPB / 32];
    __shared__ int failed;
    Ring<T, G, 3> ring = make_ring<T, G, 3>(ring_mem, full, &failed, status, stages, size, rows);
    ring.src[0] = h; ring.src[1] = dy; ring.src[2] = dx ? dsum : nullptr;
    const bool more = ring.src[2] != nullptr;
    const int t = threadIdx.x % G, mine = threadIdx.x / G;
    ring.start(t);
    float2 wv[NV][P], acc[NV][P];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = (k * G + t) * V;
        unpack<V>(j < size ? ldv<T, V>(w + j) : zerov<T, V>(), wv[k]);
#pragma unroll
        for (int e = 0; e < P; e++) acc[k][e] = twice(0.f);
    }
    int s_at = 0;
    for (int i = 0; i < ring.count; i++, s_at = s_at + 1 == stages ? 0 : s_at + 1) {
        const size_t at = (size_t)(ring.row0 + i * ring.step) * size;
        ring.wait(i);
        const T *in_h = ring.stage(s_at, 0), *in_g = ring.stage(s_at, 1), *in_d = ring.stage(s_at, 2);
        float2 hv[NV][P], gv[NV][P], s2 = twice(0.f), c2 = twice(0.f);
        Pack<T, V> dv[NV];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int j = (k * G + t) * V;
            if (j >= size) continue;
            unpack<V>(ldv<T, V>(in_h + j), hv[k]);
            unpack<V>(ldv<T, V>(in_g + j), gv[k]);
            if (more) dv[k] = ldv<T, V>(in_d + j);
#pragma unroll
            for (int e = 0; e < P; e++) {
                s2 = fma2(hv[k][e], hv[k][e], s2);
                c2 = fma2(hv[k][e], mul2(gv[k][e], wv[k][e]), c2);
            }
        }
        const float2 tot = group_reduce<G, false>(s2.x + s2.y, c2.x + c2.y, red[i & 1]);
        ring.refill(i, t);
        const float r = norm_factor(fmaf(tot.x, per, eps)), cr = tot.y * per * r * r;
        const float2 rr = twice(r), less = twice(-cr);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int j = (k * G + t) * V;
            if (j >= size) continue;
            float2 d[P];
            if (more) unpack<V>(dv[k], d);
#pragma unroll
            for (int e = 0; e < P; e++) {
                acc[k][e] = fma2(mul2(gv[k][e], hv[k][e]), rr, acc[k][e]);
                const float2 v = fma2(hv[k][e], less, mul2(gv[k][e], wv[k][e]));
                d[e] = more ? fma2(rr, v, d[e]) : mul2(rr, v);
            }
            if (dx) stv<T, V>(dx + at + j, repack<V>(d, (T *)nullptr));
        }
    }
    ring.settle(t);
    if (part) {
        float a[NV][V];
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < P; e++) { a[k][2 * e] = acc[k][e].x; a[k][2 * e + 1] = acc[k][e].y; }
        block_columns<T, G, NV, V, RG, RING_TPB>(a, part + (size_t)blockIdx.x * size, reinterpret_cast<float *>(ring_mem), size, t, mine);
    }
}
// stages per group (two at least: a group's rows are 96 KB at most for all of them together)
template <class T> static int ring_stages(int groups, int in, int size) { return std::min(RING_BYTES / (groups * in * size * (int)sizeof(T)), RING_MOST); }

// ---------------------------------------------------------------- forward
// G threads per row, a block's rows side by side, NV packs of V elements per thread; small CTAs, so that one's loads cover the other's stores.  Measured with
// x, residual, sum and y of 2^25 elements (41 us half, 82 us single at the rate of a plain copy): halves 40.4 us at 256 columns, 40.8 at 1000 and 2048, 41.4 at 8192,
// 44.8 at 16384; floats 79 us from 256 to 8192 columns, 84 at 16384; 999 columns, element by element, 58 and 80 us.  To 8 bits, with the sum: 41.7 and 40.7 us
// for halves at 2048 and 8192 columns (35.9), 75 at 999; 32.9 for 2^24 floats at 2048 (33.3).
// (CTAs per SM that the registers are held down to: 1024 threads with 4 or 8 packs each, 768 of 256 with 8, 1280 with fewer)
constexpr int fw_blocks(int g, int nv, bool few) { return g < 512 ? nv == 8 ? 3 : nv == 4 ? 4 : 5 : nv == 4 || few ? 2 : 1; }
template <class T, int MODE, int G, int NV, int V>
__global__ void __launch_bounds__(G < 256 ? 256 : G, fw_blocks(G, NV, MODE == QUANT_ROWS || V < 4)) rmsnorm_fw_kernel(const T *x, const T *res, const T *__restrict__ w, T *sum, T *y, signed char *__restrict__ q,
                                                                       float *__restrict__ scale, int rows, int size, float eps)
{
    pdl_wait();
    const float per = 1.f / (float)size;
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
    if constexpr (V >= 4) {
        constexpr int P = V / 2;
        float2 h[NV][P], s2 = twice(0.f);
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float2 c[P], ww[P];
            unpack<V>(a[k], h[k]);
            unpack<V>(b[k], c);
            if (MODE == NORM_INT8) unpack<V>(wv[k], ww);
#pragma unroll
            for (int e = 0; e < P; e++) {
                h[k][e] = add2(h[k][e], c[e]);
                s2 = fma2(h[k][e], MODE == QUANT_ROWS ? twice(0.f) : h[k][e], s2);       // (quantised alone, the sum tells only whether every value is finite)
                if (MODE != NORM_PLAIN) {
                    const float2 v = MODE == NORM_INT8 ? mul2(h[k][e], ww[e]) : h[k][e];
                    m = fmaxf(m, fmaxf(fabsf(v.x), fabsf(v.y)));
                    if (MODE == NORM_INT8) s2 = fma2(v, twice(0.f), s2);                  // (a weight that is no number shows in the sum, too)
                }
            }
        }
        const float2 tot = row_reduce<G, true>(s2.x + s2.y, m, red);     // (the largest magnitude passes over NaN: the scale carries it)
        if (row >= rows) return;
        const float r = MODE == QUANT_ROWS ? 1.f : norm_factor(fmaf(tot.x, per, eps));
        const float2 f = MODE == NORM_PLAIN ? make_float2(0.f, 0.f) : quant_factor(tot.y);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int j = (k * G + t) * V;
            if (j >= size) continue;
            if (MODE != QUANT_ROWS && sum) stv<T, V>(sum + at + j, repack<V>(h[k], (T *)nullptr));
            if (MODE != QUANT_ROWS) {
                float2 ww[P];
                unpack<V>(wv[k], ww);
#pragma unroll
                for (int e = 0; e < P; e++) h[k][e] = mul2(MODE == NORM_PLAIN ? mul2(h[k][e], twice(r)) : h[k][e], ww[e]);
            }
            if constexpr (MODE == NORM_PLAIN) stv<T, V>(y + at + j, repack<V>(h[k], (T *)nullptr));
            else stv<signed char, V>(q + at + j, quant_pairs<V, sizeof(T) == 4 || MODE == NORM_INT8>(h[k], f, tot.y, tot.x - tot.x == 0.f));
        }
        if (MODE != NORM_PLAIN && t == 0) scale[row] = quant_scale(r, tot.y, tot.x);
        return;
    }
    float s = 0.f, m = 0.f, h[NV][V];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            h[k][i] = tof(a[k].e[i]) + tof(b[k].e[i]);
            s = MODE == QUANT_ROWS ? fmaf(h[k][i], 0.f, s) : fmaf(h[k][i], h[k][i], s);                  // (quantised alone, the sum tells only whether every value is finite)
            if (MODE != NORM_PLAIN) {
                const float v = MODE == NORM_INT8 ? h[k][i] * tof(wv[k].e[i]) : h[k][i];
                m = fmaxf(m, fabsf(v));                                                                  // (passes over NaN: the scale carries it)
                if (MODE == NORM_INT8) s = fmaf(v, 0.f, s);                                              // (and a weight's that is none)
            }
        }
    const float2 tot = row_reduce<G, true>(s, m, red);
    if (row >= rows) return;
    const float r = MODE == QUANT_ROWS ? 1.f : norm_factor(fmaf(tot.x, per, eps));
    const float2 f = MODE == NORM_PLAIN ? make_float2(0.f, 0.f) : quant_factor(tot.y);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = (k * G + t) * V;
        if (j < size) norm_leave<T, MODE, V>(h[k], wv[k], r, f, tot, sum, y, q, at + j);
    }
    if (MODE != NORM_PLAIN && t == 0) scale[row] = quant_scale(r, tot.y, tot.x);
}
// A CTA per row, any width: a pass for the row's sum of squares and largest magnitude, a second one for the results.
template <class T, int MODE>
__global__ void __launch_bounds__(1024) rmsnorm_fw_wide_kernel(const T *x, const T *res, const T *__restrict__ w, T *sum, T *y, signed char *__restrict__ q,
                                                               float *__restrict__ scale, int size, float eps)
{
    pdl_wait();
    const float per = 1.f / (float)size;
    __shared__ float2 red[32];
    const size_t at = (size_t)blockIdx.x * size;
    float s = 0.f, m = 0.f;
#pragma unroll 4
    for (int j = threadIdx.x; j < size; j += 1024) {
        const float h = ld(x + at + j) + (res ? ld(res + at + j) : 0.f);
        s = MODE == QUANT_ROWS ? fmaf(h, 0.f, s) : fmaf(h, h, s);
        if (MODE != NORM_PLAIN) {
            const float v = MODE == NORM_INT8 ? h * ld(w + j) : h;
            m = fmaxf(m, fabsf(v));
            if (MODE == NORM_INT8) s = fmaf(v, 0.f, s);
        }
    }
    const float2 tot = row_reduce<1024, true>(s, m, red);
    const float r = MODE == QUANT_ROWS ? 1.f : norm_factor(fmaf(tot.x, per, eps));
    const float2 f = quant_factor(tot.y);
    for (int j = threadIdx.x; j < size; j += 1024) {
        const float h = ld(x + at + j) + (res ? ld(res + at + j) : 0.f);
        if (MODE != QUANT_ROWS && sum) st(sum + at + j, h);
        if (MODE == NORM_PLAIN) st(y + at + j, h * r * ld(w + j));
        else {
            const float v[1] = {MODE == NORM_INT8 ? h * ld(w + j) : h};
            signed char o[1];
            quant<1>(v, f, tot.y, tot.x - tot.x == 0.f, o);
            q[at + j] = o[0];
        }
    }
    if (MODE != NORM_PLAIN && threadIdx.x == 0) scale[blockIdx.x] = quant_scale(r, tot.y, tot.x);
}

// The 8-bit form of half-precision rows as they are: a CTA of G threads per row, the halves in registers as they lie, the largest magnitude two at a time.
// 4096 rows of 8192: 26 us, the bytes alone 15; the rounding's fourteen instructions per element hold it there.  (A ring in shared memory with one CTA per SM was a tenth
// slower; a second division in quant_exact made it 29: most rows have a value near a border.)
template <int G, int NV>
__global__ void __launch_bounds__(G, 1280 / G) quantize_rows_kernel(const __half *__restrict__ x, signed char *__restrict__ q, float *__restrict__ scale, int size)
{
    pdl_wait();
    constexpr int V = 8, P = V / 2;
    __shared__ float2 red[G / 32];
    const size_t at = (size_t)blockIdx.x * size;
    Pack<__half, V> raw[NV];
    __half2 m2 = __float2half2_rn(0.f);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = (k * G + threadIdx.x) * V;
        raw[k] = j < size ? ldv<__half, V>(x + at + j) : zerov<__half, V>();
    }
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int e = 0; e < P; e++) m2 = __hmax2_nan(m2, __habs2(*reinterpret_cast<const __half2 *>(&raw[k].e[2 * e])));
    const float m = __half2float(__hmax_nan(__low2half(m2), __high2half(m2)));
    const float2 tot = row_reduce<G, true>(m * 0.f, m, red);             // the sum tells only whether every value is finite
    const float2 f = quant_factor(tot.y);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = (k * G + threadIdx.x) * V;
        if (j >= size) continue;
        float2 h[P];
        unpack<V>(raw[k], h);
        stv<signed char, V>(q + at + j, quant_pairs<V, false>(h, f, tot.y, tot.x == 0.f));
    }
    if (threadIdx.x == 0) scale[blockIdx.x] = quant_scale(1.f, tot.y, tot.x);
}

template <class T, int MODE>
static void norm_forward(const T *x, const T *res, const T *w, T *sum, T *y, signed char *q, float *scale, int rows, int size, float eps)
{
    constexpr int V16 = 16 / (int)sizeof(T);
    // packs of 16 bytes where every row of every tensor starts on such a boundary (the 8-bit one on V16 bytes)
    const uintptr_t at = (uintptr_t)x | (uintptr_t)res | (uintptr_t)w | (uintptr_t)sum | (uintptr_t)y;
    const bool wide = size % V16 == 0 && at % 16 == 0 && (uintptr_t)q % V16 == 0;
    // or of two halves
    constexpr int V2 = sizeof(T) == 2 ? 2 : 1;
    const bool two = V2 == 2 && size % 2 == 0 && at % 4 == 0 && (uintptr_t)q % 2 == 0;
    const int packs = wide ? size / V16 : two ? size / 2 : size;
#define TL_NORM(G, NV, V) TL_LAUNCH((rmsnorm_fw_kernel<T, MODE, G, NV, V>), ceil_div(rows, (G < 256 ? 256 : G) / G), G < 256 ? 256 : G, 0, x, res, w, sum, y, q, scale, rows, size, eps)
#define TL_NORM_V(V)                                                                                  \
    do {                                                                                              \
        constexpr bool FEW = MODE == QUANT_ROWS || V < 4;                                             \
        if (packs <= 32) TL_NORM(32, 1, V);                                                           \
        else if (packs <= 64) TL_NORM(32, 2, V);                                                      \
        else if (packs <= 128) TL_NORM((FEW ? 32 : 64), (FEW ? 4 : 2), V);                            \
        else if (packs <= 256) TL_NORM((FEW ? 32 : 128), (FEW ? 8 : 2), V);                           \
        else if (packs <= 512) TL_NORM((FEW ? 64 : 256), (FEW ? 8 : 2), V);                           \
        else if (packs <= 1024) TL_NORM((FEW ? 128 : 256), (FEW ? 8 : 4), V);                         \
        else if (packs <= 2048) TL_NORM((FEW ? 256 : 512), (FEW ? 8 : 4), V);                         \
        else TL_NORM(512, 8, V);                                                                      \
    } while (0)
    if constexpr (MODE == QUANT_ROWS && sizeof(T) == 2) {
        if (wide && size > 512 && size <= 16384) {
            if (size <= 1024) TL_LAUNCH((quantize_rows_kernel<128, 1>), rows, 128, 0, x, q, scale, size);
            else if (size <= 2048) TL_LAUNCH((quantize_rows_kernel<128, 2>), rows, 128, 0, x, q, scale, size);
            else if (size <= 4096) TL_LAUNCH((quantize_rows_kernel<128, 4>), rows, 128, 0, x, q, scale, size);
            else if (size <= 8192) TL_LAUNCH((quantize_rows_kernel<256, 4>), rows, 256, 0, x, q, scale, size);
            else TL_LAUNCH((quantize_rows_kernel<512, 4>), rows, 512, 0, x, q, scale, size);
            return;
        }
    }
    if (packs > 4096) TL_LAUNCH((rmsnorm_fw_wide_kernel<T, MODE>), rows, 1024, 0, x, res, w, sum, y, q, scale, size, eps);
    else if (wide) TL_NORM_V(V16);
    else if (two) TL_NORM_V(V2);
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
    const float per = 1.f / (float)size;
    constexpr int TPB = G < NB_TPB ? NB_TPB : G, RG = TPB / G;
    __shared__ float2 red[2][TPB / 32];
    extern __shared__ __align__(16) float cols[];        // [RG, size], where RG > 1
    const int t = threadIdx.x % G, mine = threadIdx.x / G;
    Pack<T, V> hv[NV], gv[NV];
    float acc[NV][V];
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < V; i++) acc[k][i] = 0.f;
    auto weight = [&](int k) { const int j = (k * G + t) * V; return j < size ? ldv<T, V>(w + j) : zerov<T, V>(); };       // (from L1: registers go to the rows)
    auto fetch = [&](long long row) {
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
    for (long long base = (long long)blockIdx.x * RG; base < rows; base += (long long)gridDim.x * RG, turn ^= 1) {
        const long long row = base + mine;
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
        if (PRE) fetch(row + (long long)gridDim.x * RG);       // under way while the row's sums meet (dx may be one of the inputs: of this row, which is in registers)
        const float2 tot = row_reduce<G, false>(s, c, red[turn]);
        if (!PRE) residual();
        const float r = norm_factor(fmaf(tot.x, per, eps)), cr = tot.y * per * r * r;
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
    if (part) block_columns<T, G, NV, V, RG, TPB>(acc, part + (size_t)blockIdx.x * size, cols, size, t, mine);
}
// dw from the blocks' partial sums: 32 columns by 32 slices of the blocks, each slice in order, the slices in order (3 us behind the rows' kernel)
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
    const float per = 1.f / (float)size;
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
    const float r = norm_factor(fmaf(tot.x, per, eps));
    if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(r, tot.y * per * r * r);
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
    if (wide && size <= 512 * 16) {
        int *status = tc_status_word();
        if (!status) return set_error(TL_ERR_NO_MEMORY, "no memory for the word in which a kernel's waits report");
#define TL_NORM_BW_RING(G, NV)                                                                                                                                        \
    do {                                                                                                                                                              \
        const int stages = ring_stages<T>(RING_TPB / G, 3, size), blocks = std::min(ceil_div(rows, RING_TPB / G), sm_count());                                        \
        float *part = dw ? sc.scratch<float>((size_t)blocks * size) : nullptr;                                                                                        \
        if (dw && !part) return;                                                                                                                                      \
        static bool set = false;                                                                                                                                      \
        if (!set) set = cudaFuncSetAttribute(rmsnorm_bw_ring_kernel<T, G, NV, V16>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES) == cudaSuccess;          \
        TL_LAUNCH((rmsnorm_bw_ring_kernel<T, G, NV, V16>), blocks, RING_TPB, RING_BYTES, h, w, dy, dsum, dx, part, rows, size, stages, eps, status);                  \
        if (dw) norm_columns<T>(part, dw, size, blocks);                                                                                                              \
    } while (0)
        constexpr int E = 16 / V16;
        if (size <= 32 * 8) TL_NORM_BW_RING(32, (E + 1) / 2);
        else if (size <= 32 * 16) TL_NORM_BW_RING(32, E);
        else if (size <= 64 * 16) TL_NORM_BW_RING(64, E);
        else if (size <= 128 * 16) TL_NORM_BW_RING(128, E);
        else if (size <= 256 * 16) TL_NORM_BW_RING(256, E);
        else TL_NORM_BW_RING(512, E);
#undef TL_NORM_BW_RING
        return;
    }
#define TL_NORM_BW(G, NV, V, PRE)                                                                                                                             \
    do {                                                                                                                                                      \
        constexpr int TPB = G < NB_TPB ? NB_TPB : G, RG = TPB / G;                                                                                            \
        const int blocks = std::min(ceil_div(rows, RG), (TPB == 1024 ? 1 : 2) * sm_count());                                                                  \
        float *part = dw ? sc.scratch<float>((size_t)blocks * size) : nullptr;                                                                                \
        if (dw && !part) return;                                                                                                                              \
        TL_LAUNCH((rmsnorm_bw_kernel<T, G, NV, V, PRE>), blocks, TPB, RG > 1 ? RG * size * sizeof(float) : 0, h, w, dy, dsum, dx, part, rows, size, eps);          \
        if (dw) norm_columns<T>(part, dw, size, blocks);                                                                                                      \
    } while (0)
    if (wide) TL_NORM_BW(1024, 16 / V16, V16, false);
    else if (size <= 32) TL_NORM_BW(32, 1, 1, true);
    else if (size <= 32 * 8) TL_NORM_BW(32, 8, 1, true);
    else if (size <= 64 * 8) TL_NORM_BW(64, 8, 1, true);
    else if (size <= 128 * 8) TL_NORM_BW(128, 8, 1, true);
    else if (size <= 256 * 8) TL_NORM_BW(256, 8, 1, true);
    else if (size <= 512 * 8) TL_NORM_BW(512, 8, 1, true);
    else if (size <= 1024 * 8) TL_NORM_BW(1024, 8, 1, false);
    else TL_NORM_BW(1024, 16, 1, false);
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
