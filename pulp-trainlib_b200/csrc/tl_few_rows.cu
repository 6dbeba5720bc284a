// The forward products of the feed-forward block and the 8-bit linear layer for few tokens (a generation loop's): bound by the weights' bytes, which are
// read once, straight into the registers that the matrix instruction takes them from.
//   A CTA has 16 rows of the weights (16 of each matrix for the gate; 32 where there are many tokens and enough rows) and all tokens; its warps share K in
//   pieces of 64 bytes.  The order of K inside a piece does not matter to a sum as long as both operands keep it: a thread loads 16 neighbouring bytes of
//   its two weight rows and of its token, and they serve as the fragments of two mma.sync (m16n8k16 fp16, m16n8k32 in 8 bits): no shared memory, no
//   shuffles.  The warps' sums meet in shared memory, in order.
//   What counts is the number of loads under way: a thread issues all of a turn's, 256 bytes of weights, before it waits for the first.
//   (Rings in shared memory with even shares of all bytes for persistent CTAs, by bulk copies of 1 KB or by cp.async, keep more under way, but lose more than
//   that at the ends of the units: 8-bit 4096 -> 10240 for one token 16 us against 11, fp16 4096 x 10240 x 4096 57 us against 54.)
//   Rows that do not start on 16 bytes come as the five words around the thread's bytes, shifted into place, without a condition up to the last piece or two of
//   a row (23 tokens of 1000 x 2731 x 1000: 15.7 us; a condition around every piece's words, each waiting for the one before, 18.8; 2736: 10.5).
//   Half precision, up to eight tokens: silu(gate) * up goes from one product to the other in two halves, itself and what its rounding left: the weights' bytes
//   are what counts, and the result is rounded once (one token of 4096 x 10240 x 4096: 45.9 us, with one rounded half 44.4; 32 tokens would take 76 for 66).
//   Single precision: the same on m16n8k8 in TF32, every operand as two parts and three products of them; the sums move to others, rounded to nearest, after
//   each turn (the instruction's own sum is cut off towards zero at every step).
#include "tl_gate.cuh"
#include "tl_tc.cuh"
#include "tl_reduce.cuh"
#include <type_traits>

namespace tl {

enum { FEW_F16 = 0, FEW_I8 = 1, FEW_F32 = 2 };
template <int KIND> struct FewType { typedef __half E; typedef float S; };
template <> struct FewType<FEW_I8> { typedef signed char E; typedef int S; };
template <> struct FewType<FEW_F32> { typedef float E; typedef float S; };

template <class T> struct FewParams {
    const void *x, *x2, *w[2];          // x2: what rounding x to its type left (FFN_PLAIN in half precision)
    T *C, *C2, *g, *u;                  // C2: what rounding C left (FFN_GATE in half precision)
    const T *bias; const float *xs, *ws;
    int rows, M, K;                     // tokens, weight rows, elements of K
    long long x_stride, c_stride;       // elements
    bool words, x16;                    // every tensor starts on four bytes; x's rows on sixteen
};

// 16 neighbouring bytes of a row of K elements from element k on, zeros behind the end.  ALIGN < 16: rows start anywhere.  Inside a row (four bytes in front of the
// piece and behind it are the row's too) as whole words, at its ends element by element.
template <class E, int ALIGN> __device__ __forceinline__ uint4 few_load(const E *row, int k, int K)
{
    constexpr int N = 16 / (int)sizeof(E), WORD = 4 / (int)sizeof(E);
    uint4 v = make_uint4(0, 0, 0, 0);
    if constexpr (ALIGN == 16) { if (k < K) v = *reinterpret_cast<const uint4 *>(row + k); }
    else if (k >= WORD && k + N + WORD <= K) {
        const uintptr_t at = (uintptr_t)(row + k);
        const uint32_t *w = reinterpret_cast<const uint32_t *>(at & ~(uintptr_t)3), sh = (uint32_t)(at & 3) * 8u;
        const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3], w4 = w[4];
        v = make_uint4(__funnelshift_r(w0, w1, sh), __funnelshift_r(w1, w2, sh), __funnelshift_r(w2, w3, sh), __funnelshift_r(w3, w4, sh));
    } else if (k < K) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < N; i++) {
            uint32_t e = 0;
            if (k + i < K) { if constexpr (sizeof(E) == 4) e = *reinterpret_cast<const uint32_t *>(row + k + i); else if constexpr (sizeof(E) == 2) e = *reinterpret_cast<const unsigned short *>(row + k + i); else e = *reinterpret_cast<const unsigned char *>(row + k + i); }
            if constexpr (sizeof(E) == 4) w[i] = e; else w[i * 4 / N] |= e << (i % (N / 4) * 8 * (int)sizeof(E));
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
}
// Loads that are issued where they stand, all of a turn's in front of its first product: the weights past L1 (nobody reads them again), the tokens through it.
__device__ __forceinline__ uint4 few_stream(const void *p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 few_keep(const void *p)
{
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t few_word(const void *p)
{
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
// 16 bytes of a row that starts on four bytes or between: the five words around them as they come, to be shifted into place when they are used
struct FewRaw { uint32_t w[5]; };
template <class E> __device__ __forceinline__ FewRaw few_raw(const E *at, bool whole)
{
    FewRaw r;
    if (whole) {                                             // (the row starts on sixteen)
        const uint4 v = few_keep(at);
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w; r.w[4] = 0;
    } else {
        const uint32_t *from = reinterpret_cast<const uint32_t *>((uintptr_t)at & ~(uintptr_t)3);
#pragma unroll
        for (int i = 0; i < 5; i++) r.w[i] = few_word(from + i);
    }
    return r;
}
__device__ __forceinline__ uint4 few_place(const FewRaw &r, const void *row)
{
    const uint32_t sh = (uint32_t)((uintptr_t)row & 3) * 8u;                 // (pieces are multiples of four bytes)
    return make_uint4(__funnelshift_r(r.w[0], r.w[1], sh), __funnelshift_r(r.w[1], r.w[2], sh), __funnelshift_r(r.w[2], r.w[3], sh), __funnelshift_r(r.w[3], r.w[4], sh));
}
__device__ __forceinline__ void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void few_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void few_mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void few_split(uint4 v, uint4 &hi, uint4 &lo)
{
    tc::split_tf32_rn(__uint_as_float(v.x), hi.x, lo.x); tc::split_tf32_rn(__uint_as_float(v.y), hi.y, lo.y);
    tc::split_tf32_rn(__uint_as_float(v.z), hi.z, lo.z); tc::split_tf32_rn(__uint_as_float(v.w), hi.w, lo.w);
}
// a result: v (and w, the second matrix') of token n and weight row m
template <class T, int EPI, class S> __device__ __forceinline__ void few_result(const FewParams<T> &p, int n, int m, S v, S w)
{
    const long long at = n * p.c_stride + m;
    if constexpr (EPI == FFN_GATE) {
        if (p.g) { st(p.g + (long long)n * p.M + m, v); st(p.u + (long long)n * p.M + m, w); }
        const float h = gate_fw<sizeof(T) == 2>(v, w);
        st(p.C + at, h);
        if constexpr (sizeof(T) == 2) if (p.C2) { const float rest = h - ld(p.C + at); st(p.C2 + at, fabsf(rest) < INFINITY ? rest : 0.f); }      // (nothing is left of an infinity)
    } else if constexpr (EPI == FFN_INT8) st(p.C + at, (float)v * p.xs[n] * p.ws[m] + ld0(p.bias != nullptr, p.bias + m));
    else st(p.C + at, v);
}

// NT: groups of eight tokens; MT: groups of 16 weight rows; WARPS: that share K
template <int KIND, class T, int EPI, int NT, int MT, int ALIGN, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS) few_rows_kernel(const __grid_constant__ FewParams<T> p)
{
    pdl_wait();
    typedef typename FewType<KIND>::E E;
    typedef typename FewType<KIND>::S S;
    constexpr int MATS = EPI == FFN_GATE ? 2 : 1, N = 16 / (int)sizeof(E), PIECE = 4 * N;
    // pieces of a turn: 256 bytes of weights per thread, 128 where the tokens take as many registers
    constexpr bool F32 = KIND == FEW_F32, TWO = KIND == FEW_F16 && EPI == FFN_PLAIN && NT == 1;      // TWO: the tokens in two parts
    constexpr int U = (NT > 1 || F32 || TWO ? 4 : 8) / (MATS * MT);
    __shared__ S red[WARPS][MATS * MT * NT * 4][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, m0 = blockIdx.x * 16 * MT;
    const E *x = reinterpret_cast<const E *>(p.x);
    S acc[MATS][MT][NT][4];
#pragma unroll
    for (int a = 0; a < MATS * MT * NT * 4; a++) (&acc[0][0][0][0])[a] = 0;
    // rows behind the last are the last once more (their results are not written): no load has a condition
    const E *wp[MATS][MT][2], *xp[NT];
    const long long rest = TWO ? reinterpret_cast<const E *>(p.x2) - x : 0;
#pragma unroll
    for (int b = 0; b < MATS; b++)
#pragma unroll
        for (int a = 0; a < MT; a++)
#pragma unroll
            for (int h = 0; h < 2; h++) wp[b][a][h] = reinterpret_cast<const E *>(p.w[b]) + (long long)min(m0 + 16 * a + g + 8 * h, p.M - 1) * p.K;
#pragma unroll
    for (int n = 0; n < NT; n++) xp[n] = x + min(8 * n + g, p.rows - 1) * p.x_stride;
    constexpr int XP = TWO ? 2 : 1;
    auto multiply = [&](const uint4 (&wv)[MATS][MT][2], const uint4 (&xv)[XP * NT]) {
        if constexpr (F32) {
            uint4 xh[NT], xl[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) few_split(xv[n], xh[n], xl[n]);
#pragma unroll
            for (int b = 0; b < MATS; b++)
#pragma unroll
                for (int a = 0; a < MT; a++) {
                    uint4 ph, pl, qh, ql;
                    few_split(wv[b][a][0], ph, pl);
                    few_split(wv[b][a][1], qh, ql);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        few_mma_tf32(acc[b][a][n], pl.x, ql.x, pl.y, ql.y, xh[n].x, xh[n].y);
                        few_mma_tf32(acc[b][a][n], pl.z, ql.z, pl.w, ql.w, xh[n].z, xh[n].w);
                        few_mma_tf32(acc[b][a][n], ph.x, qh.x, ph.y, qh.y, xl[n].x, xl[n].y);
                        few_mma_tf32(acc[b][a][n], ph.z, qh.z, ph.w, qh.w, xl[n].z, xl[n].w);
                        few_mma_tf32(acc[b][a][n], ph.x, qh.x, ph.y, qh.y, xh[n].x, xh[n].y);
                        few_mma_tf32(acc[b][a][n], ph.z, qh.z, ph.w, qh.w, xh[n].z, xh[n].w);
                    }
                }
        } else {
#pragma unroll
            for (int b = 0; b < MATS; b++)
#pragma unroll
                for (int a = 0; a < MT; a++)
#pragma unroll
                    for (int n = 0; n < XP * NT; n++) {
                        const uint4 lo = wv[b][a][0], hi = wv[b][a][1], y = xv[n];
                        few_mma(acc[b][a][n % NT], lo.x, hi.x, lo.y, hi.y, y.x, y.y);
                        few_mma(acc[b][a][n % NT], lo.z, hi.z, lo.w, hi.w, y.z, y.w);
                    }
        }
    };
    constexpr int ACCS = MATS * MT * NT * 4;
    float total[F32 ? ACCS : 1];
#pragma unroll
    for (int a = 0; a < (F32 ? ACCS : 1); a++) total[a] = 0.f;
    auto settle = [&]() {
        if constexpr (F32) {
#pragma unroll
            for (int a = 0; a < ACCS; a++) { total[a] += (&acc[0][0][0][0])[a]; (&acc[0][0][0][0])[a] = 0.f; }
        }
    };
    int k0 = 0;
    constexpr int UT = ALIGN == 16 ? KIND != FEW_F16 ? 1 : MT * MATS == 1 ? U : 2 : MT * MATS == 1 ? 4 : 2;        // (pieces under way where a row ends)
    if constexpr (ALIGN == 16) {
        for (; k0 + WARPS * PIECE * U <= p.K; k0 += WARPS * PIECE * U) {
            uint4 wv[U][MATS][MT][2], xv[U][XP * NT];
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int k = k0 + (i * WARPS + warp) * PIECE + t * N;
#pragma unroll
                for (int b = 0; b < MATS; b++)
#pragma unroll
                    for (int a = 0; a < MT; a++)
#pragma unroll
                        for (int h = 0; h < 2; h++) wv[i][b][a][h] = few_stream(wp[b][a][h] + k);
            }
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int n = 0; n < XP * NT; n++) xv[i][n] = few_keep(xp[n % NT] + (n < NT ? 0 : rest) + k0 + (i * WARPS + warp) * PIECE + t * N);
#pragma unroll
            for (int i = 0; i < U; i++) multiply(wv[i], xv[i]);
            settle();
        }
    } else if (p.words && p.K > WARPS * PIECE * (F32 ? UT : 1)) {             // (shorter rows: the loop below has them under way at once)
        constexpr int WORD = 4 / (int)sizeof(E);             // (the fifth word of a piece is the row's too)
        const int last = p.K - PIECE - WORD;                 // where a piece may start at most; what lies behind is left to the loop below
        auto turn = [&](auto part) {
            constexpr bool PART = decltype(part)::value;
            FewRaw wr[U][MATS][MT][2], xr[U][XP * NT];
            const int first = k0 + warp * PIECE;
#pragma unroll
            for (int i = 0; i < U; i++) {
                if (PART && first + i * WARPS * PIECE > last) continue;
                const int k = first + i * WARPS * PIECE + t * N;
#pragma unroll
                for (int b = 0; b < MATS; b++)
#pragma unroll
                    for (int a = 0; a < MT; a++)
#pragma unroll
                        for (int h = 0; h < 2; h++) wr[i][b][a][h] = few_raw(wp[b][a][h] + k, false);
#pragma unroll
                for (int n = 0; n < XP * NT; n++) xr[i][n] = few_raw(xp[n % NT] + (n < NT ? 0 : rest) + k, p.x16);
            }
#pragma unroll
            for (int i = 0; i < U; i++) {
                if (PART && first + i * WARPS * PIECE > last) continue;
                uint4 wv[MATS][MT][2], xv[XP * NT];
#pragma unroll
                for (int b = 0; b < MATS; b++)
#pragma unroll
                    for (int a = 0; a < MT; a++)
#pragma unroll
                        for (int h = 0; h < 2; h++) wv[b][a][h] = few_place(wr[i][b][a][h], wp[b][a][h]);
#pragma unroll
                for (int n = 0; n < XP * NT; n++) xv[n] = few_place(xr[i][n], xp[n % NT] + (n < NT ? 0 : rest));
                multiply(wv, xv);
            }
            settle();
        };
        for (; k0 + (WARPS * U - 1) * PIECE <= last; k0 += WARPS * PIECE * U) turn(std::false_type{});
        if (k0 <= last) turn(std::true_type{});
        k0 = last < 0 ? 0 : (last / PIECE + 1) * PIECE;      // the one or two pieces behind
    }
    for (; k0 < p.K; k0 += WARPS * PIECE * UT) {
        uint4 wv[UT][MATS][MT][2], xv[UT][XP * NT];
#pragma unroll
        for (int i = 0; i < UT; i++) {
            const int k = k0 + (i * WARPS + warp) * PIECE + t * N;
#pragma unroll
            for (int b = 0; b < MATS; b++)
#pragma unroll
                for (int a = 0; a < MT; a++)
#pragma unroll
                    for (int h = 0; h < 2; h++) wv[i][b][a][h] = few_load<E, ALIGN>(wp[b][a][h], k, p.K);
#pragma unroll
            for (int n = 0; n < XP * NT; n++) xv[i][n] = few_load<E, ALIGN>(xp[n % NT] + (n < NT ? 0 : rest), k, p.K);
        }
#pragma unroll
        for (int i = 0; i < UT; i++) multiply(wv[i], xv[i]);
        settle();
    }
#pragma unroll
    for (int a = 0; a < MATS * MT * NT * 4; a++) { if constexpr (F32) red[warp][a][lane] = total[a]; else red[warp][a][lane] = (&acc[0][0][0][0])[a]; }
    __syncthreads();
    // accumulator c of lane (g, t): weight row g + 8 (c / 2), token 2 t + c % 2
    for (int e = threadIdx.x; e < MT * 16 * NT * 8; e += 32 * WARPS) {
        const int m = e % (MT * 16), n = e / (MT * 16);
        if (n >= p.rows || m0 + m >= p.M) continue;
        const int a = m / 16, r = m % 16, src = (r % 8) * 4 + (n % 8) / 2, c = (r / 8) * 2 + n % 2;
        S v = 0, w = 0;
#pragma unroll
        for (int k = 0; k < WARPS; k++) {
            v += red[k][(a * NT + n / 8) * 4 + c][src];
            if constexpr (MATS == 2) w += red[k][((MT + a) * NT + n / 8) * 4 + c][src];
        }
        few_result<T, EPI, S>(p, n, m0 + m, v, w);
    }
}

// Single precision, up to four tokens, on FFMA: R rows of each matrix per CTA, its warps share K, lanes along it.  V: elements per load.  Whole blocks, both products,
// weights from memory, FFMA against the tensor cores in us:  one token 3.4 / 5.1 (512 x 512 x 512), 8.6 / 11.0 (1024 x 2048 x 1024), 12.5 / 19.1 (1000 x 2731 x 1000),
// 32.2 / 37.9 (2048 x 5632 x 2048), 44.4 / 44.7 (4096 x 4096 x 4096).  Two to four tokens, which cost the same: 4.0 / 5.3, 12.6 / 11.1, 21.7 / 19.2, 51.8 / 38.1,
// 62.0 / 44.5, and 7.0 / 9.9 (257 x 1001 x 257), 10.6 / 10.3 (640 x 1712 x 640), 15.5 / 16.3 (1000 x 2736 x 1000): the bound of four is right for weights of up to
// some 10 MB that fit a wave or two of CTAs, and too high for larger ones by up to 1.4 times.
template <int EPI, int NT, int R, int V>
__global__ void __launch_bounds__(256) few_rows_fp32_kernel(const __grid_constant__ FewParams<float> p)
{
    pdl_wait();
    constexpr int MATS = EPI == FFN_GATE ? 2 : 1;
    __shared__ float red[8][MATS * R * NT];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m0 = blockIdx.x * R;
    const float *x = reinterpret_cast<const float *>(p.x);
    float acc[MATS][R][NT];
#pragma unroll
    for (int a = 0; a < MATS * R * NT; a++) (&acc[0][0][0])[a] = 0.f;
#pragma unroll 2
    for (int k = threadIdx.x * V; k < p.K; k += 256 * V) {
        float wv[MATS][R][V], xv[NT][V];
        auto load = [&](const float *row, bool live, float (&v)[V]) {
            if constexpr (V == 4) {
                const float4 q = live ? *reinterpret_cast<const float4 *>(row + k) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
            } else v[0] = live ? row[k] : 0.f;
        };
#pragma unroll
        for (int b = 0; b < MATS; b++)
#pragma unroll
            for (int r = 0; r < R; r++) load(reinterpret_cast<const float *>(p.w[b]) + (long long)(m0 + r) * p.K, m0 + r < p.M, wv[b][r]);
#pragma unroll
        for (int n = 0; n < NT; n++) load(x + n * p.x_stride, n < p.rows, xv[n]);
#pragma unroll
        for (int b = 0; b < MATS; b++)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int v = 0; v < V; v++) acc[b][r][n] = fmaf(wv[b][r][v], xv[n][v], acc[b][r][n]);
    }
#pragma unroll
    for (int a = 0; a < MATS * R * NT; a++) {
        const float s = warp_sum((&acc[0][0][0])[a]);
        if (lane == 0) red[warp][a] = s;
    }
    __syncthreads();
    const int e = threadIdx.x;
    if (e >= R * NT) return;
    const int r = e % R, n = e / R;
    if (n >= p.rows || m0 + r >= p.M) return;
    float v = 0.f, w = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        v += red[k][r * NT + n];
        if constexpr (MATS == 2) w += red[k][(R + r) * NT + n];
    }
    few_result<float, EPI, float>(p, n, m0 + r, v, w);
}

template <int KIND, class T, int EPI, int NT, int MT, int ALIGN> static void few_launch(const FewParams<T> &p)
{
    // fewer CTAs than SMs: twice the warps for each
    const int ctas = ceil_div(p.M, 16 * MT);
    constexpr int W = NT * MT * (EPI == FFN_GATE ? 2 : 1) <= 4 ? 16 : 8;           // (their sums fit the shared memory)
    if (ctas <= sm_count() && W == 16) TL_LAUNCH((few_rows_kernel<KIND, T, EPI, NT, MT, ALIGN, W>), ctas, 32 * W, 0, p);
    else TL_LAUNCH((few_rows_kernel<KIND, T, EPI, NT, MT, ALIGN, 8>), ctas, 256, 0, p);
}
template <int KIND, class T, int EPI, int ALIGN> static void few_tokens(const FewParams<T> &p)
{
    const int nt = ceil_div(p.rows, 8);
    const bool wide = EPI != FFN_GATE && p.M > 32 * sm_count();
    constexpr int WIDE = EPI != FFN_GATE ? 2 : 1;
    if (nt == 1) few_launch<KIND, T, EPI, 1, 1, ALIGN>(p);
    else if (nt == 2) few_launch<KIND, T, EPI, 2, 1, ALIGN>(p);
    else if (nt == 3) { if (wide) few_launch<KIND, T, EPI, 3, WIDE, ALIGN>(p); else few_launch<KIND, T, EPI, 3, 1, ALIGN>(p); }
    else if (wide) few_launch<KIND, T, EPI, 4, WIDE, ALIGN>(p);
    else few_launch<KIND, T, EPI, 4, 1, ALIGN>(p);
}
template <int KIND, class T, int EPI> static void few_aligned(const FewParams<T> &p, int esize)
{
    const uintptr_t at = (uintptr_t)p.x | (uintptr_t)p.x2 | (uintptr_t)p.w[0] | (uintptr_t)(EPI == FFN_GATE ? p.w[1] : nullptr) | (uintptr_t)((long long)p.K * esize) | (uintptr_t)(p.x_stride * esize);
    if (at % 16 == 0) return few_tokens<KIND, T, EPI, 16>(p);
    FewParams<T> q = p;
    q.words = (((uintptr_t)p.x | (uintptr_t)p.x2 | (uintptr_t)p.w[0] | (uintptr_t)(EPI == FFN_GATE ? p.w[1] : nullptr)) & 3) == 0;
    q.x16 = (((uintptr_t)p.x | (uintptr_t)p.x2 | (uintptr_t)(p.x_stride * esize)) & 15) == 0;
    few_tokens<KIND, T, EPI, 1>(q);
}
template <int EPI> static void few_fp32(const FewParams<float> &p)
{
    constexpr int R = EPI == FFN_GATE ? 2 : 4;
    const bool wide = (((uintptr_t)p.x | (uintptr_t)p.w[0] | (uintptr_t)(EPI == FFN_GATE ? p.w[1] : nullptr)) & 15) == 0 && p.K % 4 == 0 && p.x_stride % 4 == 0;
#define TL_FEW32(NT, V) TL_LAUNCH((few_rows_fp32_kernel<EPI, NT, R, V>), ceil_div(p.M, R), 256, 0, p)
    if (wide) { if (p.rows == 1) TL_FEW32(1, 4); else TL_FEW32(4, 4); }
    else { if (p.rows == 1) TL_FEW32(1, 1); else TL_FEW32(4, 1); }
#undef TL_FEW32
}

template <class T, int EPI> void few_rows_mm(Scope &, const FfnProduct<T> &f, long long c_stride, const T *x2, T *c2)
{
    FewParams<T> p = {};
    p.x = f.A[0]; p.w[0] = f.B[0]; p.w[1] = f.B[1]; p.C = f.C; p.g = f.g; p.u = f.u; p.rows = f.N; p.M = f.M; p.K = f.K; p.x_stride = f.a_rs; p.c_stride = c_stride; p.x2 = x2; p.C2 = c2;
    if constexpr (sizeof(T) == 2) few_aligned<FEW_F16, T, EPI>(p, 2);
    else if (p.rows <= 4) few_fp32<EPI>(p);
    else few_aligned<FEW_F32, T, EPI>(p, 4);
}
template <class T> void few_rows_int8(Scope &, const signed char *x, const float *xs, const signed char *w, const float *ws, const T *bias, T *y, int rows, int in, int out)
{
    FewParams<T> p = {};
    p.x = x; p.w[0] = w; p.C = y; p.bias = bias; p.xs = xs; p.ws = ws; p.rows = rows; p.M = out; p.K = in; p.x_stride = in; p.c_stride = out;
    few_aligned<FEW_I8, T, FFN_INT8>(p, 1);
}
#define INST(T)                                                                 \
    template void few_rows_mm<T, FFN_PLAIN>(Scope &, const FfnProduct<T> &, long long, const T *, T *);  \
    template void few_rows_mm<T, FFN_GATE>(Scope &, const FfnProduct<T> &, long long, const T *, T *);   \
    template void few_rows_int8<T>(Scope &, const signed char *, const float *, const signed char *, const float *, const T *, T *, int, int, int);
INST(float)
INST(__half)

} // namespace tl
