// The gate of the feed-forward block, and the products around it as their kernels take them.
#pragma once
#include "tl_kernels.h"

namespace tl {

// s = 1 / (1 + exp(-g)).  For half-precision results the hardware's power of two and reciprocal do (their few units of 2^-23, growing with |g| to some
// thirty at the |g| where s is no longer 0 or 1 to eleven bits), without subnormal numbers, which are nothing beside 1 and in a result of half precision;
// both ends of the range are right: exp(-g) = inf gives 0.
template <bool FAST> __device__ __forceinline__ float gate_sigmoid(float g)
{
    if constexpr (FAST) {
        float e, s;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
        return s;
    }
    else return 1.f / (1.f + expf(-g));
}
template <bool FAST> __device__ __forceinline__ float gate_fw(float g, float u) { return g * gate_sigmoid<FAST>(g) * u; }
template <bool FAST> __device__ __forceinline__ void gate_bw(float g, float u, float dh, float &h, float &dg, float &du)
{
    const float s = gate_sigmoid<FAST>(g), a = g * s;
    h = a * u;
    du = dh * a;
    dg = dh * u * fmaf(a, 1.f - s, s);
}

// C(i, j) = sum_k A(i, k) B(k, j), i < N, j < M, k < K; A(i, k) = A[i * a_rs + k * a_cs], B(k, j) = B[k * b_rs + j * b_cs],
// C, dg and du in rows of ld elements (padding is written where ld covers it), g and u dense.
//   FFN_PLAIN: C = the sum over `terms` (1 or 2) pairs of operands;  FFN_GATE: g, u (may be null) = A[0] with B[0] and B[1], C = silu(g) * u;
//   FFN_GATE_BW: dH = A[0] B[0]; reads g and u, writes C = silu(g) * u and their gradients dg, du
enum { FFN_PLAIN = 0, FFN_GATE = 1, FFN_GATE_BW = 2, FFN_INT8 = 3 };
template <class T> struct FfnProduct {
    const T *A[2], *B[2];
    T *C, *g, *u, *dg, *du;
    int N, M, K, terms, ld;
    long long a_rs, a_cs, b_rs, b_cs;
};
// On the tensor cores (tl_block_mm.cu); false: nothing launched, the error is set (no memory for an operand's copy, no tensor-map encoder)
// FFN_PLAIN: up to four products in one launch, none of which may write what another one reads.
template <class T, int EPI> bool block_mm(Scope &sc, const FfnProduct<T> *list, int count);
// Few tokens (FEW_ROWS at most), weights with K contiguous (tl_few_rows.cu): FFN_PLAIN of one term and FFN_GATE.  c_stride: elements between the
// rows of C.  Half precision, FEW_TWO tokens at most: FFN_GATE leaves what rounding C left in c2, FFN_PLAIN adds the product of x2 with the
// same weights.
static constexpr int FEW_ROWS = 32, FEW_TWO = 8;
template <class T, int EPI> void few_rows_mm(Scope &sc, const FfnProduct<T> &p, long long c_stride, const T *x2, T *c2);
template <class T> void few_rows_int8(Scope &sc, const signed char *x, const float *xs, const signed char *w, const float *ws, const T *bias, T *y, int rows, int in, int out);

} // namespace tl
