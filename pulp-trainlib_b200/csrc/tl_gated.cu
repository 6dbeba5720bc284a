// Gated feed-forward block and its backward pass:
//   G = X Wg^T, U = X Wu^T, H = silu(G) * U, Y = H Wd^T
//   dH = dY Wd;  with s = 1 / (1 + exp(-G)), a = G s:  dU = dH a,  dG = dH U (s + a (1 - s));
//   dX = dG Wg + dU Wu,  dWg = dG^T X,  dWu = dU^T X,  dWd = dY^T H
// Two of its products have an epilogue of their own: the pair G, U (the gate, the product and H leave with it) and dH (G and U come in,
// dG, dU and H leave).  The others are plain products.
#include "tl_kernels.h"

namespace tl {

// ---------------------------------------------------------------- the gate
__device__ __forceinline__ float gate_sigmoid(float g) { return 1.f / (1.f + expf(-g)); }
__device__ __forceinline__ float gate_fw(float g, float u) { return g * gate_sigmoid(g) * u; }
__device__ __forceinline__ void gate_bw(float g, float u, float dh, float &h, float &dg, float &du)
{
    const float s = gate_sigmoid(g), a = g * s;
    h = a * u;
    du = dh * a;
    dg = dh * u * fmaf(a, 1.f - s, s);
}

// ---------------------------------------------------------------- products on CUDA cores
// C(i, j) = sum_k A(i, k) B(k, j) on 64 x 64 tiles with any strides; a thread has 4 x 4 results.
enum { FFN_PLAIN = 0, FFN_GATE = 1, FFN_GATE_BW = 2 };
template <class T> struct FfnProduct {
    const T *A[2], *B[2];           // FFN_PLAIN: up to two products that are added; FFN_GATE: A[0] with both B
    T *C, *g, *u, *dg, *du;
    int N, M, K, terms;
    long long a_rs, a_cs, b_rs, b_cs, c_rs;
};
template <class T, int EPI>
__global__ void __launch_bounds__(256) ffn_product_kernel(const __grid_constant__ FfnProduct<T> p)
{
    pdl_wait();
    constexpr int NB = EPI == FFN_GATE ? 2 : 1;
    __shared__ float As[16][65], Bs[NB][16][65];
    const int row0 = blockIdx.y * 64, col0 = blockIdx.x * 64, tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    float acc[NB][4][4] = {};
    for (int term = 0; term < p.terms; term++)
        for (int k0 = 0; k0 < p.K; k0 += 16) {
            for (int e = threadIdx.x; e < 1024; e += 256) {
                // neighbouring threads read along the index that is contiguous
                const int ia = p.a_cs == 1 ? e / 16 : e % 64, ka = p.a_cs == 1 ? e % 16 : e / 64;
                As[ka][ia] = ld0(row0 + ia < p.N && k0 + ka < p.K, p.A[term] + (row0 + ia) * p.a_rs + (k0 + ka) * p.a_cs);
                const int jb = p.b_rs == 1 ? e / 16 : e % 64, kb = p.b_rs == 1 ? e % 16 : e / 64;
#pragma unroll
                for (int b = 0; b < NB; b++)
                    Bs[b][kb][jb] = ld0(col0 + jb < p.M && k0 + kb < p.K, p.B[EPI == FFN_GATE ? b : term] + (k0 + kb) * p.b_rs + (col0 + jb) * p.b_cs);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 16; k++) {
                float a[4];
#pragma unroll
                for (int i = 0; i < 4; i++) a[i] = As[k][tr + 16 * i];
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float v = Bs[b][k][tc + 16 * j];
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[b][i][j] = fmaf(a[i], v, acc[b][i][j]);
                    }
            }
            __syncthreads();
        }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = row0 + tr + 16 * i, col = col0 + tc + 16 * j;
            if (row >= p.N || col >= p.M) continue;
            const long long at = row * p.c_rs + col;
            if (EPI == FFN_PLAIN) st(p.C + at, acc[0][i][j]);
            else if (EPI == FFN_GATE) {
                if (p.g) { st(p.g + at, acc[0][i][j]); st(p.u + at, acc[NB - 1][i][j]); }
                st(p.C + at, gate_fw(acc[0][i][j], acc[NB - 1][i][j]));
            } else {
                float h, dg, du;
                gate_bw(ld(p.g + at), ld(p.u + at), acc[0][i][j], h, dg, du);
                st(p.C + at, h); st(p.dg + at, dg); st(p.du + at, du);
            }
        }
}
template <class T, int EPI> static void ffn_product(const FfnProduct<T> &p)
{
    TL_LAUNCH((ffn_product_kernel<T, EPI>), dim3(ceil_div(p.M, 64), ceil_div(p.N, 64)), 256, 0, p);
}

template <class T> void gated_ffn_fw(Scope &sc, const GatedFfn<T> &f)
{
    T *h = sc.scratch<T>((size_t)f.rows * f.hidden);
    if (!h) return;
    FfnProduct<T> p = {};
    p.A[0] = f.x; p.B[0] = f.wg; p.B[1] = f.wu; p.C = h; p.g = f.g; p.u = f.u; p.N = f.rows; p.M = f.hidden; p.K = f.in; p.terms = 1;
    p.a_rs = f.in; p.a_cs = 1; p.b_rs = 1; p.b_cs = f.in; p.c_rs = f.hidden;
    ffn_product<T, FFN_GATE>(p);
    FfnProduct<T> d = {};
    d.A[0] = h; d.B[0] = f.wd; d.C = f.y; d.N = f.rows; d.M = f.out; d.K = f.hidden; d.terms = 1;
    d.a_rs = f.hidden; d.a_cs = 1; d.b_rs = 1; d.b_cs = f.hidden; d.c_rs = f.out;
    ffn_product<T, FFN_PLAIN>(d);
}
template <class T> void gated_ffn_bw(Scope &sc, const GatedFfn<T> &f)
{
    const size_t n = (size_t)f.rows * f.hidden;
    T *h = sc.scratch<T>(n), *dg = sc.scratch<T>(n), *du = sc.scratch<T>(n);
    if (!h || !dg || !du) return;
    FfnProduct<T> p = {};
    p.A[0] = f.dy; p.B[0] = f.wd; p.C = h; p.g = f.g; p.u = f.u; p.dg = dg; p.du = du; p.N = f.rows; p.M = f.hidden; p.terms = 1;
    p.K = f.dx || f.dwg || f.dwu ? f.out : 0;            // only dWd is wanted: H alone, Wd need not be there
    p.a_rs = f.out; p.a_cs = 1; p.b_rs = f.hidden; p.b_cs = 1; p.c_rs = f.hidden;
    ffn_product<T, FFN_GATE_BW>(p);
    if (f.dx) {
        FfnProduct<T> d = {};
        d.A[0] = dg; d.A[1] = du; d.B[0] = f.wg; d.B[1] = f.wu; d.C = f.dx; d.N = f.rows; d.M = f.in; d.K = f.hidden; d.terms = 2;
        d.a_rs = f.hidden; d.a_cs = 1; d.b_rs = f.in; d.b_cs = 1; d.c_rs = f.in;
        ffn_product<T, FFN_PLAIN>(d);
    }
    auto weights = [&](const T *left, const T *right, T *dw, int N, int M) {
        if (!dw) return;
        FfnProduct<T> d = {};
        d.A[0] = left; d.B[0] = right; d.C = dw; d.N = N; d.M = M; d.K = f.rows; d.terms = 1;
        d.a_rs = 1; d.a_cs = N; d.b_rs = M; d.b_cs = 1; d.c_rs = M;
        ffn_product<T, FFN_PLAIN>(d);
    };
    weights(dg, f.x, f.dwg, f.hidden, f.in);
    weights(du, f.x, f.dwu, f.hidden, f.in);
    weights(f.dy, h, f.dwd, f.out, f.hidden);
}
template void gated_ffn_fw<float>(Scope &, const GatedFfn<float> &);
template void gated_ffn_fw<__half>(Scope &, const GatedFfn<__half> &);
template void gated_ffn_bw<float>(Scope &, const GatedFfn<float> &);
template void gated_ffn_bw<__half>(Scope &, const GatedFfn<__half> &);

} // namespace tl
