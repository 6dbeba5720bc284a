// Gated feed-forward block and its backward pass:
//   G = X Wg^T, U = X Wu^T, H = silu(G) * U, Y = H Wd^T
//   dH = dY Wd;  with s = 1 / (1 + exp(-G)), a = G s:  dU = dH a,  dG = dH U (s + a (1 - s));
//   dX = dG Wg + dU Wu,  dWg = dG^T X,  dWu = dU^T X,  dWd = dY^T H
// Two of its products have an epilogue of their own: the pair G, U (the gate, the product and H leave with it) and dH (G and U come in,
// dG, dU and H leave).  The others are plain products.
#include "tl_gate.cuh"
#include <algorithm>

namespace tl {

// H alone, for a backward pass of which only dWd is wanted: the operations of the products' epilogues
template <class T> __global__ void __launch_bounds__(256) gate_kernel(const T *__restrict__ g, const T *__restrict__ u, T *__restrict__ h, int rows, int size, int pitch)
{
    pdl_wait();
    for (int r = blockIdx.y; r < rows; r += gridDim.y)
        for (int i = blockIdx.x * 256 + threadIdx.x; i < size; i += gridDim.x * 256) {
            const size_t at = (size_t)r * size + i;
            st(h + (size_t)r * pitch + i, gate_fw<sizeof(T) == 2>(ld(g + at), ld(u + at)));
        }
}
// elements between the rows of H and of its gradients: whole lines of 128 bytes, so that the products read them where they are and in whole lines
template <class T> static int ffn_pitch(int hidden) { constexpr int E = 128 / (int)sizeof(T); return (hidden + E - 1) / E * E; }

template <class T> void gated_ffn_fw(Scope &sc, const GatedFfn<T> &f)
{
    // few tokens: H in half precision with what its rounding left beside it
    const bool few = f.rows <= FEW_ROWS, two = sizeof(T) == 2 && f.rows <= FEW_TWO;
    const int pitch = ffn_pitch<T>(f.hidden);
    T *h = sc.scratch<T>((size_t)f.rows * pitch), *rest = two ? sc.scratch<T>((size_t)f.rows * pitch) : nullptr;
    if (!h || (two && !rest)) return;
    FfnProduct<T> p = {};
    p.A[0] = f.x; p.B[0] = f.wg; p.B[1] = f.wu; p.C = h; p.g = f.g; p.u = f.u; p.N = f.rows; p.M = f.hidden; p.K = f.in; p.terms = 1;
    p.a_rs = f.in; p.a_cs = 1; p.b_rs = 1; p.b_cs = f.in; p.ld = pitch;
    if (few) few_rows_mm<T, FFN_GATE>(sc, p, pitch, nullptr, rest);
    else if (!block_mm<T, FFN_GATE>(sc, &p, 1)) return;
    FfnProduct<T> d = {};
    d.A[0] = h; d.B[0] = f.wd; d.C = f.y; d.N = f.rows; d.M = f.out; d.K = f.hidden; d.terms = 1;
    d.a_rs = pitch; d.a_cs = 1; d.b_rs = 1; d.b_cs = f.hidden; d.ld = f.out;
    if (few) few_rows_mm<T, FFN_PLAIN>(sc, d, f.out, rest, nullptr);
    else block_mm<T, FFN_PLAIN>(sc, &d, 1);
}
template <class T> void gated_ffn_bw(Scope &sc, const GatedFfn<T> &f)
{
    const int pitch = ffn_pitch<T>(f.hidden);
    const size_t n = (size_t)f.rows * pitch;
    T *h = sc.scratch<T>(n), *dg = sc.scratch<T>(n), *du = sc.scratch<T>(n);
    if (!h || !dg || !du) return;
    FfnProduct<T> p = {};
    p.A[0] = f.dy; p.B[0] = f.wd; p.C = h; p.g = f.g; p.u = f.u; p.dg = dg; p.du = du; p.N = f.rows; p.M = f.hidden; p.terms = 1;
    p.K = f.out; p.a_rs = f.out; p.a_cs = 1; p.b_rs = f.hidden; p.b_cs = 1; p.ld = pitch;
    if (!f.dx && !f.dwg && !f.dwu) TL_LAUNCH((gate_kernel<T>), dim3(std::min(ceil_div(f.hidden, 256), 64), std::min(f.rows, 4096)), 256, 0, f.g, f.u, h, f.rows, f.hidden, pitch);
    else if (!block_mm<T, FFN_GATE_BW>(sc, &p, 1)) return;
    // the gradients that are wanted, in one launch
    FfnProduct<T> list[4];
    int count = 0;
    if (f.dx) {
        FfnProduct<T> &d = list[count++] = {};
        d.A[0] = dg; d.A[1] = du; d.B[0] = f.wg; d.B[1] = f.wu; d.C = f.dx; d.N = f.rows; d.M = f.in; d.K = f.hidden; d.terms = 2;
        d.a_rs = pitch; d.a_cs = 1; d.b_rs = f.in; d.b_cs = 1; d.ld = f.in;
    }
    auto weights = [&](const T *left, int l_rows, const T *right, int r_rows, T *dw, int N, int M) {
        if (!dw) return;
        FfnProduct<T> &d = list[count++] = {};
        d.A[0] = left; d.B[0] = right; d.C = dw; d.N = N; d.M = M; d.K = f.rows; d.terms = 1;
        d.a_rs = 1; d.a_cs = l_rows; d.b_rs = r_rows; d.b_cs = 1; d.ld = M;
    };
    weights(dg, pitch, f.x, f.in, f.dwg, f.hidden, f.in);
    weights(du, pitch, f.x, f.in, f.dwu, f.hidden, f.in);
    weights(f.dy, f.out, h, pitch, f.dwd, f.out, f.hidden);
    block_mm<T, FFN_PLAIN>(sc, list, count);
}
template void gated_ffn_fw<float>(Scope &, const GatedFfn<float> &);
template void gated_ffn_fw<__half>(Scope &, const GatedFfn<__half> &);
template void gated_ffn_bw<float>(Scope &, const GatedFfn<float> &);
template void gated_ffn_bw<__half>(Scope &, const GatedFfn<__half> &);

} // namespace tl
