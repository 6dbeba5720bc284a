// Entry points of the feed-forward half of a transformer block: RMS norm of a residual sum, gated feed-forward block, linear layer in
// 8-bit integers.  Same conventions as the other entry points: host pointers are staged, device pointers pass through, errors latch.
#include "tl_kernels.h"
#include <algorithm>

using namespace tl;

namespace {

#define TL_REQUIRE(cond, ...)                                        \
    do { if (!(cond)) { set_error(TL_ERR_BAD_ARGS, __VA_ARGS__); return; } } while (0)

// The kernels' indices are 32 bits wide and run up to a few thousand beyond a size.
bool sizes_fit(const char *what, int a, int b)
{
    const int largest = std::max(a, b);
    if (largest <= 1 << 30) return true;
    set_error(TL_ERR_TOO_LARGE, "%s: a size of %d, 2^30 at most", what, largest);
    return false;
}

template <class T> void rmsnorm_fw_impl(void *args, bool int8)
{
    auto *a = (trainlib_rmsnorm_args *)args;
    TL_REQUIRE(a && a->rows > 0 && a->size > 0, "trainlib_rmsnorm: rows=%d size=%d", a ? a->rows : 0, a ? a->size : 0);
    TL_REQUIRE(a->x && a->weight && (int8 ? a->q && a->scale : a->output != nullptr), "trainlib_rmsnorm: null x, weight or output");
    if (!sizes_fit("trainlib_rmsnorm", a->rows, a->size)) return;
    Scope sc;
    const size_t n = (size_t)a->rows * a->size;
    const T *x = sc.in((T *)a->x, n), *res = sc.in((T *)a->residual, n), *w = sc.in((T *)a->weight, (size_t)a->size);
    T *sum = sc.out((T *)a->sum, n);
    if (int8) {
        signed char *q = sc.out(a->q, n);
        float *scale = sc.out(a->scale, (size_t)a->rows);
        if (sc.ok()) rmsnorm_int8_fw<T>(x, res, w, sum, q, scale, a->rows, a->size, a->eps);
    } else {
        T *y = sc.out((T *)a->output, n);
        if (sc.ok()) rmsnorm_fw<T>(x, res, w, sum, y, a->rows, a->size, a->eps);
    }
}
template <class T> void rmsnorm_bw_impl(void *args)
{
    auto *a = (trainlib_rmsnorm_args *)args;
    TL_REQUIRE(a && a->rows > 0 && a->size > 0, "trainlib_rmsnorm: rows=%d size=%d", a ? a->rows : 0, a ? a->size : 0);
    TL_REQUIRE(a->sum && a->weight && a->dy && (a->dx || a->dweight), "trainlib_rmsnorm: backward needs sum, weight, dy and a gradient to write");
    if (!sizes_fit("trainlib_rmsnorm", a->rows, a->size)) return;
    Scope sc;
    const size_t n = (size_t)a->rows * a->size;
    const T *h = sc.in((T *)a->sum, n), *w = sc.in((T *)a->weight, (size_t)a->size), *dy = sc.in((T *)a->dy, n), *dsum = sc.in((T *)a->dsum, n);
    T *dx = sc.out((T *)a->dx, n), *dw = sc.out((T *)a->dweight, (size_t)a->size);
    if (!sc.ok()) return;
    defer_settle(dw);
    rmsnorm_bw<T>(sc, h, w, dy, dsum, dx, dw, a->rows, a->size, a->eps);
}
template <class T> void quantize_rows_impl(void *args)
{
    auto *a = (trainlib_quantize_rows_args *)args;
    TL_REQUIRE(a && a->rows > 0 && a->size > 0 && a->x && a->q && a->scale, "trainlib_quantize_rows: rows=%d size=%d or a null pointer", a ? a->rows : 0, a ? a->size : 0);
    if (!sizes_fit("trainlib_quantize_rows", a->rows, a->size)) return;
    Scope sc;
    const size_t n = (size_t)a->rows * a->size;
    const T *x = sc.in((T *)a->x, n);
    signed char *q = sc.out(a->q, n);
    float *scale = sc.out(a->scale, (size_t)a->rows);
    if (sc.ok()) quantize_rows<T>(x, q, scale, a->rows, a->size);
}
template <class T> void linear_int8_impl(void *args)
{
    auto *a = (trainlib_linear_int8_args *)args;
    TL_REQUIRE(a && a->rows > 0 && a->in_size > 0 && a->out_size > 0, "trainlib_linear_int8: rows=%d in_size=%d out_size=%d", a ? a->rows : 0, a ? a->in_size : 0, a ? a->out_size : 0);
    TL_REQUIRE(a->x && a->x_scale && a->weight && a->w_scale && a->y, "trainlib_linear_int8: null operand, scale or output");
    if (!sizes_fit("trainlib_linear_int8", a->rows, a->out_size)) return;
    if (a->in_size > 131071) { set_error(TL_ERR_TOO_LARGE, "trainlib_linear_int8: in_size = %d, sums of more than 131071 products pass 32 bits", a->in_size); return; }
    Scope sc;
    const signed char *x = sc.in(a->x, (size_t)a->rows * a->in_size), *w = sc.in(a->weight, (size_t)a->out_size * a->in_size);
    const float *xs = sc.in(a->x_scale, (size_t)a->rows), *ws = sc.in(a->w_scale, (size_t)a->out_size);
    const T *bias = sc.in((T *)a->bias, (size_t)a->out_size);
    T *y = sc.out((T *)a->y, (size_t)a->rows * a->out_size);
    if (sc.ok()) linear_int8<T>(sc, x, xs, w, ws, bias, y, a->rows, a->in_size, a->out_size);
}
template <class T> bool gated_ffn_sizes(trainlib_gated_ffn_args *a)
{
    if (a && a->rows > 0 && a->in_size > 0 && a->hidden > 0 && a->out_size > 0) {
        return sizes_fit("trainlib_gated_ffn", std::max(a->rows, a->in_size), std::max(a->hidden, a->out_size));
    }
    set_error(TL_ERR_BAD_ARGS, "trainlib_gated_ffn: rows=%d in_size=%d hidden=%d out_size=%d", a ? a->rows : 0, a ? a->in_size : 0, a ? a->hidden : 0, a ? a->out_size : 0);
    return false;
}
template <class T> void gated_ffn_fw_impl(void *args)
{
    auto *a = (trainlib_gated_ffn_args *)args;
    if (!gated_ffn_sizes<T>(a)) return;
    TL_REQUIRE(a->x && a->w_gate && a->w_up && a->w_down && a->y && !a->gate == !a->up, "trainlib_gated_ffn: null x, weight or output, or one of gate and up without the other");
    Scope sc;
    const size_t nx = (size_t)a->rows * a->in_size, nw = (size_t)a->hidden * a->in_size, nh = (size_t)a->rows * a->hidden;
    GatedFfn<T> f = {};
    f.rows = a->rows; f.in = a->in_size; f.hidden = a->hidden; f.out = a->out_size;
    f.x = sc.in((T *)a->x, nx); f.wg = sc.in((T *)a->w_gate, nw); f.wu = sc.in((T *)a->w_up, nw); f.wd = sc.in((T *)a->w_down, (size_t)a->out_size * a->hidden);
    f.g = sc.out((T *)a->gate, nh); f.u = sc.out((T *)a->up, nh); f.y = sc.out((T *)a->y, (size_t)a->rows * a->out_size);
    if (sc.ok()) gated_ffn_fw<T>(sc, f);
}
template <class T> void gated_ffn_bw_impl(void *args)
{
    auto *a = (trainlib_gated_ffn_args *)args;
    if (!gated_ffn_sizes<T>(a)) return;
    const bool wide = a->dx || a->dw_gate || a->dw_up;
    TL_REQUIRE(a->dy && a->gate && a->up && (wide || a->dw_down), "trainlib_gated_ffn: backward needs dy, gate, up and a gradient to write");
    TL_REQUIRE((!wide || a->w_down) && (!a->dx || (a->w_gate && a->w_up)) && (!(a->dw_gate || a->dw_up) || a->x), "trainlib_gated_ffn: an operand of a wanted gradient is null");
    Scope sc;
    const size_t nx = (size_t)a->rows * a->in_size, nw = (size_t)a->hidden * a->in_size, nh = (size_t)a->rows * a->hidden, nd = (size_t)a->out_size * a->hidden;
    GatedFfn<T> f = {};
    f.rows = a->rows; f.in = a->in_size; f.hidden = a->hidden; f.out = a->out_size;
    f.dy = sc.in((T *)a->dy, (size_t)a->rows * a->out_size); f.g = const_cast<T *>(sc.in((T *)a->gate, nh)); f.u = const_cast<T *>(sc.in((T *)a->up, nh));
    if (wide) f.wd = sc.in((T *)a->w_down, nd);
    if (a->dx) { f.wg = sc.in((T *)a->w_gate, nw); f.wu = sc.in((T *)a->w_up, nw); }
    if (a->dw_gate || a->dw_up) f.x = sc.in((T *)a->x, nx);
    f.dx = sc.out((T *)a->dx, nx); f.dwg = sc.out((T *)a->dw_gate, nw); f.dwu = sc.out((T *)a->dw_up, nw); f.dwd = sc.out((T *)a->dw_down, nd);
    if (!sc.ok()) return;
    defer_settle(f.dwg); defer_settle(f.dwu); defer_settle(f.dwd);
    gated_ffn_bw<T>(sc, f);
}

} // namespace

#define TL_EXPORT extern "C" __attribute__((visibility("default")))
TL_EXPORT void trainlib_rmsnorm_fp32_fw_cl(void *a) { rmsnorm_fw_impl<float>(a, false); }
TL_EXPORT void trainlib_rmsnorm_fp16_fw_cl(void *a) { rmsnorm_fw_impl<__half>(a, false); }
TL_EXPORT void trainlib_rmsnorm_int8_fp32_fw_cl(void *a) { rmsnorm_fw_impl<float>(a, true); }
TL_EXPORT void trainlib_rmsnorm_int8_fp16_fw_cl(void *a) { rmsnorm_fw_impl<__half>(a, true); }
TL_EXPORT void trainlib_rmsnorm_fp32_bw_cl(void *a) { rmsnorm_bw_impl<float>(a); }
TL_EXPORT void trainlib_rmsnorm_fp16_bw_cl(void *a) { rmsnorm_bw_impl<__half>(a); }
TL_EXPORT void trainlib_quantize_rows_fp32_cl(void *a) { quantize_rows_impl<float>(a); }
TL_EXPORT void trainlib_quantize_rows_fp16_cl(void *a) { quantize_rows_impl<__half>(a); }
TL_EXPORT void trainlib_linear_int8_fp32_fw_cl(void *a) { linear_int8_impl<float>(a); }
TL_EXPORT void trainlib_linear_int8_fp16_fw_cl(void *a) { linear_int8_impl<__half>(a); }
TL_EXPORT void trainlib_gated_ffn_fp32_fw_cl(void *a) { gated_ffn_fw_impl<float>(a); }
TL_EXPORT void trainlib_gated_ffn_fp16_fw_cl(void *a) { gated_ffn_fw_impl<__half>(a); }
TL_EXPORT void trainlib_gated_ffn_fp32_bw_cl(void *a) { gated_ffn_bw_impl<float>(a); }
TL_EXPORT void trainlib_gated_ffn_fp16_bw_cl(void *a) { gated_ffn_bw_impl<__half>(a); }
