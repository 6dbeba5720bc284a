"""The operators of a transformer's feed-forward half, as cases whose time and outputs can be measured.

  norm_fw, norm_bw  RMS norm of a residual sum, forward (sum and norm) and backward
  ffn_fw, ffn_bw    gated feed-forward block y = (silu(x Wg^T) * (x Wu^T)) Wd^T, forward and backward
  int8              matrix product of 8-bit integers with a scale for each token and each output channel; its left operand is
                    given in 8 bits ("given"), quantised from a tensor within the pass ("rows"), or leaves the RMS norm of a
                    residual sum in 8 bits ("norm")

Tensors live in device memory and are handed to the library's entry points by address.
"""
import ctypes
import importlib
import math

import torch

own = False

EPS = 1e-5
DTYPE = {"fp32": torch.float32, "fp16": torch.float16}
ESIZE = {"fp32": 4, "fp16": 2}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one token of a generation loop passes the norm in front of a block: latency
        dict(name="norm_token_fp16", kind="norm_fw", dtype="fp16", rows=1, size=4096),
        # the norm of a training step's forward pass in single precision, as long as a batch of sequences is
        dict(name="norm_fw_fp32", kind="norm_fw", dtype="fp32", rows=8192, size=2048),
        # its backward pass over a ragged batch and a width that is no power of two
        dict(name="norm_bw_fp32_ragged", kind="norm_bw", dtype="fp32", rows=1023, size=1000),
        # the backward pass of a large half-precision step: what comes back through the residual path is added
        dict(name="norm_bw_fp16", kind="norm_bw", dtype="fp16", rows=16384, size=2048),
        # one token of a generation loop through a block: the weights' bytes
        dict(name="ffn_token_fp16", kind="ffn_fw", dtype="fp16", rows=1, inn=4096, hidden=10240, out=4096, save=False),
        # a few tokens (a short batch of streams) through a block whose sizes are odd
        dict(name="ffn_few_odd_fp16", kind="ffn_fw", dtype="fp16", rows=23, inn=1000, hidden=2731, out=1000, save=False),
        # forward and backward pass of a training step in half precision
        dict(name="ffn_fw_fp16", kind="ffn_fw", dtype="fp16", rows=4096, inn=2048, hidden=8192, out=2048, save=True),
        dict(name="ffn_bw_fp16", kind="ffn_bw", dtype="fp16", rows=4096, inn=2048, hidden=8192, out=2048),
        # backward pass in single precision with the sizes of the encoder block of the benchmark
        dict(name="ffn_bw_fp32", kind="ffn_bw", dtype="fp32", rows=128, inn=512, hidden=512, out=512),
        # one token of a served network: the norm leaves 8 bits for the projection behind it
        dict(name="int8_token", kind="int8", dtype="fp16", source="norm", rows=1, inn=4096, out=10240, bias=False),
        # a prompt's tokens, quantised as they come and projected
        dict(name="int8_prompt", kind="int8", dtype="fp16", source="rows", rows=4096, inn=8192, out=4096, bias=False),
        # a small ragged layer with a bias and single-precision results
        dict(name="int8_ragged_fp32", kind="int8", dtype="fp32", source="given", rows=333, inn=1001, out=777, bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """a width: odd, even, or (most often) a multiple of 64"""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.6 else n


def draw(rng):
    kind = rng.choice(["norm_fw", "norm_bw", "ffn_fw", "ffn_bw", "int8", "int8"])
    dtype = rng.choice(["fp16", "fp16", "fp32"])
    while True:
        if kind in ("norm_fw", "norm_bw"):
            c = dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 16384), size=_width(rng, 16, 16384))
        elif kind in ("ffn_fw", "ffn_bw"):
            most = 4096 if dtype == "fp16" else 1024
            c = dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 4096 if dtype == "fp16" else 1024), inn=_width(rng, 64, most), hidden=_width(rng, 64, 2 * most), out=0)
            c["out"] = c["inn"] if rng.random() < 0.8 else _width(rng, 64, most)
            if kind == "ffn_fw":
                c["save"] = rng.random() < 0.5
        else:
            # (single-precision results of integers that are given: beside a border of the quantisation two right answers are a step apart)
            c = dict(kind=kind, dtype=dtype, source="given" if dtype == "fp32" else rng.choice(["given", "rows", "norm"]), rows=_log(rng, 1, 4096), inn=_width(rng, 64, 8192),
                     out=_width(rng, 64, 8192), bias=rng.random() < 0.3)
        w = work(c)
        if w["flops"] < 3e11 and w["bytes"] < 4e8:
            return c


def work(c):
    """Bytes with every input read once and every output written once; floating-point operations at two per multiply-add."""
    es, r = ESIZE[c["dtype"]], c["rows"]
    if c["kind"] == "norm_fw":                    # x, residual in; sum, norm out; the weight
        return {"bytes": es * (4 * r * c["size"] + c["size"]), "flops": 5.0 * r * c["size"]}
    if c["kind"] == "norm_bw":                    # sum, dy, dsum in; dx out; the weight and its gradient
        return {"bytes": es * (4 * r * c["size"] + 2 * c["size"]), "flops": 12.0 * r * c["size"]}
    if c["kind"] == "int8":
        n, m = c["inn"], c["out"]
        left = {"given": r * n + 4 * r, "rows": es * r * n, "norm": es * (3 * r * n + n)}[c["source"]]
        return {"bytes": left + n * m + 4 * m + es * r * m + (es * m if c["bias"] else 0), "flops": 2.0 * r * n * m}
    n, h, m = c["inn"], c["hidden"], c["out"]
    if c["kind"] == "ffn_fw":
        return {"bytes": es * (r * (n + m) + h * (2 * n + m) + (2 * r * h if c["save"] else 0)), "flops": 2.0 * r * h * (2 * n + m)}
    return {"bytes": es * (r * (2 * n + m + 2 * h) + 2 * h * (2 * n + m)), "flops": 4.0 * r * h * (2 * n + m)}


# ------------------------------------------------------------------------------------------------ inputs
class State(object):
    """A program's tensors and, once the library has been called, its argument structs."""

    def __init__(self, case):
        self.case, self.calls, self.stream = case, None, 0


def _randn(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def prepare(case, seed):
    s, c = State(case), case
    dt, r = DTYPE[c["dtype"]], c["rows"]
    gen = torch.Generator("cuda").manual_seed(int(seed))
    new = lambda *shape, dtype=dt: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
    if c["kind"] in ("norm_fw", "norm_bw"):
        n = c["size"]
        s.w = 1 + 0.1 * _randn(gen, n)
        s.w = s.w.to(dt)
        if c["kind"] == "norm_fw":
            s.x, s.res = _randn(gen, r, n, dtype=dt), _randn(gen, r, n, scale=3.0, dtype=dt)
            s.sum, s.y = new(r, n), new(r, n)
        else:
            s.sum, s.dy, s.dsum = _randn(gen, r, n, scale=3.0, dtype=dt), _randn(gen, r, n, dtype=dt), _randn(gen, r, n, dtype=dt)
            s.dx, s.dw = new(r, n), new(n)
    elif c["kind"] == "int8":
        n, m = c["inn"], c["out"]
        # weights as a program holds them: quantised once, a scale for each output channel
        w = _randn(gen, m, n, scale=1 / math.sqrt(n))
        s.ws = w.abs().amax(1) / 127
        s.wq = torch.round(w / s.ws[:, None]).to(torch.int8)
        s.bias = _randn(gen, m, dtype=dt) if c["bias"] else None
        if c["source"] == "given":
            x = _randn(gen, r, n)
            s.xs = x.abs().amax(1) / 127
            s.xq = torch.round(x / s.xs[:, None]).to(torch.int8)
        else:
            s.x = _randn(gen, r, n, dtype=dt)
            s.xq, s.xs = new(r, n, dtype=torch.int8), new(r, dtype=torch.float32)
        if c["source"] == "norm":
            s.res, s.sum = _randn(gen, r, n, scale=3.0, dtype=dt), new(r, n)
            s.w = (1 + 0.1 * _randn(gen, n)).to(dt)
        s.y = new(r, m)
    else:
        n, h, m = c["inn"], c["hidden"], c["out"]
        s.x = _randn(gen, r, n, dtype=dt)
        s.wg, s.wu = (_randn(gen, h, n, scale=1 / math.sqrt(n), dtype=dt) for _ in range(2))
        s.wd = _randn(gen, m, h, scale=1 / math.sqrt(h), dtype=dt)
        if c["kind"] == "ffn_fw":
            s.y = new(r, m)
            s.g, s.u = (new(r, h), new(r, h)) if c["save"] else (None, None)
        else:
            s.g, s.u = s.x @ s.wg.T, s.x @ s.wu.T             # what the forward pass left
            s.dy = _randn(gen, r, m, dtype=dt)
            s.dx, s.dwg, s.dwu, s.dwd = new(r, n), new(h, n), new(h, n), new(m, h)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _mean_square(h):
    return (h * h).sum(-1, keepdim=True) / h.shape[-1]


def _quantise(y):
    """8-bit integers and a scale for each row (in 64 bits: a value beside the border of two steps)"""
    scale = y.abs().amax(-1, keepdim=True) / 127
    return torch.round(y / scale), scale


def _norm_fw(s):
    h = s.x.float() + s.res.float()
    y = h / torch.sqrt(_mean_square(h) + EPS) * s.w.float()
    return h.to(s.x.dtype), y.to(s.x.dtype)


def _norm_bw(s):
    dt = s.sum.dtype
    h, dy, w = s.sum.float(), s.dy.float(), s.w.float()
    r = 1 / torch.sqrt(_mean_square(h) + EPS)
    g = dy * w
    dx = s.dsum.float() + r * (g - h * r * r * ((g * h).sum(-1, keepdim=True) / h.shape[-1]))
    return dx.to(dt), (dy * h * r).sum(0).to(dt)


def _ffn_fw(s):
    dt, x = s.x.dtype, s.x.float()
    g, u = x @ s.wg.float().T, x @ s.wu.float().T
    y = (g / (1 + torch.exp(-g)) * u) @ s.wd.float().T
    return (y.to(dt), g.to(dt), u.to(dt)) if s.g is not None else y.to(dt)


def _ffn_bw(s):
    dt, x, g, u, dy = s.x.dtype, s.x.float(), s.g.float(), s.u.float(), s.dy.float()
    sig = 1 / (1 + torch.exp(-g))
    act = g * sig
    dh = dy @ s.wd.float()
    dg, du = dh * u * (sig + act * (1 - sig)), dh * act
    dx = dg @ s.wg.float() + du @ s.wu.float()
    return dx.to(dt), (dg.T @ x).to(dt), (du.T @ x).to(dt), (dy.T @ (act * u)).to(dt)


def _int8(s):
    c, dt = s.case, s.y.dtype
    if c["source"] == "given":
        q, scale = s.xq.double(), s.xs.double()[:, None]
    else:
        h = s.x.double()
        if c["source"] == "norm":
            h = h + s.res.double()
            total = h.to(dt)
            h = h / torch.sqrt(_mean_square(h) + EPS) * s.w.double()
        q, scale = _quantise(h)
    # whole numbers of up to 7 bits: sums of their products are exact in 64 bits
    y = (q @ s.wq.double().T) * scale * s.ws.double()
    if s.bias is not None:
        y = y + s.bias.double()
    return (y.to(dt), total) if c["source"] == "norm" else y.to(dt)


# ------------------------------------------------------------------------------------------------ the framework's kernels
_pkg = None
_on = None                                                    # the stream that the library's calls are queued on
LEGACY = 1                                                    # CUDA's handle of the default stream, which torch gives as 0


def _library():
    global _pkg
    if _pkg is None:
        _pkg = importlib.import_module("pulp-trainlib_b200")
        lib = _pkg.load()
        lib.trainlib_init(torch.cuda.current_device())
        lib.trainlib_set_memory_mode(_pkg.TL_MEM_DEVICE)      # every tensor lives on the device
    return _pkg, _pkg.load()


def _own_calls(s):
    """The program's calls and what they leave: the argument structs are filled once, as a C program keeps them."""
    pkg, lib = _library()
    c, p = s.case, s.case["dtype"]
    s.keep = pkg.Keep()
    s.stream = torch.cuda.current_stream().cuda_stream or LEGACY

    def call(name, struct, **fields):
        at = {k: v.data_ptr() if isinstance(v, torch.Tensor) else v for k, v in fields.items()}
        return getattr(lib, name), ctypes.byref(pkg.make_args(s.keep, struct, **at))

    if c["kind"] == "norm_fw":
        s.out = (s.sum, s.y)
        return [call("trainlib_rmsnorm_%s_fw_cl" % p, "trainlib_rmsnorm_args", x=s.x, residual=s.res, weight=s.w, sum=s.sum, output=s.y, eps=EPS, rows=c["rows"], size=c["size"])]
    if c["kind"] == "norm_bw":
        s.out = (s.dx, s.dw)
        return [call("trainlib_rmsnorm_%s_bw_cl" % p, "trainlib_rmsnorm_args", sum=s.sum, weight=s.w, dy=s.dy, dsum=s.dsum, dx=s.dx, dweight=s.dw, eps=EPS, rows=c["rows"], size=c["size"])]
    if c["kind"] == "int8":
        calls = []
        if c["source"] == "rows":
            calls.append(call("trainlib_quantize_rows_%s_cl" % p, "trainlib_quantize_rows_args", x=s.x, q=s.xq, scale=s.xs, rows=c["rows"], size=c["inn"]))
        if c["source"] == "norm":
            calls.append(call("trainlib_rmsnorm_int8_%s_fw_cl" % p, "trainlib_rmsnorm_args", x=s.x, residual=s.res, weight=s.w, sum=s.sum, q=s.xq, scale=s.xs, eps=EPS,
                              rows=c["rows"], size=c["inn"]))
        s.out = (s.y, s.sum) if c["source"] == "norm" else s.y
        return calls + [call("trainlib_linear_int8_%s_fw_cl" % p, "trainlib_linear_int8_args", x=s.xq, x_scale=s.xs, weight=s.wq, w_scale=s.ws, bias=s.bias, y=s.y,
                             rows=c["rows"], in_size=c["inn"], out_size=c["out"])]
    sizes = dict(rows=c["rows"], in_size=c["inn"], hidden=c["hidden"], out_size=c["out"])
    if c["kind"] == "ffn_fw":
        s.out = (s.y, s.g, s.u) if c["save"] else s.y
        return [call("trainlib_gated_ffn_%s_fw_cl" % p, "trainlib_gated_ffn_args", x=s.x, w_gate=s.wg, w_up=s.wu, w_down=s.wd, gate=s.g, up=s.u, y=s.y, **sizes)]
    s.out = (s.dx, s.dwg, s.dwu, s.dwd)
    return [call("trainlib_gated_ffn_%s_bw_cl" % p, "trainlib_gated_ffn_args", x=s.x, w_gate=s.wg, w_up=s.wu, w_down=s.wd, gate=s.g, up=s.u, dy=s.dy, dx=s.dx,
                 dw_gate=s.dwg, dw_up=s.dwu, dw_down=s.dwd, **sizes)]


def run(s):
    global _on
    if own:
        first = s.calls is None
        if first:
            s.calls = _own_calls(s)
        if _on != s.stream:                                   # behind the kernels that made the inputs, in front of those that read what leaves
            _on = s.stream
            _library()[1].trainlib_set_stream(_on)
        for fn, args in s.calls:
            fn(args)
        if first:
            _pkg.check(_pkg.load())                           # a refused call left its outputs as they were
        return s.out
    return {"norm_fw": _norm_fw, "norm_bw": _norm_bw, "ffn_fw": _ffn_fw, "ffn_bw": _ffn_bw, "int8": _int8}[s.case["kind"]](s)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    d = lambda t: t.double()  # noqa: E731
    if c["kind"] == "norm_fw":
        h = d(s.x) + d(s.res)
        return h, d(s.w) * h * (h.pow(2).mean(1, keepdim=True) + EPS).rsqrt()
    if c["kind"] == "norm_bw":                    # by differentiation of the forward formula
        h, w = d(s.sum).requires_grad_(), d(s.w).requires_grad_()
        y = w * h * (h.pow(2).mean(1, keepdim=True) + EPS).rsqrt()
        return torch.autograd.grad([y, h], [h, w], [d(s.dy), d(s.dsum)])
    if c["kind"] == "int8":
        total = None
        if c["source"] == "given":
            left = torch.mul(d(s.xq), d(s.xs).unsqueeze(1))
        else:
            left = d(s.x)
            if c["source"] == "norm":
                total = left + d(s.res)
                left = total.div((total.square().mean(1) + EPS).sqrt().unsqueeze(1)).mul(d(s.w))
            step = torch.linalg.vector_norm(left, math.inf, dim=1, keepdim=True).div(127)
            left = left.div(step).round().mul(step)
        y = torch.einsum("rk,mk->rm", left, torch.mul(d(s.wq), d(s.ws).unsqueeze(1)))
        y = y if s.bias is None else y.add(d(s.bias))
        return (y, total) if total is not None else y
    x, wg, wu, wd = d(s.x), d(s.wg), d(s.wu), d(s.wd)
    if c["kind"] == "ffn_fw":
        g, u = torch.einsum("rk,hk->rh", x, wg), torch.einsum("rk,hk->rh", x, wu)
        y = torch.einsum("rh,mh->rm", g * torch.sigmoid(g) * u, wd)
        return (y, g, u) if c["save"] else y
    g, u, wd = d(s.g).requires_grad_(), d(s.u).requires_grad_(), wd.requires_grad_()
    y = torch.einsum("rh,mh->rm", g * torch.sigmoid(g) * u, wd)
    dg, du, dwd = torch.autograd.grad(y, [g, u, wd], d(s.dy))
    return torch.einsum("rh,hk->rk", dg, wg) + torch.einsum("rh,hk->rk", du, wu), torch.einsum("rh,rk->hk", dg, x), torch.einsum("rh,rk->hk", du, x), dwd
