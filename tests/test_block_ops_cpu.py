"""CPU: refusals of the feed-forward operators' entry points (RMS norm of a residual sum, gated feed-forward block, linear layer in 8-bit
integers).  Arguments are checked before a device is asked for, so a refused call says what is wrong with it on any box."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD_ARGS, TOO_LARGE, NO_DEVICE = 3, 5, 1

# a process of its own: the first error of a process stays when it is that there is no device
RUN = r'''
import sys, ctypes
sys.path.insert(0, "tests")
import conftest, numpy as np
pkg = conftest.load_pkg(); lib = pkg.load()
name, struct, fields = sys.argv[1], sys.argv[2], eval(sys.argv[3])
keep = pkg.Keep()
out = np.full(64, 5, np.float32)
buf = {"in": np.ones(64, np.float32), "out": out}
args = pkg.make_args(keep, struct, **{k: buf.get(v, v) if isinstance(v, str) else v for k, v in fields.items()})
getattr(lib, name)(ctypes.byref(args))
print(lib.trainlib_last_error(), int(np.all(out == 5)))
'''


def outcome(name, struct, fields):
    r = subprocess.run([sys.executable, "-c", RUN, name, struct, repr(fields)], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0, r.stderr
    code, untouched = r.stdout.split()[-2:]
    return int(code), untouched == "1"


NORM = dict(x="in", weight="in", output="out", sum="out", eps=1e-5, rows=2, size=8)
NORM8 = dict(x="in", weight="in", q="out", scale="out", eps=1e-5, rows=2, size=8)
NORM_BW = dict(sum="in", weight="in", dy="in", dx="out", eps=1e-5, rows=2, size=8)
FFN = dict(x="in", w_gate="in", w_up="in", w_down="in", y="out", rows=2, in_size=4, hidden=4, out_size=4)
FFN_BW = dict(x="in", w_gate="in", w_up="in", w_down="in", gate="in", up="in", dy="in", dx="out", rows=2, in_size=4, hidden=4, out_size=4)
LIN8 = dict(x="in", x_scale="in", weight="in", w_scale="in", y="out", rows=2, in_size=4, out_size=4)
ROWS8 = dict(x="in", q="out", scale="out", rows=2, size=8)

REFUSED = [("trainlib_rmsnorm_%s_fw_cl", "trainlib_rmsnorm_args", NORM, d) for d in (dict(rows=0), dict(rows=-1), dict(size=0), dict(x=None), dict(weight=None), dict(output=None))]
REFUSED += [("trainlib_rmsnorm_int8_%s_fw_cl", "trainlib_rmsnorm_args", NORM8, d) for d in (dict(rows=0), dict(size=-3), dict(q=None), dict(scale=None))]
REFUSED += [("trainlib_rmsnorm_%s_bw_cl", "trainlib_rmsnorm_args", NORM_BW, d) for d in (dict(rows=0), dict(size=0), dict(sum=None), dict(dy=None), dict(weight=None), dict(dx=None))]
REFUSED += [("trainlib_gated_ffn_%s_fw_cl", "trainlib_gated_ffn_args", FFN, d)
            for d in (dict(rows=0), dict(in_size=0), dict(hidden=0), dict(out_size=-1), dict(x=None), dict(w_gate=None), dict(w_up=None), dict(w_down=None), dict(y=None), dict(gate="out"), dict(up="out"))]
REFUSED += [("trainlib_gated_ffn_%s_bw_cl", "trainlib_gated_ffn_args", FFN_BW, d)
            for d in (dict(rows=0), dict(hidden=-5), dict(dy=None), dict(gate=None), dict(up=None), dict(w_down=None), dict(w_gate=None), dict(w_up=None), dict(dx=None), dict(dw_up="out", x=None))]
REFUSED += [("trainlib_linear_int8_%s_fw_cl", "trainlib_linear_int8_args", LIN8, d)
            for d in (dict(rows=0), dict(in_size=0), dict(out_size=0), dict(x=None), dict(x_scale=None), dict(weight=None), dict(w_scale=None), dict(y=None))]
REFUSED += [("trainlib_quantize_rows_%s_cl", "trainlib_quantize_rows_args", ROWS8, d) for d in (dict(rows=0), dict(size=0), dict(x=None), dict(q=None), dict(scale=None))]


@pytest.mark.parametrize("name,struct,fields,change", REFUSED, ids=["%s-%s" % (r[0].split("_%s")[0][9:] + r[0].split("%s")[1], "-".join("%s=%s" % i for i in r[3].items())) for r in REFUSED])
def test_refused(name, struct, fields, change):
    assert outcome(name % "fp32", struct, {**fields, **change}) == (BAD_ARGS, True)


@pytest.mark.parametrize("p", ["fp32", "fp16"])
def test_sums_that_pass_32_bits_are_refused(p):
    assert outcome("trainlib_linear_int8_%s_fw_cl" % p, "trainlib_linear_int8_args", {**LIN8, "in_size": 131072}) == (TOO_LARGE, True)


@pytest.mark.parametrize("size", ["rows", "in_size", "hidden", "out_size"])
@pytest.mark.parametrize("p", ["fp32", "fp16"])
def test_sizes_beyond_the_index_arithmetic_are_refused(p, size):
    for name, fields in (("trainlib_gated_ffn_%s_fw_cl", FFN), ("trainlib_gated_ffn_%s_bw_cl", FFN_BW)):
        assert outcome(name % p, "trainlib_gated_ffn_args", {**fields, size: (1 << 30) + 1}) == (TOO_LARGE, True)


def test_null_arguments_and_a_machine_without_a_device(pkg):
    lib = pkg.load()
    for name in pkg.EXT_FUNCTIONS:
        if any(w in name for w in ("rmsnorm", "gated_ffn", "int8", "quantize_rows")):
            r = subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, 'tests'); import conftest; lib = conftest.load_pkg().load(); lib.%s(None); print(lib.trainlib_last_error())" % name],
                               capture_output=True, text=True, cwd=ROOT)
            assert r.returncode == 0 and r.stdout.split()[-1] == str(BAD_ARGS), (name, r.stdout, r.stderr)
    if lib.trainlib_init(-1) != 0:
        for name, struct, fields in (("trainlib_rmsnorm_fp32_fw_cl", "trainlib_rmsnorm_args", NORM), ("trainlib_gated_ffn_fp32_bw_cl", "trainlib_gated_ffn_args", FFN_BW),
                                     ("trainlib_linear_int8_fp32_fw_cl", "trainlib_linear_int8_args", LIN8)):
            assert outcome(name, struct, fields) == (NO_DEVICE, True)


LIMITS = [("trainlib_rmsnorm_%s_fw_cl", "trainlib_rmsnorm_args", NORM, ("rows", "size")), ("trainlib_rmsnorm_int8_%s_fw_cl", "trainlib_rmsnorm_args", NORM8, ("rows", "size")),
          ("trainlib_rmsnorm_%s_bw_cl", "trainlib_rmsnorm_args", NORM_BW, ("rows", "size")), ("trainlib_quantize_rows_%s_cl", "trainlib_quantize_rows_args", ROWS8, ("rows", "size")),
          ("trainlib_linear_int8_%s_fw_cl", "trainlib_linear_int8_args", LIN8, ("rows", "out_size"))]


@pytest.mark.parametrize("p", ["fp32", "fp16"])
@pytest.mark.parametrize("name,struct,fields,sizes", LIMITS, ids=[r[0][9:].replace("_%s", "").replace("_cl", "") for r in LIMITS])
def test_sizes_that_wrap_around_are_refused(p, name, struct, fields, sizes):
    """above 2^30 in every operator: a row's or a column's index plus what a pass adds to it stays below 2^31"""
    for size in sizes:
        for n in ((1 << 30) + 1, (1 << 31) - 1):
            assert outcome(name % p, struct, {**fields, size: n}) == (TOO_LARGE, True), (size, n)
