"""Microscaled arrays without a GPU: the float64 oracle against known values, the stored layout, and the
refusals of the C entry points and of the Python functions (all of them before any launch)."""
import ctypes as C

import numpy as np
import pytest
import torch

from ancha_b200 import _native as N
from ancha_b200 import microscaled as mx
from oracle import microscaled as O

FORMATS = ("mxf8", "mxf4", "nvf4")


def test_oracle_grids_match_torch():
    codes = torch.arange(127, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).double().numpy(), O.E4M3)
    # Rounding to E4M3 is torch's (to nearest, ties to even) up to the largest value.
    t = np.linspace(0, 448, 100001)
    want = torch.from_numpy(t).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(O.nearest(t, O.E4M3), want)
    # E2M1 ties go to the even code: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4.
    assert O.E2M1[O.nearest([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7], O.E2M1)].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]


def test_oracle_scale_borders():
    # The largest magnitude rounds into the range: 464 still does (a tie to the even 448), beyond it the
    # scale doubles; for E2M1 everything below 7 rounds to at most 6.
    assert O.scale_codes([448, 464, np.nextafter(464, 500), 511, 512], "mxf8").tolist() == [127, 127, 128, 128, 128]
    assert O.scale_codes([6, np.nextafter(7, 0), 7, 8, 3.4], "mxf4").tolist() == [127, 127, 128, 128, 126]
    assert O.scale_codes([0, 1e-45, 2.0 ** -126], "mxf8").tolist() == [0, 0, 0]
    top = float(np.finfo(np.float32).max)
    assert O.scale_codes([top], "mxf8").tolist() == [247] and O.scale_codes([top], "mxf4").tolist() == [253]
    assert O.scale_values(O.scale_codes([6 * 448.0, 1e9, 6.0], "nvf4"), "nvf4").tolist() == [448, 448, 1]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (127, 33), (128, 128), (129, 515), (300, 1000)])
def test_layout(fmt, rows, cols):
    """ancha_mx_layout, the Python shapes and the oracle's packing agree."""
    ld, data, scales = C.c_int64(), C.c_size_t(), C.c_size_t()
    assert N.lib().ancha_mx_layout(mx.FORMATS[fmt], rows, cols, C.byref(ld), C.byref(data), C.byref(scales)) == N.OK
    q = mx.empty(fmt, rows, cols, "cpu")
    assert q.data.shape == (rows, ld.value) and q.data.numel() == data.value and q.scales.numel() == scales.value
    rng = np.random.default_rng(rows + cols)
    e, c = O.quantize(rng.standard_normal((rows, cols)), fmt)
    assert O.pack(e, fmt).shape == tuple(q.data.shape)
    assert np.array_equal(O.unpack(O.pack(e, fmt), fmt, cols), e)
    t = O.tile(c)
    assert t.size == scales.value and np.array_equal(O.untile(t, rows, c.shape[1]), c)
    q.scales.copy_(torch.from_numpy(t).view(q.scales.shape))
    assert np.array_equal(q.scale_codes().numpy(), c)


@pytest.mark.parametrize("fmt", FORMATS)
def test_oracle_error_is_half_a_step(fmt):
    v = np.random.default_rng(3).standard_normal((50, 200)) * np.exp(np.random.default_rng(4).standard_normal((50, 1)))
    g = np.abs(v).max() / (6 * 448) if fmt == "nvf4" else 1.0
    e, c = O.quantize(v, fmt, g)
    d = np.abs(O.expand(e, c, fmt, g) - v)
    s = np.repeat(O.scale_values(c, fmt, g), O.BLOCK[fmt], 1)[:, :200]
    if fmt == "mxf8":
        assert (d <= np.maximum(np.abs(v) * 2.0 ** -4, s * 2.0 ** -10)).all()
    else:
        t = np.abs(v) / s
        # nvf4's rounded scale lets the largest element reach 6 (1 + 2^-4) before it saturates.
        assert (d <= s * np.where(t < 2, .25, np.where(t < 4, .5, 1)) * (1 + 1e-12)).all()


# ------------------------------------------------------------------------------------- refusals

P = 1 << 20  # a 16-byte aligned address that is never read


def array(fmt="mxf8", rows=4, cols=64, ld=None, data=P, scales=P, g=None):
    per = 1 if fmt == "mxf8" else 2
    return N.MxArray(mx.FORMATS.get(fmt, 9), rows, cols, data, ld or -(-cols // (16 * per)) * 16, scales, g)


BAD_ARRAYS = [dict(fmt="?"), dict(rows=-1), dict(cols=0), dict(cols=1 << 31), dict(rows=1 << 31), dict(data=P + 8),
              dict(scales=P + 4), dict(ld=72), dict(ld=48), dict(data=None), dict(scales=None), dict(g=P),
              dict(fmt="nvf4", g=P + 2), dict(ld=1 << 40)]


@pytest.mark.parametrize("bad", BAD_ARRAYS)
def test_bad_arrays_are_refused(bad):
    L = N.lib()
    q, ok = array(**bad), array()
    assert L.ancha_mx_quantize(P, N.F32, 64, C.byref(q), None) != N.OK
    assert L.ancha_mx_dequantize(C.byref(q), P, N.F32, 64, None) != N.OK
    d = N.MxNormDesc(N.F32, N.F32, 64, 64, 64, 1e-6)
    assert L.ancha_mx_add_rms_norm_fwd(C.byref(d), P, P, None, P, C.byref(q), None) != N.OK
    ld = N.MxLinearDesc(N.ACT_NONE, N.F32, N.F32, 64, 64)
    for x, w in ((q, ok), (ok, q)):
        assert L.ancha_mx_linear_fwd(C.byref(ld), C.byref(x), C.byref(w), None, None, P, None, None) in \
            (N.E_INVALID, N.E_UNSUPPORTED)
    assert N.last_error().startswith("mx_linear")


@pytest.mark.parametrize("args", [(None, N.F32, 64), (P, 7, 64), (P, N.F32, 63), (P + 2, N.F32, 64), (P + 1, N.F16, 64),
                                  (P, N.BF16, 1 << 40)])
def test_bad_matrices_are_refused(args):
    L = N.lib()
    q = array()
    x, t, ld = args
    assert L.ancha_mx_quantize(x, t, ld, C.byref(q), None) == N.E_INVALID
    assert L.ancha_mx_dequantize(C.byref(q), x, t, ld, None) == N.E_INVALID
    d = N.MxNormDesc(t, t, ld, ld, ld, 1e-6)
    assert L.ancha_mx_add_rms_norm_fwd(C.byref(d), x, None, None, None, C.byref(q), None) == N.E_INVALID
    w = array(rows=64)
    o = N.MxLinearDesc(N.ACT_NONE, t, N.F32, ld, 64)
    assert L.ancha_mx_linear_fwd(C.byref(o), C.byref(q), C.byref(w), None, None, x, None, None) == N.E_INVALID
    if x is not None:
        o = N.MxLinearDesc(N.ACT_NONE, N.F32, t, 64, ld)
        assert L.ancha_mx_linear_fwd(C.byref(o), C.byref(q), C.byref(w), None, x, P, None, None) == N.E_INVALID


def test_null_arguments_are_refused():
    L = N.lib()
    assert L.ancha_mx_quantize(P, N.F32, 64, None, None) == N.E_INVALID
    assert L.ancha_mx_dequantize(None, P, N.F32, 64, None) == N.E_INVALID
    assert L.ancha_mx_add_rms_norm_fwd(None, P, None, None, None, C.byref(array()), None) == N.E_INVALID
    assert L.ancha_mx_linear_fwd(None, C.byref(array()), C.byref(array()), None, None, P, None, None) == N.E_INVALID
    assert L.ancha_mx_layout(5, 1, 1, None, None, None) == N.E_INVALID


def test_norm_refusals():
    L = N.lib()

    def call(x=P, r=P, gain=None, ro=2 * P, q=None, **k):
        d = dict(dtype=N.F32, residual_dtype=N.F32, ldx=64, ldres=64, ldres_out=64, eps=1e-6)
        d.update(k)
        return L.ancha_mx_add_rms_norm_fwd(C.byref(N.MxNormDesc(**d)), x, r, gain, ro, C.byref(q or array()), None)

    for eps in (0.0, -1.0, float("nan"), float("inf")):
        assert call(eps=eps) == N.E_INVALID
    assert call(ro=None) == N.E_INVALID                                      # a residual without a place for the sum
    assert call(ro=P, ldres_out=128) == N.E_INVALID                          # over the residual, another stride
    assert call(x=3 * P, r=P, ro=3 * P, dtype=N.F16, ldx=64) == N.E_INVALID  # over x, another type
    assert call(r=None, residual_dtype=N.F16) == N.E_INVALID
    assert call(gain=P + 2) == N.E_INVALID
    assert call(q=array(cols=32769), ldx=1 << 16, ldres=1 << 16, ldres_out=1 << 16) == N.E_UNSUPPORTED


def test_linear_refusals():
    L = N.lib()

    def call(x=None, w=None, bias=None, res=None, out=P, om=None, **k):
        d = dict(act=N.ACT_NONE, out_dtype=N.F32, residual_dtype=N.F32, ldout=4, ldres=4)
        d.update(k)
        return L.ancha_mx_linear_fwd(C.byref(N.MxLinearDesc(**d)), C.byref(x or array()), C.byref(w or array()), bias, res,
                                     out, None if om is None else C.byref(om), None)

    assert call(w=array("mxf4")) == N.E_INVALID
    assert call(w=array(cols=65, ld=80)) == N.E_INVALID
    assert call(w=array(rows=0)) == N.E_INVALID
    assert call(act=N.ACT_GLU) == N.E_UNSUPPORTED
    assert call(act=17) == N.E_UNSUPPORTED
    assert call(out=None) == N.E_INVALID
    assert call(om=array(rows=4, cols=4)) == N.E_INVALID                     # both
    assert call(out=None, om=array(rows=4, cols=5)) == N.E_INVALID           # another shape
    assert call(out=None, om=array("mxf4", rows=4, cols=4, g=P)) == N.E_INVALID
    assert call(bias=P + 1) == N.E_INVALID
    assert call(res=P, out=P, residual_dtype=N.F16) == N.E_INVALID           # in place with another type
    assert call(res=P, out=P, ldres=8) == N.E_INVALID


def test_empty_rows_need_no_gpu():
    L = N.lib()
    e = array(rows=0, data=None, scales=None)
    assert L.ancha_mx_quantize(None, N.F32, 64, C.byref(e), None) == N.OK
    assert L.ancha_mx_dequantize(C.byref(e), None, N.F32, 64, None) == N.OK
    d = N.MxNormDesc(N.F32, N.F32, 64, 64, 64, 1e-6)
    assert L.ancha_mx_add_rms_norm_fwd(C.byref(d), None, None, None, None, C.byref(e), None) == N.OK
    o = N.MxLinearDesc(N.ACT_NONE, N.F32, N.F32, 4, 0)
    assert L.ancha_mx_linear_fwd(C.byref(o), C.byref(e), C.byref(array()), None, None, None, None, None) == N.OK


def test_python_refusals():
    x = torch.zeros(4, 64)
    q = mx.empty("mxf8", 4, 64, "cpu")
    for call in (lambda: mx.quantize(x), lambda: mx.dequantize(q), lambda: mx.add_rms_norm(x), lambda: mx.linear(q, q)):
        with pytest.raises(N.AnchaError, match="CUDA device"):
            call()
    with pytest.raises(N.AnchaError, match="unknown format"):
        mx.empty("mxf6", 4, 64, "cpu")
    with pytest.raises(N.AnchaError, match="without elements"):
        mx.empty("mxf8", 4, 0, "cpu")


def test_struct_layouts_match_the_c_compiler(tmp_path):
    import os
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    structs = {"ancha_mx_array": N.MxArray, "ancha_mx_norm_desc": N.MxNormDesc, "ancha_mx_linear_desc": N.MxLinearDesc}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "ancha_b200.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for cname, py in structs.items():
        assert int(got[cname]) == C.sizeof(py)
        for f, _ in py._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(py, f).offset
