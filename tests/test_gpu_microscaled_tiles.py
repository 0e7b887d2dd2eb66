"""Microscaled products whose CTAs and CTA pairs take several tiles each, in every shape of kernel, against a float64
product on the device: all rows and columns, two tolerances.

Worst case, as test_gpu_microscaled.py: (k + 2) * 2^-23 * sum |x w|. And over the whole output: the tensor core adds 32
bytes of both rows at a time, so a sum takes S = k / 32 (8 bits) or k / 64 additions into f32 with an error of at most
2^-23 of the sum so far (truncated at worst). That is at most final in the mean square, so the root mean square error is at
most S * 2^-23 of the outputs' own. A sum kept in fewer bits, or a lost slab, exceeds it."""
import os
import subprocess
import sys
from ctypes import byref

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ancha_b200 import _native as N  # noqa: E402
from ancha_b200 import microscaled as mx  # noqa: E402
from test_gpu_microscaled import FORMATS, HALF_STEP, operands, poisoned_memory, rows_of, scalar  # noqa: E402,F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def product64(x, w):
    """(x . w^T, sum |x w|) in float64 on the device. Expanded f32 values are exact but for nvf4's array scales."""
    gx, gw = x.global_scale, w.global_scale
    g = 1.0 if gx is None else gx.double() * gw.double()
    a, b = (mx.dequantize(mx.Microscaled(q.format, q.rows, q.cols, q.data, q.scales)).double() for q in (x, w))
    return (a @ b.T) * g, (a.abs() @ b.abs().T) * g


def steps(fmt, k):
    return -(-k // (32 if fmt == "mxf8" else 64))


def check(got, y, mass, fmt, k, terms=0.0):
    """`terms`: the largest magnitudes added behind the product."""
    half = HALF_STEP[got.dtype]
    tol = (k + 2) * 2.0 ** -23 * mass + 2.0 ** -22 * (mass + terms)
    err = (got.double() - y).abs()
    assert (err <= tol + half * (y.abs() + tol)).all(), float((err / tol).max())
    rms, own = (float(t.square().mean().sqrt()) for t in (err, y))
    assert rms <= (steps(fmt, k) * 2.0 ** -23 + half + 2.0 ** -23) * own, rms / own


# Rows, columns, depth in units of the 8-bit one: three tiles or so for each CTA (148) or CTA pair (74), each with several
# K slabs. 256-column pairs (whole, odd and ragged widths), 192-column pairs, single CTAs.
TILES = [(5300, 2560, 2304), (5300, 2555, 2340), (12000, 1000, 900), (12000, 965, 520), (60000, 96, 300), (60000, 128, 520)]


def case(fmt, m, n, k, seed=0):
    k = k if fmt == "mxf8" else 2 * k
    x, w = operands(fmt, m, n, k, seed)
    return k, x, w


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", TILES)
def test_products_of_several_tiles(fmt, m, n, k):
    k, x, w = case(fmt, m, n, k)
    y, mass = product64(x, w)
    bias = rows_of(1, n, torch.float32, 4)[0]
    for out in (torch.float32, torch.bfloat16):
        check(mx.linear(x, w, dtype=out), y, mass, fmt, k)
        check(mx.linear(x, w, bias, dtype=out), y + bias.double(), mass, fmt, k, bias.double().abs())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", TILES)
def test_residuals_of_several_tiles(fmt, m, n, k):
    k, x, w = case(fmt, m, n, k)
    y, mass = product64(x, w)
    for r, out in ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16),
                   (torch.float16, torch.float32)):
        res = rows_of(m, n, r, 5, 0.2)
        got = mx.linear(x, w, None, "none", res, dtype=out)
        check(got, y + res.double(), mass, fmt, k, res.double().abs())
        if r == out:  # onto the residual itself
            d = N.MxLinearDesc(N.ACT_NONE, mx._DTYPES[out], mx._DTYPES[r], n, n)
            stream = torch.cuda.current_stream().cuda_stream
            N.check(N.lib().ancha_mx_linear_fwd(byref(d), byref(mx._array(x, 0, "x")), byref(mx._array(w, 0, "w")), None,
                                                res.data_ptr(), res.data_ptr(), None, stream))
            assert torch.equal(res, got)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("out", FORMATS)
@pytest.mark.parametrize("m,n,k", TILES)
def test_quantized_outputs_of_several_tiles(fmt, out, m, n, k):
    """The quantisation of the f32 output, bit for bit, whose values the tests above hold to float64."""
    k, x, w = case(fmt, m, n, k)
    bias, res = rows_of(1, n, torch.float32, 10)[0], rows_of(m, n, torch.bfloat16, 11, 0.2)
    g = scalar(0.01) if out == "nvf4" else None
    for args in ((bias, "gelu", None), (bias, "tanh", res)):
        got = mx.linear(x, w, *args, format=out, global_scale=g)
        want = mx.quantize(mx.linear(x, w, *args, dtype=torch.float32), out, g)
        assert torch.equal(got.data, want.data) and torch.equal(got.scales, want.scales)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 1000, 2000), (40, 700, 2000), (133, 1544, 1000), (300, 520, 2000), *TILES])
def test_rows_do_not_depend_on_one_another(fmt, m, n, k):
    """Rows keep their bits when every other row of x, or of w, becomes another one."""
    k, x, w = case(fmt, m, n, k)
    y = mx.linear(x, w, dtype=torch.float32)
    keep = torch.arange(0, m, 3, device="cuda")
    other = torch.ones(m, dtype=torch.bool, device="cuda")
    other[keep] = False
    x2, w2 = operands(fmt, m, n, k, 77)
    x2.data[keep] = x.data[keep]
    r = keep  # their scales, at (row // 128, :, row % 32, row % 128 // 32, :)
    x2.scales[r // 128, :, r % 32, r % 128 // 32] = x.scales[r // 128, :, r % 32, r % 128 // 32]
    got = mx.linear(x2, w, dtype=torch.float32)
    assert torch.equal(got[keep], y[keep]) and (m == 1 or not torch.equal(got[other], y[other]))
    c = torch.arange(0, n, 3, device="cuda")
    w2.data[c] = w.data[c]
    w2.scales[c // 128, :, c % 32, c % 128 // 32] = w.scales[c // 128, :, c % 32, c % 128 // 32]
    assert torch.equal(mx.linear(x, w2, dtype=torch.float32)[:, c], y[:, c])


def same_codes(q, last, first):
    """The last rows of q, at a multiple of 128, and an array of those rows alone."""
    assert first % 128 == 0
    return torch.equal(q.data[first:], last.data) and torch.equal(q.scale_codes()[first:], last.scale_codes())


def test_operands_beyond_32_bits():
    """Rows of x, and of the stream of a norm, that begin beyond 2^32 bytes: against the same rows alone."""
    m, k, first = 70000, 65504, 69888
    x = torch.empty((m, k), dtype=torch.bfloat16, device="cuda")
    x[:first] = 1
    x[first:] = rows_of(m - first, k, torch.bfloat16, 3)
    w = mx.quantize(rows_of(64, k, torch.float32, 4, 0), "mxf8")
    q = mx.quantize(x, "mxf8")
    last = mx.quantize(x[first:], "mxf8")
    assert same_codes(q, last, first)
    # The same kernel shape: 128 rows a tile, one CTA each.
    rest = mx.quantize(x[first - 128 * 200:], "mxf8")
    assert torch.equal(mx.linear(q, w, dtype=torch.float32)[first:], mx.linear(rest, w, dtype=torch.float32)[128 * 200:])
    del q, rest
    x, r = x[:, :32768], x[:, 32736:]  # rows 131008 bytes apart
    q, s = mx.add_rms_norm(x, r)
    one, t = mx.add_rms_norm(x[first:], r[first:])
    assert torch.equal(s[first:], t) and same_codes(q, one, first)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 333, 1504])
def test_gain_at_an_odd_address(fmt, dim):
    x = rows_of(20, dim, torch.float32, 1)
    gain = rows_of(1, dim + 3, torch.float32, 2, 0)[0]
    for lo in range(4):
        q, _ = mx.add_rms_norm(x, gain=gain[lo:lo + dim], format=fmt)
        want, _ = mx.add_rms_norm(x, gain=gain[lo:lo + dim].clone(), format=fmt)
        assert torch.equal(q.data, want.data) and torch.equal(q.scales, want.scales)


def test_calls_from_several_threads():
    """Threads with a stream each, in shapes of every kernel, get what one thread gets."""
    import threading
    shapes = [("mxf8", 3, 700, 2000), ("nvf4", 300, 520, 600), ("mxf4", 3000, 96, 300), ("mxf8", 133, 1544, 1000)]
    work = [(*operands(f, m, n, k, m), rows_of(1, n, torch.float32, 9)[0]) for f, m, n, k in shapes]
    want = [mx.linear(x, w, b, "gelu", format="mxf8") for x, w, b in work]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        x, w, b = work[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                y = mx.linear(x, w, b, "gelu", format="mxf8")
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(y.data, want[i].data) and torch.equal(y.scales, want[i].scales)):
                    wrong.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


CAPTURE_FIRST = """
import torch
from ancha_b200 import microscaled as mx
x, r = torch.randn({m}, 384, device="cuda"), torch.randn({m}, 384, device="cuda")
v = torch.randn(512, 384, device="cuda")
torch.cuda.synchronize()
def block():
    q, s = mx.add_rms_norm(x, r, format="{fmt}")
    w = mx.quantize(v, "{fmt}")
    h = mx.linear(q, w, None, "gelu", format="{fmt}")
    return mx.dequantize(h), mx.linear(q, w, dtype=torch.float32), s
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = block()
g.replay()
b = block()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(a, b))
print("same")
"""


@pytest.mark.parametrize("fmt,m", [("mxf8", 3), ("nvf4", 600)])
def test_the_first_calls_of_a_process_can_be_captured(fmt, m):
    code = CAPTURE_FIRST.format(fmt=fmt, m=m)
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]
