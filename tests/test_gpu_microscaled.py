"""Microscaled operators on the GPU against float64 (oracle/microscaled.py).

Tolerances. Quantisation: scale codes and elements equal the oracle's bit for bit, but for nvf4 elements whose
quotient lies within 2^-22 of a border without being on it (its divisor scale * array scale and the
quotient are rounded to f32, 2^-24 each). Norm: three f32 roundings (1/rms, times s, times gain), 4 * 2^-24
of |y|. Products: operands and their products are exact in f32, so the sum of k of them is off by at most
(k + 2) * 2^-23 * sum |x w| (every addition truncated at worst); the epilogue adds 2^-23 of its terms, GELU
7e-7 + 5e-6 |y| and tanh 3e-7 (the errors that tc.cuh derives for its polynomials), the output's type half a
step. A quantised result is off by half a step of its elements more, and its scale is that of a maximum within
the tolerance."""
import math
from ctypes import byref

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ancha_b200 import _native as N  # noqa: E402
from ancha_b200 import microscaled as mx  # noqa: E402
from oracle import microscaled as O  # noqa: E402

FORMATS = ("mxf8", "mxf4", "nvf4")
BLOCK = O.BLOCK
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def poisoned_memory(monkeypatch):
    """New arrays hold 0xAB everywhere, so that a byte that a call has to write and does not is seen."""
    plain = mx.Microscaled._new.__func__

    def poisoned(cls, *args):
        q = plain(cls, *args)
        q._buffer.fill_(0xAB)
        return q

    monkeypatch.setattr(mx.Microscaled, "_new", classmethod(poisoned))


def f64(t):
    return t.detach().double().cpu().numpy()


def rows_of(rows, cols, dtype, seed=0, spread=1.0):
    rng = np.random.default_rng(seed)
    v = rng.standard_normal((rows, cols)) * np.exp(spread * rng.standard_normal((rows, 1)))
    return torch.from_numpy(v).to(dtype).cuda()


def scalar(g):
    return None if g is None else torch.full((1,), g, dtype=torch.float32, device="cuda")


def stored(q):
    """(element codes, scale codes, all stored scale bytes, element bytes behind the columns) on the host."""
    data = q.data.cpu().numpy()
    nb = -(-q.cols // O.BLOCK[q.format])
    scales = q.scales.cpu().numpy().reshape(-1)
    tail = data[:, (q.cols if q.format == "mxf8" else (q.cols + 1) // 2):]
    return O.unpack(data, q.format, q.cols), O.untile(scales, q.rows, nb), scales, tail


def gval(q):
    return 1.0 if q.global_scale is None else float(q.global_scale.double().item())


def check_exact(q, v, g=1.0, rounded=True):
    """q holds exactly the oracle's quantisation of the float64 rows v; with nvf4 and `rounded` (a divisor that
    is no power of two), either neighbour within 2^-22 of a border."""
    e, c = O.quantize(v, q.format, g)
    ge, gc, scales, tail = stored(q)
    assert np.array_equal(gc, c)
    assert np.array_equal(scales, O.tile(c))  # zeros behind the last row and block
    assert not tail.any()
    if q.format == "nvf4" and rounded:
        s = np.repeat(O.scale_values(c, "nvf4", g), 16, 1)[:, :q.cols]
        dead = ~(s > 0)
        t = np.abs(np.where(np.isfinite(v), v, 0)) / np.where(dead, 1, s)
        sign = e & 8
        lo, hi = (np.where(dead, 0, O.nearest(t * (1 + d), O.E2M1)) for d in (-2.0 ** -22, 2.0 ** -22))
        on = np.isin(t, (O.E2M1[1:] + O.E2M1[:-1]) / 2)  # exact ties stay exact
        e = np.where((ge >= sign + lo) & (ge <= sign + hi) & ~on, ge, e)
    assert np.array_equal(ge, e)


def check_near(q, y, tol):
    """q is a quantisation of rows within tol of the float64 rows y."""
    g, fmt = gval(q), q.format
    ge, gc, scales, tail = stored(q)
    assert not tail.any()
    assert np.array_equal(scales, O.tile(gc))
    a = np.abs(O.blocks(y, fmt)).max(-1)
    ta = O.blocks(np.broadcast_to(tol, y.shape), fmt).max(-1)
    # nvf4's quotient with the array scale is rounded to f32 before it is rounded to E4M3.
    ta = ta + 2.0 ** -22 * a * (fmt == "nvf4")
    assert (gc >= O.scale_codes(np.maximum(a - ta, 0), fmt, g)).all() and (gc <= O.scale_codes(a + ta, fmt, g)).all()
    s = np.repeat(O.scale_values(gc, fmt, g), O.BLOCK[fmt], 1)[:, :q.cols]
    d = np.abs(O.expand(ge, gc, fmt, g) - y)
    t = (np.abs(y) + tol) * (1 + 2.0 ** -20)
    if fmt == "mxf8":
        half = np.maximum(t * 2.0 ** -4, s * 2.0 ** -10)
    else:
        half = s * np.where(t < 2 * s, .25, np.where(t < 4 * s, .5, 1))
        half = np.maximum(half, t - 6 * s)  # nvf4: a block scale saturated at 448 saturates its elements
        half = np.where(s == 0, t, half)  # nvf4: a block below the least scale
    assert (d <= half * (1 + 2.0 ** -20) + tol).all()


# -------------------------------------------------------------------------------- quantise, expand

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 31), (5, 64), (127, 129), (130, 515), (257, 1000)])
def test_quantize_matches_oracle(fmt, dtype, rows, cols):
    x = rows_of(rows, cols, DTYPES[dtype], seed=rows * cols)
    g = float(np.float32(f64(x.abs().max()) / (6 * 448))) if fmt == "nvf4" else None
    q = mx.quantize(x, fmt, scalar(g))
    check_exact(q, f64(x), 1.0 if g is None else g)
    if fmt == "nvf4":
        check_exact(mx.quantize(x, fmt), f64(x))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 37), (130, 515), (64, 96)])
def test_dequantize_matches_oracle(fmt, dtype, rows, cols):
    q = mx.quantize(rows_of(rows, cols, torch.float32, seed=cols), fmt, scalar(0.01) if fmt == "nvf4" else None)
    e, c, _, _ = stored(q)
    want = O.expand(e, c, fmt, gval(q))
    got = f64(mx.dequantize(q, DTYPES[dtype]))
    # Two f32 roundings at most (scale * array scale, times the element), then the output's.
    tiny = 2.0 ** -149 if dtype != "f16" else 2.0 ** -25
    assert (np.abs(got - want) <= np.abs(want) * (HALF_STEP[DTYPES[dtype]] + 2.0 ** -23) + tiny).all()
    if fmt != "nvf4" and dtype != "f16":
        assert np.array_equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_borders_of_the_grid(fmt):
    """Every element value, every tie, and the values next to the ties, under scales from the least up."""
    grid = O.GRID[fmt]
    mid = (grid[1:] + grid[:-1]) / 2
    vals = np.concatenate((grid, mid, np.nextafter(mid.astype(np.float32), np.float32(0)).astype(np.float64),
                           np.nextafter(mid.astype(np.float32), np.float32(1e9)).astype(np.float64)))
    vals = np.concatenate((vals, -vals))
    b = O.BLOCK[fmt]
    per = b - 1
    vals = np.pad(vals, (0, -len(vals) % per)).reshape(-1, per)
    block = np.concatenate((np.full((len(vals), 1), grid[-1]), vals), 1)  # the first element fixes the scale
    exps = (-120, -60, -1, 0, 5, 100) if fmt != "nvf4" else (-8, -1, 0, 5)
    x = np.concatenate([block * 2.0 ** e for e in exps]).astype(np.float32)
    x = x.reshape(len(exps), -1)
    # Every divisor is a power of two: no quotient rounds.
    check_exact(mx.quantize(torch.from_numpy(x).cuda(), fmt), x.astype(np.float64), rounded=False)


@pytest.mark.parametrize("fmt", FORMATS)
def test_scale_borders_and_extremes(fmt):
    """Blocks of one value next to every border of the scale's choice, tiny and huge ones, and zeros."""
    b = O.BLOCK[fmt]
    tops = []
    for e in (-126, -120, -10, 0, 20, 118):
        for r in (1.0, 1.75, 1.8125, 464 / 256, 448 / 256, 1.5):
            v = np.float32(r * 2.0 ** e)
            tops += [np.nextafter(v, np.float32(0)), v, np.nextafter(v, np.float32(np.inf))]
    tops += [np.float32(0), np.float32(-0.0), np.float32(1e-45), np.float32(1e-40), np.finfo(np.float32).max,
             np.float32(2.0 ** -10 * 6), np.float32(2.0 ** -11 * 6)]
    x = np.zeros((len(tops), 2 * b), np.float32)
    x[:, 3] = tops
    x[:, 4] = -np.array(tops) * np.float32(0.3)
    x[:, b] = -np.array(tops)
    check_exact(mx.quantize(torch.from_numpy(x).cuda(), fmt), x.astype(np.float64))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_infinities_and_nan_poison_their_block_alone(fmt, bad):
    x = rows_of(3, 200, torch.float32, seed=5)
    x[1, 70] = bad
    q = mx.quantize(x, fmt)
    check_exact(q, f64(x))
    y = f64(mx.dequantize(q))
    b = O.BLOCK[fmt]
    lo = 70 // b * b
    assert np.isnan(y[1, lo:lo + b]).all()
    y[1, lo:lo + b] = 0
    assert np.isfinite(y).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_strides_offsets_and_memory_behind_the_array(fmt):
    """Rows at any element offset and stride; wider rows of `data` and its rows behind the last are left alone."""
    base = rows_of(40, 700, torch.bfloat16, seed=9)
    for lo, cols in ((0, 264), (1, 264), (7, 333), (8, 128)):
        x = base[:, lo:lo + cols]
        check_exact(mx.quantize(x, fmt), f64(x))
        x = base[::3, lo:lo + cols]
        check_exact(mx.quantize(x, fmt), f64(x))
    cols, rows = 333, 37
    x = base[:rows, :cols]
    wide = torch.full((40, 512), 0xAB, dtype=torch.uint8, device="cuda")
    q = mx.empty(fmt, rows, cols)
    q = mx.Microscaled(fmt, rows, cols, wide[:rows], q.scales)
    N.check(N.lib().ancha_mx_quantize(x.data_ptr(), N.BF16, 700, byref(mx._array(q, 0, "q")), 0))
    width = -(-(cols if fmt == "mxf8" else (cols + 1) // 2) // 16) * 16
    assert (wide[rows:] == 0xAB).all() and (wide[:, width:] == 0xAB).all()
    check_exact(mx.Microscaled(fmt, rows, cols, wide[:rows, :width].contiguous(), q.scales), f64(x))
    assert np.array_equal(f64(mx.dequantize(q)), f64(mx.dequantize(mx.quantize(x, fmt))))


def test_empty_arrays():
    for fmt in FORMATS:
        x = torch.zeros((0, 64), device="cuda")
        q = mx.quantize(x, fmt)
        assert q.data.shape[0] == 0 and mx.dequantize(q).shape == (0, 64)
        q, s = mx.add_rms_norm(x, x, None, format=fmt)
        assert q.rows == 0 and s.shape == (0, 64)
        w = mx.quantize(rows_of(8, 64, torch.float32), fmt)
        assert mx.linear(q, w).shape == (0, 8)
        assert mx.linear(q, w, format=fmt).data.shape[0] == 0


def test_offsets_beyond_32_bits():
    """An array of more than 2^32 elements: its last rows, against the same rows alone."""
    rows, cols = 70000, 65536 - 32
    x = torch.empty((rows, cols), dtype=torch.float16, device="cuda")
    x[:-300] = 1
    x[-300:] = rows_of(300, cols, torch.float16, seed=2)
    q = mx.quantize(x, "mxf4")
    tail = mx.quantize(x[-300:], "mxf4")
    assert torch.equal(q.data[-300:], tail.data)
    assert torch.equal(q.scale_codes()[-300:], tail.scale_codes())
    y = mx.dequantize(q, torch.float16)
    assert torch.equal(y[-300:], mx.dequantize(tail, torch.float16))
    assert (y[:-300] == 1).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_very_wide_rows(fmt):
    """Two rows of fifty million columns: their blocks are those of the same elements in short rows."""
    cols, whole = 50_000_001, 49_999_872
    x = rows_of(2, 4096, torch.bfloat16, seed=3).repeat(1, cols // 4096 + 1)[:, :cols]
    q, short = mx.quantize(x, fmt), mx.quantize(x[:, :whole].reshape(-1, 1024), fmt)
    n = whole if fmt == "mxf8" else whole // 2
    assert torch.equal(q.data[:, :n].reshape(-1), short.data.reshape(-1))
    assert torch.equal(q.scale_codes()[:, :whole // BLOCK[fmt]].reshape(-1), short.scale_codes().reshape(-1))
    assert torch.equal(mx.dequantize(q, torch.bfloat16)[:, :whole].reshape(-1, 1024), mx.dequantize(short, torch.bfloat16))
    tail = mx.quantize(x[:, whole:].contiguous(), fmt)
    assert torch.equal(mx.dequantize(q)[:, whole:], mx.dequantize(tail))


# ---------------------------------------------------------------------------------------- norm

def check_norm(x, residual, gain, eps, fmt, g=None, **kw):
    q, s = mx.add_rms_norm(x, residual, gain, eps, fmt, scalar(g), **kw)
    if residual is not None:
        assert s.dtype == residual.dtype
        want = (residual.float() + x.float()).to(residual.dtype)
        assert torch.equal(s, want)
    y = O.rms_norm(f64(s), 1.0 if gain is None else f64(gain), eps)
    check_near(q, y, 4 * 2.0 ** -24 * np.abs(y))
    return q, s


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 512), (2, 8), (5, 31), (9, 384), (130, 129), (3, 520), (33, 1001),
                                      (2, 1024), (7, 1032), (3, 4096), (2, 5000), (2, 8200), (1, 20000), (1, 32768)])
def test_add_rms_norm_matches_oracle(fmt, rows, dim):
    x = rows_of(rows, dim, torch.bfloat16, seed=dim)
    r = rows_of(rows, dim, torch.float32, seed=dim + 1)
    gain = 1 + 0.1 * rows_of(1, dim, torch.float32, seed=3)[0]
    check_norm(x, r, gain, 1e-6, fmt, 0.01 if fmt == "nvf4" else None)


@pytest.mark.parametrize("x_type", DTYPES)
@pytest.mark.parametrize("r_type", [None, *DTYPES])
@pytest.mark.parametrize("dim", [384, 515])
def test_add_rms_norm_types(x_type, r_type, dim):
    x = rows_of(6, dim, DTYPES[x_type], seed=1)
    r = None if r_type is None else rows_of(6, dim, DTYPES[r_type], seed=2)
    for gain in (None, 1 + 0.1 * rows_of(1, dim, torch.float32, seed=3)[0]):
        q, s = check_norm(x, r, gain, 1e-5, "mxf8")
        if r is None:
            assert s is x


def test_add_rms_norm_in_place_and_strided():
    base = rows_of(20, 900, torch.float32, seed=4)
    for lo, dim in ((0, 384), (3, 385), (4, 384)):
        r = base.clone()[:, lo:lo + dim]
        x = rows_of(20, dim, torch.float16, seed=5)
        want, s = mx.add_rms_norm(x, r, None, format="mxf4")
        before = r.clone()
        whole = r._base.clone()
        q, s2 = mx.add_rms_norm(x, r, None, format="mxf4", residual_out=r)
        assert s2 is r and torch.equal(r, s) and not torch.equal(r, before)
        assert torch.equal(q.data, want.data) and torch.equal(q.scales, want.scales)
        whole[:, lo:lo + dim] = s
        assert torch.equal(r._base, whole)


@pytest.mark.parametrize("dim", [600, 1501, 5003, 20001])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_add_rms_norm_in_place_at_odd_widths(dim, kind):
    """The stream written over the residual, and over x, where rows cannot be read in vectors."""
    x, r = rows_of(5, dim, DTYPES[kind], 1), rows_of(5, dim, DTYPES[kind], 2)
    want, s = mx.add_rms_norm(x, r)
    for over in (0, 1):
        a, b = x.clone(), r.clone()
        q, s2 = mx.add_rms_norm(a, b, residual_out=(b, a)[over])
        assert torch.equal(s2, s) and torch.equal(q.data, want.data) and torch.equal(q.scales, want.scales)
        assert torch.equal((a, b)[over], (x, r)[over])  # the other one as it was


def test_add_rms_norm_does_not_depend_on_the_split():
    """The codes of a row are the same alone, among others, and at unaligned addresses."""
    for dim in (384, 1000, 4000, 9000):
        x, r = rows_of(40, dim, torch.float32, seed=6), rows_of(40, dim, torch.float32, seed=7)
        q, _ = mx.add_rms_norm(x, r, None)
        one, _ = mx.add_rms_norm(x[17:18], r[17:18], None)
        assert torch.equal(one.data[0], q.data[17])
        pad = torch.zeros(40, dim + 1, device="cuda")
        pad[:, 1:] = x
        odd, _ = mx.add_rms_norm(pad[:, 1:], r, None)
        assert torch.equal(odd.data, q.data) and torch.equal(odd.scales, q.scales)


@pytest.mark.parametrize("fmt", FORMATS)
def test_add_rms_norm_extreme_rows(fmt):
    """Zeros, values whose squares leave f32 in both directions, and NaN or infinities, row by row."""
    x = rows_of(6, 320, torch.float32, seed=8, spread=0)
    x[0] = 0
    x[1] *= 1e25
    x[2] *= 1e-25
    x[3] *= 1e-4
    y = O.rms_norm(f64(x), 1.0, 1e-6)
    q, _ = mx.add_rms_norm(x, format=fmt)
    check_near(q, y, 4 * 2.0 ** -24 * np.abs(y))
    check_near(mx.add_rms_norm(x, format=fmt, eps=1e-60)[0], O.rms_norm(f64(x), 1.0, 1e-60),
               4 * 2.0 ** -24 * np.abs(O.rms_norm(f64(x), 1.0, 1e-60)))
    x[4, 7] = math.nan
    x[5, 9] = math.inf
    d = f64(mx.dequantize(mx.add_rms_norm(x, format=fmt)[0]))
    assert np.isnan(d[4]).all()
    # inf / rms(inf) is NaN in its own block, and the other blocks' values are 0.
    b = O.BLOCK[fmt]
    assert np.isnan(d[5, 9 // b * b:9 // b * b + b]).all() and np.nansum(np.abs(d[5])) == 0
    assert np.isfinite(d[:4]).all()


# -------------------------------------------------------------------------------------- product

def gelu64(y):
    return 0.5 * y * (1 + np.vectorize(math.erf)(y / math.sqrt(2)))


def linear64(x, w, bias=None, act="none", residual=None):
    """(y, tolerance before the output's rounding) of quantised x and w in float64."""
    a, b = f64(mx.dequantize(x)), f64(mx.dequantize(w))
    # The expanded f32 values are exact but for nvf4, whose array scales multiply once more in f32.
    y, mass = a @ b.T, np.abs(a) @ np.abs(b).T
    tol = (x.cols + 2) * 2.0 ** -23 * mass + 2.0 ** -21 * mass * (x.format == "nvf4")
    if bias is not None:
        y = y + f64(bias)
        tol = tol + 2.0 ** -23 * (np.abs(f64(bias)) + mass)
    if act == "gelu":
        tol = 1.13 * tol + 7e-7  # |GELU'| < 1.13
        y = gelu64(y)
        tol = tol + 5e-6 * np.abs(y)
    elif act == "tanh":
        y = np.tanh(y)
        tol = tol + 3e-7
    if residual is not None:
        tol = tol + 2.0 ** -23 * (np.abs(y) + np.abs(f64(residual)))
        y = y + f64(residual)
    return y, tol


def check_linear(x, w, bias=None, act="none", residual=None, dtype=torch.float32):
    y, tol = linear64(x, w, bias, act, residual)
    got = mx.linear(x, w, bias, act, residual, dtype=dtype)
    assert got.dtype == dtype and got.shape == y.shape
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0
    err = np.abs(f64(got) - y)
    assert (err <= tol + HALF_STEP[dtype] * (np.abs(y) + tol) + tiny).all(), float((err / (tol + 1e-30)).max())
    return got


def operands(fmt, m, n, k, seed=0):
    g = (0.002, 0.0005) if fmt == "nvf4" else (None, None)
    x = mx.quantize(rows_of(m, k, torch.float32, seed, 0.3), fmt, scalar(g[0]))
    w = mx.quantize(rows_of(n, k, torch.float32, seed + 1, 0.3) / math.sqrt(k), fmt, scalar(g[1]))
    return x, w


SHAPES = [(1, 1, 1), (1, 7, 16), (1, 128, 32), (2, 130, 64), (3, 384, 384), (8, 96, 100), (16, 512, 1000), (17, 129, 129),
          (33, 65, 31), (64, 200, 256), (65, 257, 260), (100, 128, 2048), (127, 127, 127), (128, 128, 128), (128, 256, 256),
          (129, 385, 384), (200, 1544, 384), (256, 192, 640), (300, 520, 777), (1000, 384, 1536)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_matches_float64(fmt, m, n, k):
    x, w = operands(fmt, m, n, k, m + n + k)
    check_linear(x, w)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 300, 200), (40, 129, 96), (200, 391, 260), (260, 512, 300)])
@pytest.mark.parametrize("act", ["none", "gelu", "tanh"])
@pytest.mark.parametrize("out", DTYPES)
def test_linear_epilogues(fmt, m, n, k, act, out):
    x, w = operands(fmt, m, n, k, 3)
    bias = rows_of(1, n, torch.float32, 4)[0]
    check_linear(x, w, bias, act, None, DTYPES[out])
    for r in DTYPES.values():
        check_linear(x, w, bias, act, rows_of(m, n, r, 5, 0.2), DTYPES[out])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n", [(4, 256), (150, 300)])
def test_linear_strides_and_offsets(fmt, m, n):
    """A residual and a bias at odd offsets, rows of x and w wider than they need to be, out in place of the
    residual, and memory around the output left alone."""
    x, w = operands(fmt, m, n, 200, 6)
    wide = lambda q: mx.Microscaled(q.format, q.rows, q.cols, torch.nn.functional.pad(q.data, (0, 48), value=0xFF),  # noqa: E731
                                    q.scales, q.global_scale)
    bias = rows_of(1, n + 1, torch.float32, 7)[0, 1:]
    res = rows_of(m, n + 3, torch.bfloat16, 8)[:, 3:]
    want = mx.linear(x, w, bias, "gelu", res, dtype=torch.bfloat16)
    assert torch.equal(mx.linear(wide(x), wide(w), bias.clone(), "gelu", res.contiguous(), dtype=torch.bfloat16), want)
    for lo, ld in ((0, n + 8), (1, n + 5), (8, n + 8)):
        buf = torch.full((m + 2, ld + 8), 3.0, dtype=torch.bfloat16, device="cuda")
        view = buf[1:m + 1, lo:lo + n]
        view.copy_(res)
        ref = buf.clone()
        ref[1:m + 1, lo:lo + n] = want
        d = N.MxLinearDesc(N.ACT_GELU, N.BF16, N.BF16, ld + 8, ld + 8)
        N.check(N.lib().ancha_mx_linear_fwd(byref(d), byref(mx._array(x, 0, "x")), byref(mx._array(w, 0, "w")),
                                            bias.data_ptr(), view.data_ptr(), view.data_ptr(), None, 0))
        assert torch.equal(buf, ref)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("out", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 40), (1, 512, 256), (30, 100, 96), (129, 300, 384), (256, 515, 200), (384, 768, 128),
                                   (200, 65, 64), (300, 130, 64), (300, 321, 96), (130, 577, 64), (260, 449, 2080)])
def test_linear_with_quantized_output(fmt, out, m, n, k):
    """The quantised output is the quantisation of the f32 output, bit for bit."""
    x, w = operands(fmt, m, n, k, 9)
    bias, res = rows_of(1, n, torch.float32, 10)[0], rows_of(m, n, torch.float16, 11)
    g = scalar(0.01) if out == "nvf4" else None
    for args in ((bias, "gelu", None), (None, "none", res), (bias, "tanh", res)):
        got = mx.linear(x, w, *args, format=out, global_scale=g)
        want = mx.quantize(mx.linear(x, w, *args, dtype=torch.float32), out, g)
        assert torch.equal(got.data, want.data) and torch.equal(got.scales, want.scales)
        y, tol = linear64(x, w, *args)
        check_near(got, y, tol)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n", [(3, 200), (140, 200)])
def test_linear_with_poisoned_and_empty_rows(fmt, m, n):
    """A NaN block makes its row of x, or its column of w, NaN, and nothing else; zero rows give the bias."""
    k = 256
    xv, wv = rows_of(m, k, torch.float32, 1, 0), rows_of(n, k, torch.float32, 2, 0)
    bias = rows_of(1, n, torch.float32, 3)[0]
    xv[1] = 0
    xv[2, 100] = math.inf
    wv[7, 3] = math.nan
    x, w = mx.quantize(xv, fmt), mx.quantize(wv, fmt)
    y = f64(mx.linear(x, w, bias, dtype=torch.float32))
    assert np.isnan(y[2]).all() and np.isnan(y[:, 7]).all()
    ok = np.ones((m, n), bool)
    ok[2], ok[:, 7] = False, False
    assert np.isfinite(y[ok]).all()
    row = np.delete(y[1], 7)
    assert np.array_equal(row, np.delete(f64(bias), 7))
    keep = [i for i in range(m) if i != 2]
    keep_n = [i for i in range(n) if i != 7]
    check_linear(mx.quantize(xv[keep], fmt), mx.quantize(wv[keep_n], fmt), bias[keep_n].contiguous())


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("act", ["gelu", "tanh"])
def test_activations_at_their_ends(m, act):
    """Large sums, sums near zero, infinities (an overflowing sum) and NaN through the activations."""
    k, n = 64, 160
    w = mx.quantize(torch.eye(n, k, device="cuda"), "mxf8")
    x = torch.zeros((m, k), device="cuda")
    tops = [0.0, 1e-30, -1e-30, 1e-4, -1e-4, 3.0, -3.0, 5.5, -5.5, 8.0, -8.0, 256.0, -256.0, 2.0 ** 60, -2.0 ** 60]
    vals = torch.tensor([tops[i % len(tops)] for i in range(2 * m)], device="cuda").view(m, 2)
    x[:, 0], x[:, 32] = vals[:, 0], vals[:, 1]  # one value to a block
    x[1, 1] = math.nan
    bias = torch.zeros(n, device="cuda")
    bias[40], bias[41], bias[42] = math.inf, -math.inf, math.nan
    y = f64(mx.linear(mx.quantize(x, "mxf8"), w, bias, act, dtype=torch.float32))
    z = f64(mx.dequantize(mx.quantize(x, "mxf8"))) @ f64(mx.dequantize(w)).T + f64(bias)
    with np.errstate(invalid="ignore", over="ignore"):
        want = gelu64(z) if act == "gelu" else np.tanh(z)
    want = np.where(np.isneginf(z), 0.0 if act == "gelu" else -1.0, want)
    assert np.array_equal(np.isnan(y), np.isnan(want))
    ok = np.isfinite(want)
    assert np.array_equal(y[~ok & ~np.isnan(want)], want[~ok & ~np.isnan(want)])
    assert (np.abs(y[ok] - want[ok]) <= 7e-7 + 5e-6 * np.abs(want[ok])).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_is_deterministic_and_rows_are_independent(fmt):
    x, w = operands(fmt, 300, 520, 2000, 12)
    y = mx.linear(x, w, dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(mx.linear(x, w, dtype=torch.float32), y)


@pytest.mark.parametrize("n", [32768, 32771])
@pytest.mark.parametrize("kind", ["bf16", "mxf8", "mxf4"])
def test_linear_outputs_beyond_32_bits(n, kind):
    """An output of more than 2^31 elements: its last rows against float64."""
    m, k = 70016, 32
    x, w = operands("mxf8", m, n, k, 4)
    bias = rows_of(1, n, torch.float32, 5)[0]
    last = mx.quantize(mx.dequantize(x)[-100:], "mxf8")  # values of the format: quantised to themselves
    assert torch.equal(mx.dequantize(last), mx.dequantize(x)[-100:])
    y, tol = linear64(last, w, bias)
    if kind == "bf16":
        got = f64(mx.linear(x, w, bias)[-100:])
        assert (np.abs(got - y) <= tol + 2.0 ** -8 * (np.abs(y) + tol)).all()
        return
    q = mx.linear(x, w, bias, format=kind)
    width = -(-(n if kind == "mxf8" else (n + 1) // 2) // 16) * 16
    tail = mx.empty(kind, 100, n)
    tail.data.copy_(q.data[-100:, :width])
    codes = q.scale_codes()[-100:].cpu().numpy()
    tail.scales.copy_(torch.from_numpy(O.tile(codes)).view(tail.scales.shape))
    check_near(tail, y, tol)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [2, 200])
def test_linear_with_a_very_long_depth(fmt, m):
    x, w = operands(fmt, m, 5, 300_001, 6)
    check_linear(x, w)


# ------------------------------------------------------------------------------------- together

def feed_forward(branch, stream, gain, w1, b1, w2, b2, fmt, g):
    q, s = mx.add_rms_norm(branch, stream, gain, 1e-6, fmt, g)
    hidden = mx.linear(q, w1, b1, "gelu", format=fmt, global_scale=g)
    return q, s, hidden, mx.linear(hidden, w2, b2, "none", s, dtype=torch.float32)


def block(fmt, rows, dim, hidden, seed=0):
    g = scalar(0.01) if fmt == "nvf4" else None
    w1 = mx.quantize(rows_of(hidden, dim, torch.float32, seed + 1, 0) / math.sqrt(dim), fmt, g)
    w2 = mx.quantize(rows_of(dim, hidden, torch.float32, seed + 2, 0) / math.sqrt(hidden), fmt, g)
    return (rows_of(rows, dim, torch.bfloat16, seed + 3, 0), rows_of(rows, dim, torch.float32, seed + 4, 0),
            1 + 0.1 * rows_of(1, dim, torch.float32, seed + 5, 0)[0], w1, rows_of(1, hidden, torch.float32, seed + 6, 0)[0],
            w2, rows_of(1, dim, torch.float32, seed + 7, 0)[0], fmt, g)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,dim,hidden", [(1, 384, 1536), (70, 200, 520), (801, 384, 1536)])
def test_feed_forward_block(fmt, rows, dim, hidden):
    """Norm, product with quantised GELU output, product onto the stream: each step against float64 on what
    the step before it gave."""
    args = block(fmt, rows, dim, hidden)
    q, s, h, y = feed_forward(*args)
    assert torch.equal(s, args[1] + args[0].float())
    y64 = O.rms_norm(f64(s), f64(args[2]), 1e-6)
    check_near(q, y64, 4 * 2.0 ** -24 * np.abs(y64))
    y64, tol = linear64(q, args[3], args[4], "gelu")
    check_near(h, y64, tol)
    y64, tol = linear64(h, args[5], args[6], "none", s)
    assert (np.abs(f64(y) - y64) <= tol + 2.0 ** -24 * np.abs(y64)).all()


def test_two_streams_at_once_and_graphs():
    """Blocks on two streams at once, and two captured graphs replayed at once on new inputs, give what the
    blocks give one after the other."""
    a, b = block("mxf8", 500, 384, 1536, 0), block("nvf4", 3, 512, 2048, 50)
    want = [feed_forward(*a)[3], feed_forward(*b)[3]]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s1):
            y1 = feed_forward(*a)[3]
        with torch.cuda.stream(s2):
            y2 = feed_forward(*b)[3]
        torch.cuda.synchronize()
        assert torch.equal(y1, want[0]) and torch.equal(y2, want[1])
    graphs, outs = [], []
    for args in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(feed_forward(*args)[3])
        graphs.append(g)
    for scale in (1.0, 0.5, -2.0):
        a[0].copy_(rows_of(500, 384, torch.bfloat16, 77, 0) * scale)
        b[1].copy_(rows_of(3, 512, torch.float32, 78, 0) * scale)
        want = [feed_forward(*a)[3], feed_forward(*b)[3]]
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(s1):
                graphs[0].replay()
            with torch.cuda.stream(s2):
                graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_wrong_tensors_are_refused():
    x = rows_of(4, 64, torch.float32)
    q = mx.quantize(x, "mxf8")
    f = mx.quantize(x, "mxf4")
    bad = [lambda: mx.quantize(x.double()), lambda: mx.quantize(x[0]), lambda: mx.quantize(x.t()),
           lambda: mx.quantize(x, "mxf8", scalar(1.0)), lambda: mx.quantize(x, "nvf4", torch.ones(1)),
           lambda: mx.quantize(x, "nvf4", torch.ones(2, device="cuda")), lambda: mx.dequantize(q, torch.float64),
           lambda: mx.add_rms_norm(x, x[:3]), lambda: mx.add_rms_norm(x, x.cpu()), lambda: mx.add_rms_norm(x, gain=x),
           lambda: mx.add_rms_norm(x, eps=0.0), lambda: mx.add_rms_norm(x, x, residual_out=x.half()),
           lambda: mx.linear(q, f), lambda: mx.linear(q, mx.quantize(x[:, :32])), lambda: mx.linear(q, q, act="glu"),
           lambda: mx.linear(q, q, x[0]), lambda: mx.linear(q, q, residual=x), lambda: mx.linear(q, q, dtype=torch.int32),
           lambda: mx.linear(q, q, dtype=torch.float32, format="mxf8"), lambda: mx.linear(q, q, global_scale=scalar(1.0)),
           lambda: mx.linear(q, q, format="mxf8", global_scale=scalar(1.0)),
           lambda: mx.dequantize(mx.Microscaled("mxf8", 4, 64, q.data[:, :48], q.scales)),
           lambda: mx.dequantize(mx.Microscaled("mxf8", 4, 200, q.data, q.scales)),
           lambda: mx.dequantize(mx.Microscaled("mxf8", 4, 64, q.data, q.scales[..., :2])),
           lambda: mx.dequantize(mx.Microscaled("mxf8", 4, 64, q.data.int(), q.scales))]
    for call in bad:
        with pytest.raises(N.AnchaError):
            call()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_device_than_the_current_one():
    args = [a.to("cuda:1") if isinstance(a, torch.Tensor) else a for a in block("mxf4", 9, 384, 512)]
    move = lambda q: mx.Microscaled(q.format, q.rows, q.cols, q.data.to("cuda:1"), q.scales.to("cuda:1"))  # noqa: E731
    args[3], args[5] = move(args[3]), move(args[5])
    want = feed_forward(*block("mxf4", 9, 384, 512))[3]
    assert torch.cuda.current_device() == 0
    assert torch.equal(feed_forward(*args)[3].cpu(), want.cpu())
