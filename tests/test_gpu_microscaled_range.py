"""Microscaled operators at the ends of the value range, against float64.

Tolerances, beside test_gpu_microscaled.py's. The inputs of the activations here are sums of one product, which are
exact, so what is off is the activation alone:

* tanh: relative 1e-6 (below 0.5 an odd polynomial, off by less than 1e-7 in f32; above it 1 - 2 / (e^2x + 1), whose
  exponential is off by 2^-22, whose reciprocal by 2^-23 and whose other steps by 2^-24 each, so 9.1e-7 of tanh);
* GELU: 2.5e-7 absolute and half a step of f32 (the fit is off by 8e-8, the polynomial's f32 steps and the exponential by
  1.3e-7 together), and for negative arguments also relative: 1e-3 down to -5.5, 8e-3 below (the fit of log2 Phi is off by
  8e-4 and 6e-3 of Phi), down to f32's least normal number, below which the exponential is 0."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ancha_b200 import microscaled as mx  # noqa: E402
from oracle import microscaled as O  # noqa: E402
from test_gpu_microscaled import FORMATS, check_near, f64, poisoned_memory, rows_of, scalar  # noqa: E402,F401

LEAST = 2.0 ** -126  # f32's least normal number


# ---------------------------------------------------------------------------------------- norm

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [1, 320, 600, 1500, 4000, 8192, 20001])
def test_norm_of_zero_and_extreme_rows_with_any_eps(fmt, dim):
    """Rows of zeros are zeros whatever eps is; rows of subnormal numbers and of numbers next to f32's largest have
    the norm of any other row."""
    x = rows_of(6, dim, torch.float32, seed=dim, spread=0)
    x[0] = 0
    x[1] *= 1e-44
    x[2] *= 1e-40
    x[3] *= 1e-30
    x[4] = torch.clamp(x[4], -3, 3) * 1e38
    for eps in (1e-30, 1e-76, 1e-78, 1e-100, 1e-300, 5e-324):
        y = O.rms_norm(f64(x), 1.0, eps)
        q, _ = mx.add_rms_norm(x, None, None, eps, fmt)
        assert not f64(mx.dequantize(q))[0].any()
        check_near(q, y, 4 * 2.0 ** -24 * np.abs(y))


# --------------------------------------------------------------------------------- activations

def sums(m, top):
    """x and w whose product is x itself: [m, 256] numbers up to about 4 `top`, a row of one size each, from `top` down
    by 2^-40 over the rows, their blocks' elements from full size to nothing."""
    k = 256
    rng = np.random.default_rng(m)
    v = rng.standard_normal((m, k)) * np.exp2(-rng.uniform(0, 8, (m, k))) * np.exp2(-40 * np.arange(m) / m)[:, None] * top
    x = mx.quantize(torch.from_numpy(v).float().cuda(), "mxf8")
    return x, mx.quantize(torch.eye(k, device="cuda"), "mxf8"), f64(mx.dequantize(x))


def gelu64(z):
    return np.vectorize(lambda t: 0.5 * t * math.erfc(-t / math.sqrt(2)))(z)


def activation(act, z):
    """(activation, tolerance) in float64."""
    if act == "tanh":
        y = np.tanh(z)
        return y, 1e-6 * np.abs(y)
    y = gelu64(z)
    tol = 2.5e-7 + 2.0 ** -24 * np.abs(y)
    rel = np.where(z < -5.5, 8e-3, 1e-3)
    return y, np.where(z < 0, np.minimum(tol, rel * np.abs(y) + 16 * LEAST), tol)


@pytest.mark.parametrize("m", [3, 40, 300])
@pytest.mark.parametrize("act", ["tanh", "gelu"])
@pytest.mark.parametrize("top", [4.0, 0.05])
def test_activations_over_their_range(m, act, top):
    x, w, z = sums(m, top)
    y, tol = activation(act, z)
    got = f64(mx.linear(x, w, None, act, dtype=torch.float32))
    assert (np.abs(got - y) <= tol).all(), float((np.abs(got - y) / (tol + 1e-300)).max())


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("fmt", FORMATS)
def test_small_tanh_keeps_its_blocks(m, fmt):
    """Blocks of small sums, whose scale and codes are those of tanh and not of its rounding."""
    x, w, z = sums(m, 0.05)
    y, tol = activation("tanh", z)
    g = 2.0 ** -30 if fmt == "nvf4" else None
    check_near(mx.linear(x, w, None, "tanh", format=fmt, global_scale=scalar(g)), y, tol)


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lo,hi", [(-5.5, -4.0), (-7.0, -5.6), (-12.5, -9.0), (-6.0, -5.0), (-3e4, -20.0)])
def test_gelu_of_negative_sums_keeps_its_blocks(m, fmt, lo, hi):
    """Blocks of sums so negative that GELU is next to nothing: their scale and codes are those of what is left."""
    k = 256
    v = np.random.default_rng(m).uniform(lo, hi, (m, k))
    x = mx.quantize(torch.from_numpy(v).float().cuda(), "mxf8")
    z = f64(mx.dequantize(x))
    y, tol = activation("gelu", z)
    w = mx.quantize(torch.eye(k, device="cuda"), "mxf8")
    got = f64(mx.linear(x, w, None, "gelu", dtype=torch.float32))
    assert (np.abs(got - y) <= tol).all(), float((np.abs(got - y) / tol).max())
    g = max(np.abs(y).max() / (6 * 448), 2.0 ** -120) if fmt == "nvf4" else None
    check_near(mx.linear(x, w, None, "gelu", format=fmt, global_scale=scalar(g)), y, tol)


def test_gelu_does_not_depend_on_its_neighbours():
    """The same sums give the same bits beside very negative ones and without them."""
    k, m = 256, 300
    v = torch.from_numpy(np.random.default_rng(7).uniform(-5.4, 9, (m, k))).float().cuda()
    far = v.clone()
    far[:, ::64] = -7.0
    w = mx.quantize(torch.eye(k, device="cuda"), "mxf8")
    a, b = (mx.linear(mx.quantize(t, "mxf8"), w, None, "gelu", dtype=torch.float32) for t in (v, far))
    same = mx.dequantize(mx.quantize(v, "mxf8")) == mx.dequantize(mx.quantize(far, "mxf8"))
    assert same.float().mean() > 0.9 and torch.equal(a[same], b[same])


# -------------------------------------------------------------------------------- array scales

@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gx,gw,size", [(3e-22, 5e-22, 1.0), (7e-20, 2e-25, 1.0), (1e-30, 1e-30, 1.0), (2e30, 1e9, 2.0 ** -7),
                                        (1e30, 1e-31, 1.0)])
def test_products_of_extreme_array_scales(m, out, gx, gw, size):
    """Array scales whose product leaves f32's normal numbers: the products of the arrays need not."""
    n, k = 200, 96

    def operand(rows, seed):  # an array without an array scale, whose row 1 holds zeros
        v = np.random.default_rng(seed).standard_normal((rows, k)) * (2000 if size == 1.0 else size)
        v[1] = 0
        return mx.quantize(torch.from_numpy(v).float().cuda(), "nvf4")

    x, w = operand(m, 1), operand(n, 2)
    a, b = f64(mx.dequantize(x)), f64(mx.dequantize(w))
    x.global_scale, w.global_scale = scalar(gx), scalar(gw)
    g = float(np.float32(gx)) * float(np.float32(gw))
    y, mass = (a @ b.T) * g, (np.abs(a) @ np.abs(b).T) * g
    top = float(torch.finfo(out).max)
    got = f64(mx.linear(x, w, dtype=out))
    assert np.isfinite(got[np.abs(y) < top * 0.99]).all() and not got[1].any()
    ok = np.isfinite(got)
    assert ok.mean() > 0.9
    # Sum and product as ever; what is below f32's least normal number rounds to its subnormal step.
    tol = (k + 4) * 2.0 ** -23 * mass + (0 if out == torch.float32 else 2.0 ** -8) * np.abs(y) + 2.0 ** -132
    assert (np.abs(got - y)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("g", [2.0 ** -149, 1e-38, 5e37, 2.0 ** 125])
def test_quantisation_with_the_ends_of_the_array_scale(g):
    """The least number of f32, and the largest of which six are one."""
    x = torch.clamp(rows_of(20, 200, torch.float32, 1, 0), -3, 3) * (1e38 if g > 1 else 1e-37)
    x[3] = 0
    q = mx.quantize(x, "nvf4", scalar(g))
    check_near(q, f64(x), 2.0 ** -22 * np.abs(f64(x)) + 2.0 ** -149)
    assert f64(mx.dequantize(q)).any()


@pytest.mark.parametrize("m", [3, 300])
def test_zeros_with_the_array_scale_of_zeros(m):
    """max|x| / (6 * 448) of an array of zeros is 0: the array and its products are zeros."""
    x, v = torch.zeros((m, 200), device="cuda"), rows_of(130, 200, torch.float32, 2)
    q, w = mx.quantize(x, "nvf4", x.abs().max().view(1) / (6 * 448)), mx.quantize(v, "nvf4", scalar(0.001))
    assert not mx.dequantize(q).any() and not mx.linear(q, w).any() and not mx.linear(w, q).any()
    s, _ = mx.add_rms_norm(x, None, None, format="nvf4", global_scale=q.global_scale)
    assert not mx.dequantize(s).any() and not mx.linear(s, w).any()
    y = mx.linear(q, w, format="nvf4", global_scale=q.global_scale)
    assert not mx.dequantize(y).any()


# --------------------------------------------------------------------------- rounding of the stream

@pytest.mark.parametrize("kind,half", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_the_stream_is_added_in_f32_and_then_rounded(kind, half):
    """A sum just above a tie of the stream's type, by less than f32 holds: the f32 sum is the tie, which goes to
    the even number. A sum of two 16-bit numbers that f32 does not hold is never next to a tie."""
    x = torch.full((2, 64), half, device="cuda")
    x[:, 1::2] *= 1 + 2.0 ** -20
    r = torch.ones((2, 64), dtype=kind, device="cuda")
    _, s = mx.add_rms_norm(x, r)
    assert s.dtype == kind and (s == 1).all()
    x[:, 0::2] *= 1 + 2.0 ** -10  # f32 holds this one
    _, s = mx.add_rms_norm(x, r)
    assert (s[:, 0::2].double() == 1 + 2 * half).all() and (s[:, 1::2] == 1).all()
