"""symmetric.rms_norm_quantize and silu_mul_quantize where fp32 runs out of range on the way: eps of 0, squares below fp32's smallest
number, gates whose exponential passes it.

Tolerances, in units of u = 2^-24 (half a step of fp32 relative to the value).  Norm: the codes are exact.  Its scale: at most `adds`
additions of the squares one after the other, the squares' own rounding, mean and eps (the root halves all of these), then root, reciprocal,
top / 127 and the product, one each.  The gated activation: see `_gated`."""
import numpy as np
import pytest
import torch

import quik

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]
WIDTHS = [8, 63, 64, 1001, 4096, 16390, 32768, 40001]   # one chunk of eight and its ends, every number of chunks per lane, beyond the registers


def _up(t):
    return t.double().cpu().numpy()


def _random(rows, cols, seed):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed))


def _norm_tolerance(cols):
    adds = 40 if cols <= 32768 else 40 + cols // 1024
    return ((adds + 3) / 2 + 4) * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_rows_of_zeros_without_eps(cols, dtype):
    """Codes 0 and scale 0, whatever eps is; also where the weight makes them so."""
    x, w = _random(3, cols, 1).to(dtype).to(DEV), torch.ones(cols, dtype=dtype, device=DEV)
    r = _random(3, cols, 2).to(dtype).to(DEV)
    r[1], x[1] = 1, -1
    zero = torch.zeros_like(x)
    for eps in (0.0, 1e-60, 1e-5):                     # (1e-60: 0 in fp32)
        q, scale, _ = quik.symmetric.rms_norm_quantize(zero, w, eps)
        assert not q.any() and torch.equal(scale, torch.zeros_like(scale))
        q, scale, _ = quik.symmetric.rms_norm_quantize(x, torch.zeros_like(w), eps)
        assert not q.any() and torch.equal(scale, torch.zeros_like(scale))
        q, scale, h = quik.symmetric.rms_norm_quantize(x, w, eps, residual=r)
        assert not h[1].any() and not q[1].any() and scale[1] == 0
        assert (scale[[0, 2]] > 0).all() and scale.isfinite().all() and q[0].any() and q[2].any()
    x[0, cols - 1] = float("nan")                      # and a row that is no number stays one
    q, scale, _ = quik.symmetric.rms_norm_quantize(x, torch.zeros_like(w), 0.0)
    assert scale[0].isnan() and scale[1] == 0 and not q.any()


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -149, 1e-38, 1e-31, 1e-12])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("cols", WIDTHS)
def test_norm_of_tiny_numbers(cols, with_residual, eps):
    """bf16 rows from the smallest subnormal up, whose squares fp32 does not hold: the scale is that of the formula."""
    powers = [-133, -130, -126, -110, -80, -64, -55, -49, -40, 0]
    x = torch.zeros(len(powers), cols, dtype=torch.float64)
    for i, p in enumerate(powers):
        x[i] = (_random(1, cols, 10 + i)[0].double() * 2.0 ** p).float().double()
        x[i, i % cols] = 2.0 ** p                      # (something is left of each)
    x = x.to(torch.bfloat16).to(DEV)
    w = (1 + 0.25 * _random(1, cols, 3)[0].clamp(-2, 2)).to(torch.bfloat16).to(DEV)
    q, scale, h = quik.symmetric.rms_norm_quantize(x, w, eps, residual=torch.zeros_like(x) if with_residual else None)
    assert h is None or torch.equal(h, x)
    u = _up(x) * _up(w)                                # (products of 8 bits at 2^-133 and 2^-8: whole steps of fp32)
    top = np.abs(u).max(1, keepdims=True)
    want = top / 127 / np.sqrt((_up(x) ** 2).mean(1, keepdims=True) + np.float64(np.float32(eps)))
    got = scale.double().cpu().numpy()
    assert np.isfinite(got).all()
    # (a scale below fp32's normal numbers: whole steps)
    assert (np.abs(got - want) <= _norm_tolerance(cols) * want + (want < 2.0 ** -126) * 2.0 ** -149).all()
    codes = 127 * u / top
    assert (np.abs(codes - q.cpu().numpy()) <= 0.5 + 127 * 2 * 2.0 ** -24).all()
    assert (np.abs(q.cpu().numpy().astype(int)).max(1) == 127).all()


def _gated(g, u):
    """The value in 64 bits and what it may be off by, relative to it: exp2's argument is |g| times a rounded constant, rounded (log2 e is off by
    a quarter of u: 1.25 u |g| of the exponential; 1.5 here), and exp2 is good to an ulp (2 u), reciprocal likewise, the sum and up to four
    products 1 u each: 9 u, and one for what these have in common.  Below -86 two exponentials of half the gate: the same |g| in all, 4 u and
    three products."""
    g, u = _up(g), _up(u)
    with np.errstate(over="ignore"):
        return np.where(g < 0, g * np.exp(g) / (1 + np.exp(np.minimum(g, 0))), g / (1 + np.exp(-np.abs(g)))) * u, (1.5 * np.abs(g) + 10) * 2.0 ** -24


def _check_gated(q, scale, g, u):
    v, off = _gated(g, u)
    top, at = np.abs(v).max(1, keepdims=True), np.abs(v).argmax(1)
    most = (off * np.abs(v)).max(1, keepdims=True) / top   # of the row's largest
    got = scale.double().cpu().numpy()
    assert (np.abs(got - top / 127) <= (most + 2.0 ** -23) * top / 127 + (top < 2.0 ** -119) * 2.0 ** -149).all()
    codes = 127 * v / top
    assert (np.abs(codes - q.cpu().numpy()) <= 0.5 + 127 * (most + off * np.abs(v) / top + 2.0 ** -22)).all()
    assert (np.abs(q.cpu().numpy().astype(int)).max(1) == 127).all()


@pytest.mark.parametrize("cols", WIDTHS)
def test_gates_whose_exponential_passes_fp32(cols):
    """bf16: gates down to -170 with the largest factors there are, each row around one gate."""
    gates = [-20, -44, -60, -86, -87.5, -88, -88.5, -89, -100, -126, -140, -160, -170]
    g = torch.tensor(gates).reshape(-1, 1) + 2 * _random(len(gates), cols, 5).clamp(-1, 1)
    u = _random(len(gates), cols, 6) * 2.0 ** 124
    g, u = g.to(torch.bfloat16).to(DEV), u.to(torch.bfloat16).to(DEV)
    q, scale = quik.symmetric.silu_mul_quantize(g, u)
    _check_gated(q, scale, g, u)


@pytest.mark.parametrize("cols", WIDTHS)
def test_gates_of_one_row_from_end_to_end(cols):
    """A row's largest value at a gate of -88: gates above it have small factors."""
    g = torch.linspace(-100, 40, cols).reshape(1, -1).repeat(2, 1)
    g[:, cols // 2] = -88
    u = _random(2, cols, 7)
    u[:, cols // 2] = 2.0 ** 127
    u[:, g[0] > -88] *= 2.0 ** -4
    g, u = g.to(torch.bfloat16).to(DEV), u.to(torch.bfloat16).to(DEV)
    q, scale = quik.symmetric.silu_mul_quantize(g, u)
    _check_gated(q, scale, g, u)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_rows_of_closed_gates(cols, dtype):
    """Nothing but gates around -88: values of 1e-37 and the like, which fp32 holds."""
    g = (-88 + _random(4, cols, 8).clamp(-2, 2)).to(dtype).to(DEV)
    u = (500 * _random(4, cols, 9)).to(dtype).to(DEV)
    q, scale = quik.symmetric.silu_mul_quantize(g, u)
    _check_gated(q, scale, g, u)


@pytest.mark.parametrize("dtype", TYPES)
def test_gates_that_are_shut(dtype):
    """Beyond that a gate counts as 0; infinities and NaNs are no numbers."""
    big = torch.finfo(dtype).max
    g, u = torch.full((6, 100), -200.0), torch.full((6, 100), 3.0)
    g[1], u[1] = -big, big
    g[2, 5], u[2, 5] = -float("inf"), 1
    g[3, 5], u[3, 5] = -180, float("inf")
    g[4, 5], u[4, 5] = 0, -float("inf")
    g[5, 5], u[5, 5] = float("nan"), 0
    q, scale = quik.symmetric.silu_mul_quantize(g.to(dtype).to(DEV), u.to(dtype).to(DEV))
    assert not q.any() and (scale[:2] == 0).all() and scale[2:].isnan().all()
