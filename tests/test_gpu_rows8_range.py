"""symmetric.rms_norm_quantize where fp32 runs out of range on the way: eps of 0, squares below fp32's smallest number.

Tolerances, in units of u = 2^-24 (half a step of fp32 relative to the value).  Norm: the codes are exact.  Its scale: at most `adds`
additions of the squares one after the other, the squares' own rounding, mean and eps (the root halves all of these), then root, reciprocal,
top / 127 and the product, one each."""
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
