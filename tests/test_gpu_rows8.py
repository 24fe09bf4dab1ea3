"""symmetric.rms_norm_quantize and silu_mul_quantize against their formulas in 64 bits.

The norm's codes are exact: h is one rounding of x + residual, u = h * weight has at most 22 significant bits, and 127 / top and its
product with u are single fp32 operations, which numpy does the same way.  Scales: the squares' sum goes through at most `adds`
additions one after the other (its square root halves that), then mean, eps, root, quotient, top / 127 and the product round once each.
The gated activation: exp2 takes a product and a constant rounded to 24 bits, so exp(-g) is off by at most 2 |g| 2^-24 and an ulp; with
reciprocal, two products and the sum behind it (2 |g| + 8) 2^-24 of a value, and the same of the row's largest."""
import numpy as np
import pytest
import torch

import quik

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]

# one to eight chunks of eight columns per lane and their ends, every workgroup size, odd widths, rows beyond the registers
SHAPES = [(1, 1), (1, 7), (3, 8), (2, 63), (5, 64), (1, 512), (4, 520), (2, 1000), (3, 1725), (33, 2048), (1, 4096), (7, 4099), (2, 5120),
          (3, 8200), (1, 11008), (5, 13824), (2, 16392), (1, 28672), (2, 32768), (2, 32767), (1, 32776), (3, 40001)]


def _adds(cols):
    return 40 if cols <= 32768 else 40 + cols // 1024


def _up(t):
    return t.double().cpu().numpy()


def _f32(t):
    return t.float().cpu().numpy()


def _norm_oracle(x, weight, eps, residual):
    h = x.cpu() if residual is None else (x.cpu().float() + residual.cpu().float()).to(x.dtype)
    with np.errstate(all="ignore"):
        u = _f32(h) * _f32(weight)
        top = np.abs(u).max(1, keepdims=True)
        inv = np.where(top > 0, np.float32(127) / top, np.float32(0)).astype(np.float32)
        q = np.nan_to_num(np.rint(u * inv))
        scale = top.astype(np.float64) / 127 / np.sqrt((_up(h) ** 2).mean(1, keepdims=True) + np.float64(np.float32(eps)))
    bad = ~np.isfinite(u).all(1) | ~np.isfinite(_f32(h)).all(1)
    q[bad] = 0
    scale[bad] = np.nan
    return np.clip(q, -127, 127).astype(np.int8), scale, h


def _check_scale(got, want, tol):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert (np.abs(got - want)[fine] <= tol * np.abs(want)[fine]).all()


def _input(rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * scale
    x[:, ::97] *= 30
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm(rows, cols, with_residual, dtype):
    x, r, w = _input(rows, cols, dtype, 1), _input(rows, cols, dtype, 2), _input(1, cols, dtype, 3)[0]
    q, scale, h = quik.symmetric.rms_norm_quantize(x, w, 1e-5, residual=r if with_residual else None)
    wq, ws, wh = _norm_oracle(x, w, 1e-5, r if with_residual else None)
    assert (h is None) == (not with_residual)
    if with_residual:
        assert torch.equal(h.cpu(), wh)
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and scale.shape == (rows, 1)
    assert np.array_equal(q.cpu().numpy(), wq)
    _check_scale(scale, ws, (_adds(cols) / 2 + 7) * 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_silu_mul(rows, cols, dtype):
    g, u = _input(rows, cols, dtype, 4).clamp(-30, 30), _input(rows, cols, dtype, 5)
    q, scale = quik.symmetric.silu_mul_quantize(g, u)
    _check_gated(q, scale, g, u)


def _check_gated(q, scale, g, u):
    v = _up(g) / (1 + np.exp(-_up(g))) * _up(u)
    top = np.abs(v).max(1, keepdims=True)
    off = (2 * 30 + 8) * 2.0 ** -24
    _check_scale(scale, top / 127, off + 2.0 ** -24)
    codes = np.divide(127 * v, top, out=np.zeros_like(v), where=top > 0)
    assert (np.abs(codes - q.cpu().numpy()) <= 0.5 + 127 * 2 * off).all()
    assert ((np.abs(q.cpu().numpy().astype(int)).max(1) == 127) | (top[:, 0] == 0)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [64, 1001, 4096, 33000])
def test_rows_that_hold_something_else(cols, dtype):
    """Zeros, one value, the type's largest, tiny numbers, NaN and infinities at either end; each row is on its own."""
    x, r, w = (_input(9, cols, dtype, s) for s in (6, 7, 8))
    w = w[0]
    big = torch.finfo(dtype).max
    x[0], r[0] = 0, 0
    x[1], r[1] = 0, 0
    x[1, cols - 1] = 3
    x[2, 0], r[2, 0] = big, big                      # the sum passes the type: an infinity
    x[3, cols - 1] = float("nan")
    r[4, cols // 2] = float("inf")
    r[5, 0], x[5, 0] = float("-inf"), float("inf")   # their sum is no number
    x[6], r[6] = 0, 0
    x[6, :7] = torch.finfo(dtype).smallest_normal / 8  # subnormals
    x[7], r[7] = 1, -1
    q, scale, h = quik.symmetric.rms_norm_quantize(x, w, 1e-5, residual=r)
    wq, ws, wh = _norm_oracle(x, w, 1e-5, r)
    if dtype == torch.bfloat16:   # products of 1e-39 and less: subnormal in fp32, made larger by 2^100 before the quotient
        small = _f32(wh)[6] * _f32(w) * np.float32(2.0 ** 100)
        inv = np.float32(127) / np.abs(small).max()
        wq[6] = np.rint(small * inv)
        assert abs(wq[6]).max() == 127
        ws[6] = np.nan                                # (its scale is subnormal: checked to whole steps below)
        assert abs(float(scale[6]) - float(np.abs(_f32(wh)[6] * _f32(w)).max()) / 127 / np.sqrt(1e-5)) <= 400 * 2.0 ** -149
        scale[6] = float("nan")
    assert np.isnan(ws[2:6]).all() and ws[0] == 0 and not q[0].any() and ws[7] == 0
    assert np.array_equal(q.cpu().numpy(), wq)
    assert torch.equal(h.cpu().isnan(), wh.isnan()) and torch.equal(h.cpu().nan_to_num(1), wh.nan_to_num(1))
    _check_scale(scale, ws, (_adds(cols) / 2 + 7) * 2.0 ** -24)
    # a weight that is no number is in every row
    w[3] = float("nan")
    q, scale, _ = quik.symmetric.rms_norm_quantize(x, w, 1e-5)
    assert scale.isnan().all() and not q.any()

    g, u = _input(5, cols, dtype, 9).clamp(-30, 30), _input(5, cols, dtype, 10)
    g[0], u[1] = 0, 0
    g[2, cols - 1], u[3, 0] = float("nan"), float("inf")
    g[4] = -200                                       # exp(200) passes fp32: the value is 0
    q, scale = quik.symmetric.silu_mul_quantize(g, u)
    assert scale[[0, 1, 4]].abs().max() == 0 and scale[[2, 3]].isnan().all() and not q.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,pitch,shift", [(64, 200, 8), (64, 201, 0), (1000, 1003, 3), (4096, 8192, 4096), (4096, 8196, 1), (13824, 27648, 0)])
def test_column_views(cols, pitch, shift, dtype):
    """Rows that lie apart, at any distance and alignment; what is not theirs is not read."""
    rows = 6
    whole, other, w = torch.full((rows, pitch), float("nan"), dtype=dtype, device=DEV), _input(rows, pitch, dtype, 11), _input(1, cols, dtype, 12)[0]
    shift = min(shift, pitch - cols)
    whole[:, shift:shift + cols] = _input(rows, cols, dtype, 13).clamp(-30, 30)
    x, r = whole[:, shift:shift + cols], other[:, :cols]
    for residual in (None, r):
        got, want = quik.symmetric.rms_norm_quantize(x, w, residual=residual), \
            quik.symmetric.rms_norm_quantize(x.contiguous(), w, residual=None if residual is None else residual.contiguous())
        wq, ws, _ = _norm_oracle(x, w, 1e-6, residual)
        assert np.array_equal(got[0].cpu().numpy(), wq)
        _check_scale(got[1], ws, (_adds(cols) / 2 + 7) * 2.0 ** -24)
        assert torch.equal(got[0], want[0]) and (residual is None or torch.equal(got[2], want[2]))
    q, scale = quik.symmetric.silu_mul_quantize(x, r)
    _check_gated(q, scale, x, r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale_dtype", TYPES)
def test_scales_of_16_bits(dtype, scale_dtype):
    x, w = _input(40, 1000, dtype, 14), _input(1, 1000, dtype, 15)[0]
    q, s, _ = quik.symmetric.rms_norm_quantize(x, w)
    q16, s16, _ = quik.symmetric.rms_norm_quantize(x, w, scale_dtype=scale_dtype)
    assert torch.equal(q, q16) and s16.dtype == scale_dtype and torch.equal(s.to(scale_dtype), s16)
    q, s = quik.symmetric.silu_mul_quantize(x, x)
    q16, s16 = quik.symmetric.silu_mul_quantize(x, x, scale_dtype=scale_dtype)
    assert torch.equal(q, q16) and torch.equal(s.to(scale_dtype), s16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [64, 1001, 4096, 16384, 30000, 40000])
def test_sum_in_the_place_of_an_input(cols, dtype):
    from quik_amd import _lib as L
    rows, x, r, w = 5, _input(5, cols, dtype, 19), _input(5, cols, dtype, 20), _input(1, cols, dtype, 21)[0]
    wq, ws, wh = quik.symmetric.rms_norm_quantize(x, w, residual=r)
    for place in (0, 1):
        both = [x.clone(), r.clone()]
        q, scale = torch.empty_like(wq), torch.empty_like(ws)
        L.check(L.load().quik_rms_norm_quantize(L.ptr(both[0]), cols, L.ptr(both[1]), cols, L.ptr(w), 1e-6, L.dtype_id(x, "", True), rows, cols,
                                                L.ptr(both[place]), L.ptr(q), L.ptr(scale), L.QUIK_F32, L.stream()), "")
        assert torch.equal(both[place], wh) and torch.equal(q, wq) and torch.equal(scale, ws)
        assert torch.equal(both[1 - place], (r, x)[place])


def test_more_rows_than_workgroups_and_offsets_past_32_bits():
    w = _input(1, 8, torch.float16, 22)[0]
    x = torch.ones((1 << 20) + 3, 8, dtype=torch.float16, device=DEV)
    x[-1] = _input(1, 8, torch.float16, 23)[0]
    q, scale, _ = quik.symmetric.rms_norm_quantize(x, w)
    for i in (0, 1 << 20, -1):
        one = quik.symmetric.rms_norm_quantize(x[i:][:1], w)
        assert torch.equal(q[i], one[0][0]) and torch.equal(scale[i], one[1][0])
    cols, rows = 32768, (1 << 16) + 2                 # 2^31 and some elements
    g = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    g[-2:] = _input(2, cols, torch.bfloat16, 24)
    w = _input(1, cols, torch.bfloat16, 25)[0]
    q, scale, h = quik.symmetric.rms_norm_quantize(g, w, residual=g)
    a, b, c = quik.symmetric.rms_norm_quantize(g[-2:], w, residual=g[-2:])
    assert torch.equal(q[-2:], a) and torch.equal(scale[-2:], b) and torch.equal(h[-2:], c) and not scale[:-2].any()
    del h
    q, scale = quik.symmetric.silu_mul_quantize(g, g)
    a, b = quik.symmetric.silu_mul_quantize(g[-2:], g[-2:])
    assert torch.equal(q[-2:], a) and torch.equal(scale[-2:], b) and not scale[:-2].any()


def test_empty_batch():
    x = torch.empty(0, 64, dtype=torch.float16, device=DEV)
    q, s, h = quik.symmetric.rms_norm_quantize(x, torch.ones(64, dtype=torch.float16, device=DEV), residual=x)
    assert q.shape == (0, 64) and s.shape == (0, 1) and h.shape == (0, 64)
    q, s = quik.symmetric.silu_mul_quantize(x, x)
    assert q.shape == (0, 64) and s.shape == (0, 1)


def test_into_the_eight_bit_product():
    """The norm's rows in the product that takes int8 operands and fp16 row scales."""
    x, w = _input(64, 512, torch.float16, 16), _input(1, 512, torch.float16, 17)[0]
    q, s, _ = quik.symmetric.rms_norm_quantize(x, w, scale_dtype=torch.float16)
    g = torch.Generator().manual_seed(18)
    b = torch.randint(-127, 128, (96, 512), generator=g, dtype=torch.int8).to(DEV)
    sc, y = torch.full((1, 96), 2.0 ** -10, dtype=torch.float16, device=DEV), torch.zeros(64, 96, dtype=torch.float16, device=DEV)
    acc = quik.matmul.int8Matmul(q, b)
    assert np.array_equal(acc.cpu().numpy(), q.cpu().numpy().astype(np.int64) @ b.cpu().numpy().astype(np.int64).T)
    assert torch.equal(quik.symmetric.int8FusedDequantize(q, b, s, sc, y), quik.symmetric.dequantize(acc, s, sc, y, 32))
