"""Rows in blocks of 32: codes and exponent bytes against 64-bit arithmetic, element by element."""
import pytest
import torch

import mx_plain as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]


def ms():
    from quik import microscaled
    return microscaled


def check_codes(got, v, bits):
    q, scale = (t.cpu() for t in got)
    c, e = P.codes(v, bits)
    assert torch.equal(scale.to(torch.int64), e)
    assert torch.equal(P.unpack(q), c)


def hard_rows(gen, rows, cols, dtype):
    """Numbers of all magnitudes, ties of the codes among them, blocks of zeros, of one number, of the type's smallest and largest."""
    x = torch.randn(rows, cols, generator=gen) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=gen).float())
    x = x.to(dtype)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.5, 6.0, -0.25, -1.25, -5.0, 0.0, -0.0, 7.0, 4.0], dtype=dtype)
    x[0, :min(cols, 16)] = ties[:min(cols, 16)]
    if rows > 1:
        x[1] = 0
    if rows > 2:
        x[2] = torch.finfo(dtype).smallest_normal / 4
        x[2, ::3] = -torch.finfo(dtype).max
    if rows > 3:
        x[3] = torch.finfo(dtype).smallest_normal / 8
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,cols", [(1, 2), (1, 32), (3, 30), (5, 34), (4, 64), (7, 250), (2, 4096), (33, 1000), (300, 4544), (1, 40000)])
def test_quantize(dtype, bits, rows, cols):
    x = hard_rows(torch.Generator().manual_seed(rows * cols), rows, cols, dtype)
    check_codes(ms().quantize(x.to(DEV), bits), x.double(), bits)


def test_quantize_8_bits_of_odd_widths():
    for cols in (1, 31, 33, 77):
        x = hard_rows(torch.Generator().manual_seed(cols), 5, cols, torch.float16)
        check_codes(ms().quantize(x.to(DEV), 8), x.double(), 8)


@pytest.mark.parametrize("bits", [4, 8])
def test_every_bf16_number(bits):
    """Each number beside 31 that lie 0 to 30 binades below it."""
    top = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(torch.bfloat16)
    top = top[torch.isfinite(top)]
    x = (top.double().unsqueeze(1) * torch.exp2(-torch.arange(32, dtype=torch.float64) / 2)).to(torch.bfloat16)
    check_codes(ms().quantize(x.to(DEV), bits), x.double(), bits)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
def test_strided_rows_and_unaligned_starts(dtype, bits):
    gen = torch.Generator().manual_seed(3)
    wide = hard_rows(gen, 9, 4 * 96 + 3, dtype).to(DEV)
    for lo, hi in ((0, 96), (1, 97), (3, 3 + 4 * 96), (2, 72)):
        part = wide[:, lo:hi]
        check_codes(ms().quantize(part, bits), part.cpu().double(), bits)
    check_codes(ms().quantize(wide[::2, 8:72], bits), wide[::2, 8:72].cpu().double(), bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_blocks_without_a_number(bits, bad):
    x = torch.randn(3, 100, generator=torch.Generator().manual_seed(1)).half()
    x[1, 40], x[2, 99] = bad, bad
    q, scale = ms().quantize(x.to(DEV), bits)
    check_codes((q, scale), x.double(), bits)
    back = ms().dequantize(q, scale).cpu()
    want = torch.zeros(3, 100, dtype=torch.bool)
    want[1, 32:64] = want[2, 96:] = True
    assert torch.equal(back.isnan(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shape", [(1, 2), (5, 32), (6, 250), (4, 3, 80), (2, 5, 3, 34), (130, 8, 128)])
def test_dequantize(dtype, bits, shape):
    gen = torch.Generator().manual_seed(len(shape) + shape[-1])
    rows = 1
    for n in shape[:-1]:
        rows *= n
    c, e = P.random_rows(gen, rows, shape[-1], bits, 12)
    q, scale = P.pack(c, bits).reshape(*shape[:-1], -1).to(DEV), e.to(torch.uint8).reshape(*shape[:-1], -1).to(DEV)
    v = P.numbers(c, e, bits)
    assert torch.equal(ms().dequantize(q, scale, dtype).cpu(), v.to(dtype).reshape(shape))
    index = torch.randint(-1, shape[0] + 1, (7,), generator=gen)
    index[0], index[1] = -2 ** 62, 2 ** 62
    got = ms().dequantize(q, scale, dtype, rows=index.to(DEV)).cpu()
    there = (index >= 0) & (index < shape[0])
    want = torch.where(there.view(-1, *[1] * (len(shape) - 1)), v.to(dtype).reshape(shape)[index.clamp(0, shape[0] - 1)], 0)
    assert torch.equal(got, want)
    factor = torch.rand(7, 1, generator=gen) + 0.5
    got = ms().dequantize(q, scale, dtype, rows=index.to(DEV), scale_row=factor.to(DEV)).cpu()
    # one product in fp32, then the rounding to the type
    scaled = v.float().reshape(shape)[index.clamp(0, shape[0] - 1)] * factor.view(-1, *[1] * (len(shape) - 1))
    assert torch.equal(got, torch.where(there.view(-1, *[1] * (len(shape) - 1)), scaled, 0).to(dtype))


def test_every_code_and_exponent_comes_back():
    for bits in (4, 8):
        n = 16 if bits == 4 else 256
        c = torch.arange(n).repeat(256, 32 // n if n < 32 else 1)
        e = torch.arange(256).unsqueeze(1).expand(256, c.shape[1] // 32).contiguous()
        got = ms().dequantize(P.pack(c, bits).to(DEV), e.to(torch.uint8).to(DEV), torch.bfloat16).cpu()
        want = P.numbers(c, e, bits).to(torch.bfloat16)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))


def norm_reference(x, residual, gain, eps):
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    d = h.double()
    return h, d * gain.double(), 1 / torch.sqrt(d.pow(2).mean(1, keepdim=True) + eps)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 2), (1, 64), (5, 34), (3, 250), (2, 4096), (37, 5120), (2, 8200), (1, 40000), (800, 5120), (1030, 4114)])
def test_norm(dtype, bits, with_residual, rows, cols):
    gen = torch.Generator().manual_seed(rows + cols)
    x = (torch.randn(rows, cols, generator=gen) * 3).to(dtype)
    x[:, ::128] *= 10
    r = torch.randn(rows, cols, generator=gen).to(dtype) if with_residual else None
    gain = (1 + 0.2 * torch.randn(cols, generator=gen)).to(dtype)
    if rows > 2:
        x[1] = 0
        if r is not None:
            r[1] = 0
    q, scale, factor, h = ms().rms_norm_quantize(x.to(DEV), gain.to(DEV), 1e-5, None if r is None else r.to(DEV), bits)
    want_h, u, f = norm_reference(x, r, gain, 1e-5)
    assert (h is None) == (r is None) and (h is None or torch.equal(h.cpu(), want_h))
    check_codes((q, scale), u, bits)
    # a thread's squares one after the other, then ten sums of pairs or of sixteen waves: each adds half a unit of 2^-23 to a sum of one sign; root and
    # quotients three more
    terms = -(-cols // 8192) * 8 + 26
    assert ((factor.cpu().double() - f).abs() <= (terms / 2 + 3) * 2.0 ** -24 * f).all()


@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_norm_of_extreme_rows(eps):
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(6, 320, generator=gen).bfloat16()
    x[0], x[1], x[2] = 0, x[1] * 2.0 ** -70, x[2] * 2.0 ** 70     # zeros; squares below and above fp32's numbers
    x[3, 7], x[4, 300] = float("inf"), float("nan")
    gain = torch.ones(320).bfloat16()
    q, scale, factor, _ = ms().rms_norm_quantize(x.to(DEV), gain.to(DEV), eps)
    check_codes((q, scale), x.double(), 4)
    f = factor.cpu().double().flatten()
    assert f[0] == (0 if eps == 0 else 1 / torch.tensor(eps, dtype=torch.float32).double().sqrt().float().double()) or abs(f[0] * eps ** 0.5 - 1) < 1e-6
    assert f[2].isnan() and f[3].isnan() and f[4].isnan()
    want = 1 / torch.sqrt(x[1].double().pow(2).mean() + torch.tensor(eps, dtype=torch.float32).double())
    assert abs(f[1] / want - 1) <= 40 * 2.0 ** -24
    want = 1 / torch.sqrt(x[5].double().pow(2).mean() + eps)
    assert abs(f[5] / want - 1) <= 40 * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,cols", [(1, 2), (1, 32), (5, 34), (3, 250), (64, 13824), (2, 40000)])
def test_silu_mul(dtype, bits, rows, cols):
    """The values are off by (1.5 |gate| + 10) 2^-24 of them: a code is one between those of the ends of that range, with a byte of such an end."""
    gen = torch.Generator().manual_seed(rows * 7 + cols)
    both = (torch.randn(rows, 2 * cols, generator=gen) * 4).to(dtype)
    both[0, :min(cols, 3)] = torch.tensor([-100.0, -90.0, 60.0]).to(dtype)[:min(cols, 3)]
    gate, up = both[:, :cols], both[:, cols:]
    dev = both.to(DEV)
    q, scale = ms().silu_mul_quantize(dev[:, :cols], dev[:, cols:], bits)
    g = gate.double()
    v = g * torch.sigmoid(g) * up.double()
    off = (1.5 * g.abs() + 10) * 2.0 ** -24
    lo, hi = v.abs() * (1 - off), v.abs() * (1 + off)
    e = scale.cpu().to(torch.int64)
    assert ((e >= P.exponent_bytes(lo, bits)) & (e <= P.exponent_bytes(hi, bits))).all()
    half = 8 if bits == 4 else 128
    c = P.unpack(q.cpu())
    assert ((c % half >= P.codes(lo, bits, e)[0] % half) & (c % half <= P.codes(hi, bits, e)[0] % half)).all()
    assert torch.equal((c >= half)[c % half > 0], torch.signbit(v)[c % half > 0])


def test_silu_mul_of_no_numbers():
    g, u = torch.randn(2, 96).half(), torch.randn(2, 96).half()
    g[0, 40], u[1, 70] = float("nan"), float("inf")
    _, scale = ms().silu_mul_quantize(g.to(DEV), u.to(DEV))
    assert torch.equal(scale.cpu() == 255, torch.tensor([[False, True, False], [False, False, True]]))


def test_no_rows():
    x = torch.empty(0, 64, dtype=torch.float16, device=DEV)
    q, s = ms().quantize(x)
    assert q.shape == (0, 32) and s.shape == (0, 2) and ms().dequantize(q, s).shape == (0, 64)
    q, s, f, h = ms().rms_norm_quantize(x, torch.ones(64, dtype=torch.float16, device=DEV), residual=x)
    assert f.shape == (0, 1) and h.shape == (0, 64)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    q, s = ms().quantize(torch.ones(4, 64, dtype=torch.float16, device=DEV))
    assert ms().dequantize(q, s, rows=none).shape == (0, 64)
