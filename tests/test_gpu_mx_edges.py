"""Calls in blocks of 32 at the ends of what is allowed: widths of an odd number of 8-bit columns, caches and tables of nothing, codes of
five dimensions, the longest rows and the most columns of a product."""
import pytest
import torch

import mx_plain as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]
ODD = (1, 7, 31, 33, 77, 255, 4097)


def ms():
    from quik import microscaled
    return microscaled


@pytest.fixture(autouse=True)
def memory_back():
    yield
    torch.cuda.empty_cache()


def check_codes(got, v):
    c, e = P.codes(v, 8)
    assert torch.equal(got[1].cpu().to(torch.int64), e) and torch.equal(P.unpack(got[0].cpu()), c)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", ODD)
def test_odd_widths(cols, dtype):
    gen = torch.Generator().manual_seed(cols)
    x, r = (torch.randn(5, cols, generator=gen).to(dtype) for _ in range(2))
    gain = (1 + 0.2 * torch.randn(cols, generator=gen)).to(dtype)
    for residual in (None, r):
        q, s, factor, h = ms().rms_norm_quantize(x.to(DEV), gain.to(DEV), 1e-5, None if residual is None else r.to(DEV), bits=8)
        v = x if residual is None else (x.double() + r.double()).to(dtype)
        assert (h is None) == (residual is None) and (h is None or torch.equal(h.cpu(), v))
        check_codes((q, s), v.double() * gain.double())
        want = 1 / torch.sqrt(v.double().pow(2).mean(1, keepdim=True) + 1e-5)
        assert ((factor.cpu().double() - want).abs() <= 20 * 2.0 ** -24 * want).all()      # (eight squares, nine sums of pairs, root and quotients)
    for shape in ((5, cols), (5, 1, cols)):
        codes, e = P.random_rows(gen, 5, cols, 8, 9)
        back = ms().dequantize(P.pack(codes, 8).view(shape).to(DEV), e.to(torch.uint8).view(*shape[:-1], -1).to(DEV), dtype)
        assert torch.equal(back.cpu(), P.numbers(codes, e, 8).to(dtype).view(shape))
    both = torch.randn(5, 2 * cols, generator=gen).to(dtype).to(DEV)
    q, s = ms().silu_mul_quantize(both[:, :cols], both[:, cols:], 8)
    g, u = both.cpu().double().split(cols, 1)
    v = g * torch.sigmoid(g) * u
    off = (1.5 * g.abs() + 10) * 2.0 ** -24                # (of a value, relative)
    e, c = s.cpu().to(torch.int64), P.unpack(q.cpu()) % 128
    lo, hi = v.abs() * (1 - off), v.abs() * (1 + off)
    assert ((e >= P.exponent_bytes(lo, 8)) & (e <= P.exponent_bytes(hi, 8))).all()
    assert ((c >= P.codes(lo, 8, e)[0] % 128) & (c <= P.codes(hi, 8, e)[0] % 128)).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_codes_of_five_dimensions(bits):
    gen = torch.Generator().manual_seed(bits)
    c, e = P.random_rows(gen, 48, 34, bits, 5)
    q, s = P.pack(c, bits).view(2, 3, 4, 2, -1).to(DEV), e.to(torch.uint8).view(2, 3, 4, 2, -1).to(DEV)
    v = P.numbers(c, e, bits).to(torch.bfloat16).view(2, 3, 4, 2, 34)
    assert torch.equal(ms().dequantize(q, s, torch.bfloat16).cpu(), v)
    rows = torch.tensor([1, 2, 0, -1], device=DEV)
    got = ms().dequantize(q, s, torch.bfloat16, rows=rows).cpu()
    assert torch.equal(got[0], v[1]) and torch.equal(got[2], v[0]) and not got[[1, 3]].any()


@pytest.mark.parametrize("bits", [4, 8])
def test_a_cache_of_no_slots_and_a_table_of_no_positions(bits):
    x = torch.randn(3, 2, 64, device=DEV).half()
    angles, none = torch.ones(1, 32, device=DEV), torch.ones(0, 32, device=DEV)
    zero = torch.zeros(3, dtype=torch.int64, device=DEV)
    cache = lambda n: (torch.full((n, 2, 64 * bits // 8), 9, dtype=torch.uint8, device=DEV).view(torch.uint8 if bits == 4 else torch.float8_e4m3fn),
                       torch.full((n, 2, 2), 9, dtype=torch.uint8, device=DEV))
    (k, ks), (v, vs) = cache(0), cache(0)
    out = ms().rotate_to_cache(x, x, x, angles, torch.zeros_like(angles), zero, zero, k, ks, v, vs)
    assert torch.equal(out, x)
    assert not ms().dequantize(k, ks, rows=zero).any() and ms().dequantize(k, ks).shape == (0, 2, 64)
    (k, ks), (v, vs) = cache(4), cache(4)
    slots = torch.tensor([2, 7, 0], device=DEV)
    out = ms().rotate_to_cache(x, x, x, none, none, zero, slots, k, ks, v, vs)
    assert out.isnan().all() and torch.equal(ks.cpu()[:, 0, 0], torch.tensor([255, 9, 255, 9], dtype=torch.uint8))
    want = ms().quantize(x.view(6, 64), bits)
    assert torch.equal(vs[2], want[1].view(3, 2, 2)[0]) and torch.equal(v.view(torch.uint8)[0], want[0].view(torch.uint8).view(3, 2, -1)[2])


def whole_numbers(gen, rows, K, bits, largest, spread):
    """(numbers, codes, exponent bytes): whole numbers up to `spread`, the first of each 32 as `largest`, which is the block's exponent."""
    v = torch.randint(-spread, spread + 1, (rows, K), generator=gen, device=DEV).to(torch.int8)
    v[:, ::32] = (largest * (1 - 2 * torch.randint(0, 2, (rows, K // 32), generator=gen, device=DEV))).to(torch.int8)
    return v, *ms().quantize(v.half(), bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [1, 9, 20, 40, 150])
def test_the_longest_rows(M, bits):
    """K of 2^20, where sums are whole numbers below 2^24; and half a stage less."""
    for K in (1 << 20, (1 << 20) - 96):
        gen = torch.Generator(DEV).manual_seed(M)
        (x, xq, xs), (w, wq, ws) = whole_numbers(gen, M, K, bits, 4, 2), whole_numbers(gen, 192, K, 4, 6, 1)
        sums = x.double() @ w.double().t()
        assert torch.equal(ms().matmul(xq, xs, wq, ws, torch.bfloat16), sums.to(torch.bfloat16))
        row = torch.full((M, 1), 2.0 ** -9, device=DEV)
        both = (sums * 2.0 ** -9).to(torch.bfloat16)
        got, want = ms().gated_matmul(xq, xs, wq, ws, torch.bfloat16, row), ms().silu_mul_quantize(both[:, :96], both[:, 96:])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [1, 12, 20, 40])
def test_the_most_columns(M, bits):
    """2^29 and some columns of 32 numbers: weights, results and tiles past 32 bits."""
    N, gen = (1 << 29) + 37, torch.Generator(DEV).manual_seed(M)
    x, xq, xs = whole_numbers(gen, M, 32, bits, 4, 2)
    wq, ws = torch.zeros(N, 16, dtype=torch.uint8, device=DEV), torch.full((N, 1), 127, dtype=torch.uint8, device=DEV)
    at = torch.cat([torch.arange(a, b, device=DEV) for a, b in ((0, 300), (N // 2 - 300, N // 2 + 300), (N - 300, N))])
    w, wq[at], ws[at] = whole_numbers(gen, len(at), 32, 4, 6, 1)
    out = ms().matmul(xq, xs, wq, ws, torch.float16)
    assert torch.equal(out[:, at], (x.double() @ w.double().t()).half())
    out[:, at] = 0
    assert not out.any()


@pytest.mark.parametrize("kind", ["apart", "zeros", "low", "high"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,N,K", [(1, 200, 256), (16, 70, 544), (24, 300, 4096), (64, 70, 544), (300, 300, 4096)])
def test_exponents_at_their_ends(M, N, K, bits, kind):
    """Exponent bytes of either side up to 115 from the middle whose products are ordinary numbers; blocks of zeros with the largest exponents on both; the
    least and the largest byte against weights that make up for it.  The bound is test_gpu_mx_matmul's, and bf16's last subnormal."""
    gen = torch.Generator().manual_seed(M + K)
    (c, e), (w, we) = P.random_rows(gen, M, K, bits, 0), P.random_rows(gen, N, K, 4, 0)
    blocks = K // 32
    if kind == "apart":
        d = torch.randint(-115, 116, (blocks,), generator=gen)
        e, we = (127 - (3 if bits == 4 else 8) + d).expand(M, blocks), (127 - d).expand(N, blocks)
    elif kind == "zeros":
        c[:, torch.arange(K) // 32 % 2 == 1] = 0
        e[:, 1::2], we[:, 1::2] = 254, 254
    else:
        e, we = torch.full_like(e, 0 if kind == "low" else 254), torch.full_like(we, 200 if kind == "low" else 20)
    x, v = P.numbers(c, e, bits), P.numbers(w, we, 4)
    on = lambda q, s, b: (P.pack(q, b).to(DEV), s.to(torch.uint8).contiguous().to(DEV))
    out = ms().matmul(*on(c, e, bits), *on(w, we, 4), torch.bfloat16).cpu().double()
    y, steps = x @ v.t(), -(-K // 64) * (bits // 4) + 20
    assert ((out - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -134 + x.abs() @ v.abs().t() * (steps * 2.0 ** -24)).all()


@pytest.mark.parametrize("M", [1, 8, 16, 24, 64, 300])
@pytest.mark.parametrize("code", [0x7F, 0xFF])
def test_a_code_without_a_number(M, code):
    """e4m3's NaN among 8-bit codes, which quantize never writes: its row of a product is NaNs, and a number read back is one."""
    gen = torch.Generator().manual_seed(M)
    (c, e), (w, we) = P.random_rows(gen, M, 544, 8), P.random_rows(gen, 70, 544, 4)
    c[M // 2, 543] = code
    q, s, wq, ws = P.pack(c, 8).to(DEV), e.to(torch.uint8).to(DEV), P.pack(w, 4).to(DEV), we.to(torch.uint8).to(DEV)
    bad = torch.zeros(M, dtype=torch.bool)
    bad[M // 2] = True
    out = ms().matmul(q, s, wq, ws, torch.bfloat16).cpu()
    assert torch.equal(out.isnan(), bad.unsqueeze(1).expand(M, 70))
    back = ms().dequantize(q, s, torch.bfloat16).cpu().isnan()
    assert back[M // 2, 543] and back.sum() == 1
