"""Products of rows in blocks of 32 with 4-bit weights, and the gated one, against 64-bit arithmetic."""
import pytest
import torch

import mx_plain as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ms():
    from quik import microscaled
    return microscaled


def operands(seed, M, N, K, bits, spread=3):
    gen = torch.Generator().manual_seed(seed)
    x, w = P.random_rows(gen, M, K, bits, spread), P.random_rows(gen, N, K, 4, spread)
    on = lambda c, e, b: (P.pack(c, b).to(DEV), e.to(torch.uint8).to(DEV))
    return gen, P.numbers(*x, bits), P.numbers(*w, 4), on(*x, bits), on(*w, 4)


def allowed(x, w, y, bits, dtype):
    """The rounding to the type; per instruction of 64 columns (8 bits: two of them) an alignment to 2^-24 of its largest term and a rounding of
    the sum so far, sixteen parts of K joined, row factor and bias."""
    total = x.abs() @ w.abs().t()
    steps = -(-x.shape[1] // 64) * (bits // 4) + 20
    return torch.finfo(dtype).eps / 2 * y.abs() + 2.0 ** -24 * (1 if dtype == torch.float16 else 0) + total * (steps * 2.0 ** -24)


SHAPES = [(1, 1, 32), (1, 5, 64), (1, 4096, 4096), (1, 1000, 11008), (2, 33, 96), (4, 64, 128), (5, 257, 160), (8, 8200, 512), (9, 100, 1056), (16, 300, 4544),
          (16, 5120, 1024), (17, 64, 32), (17, 4096, 4096), (31, 129, 224), (32, 128, 640), (33, 131, 4544), (64, 5120, 2048), (65, 1, 128), (100, 4541, 544),
          (128, 256, 13824), (200, 333, 1120), (300, 4541, 4544), (257, 513, 384), (512, 1024, 1024), (777, 700, 256), (32, 300, 4544), (25, 5121, 1056), (29, 28672, 1024),
          (18, 4100, 96), (32, 9000, 2080), (24, 16, 128)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(M, N, K, bits):
    gen, x, w, xq, wq = operands(M + N + K, M, N, K, bits)
    dtype = torch.float16 if (M + K) % 3 else torch.bfloat16
    out = ms().matmul(*xq, *wq, dtype)
    assert out.shape == (M, N) and out.dtype == dtype
    y = x @ w.t()
    assert ((out.cpu().double() - y).abs() <= allowed(x, w, y, bits, dtype)).all()
    row, bias = torch.rand(M, 1, generator=gen) + 0.5, torch.randn(N, generator=gen).to(dtype)
    out = ms().matmul(*xq, *wq, dtype, scale_row=row.to(DEV), bias=bias.to(DEV))
    y = y * row.double() + bias.double()
    limit = allowed(x * row.double(), w, y, bits, dtype) + 2.0 ** -23 * y.abs()
    assert ((out.cpu().double() - y).abs() <= limit).all()


@pytest.mark.parametrize("M", [1, 8, 13, 27, 40, 100, 300])
def test_all_of_an_8_bit_code_counts(M):
    """Numbers over all of e4m3's range next to each other: the largest cancel each other, and what remains of each sixteen is a sum of multiples of 2^-10
    below 2^12 apart, which is a number of fp32."""
    K, N = 256, 70
    gen = torch.Generator().manual_seed(M)
    v = torch.randint(0, 120, (M, K), generator=gen)
    e = torch.full((M, K // 32), 127)
    v[:, 0::16], v[:, 15::16] = 126, 254                      # 448 and -448
    small = torch.randint(1, 16, (M, K // 4), generator=gen)  # multiples of 2^-9 up to 2^-5
    v[:, 1::16] = small[:, :K // 16]
    v[:, 2::16] = 128 + small[:, K // 16:K // 8]
    for i in range(3, 15):
        v[:, i::16] = torch.randint(0, 64, (M, K // 16), generator=gen)   # below 2
    w = torch.randint(0, 16, (N, K), generator=gen)
    w[:, 0::16] = w[:, 15::16] = 7                            # 6
    we = torch.full((N, K // 32), 127)
    y = P.numbers(v, e, 8) @ P.numbers(w, we, 4).t()
    out = ms().matmul(P.pack(v, 8).to(DEV), e.to(torch.uint8).to(DEV), P.pack(w, 4).to(DEV), we.to(torch.uint8).to(DEV), torch.float16)
    assert torch.equal(out.cpu(), y.to(torch.float16))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [1, 16, 24, 40, 150])
def test_exact_sums(M, bits):
    """Equal exponents and small codes: every sum is a number of fp16, and comes out as it is."""
    K, N = 512, 200
    gen = torch.Generator().manual_seed(M)
    v = torch.randint(-2, 3, (M, K), generator=gen).double()
    v[:, ::32] = 4.0
    w = torch.randint(-1, 2, (N, K), generator=gen).double()
    w[:, ::32] = 6.0
    (xc, xe), (wc, we) = P.codes(v, bits), P.codes(w, 4)
    out = ms().matmul(P.pack(xc, bits).to(DEV), xe.to(torch.uint8).to(DEV), P.pack(wc, 4).to(DEV), we.to(torch.uint8).to(DEV), torch.bfloat16)
    assert torch.equal(out.cpu(), (v @ w.t()).to(torch.bfloat16))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,K", [(3, 128), (3, 160), (23, 128), (32, 160), (40, 256), (40, 96)])
def test_each_code_meets_its_own(M, K, bits):
    """Weights that are one number in one column each: the product is that column of x."""
    gen = torch.Generator().manual_seed(K)
    c, e = P.random_rows(gen, M, K, bits, 6)
    w = torch.eye(K, dtype=torch.float64)
    wc, we = P.codes(w, 4)
    out = ms().matmul(P.pack(c, bits).to(DEV), e.to(torch.uint8).to(DEV), P.pack(wc, 4).to(DEV), we.to(torch.uint8).to(DEV), torch.bfloat16)
    assert torch.equal(out.cpu().double(), P.numbers(c, e, bits).to(torch.bfloat16).double())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,N,K", [(2, 40, 96), (16, 200, 256), (32, 70, 544), (50, 70, 544), (300, 300, 512)])
def test_rows_without_a_number(M, N, K, bits):
    """A NaN byte of x is a row of NaNs, one of the weights a column; nothing else is touched."""
    _, x, w, (xq, xs), (wq, ws) = operands(7, M, N, K, bits)
    xs[M // 2, K // 32 - 1] = 255
    ws[N // 3, 0] = 255
    want = torch.zeros(M, N, dtype=torch.bool)
    want[M // 2], want[:, N // 3] = True, True
    out = ms().matmul(xq, xs, wq, ws, torch.bfloat16).cpu()
    assert torch.equal(out.isnan(), want)
    y = x @ w.t()
    assert ((out.double() - y).abs() <= allowed(x, w, y, bits, torch.bfloat16))[~want].all()


@pytest.mark.parametrize("M", [1, 20, 40])
def test_views_and_scales_at_any_byte(M):
    """Exponent bytes that start between multiples of four; codes that start between multiples of sixteen are refused."""
    _, x, w, (xq, xs), (wq, ws) = operands(9, M, 100, 256, 4)
    shifted = [torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape) for t in (xs, ws)]
    assert shifted[0].data_ptr() % 4
    assert torch.equal(ms().matmul(xq, shifted[0], wq, shifted[1]), ms().matmul(xq, xs, wq, ws))
    with pytest.raises(RuntimeError, match="align"):
        ms().matmul(torch.cat((xq.new_zeros(8), xq.flatten()))[8:].view(xq.shape), xs, wq, ws)


def test_range_of_exponents():
    """Sums near both ends of bf16's numbers."""
    for e in (60, 190):
        gen = torch.Generator().manual_seed(e)
        c, b = P.random_rows(gen, 20, 128, 4, 0)
        w, wb = P.random_rows(gen, 40, 128, 4, 0)
        b, wb = torch.full_like(b, e), torch.full_like(wb, 127 if e > 127 else 70)
        out = ms().matmul(P.pack(c, 4).to(DEV), b.to(torch.uint8).to(DEV), P.pack(w, 4).to(DEV), wb.to(torch.uint8).to(DEV), torch.bfloat16).cpu().double()
        x, v = P.numbers(c, b, 4), P.numbers(w, wb, 4)
        y = x @ v.t()
        assert ((out - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -20 * (x.abs() @ v.abs().t())).all()


GATED = [(1, 32, 32), (1, 11008, 512), (3, 96, 4096), (8, 64, 96), (9, 64, 1056), (16, 352, 640), (17, 64, 128), (40, 1024, 512), (64, 2304, 544), (100, 96, 4544),
         (130, 160, 512), (300, 1056, 1024), (520, 544, 256)]


@pytest.mark.parametrize("q_bits", [4, 8])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M,inner,K", GATED)
def test_gated_product_is_the_two_after_each_other(M, inner, K, bits, q_bits):
    """Bit for bit what matmul (its K not split) and silu_mul_quantize give."""
    gen, x, w, xq, wq = operands(M + inner, M, 2 * inner, K, bits)
    dtype = torch.float16 if M % 2 else torch.bfloat16
    row = ((torch.rand(M, 1, generator=gen) + 0.5) / K ** 0.5).to(DEV)
    q, scale = ms().gated_matmul(*xq, *wq, dtype, scale_row=row, bits=q_bits)
    assert q.shape == (M, inner // 2 if q_bits == 4 else inner) and scale.shape == (M, inner // 32)
    # the values: gate and up within the product's bound, then silu's slope (at most 1.1) and the codes' half a step of the largest number
    y = (x @ w.t()) * row.cpu().double()
    off = allowed(x * row.cpu().double(), w, y, bits, dtype) + 2.0 ** -23 * y.abs()
    g, u = y[:, :inner], y[:, inner:]
    v = g * torch.sigmoid(g) * u
    dv = 1.1 * off[:, :inner] * (u.abs() + off[:, inner:]) + g.abs() * off[:, inner:] + 1e-5 * v.abs()
    got = P.numbers(P.unpack(q.cpu()), scale.cpu().to(torch.int64), q_bits)
    top = (P.split(v.abs() + dv).amax(-1, keepdim=True) * torch.ones(32)).flatten(-2)
    step = top / 4 if q_bits == 4 else top * 2.0 ** -3      # half the widest step, or what the largest code cuts off
    assert ((got - v).abs() <= dv + step).all()
    both = _whole_product(xq, wq, dtype, row, M)
    want = ms().silu_mul_quantize(both[:, :inner], both[:, inner:], q_bits)
    if both.whole:
        assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scale, want[1])


def _whole_product(xq, wq, dtype, row, M):
    """matmul without a workspace: K is one part."""
    from quik_amd import _lib as L
    lib = L.load()
    (x, xs), (w, ws) = xq, wq
    N, K = w.shape[0], 2 * w.shape[1]
    out = torch.empty(M, N, dtype=dtype, device=DEV)
    L.check(lib.quik_mx_matmul(L.ptr(x), 4 if x.dtype == torch.uint8 else 8, L.ptr(xs), L.ptr(w), L.ptr(ws), L.ptr(row), None,
                               L.QUIK_BF16 if dtype == torch.bfloat16 else L.QUIK_F16, M, N, K, L.ptr(out), None, 0, L.stream()), "matmul")
    out.whole = M > 16      # (up to 16 rows the waves that share K differ between the two)
    return out


def test_without_a_workspace_within_the_rounding():
    for M, N, K in ((64, 512, 13824), (20, 256, 8192)):
        _, x, w, xq, wq = operands(1, M, N, K, 4)
        out = _whole_product(xq, wq, torch.bfloat16, None, M)
        y = x @ w.t()
        assert ((out.cpu().double() - y).abs() <= allowed(x, w, y, 4, torch.bfloat16)).all()


def test_no_rows_and_no_columns():
    _, _, _, (xq, xs), (wq, ws) = operands(1, 3, 64, 64, 4)
    assert ms().matmul(xq[:0], xs[:0], wq, ws).shape == (0, 64) and ms().matmul(xq, xs, wq[:0], ws[:0]).shape == (3, 0)
    assert ms().gated_matmul(xq[:0], xs[:0], wq, ws)[0].shape == (0, 16)


def test_the_python_functions_and_the_front_end_agree():
    from quik_amd import _lib as L
    _, _, _, xq, wq = operands(2, 30, 128, 256, 8)
    with_front = ms().matmul(*xq, *wq), *ms().gated_matmul(*xq, *wq)
    front, L._front = L._front, L._NoFront()
    try:
        without = ms().matmul(*xq, *wq), *ms().gated_matmul(*xq, *wq)
    finally:
        L._front = front
    for a, b in zip(with_front, without):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and a.dtype == b.dtype
