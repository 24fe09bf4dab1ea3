"""Calls in blocks of 32 with more work than one launch holds: every input goes on where the launch before ended.  The rows next to
the border and the last ones are compared with calls of few rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS = (1 << 29) + 9                 # of four lanes each: 2^31 - 4097 in a launch
BORDER = (2 ** 31 - 1 - 4096) // 4   # the second launch's first row


def ms():
    from quik import microscaled
    return microscaled


@pytest.fixture(autouse=True)
def memory_back():
    yield
    torch.cuda.empty_cache()


def places(n=ROWS):
    """Rows at the start, on both sides of the border, at the end."""
    return torch.cat([torch.arange(a, b, device=DEV) for a, b in ((0, 5), (BORDER - 6, BORDER + 6), (n - 5, n))])


def heads_of_two(n, gen):
    """(codes [n, 4, 1], exponent bytes [n, 4, 1]) of zeros but for the rows that are looked at."""
    q, s = torch.zeros(n, 4, 1, dtype=torch.uint8, device=DEV), torch.full((n, 4, 1), 127, dtype=torch.uint8, device=DEV)
    at = places(n)
    q[at] = torch.randint(1, 256, (len(at), 4, 1), generator=gen, device=DEV).to(torch.uint8)
    s[at] = torch.randint(120, 130, (len(at), 4, 1), generator=gen, device=DEV).to(torch.uint8)
    return q, s, at


@pytest.mark.parametrize("scaled", [False, True])
def test_all_rows_read_back(scaled):
    gen = torch.Generator(DEV).manual_seed(1)
    q, s, at = heads_of_two(ROWS, gen)
    factor = torch.rand(ROWS, generator=gen, device=DEV) + 0.5 if scaled else None
    out = ms().dequantize(q, s, torch.bfloat16, scale_row=factor)
    want = ms().dequantize(q[at], s[at], torch.bfloat16, scale_row=factor[at] if scaled else None)
    assert out.shape == (ROWS, 4, 2) and torch.equal(out[at], want) and want.any()
    out[at] = 0
    assert not out.any()       # (every other row is there, as the zeros that it is)


@pytest.mark.parametrize("scaled", [False, True])
def test_a_list_of_rows_read_back(scaled):
    gen = torch.Generator(DEV).manual_seed(2)
    q, s = torch.randint(1, 256, (7, 4, 1), generator=gen, device=DEV).to(torch.uint8), torch.randint(120, 130, (7, 4, 1), generator=gen, device=DEV).to(torch.uint8)
    rows = torch.randint(-1, 8, (ROWS,), generator=gen, device=DEV)
    factor = torch.rand(ROWS, generator=gen, device=DEV) + 0.5 if scaled else None
    out = ms().dequantize(q, s, rows=rows, scale_row=factor)
    part = 1 << 27
    for i in range(0, ROWS, part):
        assert torch.equal(out[i:i + part], ms().dequantize(q, s, rows=rows[i:i + part], scale_row=factor[i:i + part] if scaled else None))
    table = ms().dequantize(q, s)
    one = rows[BORDER - 6:BORDER + 6]
    want = torch.where(((one >= 0) & (one < 7)).view(-1, 1, 1), table[one.clamp(0, 6)].float() * (factor[BORDER - 6:BORDER + 6].view(-1, 1, 1) if scaled else 1), 0).half()
    assert torch.equal(out[BORDER - 6:BORDER + 6], want)


def test_gated_activations():
    gen = torch.Generator(DEV).manual_seed(3)
    both = torch.zeros(ROWS, 4, dtype=torch.float16, device=DEV)
    at = places()
    both[at] = torch.randn(len(at), 4, generator=gen, device=DEV).half()
    q, s = ms().silu_mul_quantize(both[:, :2], both[:, 2:])
    want = ms().silu_mul_quantize(both[at][:, :2], both[at][:, 2:])
    assert torch.equal(q[at], want[0]) and torch.equal(s[at], want[1]) and want[0].any()
    q[at], s[at] = 0, 0
    assert not q.any() and not s.any()


@pytest.mark.parametrize("bits", [4, 8])
def test_gated_products(bits):
    """Rows of 32 columns, 32 results of each; a launch holds up to 2^30 rows."""
    n = (1 << 30) + (1 << 24) + 7
    gen = torch.Generator(DEV).manual_seed(4)
    kind = (lambda t: t) if bits == 4 else (lambda t: t.view(torch.float8_e4m3fn))
    x, s = torch.zeros(n, 4 * bits, dtype=torch.uint8, device=DEV), torch.full((n, 1), 127, dtype=torch.uint8, device=DEV)
    at = torch.cat((torch.arange(3, device=DEV), *(torch.arange(b - 260, b + 260, device=DEV) for b in (1 << 29, 1 << 30)), torch.arange(n - 40, n, device=DEV)))
    x[at] = torch.randint(0, 127, (len(at), 4 * bits), generator=gen, device=DEV).to(torch.uint8)
    row = torch.zeros(n, device=DEV)
    row[at] = torch.exp2(torch.randint(-3, 3, (len(at),), generator=gen, device=DEV).float()) / 8
    w, ws = ms().quantize(torch.randn(64, 32, generator=gen, device=DEV).half())
    q, scale = ms().gated_matmul(kind(x), s, w, ws, torch.bfloat16, row)
    want = ms().gated_matmul(kind(x[at]), s[at], w, ws, torch.bfloat16, row[at])
    assert torch.equal(q[at], want[0]) and torch.equal(scale[at], want[1]) and want[0].any()
    q[at], scale[at] = 0, 0
    assert not (q & 0x77).any() and not scale.any()


@pytest.mark.parametrize("bits", [4, 8])
def test_products_with_a_factor_per_row(bits):
    n = (1 << 30) + (1 << 24) + 7
    gen = torch.Generator(DEV).manual_seed(5)
    kind = (lambda t: t) if bits == 4 else (lambda t: t.view(torch.float8_e4m3fn))
    x, s = torch.zeros(n, 4 * bits, dtype=torch.uint8, device=DEV), torch.full((n, 1), 127, dtype=torch.uint8, device=DEV)
    at = torch.cat((torch.arange(3, device=DEV), *(torch.arange(b - 260, b + 260, device=DEV) for b in (1 << 28, 1 << 29, 1 << 30)), torch.arange(n - 40, n, device=DEV)))
    x[at] = torch.randint(0, 127, (len(at), 4 * bits), generator=gen, device=DEV).to(torch.uint8)
    row = torch.rand(n, generator=gen, device=DEV) + 0.5
    w, ws = ms().quantize(torch.randn(1, 32, generator=gen, device=DEV).half())
    out = ms().matmul(kind(x), s, w, ws, torch.bfloat16, row)
    assert torch.equal(out[at], ms().matmul(kind(x[at]), s[at], w, ws, torch.bfloat16, row[at]))
    out[at] = 0
    assert not out.any()
