"""Operators in blocks of 32 as a decoder block runs them: one after the other, as modules, from graphs between eager calls, on streams of their own,
over caches and row counts that pass 32 bits."""
import pytest
import torch

import mx_plain as P
from quik_amd.qlinear import MicroscaledLinear4bit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ms():
    from quik import microscaled
    return microscaled


class Block:
    """Norm, one product for q, k and v, heads into a cache, (the queries stand for the attention's result,) a product, norm, gated product, product."""

    def __init__(self, hidden, heads, kv_heads, size, inner, bits, dtype, slots=200, seed=0):
        torch.manual_seed(seed)
        lin = lambda n, m, bias: MicroscaledLinear4bit.from_float(torch.nn.Linear(n, m, bias=bias, dtype=dtype, device=DEV), bits)
        self.qkv, self.out = lin(hidden, (heads + 2 * kv_heads) * size, True), lin(heads * size, hidden, False)
        self.up, self.down = lin(hidden, 2 * inner, False), lin(inner, hidden, False)
        self.gains = [(1 + 0.1 * torch.randn(n, device=DEV)).to(dtype) for n in (hidden, hidden, size, size)]
        angle = torch.outer(torch.arange(64.0), 100.0 ** (-torch.arange(size // 2) / (size // 2)))
        self.cos, self.sin = angle.cos().to(DEV), angle.sin().to(DEV)
        self.shape, self.bits, self.dtype = (heads, kv_heads, size), bits, dtype
        empty = lambda b: torch.zeros(slots, kv_heads, size // 2 if b == 4 else size, dtype=torch.uint8, device=DEV)
        self.kc, self.vc = empty(8).view(torch.float8_e4m3fn), empty(4)
        self.ks, self.vs = (torch.zeros(slots, kv_heads, -(-size // 32), dtype=torch.uint8, device=DEV) for _ in range(2))

    def run(self, x, residual, positions, slots):
        """(result, the next residual, keys, values, and what lies between)"""
        heads, kv_heads, size = self.shape
        m = ms()
        q, scale, row, h = m.rms_norm_quantize(x, self.gains[0], 1e-5, residual, self.bits)
        qkv = self.qkv(q, scale, row)
        q, k, v = (t.unflatten(1, (-1, size)) for t in qkv.split((heads * size, kv_heads * size, kv_heads * size), 1))
        queries = m.rotate_to_cache(q, k, v, self.cos, self.sin, positions, slots, self.kc, self.ks, self.vc, self.vs, self.gains[2], self.gains[3])
        keys = m.dequantize(self.kc, self.ks, self.dtype, rows=slots)
        values = m.dequantize(self.vc, self.vs, self.dtype, rows=slots)
        a = self.out(queries.flatten(1))
        q, scale, row, last = m.rms_norm_quantize(a, self.gains[1], 1e-5, h, self.bits)
        q, scale = self.up.gated(q, scale, row)
        return self.down(q, scale), last, keys, values, h, qkv, queries, a, m.dequantize(q, scale, self.dtype)


def held(v, bits):
    return P.numbers(*P.codes(v, bits), bits)


def weight(mod):
    return P.numbers(P.unpack(mod.weight.cpu()), mod.weight_scale.cpu().to(torch.int64), 4)


def inputs(rows, hidden, dtype, seed=1):
    gen = torch.Generator(DEV).manual_seed(seed)
    x, r = (torch.randn(rows, hidden, device=DEV, generator=gen).to(dtype) for _ in range(2))
    return x, r, torch.randint(0, 64, (rows,), device=DEV, generator=gen), torch.randperm(200, device=DEV, generator=gen)[:rows]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows", [1, 7, 16, 40, 150])
def test_block(rows, bits, dtype):
    """Each step against 64 bits, from what the steps before it left.  Sums are exact but for `near`, relative to the result's norm: a rounding to 16
    bits (eps / 2) and the norm's factor.  A value that is off by d goes to the neighbouring code with the probability d / step, so that behind a quantization the
    squares of the differences are d * step of the values' own, step 2^-1 and 2^-3 (4 and 8 bits: a step over the smallest number that has it)."""
    block = Block(512, 8, 2, 64, 1376, bits, dtype)
    x, residual, positions, slots = inputs(rows, 512, dtype)
    out, last, keys, values, h, qkv, queries, a, gated = (t.double().cpu() for t in block.run(x, residual, positions, slots))
    heads, kv_heads, size = block.shape
    gains, cos, sin = [g.double().cpu() for g in block.gains], block.cos.double().cpu()[positions.cpu()], block.sin.double().cpu()[positions.cpu()]
    near = torch.finfo(dtype).eps / 2 + 2.0 ** -18
    apart = lambda got, want: ((got - want).norm() / want.norm()).item()

    def norm(t, gain):  # (the codes are those of t * gain, the row's factor is apart from them)
        return held(t * gain, bits) / torch.sqrt(t.pow(2).mean(1, keepdim=True) + 1e-5)

    def turn(t, gain):
        t = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * gain
        a, b = t.chunk(2, -1)
        return torch.cat((a * cos.unsqueeze(1) - b * sin.unsqueeze(1), b * cos.unsqueeze(1) + a * sin.unsqueeze(1)), -1)
    assert torch.equal(h, (x.float() + residual.float()).to(dtype).double().cpu())
    assert apart(qkv, norm(h, gains[0]) @ weight(block.qkv).t() + block.qkv.bias.double().cpu()) <= near
    q, k, v = (t.unflatten(1, (-1, size)) for t in qkv.split((heads * size, kv_heads * size, kv_heads * size), 1))
    assert apart(queries, turn(q, gains[2])) <= torch.finfo(dtype).eps / 2 + 2.0 ** -18
    assert apart(keys, held(turn(k, gains[3]), 8)) <= (2.0 ** -18 * 0.125) ** 0.5 + torch.finfo(dtype).eps / 2
    assert torch.equal(values, held(v, 4).to(dtype).double())
    assert apart(a, held(queries.flatten(1), bits) @ weight(block.out).t()) <= near
    assert torch.equal(last, (a.float() + h.float()).to(dtype).double())
    g, u = (norm(last, gains[1]) @ weight(block.up).t()).chunk(2, 1)
    assert apart(gated, held(g / (1 + torch.exp(-g)) * u, bits)) <= (3 * near * (0.5 if bits == 4 else 0.125)) ** 0.5 + 3 * near
    assert apart(out, gated @ weight(block.down).t()) <= near


@pytest.mark.parametrize("rows", [1, 16, 70, 150])
def test_replayed_between_eager_calls(rows):
    """Two captured runs of a block, replayed with new inputs between eager runs of the same and of other sizes, equal the eager run each time.  70 rows: K
    is split, so that each graph holds the memory of the parts."""
    block = Block(1024, 8, 8, 128, 4096, 8, torch.float16)
    args = inputs(rows, 1024, torch.float16)
    block.run(*args)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block.run(*args)
        graphs.append((g, out))
    for i in range(4):
        for t, new in zip(args, inputs(rows, 1024, torch.float16, seed=10 + i)):
            t.copy_(new)
        want = [t.clone() for t in block.run(*args)]
        block.run(*inputs(33, 1024, torch.float16, seed=99))
        for g, out in graphs:
            g.replay()
        if i % 2:
            torch.cuda.synchronize()
        for g, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    sizes = (64, 90)
    blocks = [Block(1024, 8, 2, 64, 2752, 4, torch.bfloat16, seed=k) for k in range(2)]
    args = [inputs(n, 1024, torch.bfloat16, seed=n) for n in sizes]
    want = [b.run(*a) for b, a in zip(blocks, args)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sizes], [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(blocks[k].run(*args[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            for a, b in zip(out, want[k]):
                assert torch.equal(a, b)


def test_captured_first():
    """Sizes that no eager call has had are captured like any other."""
    x = torch.randn(19, 640, device=DEV).half()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w, ws = ms().quantize(x)
        out = ms().matmul(w, ws, w, ws)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ms().matmul(*ms().quantize(x), *ms().quantize(x)))


@pytest.mark.parametrize("act_bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_module(dtype, act_bits):
    torch.manual_seed(3)
    lin = torch.nn.Linear(352, 96, dtype=dtype, device=DEV)
    lin.weight.data[5] = 0
    mod = MicroscaledLinear4bit.from_float(lin, act_bits)
    kind = torch.float16 if dtype == torch.float32 else dtype
    assert torch.equal(weight(mod), held(lin.weight.detach().to(kind).double().cpu(), 4)) and mod.dtype == kind
    x = torch.randn(2, 7, 352, device=DEV).to(kind)
    out = mod(x)
    assert out.shape == (2, 7, 96) and out.dtype == kind
    q, s = ms().quantize(x.view(14, 352), act_bits)
    assert torch.equal(out.view(14, 96), ms().matmul(q, s, mod.weight, mod.weight_scale, kind, bias=mod.bias))
    assert torch.equal(mod(q.view(2, 7, -1), s.view(2, 7, -1)), out)
    back = x.transpose(1, 2).contiguous().transpose(1, 2)     # columns apart
    assert torch.equal(mod(back), out) and torch.equal(mod(x[:1, :1].expand(2, 3, 352))[1, 2], out[0, 0])
    assert mod(x[:, :0]).shape == (2, 0, 96)
    twin = MicroscaledLinear4bit(352, 96, act_bits, True, kind).to(DEV)
    twin.load_state_dict(mod.state_dict())
    assert torch.equal(twin(x), out)
    assert twin.to(torch.bfloat16)(x).dtype == torch.bfloat16
    with pytest.raises(ValueError, match="no bias"):
        mod.gated(x)
    with pytest.raises(ValueError, match="scale_row"):
        mod(x, scale_row=torch.ones(14, device=DEV))
    both = MicroscaledLinear4bit(352, 128, act_bits, False, kind).to(DEV)
    both.weight, both.weight_scale = ms().quantize(torch.randn(128, 352, device=DEV).to(kind))
    a, b = both.gated(x), ms().gated_matmul(q, s, both.weight, both.weight_scale, kind, bits=act_bits)
    assert a[0].shape[:2] == (2, 7) and torch.equal(a[0].view(torch.uint8).flatten(), b[0].view(torch.uint8).flatten()) and torch.equal(a[1].view(14, -1), b[1])


def test_an_angle_without_a_number_stays_with_its_columns():
    """Heads of 48: the second block is half behind the head's end, and has numbers whatever the angle of column 0 is."""
    x = torch.randn(2, 1, 48, device=DEV).half()
    cos, sin = torch.ones(1, 24, device=DEV), torch.zeros(1, 24, device=DEV)
    cos[0, 0] = float("nan")
    kc, ks = torch.zeros(2, 1, 48, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.zeros(2, 1, 2, dtype=torch.uint8, device=DEV)
    vc, vs = kc.clone(), ks.clone()
    zero = torch.zeros(2, dtype=torch.int64, device=DEV)
    out = ms().rotate_to_cache(x, x, x, cos, sin, zero, torch.arange(2, device=DEV), kc, ks, vc, vs)
    assert torch.equal(out.isnan().any(0).any(0).nonzero().flatten().cpu(), torch.tensor([0, 24]))
    q, s = ms().quantize(x.flatten(1), 8)
    assert (ks[:, 0, 0] == 255).all() and torch.equal(ks[:, 0, 1], s[:, 1])
    assert torch.equal(kc.view(torch.uint8)[:, 0, 32:], q.view(torch.uint8)[:, 32:]) and torch.equal(vc.view(torch.uint8)[:, 0], q.view(torch.uint8))


@pytest.mark.parametrize("bits", [4, 8])
def test_a_cache_past_32_bits(bits):
    slots, heads, size = (1 << 23) + 5 if bits == 4 else (1 << 22) + 5, 8, 128
    cache = torch.empty(slots, heads, size // 2 if bits == 4 else size, dtype=torch.uint8, device=DEV)
    assert cache.numel() > 1 << 32
    cache = cache if bits == 4 else cache.view(torch.float8_e4m3fn)
    scale = torch.zeros(slots, heads, 4, dtype=torch.uint8, device=DEV)
    x = torch.randn(3, heads, size, device=DEV).half()
    at = torch.tensor([slots - 1, 0, slots - 4], device=DEV)
    cos, sin = torch.ones(1, 64, device=DEV), torch.zeros(1, 64, device=DEV)
    zero = torch.zeros(3, dtype=torch.int64, device=DEV)
    vc, vs = cache[:1].clone(), scale[:1].clone()
    with pytest.raises(RuntimeError, match="v_cache to have size"):
        ms().rotate_to_cache(x, x, x, cos, sin, zero, at, cache, scale, vc, vs)
    ms().rotate_to_cache(x, x, x, cos, sin, zero, at, cache, scale, cache, scale)   # (keys and values are the same numbers here)
    q, s = ms().quantize(x.flatten(0, 1), bits)
    want = ms().dequantize(q, s).view(3, heads, size)
    got = ms().dequantize(cache, scale, rows=torch.cat((at, torch.tensor([slots, -1], device=DEV))))
    assert torch.equal(got[:3], want) and not got[3:].any()


def test_row_counts_past_one_launch():
    """Rows of two columns, more than 2^31 threads' worth: further launches go on where the first ends."""
    n = (1 << 29) + 9
    x = torch.zeros(n, 2, dtype=torch.float16, device=DEV)
    x[-3:] = torch.tensor([[1.0, 6.0], [-3.0, 0.5], [0.0, 2.0]], device=DEV)
    q, s = ms().quantize(x)
    want = ms().quantize(x[-3:].clone())
    assert torch.equal(q[-3:], want[0]) and torch.equal(s[-3:], want[1]) and not q[:-3].any() and not s[:-3].any()
    del x
    back = ms().dequantize(q[-3:].repeat(1, 1), s[-3:].clone())
    assert torch.equal(back.cpu(), torch.tensor([[1.0, 6.0], [-3.0, 0.5], [0.0, 2.0]]).half())
    del q, s
    n = (1 << 20) + 3
    x = torch.randn(n, 34, device=DEV).half()
    w = torch.ones(34, device=DEV).half()
    q, s, row, h = ms().rms_norm_quantize(x, w, 1e-5, x)
    tail = ms().rms_norm_quantize(x[-5:], w, 1e-5, x[-5:])
    assert all(torch.equal(a[-5:], b) for a, b in zip((q, s, row, h), tail))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("bits", [4, 8])
def test_tokens_and_rows_of_a_product_past_one_launch(bits):
    n = (1 << 30) + (1 << 24) + 7                 # rows of 32 columns, one result column
    x = torch.zeros(n, 4 * bits, dtype=torch.uint8, device=DEV)
    s = torch.full((n, 1), 127, dtype=torch.uint8, device=DEV)
    x[-40:] = torch.randint(0, 127, (40, 4 * bits), dtype=torch.uint8, device=DEV)
    kind = (lambda t: t) if bits == 4 else (lambda t: t.view(torch.float8_e4m3fn))
    w, ws = ms().quantize(torch.randn(1, 32, device=DEV).half())
    out = ms().matmul(kind(x), s, w, ws)
    assert torch.equal(out[-40:], ms().matmul(kind(x[-40:].clone()), s[-40:].clone(), w, ws)) and not out[:-40].any()
    del x, s, out
    torch.cuda.empty_cache()


def test_tokens_past_one_launch():
    n = (2 ** 31 - 1) // 256 + 6
    gen = torch.Generator(DEV).manual_seed(4)
    x = torch.randn(n, 1, 2, device=DEV, generator=gen).half()
    cos, sin = torch.full((3, 1), 0.6, device=DEV), torch.full((3, 1), 0.8, device=DEV)
    cos[2], sin[2] = 0.0, 1.0
    positions, slots = torch.zeros(n, dtype=torch.int64, device=DEV), torch.full((n,), -1, dtype=torch.int64, device=DEV)
    positions[-4:], slots[-4:] = 2, torch.arange(4, device=DEV)
    cache = [torch.full(s, 9, dtype=torch.uint8, device=DEV) for s in ((6, 1, 1), (6, 1, 1), (6, 1, 1), (6, 1, 1))]
    out = ms().rotate_to_cache(x, x, x, cos, sin, positions, slots, *cache)
    tail = [torch.full_like(t, 9) for t in cache]
    assert torch.equal(out[-9:], ms().rotate_to_cache(x[-9:], x[-9:], x[-9:], cos, sin, positions[-9:], slots[-9:], *tail))
    assert all(torch.equal(a, b) for a, b in zip(cache, tail)) and (cache[0][:4] != 9).any() and all((t[4:] == 9).all() for t in cache)
    a, b = x[:1000, 0].double().unbind(1)
    assert (out[:1000, 0].double() - torch.stack((0.6 * a - 0.8 * b, 0.6 * b + 0.8 * a), 1)).abs().max() <= 2.0 ** -10 * 4


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("over", ["x", "residual"])
def test_the_sum_over_one_of_its_terms(over, bits):
    """The C entry point takes x or the residual as the place of their sum; bf16 rows of tiny numbers are read again for their squares."""
    from quik_amd import _lib as L
    x, r, w = torch.randn(5, 200, device=DEV).bfloat16(), torch.randn(5, 200, device=DEV).bfloat16(), torch.rand(200, device=DEV).bfloat16()
    x[3], r[3] = x[3] * 2.0 ** -70, r[3] * 2.0 ** -70
    want = ms().rms_norm_quantize(x, w, 0.0, r, bits)
    q, s, f = (torch.empty_like(t) for t in want[:3])
    place = x if over == "x" else r
    L.check(L.load().quik_mx_rms_norm_quantize(L.ptr(x), 200, L.ptr(r), 200, L.ptr(w), 0.0, L.dtype_id(x, "norm", allow_bf16=True), 5, 200, bits, L.ptr(place),
                                               L.ptr(q), L.ptr(s), L.ptr(f), L.stream()), "norm")
    for a, b in zip((q, s, f, place), want):
        assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
