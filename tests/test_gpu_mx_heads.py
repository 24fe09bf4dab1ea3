"""Heads normed, turned and put into a cache in blocks of 32, against 64-bit arithmetic."""
import pytest
import torch

import mx_plain as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ms():
    from quik import microscaled
    return microscaled


def table(positions, half, base=10000.0):
    angle = torch.outer(torch.arange(positions, dtype=torch.float64), base ** (-torch.arange(half, dtype=torch.float64) / half))
    return angle.cos().float(), angle.sin().float()


def empty_cache(slots, heads, size, bits, fill=7):
    q = torch.full((slots, heads, size // 2 if bits == 4 else size), fill, dtype=torch.uint8)
    return (q if bits == 4 else q.view(torch.float8_e4m3fn)).to(DEV), torch.full((slots, heads, -(-size // 32)), 99, dtype=torch.uint8, device=DEV)


def turned(x, gain, eps, cos, sin):
    """(values, how far fp32 arithmetic may be from them): a norm's factor within 40 units of 2^-24, four products and a sum."""
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * gain.double()
    r = cos.shape[-1]
    c, s = cos.double().unsqueeze(1), sin.double().unsqueeze(1)
    a, b = x[..., :r], x[..., r:2 * r]
    y = torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * r:]), -1)
    mag = torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), x[..., 2 * r:].abs()), -1)
    return y, mag * ((40 if gain is not None else 3) * 2.0 ** -24)


def check_cached(q, scale, v, off, bits):
    """Each code between those of the ends of its value's range."""
    e = scale.cpu().to(torch.int64)
    lo, hi = (v.abs() - off).clamp(min=0), v.abs() + off
    assert ((e >= P.exponent_bytes(lo, bits)) & (e <= P.exponent_bytes(hi, bits))).all()
    half = 8 if bits == 4 else 128
    c = P.unpack(q.cpu()) % half
    assert ((c >= P.codes(lo, bits, e)[0] % half) & (c <= P.codes(hi, bits, e)[0] % half)).all()
    sure = (c > 0) & (v.abs() > off)
    assert torch.equal((P.unpack(q.cpu()) >= half)[sure], (v < 0)[sure])


CASES = [(1, 1, 1, 2, 1), (1, 32, 8, 128, 64), (5, 4, 4, 64, 32), (3, 16, 2, 80, 40), (7, 3, 1, 96, 16), (9, 2, 2, 34, 17), (4, 5, 3, 256, 128), (2, 2, 1, 512, 256),
         (33, 8, 8, 128, 32), (6, 2, 2, 40, 10), (300, 12, 4, 64, 32), (2, 0, 3, 64, 32), (2, 3, 0, 64, 32), (5, 6, 2, 18, 4), (70, 40, 40, 128, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k_bits,v_bits,norm", [(8, 8, True), (8, 4, False), (4, 4, True), (4, 8, False)])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,size,half", CASES)
def test_heads(tokens, q_heads, kv_heads, size, half, k_bits, v_bits, norm, dtype):
    gen = torch.Generator().manual_seed(tokens * size + half)
    pad = 3 if size % 8 else 8
    qkv = torch.randn(tokens, (q_heads + 2 * kv_heads) * size + pad, generator=gen).to(dtype)
    host = [t.unflatten(1, (-1, size)) if t.shape[1] else t.reshape(tokens, 0, size)
            for t in qkv[:, :-pad].split((q_heads * size, kv_heads * size, kv_heads * size), 1)]
    dev = qkv.to(DEV)
    q, k, v = [t.unflatten(1, (-1, size)) if t.shape[1] else t.reshape(tokens, 0, size)
               for t in dev[:, :-pad].split((q_heads * size, kv_heads * size, kv_heads * size), 1)]
    gains = [(1 + 0.2 * torch.randn(size, generator=gen)).to(dtype) if norm else None for _ in range(2)]
    cos, sin = table(50, half)
    positions = torch.randint(0, 50, (tokens,), generator=gen)
    slots = torch.randperm(2 * tokens + 3, generator=gen)[:tokens]
    kc, ks = empty_cache(2 * tokens + 3, kv_heads, size, k_bits)
    vc, vs = empty_cache(2 * tokens + 3, kv_heads, size, v_bits)
    out = ms().rotate_to_cache(q, k, v, cos.to(DEV), sin.to(DEV), positions.to(DEV), slots.to(DEV), kc, ks, vc, vs,
                               *(None if g is None else g.to(DEV) for g in gains), 1e-5)
    want, off = turned(host[0], gains[0], 1e-5, cos[positions], sin[positions])
    assert out.shape == want.shape and out.dtype == dtype
    assert ((out.cpu().double() - want).abs() <= off + torch.finfo(dtype).eps / 2 * (want.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
    if kv_heads:
        want, off = turned(host[1], gains[1], 1e-5, cos[positions], sin[positions])
        check_cached(kc.view(torch.uint8).cpu()[slots].view(kc.dtype), ks.cpu()[slots], want, off, k_bits)
        c, e = P.codes(host[2].double(), v_bits)
        assert torch.equal(P.unpack(vc.view(torch.uint8).cpu()[slots].view(vc.dtype)), c) and torch.equal(vs.cpu()[slots].to(torch.int64), e)
    rest = torch.ones(2 * tokens + 3, dtype=torch.bool)
    rest[slots] = False
    for t, fill in ((kc, 7), (ks, 99), (vc, 7), (vs, 99)):   # rows that no token names stay as they are
        assert (t.view(torch.uint8).cpu()[rest] == fill).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which", ["both", "q", "k"])
def test_many_heads_of_many_tokens(which, dtype):
    """So many that a workgroup goes through several rounds of heads; heads of zeros, of tiny numbers and without a number among them."""
    tokens, q_heads, kv_heads, size, half = 1100, 40, 12, 128, 64
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn(tokens, q_heads + 2 * kv_heads, size, generator=gen).to(dtype)
    qkv[3, 7], qkv[4, q_heads + 3], qkv[5, 9, 100], qkv[6, q_heads + 1, 2] = 0, 0, float("nan"), float("inf")
    if dtype == torch.bfloat16:
        qkv[7] *= 2.0 ** -120
    q, k, v = qkv.split((q_heads, kv_heads, kv_heads), 1)
    gains = [(1 + 0.2 * torch.randn(size, generator=gen)).to(dtype) if which in (name, "both") else None for name in "qk"]
    cos, sin = table(50, half)
    positions, slots = torch.randint(0, 50, (tokens,), generator=gen), torch.randperm(tokens + 3, generator=gen)[:tokens]
    (kc, ks), (vc, vs) = empty_cache(tokens + 3, kv_heads, size, 8), empty_cache(tokens + 3, kv_heads, size, 4)
    dev = [t.unflatten(1, (-1, size)) for t in qkv.flatten(1).to(DEV).split((q_heads * size, kv_heads * size, kv_heads * size), 1)]
    out = ms().rotate_to_cache(*dev, cos.to(DEV), sin.to(DEV), positions.to(DEV), slots.to(DEV), kc, ks, vc, vs, *(None if g is None else g.to(DEV) for g in gains), 0.0)
    bad = torch.zeros(tokens, q_heads, dtype=torch.bool)
    bad[5, 9] = True
    want, off = turned(q, gains[0], 1e-300, cos[positions], sin[positions])    # (eps 0; a head of zeros is zeros)
    got = out.cpu().double()
    if gains[0] is not None:
        assert got[bad].isnan().all()
    good = ~bad
    assert ((got - want).abs() <= off + torch.finfo(dtype).eps / 2 * (want.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134))[good].all()
    want, off = turned(k, gains[1], 1e-300, cos[positions], sin[positions])
    keys, scales = kc.view(torch.uint8).cpu()[slots].view(kc.dtype), ks.cpu()[slots]
    assert (scales[6, 1] == 255).any() if gains[1] is None else (scales[6, 1] == 255).all()
    keep = torch.ones(tokens, kv_heads, dtype=torch.bool)
    keep[6, 1] = False
    check_cached(keys.view(torch.uint8)[keep].view(kc.dtype), scales[keep], want[keep], off[keep] + 2.0 ** -149, 8)
    check_cached(vc.cpu()[slots], vs.cpu()[slots], v.double(), torch.zeros(()).double(), 4)


def simple(tokens=4, heads=2, size=64, bits=8, dtype=torch.float16):
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(tokens, heads, size, generator=gen).to(dtype).to(DEV) for _ in range(3))
    cos, sin = (t.to(DEV) for t in table(10, size // 2))
    return [q, k, v, cos, sin, torch.arange(tokens, device=DEV), torch.arange(tokens, device=DEV), *empty_cache(tokens + 2, heads, size, bits),
            *empty_cache(tokens + 2, heads, size, bits)]


@pytest.mark.parametrize("bits", [4, 8])
def test_slots_that_are_not_there(bits):
    a = simple(bits=bits)
    a[6] = torch.tensor([1, -1, 6, 2 ** 40], device=DEV)
    out = ms().rotate_to_cache(*a)
    assert out.isfinite().all()
    assert (a[8].cpu()[[0, 2, 3, 4, 5]] == 99).all() and (a[8].cpu()[1] != 99).all()
    assert (a[7].view(torch.uint8).cpu()[[0, 2, 3, 4, 5]] == 7).all()
    back = ms().dequantize(a[9], a[10], rows=a[6]).cpu()
    assert (back[1:] == 0).all() and (back[0] != 0).any()


@pytest.mark.parametrize("position", [-1, 10, 2 ** 40])
def test_positions_that_are_not_there(position):
    a = simple()
    a[5] = torch.tensor([0, position, 2, 3], device=DEV)
    out = ms().rotate_to_cache(*a).cpu()
    assert out[1].isnan().all() and out[[0, 2, 3]].isfinite().all()
    assert (a[8].cpu()[1] == 255).all() and (a[8].cpu()[[0, 2, 3]] != 255).all() and (a[10].cpu()[1] != 255).all()


def test_heads_without_a_number_and_of_zeros():
    a = simple(dtype=torch.bfloat16)
    gain = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    a[0][0, 0], a[0][1, 1, 3], a[1][2, 0, 5], a[2][3, 1, 40] = 0, float("nan"), float("inf"), float("inf")
    a[0][2, 0] *= 2.0 ** 80                                     # squares beyond fp32
    out = ms().rotate_to_cache(*a, gain, gain, eps=0.0).cpu()
    assert (out[0, 0] == 0).all() and out[1, 1].isnan().all() and out[2, 0].isnan().all()
    mask = torch.ones(4, 2, dtype=torch.bool)
    mask[1, 1] = mask[2, 0] = False
    assert out[mask].isfinite().all()
    assert (a[8].cpu()[2, 0] == 255).all() and (a[8].cpu()[:4] == 255).sum() == 2
    assert a[10].cpu()[3, 1].tolist()[1] == 255 and (a[10].cpu()[:4] == 255).sum() == 1


def test_a_head_of_tiny_numbers_is_normed():
    a = simple(dtype=torch.bfloat16)
    gain = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    plain = ms().rotate_to_cache(*a, gain, gain, eps=0.0)
    a[0] = a[0] * 2.0 ** -100
    assert torch.equal(ms().rotate_to_cache(*a, gain, gain, eps=0.0), plain)


def test_no_tokens():
    a = simple()
    for i in (0, 1, 2, 5, 6):
        a[i] = a[i][:0]
    assert ms().rotate_to_cache(*a).shape == (0, 2, 64) and (a[8] == 99).all()


def test_the_python_function_and_the_front_end_agree():
    from quik_amd import _lib as L
    outs = []
    for front in (None, L._NoFront()):
        a = simple(bits=4)
        kept = L.front()
        if front is not None:
            L._front = front
        try:
            outs.append([ms().rotate_to_cache(*a), *a[7:]])
            outs[-1].append(ms().dequantize(a[7], a[8], torch.bfloat16, rows=a[6]))
        finally:
            L._front = kept
    for x, y in zip(*outs):
        assert torch.equal(x, y)
