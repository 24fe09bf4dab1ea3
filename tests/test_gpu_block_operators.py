"""The 8-bit row operators and the grouped 4-bit product as a decoder block runs them: one after the other, as modules, from graphs
between eager calls, on streams of their own, with and without the native front end."""
import numpy as np
import pytest
import torch

import quik
from quik_amd.qlinear import GroupLinear4bit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _block(hidden, inner, dtype, symm, seed=0):
    torch.manual_seed(seed)
    lin = lambda n, m: GroupLinear4bit.from_float(torch.nn.Linear(n, m, bias=not symm, dtype=dtype, device=DEV), 128, symm)
    return lin(hidden, 2 * inner), lin(inner, hidden), (1 + 0.1 * torch.randn(hidden, device=DEV)).to(dtype)


def _run(block, x, residual):
    up, down, gain = block
    q, scale, h = quik.symmetric.rms_norm_quantize(x, gain, 1e-5, residual=residual)
    both = up(q, scale)
    q, scale = quik.symmetric.silu_mul_quantize(*both.chunk(2, -1))
    return down(q, scale), h


def _weight(mod):
    by = mod.int_weight.cpu().numpy()
    q = np.empty((by.shape[0], 2 * by.shape[1]))
    q[:, 0::2], q[:, 1::2] = ((by & 15) ^ 8).astype(int) - 8, ((by >> 4) ^ 8).astype(int) - 8
    at = np.arange(q.shape[1]) // mod.group_size
    z = 0 if mod.zeros is None else mod.zeros.double().cpu().numpy()[:, at]
    return (q - z) * mod.scales.double().cpu().numpy()[:, at]


def _rows(v):
    step = np.abs(v).max(1, keepdims=True) / 127
    return np.rint(v / step) * step


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("symm", [True, False])
@pytest.mark.parametrize("rows", [1, 5, 16, 48, 200])
def test_mlp(rows, symm, dtype):
    """Against the block in 64 bits.  Differences: 16-bit results of both products (half a step each), and codes that a value next to a
    border rounds to the other side: a step of a row's scale, for few values, so norms are compared."""
    block = _block(512, 1376, dtype, symm)
    x, r = torch.randn(rows, 512, device=DEV).to(dtype), torch.randn(rows, 512, device=DEV).to(dtype)
    out, h = _run(block, x, r)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    hd = h.double().cpu().numpy()
    v = _rows(hd / np.sqrt((hd ** 2).mean(1, keepdims=True) + 1e-5) * block[2].double().cpu().numpy())
    bias = lambda m: 0 if m.bias is None else m.bias.double().cpu().numpy()
    both = v @ _weight(block[0]).T + bias(block[0])
    g, u = both[:, :1376], both[:, 1376:]
    want = _rows(g / (1 + np.exp(-g)) * u) @ _weight(block[1]).T + bias(block[1])
    got = out.double().cpu().numpy()
    # gate and up are rounded (each by eps / 2 at most, so their product by eps), what that moves in the codes is of a step's size for
    # few values; the result is rounded once
    eps = torch.finfo(dtype).eps
    assert np.linalg.norm(got - want) <= (eps / 2 + 2 * eps + 2.0 ** -8) * np.linalg.norm(want)


@pytest.mark.parametrize("symm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_module_from_float(dtype, symm):
    torch.manual_seed(3)
    lin = torch.nn.Linear(352, 96, dtype=dtype, device=DEV)
    lin.weight.data[5] = 0
    lin.weight.data[6, 64:128] = lin.weight.data[6, 64:128].abs() + 1   # a group on one side of zero
    mod = GroupLinear4bit.from_float(lin, 64, symm)
    w, want = _weight(mod), lin.weight.double().cpu().detach().numpy()
    at = np.arange(352) // 64
    step = mod.scales.double().cpu().numpy()[:, at]
    # half a step; the scale is rounded to 16 bits before the codes, which moves the largest code's value by 8 (15) half steps of the type
    assert (np.abs(w - want) <= step * (0.5 + 16 * torch.finfo(mod.scales.dtype).eps / 2 + 1e-6)).all()
    assert not w[5].any()
    x = torch.randn(2, 7, 352, device=DEV).to(mod.scales.dtype)
    out = mod(x)
    assert out.shape == (2, 7, 96) and out.dtype == mod.scales.dtype
    y = x.double().cpu().numpy() @ w.T + mod.bias.double().cpu().numpy()
    assert np.linalg.norm(out.double().cpu().numpy() - y) <= torch.finfo(out.dtype).eps / 2 * np.linalg.norm(y)
    twin = GroupLinear4bit(352, 96, 64, not symm, True, mod.scales.dtype).to(DEV)
    twin.load_state_dict(mod.state_dict())
    assert torch.equal(twin(x), out)


@pytest.mark.parametrize("rows", [1, 16, 70, 300])
def test_replayed_between_eager_calls(rows):
    """A captured block, replayed with new inputs between eager runs of the same and of other sizes, equals the eager run each time.  70 rows:
    K is split, so that the graph holds the memory of the parts."""
    block = _block(1024, 4096, torch.float16, True)
    x, r = torch.randn(rows, 1024, device=DEV).half(), torch.randn(rows, 1024, device=DEV).half()
    want = _run(block, x, r)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _run(block, x, r)
        graphs.append((g, out))
    for i in range(4):
        x.copy_(torch.randn(rows, 1024, device=DEV))
        want = _run(block, x, r)
        _run(block, torch.randn(33, 1024, device=DEV).half(), torch.randn(33, 1024, device=DEV).half())
        for g, out in graphs:
            g.replay()
        if i % 2:
            torch.cuda.synchronize()
        for g, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_captured_first():
    """A call whose sizes no eager call has had is captured like any other."""
    x, w = torch.randn(19, 640, device=DEV).half(), torch.randint(0, 256, (170, 320), device=DEV, dtype=torch.uint8)
    s = torch.rand(170, 5, device=DEV).half()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = quik.matmul.int4GroupMatmul(x, w, s, 128)
        q, sc, _ = quik.symmetric.rms_norm_quantize(x, x[0])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, quik.matmul.int4GroupMatmul(x, w, s, 128))
    assert torch.equal(q, quik.symmetric.rms_norm_quantize(x, x[0])[0])


def test_two_streams_at_once():
    block = _block(1024, 2752, torch.bfloat16, False)
    inputs = [[torch.randn(n, 1024, device=DEV).bfloat16() for _ in range(2)] for n in (64, 90)]
    want = [_run(block, *i) for i in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in inputs], [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(_run(block, *inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out, h in got[k]:
            assert torch.equal(out, want[k][0]) and torch.equal(h, want[k][1])


def test_same_bits_without_the_front_end(monkeypatch):
    from quik_amd import _lib as L
    block = _block(512, 1376, torch.float16, False)
    for rows in (1, 40):
        x, r = torch.randn(rows, 512, device=DEV).half(), torch.randn(rows, 512, device=DEV).half()
        want = _run(block, x, r)
        with monkeypatch.context() as m:
            m.setattr(L, "_front", L._NoFront())
            got = _run(block, x, r)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_parameters_and_views_take_the_python_path():
    x, w = torch.randn(3, 256, device=DEV).half(), torch.nn.Parameter(torch.randn(256, device=DEV).half())
    a, b = quik.symmetric.rms_norm_quantize(x, w), quik.symmetric.rms_norm_quantize(x, w.detach())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not a[1].requires_grad
    q, s, _ = quik.symmetric.rms_norm_quantize(x, w, 1)      # a whole number as eps
    assert s.isfinite().all()
