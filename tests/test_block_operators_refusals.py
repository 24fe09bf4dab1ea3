"""What the 8-bit row operators and the product with grouped 4-bit weights refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch

import quik

null, one, odd = ctypes.c_void_p(None), ctypes.c_void_p(256), ctypes.c_void_p(257)


def _lib():
    from quik_amd import _lib as L
    return L.load()


def test_norm_checks_its_arguments():
    def f(x=one, xp=64, r=one, rp=64, g=one, eps=1e-5, dt=0, rows=4, cols=64, h=one, q=one, s=one, st=2):
        return _lib().quik_rms_norm_quantize(x, xp, r, rp, g, ctypes.c_float(eps), dt, rows, cols, h, q, s, st, null)
    assert f(rows=0) == 0
    assert f(dt=2) == -3 and f(dt=-1) == -3 and f(st=3) == -3 and f(st=-1) == -3
    assert f(rows=-1) == -2 and f(cols=0) == -2 and f(xp=63) == -2 and f(rp=63) == -2
    assert f(eps=-1.0) == -6 and f(eps=float("nan")) == -6 and f(cols=1 << 31, xp=1 << 31, rp=1 << 31) == -6 and f(rows=1 << 31) == -6
    assert f(x=null) == -5 and f(g=null) == -5 and f(h=null) == -5 and f(q=null) == -5 and f(s=null) == -5
    assert f(x=odd) == -4 and f(r=odd) == -4 and f(g=odd) == -4 and f(h=odd) == -4 and f(s=ctypes.c_void_p(258)) == -4


def test_activation_checks_its_arguments():
    def f(g=one, gp=64, u=one, up=64, dt=0, rows=4, cols=64, q=one, s=one, st=2):
        return _lib().quik_silu_mul_quantize(g, gp, u, up, dt, rows, cols, q, s, st, null)
    assert f(rows=0) == 0
    assert f(dt=2) == -3 and f(st=3) == -3 and f(rows=-1) == -2 and f(cols=0) == -2 and f(gp=63) == -2 and f(up=63) == -2
    assert f(cols=1 << 31, gp=1 << 31, up=1 << 31) == -6 and f(rows=1 << 31) == -6
    assert f(g=null) == -5 and f(u=null) == -5 and f(q=null) == -5 and f(s=null) == -5
    assert f(g=odd) == -4 and f(u=odd) == -4 and f(s=ctypes.c_void_p(258)) == -4


def test_product_checks_its_arguments():
    def f(x=one, bits=16, w=one, s=one, z=null, sr=null, b=null, dt=0, M=4, N=8, K=256, G=128, out=one, ws=null):
        return _lib().quik_int4_group_matmul(x, bits, w, s, z, sr, b, dt, M, N, K, G, out, ws, 0, null)
    assert f(M=0) == 0 and f(N=0) == 0
    assert f(bits=4) == -1 and f(dt=2) == -3
    assert f(M=-1) == -2 and f(N=-1) == -2 and f(K=0) == -2 and f(G=0) == -2 and f(G=-32) == -2
    assert f(K=240) == -4 and f(G=48) == -4
    assert f(K=(1 << 20) + 32) == -6 and f(N=1 << 31) == -6 and f(M=1 << 31) == -6
    assert f(x=null) == -5 and f(w=null) == -5 and f(s=null) == -5 and f(out=null) == -5 and f(bits=8) == -5
    at8 = ctypes.c_void_p(264)
    assert f(x=at8) == -4 and f(w=at8) == -4 and f(s=odd) == -4 and f(z=odd) == -4 and f(b=odd) == -4 and f(out=odd) == -4 and f(ws=at8) == -4
    assert f(bits=8, sr=ctypes.c_void_p(258)) == -4


def test_tensors_that_are_not_on_a_gpu():
    x, w = torch.zeros(2, 64, dtype=torch.float16), torch.zeros(4, 32, dtype=torch.uint8)
    for call in (lambda: quik.symmetric.rms_norm_quantize(x, x[0]), lambda: quik.symmetric.silu_mul_quantize(x, x),
                 lambda: quik.matmul.int4GroupMatmul(x, w, x[:, :1], 64)):
        with pytest.raises(RuntimeError, match="on a CUDA"):
            call()
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        quik.symmetric.rms_norm_quantize([1.0], x[0])


@pytest.mark.gpu
def test_shapes_types_and_layouts():
    dev = "cuda:0"
    x, w = torch.zeros(2, 64, dtype=torch.float16, device=dev), torch.ones(64, dtype=torch.float16, device=dev)
    norm, silu = quik.symmetric.rms_norm_quantize, quik.symmetric.silu_mul_quantize
    for args, kw, word in (((x.float(), w), {}, "float16 or bfloat16"), ((x, w.bfloat16()), {}, "weight of dtype"), ((x, w[:63]), {}, "weight to have size"),
                           ((x, w), {"residual": x[:1]}, "residual to have size"), ((x, w), {"residual": x.bfloat16()}, "residual of dtype"),
                           ((x.t(), w[:2]), {}, "contiguous rows"), ((x[0], w), {}, "matrix"), ((x[:1].expand(2, 64), w), {}, "do not overlap"),
                           ((x, w, -1.0), {}, "eps"), ((x[:, :0], w[:0]), {}, "no columns"), ((x, w), {"scale_dtype": torch.int8}, "scale_dtype"),
                           ((x, w.cpu()), {}, "CUDA"), ((x, w[::2].repeat(2)[::2]), {}, "contiguous")):
        with pytest.raises(RuntimeError, match=word):
            norm(*args, **kw)
    for args, word in (((x, x.bfloat16()), "up of dtype"), ((x, x[:, :32]), "same size"), ((x.int(), x), "float16"), ((x.t(), x.t()), "contiguous rows")):
        with pytest.raises(RuntimeError, match=word):
            silu(*args)
    q = torch.zeros(2, 64, dtype=torch.int8, device=dev)
    p, s, sr = torch.zeros(4, 32, dtype=torch.uint8, device=dev), torch.ones(4, 1, dtype=torch.float16, device=dev), torch.ones(2, 1, device=dev)
    for args, kw, word in (((x, p, s.float(), 64), {}, "float16"), ((x.bfloat16(), p, s, 64), {}, "x of dtype"), ((x, p.char(), s, 64), {}, "weight of dtype"),
                           ((q, p, s, 64), {}, "scale_row"), ((x, p, s, 64), {"scale_row": sr}, "scale_row"), ((q, p, s, 64), {"scale_row": sr.half()}, "scale_row of dtype"),
                           ((q, p, s, 64), {"scale_row": sr[:1]}, "scale_row to have"), ((x, p, s, 32), {}, "scales to have size"), ((x, p, s, 48), {}, "multiples of 32"),
                           ((x, p, s, 0), {}, "multiples of 32"), ((x, p[:, :16].contiguous(), s, 64), {}, "agree in K"), ((x[0], p, s, 64), {}, "agree in K"),
                           ((x, p, s, 64), {"zeros": s[:2]}, "zeros to have size"), ((x, p, s, 64), {"zeros": s.float()}, "zeros of dtype"),
                           ((x, p, s, 64), {"bias": s[:3]}, "bias to have"), ((x, p, s, 64), {"bias": s.float()}, "bias of dtype"),
                           ((x[:, ::2].repeat(1, 2)[:, ::1], p.t(), s, 64), {}, "contiguous")):
        with pytest.raises(RuntimeError, match=word):
            quik.matmul.int4GroupMatmul(*args, **kw)
    shifted = torch.zeros(2 * 64 + 1, dtype=torch.float16, device=dev)[1:].view(2, 64)
    with pytest.raises(RuntimeError, match="alignment"):
        quik.matmul.int4GroupMatmul(shifted, p, s, 64)


def test_product_says_what_it_makes_use_of():
    f = _lib().quik_int4_group_matmul_workspace_bytes
    assert f(16, 0, 16, 4096, 4096) == 0 and f(16, 0, 0, 4096, 4096) == 0 and f(8, 0, 64, 0, 4096) == 0
    assert f(16, 0, 2048, 8192, 8192) == 0                        # tiles for every CU
    n = f(8, 1, 64, 5121, 13824)                                  # few tiles, long rows: whole parts of [64, 5124] sums
    assert n > 0 and n % (64 * 5124 * 4) == 0
