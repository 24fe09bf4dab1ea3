"""What the rows, products and caches in blocks of 32 refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch

import quik

ms = quik.microscaled
null, one, odd, at2, at8 = (ctypes.c_void_p(n) for n in (None, 256, 257, 258, 264))
BITS, SHAPE, DTYPE, ALIGN, NULL, RANGE = -1, -2, -3, -4, -5, -6


def _lib():
    from quik_amd import _lib as L
    return L.load()


def test_quantize_checks_its_arguments():
    def f(x=one, pitch=64, dt=0, rows=4, cols=64, bits=4, q=one, s=one):
        return _lib().quik_mx_quantize(x, pitch, dt, rows, cols, bits, q, s, null)
    assert f(rows=0) == 0
    assert f(bits=5) == BITS and f(bits=16) == BITS and f(dt=2) == DTYPE and f(dt=-1) == DTYPE
    assert f(rows=-1) == SHAPE and f(cols=0) == SHAPE and f(pitch=63) == SHAPE
    assert f(cols=63) == ALIGN and f(x=odd) == ALIGN
    assert f(rows=1 << 31) == RANGE and f(cols=(1 << 30) + 2, pitch=1 << 31) == RANGE
    assert f(x=null) == NULL and f(q=null) == NULL and f(s=null) == NULL


def test_activation_checks_its_arguments():
    def f(g=one, gp=64, u=one, up=64, dt=1, rows=4, cols=64, bits=8, q=one, s=one):
        return _lib().quik_mx_silu_mul_quantize(g, gp, u, up, dt, rows, cols, bits, q, s, null)
    assert f(rows=0) == 0
    assert f(bits=0) == BITS and f(dt=2) == DTYPE
    assert f(rows=-1) == SHAPE and f(cols=0) == SHAPE and f(gp=63) == SHAPE and f(up=63) == SHAPE
    assert f(cols=63, bits=4) == ALIGN and f(g=odd) == ALIGN and f(u=odd) == ALIGN
    assert f(rows=1 << 31) == RANGE and f(cols=(1 << 30) + 2, gp=1 << 31, up=1 << 31) == RANGE
    assert f(g=null) == NULL and f(u=null) == NULL and f(q=null) == NULL and f(s=null) == NULL


def test_norm_checks_its_arguments():
    def f(x=one, xp=64, r=one, rp=64, g=one, eps=1e-5, dt=0, rows=4, cols=64, bits=4, h=one, q=one, s=one, sr=one):
        return _lib().quik_mx_rms_norm_quantize(x, xp, r, rp, g, ctypes.c_float(eps), dt, rows, cols, bits, h, q, s, sr, null)
    assert f(rows=0) == 0
    assert f(bits=6) == BITS and f(dt=3) == DTYPE
    assert f(rows=-1) == SHAPE and f(cols=0) == SHAPE and f(xp=63) == SHAPE and f(rp=63) == SHAPE
    assert f(eps=-1e-9) == RANGE and f(eps=float("nan")) == RANGE and f(rows=1 << 31) == RANGE
    assert f(x=null) == NULL and f(g=null) == NULL and f(h=null) == NULL and f(q=null) == NULL and f(s=null) == NULL and f(sr=null) == NULL
    assert f(x=odd) == ALIGN and f(r=odd) == ALIGN and f(g=odd) == ALIGN and f(h=odd) == ALIGN and f(sr=at2) == ALIGN and f(cols=62 + 1) == ALIGN


def test_reading_checks_its_arguments():
    def f(q=one, bits=4, s=one, index=one, sr=null, dt=0, rows=4, source=4, heads=2, cols=64, out=one):
        return _lib().quik_mx_dequantize(q, bits, s, index, sr, dt, rows, source, heads, cols, out, null)
    assert f(rows=0) == 0 and f(heads=0) == 0
    assert f(bits=2) == BITS and f(dt=2) == DTYPE
    assert f(rows=-1) == SHAPE and f(source=-1) == SHAPE and f(heads=-1) == SHAPE and f(cols=0) == SHAPE and f(index=null, rows=3) == SHAPE
    assert f(heads=(1 << 30) + 1) == RANGE and f(cols=(1 << 30) + 2) == RANGE and f(heads=1 << 30, cols=1 << 10) == RANGE and f(rows=1 << 31) == RANGE
    assert f(q=null) == NULL and f(s=null) == NULL and f(out=null) == NULL
    assert f(cols=63) == ALIGN and f(out=odd) == ALIGN and f(index=ctypes.c_void_p(260)) == ALIGN and f(sr=at2) == ALIGN


def test_heads_check_their_arguments():
    from quik_amd import _lib as L
    given = dict(struct_bytes=ctypes.sizeof(L.QuikMxHeads), dtype=0, k_bits=8, v_bits=4, tokens=4, q_heads=8, kv_heads=2, size=64, half=32, positions=16,
                 slots=16, q_pitch=512, k_pitch=128, v_pitch=128, eps=1e-6, reserved=0)
    given.update({name: 256 for name in ("q", "k", "v", "cos", "sin", "position", "slot", "q_gain", "k_gain", "q_out", "k_codes", "k_scale", "v_codes",
                                         "v_scale")})

    def f(**kw):
        return _lib().quik_mx_rotate_to_cache(ctypes.byref(L.QuikMxHeads(**{**given, **kw})), null)
    assert _lib().quik_mx_rotate_to_cache(None, null) == NULL
    assert f(tokens=0) == 0 and f(q_heads=0, kv_heads=0) == 0
    assert f(struct_bytes=given["struct_bytes"] - 8) == SHAPE
    assert f(k_bits=5) == BITS and f(v_bits=16) == BITS and f(dtype=2) == DTYPE
    for name in ("tokens", "q_heads", "kv_heads", "positions", "slots"):
        assert f(**{name: -1}) == SHAPE, name
    assert f(size=0) == SHAPE and f(half=0) == SHAPE and f(half=33) == SHAPE
    assert f(q_pitch=511) == SHAPE and f(k_pitch=127) == SHAPE and f(v_pitch=127) == SHAPE
    assert f(size=63, half=31) == ALIGN and f(size=514, q_pitch=1 << 20, k_pitch=1 << 20, v_pitch=1 << 20) == RANGE
    assert f(tokens=1 << 31) == RANGE and f(q_heads=(1 << 20) + 1, q_pitch=1 << 40) == RANGE and f(kv_heads=(1 << 20) + 1) == RANGE
    assert f(eps=-1.0) == RANGE and f(eps=float("nan")) == RANGE
    for name in ("q", "k", "v", "cos", "sin", "position", "slot", "q_out", "k_codes", "k_scale", "v_codes", "v_scale"):
        assert f(**{name: None}) == NULL, name
    for name in ("q", "k", "v", "q_gain", "k_gain", "q_out"):
        assert f(**{name: 257}) == ALIGN, name
    for name, at in (("cos", 258), ("sin", 258), ("position", 260), ("slot", 260)):
        assert f(**{name: at}) == ALIGN, name


@pytest.mark.parametrize("gated", [False, True])
def test_products_check_their_arguments(gated):
    def f(x=one, bits=4, xs=one, w=one, ws=one, sr=null, b=null, dt=0, M=4, N=64, K=256, out=one, q_bits=4, q_scale=one, work=null):
        if gated:
            return _lib().quik_mx_gated_matmul(x, bits, xs, w, ws, sr, dt, M, N, K, q_bits, out, q_scale, null)
        return _lib().quik_mx_matmul(x, bits, xs, w, ws, sr, b, dt, M, N, K, out, work, 0, null)
    assert f(M=0) == 0 and f(N=0) == 0
    assert f(bits=16) == BITS and f(bits=2) == BITS and f(dt=2) == DTYPE
    assert f(M=-1) == SHAPE and f(N=-1) == SHAPE and f(K=0) == SHAPE and f(K=-32) == SHAPE
    assert f(K=240) == ALIGN and f(K=16) == ALIGN
    assert f(M=1 << 31) == RANGE and f(N=1 << 30) == RANGE and f(K=(1 << 20) + 32) == RANGE
    for name in ("x", "xs", "w", "ws", "out"):
        assert f(**{name: null}) == NULL, name
    assert f(x=at8) == ALIGN and f(w=at8) == ALIGN and f(sr=at2) == ALIGN
    if gated:
        assert f(q_bits=16) == BITS and f(N=48) == ALIGN and f(q_scale=null) == NULL
        assert f(N=1 << 20, K=1 << 17) == RANGE  # up's exponent bytes would start past 32 bits
    else:
        assert f(b=odd) == ALIGN and f(out=odd) == ALIGN and f(work=at8) == ALIGN


def test_product_says_what_it_makes_use_of():
    f = _lib().quik_mx_matmul_workspace_bytes
    assert f(4, 16, 4096, 4096) == 0 and f(8, 0, 4096, 4096) == 0 and f(4, 64, 0, 4096) == 0 and f(4, 64, 64, 0) == 0 and f(4, 64, 64, -32) == 0
    assert f(4, 2048, 8192, 8192) == 0 and f(4, 1 << 31, 64, 64) == 0 and f(4, 64, 1 << 30, 64) == 0 and f(4, 64, 64, (1 << 20) + 32) == 0
    n = f(4, 64, 5121, 13824)
    assert n > 0 and n % (64 * 5124 * 4) == 0  # whole parts of [64, 5124] sums


def test_tensors_that_are_not_on_a_gpu():
    x = torch.zeros(2, 64, dtype=torch.float16)
    q, s = torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    h, i = x.view(2, 1, 64), torch.zeros(2, dtype=torch.int64)
    cache, cs = q.view(2, 1, 32), s.view(2, 1, 2)
    angles = torch.zeros(4, 32)
    for call in (lambda: ms.quantize(x), lambda: ms.dequantize(q, s), lambda: ms.rms_norm_quantize(x, x[0]), lambda: ms.silu_mul_quantize(x, x),
                 lambda: ms.matmul(q, s, q, s), lambda: ms.gated_matmul(q, s, q, s),
                 lambda: ms.rotate_to_cache(h, h, h, angles, angles, i, i, cache, cs, cache, cs)):
        with pytest.raises(RuntimeError, match="on a CUDA"):
            call()
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        ms.quantize([1.0])


@pytest.mark.gpu
def test_rows_shapes_types_and_layouts():
    dev = "cuda:0"
    x, w = torch.zeros(2, 64, dtype=torch.float16, device=dev), torch.ones(64, dtype=torch.float16, device=dev)
    for args, kw, word in (((x.float(),), {}, "float16 or bfloat16"), ((x, 5), {}, "bits"), ((x[0],), {}, "matrix"), ((x.t(),), {}, "contiguous rows"),
                           ((x[:, :0],), {}, "no columns"), ((x[:, :63],), {}, "even"), ((x[:1].expand(2, 64),), {}, "do not overlap")):
        with pytest.raises(RuntimeError, match=word):
            ms.quantize(*args, **kw)
    for args, kw, word in (((x.float(), w), {}, "float16 or bfloat16"), ((x, w.bfloat16()), {}, "weight of dtype"), ((x, w[:63]), {}, "weight to have size"),
                           ((x, w), {"residual": x[:1]}, "size"), ((x, w), {"residual": x.bfloat16()}, "residual of dtype"), ((x, w, -1.0), {}, "eps"),
                           ((x, w, float("nan")), {}, "eps"), ((x, w), {"bits": 16}, "bits"), ((x, w.cpu()), {}, "CUDA"), ((x[:, :63], w[:63]), {}, "even"),
                           ((x, w[::2].repeat(2)[::2]), {}, "contiguous")):
        with pytest.raises(RuntimeError, match=word):
            ms.rms_norm_quantize(*args, **kw)
    for args, word in (((x, x.bfloat16()), "up of dtype"), ((x, x[:, :32]), "size"), ((x.int(), x), "float16"), ((x.t(), x.t()), "contiguous rows"), ((x, x, 1), "bits")):
        with pytest.raises(RuntimeError, match=word):
            ms.silu_mul_quantize(*args)
    q, s = ms.quantize(x)
    rows = torch.zeros(3, dtype=torch.int64, device=dev)
    for args, kw, word in (((q.char(), s), {}, "dtype torch.uint8"), ((q, s, torch.float32), {}, "float16 or bfloat16"), ((q[0], s[0]), {}, "two dimensions"),
                           ((q, s[:1]), {}, "scale to have size"), ((q, s.char()), {}, "scale of dtype"), ((q, s), {"rows": rows.int()}, "int64"),
                           ((q, s), {"rows": rows.view(3, 1)}, "int64"), ((q, s), {"scale_row": torch.ones(3, device=dev)}, "scale_row"),
                           ((q, s), {"rows": rows, "scale_row": torch.ones(2, device=dev)}, "scale_row"), ((q, s), {"rows": rows.cpu()}, "CUDA"),
                           ((q.t(), s), {}, "contiguous"), ((q[:, :0].contiguous(), s[:, :0].contiguous()), {}, "no columns")):
        with pytest.raises(RuntimeError, match=word):
            ms.dequantize(*args, **kw)


@pytest.mark.gpu
def test_products_shapes_types_and_layouts():
    dev = "cuda:0"
    x = torch.zeros(2, 64, dtype=torch.float16, device=dev)
    (q, s), (w, ws) = ms.quantize(x), ms.quantize(torch.zeros(64, 64, dtype=torch.float16, device=dev))
    row, bias = torch.ones(2, 1, device=dev), torch.zeros(64, dtype=torch.float16, device=dev)
    both = (((q.char(), s, w, ws), {}, "dtype torch.uint8"), ((q, s, w.char(), ws), {}, "weight of dtype"), ((q, s, w, ws, torch.float32), {}, "float16 or bfloat16"),
            ((q[0], s, w, ws), {}, "agree in K"), ((q, s, w[:, :16].contiguous(), ws), {}, "agree in K"), ((q, s[:1], w, ws), {}, "x_scale to have size"),
            ((q, s, w, ws[:, :1].contiguous()), {}, "weight_scale to have size"), ((q, s.char(), w, ws), {}, "x_scale of dtype"),
            ((q, s, w, ws), {"scale_row": row.half()}, "scale_row"), ((q, s, w, ws), {"scale_row": row[:1]}, "scale_row"),
            ((q[:, :24].contiguous(), s, w[:, :24].contiguous(), ws), {}, "multiple of 32"), ((q[:, :0].contiguous(), s, w[:, :0].contiguous(), ws), {}, "multiple of 32"),
            ((q, s, w.t(), ws), {}, "contiguous"), ((q, s, w.cpu(), ws), {}, "CUDA"))
    for op, more in ((ms.matmul, (((q, s, w, ws), {"bias": bias[:3]}, "bias"), ((q, s, w, ws), {"bias": bias.float()}, "bias"))),
                     (ms.gated_matmul, (((q, s, w[:32], ws[:32]), {}, "multiple of 32"), ((q, s, w[:0], ws[:0]), {}, "multiple of 32"), ((q, s, w, ws), {"bits": 3}, "bits")))):
        for args, kw, word in both + more:
            with pytest.raises(RuntimeError, match=word):
                op(*args, **kw)
    shifted = torch.zeros(2 * 32 + 8, dtype=torch.uint8, device=dev)[8:].view(2, 32)
    for op in (ms.matmul, ms.gated_matmul):
        with pytest.raises(RuntimeError, match="alignment"):
            op(shifted, s, w, ws)


@pytest.mark.gpu
def test_heads_shapes_types_and_layouts():
    dev = "cuda:0"
    h = torch.zeros(2, 4, 64, dtype=torch.float16, device=dev)
    kv = h[:, :2].contiguous()
    angles, i, gain = torch.zeros(8, 32, device=dev), torch.zeros(2, dtype=torch.int64, device=dev), torch.ones(64, dtype=torch.float16, device=dev)
    c4, c8 = torch.zeros(5, 2, 32, dtype=torch.uint8, device=dev), torch.zeros(5, 2, 64, device=dev).to(torch.float8_e4m3fn)
    sc = torch.zeros(5, 2, 2, dtype=torch.uint8, device=dev)
    good = dict(q=h, k=kv, v=kv, cos=angles, sin=angles, positions=i, slots=i, k_cache=c8, k_scale=sc, v_cache=c4, v_scale=sc.clone())
    assert ms.rotate_to_cache(**good).shape == h.shape
    for change, word in (({"q": h.float()}, "float16 or bfloat16"), ({"k": kv.bfloat16()}, "k of dtype"), ({"v": kv[:1]}, "v to have size"), ({"q": h[0]}, "heads, size"),
                         ({"q": h.transpose(1, 2)}, "contiguous heads"), ({"cos": angles[0]}, "cos"), ({"cos": angles.half()}, "cos of dtype"),
                         ({"sin": angles[:7]}, "sin to have size"), ({"cos": angles[:, :0].contiguous()}, "cos"),
                         ({"cos": torch.zeros(8, 33, device=dev), "sin": torch.zeros(8, 33, device=dev)}, "cos"), ({"positions": i.int()}, "positions of dtype"),
                         ({"slots": i[:1]}, "slots to have size"), ({"k_cache": c8.half()}, "dtype torch.uint8"), ({"k_cache": c8[0]}, "k_cache"),
                         ({"k_cache": c4[0, 0, 0]}, "k_cache"), ({"k_cache": c8[:, :1].contiguous()}, "k_cache to have size"), ({"v_cache": c4[:4]}, "v_cache to have size"),
                         ({"v_scale": sc[:4]}, "v_scale to have size"), ({"k_scale": sc.char()}, "k_scale of dtype"), ({"q_weight": gain[:63]}, "q_weight to have size"),
                         ({"k_weight": gain.float()}, "k_weight of dtype"), ({"eps": -1.0}, "eps"), ({"slots": i.cpu()}, "CUDA"),
                         ({"k_cache": c8.transpose(0, 1)}, "contiguous")):
        with pytest.raises(RuntimeError, match=word):
            ms.rotate_to_cache(**{**good, **change})


def test_the_typed_stub_describes_the_module():
    import ast
    import inspect
    import pathlib
    stub = ast.parse((pathlib.Path(quik.__file__).parent / "_C" / "microscaled.pyi").read_text())
    given = {f.name: [a.arg for a in f.args.args] for f in stub.body if isinstance(f, ast.FunctionDef)}
    assert given == {name: list(inspect.signature(getattr(ms, name)).parameters) for name in ms.__all__}
