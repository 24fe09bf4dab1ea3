"""quik.microscaled: rows, products and caches in blocks of 32 numbers that share a power of two.  No counterpart in the reference.

32 neighbouring columns are held as 4-bit (e2m1) or 8-bit (e4m3) floating-point codes and one exponent byte e, for 2^(e - 127):
  4 bits  q [.., cols / 2] uint8, two codes per byte, the even column in the low half
  8 bits  q [.., cols] float8_e4m3fn
  scale   [.., ceil(cols / 32)] uint8
e is the exponent of the block's largest magnitude less that of the format's largest number (2 and 8), a code the nearest number of the
format, of two the even code, at most 6 and 448.  A block with a NaN or an infinity has e = 255 and gives NaNs wherever it is read.
The calls run on the current stream of the tensors' GPU, allocate their results and workspaces through torch, and can be captured.
There are no gradients: the rows are a serving program's."""
from __future__ import annotations

import ctypes

import torch

from . import _lib as L

__all__ = ["quantize", "dequantize", "rms_norm_quantize", "silu_mul_quantize", "matmul", "gated_matmul", "rotate_to_cache"]

BLOCK = 32


def _bits_of(op, name, q):
    if q.dtype == torch.uint8:
        return 4
    if q.dtype == torch.float8_e4m3fn:
        return 8
    raise RuntimeError(f"{op}: expected {name} of dtype torch.uint8 (4-bit codes) or torch.float8_e4m3fn but got {q.dtype}")


def _check_bits(op, bits, cols):
    if bits not in (4, 8):
        raise RuntimeError(f"{op}: expected bits to be 4 or 8 but got {bits}")
    if cols == 0:
        raise RuntimeError(f"{op}: rows of no columns have no blocks")
    if bits == 4 and cols % 2:
        raise RuntimeError(f"{op}: 4-bit codes lie two to a byte: the number of columns must be even, got {cols}")


def _codes(shape, bits, dev):
    """Uninitialised (q, scale) of a tensor of numbers."""
    *lead, cols = shape
    q = torch.empty((*lead, cols // 2), dtype=torch.uint8, device=dev) if bits == 4 else \
        torch.empty((*lead, cols), dtype=torch.float8_e4m3fn, device=dev)
    return q, torch.empty((*lead, -(-cols // BLOCK)), dtype=torch.uint8, device=dev)


def _expect(op, name, t, dtype, shape):
    if t.dtype != dtype:
        raise RuntimeError(f"{op}: expected {name} of dtype {dtype} but got {t.dtype}")
    if t.shape != torch.Size(shape):
        raise RuntimeError(f"{op}: expected {name} to have size {tuple(shape)}, got {tuple(t.shape)}")


def _same_gpu(op, dev, **tensors):
    given = {name: t for name, t in tensors.items() if t is not None}
    if given and L.check_cuda_contiguous(op, **given) != dev:
        raise RuntimeError(f"{op}: expected all tensors on the same GPU, but {', '.join(given)} are not on {dev}")


def _float_type(op, dtype):
    if dtype == torch.float16:
        return L.QUIK_F16
    if dtype == torch.bfloat16:
        return L.QUIK_BF16
    raise RuntimeError(f"{op}: expected dtype to be float16 or bfloat16 but got {dtype}")


def quantize(src: torch.Tensor, bits: int = 4):
    """(q, scale) of src [rows, cols] fp16 or bf16, whose rows may lie apart."""
    op = "quantize"
    out = L.front().mx_quantize(src, bits)
    if out is not None:
        return out
    dev = L.check_cuda_rows(op, src=src)
    dt = L.dtype_id(src, op, allow_bf16=True)
    rows, cols = src.shape
    _check_bits(op, bits, cols)
    lib = L.load()
    with L.device_guard(dev):
        q, scale = _codes(src.shape, bits, dev)
        L.check(lib.quik_mx_quantize(L.ptr(src), src.stride(0), dt, rows, cols, bits, L.ptr(q), L.ptr(scale), L.stream()), op)
    return q, scale


def dequantize(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float16, rows: torch.Tensor = None,
               scale_row: torch.Tensor = None) -> torch.Tensor:
    """The numbers that codes stand for, in fp16 or bf16 [.., cols]; with scale_row [rows] or [rows, 1] fp32 times a factor per row.
    rows (int64, any number of them): of the first dimension, those rows in that order; one that is not there gives zeros (a cache's slots;
    scale_row then goes by the result's rows)."""
    op = "dequantize"
    out = L.front().mx_dequantize(q, scale, dtype, rows, scale_row)
    if out is not None:
        return out
    dev = L.check_cuda_contiguous(op, q=q, scale=scale)
    bits, dt = _bits_of(op, "q", q), _float_type(op, dtype)
    if q.dim() < 2:
        raise RuntimeError(f"{op}: expected q to have at least two dimensions, got {tuple(q.shape)}")
    source_rows, *lead, width = q.shape
    cols = width * 2 if bits == 4 else width
    _check_bits(op, bits, cols)
    _expect(op, "scale", scale, torch.uint8, (source_rows, *lead, -(-cols // BLOCK)))
    _same_gpu(op, dev, rows=rows, scale_row=scale_row)
    if rows is not None and (rows.dtype != torch.int64 or rows.dim() != 1):
        raise RuntimeError(f"{op}: expected rows to be a list of int64, got {rows.dtype} {tuple(rows.shape)}")
    count = source_rows if rows is None else rows.numel()
    if scale_row is not None and (scale_row.dtype != torch.float32 or scale_row.numel() != count):
        raise RuntimeError(f"{op}: expected scale_row to be {count} float32 numbers, got {scale_row.dtype} {tuple(scale_row.shape)}")
    heads = 1
    for n in lead:
        heads *= n
    lib = L.load()
    with L.device_guard(dev):
        out = torch.empty((count, *lead, cols), dtype=dtype, device=dev)
        L.check(lib.quik_mx_dequantize(L.ptr(q), bits, L.ptr(scale), L.ptr(rows), L.ptr(scale_row), dt, count, source_rows, heads, cols,
                                       L.ptr(out), L.stream()), op)
    return out


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor = None, bits: int = 4):
    """Root-mean-square norm in blocks of 32, in one launch: h = x + residual (rounded to x's type; residual None: h = x), value = h * weight *
    scale_row with scale_row = 1 / sqrt(mean(h^2) + eps).  Returns (q, scale, scale_row, h): the codes are those of h * weight, scale_row
    [rows, 1] fp32 goes to matmul and gated_matmul; h is the next residual (None without one).  A row with a NaN, or whose squares' sum passes fp32's
    range, has the factor NaN.

    x, residual [rows, cols] fp16 or bf16 (rows may lie apart), weight [cols] of the same type."""
    op = "rms_norm_quantize"
    out = L.front().mx_rms_norm_quantize(x, weight, eps, residual, bits)
    if out is not None:
        return out
    rows_of = dict(x=x) if residual is None else dict(x=x, residual=residual)
    dev = L.check_cuda_rows(op, **rows_of)
    _same_gpu(op, dev, weight=weight)
    dt = L.dtype_id(x, op, allow_bf16=True)
    rows, cols = x.shape
    _check_bits(op, bits, cols)
    _expect(op, "weight", weight, x.dtype, (cols,))
    if residual is not None:
        _expect(op, "residual", residual, x.dtype, x.shape)
    if not eps >= 0:
        raise RuntimeError(f"{op}: expected eps to be at least 0 but got {eps}")
    lib = L.load()
    with L.device_guard(dev):
        q, scale = _codes(x.shape, bits, dev)
        scale_row = torch.empty((rows, 1), dtype=torch.float32, device=dev)
        h = None if residual is None else torch.empty((rows, cols), dtype=x.dtype, device=dev)
        L.check(lib.quik_mx_rms_norm_quantize(L.ptr(x), x.stride(0), L.ptr(residual), 0 if residual is None else residual.stride(0),
                                              L.ptr(weight), eps, dt, rows, cols, bits, L.ptr(h), L.ptr(q), L.ptr(scale), L.ptr(scale_row),
                                              L.stream()), op)
    return q, scale, scale_row, h


def silu_mul_quantize(gate: torch.Tensor, up: torch.Tensor, bits: int = 4):
    """(q, scale) of gate * sigmoid(gate) * up, in one launch.  gate and up [rows, cols] of one type, fp16 or bf16; their rows may lie apart
    (the two halves of one product)."""
    op = "silu_mul_quantize"
    out = L.front().mx_silu_mul_quantize(gate, up, bits)
    if out is not None:
        return out
    dev = L.check_cuda_rows(op, gate=gate, up=up)
    dt = L.dtype_id(gate, op, allow_bf16=True)
    rows, cols = gate.shape
    _check_bits(op, bits, cols)
    _expect(op, "up", up, gate.dtype, gate.shape)
    lib = L.load()
    with L.device_guard(dev):
        q, scale = _codes(gate.shape, bits, dev)
        L.check(lib.quik_mx_silu_mul_quantize(L.ptr(gate), gate.stride(0), L.ptr(up), up.stride(0), dt, rows, cols, bits, L.ptr(q), L.ptr(scale),
                                              L.stream()), op)
    return q, scale


def _product_checks(op, x, x_scale, weight, weight_scale, scale_row, bias, dtype):
    given = {name: t for name, t in (("scale_row", scale_row), ("bias", bias)) if t is not None}
    dev = L.check_cuda_contiguous(op, x=x, x_scale=x_scale, weight=weight, weight_scale=weight_scale, **given)
    bits, dt = _bits_of(op, "x", x), _float_type(op, dtype)
    if weight.dtype != torch.uint8:
        raise RuntimeError(f"{op}: expected weight of dtype torch.uint8 but got {weight.dtype}")
    if x.dim() != 2 or weight.dim() != 2 or x.size(1) * (8 // bits) != 2 * weight.size(1):
        raise RuntimeError(f"{op}: x and weight [N, K/2] must be matrices that agree in K, got {tuple(x.shape)} and {tuple(weight.shape)}")
    M, N, K = x.size(0), weight.size(0), 2 * weight.size(1)
    if K == 0 or K % BLOCK:
        raise RuntimeError(f"{op}: K must be a multiple of 32, got {K}")
    _expect(op, "x_scale", x_scale, torch.uint8, (M, K // BLOCK))
    _expect(op, "weight_scale", weight_scale, torch.uint8, (N, K // BLOCK))
    if scale_row is not None and (scale_row.dtype != torch.float32 or scale_row.numel() != M):
        raise RuntimeError(f"{op}: expected scale_row to be {M} float32 numbers, got {scale_row.dtype} {tuple(scale_row.shape)}")
    if bias is not None and (bias.dtype != dtype or bias.numel() != N):
        raise RuntimeError(f"{op}: expected bias to be {N} numbers of {dtype}, got {bias.dtype} {tuple(bias.shape)}")
    return dev, bits, dt, M, N, K


def matmul(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, dtype: torch.dtype = torch.float16,
           scale_row: torch.Tensor = None, bias: torch.Tensor = None) -> torch.Tensor:
    """out[m, n] = scale_row[m] * sum_k x[m, k] * weight[n, k] + bias[n], of dtype (fp16 or bf16).

    x, x_scale: 4- or 8-bit rows [M, K] as quantize, rms_norm_quantize, silu_mul_quantize and gated_matmul give them; weight [N, K/2] uint8 and
    weight_scale [N, K/32] 4-bit ones; scale_row [M] or [M, 1] fp32 (rms_norm_quantize); bias [N] of dtype.  K is a multiple of 32; x and weight start
    at a multiple of 16 bytes.  Sums in fp32, one rounding."""
    op = "matmul"
    out = L.front().mx_matmul(x, x_scale, weight, weight_scale, dtype, scale_row, bias)
    if out is not None:
        return out
    dev, bits, dt, M, N, K = _product_checks(op, x, x_scale, weight, weight_scale, scale_row, bias, dtype)
    lib = L.load()
    with L.device_guard(dev):
        out = torch.empty((M, N), dtype=dtype, device=dev)
        need = lib.quik_mx_matmul_workspace_bytes(bits, M, N, K)
        ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
        L.check(lib.quik_mx_matmul(L.ptr(x), bits, L.ptr(x_scale), L.ptr(weight), L.ptr(weight_scale), L.ptr(scale_row), L.ptr(bias), dt, M, N, K,
                                   L.ptr(out), L.ptr(ws), need, L.stream()), op)
    return out


def gated_matmul(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, dtype: torch.dtype = torch.float16,
                 scale_row: torch.Tensor = None, bits: int = 4):
    """The first half of a gated feed-forward block in one launch: (q, scale) [M, inner] of silu(gate) * up, gate = x weight[:inner]^T, up = x
    weight[inner:]^T (times scale_row), both rounded to dtype.  weight [2 * inner, K/2] is gate's and up's one after the other, inner a multiple of
    32; everything else as in matmul.  The codes are those that silu_mul_quantize makes of matmul's result, up to the order of the sums over K."""
    op = "gated_matmul"
    out = L.front().mx_gated_matmul(x, x_scale, weight, weight_scale, dtype, scale_row, bits)
    if out is not None:
        return out
    dev, x_bits, dt, M, N, K = _product_checks(op, x, x_scale, weight, weight_scale, scale_row, None, dtype)
    if N % (2 * BLOCK) or N == 0:
        raise RuntimeError(f"{op}: expected weight to have 2 * inner rows, inner a multiple of 32, got {N}")
    _check_bits(op, bits, N // 2)
    lib = L.load()
    with L.device_guard(dev):
        q, scale = _codes((M, N // 2), bits, dev)
        L.check(lib.quik_mx_gated_matmul(L.ptr(x), x_bits, L.ptr(x_scale), L.ptr(weight), L.ptr(weight_scale), L.ptr(scale_row), dt, M, N // 2, K,
                                         bits, L.ptr(q), L.ptr(scale), L.stream()), op)
    return q, scale


def _check_heads(op, **tensors):
    """[tokens, heads, size] whose heads follow each other and whose tokens may lie apart."""
    def laid_out(t):
        if t.dim() != 3:
            return False
        n, heads, size = t.shape
        return (size <= 1 or t.stride(2) == 1) and (heads <= 1 or t.stride(1) == size) and (n <= 1 or t.stride(0) >= heads * size)
    return L._check_cuda(op, laid_out, "[tokens, heads, size] with contiguous heads and tokens that do not overlap", tensors)


def rotate_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                    slots: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor, v_cache: torch.Tensor, v_scale: torch.Tensor,
                    q_weight: torch.Tensor = None, k_weight: torch.Tensor = None, eps: float = 1e-6) -> torch.Tensor:
    """Heads on their way from a block's first product to its attention, in one launch: queries and keys are normed per head (where there is a
    weight: x / sqrt(mean(x^2) + eps) * weight), turned by their token's position, and keys and values are put into the cache in blocks of 32 columns of a
    head.  Returns the queries [tokens, q_heads, size] in their type; reads the cache back: dequantize(k_cache, k_scale, dtype, rows=slots).

    q [tokens, q_heads, size], k and v [tokens, kv_heads, size] of one type, fp16 or bf16; tokens may lie apart (columns of one product); size even,
    at most 512.  cos, sin [positions, r] fp32 with 2 r <= size: columns i and i + r turn by the angle i < r of the token's position (columns from
    2 r on stay); positions, slots [tokens] int64.  k_cache, v_cache [slots, kv_heads, size / 2] uint8 or [slots, kv_heads, size] float8_e4m3fn, k_scale,
    v_scale [slots, kv_heads, ceil(size / 32)] uint8 (pages of a cache as one list of slots); keys and values may be held in different bits.
    A token whose slot is negative or behind the end writes nothing to the cache, other rows of it stay as they are; two tokens may not name the same
    slot (its row is then of neither for certain).  A position that cos does not have gives NaNs."""
    op = "rotate_to_cache"
    out = L.front().mx_rotate_to_cache(q, k, v, cos, sin, positions, slots, k_cache, k_scale, v_cache, v_scale, q_weight, k_weight, eps)
    if out is not None:
        return out
    dev = _check_heads(op, q=q, k=k, v=v)
    weights = {name: t for name, t in (("q_weight", q_weight), ("k_weight", k_weight)) if t is not None}
    _same_gpu(op, dev, cos=cos, sin=sin, positions=positions, slots=slots, k_cache=k_cache, k_scale=k_scale, v_cache=v_cache, v_scale=v_scale, **weights)
    dt = L.dtype_id(q, op, allow_bf16=True)
    tokens, q_heads, size = q.shape
    kv_heads = k.size(1)
    _expect(op, "k", k, q.dtype, (tokens, kv_heads, size))
    _expect(op, "v", v, q.dtype, (tokens, kv_heads, size))
    if size == 0 or size % 2 or size > 512:
        raise RuntimeError(f"{op}: the heads' size must be even and at most 512, got {size}")
    if cos.dim() != 2 or cos.size(1) == 0 or 2 * cos.size(1) > size:
        raise RuntimeError(f"{op}: expected cos [positions, r] with 2 r <= {size}, got {tuple(cos.shape)}")
    _expect(op, "cos", cos, torch.float32, cos.shape)
    _expect(op, "sin", sin, torch.float32, cos.shape)
    _expect(op, "positions", positions, torch.int64, (tokens,))
    _expect(op, "slots", slots, torch.int64, (tokens,))
    bits = {}
    if k_cache.dim() != 3:
        raise RuntimeError(f"{op}: expected k_cache to have three dimensions, got {tuple(k_cache.shape)}")
    for name, cache, scale in (("k", k_cache, k_scale), ("v", v_cache, v_scale)):
        bits[name] = _bits_of(op, f"{name}_cache", cache)
        _expect(op, f"{name}_cache", cache, cache.dtype, (k_cache.size(0), kv_heads, size // 2 if bits[name] == 4 else size))
        _expect(op, f"{name}_scale", scale, torch.uint8, (k_cache.size(0), kv_heads, -(-size // BLOCK)))
    for name, t in weights.items():
        _expect(op, name, t, q.dtype, (size,))
    if not eps >= 0:
        raise RuntimeError(f"{op}: expected eps to be at least 0 but got {eps}")
    lib = L.load()
    with L.device_guard(dev):
        out = torch.empty((tokens, q_heads, size), dtype=q.dtype, device=dev)
        args = L.QuikMxHeads(ctypes.sizeof(L.QuikMxHeads), dt, bits["k"], bits["v"], tokens, q_heads, kv_heads, size, cos.size(1), cos.size(0),
                             k_cache.size(0), L.ptr(q), L.ptr(k), L.ptr(v), q.stride(0), k.stride(0), v.stride(0), L.ptr(cos), L.ptr(sin),
                             L.ptr(positions), L.ptr(slots), L.ptr(q_weight), L.ptr(k_weight), L.ptr(out), L.ptr(k_cache), L.ptr(k_scale),
                             L.ptr(v_cache), L.ptr(v_scale), eps, 0)
        L.check(lib.quik_mx_rotate_to_cache(ctypes.byref(args), L.stream()), op)
    return out
