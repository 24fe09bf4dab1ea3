"""Microscaled operators: rows and caches in blocks of 32 numbers that share a power of two, and products of such rows.

A block of 32 neighbouring columns is held as 4-bit (e2m1) or 8-bit (e4m3) floating-point codes and one byte, the exponent of a
power of two, so that a matrix instruction takes both as they are.  A decoder whose linears run in that form makes its rows where
they arise (norm, gated activation, any matrix), multiplies them with 4-bit weights, and keeps keys and values in the same form.
`listed()` names the measured calls, `draw(rng)` gives further ones of the same ranges, `prepare` makes what a program holds
before the call, `run` is the call: the framework's own operators where `own` is true, elementary torch operations elsewhere.

Kinds of call:
  rows    microscaled.quantize and dequantize: a matrix to codes, and back
  norm    microscaled.rms_norm_quantize: root-mean-square norm of x (+ residual) with such rows and one fp32 factor per row
  silu    microscaled.silu_mul_quantize: silu(gate) * up of the two halves of one product
  linear  microscaled.matmul: rows in 4 or 8 bits times 4-bit weights
  mlp     a decoder block's: norm, microscaled.gated_matmul (gate and up, the activation and its codes in one kernel), matmul
  heads   microscaled.rotate_to_cache: norm of each query and key head, rotation by position, keys and values into the cache; then what
          was written is read back
  read    microscaled.dequantize of the cache rows that a list of slots names

Codes are compared as the values that they stand for, in the 16-bit type of the call.
"""
import torch

own = False

EPS = 1e-5
BLOCK = 32
# (in, out) of the 7B, 13B and 70B configurations of this repository
SHAPES = ((4096, 4096), (4096, 11008), (11008, 4096), (5120, 5120), (5120, 13824), (13824, 5120), (8192, 8192), (8192, 10240),
          (8192, 1024), (8192, 28672), (28672, 8192))
# (query heads, key heads, size) of the same, and two generic ones
HEADS = ((32, 32, 128), (40, 40, 128), (64, 8, 128), (16, 2, 80), (12, 4, 64))
_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _rows(rows, cols, bits=4, dtype="float16"):
    return {"kind": "rows", "rows": rows, "cols": cols, "bits": bits, "dtype": dtype}


def _norm(rows, cols, bits=4, dtype="float16", residual=True):
    return {"kind": "norm", "rows": rows, "cols": cols, "bits": bits, "dtype": dtype, "residual": residual}


def _silu(rows, cols, dtype="float16"):
    return {"kind": "silu", "rows": rows, "cols": cols, "dtype": dtype}


def _linear(rows, n_in, out, bits=4, dtype="float16", bias=False):
    return {"kind": "linear", "rows": rows, "in": n_in, "out": out, "bits": bits, "dtype": dtype, "bias": bias}


def _mlp(rows, hidden, inner, bits=4, dtype="float16"):
    return {"kind": "mlp", "rows": rows, "hidden": hidden, "inner": inner, "bits": bits, "dtype": dtype}


def _heads(tokens, q_heads, kv_heads, size, v_bits=8, dtype="float16", norm=False, positions=4096):
    """Keys in 8 bits (a power of two is a coarse scale for 4-bit keys), values in 4 or 8; positions: of the rotation's table."""
    return {"kind": "heads", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "size": size, "v_bits": v_bits, "dtype": dtype,
            "norm": norm, "positions": positions}


def _read(tokens, kv_heads, size, bits=8, dtype="float16"):
    return {"kind": "read", "tokens": tokens, "kv_heads": kv_heads, "size": size, "bits": bits, "dtype": dtype}


def listed():
    return [
        # a prompt's activations in front of a product whose input no norm or activation makes (the attention's output)
        dict(_rows(2048, 8192, 4, "bfloat16"), name="prefill_2048_rows"),
        # a prompt of no particular length: the norm in front of a block's first product
        dict(_norm(777, 5120), name="prompt_777_norm"),
        # the activation between gate/up and down of a prompt, 8 bits where 4 lose too much
        dict(_silu(2048, 13824, "bfloat16"), name="prefill_2048_silu"),
        # single-token products: the smallest projection, and the largest on 8-bit activations
        dict(_linear(1, 4096, 4096), name="decode_1_q"),
        dict(_linear(1, 8192, 28672, bits=8, dtype="bfloat16"), name="decode_1_gate_8"),
        # a prompt at widths that are no multiples of a tile, with a bias
        dict(_linear(300, 4544, 4541, bias=True), name="prompt_300_odd_width"),
        # prefill of the widest projection
        dict(_linear(2048, 8192, 28672, dtype="bfloat16"), name="prefill_2048_gate"),
        # a whole block's MLP: the decode step of a batch of 64, and one token on 8-bit rows
        dict(_mlp(64, 5120, 13824, 4, "bfloat16"), name="decode_64_mlp"),
        dict(_mlp(1, 4096, 11008, 8), name="decode_1_mlp_8"),
        # the decode step of a batch of 64 with normed heads; a prompt with values in 4 bits
        dict(_heads(64, 64, 8, 128, 8, "bfloat16", norm=True, positions=32768), name="decode_64_heads"),
        dict(_heads(4096, 40, 40, 128, 4), name="prefill_4096_heads"),
        # one long sequence's keys or values read back for attention in 16 bits
        dict(_read(32768, 8, 128, 8, "bfloat16"), name="read_32768"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("rows", "norm", "silu", "linear", "linear", "linear", "mlp", "heads", "read"))
    dtype, bits = rng.choice(("float16", "bfloat16")), rng.choice((4, 8))
    if kind in ("rows", "norm", "silu"):
        cols = rng.choice(SHAPES)[rng.randint(0, 1)] if rng.random() < 0.5 else 2 * _log(rng, 32, 14336)
        rows = min(_log(rng, 1, 8192), max(1, 2048 * 8192 // cols))
        return _rows(rows, cols, bits, dtype) if kind == "rows" else _silu(rows, cols, dtype) if kind == "silu" else \
            _norm(rows, cols, bits, dtype, rng.random() < 0.7)
    if kind == "mlp":
        hidden, inner = rng.choice(((4096, 11008), (5120, 13824), (32 * _log(rng, 32, 160), 32 * _log(rng, 64, 432))))
        return _mlp(_log(rng, 1, 64), hidden, inner, bits, dtype)
    if kind in ("heads", "read"):
        q_heads, kv_heads, size = rng.choice(HEADS)
        if kind == "read":
            return _read(_log(rng, 1, 32768 * 8 // max(8, kv_heads)), kv_heads, size, bits, dtype)
        return _heads(_log(rng, 1, 4096), q_heads, kv_heads, size, bits, dtype, rng.random() < 0.5, rng.choice((2048, 4096, 32768)))
    n_in, out = rng.choice(SHAPES) if rng.random() < 0.5 else (32 * _log(rng, 8, 448), _log(rng, 64, 28672))
    rows = min(_log(rng, 1, 2048), max(1, 2048 * 8192 * 28672 // (n_in * out)))
    return _linear(rows, n_in, out, bits, dtype, rng.random() < 0.3)


# -------------------------------------------------------------------------------------------------------- plain forms
def _blocks(v):
    """[..., C] -> [..., C / 32, 32], the last block filled with zeros."""
    pad = -v.shape[-1] % BLOCK
    if pad:
        v = torch.nn.functional.pad(v, (0, pad))
    return v.unflatten(-1, (-1, BLOCK))


def _block_codes(v, bits):
    """fp32 [..., C] -> what the codes stand for within their blocks [..., C / 32, 32] and the blocks' exponents [..., C / 32, 1].
    The exponent is that of the largest magnitude less the format's largest (2 and 8); ties of a code go to the even one."""
    v = _blocks(v)
    top = v.abs().amax(-1, keepdim=True)
    exponent = torch.where(top > 0, torch.frexp(top).exponent - 1 - (2 if bits == 4 else 8), -127).clamp(min=-127)
    t = torch.ldexp(v, -exponent)
    lowest, digits, most = (0, 1, 6.0) if bits == 4 else (-6, 3, 448.0)
    binade = (torch.frexp(t).exponent - 1).clamp(min=lowest) - digits
    return torch.ldexp(torch.round(torch.ldexp(t, -binade)), binade).clamp(-most, most), exponent


def _rounded(v, bits):
    """fp32 numbers -> the numbers that their codes stand for."""
    t, exponent = _block_codes(v, bits)
    return torch.ldexp(t, exponent).flatten(-2)[..., :v.shape[-1]]


def _numbers(q, scale, cols):
    """Codes and exponents -> fp32 numbers."""
    if q.dtype == torch.uint8:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=q.device)
        v = table[torch.stack((q & 15, q >> 4), -1).flatten(-2).long()]
    else:
        v = q.float()
    return torch.ldexp(_blocks(v), scale.unsqueeze(-1).int() - 127).flatten(-2)[..., :cols]


def _normed(x, gain):
    h = x.float()
    return h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * (1 if gain is None else gain.float())


def _plain_norm(s):
    """The rows before their factor are rounded: the factor is the same for a whole row and stays in fp32."""
    x = s["x"] if s["residual"] is None else s["x"] + s["residual"]
    h = x.float()
    return _rounded(h * s["gain"].float(), s["bits"]), torch.rsqrt((h * h).mean(1, keepdim=True) + EPS), x


def _plain_silu(gate, up, bits):
    g = gate.float()
    return _rounded(g / (1 + torch.exp(-g)) * up.float(), bits)


def _plain_linear(x, w, dtype, bias=None):
    y = x @ _numbers(w["q"], w["scale"], x.shape[1]).t()
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_heads(s):
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    q, k = (s["q"], s["k"]) if s["q_gain"] is None else (_normed(s["q"], s["q_gain"]), _normed(s["k"], s["k_gain"]))
    q, k = _rotated(q.float(), cos, sin), _rotated(k.float(), cos, sin)
    keys, values = s["plain_cache"]
    keys[s["slots"]] = _rounded(k, 8).to(s["dtype"])
    values[s["slots"]] = _rounded(s["v"].float(), s["v_bits"]).to(s["dtype"])
    return {"q": q.to(s["dtype"]), "k": keys[s["slots"]], "v": values[s["slots"]]}


def _run_plain(s):
    kind, dtype = s["kind"], s["dtype"]
    if kind == "rows":
        return _rounded(s["x"].float(), s["bits"]).to(dtype)
    if kind == "norm":
        v, factor, h = _plain_norm(s)
        v = (v * factor).to(dtype)
        return {"values": v} if s["residual"] is None else {"values": v, "sum": h}
    if kind == "silu":
        return _plain_silu(s["gate"], s["up"], s["bits"]).to(dtype)
    if kind == "linear":
        return _plain_linear(_numbers(s["xq"], s["x_scale"], s["in"]), s["w"], dtype, s["bias"])
    if kind == "read":
        return _numbers(s["cache"][s["slots"]], s["scale"][s["slots"]], s["size"]).to(dtype)
    if kind == "heads":
        return _plain_heads(s)
    v, factor, h = _plain_norm(s)
    both = _plain_linear(v * factor, s["gate_up"], dtype)
    return {"out": _plain_linear(_plain_silu(*both.chunk(2, 1), s["bits"]), s["down"], dtype), "sum": h}


# ------------------------------------------------------------------------------------------------------------ inputs
def _codes(v, bits):
    """fp32 numbers -> (codes, exponent bytes) as a program holds them."""
    t, exponent = _block_codes(v, bits)
    t = t.flatten(-2)[..., :v.shape[-1]]
    if bits == 8:
        return t.to(torch.float8_e4m3fn).contiguous(), (exponent.squeeze(-1) + 127).to(torch.uint8)
    of = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], device=v.device, dtype=torch.uint8)
    code = of[(t.abs() * 2).long()] | (torch.signbit(t).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), (exponent.squeeze(-1) + 127).to(torch.uint8)


def _weights(gen, n_in, out):
    """Codes of weights around 0.02: the exponents of their blocks lie in a narrow range."""
    return {"q": torch.randint(0, 256, (out, n_in // 2), generator=gen, device="cuda", dtype=torch.uint8),
            "scale": torch.randint(117, 122, (out, n_in // BLOCK), generator=gen, device="cuda", dtype=torch.uint8)}


def _hidden(gen, rows, cols, dtype):
    """A hidden state: N(0, 1), every 128th column ten times as large."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x[:, ::128] *= 10
    return x.to(dtype)


def _gain(gen, n, dtype):
    return (1 + 0.1 * torch.randn(n, generator=gen, device="cuda")).to(dtype)


def _prepare_heads(s, case, gen):
    tokens, hq, hk, size, dtype = case["tokens"], case["q_heads"], case["kv_heads"], case["size"], s["dtype"]
    # one product's columns: queries, keys, values; keys have columns that stand out, as they do in models
    qkv = torch.randn(tokens, (hq + 2 * hk) * size, generator=gen, device="cuda")
    qkv[:, hq * size:(hq + hk) * size:size // 2] *= 6
    qkv = qkv.to(dtype)
    s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, size)) for t in qkv.split((hq * size, hk * size, hk * size), 1))
    s["q_gain"], s["k_gain"] = (_gain(gen, size, dtype), _gain(gen, size, dtype)) if case["norm"] else (None, None)
    s["v_bits"] = case["v_bits"]
    angle = torch.outer(torch.arange(case["positions"], device="cuda", dtype=torch.float64),
                        10000.0 ** (-torch.arange(0, size, 2, device="cuda", dtype=torch.float64) / size))
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["positions"] = torch.randint(0, case["positions"], (tokens,), generator=gen, device="cuda")
    slots = tokens + tokens // 2 + 16
    s["slots"] = torch.randperm(slots, generator=gen, device="cuda")[:tokens]
    if own:
        s["cache"] = [t for bits in (8, case["v_bits"]) for t in
                      (torch.zeros(slots, hk, size // 2, dtype=torch.uint8, device="cuda") if bits == 4 else
                       torch.zeros(slots, hk, size, dtype=torch.float8_e4m3fn, device="cuda"),
                       torch.zeros(slots, hk, -(-size // BLOCK), dtype=torch.uint8, device="cuda"))]
    else:
        s["plain_cache"] = torch.zeros(2, slots, hk, size, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, dtype = case["kind"], case.get("rows"), _TYPES[case["dtype"]]
    s = {"kind": kind, "dtype": dtype, "bits": case.get("bits", 8)}
    if kind == "rows":
        s["x"] = _hidden(gen, rows, case["cols"], dtype)
    if kind in ("norm", "mlp"):
        cols = case["cols"] if kind == "norm" else case["hidden"]
        s["x"] = _hidden(gen, rows, cols, dtype)
        s["residual"] = _hidden(gen, rows, cols, dtype) if case.get("residual", True) else None
        s["gain"] = _gain(gen, cols, dtype)
    if kind == "silu":  # gate and up are column views of one product
        both = torch.randn(rows, 2 * case["cols"], generator=gen, device="cuda").to(dtype)
        s["gate"], s["up"] = both[:, :case["cols"]], both[:, case["cols"]:]
    if kind == "linear":
        s["in"] = case["in"]
        s["xq"], s["x_scale"] = _codes(_hidden(gen, rows, case["in"], torch.float32), case["bits"])
        s["w"] = _weights(gen, case["in"], case["out"])
        s["bias"] = torch.randn(case["out"], generator=gen, device="cuda").to(dtype) if case["bias"] else None
    if kind == "mlp":
        s["gate_up"], s["down"] = _weights(gen, case["hidden"], 2 * case["inner"]), _weights(gen, case["inner"], case["hidden"])
    if kind == "heads":
        _prepare_heads(s, case, gen)
    if kind == "read":
        slots = case["tokens"] + case["tokens"] // 2 + 16
        s["cache"], s["scale"] = _codes(torch.randn(slots, case["kv_heads"], case["size"], generator=gen, device="cuda"), case["bits"])
        s["slots"], s["size"] = torch.randperm(slots, generator=gen, device="cuda")[:case["tokens"]], case["size"]
    return s


# --------------------------------------------------------------------------------------------------- the framework's
def _own_heads(ms, s):
    keys, key_scale, values, value_scale = s["cache"]
    q = ms.rotate_to_cache(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], keys, key_scale, values, value_scale,
                           q_weight=s["q_gain"], k_weight=s["k_gain"], eps=EPS)
    return {"q": q, "k": ms.dequantize(keys, key_scale, s["dtype"], rows=s["slots"]),
            "v": ms.dequantize(values, value_scale, s["dtype"], rows=s["slots"])}


def _run_own(s):
    from quik import microscaled as ms
    kind, dtype = s["kind"], s["dtype"]
    if kind == "rows":
        return ms.dequantize(*ms.quantize(s["x"], s["bits"]), dtype)
    if kind == "silu":
        return ms.dequantize(*ms.silu_mul_quantize(s["gate"], s["up"], s["bits"]), dtype)
    if kind == "linear":
        return ms.matmul(s["xq"], s["x_scale"], s["w"]["q"], s["w"]["scale"], dtype, bias=s["bias"])
    if kind == "read":
        return ms.dequantize(s["cache"], s["scale"], dtype, rows=s["slots"])
    if kind == "heads":
        return _own_heads(ms, s)
    q, scale, factor, h = ms.rms_norm_quantize(s["x"], s["gain"], EPS, residual=s["residual"], bits=s["bits"])
    if kind == "norm":
        v = ms.dequantize(q, scale, dtype, scale_row=factor)
        return {"values": v} if h is None else {"values": v, "sum": h}
    q, scale = ms.gated_matmul(q, scale, s["gate_up"]["q"], s["gate_up"]["scale"], dtype, scale_row=factor, bits=s["bits"])
    return {"out": ms.matmul(q, scale, s["down"]["q"], s["down"]["scale"], dtype), "sum": h}


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ----------------------------------------------------------------------------------------------------------- in 64 bits
def _grid(bits):
    """The numbers of a format that are not negative, by code."""
    if bits == 4:
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]


def _nearest(v, bits):
    """float64 numbers -> the nearest numbers of the format within blocks of 32, of two the one with the even code."""
    grid = torch.tensor(_grid(bits), dtype=torch.float64, device=v.device)
    border = (grid[1:] + grid[:-1]) / 2
    out = torch.empty_like(v)
    for c in range(0, v.shape[-1], BLOCK):
        part = v[..., c:c + BLOCK]
        top = part.abs().max(-1, keepdim=True).values
        power = torch.floor(torch.log2(top.clamp(min=1e-300)))
        power = torch.where(torch.exp2(power) > top, power - 1, torch.where(torch.exp2(power + 1) <= top, power + 1, power))
        unit = torch.exp2((power - (2 if bits == 4 else 8)).clamp(min=-127))
        t = (part.abs() / unit).contiguous()
        code = torch.searchsorted(border, t)
        code = torch.where((code < border.numel()) & (t == border[code.clamp(max=border.numel() - 1)]) & (code % 2 == 1), code + 1, code)
        out[..., c:c + BLOCK] = torch.where(part < 0, -grid[code], grid[code]) * unit
    return out


def _exact_numbers(q, scale):
    if q.dtype == torch.uint8:
        byte = q.to(torch.int64)
        code = torch.empty(*q.shape[:-1], 2 * q.shape[-1], dtype=torch.int64, device=q.device)
        code[..., 0::2], code[..., 1::2] = byte % 16, byte // 16
        bits, negative, code = 4, code >= 8, code % 8
    else:
        code = q.view(torch.uint8).to(torch.int64)
        bits, negative, code = 8, code >= 128, code % 128
    v = torch.tensor(_grid(bits) + [float("nan")], dtype=torch.float64, device=q.device)[code]
    unit = torch.exp2(scale.double() - 127).repeat_interleave(BLOCK, -1)[..., :v.shape[-1]]
    return torch.where(negative, -v, v) * unit


def _exact_norm(s):
    h = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["dtype"])
    d = h.double()
    return _nearest(d * s["gain"].double(), s["bits"]) / torch.sqrt(d.pow(2).mean(1, keepdim=True) + EPS), h


def _exact_silu(g, u, bits):
    return _nearest(g * torch.sigmoid(g) * u, bits)


def _exact_turned(x, gain, cos, sin):
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * gain.double()
    z = torch.complex(x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]) * torch.complex(cos.double(), sin.double()).unsqueeze(1)
    return torch.cat((z.real, z.imag), -1)


def exact(case, seed):
    s = prepare(case, seed)
    kind, dtype = case["kind"], s["dtype"]
    if kind == "rows":
        return _nearest(s["x"].double(), s["bits"])
    if kind == "silu":
        return _exact_silu(s["gate"].double(), s["up"].double(), s["bits"])
    if kind == "linear":
        y = _exact_numbers(s["xq"], s["x_scale"]) @ _exact_numbers(s["w"]["q"], s["w"]["scale"]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    if kind == "read":
        return _exact_numbers(s["cache"][s["slots"]], s["scale"][s["slots"]])
    if kind == "heads":
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return {"q": _exact_turned(s["q"], s["q_gain"], cos, sin), "k": _nearest(_exact_turned(s["k"], s["k_gain"], cos, sin), 8),
                "v": _nearest(s["v"].double(), s["v_bits"])}
    v, h = _exact_norm(s)
    if kind == "norm":
        return {"values": v} if s["residual"] is None else {"values": v, "sum": h}
    both = (v @ _exact_numbers(s["gate_up"]["q"], s["gate_up"]["scale"]).t()).to(dtype).double()  # gate and up are held in 16 bits
    inner = both.shape[1] // 2
    return {"out": _exact_silu(both[:, :inner], both[:, inner:], s["bits"]) @ _exact_numbers(s["down"]["q"], s["down"]["scale"]).t(), "sum": h}


# ------------------------------------------------------------------------------------------------------------- work
def _held(n, bits):
    """Bytes of n numbers in blocks."""
    return n * bits // 8 + n // BLOCK


def work(case):
    kind, bits = case["kind"], case.get("bits", 8)
    if kind in ("rows", "norm", "silu"):  # the call's codes are written, and read for the values that they stand for
        n = case["rows"] * case["cols"]
        read = {"rows": 2, "silu": 4, "norm": 6 if case.get("residual") else 2}[kind]
        return {"bytes": n * (read + 2) + 2 * _held(n, bits), "flops": 8 * n}
    if kind == "linear":
        rows, n_in, out = case["rows"], case["in"], case["out"]
        return {"bytes": _held(out * n_in, 4) + _held(rows * n_in, bits) + 2 * rows * out, "flops": 2 * rows * n_in * out}
    if kind == "mlp":
        rows, hidden, inner = case["rows"], case["hidden"], case["inner"]
        return {"bytes": _held(3 * hidden * inner, 4) + 8 * rows * hidden, "flops": 6 * rows * hidden * inner}
    n = case["tokens"] * case["kv_heads"] * case["size"]
    if kind == "read":
        return {"bytes": _held(n, bits) + 2 * n, "flops": n}
    nq = case["tokens"] * case["q_heads"] * case["size"]
    return {"bytes": 4 * nq + 4 * n + 2 * (_held(n, 8) + _held(n, case["v_bits"])) + 4 * n + 4 * case["tokens"] * case["size"],
            "flops": 12 * (nq + 2 * n)}
