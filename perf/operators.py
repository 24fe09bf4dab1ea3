"""The operators around 8-bit activations and 4-bit weights with group scales, with their inputs and plain forms.

A decoder whose linears take 8-bit activations and weights of 4 bits runs, per block: the norm that adds the residual and
gives codes, the product of codes and grouped weights, the gated activation that gives codes again, and the next product.
`listed()` names the measured calls, `draw(rng)` gives further ones of the same ranges, `prepare` makes what a program holds
before the call, `run` is the call: the framework's own operators where `own` is true, elementary torch operations elsewhere.

Kinds of call:
  norm    symmetric.rms_norm_quantize: root-mean-square norm of x (+ residual), int8 codes and one scale per row
  silu    symmetric.silu_mul_quantize: silu(gate) * up of the two halves of one product, int8 codes and one scale per row
  linear  matmul.int4GroupMatmul: 16-bit or int8 activations times 4-bit weights with one scale (and zero) per group of a row
  mlp     the four of them as a decoder block calls them: norm, gate and up in one product, activation, down

Codes are compared as the values that they stand for (code * scale, in the 16-bit type of the call).
"""
import torch

own = False

EPS = 1e-5
# (in, out) of the 7B, 13B and 70B configurations of this repository
SHAPES = ((4096, 4096), (4096, 11008), (11008, 4096), (5120, 5120), (5120, 13824), (13824, 5120), (8192, 8192), (8192, 10240),
          (8192, 1024), (8192, 28672), (28672, 8192))
_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _norm(rows, cols, dtype="float16", residual=True):
    return {"kind": "norm", "rows": rows, "cols": cols, "dtype": dtype, "residual": residual}


def _silu(rows, cols, dtype="float16"):
    return {"kind": "silu", "rows": rows, "cols": cols, "dtype": dtype}


def _linear(rows, n_in, out, group=128, acts="float16", dtype="float16", zeros=False, bias=False):
    """acts: the activations' type (int8: codes with a scale per row); dtype: of scales, zeros, bias and the result."""
    return {"kind": "linear", "rows": rows, "in": n_in, "out": out, "group": group, "acts": acts, "dtype": dtype, "zeros": zeros,
            "bias": bias}


def _mlp(rows, hidden, inner, dtype="float16"):
    return {"kind": "mlp", "rows": rows, "hidden": hidden, "inner": inner, "dtype": dtype}


def listed():
    return [
        # one sequence, token by token: the norm in front of a block's first product
        dict(_norm(1, 4096), name="decode_1_norm"),
        # a prompt's rows, the widest hidden size; the first norm of a model, which has no residual yet, at an odd row count
        dict(_norm(4096, 8192, "bfloat16"), name="prefill_4096_norm"),
        dict(_norm(777, 5120, "float16", residual=False), name="prompt_777_norm_first"),
        # the activation between gate/up and down: a batch of 64 sequences, and a prompt
        dict(_silu(64, 13824), name="decode_64_silu"),
        dict(_silu(2048, 28672, "bfloat16"), name="prefill_2048_silu"),
        # single-token products, weights only in 4 bits: the smallest projection, and the largest with zero points
        dict(_linear(1, 4096, 4096), name="decode_1_q"),
        dict(_linear(1, 8192, 28672, acts="bfloat16", dtype="bfloat16", zeros=True), name="decode_1_gate_zeros"),
        # a few sequences together on 8-bit activations, the projection with long rows
        dict(_linear(16, 13824, 5120, acts="int8"), name="decode_16_down_int8"),
        # a prompt of no particular length at widths that are no multiples of a tile, groups of 64 with zero points, a bias
        dict(_linear(300, 4544, 4541, group=64, zeros=True, bias=True), name="prompt_300_odd_width"),
        # prefill on 8-bit activations
        dict(_linear(2048, 4096, 11008, acts="int8", dtype="bfloat16"), name="prefill_2048_gate_int8"),
        # a whole block's MLP: one token, and the decode step of a batch of 64
        dict(_mlp(1, 4096, 11008), name="decode_1_mlp"),
        dict(_mlp(64, 5120, 13824, "bfloat16"), name="decode_64_mlp"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("norm", "silu", "linear", "linear", "linear", "mlp"))
    dtype = rng.choice(("float16", "bfloat16"))
    if kind in ("norm", "silu"):
        cols = rng.choice(SHAPES)[rng.randint(0, 1)] if rng.random() < 0.5 else _log(rng, 64, 28672)
        rows = min(_log(rng, 1, 8192), max(1, 4096 * 8192 // cols))
        return _norm(rows, cols, dtype, rng.random() < 0.7) if kind == "norm" else _silu(rows, cols, dtype)
    if kind == "mlp":
        hidden, inner = rng.choice(((4096, 11008), (5120, 13824), (32 * _log(rng, 32, 160), 32 * _log(rng, 64, 432))))
        return _mlp(_log(rng, 1, 64), hidden, inner, dtype)
    n_in, out = rng.choice(SHAPES) if rng.random() < 0.5 else (32 * _log(rng, 8, 448), _log(rng, 64, 28672))
    rows = min(_log(rng, 1, 2048), max(1, 2048 * 4096 * 11008 // (n_in * out)))
    return _linear(rows, n_in, out, rng.choice((32, 64, 128, 128, 128, 256)), rng.choice((dtype, "int8")), dtype,
                   rng.random() < 0.4, rng.random() < 0.3)


# ------------------------------------------------------------------------------------------------------------ inputs
def _weights(gen, n_in, out, group, dtype, zeros):
    groups = -(-n_in // group)
    w = {"weight": torch.randint(0, 256, (out, n_in // 2), generator=gen, device="cuda", dtype=torch.uint8),
         "scales": (torch.rand(out, groups, generator=gen, device="cuda") * 0.009 + 0.001).to(dtype),
         "zeros": None, "group": group}
    if zeros:  # where a group's value 0 lies among its codes -8 .. 7
        w["zeros"] = torch.randint(-4, 4, (out, groups), generator=gen, device="cuda").to(dtype)
    return w


def _hidden(gen, rows, cols, dtype):
    """A hidden state: N(0, 1), every 128th column ten times as large."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x[:, ::128] *= 10
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, dtype = case["kind"], case["rows"], _TYPES[case["dtype"]]
    s = {"kind": kind, "dtype": dtype}
    if kind == "norm" or kind == "mlp":
        cols = case["cols"] if kind == "norm" else case["hidden"]
        s["x"] = _hidden(gen, rows, cols, dtype)
        s["residual"] = _hidden(gen, rows, cols, dtype) if case.get("residual", True) else None
        s["gain"] = (1 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(dtype)
    if kind == "silu":  # gate and up are column views of one product
        both = torch.randn(rows, 2 * case["cols"], generator=gen, device="cuda").to(dtype)
        s["gate"], s["up"] = both[:, :case["cols"]], both[:, case["cols"]:]
    if kind == "linear":
        s["w"] = _weights(gen, case["in"], case["out"], case["group"], dtype, case["zeros"])
        s["scale_row"] = s["bias"] = None
        if case["acts"] == "int8":
            s["x"] = torch.randint(-127, 128, (rows, case["in"]), generator=gen, device="cuda", dtype=torch.int8)
            s["scale_row"] = torch.rand(rows, 1, generator=gen, device="cuda") * 0.02 + 0.01
        else:
            s["x"] = _hidden(gen, rows, case["in"], dtype)
        if case["bias"]:
            s["bias"] = torch.randn(case["out"], generator=gen, device="cuda").to(dtype)
    if kind == "mlp":
        s["gate_up"] = _weights(gen, case["hidden"], 2 * case["inner"], 128, dtype, False)
        s["down"] = _weights(gen, case["inner"], case["hidden"], 128, dtype, False)
    return s


# -------------------------------------------------------------------------------------------------------- plain forms
def _codes(v):
    """Rows of numbers -> int8 codes round(127 v / max |v|) and the largest magnitudes; a row of zeros has codes 0."""
    top = v.abs().amax(1, keepdim=True)
    q = torch.round(v * torch.where(top > 0, 127 / top, torch.zeros_like(top)))
    return q, top / 127


def _plain_norm(s):
    x = s["x"] if s["residual"] is None else s["x"] + s["residual"]
    h = x.float()
    q, step = _codes(h * s["gain"].float())
    return q, step * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS), x


def _plain_silu(gate, up):
    g = gate.float()
    return _codes(g / (1 + torch.exp(-g)) * up.float())


def _plain_linear(x, w, dtype, scale_row=None, bias=None):
    q = torch.stack((w["weight"] & 15, w["weight"] >> 4), 2).flatten(1)
    q = ((q ^ 8).to(torch.int8) - 8).float()
    at = torch.arange(q.shape[1], device=q.device) // w["group"]
    if w["zeros"] is not None:
        q = q - w["zeros"].float()[:, at]
    y = x.float() @ (q * w["scales"].float()[:, at]).t()
    if scale_row is not None:
        y = y * scale_row
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def _run_plain(s):
    kind, dtype = s["kind"], s["dtype"]
    if kind == "norm":
        q, scale, h = _plain_norm(s)
        return {"values": (q * scale).to(dtype)} if s["residual"] is None else {"values": (q * scale).to(dtype), "sum": h}
    if kind == "silu":
        q, scale = _plain_silu(s["gate"], s["up"])
        return (q * scale).to(dtype)
    if kind == "linear":
        return _plain_linear(s["x"], s["w"], dtype, s["scale_row"], s["bias"])
    q, scale, h = _plain_norm(s)
    both = _plain_linear(q, s["gate_up"], dtype, scale)
    inner = both.shape[1] // 2
    q, scale = _plain_silu(both[:, :inner], both[:, inner:])
    return {"out": _plain_linear(q, s["down"], dtype, scale), "sum": h}


# --------------------------------------------------------------------------------------------------- the framework's
def _values(q, scale, dtype):
    """What the codes stand for, in one pass over them."""
    return torch.mul(q, scale, out=torch.empty(q.shape, dtype=dtype, device=q.device))


def _own_linear(quik, x, w, scale_row=None, bias=None):
    return quik.matmul.int4GroupMatmul(x, w["weight"], w["scales"], w["group"], zeros=w["zeros"], scale_row=scale_row, bias=bias)


def _run_own(s):
    import quik
    kind, dtype = s["kind"], s["dtype"]
    if kind == "linear":
        return _own_linear(quik, s["x"], s["w"], s["scale_row"], s["bias"])
    if kind == "silu":
        return _values(*quik.symmetric.silu_mul_quantize(s["gate"], s["up"]), dtype)
    q, scale, h = quik.symmetric.rms_norm_quantize(s["x"], s["gain"], EPS, residual=s["residual"])
    if kind == "norm":
        return {"values": _values(q, scale, dtype)} if h is None else {"values": _values(q, scale, dtype), "sum": h}
    both = _own_linear(quik, q, s["gate_up"], scale)
    inner = both.shape[1] // 2
    q, scale = quik.symmetric.silu_mul_quantize(both[:, :inner], both[:, inner:])
    return {"out": _own_linear(quik, q, s["down"], scale), "sum": h}


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ----------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_rows(v):
    """The quantized values of rows of numbers: multiples of max |v| / 127."""
    step = v.abs().max(1, keepdim=True).values / 127
    return torch.where(step > 0, torch.round(v / step) * step, 0.0)


def _exact_matrix(w):
    """The dequantized weights [out, in], column pair by column pair from the bytes."""
    byte = w["weight"].to(torch.int64)
    m = torch.empty(byte.shape[0], 2 * byte.shape[1], dtype=torch.float64, device=byte.device)
    m[:, 0::2] = (byte % 16 + 8) % 16 - 8
    m[:, 1::2] = (byte // 16 + 8) % 16 - 8
    for g in range(w["scales"].shape[1]):
        part = m[:, g * w["group"]:(g + 1) * w["group"]]
        if w["zeros"] is not None:
            part -= w["zeros"][:, g:g + 1].double()
        part *= w["scales"][:, g:g + 1].double()
    return m


def _exact_normed(x, gain):
    h = x.double()
    return h / torch.sqrt(h.pow(2).mean(1, keepdim=True) + EPS) * gain.double()


def _exact_gated(g, u):
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "silu":
        return _exact_rows(_exact_gated(s["gate"].double(), s["up"].double()))
    if kind == "linear":
        x = s["x"].double() if s["scale_row"] is None else s["x"].double() * s["scale_row"].double()
        y = x @ _exact_matrix(s["w"]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    # the sum is held in the type of its parts: it is the next block's residual, and the norm is of what is held
    h = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["dtype"])
    v = _exact_rows(_exact_normed(h, s["gain"]))
    if kind == "norm":
        return {"values": v} if s["residual"] is None else {"values": v, "sum": h}
    both = (v @ _exact_matrix(s["gate_up"]).t()).to(s["dtype"]).double()  # gate and up are held in 16 bits too
    inner = both.shape[1] // 2
    return {"out": _exact_rows(_exact_gated(both[:, :inner], both[:, inner:])) @ _exact_matrix(s["down"]).t(), "sum": h}


# ------------------------------------------------------------------------------------------------------------- work
def _linear_work(rows, n_in, out, group, acts, zeros, bias=False):
    groups = -(-n_in // group)
    moved = out * n_in // 2 + out * groups * (4 if zeros else 2) + rows * n_in * acts + rows * out * 2 + (out * 2 if bias else 0)
    return moved, 2 * rows * n_in * out


def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "norm":
        n = rows * case["cols"]
        return {"bytes": n * (7 if case["residual"] else 3) + 2 * case["cols"] + 4 * rows, "flops": 6 * n}
    if kind == "silu":
        n = rows * case["cols"]
        return {"bytes": 5 * n + 4 * rows, "flops": 8 * n}
    if kind == "linear":
        b, f = _linear_work(rows, case["in"], case["out"], case["group"], 1 if case["acts"] == "int8" else 2, case["zeros"], case["bias"])
        return {"bytes": b + (4 * rows if case["acts"] == "int8" else 0), "flops": f}
    hidden, inner = case["hidden"], case["inner"]
    up, down = _linear_work(rows, hidden, 2 * inner, 128, 0, False), _linear_work(rows, inner, hidden, 128, 0, False)
    return {"bytes": up[0] - rows * 4 * inner + down[0] + rows * hidden * 6 + 2 * hidden, "flops": up[1] + down[1]}
