"""MicroscaledLinear4bit: which types it has, takes and gives, and what it is made of."""
import pytest
import torch

import mx_plain as P
from quik_amd.qlinear import MicroscaledLinear4bit

DEV = "cuda:0"


def ms():
    from quik import microscaled
    return microscaled


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.int8])
def test_results_of_other_types_are_refused(dtype):
    with pytest.raises(ValueError, match="dtype must be"):
        MicroscaledLinear4bit(64, 32, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
def test_a_module_that_is_cast_to_32_bits_keeps_its_type(bias, dtype):
    mod = MicroscaledLinear4bit(64, 32, bias=bias, dtype=dtype)
    if bias:
        mod.bias.copy_(torch.arange(32) / 8)
    mod.weight.fill_(0x12)
    outer = torch.nn.Sequential(mod, torch.nn.Linear(32, 2)).float().double()
    assert mod.dtype == dtype and outer[1].weight.dtype == torch.float64
    assert mod.weight.dtype == mod.weight_scale.dtype == torch.uint8 and (mod.weight == 0x12).all()
    if bias:
        assert mod.bias.dtype == dtype and torch.equal(mod.bias, (torch.arange(32) / 8).to(dtype)) and "bias" in mod.state_dict()
    assert mod.to(torch.bfloat16).dtype == torch.bfloat16 and mod.half().dtype == torch.float16 and (not bias or mod.bias.dtype == torch.float16)


@pytest.mark.gpu
def test_a_module_that_was_cast_to_32_bits_runs():
    lin = torch.nn.Linear(64, 32, dtype=torch.bfloat16, device=DEV)
    mod, x = MicroscaledLinear4bit.from_float(lin), torch.randn(3, 64, device=DEV).bfloat16()
    want = mod(x)
    assert torch.equal(mod.float()(x), want) and want.dtype == torch.bfloat16


def test_activations_of_a_wider_range_than_the_results_are_refused():
    """A module of fp16 would turn results of bf16 activations into infinities; one of bf16 holds those of fp16."""
    mod = MicroscaledLinear4bit(64, 64)
    for call in (mod, mod.gated):
        with pytest.raises(ValueError, match="bfloat16"):
            call(torch.zeros(2, 64, dtype=torch.bfloat16))
        with pytest.raises(RuntimeError, match="float16 or bfloat16|CUDA"):
            call(torch.zeros(2, 64))


@pytest.mark.gpu
def test_activations_of_either_type():
    lin = torch.nn.Linear(64, 32, dtype=torch.float16, device=DEV)
    mod, x = MicroscaledLinear4bit.from_float(lin), torch.randn(3, 64, device=DEV).half()
    with pytest.raises(ValueError, match="bfloat16"):
        mod(x.bfloat16() * 2.0 ** 20)
    assert mod(x).dtype == torch.float16
    q, s = ms().quantize(x.bfloat16() * 2.0 ** 20)           # rows of codes have no type: what does not fit is the caller's
    assert mod(q, s).dtype == torch.float16
    assert mod.to(torch.bfloat16)(x.bfloat16() * 2.0 ** 20).isfinite().all() and mod(x).dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_a_weight_whose_columns_lie_apart(dtype):
    """Another matrix' transpose (tied weights), and every other row of one."""
    lin, w = torch.nn.Linear(96, 64, dtype=dtype, device=DEV), torch.randn(96, 64, dtype=dtype, device=DEV)
    for weight in (w.t(), torch.randn(128, 96, dtype=dtype, device=DEV)[::2]):
        lin.weight = torch.nn.Parameter(weight)
        mod = MicroscaledLinear4bit.from_float(lin)
        kind = torch.float16 if dtype == torch.float32 else dtype
        c, e = P.codes(weight.to(kind).double().cpu(), 4)
        assert torch.equal(P.unpack(mod.weight.cpu()), c) and torch.equal(mod.weight_scale.cpu().to(torch.int64), e)


def test_numbers_beyond_the_range_of_the_type_are_refused():
    for name in ("weight", "bias"):
        lin = torch.nn.Linear(64, 32)
        getattr(lin, name).data.view(-1)[5] = -7e4
        with pytest.raises(ValueError, match=f"{name} has numbers beyond"):
            MicroscaledLinear4bit.from_float(lin)


@pytest.mark.gpu
def test_the_largest_numbers_of_the_type_and_none_at_all():
    lin = torch.nn.Linear(64, 4, device=DEV)
    lin.weight.data[0, 3], lin.bias.data[1] = 65504.0, -65519.0      # (which rounds to fp16's last)
    lin.weight.data[2, 40] = float("inf")                            # an infinity of the module's own: its block has no numbers
    mod = MicroscaledLinear4bit.from_float(lin)
    assert mod.bias[1] == -65504 and torch.equal(mod.weight_scale == 255, torch.tensor([[0, 0], [0, 0], [0, 1], [0, 0]], device=DEV) == 1)
    lin = torch.nn.Linear(64, 4, device=DEV, dtype=torch.bfloat16)
    lin.weight.data[0, 3] = 1e30
    assert (MicroscaledLinear4bit.from_float(lin).weight_scale != 255).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act_bits", [4, 8])
def test_rows_of_codes_of_any_layout(act_bits):
    """Codes that start between 16-byte borders, and codes, bytes and factors whose rows lie apart, are copied as activations are."""
    lin = torch.nn.Linear(96, 64, bias=False, dtype=torch.float16, device=DEV)
    mod, x, gain = MicroscaledLinear4bit.from_float(lin, act_bits), torch.randn(10, 96, device=DEV).half(), torch.ones(96, device=DEV).half()
    q, s, row, _ = ms().rms_norm_quantize(x, gain, bits=act_bits)
    raw = q.view(torch.uint8)
    moved = torch.cat((raw.new_zeros(8), raw.flatten()))[8:].view(raw.shape).view(q.dtype)
    assert moved.data_ptr() % 16 and moved.is_contiguous()
    wide = torch.cat((raw, raw), 1)[:, raw.shape[1]:].view(q.dtype)
    assert not wide.is_contiguous()
    for call in (mod, lambda *a: torch.cat([t.view(torch.uint8) for t in mod.gated(*a)], 1)):
        want = call(q, s, row)
        assert torch.equal(call(moved, s, row), want)
        assert torch.equal(call(wide, torch.cat((s, s), 1)[:, s.shape[1]:], torch.cat((row, row), 1)[:, 1:]), want)
        assert torch.equal(call(q[::2], s[::2], row[::2]), want[::2])
        assert torch.equal(call(q[1:], s[1:], row[1:]), want[1:])
