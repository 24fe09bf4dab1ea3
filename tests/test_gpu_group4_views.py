"""qlinear.GroupLinear4bit on activations that are views: at any start and stride."""
import pytest
import torch

from quik_amd.qlinear import GroupLinear4bit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("rows", [1, 16, 40])
def test_activations_at_any_start(rows, codes, dtype):
    """The result is that of a copy of the view, bit for bit."""
    torch.manual_seed(rows)
    mod = GroupLinear4bit.from_float(torch.nn.Linear(96, 40, dtype=dtype, device=DEV), 32, False)
    scale = torch.rand(rows, 1, device=DEV) if codes else None

    def numbers(*shape):
        return torch.randint(-127, 128, shape, device=DEV, dtype=torch.int8) if codes else torch.randn(*shape, device=DEV).to(dtype)

    whole = numbers(rows * 96 + 64)
    for start in (0, 1, 3, 8, 16, 33):
        x = whole[start:start + rows * 96].view(rows, 96)      # contiguous, from any element on
        assert x.is_contiguous()
        assert torch.equal(mod(x, scale), mod(x.clone(), scale))
    x = numbers(rows, 200)[:, 5:101]                           # rows apart
    assert torch.equal(mod(x, scale), mod(x.clone(memory_format=torch.contiguous_format), scale))
    x = numbers(96, rows).t()
    assert torch.equal(mod(x, scale), mod(x.clone(memory_format=torch.contiguous_format), scale))
