"""symmetric.rms_norm_quantize where fp32 runs out of range on the way: eps of 0."""
import pytest
import torch

import quik

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]
WIDTHS = [8, 63, 64, 1001, 4096, 16390, 32768, 40001]   # one chunk of eight and its ends, every number of chunks per lane, beyond the registers


def _random(rows, cols, seed):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_rows_of_zeros_without_eps(cols, dtype):
    """Codes 0 and scale 0, whatever eps is; also where the weight makes them so."""
    x, w = _random(3, cols, 1).to(dtype).to(DEV), torch.ones(cols, dtype=dtype, device=DEV)
    r = _random(3, cols, 2).to(dtype).to(DEV)
    r[1], x[1] = 1, -1
    zero = torch.zeros_like(x)
    for eps in (0.0, 1e-60, 1e-5):                     # (1e-60: 0 in fp32)
        q, scale, _ = quik.symmetric.rms_norm_quantize(zero, w, eps)
        assert not q.any() and torch.equal(scale, torch.zeros_like(scale))
        q, scale, _ = quik.symmetric.rms_norm_quantize(x, torch.zeros_like(w), eps)
        assert not q.any() and torch.equal(scale, torch.zeros_like(scale))
        q, scale, h = quik.symmetric.rms_norm_quantize(x, w, eps, residual=r)
        assert not h[1].any() and not q[1].any() and scale[1] == 0
        assert (scale[[0, 2]] > 0).all() and scale.isfinite().all() and q[0].any() and q[2].any()
    x[0, cols - 1] = float("nan")                      # and a row that is no number stays one
    q, scale, _ = quik.symmetric.rms_norm_quantize(x, torch.zeros_like(w), 0.0)
    assert scale[0].isnan() and scale[1] == 0 and not q.any()
