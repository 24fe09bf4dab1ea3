"""matmul.int4GroupMatmul where rows and columns are more than one launch holds."""
import pytest
import torch

import quik

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_more_rows_than_one_launch():
    """2^28 rows and some in tiles of 64 rows: the last ones are a launch of their own.  Sums of 32 products of 16-bit whole numbers, scales of
    powers of two: exact but for the rounding of the result."""
    rows, last = (1 << 28) + 70, 300
    g = torch.Generator().manual_seed(0)
    x = torch.zeros(rows, 32, dtype=torch.int8, device=DEV)
    x[-last:] = torch.randint(-128, 128, (last, 32), generator=g, dtype=torch.int8).to(DEV)
    scale = torch.ones(rows, 1, device=DEV)
    scale[-last:] = 2.0 ** -torch.randint(0, 4, (last, 1), generator=g).float().to(DEV)
    w = torch.randint(0, 256, (1, 16), generator=g, dtype=torch.uint8).to(DEV)
    out = quik.matmul.int4GroupMatmul(x, w, torch.full((1, 1), 0.125, dtype=torch.float16, device=DEV), 32, scale_row=scale)
    q = torch.stack((((w & 15) ^ 8).to(torch.int8) - 8, ((w >> 4) ^ 8).to(torch.int8) - 8), 2).flatten(1)
    want = (x[-last:].double() @ q.double().t() * scale[-last:].double() * 0.125).half()
    assert torch.equal(out[-last:], want) and want.any()
    assert not out[:-last].any()
