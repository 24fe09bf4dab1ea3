"""matmul.int4GroupMatmul in every tile that its rules choose among, against its formula in 64 bits on the same GPU.

Tolerance of one value: half a step of the result's type, and the roundings of the sums: products are exact, and a result goes through at
most `32 + K / 32 + 24` additions one after the other in fp32 (a matrix instruction's own, those of the blocks, of the waves and of K's
parts), each 2^-24 of sum |x| (|q| + c + |z|) s, with c what the widened codes carry: 136 (bf16), 8 (fp16 with up to 16 rows), 0 (int8, whose
blocks are summed exactly)."""
import pytest
import torch

import quik
from quik_amd import _lib as L

DEV = "cuda:0"
ACTS = [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.int8, torch.float16), (torch.int8, torch.bfloat16)]
NAMES = ["fp16", "bf16", "int8_fp16", "int8_bf16"]


def make(M, N, K, G, acts, dtype, zeros, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + M + N + K + G)
    rand = lambda *shape: torch.rand(*shape, generator=g, device=DEV)
    groups = -(-K // G)
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device=DEV)
    s = (rand(N, groups) * 0.009 + 0.001).to(dtype)
    z = (rand(N, groups) * 16 - 8).to(dtype) if zeros else None
    if acts == torch.int8:
        return torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device=DEV), w, s, z, rand(M, 1) * 0.02 + 0.01
    x = torch.randn(M, K, generator=g, device=DEV)
    x[:, ::128] *= 10
    return x.to(acts), w, s, z, None


class Oracle:
    """The weights in 64 bits, once for several calls."""

    def __init__(self, w, s, z, G, acts):
        q = torch.stack((((w & 15) ^ 8).to(torch.int8) - 8, ((w >> 4) ^ 8).to(torch.int8) - 8), 2).flatten(1).double()
        at = torch.arange(q.shape[1], device=DEV) // G
        scale, zero = s.double()[:, at], 0.0 if z is None else z.double()[:, at]
        extra = {torch.bfloat16: 136, torch.float16: 8, torch.int8: 0}[acts]
        self.weight = ((q - zero) * scale).t().contiguous()
        self.size = ((q.abs() + extra + (0 if z is None else zero.abs())) * scale).t().contiguous()

    def check(self, out, x, sr):
        y, size = x.double() @ self.weight, x.double().abs() @ self.size
        if sr is not None:
            y, size = y * sr.double(), size * sr.double()
        half = torch.finfo(out.dtype).eps / 2
        adds = 32 + x.shape[1] / 32 + 24
        off = (out.double() - y).abs_()
        assert out.shape == y.shape and bool((off <= half * y.abs() + adds * 2.0 ** -24 * (size + y.abs())).all())
        assert off.norm() <= half * y.norm()


def call(x, w, s, z, sr, G):
    return quik.matmul.int4GroupMatmul(x, w, s, G, zeros=z, scale_row=sr)


def tile_of(acts, dtype, zeros, M, N, K):
    lib, bits, dt = L.load(), 8 if acts == torch.int8 else 16, L.QUIK_BF16 if dtype == torch.bfloat16 else L.QUIK_F16
    t = lib.quik_int4_group_matmul_tile(bits, dt, int(zeros), M, N, K, lib.quik_int4_group_matmul_workspace_bytes(bits, dt, M, N, K))
    return t >> 16, t & 0xFFFF


# ------------------------------------------------------------------------------------------------- up to 16 rows
# Odd column counts from one column per workgroup to several tiles for each (at most two of them run on a CU at a time); nine blocks of K for the
# eight waves, the last one a part of a block
FEW_ROWS, FEW_COLUMNS, FEW_K = (1, 4, 7, 9, 16), (211, 4101, 8189, 11003, 28669, 57341), 1120


def _few(acts, dtype, zeros):
    for N in FEW_COLUMNS:
        for M in FEW_ROWS:
            rows, width = tile_of(acts, dtype, zeros, M, N, FEW_K)
            yield rows, 1 if width <= 16 else 2 if width <= 32 else 4, -(-N // width) > 512


@pytest.mark.parametrize("acts,dtype", ACTS, ids=NAMES)
@pytest.mark.parametrize("zeros", [False, True])
def test_the_calls_of_few_rows_reach_every_kernel(zeros, acts, dtype):
    """Each row count with one, two and (16 rows) four matrix tiles, and with more tiles than there are workgroups at a time."""
    seen = set(_few(acts, dtype, zeros))
    assert {(r, f) for r, f, _ in seen} == {(4, 1), (4, 2), (8, 1), (8, 2), (16, 1), (16, 2), (16, 4)}
    assert {r for r, _, more in seen if more} == {4, 8, 16} and (16, 4, True) in seen and {f for _, f, more in seen if more} >= {2, 4}


@pytest.mark.gpu
@pytest.mark.parametrize("acts,dtype", ACTS, ids=NAMES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("G", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("N", FEW_COLUMNS)
def test_few_rows(N, G, zeros, acts, dtype):
    x, w, s, z, sr = make(16, N, FEW_K, G, acts, dtype, zeros)
    oracle = Oracle(w, s, z, G, acts)
    for M in FEW_ROWS:
        xx, ss = x[16 - M:], None if sr is None else sr[16 - M:]
        oracle.check(call(xx, w, s, z, ss, G), xx, ss)


# ------------------------------------------------------------------------------------------------- more than 16 rows
# (rows, columns, K) whose tiles are those of the key, ending inside one on both sides; K ends inside a block (and a step)
MANY = {(32, 128): dict(all=(77, 1155, 1120)),
        (64, 128): dict(fp16=(1030, 8197, 2080), bf16=(129, 13829, 1120), int8=(1030, 8197, 2080)),
        (128, 256): dict(all=(2050, 11011, 1120))}


def _many(tile, acts):
    sizes = MANY[tile]
    return sizes.get("all") or sizes[{torch.float16: "fp16", torch.bfloat16: "bf16", torch.int8: "int8"}[acts]]


@pytest.mark.parametrize("acts,dtype", ACTS, ids=NAMES)
@pytest.mark.parametrize("tile", MANY)
def test_the_calls_of_many_rows_reach_their_tiles(tile, acts, dtype):
    assert tile_of(acts, dtype, False, *_many(tile, acts)) == tile
    assert tile_of(acts, dtype, True, *_many(tile, acts)) == tile


@pytest.mark.gpu
@pytest.mark.parametrize("acts,dtype", ACTS, ids=NAMES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("G", [32, 64, 96, 128, 192, 256, 1 << 20])
@pytest.mark.parametrize("tile", MANY)
def test_many_rows(tile, G, zeros, acts, dtype):
    M, N, K = _many(tile, acts)
    assert tile_of(acts, dtype, zeros, M, N, K) == tile
    x, w, s, z, sr = make(M, N, K, G, acts, dtype, zeros)
    Oracle(w, s, z, G, acts).check(call(x, w, s, z, sr, G), x, sr)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("tile", MANY)
def test_a_row_that_is_no_number_stays_alone(tile, G, dtype):
    """Also where waves exchange the sums of the activations."""
    M, N, K = _many(tile, dtype)
    x, w, s, z, _ = make(M, N, K, G, dtype, dtype, True)
    want, row = call(x, w, s, z, None, G), M - 5
    for at, bad in ((0, float("nan")), (K - 1, float("inf")), (K // 2, float("-inf"))):
        y = x.clone()
        y[row, at] = bad
        got = call(y, w, s, z, None, G)
        assert not got[row].isfinite().any()
        assert torch.equal(got[:row], want[:row]) and torch.equal(got[row + 1:], want[row + 1:])


@pytest.mark.gpu
@pytest.mark.parametrize("acts,dtype", ACTS, ids=NAMES)
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 4101, 1120), (12, 11003, 1120), (77, 1155, 1120), (1030, 8197, 2080), (2050, 11011, 1120)])
def test_rows_far_from_zero(M, N, K, zeros, G, acts, dtype):
    """Activations of a large common mean and codes whose sums are 0 in every group (with zeros: at the zero), where what the offset of
    widened codes and the zeros add has to leave again: the result is small beside what it is made of."""
    x, w, s, _, sr = make(M, N, K, G, acts, dtype, False)
    x = torch.randint(90, 128, x.shape, dtype=torch.int8, device=DEV) if acts == torch.int8 else (x * 0.1 + 100).to(acts)
    w = ((w & 15) | ((16 - (w & 15)) % 16 << 4))   # q, -q (and -8, -8) side by side
    z = None
    if zeros:  # codes 0 .. 6 and 4 less them, at a zero of 2: the same value either way
        q = (w & 15).to(torch.int8) % 7
        w = ((q & 15) | ((4 - q) & 15) << 4).to(torch.uint8)
        z = torch.full_like(s, 2.0)
    oracle, out = Oracle(w, s, z, G, acts), call(x, w, s, z, sr, G)
    y, size = x.double() @ oracle.weight, x.double().abs() @ oracle.size
    if sr is not None:
        y, size = y * sr.double(), size * sr.double()
    off = (out.double() - y).abs_()
    assert (off <= torch.finfo(dtype).eps / 2 * y.abs() + (56 + K / 32) * 2.0 ** -24 * (size + y.abs())).all()
