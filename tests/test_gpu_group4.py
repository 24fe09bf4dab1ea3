"""matmul.int4GroupMatmul against its formula in 64 bits.

Tolerance of one value: half a step of the result's type, and the roundings of the sums.  A group's 32-column steps and the groups
themselves are added one after the other in fp32, each product exact: at most `32 + K / 32 + 24` additions of 2^-24 each of
sum |x| (|q| + c) s, with c the constant that the widened codes carry and zero points add: 136 for bf16 (its codes are widened to 136 +
q), |z| for zeros.  int8 activations: the groups' sums are exact, the groups are added in fp32."""
import numpy as np
import pytest
import torch

import quik

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]


def make(M, N, K, G, acts, dtype, zeros=False, bias=False, seed=0, whole=True):
    g = torch.Generator().manual_seed(seed + M + N + K + G)
    groups = -(-K // G)
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand(N, groups, generator=g) * 0.009 + 0.001).to(dtype)
    z = None
    if zeros:
        z = torch.randint(-8, 8, (N, groups), generator=g).to(dtype) if whole else (torch.rand(N, groups, generator=g) * 16 - 8).to(dtype)
    sr = None
    if acts == torch.int8:
        x = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8)
        sr = torch.rand(M, 1, generator=g) * 0.02 + 0.01
    else:
        x = torch.randn(M, K, generator=g)
        x[:, ::128] *= 10
        x = x.to(acts)
    b = torch.randn(N, generator=g).to(dtype) if bias else None
    move = lambda t: None if t is None else t.to(DEV)
    return tuple(move(t) for t in (x, w, s, z, sr, b))


def oracle(x, w, s, z, sr, b, G):
    """(value, sum of magnitudes) in 64 bits"""
    up = lambda t: t.double().cpu().numpy()
    by = w.cpu().numpy()
    q = np.empty((by.shape[0], 2 * by.shape[1]))
    q[:, 0::2], q[:, 1::2] = ((by & 15) ^ 8).astype(int) - 8, ((by >> 4) ^ 8).astype(int) - 8
    at = np.arange(q.shape[1]) // G
    zz = 0 if z is None else up(z)[:, at]
    extra = (136 if x.dtype == torch.bfloat16 else 0) + np.abs(zz)
    y = up(x) @ ((q - zz) * up(s)[:, at]).T
    size = np.abs(up(x)) @ ((np.abs(q) + extra) * up(s)[:, at]).T
    if sr is not None:
        y, size = y * up(sr).reshape(-1, 1), size * up(sr).reshape(-1, 1)
    if b is not None:
        y = y + up(b)
    return y, size


def check(out, args, G):
    y, size = oracle(*args, G)
    K = args[0].shape[1]
    half = torch.finfo(out.dtype).eps / 2
    got = out.double().cpu().numpy()
    assert got.shape == y.shape
    adds = 32 + K / 32 + 24 if args[0].dtype != torch.int8 else K / 32 + 24
    assert (np.abs(got - y) <= half * np.abs(y) + adds * 2.0 ** -24 * (size + np.abs(y))).all()
    if y.size > 64:
        assert np.linalg.norm(got - y) <= half * np.linalg.norm(y)


def call(args, G):
    x, w, s, z, sr, b = args
    return quik.matmul.int4GroupMatmul(x, w, s, G, zeros=z, scale_row=sr, bias=b)


# every number of token rows per matrix tile and its ends; columns that fill no tile; K that ends inside a block of 128
SIZES = [(1, 1, 32), (1, 16, 128), (1, 33, 4096), (2, 100, 160), (3, 7, 1024), (4, 64, 992), (5, 40, 256), (8, 200, 2080), (9, 31, 512),
         (16, 65, 1056), (17, 48, 640), (32, 130, 384), (33, 17, 96), (63, 129, 1184), (64, 512, 256), (65, 70, 544), (100, 300, 1024),
         (128, 128, 2048), (129, 257, 416), (300, 141, 768), (515, 96, 1280)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(M, N, K, codes, dtype):
    args = make(M, N, K, 128, torch.int8 if codes else dtype, dtype)
    check(call(args, 128), args, 128)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("G", [32, 64, 96, 128, 160, 256, 384, 1 << 20])
@pytest.mark.parametrize("M,N,K", [(1, 50, 1120), (6, 80, 2048), (13, 33, 352), (40, 96, 1184), (150, 130, 1120)])
def test_groups(M, N, K, G, zeros, codes, dtype):
    args = make(M, N, K, G, torch.int8 if codes else dtype, dtype, zeros, bias=G == 64)
    check(call(args, G), args, G)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 257, 11008), (16, 128, 13824), (70, 160, 8192)])
def test_long_rows_zeros_between_codes_and_bias(M, N, K, codes, dtype):
    args = make(M, N, K, 128, torch.int8 if codes else dtype, dtype, True, True, whole=False)
    check(call(args, 128), args, 128)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("G,zeros", [(128, False), (64, True), (32, True)])
def test_the_widest_tiles(G, zeros, codes, dtype):
    """Rows and columns for the tiles of 128 x 256, ending inside one on both sides; K that ends inside a block."""
    args = make(1030, 8197, 2080, G, torch.int8 if codes else dtype, dtype, zeros)
    check(call(args, G), args, G)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("M,N,K,G", [(20, 130, 4096, 128), (64, 516, 8224, 64), (90, 257, 6016, 128)])
def test_split_rows(M, N, K, G, codes, dtype):
    """K split over workgroups, and the same call without the memory for it."""
    from quik_amd import _lib as L
    args = make(M, N, K, G, torch.int8 if codes else dtype, dtype, True, True)
    x, w, s, z, sr, b = args
    lib, dt, bits = L.load(), L.dtype_id(s, "", True), 8 if codes else 16
    need = lib.quik_int4_group_matmul_workspace_bytes(bits, dt, M, N, K)
    assert need > 0
    split = call(args, G)
    check(split, args, G)
    out = torch.empty_like(split)
    for ws, size in ((None, 0), (torch.empty(need, dtype=torch.uint8, device=DEV), need - 1)):
        out.fill_(7)
        L.check(lib.quik_int4_group_matmul(L.ptr(x), bits, L.ptr(w), L.ptr(s), L.ptr(z), L.ptr(sr), L.ptr(b), dt, M, N, K, G, L.ptr(out), L.ptr(ws),
                                           size, L.stream()), "")
        check(out, args, G)
    assert torch.equal(split, call(args, G))


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("M", [1, 4, 12, 50, 200])
def test_extreme_codes(M, codes):
    """Every code at its lowest: the largest sums that there are; and rows of zeros."""
    x, w, s, z, sr, b = make(M, 40, 2048, 128, torch.int8 if codes else torch.float16, torch.float16)
    w.fill_(0x88)
    x.fill_(-128 if codes else 2)
    s.fill_(0.0009765625)
    if codes:
        sr.fill_(0.015625)
    out = call((x, w, s, z, sr, b), 128)
    want = 8 * 128 * 2048 / 1024 / 64 if codes else -8 * 2 * 2048 / 1024
    assert (out == want).all()
    assert not call((torch.zeros_like(x), w, s, z, sr, b), 128).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 7, 16, 60, 140])
def test_a_row_that_is_no_number_stays_alone(M, dtype):
    args = make(M, 70, 608, 128, dtype, dtype, True)
    want = call(args, 128)
    for bad in (float("nan"), float("inf")):
        x = args[0].clone()
        x[M // 2, 607] = bad
        got = call((x,) + args[1:], 128)
        assert not got[M // 2].isfinite().any()
        keep = torch.arange(M, device=DEV) != M // 2
        assert torch.equal(got[keep], want[keep])


def test_empty():
    args = make(1, 40, 128, 128, torch.float16, torch.float16)
    assert call((args[0][:0],) + args[1:], 128).shape == (0, 40)
    assert call((args[0], args[1][:0], args[2][:0], None, None, None), 128).shape == (1, 0)


@pytest.mark.parametrize("codes", [False, True])
def test_offsets_past_32_bits(codes):
    """Activations, results and weights of more than 2^31 elements and bytes."""
    x, w, s, z, sr, b = make(8, 48, 16384, 128, torch.int8 if codes else torch.float16, torch.float16)
    rows = (1 << 17) + 8
    many = torch.zeros(rows, 16384, dtype=x.dtype, device=DEV)
    many[-8:] = x
    scale = None if sr is None else torch.ones(rows, 1, device=DEV)
    if scale is not None:
        scale[-8:] = sr
    out = call((many, w, s, z, scale, b), 128)
    check(out[-8:], (x, w, s, z, sr, b), 128)
    assert not out[:-8].any()
    del many, out
    cols = (1 << 18) + 48
    wide = torch.full((cols, 8192), 0x88, dtype=torch.uint8, device=DEV)
    wide[-48:] = w
    scales = torch.zeros(cols, 128, dtype=torch.float16, device=DEV)
    scales[-48:] = s
    for rows in (8, 24):
        xx = x.repeat(3, 1)[:rows]
        ss = None if sr is None else sr.repeat(3, 1)[:rows]
        out = call((xx, wide, scales, None, ss, None), 128)
        check(out[:, -48:], (xx, w, s, None, ss, None), 128)
        assert not out[:, :-48].any()


def test_one_group_of_all_columns_and_long_rows():
    """The longest rows there are."""
    K = 1 << 20
    for M in (1, 20):
        for G in (K, 64):
            args = make(M, 18, K, G, torch.int8, torch.float16, True)
            args[2].mul_(2.0 ** -9)
            check(call(args, G), args, G)
