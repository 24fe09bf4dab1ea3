"""Products in blocks of 32 in every tile that their rules choose among, with K in one part and in several, and the gated ones, on the
same GPU against 64 bits: sums that fp32 holds exactly have to come out as they are, others within the bound of test_gpu_mx_matmul.

The bound: half a step of the result's type; per instruction of 64 columns (8 bits: two of them) an alignment to 2^-24 of its largest term and
a rounding of the sum so far; sixteen parts of K joined, row factor and bias."""
import pytest
import torch

from quik_amd import _lib as L

DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]
# K that ends inside its first stage of 256 columns, behind two whole ones, with the first block of a third, inside a fifth, a ninth
WHOLE_K = (160, 512, 544, 1056, 2080)
# (rows, columns) of a tile's calls, ending inside one on both sides, with more than one band of four row tiles; columns of the gated ones: of either half
WHOLE = {4: {(32, 128): (170, 299), (64, 128): (193, 5121), (128, 128): (385, 5121), (256, 256): (2050, 13829)},
         8: {(32, 128): (170, 299), (64, 128): (193, 5121), (128, 128): (385, 5121), (128, 256): (333, 11011)}}
SPLIT = {4: {(32, 128): (47, 299, 13792), (64, 128): (65, 4101, 4544), (128, 128): (77, 2081, 13792), (256, 256): (520, 4101, 13792)},
         8: {(32, 128): (47, 299, 13792), (64, 128): (257, 1155, 4544), (128, 128): (193, 3001, 4544), (128, 256): (385, 5121, 4544)}}
GATED = {4: {(64, 64): (129, 288), (128, 64): (333, 2976), (256, 128): (2050, 2976)},
         8: {(64, 64): (129, 288), (128, 64): (333, 2976), (128, 128): (385, 5120)}}
CALLS = [(bits, tile) for bits in (4, 8) for tile in WHOLE[bits]]
GATED_CALLS = [(bits, tile) for bits in (4, 8) for tile in GATED[bits]]


def tile_of(bits, M, N, K, gated=False):
    """(parts of K, (rows, columns) of a workgroup); 0 parts: the kernel of few rows."""
    lib = L.load()
    t = lib.quik_mx_matmul_tile(bits, int(gated), M, N, K, 0 if gated else lib.quik_mx_matmul_workspace_bytes(bits, M, N, K))
    return t >> 24, (t >> 12 & 0xFFF, t & 0xFFF)


# ------------------------------------------------------------------------------------------------ the choice (no GPU)
def test_the_calls_reach_every_tile():
    for bits in (4, 8):
        for tile, (M, N) in WHOLE[bits].items():
            for K in WHOLE_K:
                assert tile_of(bits, M, N, K) == (1, tile), (bits, M, N, K)
        for tile, call in SPLIT[bits].items():
            parts, got = tile_of(bits, *call)
            assert parts > 1 and got == tile, (bits, call, parts, got)
        for tile, (M, inner) in GATED[bits].items():
            for K in WHOLE_K:
                assert tile_of(bits, M, inner, K, True) == (1, tile), (bits, M, inner, K)


def test_no_call_has_another_tile():
    """Over the sizes of models: the tiles of the tables above, the kernel of few rows up to 32 rows (gated 16), and nothing else."""
    for bits in (4, 8):
        seen, gated = set(), set()
        for M in (17, 24, 32, 33, 48, 64, 100, 128, 200, 256, 300, 512, 777, 1024, 2048, 4096):
            for N in (1, 128, 1024, 4096, 5120, 8192, 11008, 28672):
                for K in (32, 1024, 4096, 8192, 28672):
                    parts, tile = tile_of(bits, M, N, K)
                    assert parts or (M <= 32 and tile[0] == 32 and tile[1] <= 32)
                    seen.add(tile if parts else None)
                    gated.add(tile_of(bits, M, (N + 31) // 32 * 32, K, True))
        assert seen == {None, *WHOLE[bits]} and gated == {(1, tile) for tile in GATED[bits]}


def test_the_tile_of_few_rows_and_of_nothing():
    tile = L.load().quik_mx_matmul_tile
    for bits in (4, 8):
        assert [tile_of(bits, M, 4096, 4096) for M in (1, 8, 9, 16)] == [(0, (8, 16))] * 2 + [(0, (16, 16))] * 2
        assert [tile_of(bits, M, 4096, 4096, True) for M in (1, 8, 9, 16)] == [(0, (8, 32))] * 2 + [(0, (16, 32))] * 2
        # without its memory K is one part
        assert tile_of(bits, 64, 4096, 13824)[0] > 1 and tile(bits, 0, 64, 4096, 13824, 0) >> 24 == 1
    for call in ((6, 0, 64, 64, 64, 0), (4, 0, 0, 64, 64, 0), (4, 0, 64, 0, 64, 0), (4, 1, 64, 64, 0, 0), (4, 0, 1 << 31, 64, 64, 0), (4, 0, 64, 1 << 30, 64, 0),
                 (8, 1, 64, 64, (1 << 20) + 32, 0)):
        assert tile(*call) == 0


# -------------------------------------------------------------------------------------------------------- the products
def ms():
    from quik import microscaled
    return microscaled


def whole_numbers(gen, rows, K, bits, largest, spread):
    """(numbers, codes, exponent bytes): whole numbers up to `spread`, the first of each 32 as `largest`, which is the block's exponent."""
    v = torch.randint(-spread, spread + 1, (rows, K), generator=gen, device=DEV)
    v[:, ::32] = largest * (1 - 2 * torch.randint(0, 2, (rows, K // 32), generator=gen, device=DEV))
    return v.double(), *ms().quantize(v.half(), bits)


def exact_operands(seed, M, N, K, bits):
    gen = torch.Generator(DEV).manual_seed(seed)
    return gen, whole_numbers(gen, M, K, bits, 4, 2), whole_numbers(gen, N, K, 4, 6, 1)


def random_operands(seed, M, N, K, bits):
    """Numbers of blocks whose exponents lie up to six apart; what the codes stand for are numbers of bf16."""
    gen = torch.Generator(DEV).manual_seed(seed)

    def rows(n, b):
        v = torch.randn(n, K // 32, 32, generator=gen, device=DEV) * torch.exp2(torch.randint(-3, 4, (n, K // 32, 1), generator=gen, device=DEV).float())
        q, s = ms().quantize(v.view(n, K).bfloat16(), b)
        return ms().dequantize(q, s, torch.bfloat16).double(), q, s
    return gen, rows(M, bits), rows(N, 4)


def row_and_bias(gen, M, N, dtype):
    """Factors that are powers of two, and whole numbers: what they make of an exact sum is exact."""
    return torch.exp2(torch.randint(-3, 4, (M, 1), generator=gen, device=DEV).float()), torch.randint(-64, 65, (N,), generator=gen, device=DEV).to(dtype)


def check_call(bits, M, N, K, dtype):
    gen, (x, xq, xs), (w, wq, ws) = exact_operands(M + K, M, N, K, bits)
    row, bias = row_and_bias(gen, M, N, dtype)
    sums = x @ w.t()      # (below 2^24: numbers of fp32 in any order)
    out = ms().matmul(xq, xs, wq, ws, dtype)
    assert out.dtype == dtype and torch.equal(out, sums.to(dtype))
    assert torch.equal(ms().matmul(xq, xs, wq, ws, dtype, row, bias), (sums * row.double() + bias.double()).to(dtype))
    gen, (x, xq, xs), (w, wq, ws) = random_operands(N + K, M, N, K, bits)
    out = ms().matmul(xq, xs, wq, ws, dtype, row, bias)
    y = x @ w.t() * row.double() + bias.double()
    steps = -(-K // 64) * (bits // 4) + 20
    limit = torch.finfo(dtype).eps / 2 * y.abs() + 2.0 ** -24 * (dtype == torch.float16) + (x.abs() @ w.abs().t()) * row.double() * (steps * 2.0 ** -24) + 2.0 ** -23 * y.abs()
    assert ((out.double() - y).abs() <= limit).all()
    assert torch.equal(ms().matmul(xq, xs, wq, ws, dtype, row, bias), out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", WHOLE_K)
@pytest.mark.parametrize("bits,tile", CALLS)
def test_product(bits, tile, K, dtype):
    M, N = WHOLE[bits][tile]
    assert tile_of(bits, M, N, K) == (1, tile)
    check_call(bits, M, N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits,tile", CALLS)
def test_product_with_k_in_parts(bits, tile, dtype):
    parts, got = tile_of(bits, *SPLIT[bits][tile])
    assert parts > 1 and got == tile
    check_call(bits, *SPLIT[bits][tile], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("bits,tile", CALLS)
def test_what_is_no_number_stays_alone(bits, tile, split):
    """A block of x without a number is a row of NaNs, one of the weights a column; every other result is as before.  The blocks are the last and one in
    the middle of K."""
    M, N, K = SPLIT[bits][tile] if split else (*WHOLE[bits][tile], 1056)
    _, (_, xq, xs), (_, wq, ws) = random_operands(5, M, N, K, bits)
    want = ms().matmul(xq, xs, wq, ws, torch.bfloat16)
    xs[M - 3, K // 32 - 1], xs[7, K // 64] = 255, 255
    ws[N - 2, K // 32 - 1], ws[11, K // 64] = 255, 255
    bad = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    bad[M - 3], bad[7], bad[:, N - 2], bad[:, 11] = True, True, True, True
    got = ms().matmul(xq, xs, wq, ws, torch.bfloat16)
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("bits,tile", CALLS)
def test_exponent_bytes_at_any_address(bits, tile):
    M, N = WHOLE[bits][tile]
    for K in (160, 1056):
        _, (_, xq, xs), (_, wq, ws) = random_operands(6, M, N, K, bits)
        want = ms().matmul(xq, xs, wq, ws, torch.bfloat16)
        for shift in (1, 2, 3):
            moved = [torch.cat((t.new_full((shift,), 255), t.flatten()))[shift:].view(t.shape) for t in (xs, ws)]
            assert moved[0].data_ptr() % 4 == shift and torch.equal(ms().matmul(xq, moved[0], wq, moved[1], torch.bfloat16), want)


# ---------------------------------------------------------------------------------------------------- gated products
def check_gated(bits, M, inner, K, dtype, q_bits):
    """Of exact sums, whatever their order, gate and up are those of matmul, and the codes bit for bit those of silu_mul_quantize."""
    gen, (x, xq, xs), (w, wq, ws) = exact_operands(M + K, M, 2 * inner, K, bits)
    row = torch.exp2(torch.randint(-7, -3, (M, 1), generator=gen, device=DEV).float())
    both = (x @ w.t() * row.double()).to(dtype)
    assert torch.equal(ms().matmul(xq, xs, wq, ws, dtype, row), both)
    got, want = ms().gated_matmul(xq, xs, wq, ws, dtype, row, q_bits), ms().silu_mul_quantize(both[:, :inner], both[:, inner:], q_bits)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("q_bits", [4, 8])
@pytest.mark.parametrize("K", WHOLE_K)
@pytest.mark.parametrize("bits,tile", GATED_CALLS)
def test_gated_product(bits, tile, K, q_bits):
    M, inner = GATED[bits][tile]
    assert tile_of(bits, M, inner, K, True) == (1, tile)
    check_gated(bits, M, inner, K, torch.bfloat16 if K % 512 else torch.float16, q_bits)


@pytest.mark.gpu
@pytest.mark.parametrize("q_bits", [4, 8])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 5, 8, 9, 16, 17, 24, 32, 33])
@pytest.mark.parametrize("bits", [4, 8])
def test_gated_product_of_few_rows(bits, M, dtype, q_bits):
    """Also where matmul of as many rows has the kernel of few rows and the gated product tiles: 17 to 32 rows."""
    for inner, K in ((96, 160), (288, 544), (11008, 1056)):
        check_gated(bits, M, inner, K, dtype, q_bits)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,tile", GATED_CALLS)
def test_gated_blocks_without_a_number_stay_alone(bits, tile):
    M, inner = GATED[bits][tile]
    _, (_, xq, xs), (_, wq, ws) = random_operands(8, M, 2 * inner, 1056, bits)
    want = ms().gated_matmul(xq, xs, wq, ws, torch.bfloat16)
    xs[M - 2, 32], ws[inner - 1, 5], ws[inner + 40, 0] = 255, 255, 255      # a row; a gate of the last block, up of the second
    bad = torch.zeros(M, inner // 32, dtype=torch.bool, device=DEV)
    bad[M - 2], bad[:, -1], bad[:, 1] = True, True, True
    got = ms().gated_matmul(xq, xs, wq, ws, torch.bfloat16)
    assert torch.equal(got[1] == 255, bad) and torch.equal(got[1][~bad], want[1][~bad])
    codes = lambda t: t.view(M, inner // 32, 16)
    assert torch.equal(codes(got[0])[~bad], codes(want[0])[~bad]) and not codes(got[0])[bad].any()
