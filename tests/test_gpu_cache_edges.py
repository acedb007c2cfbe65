"""The cache operators where their arithmetic or their arguments are at an edge: weights that
cancel, bounds of any width, scales at the ends of float32, strides of a single row."""
import math

import numpy as np
import pytest
import torch

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X GPU", allow_module_level=True)

from oracle import blocks as O
from paged_decode.block_decode import (allocate_block_resources, fp8_decode, select_blocks,
                                       sparse_decode)
from paged_decode.kv_append import allocate_bounds, append_kv, block_bounds
from paged_decode.spec import DecodeSpec
from test_gpu_append import bits
from test_gpu_blocks import attend, bounds_of, check, dev, make, spec_of

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
KINDS = [torch.bfloat16, E4M3]
IDS = ["bf16", "e4m3"]


def two_tokens(scores, values, dim, kind, scale, heads=4):
    """Attention over two tokens a sequence: scores [B, 2], held exactly by `kind` and times
    `scale`, values [B, 2, D]."""
    batch = len(scores)
    k, v = torch.zeros((batch, 256, 1, dim)), torch.zeros((batch, 256, 1, dim))
    k[:, :2, 0, 1], v[:, :2, 0] = scores, values
    k, v = (t.to(kind).cuda() for t in (k, v))
    assert torch.equal(k[:, :2, 0, 1].float().cpu(), scores)
    q = torch.zeros((batch, heads, dim), dtype=torch.bfloat16, device="cuda")
    q[..., 1] = 1.0
    tables = torch.arange(batch, dtype=torch.int32, device="cuda")[:, None].contiguous()
    lengths = torch.full((batch,), 2, dtype=torch.int32, device="cuda")
    spec = DecodeSpec(batch, heads, 1, dim, 256)
    if kind == E4M3:
        return fp8_decode(q, k, v, tables, lengths, scale=scale,
                          resources=allocate_block_resources(spec, "cuda")).cpu()
    blocks = torch.zeros((batch, 1, 1), dtype=torch.int32, device="cuda")
    return sparse_decode(q, k, v, tables, lengths, blocks, scale=scale,
                         resources=allocate_block_resources(spec, "cuda", kept=1)).cpu()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_weights_that_cancel(dim, kind):
    """Two tokens of values 1 and -1 whose weights differ by 2^-13 to 2^-10 of themselves: the
    output (1 - p) / (1 + p) is as exact as the weights.

    Float32: p = 2^x, x = -score scale log2 e below 2^-9 in size, so that its roundings move p by
    2^-32 and the exponential by 2^-22; the numerator's sum has up to four additions of numbers
    up to 1, 2^-23 each where an instruction truncates.  (2^-22 + 2^-21) / (1 + p) is below 2^-21,
    the quotient's own rounding 2^-23 of it; then the output's half step, 2^-8 of it."""
    sizes = torch.arange(8, 16) / 8.0                       # 1 to 1.875: exact in e4m3
    scores = torch.stack([torch.zeros(8), -sizes], 1)
    values = torch.tensor([1.0, -1.0])[None, :, None].expand(8, 2, dim)
    for i in range(24):
        scale = 2.0 ** -13 * (1 + i / 7)
        p = torch.exp(-sizes.double() * scale)
        exact = ((1 - p) / (1 + p))[:, None, None]
        got = two_tokens(scores, values, dim, kind, scale).double()
        allowed = 2.0 ** -21 + 2.0 ** -8 * (exact + 2.0 ** -21)
        error = (got - exact).abs()
        assert (error <= allowed).all(), (i, float((error / allowed).max()))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinite_and_huge_values_of_small_weights(dim, kind):
    """A weight of 2^-x: an infinite value (bf16 alone holds one) makes its channel infinite,
    the largest finite one adds what it is worth, and nothing once the weight is zero."""
    steps = [0.0, 8, 24, 30, 60, 88, 96, 104, 120, 160, 448]
    scores = torch.tensor([[0.0, -s] for s in steps])
    big = 448.0 if kind == E4M3 else float(torch.finfo(torch.bfloat16).max)
    values = torch.ones((len(steps), 2, dim))
    values[:, 1, 0] = big
    values[:, 1, dim - 1] = -big
    if kind != E4M3:
        values[:9, 1, 1], values[:9, 1, 2] = math.inf, -math.inf
    got = two_tokens(scores, values, dim, kind, math.log(2.0)).double()
    for i, s in enumerate(steps):
        p = 2.0 ** -s
        for c, value in ((0, big), (dim - 1, -big), (3, 1.0)):
            exact = (1 + p * value) / (1 + p)
            # x = -s: the two roundings of its factor, 2^-23 s; the exponential's 2^-22; sums
            # and quotient 2^-21.  A weight below 2^-126 is zero.
            lost = p * abs(value) if s > 120 else 0.0
            allowed = (2.0 ** -23 * s + 2.0 ** -20) * (1 + p * abs(value)) + lost
            allowed += 2.0 ** -8 * (abs(exact) + allowed)
            assert ((got[i, :, c] - exact).abs() <= allowed).all(), (s, c)
        if kind != E4M3 and i < 9:
            assert (got[i, :, 1] == math.inf).all() and (got[i, :, 2] == -math.inf).all(), s


@pytest.mark.parametrize("power", [40, 60, None], ids=["2^40", "2^60", "lowest"])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (4, 2, 128), (16, 4, 256), (32, 8, 128), (9, 3, 64),
                                      (32, 4, 256), (17, 1, 64), (40, 2, 128)])
def test_select_by_bounds_of_any_width(hq, hkv, d, power):
    """The corner that a query's sign leaves out moves no score, however large: a channel of
    positive queries whose smallest keys are far below, one of negative queries whose largest
    are far above.  With whole numbers, scores that tie."""
    far = float(torch.finfo(torch.bfloat16).max) if power is None else 2.0 ** power
    lengths = [64 * 300, 64 * 201 - 5, 700]
    x = make(lengths, hq, hkv, d, torch.bfloat16, seed=hq + d)
    gen = torch.Generator().manual_seed(hq)
    for integers in (False, True):
        q = (x["q"].float().round() if integers else x["q"].float())
        q[..., 3] = q[..., 3].abs() + 1
        q[..., d - 6] = -q[..., d - 6].abs() - 1
        q = q.bfloat16()
        bounds = bounds_of(x, hq + d, integers)
        wide = torch.rand((2, *bounds.shape[:3]), generator=gen) < 0.3
        bounds[..., 0, 3][wide[0]] = -far
        bounds[..., 1, d - 6][wide[1]] = far
        res = allocate_block_resources(spec_of(x), "cuda", kept=40)
        got = select_blocks(q.cuda(), bounds.cuda(), x["tables"].cuda(), x["lengths"].cuda(),
                            resources=res)
        assert torch.equal(got.cpu(), O.select(q, bounds, x["tables"], x["lengths"], 40))


def test_select_beside_bounds_that_are_not_finite():
    """Blocks of wide, of infinite and of NaN bounds next to one another."""
    x = make([64 * 300], 8, 2, 64, torch.bfloat16, seed=5)
    bounds = bounds_of(x, 5)
    gen = torch.Generator().manual_seed(5)
    x["q"][..., 3] = x["q"][..., 3].abs() + 1
    x["q"][0, 2, 8] = 0.0
    wide = torch.rand(bounds.shape[:3], generator=gen) < 0.5
    bounds[..., 0, 3][wide] = -float(torch.finfo(torch.bfloat16).max)
    for value, corner, channel in ((math.inf, 1, 8), (-math.inf, 0, 3), (math.nan, 1, 40),
                                   (math.nan, 0, 0)):
        odd = torch.rand(bounds.shape[:3], generator=gen) < 0.02
        bounds[..., corner, channel][odd] = value
    for kept in (4, 20, 60):
        res = allocate_block_resources(spec_of(x), "cuda", kept=kept)
        got = select_blocks(x["q"].cuda(), bounds.cuda(), x["tables"].cuda(), x["lengths"].cuda(),
                            resources=res)
        assert torch.equal(got.cpu(), O.select(x["q"], bounds, x["tables"], x["lengths"], kept))


@pytest.mark.parametrize("scale", [1e-40, 2.0 ** -126, 1.1464847e-36, 1.7e-38, 3.3e-35, 1e-32, 7e-31, 1.3e-25,
                                   2.1e-19, 5e18, 1e30, 8.6e37, 1.2e38, 3.3e38])
def test_quotients_by_scales_of_any_size(scale):
    """The stored value is the rounded division's, as at ordinary scales: products of the scale
    with values and midpoints of e4m3 and the floats next to them, through a rotation by
    (cos, 0)."""
    n, d = 2048, 64
    scale = torch.tensor([scale], dtype=torch.float32)
    rng = np.random.default_rng(34)
    grid = torch.arange(127, dtype=torch.uint8).view(E4M3).float()
    grid = torch.cat([grid, (grid[1:] + grid[:-1]) / 2])
    grid = grid[(grid * scale) < 1e38]
    x = grid[torch.from_numpy(rng.integers(0, len(grid), (n, d // 2)))] * scale
    near = torch.from_numpy(rng.integers(-2, 3, (n, d // 2)).astype(np.int32))
    x = (x.view(torch.int32) + near * (x > 0)).view(torch.float32)
    rope = torch.stack([x, torch.zeros_like(x)], -1).cuda()
    k = torch.cat([torch.ones(n, 1, d // 2), torch.zeros(n, 1, d // 2)], 2).bfloat16().cuda()
    cache = [torch.zeros((8, 256, 1, d), device="cuda").to(E4M3) for _ in range(2)]
    at = torch.arange(n, device="cuda")
    append_kv(None, k, k, at, rope, *cache, at.int(), k_scale=scale.cuda())
    want = O.stored(x[:, None], scale, E4M3)
    assert torch.equal(bits(cache[0]).view(n, d)[:, :d // 2], bits(want)[:, 0])


@pytest.mark.parametrize("scale", [1e-42, 2.0 ** -126, 3e-37, 2.0 ** -62, 1.5 * 2.0 ** 62, 3.3e38])
def test_special_values_by_scales_of_any_size(scale):
    special = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 3.3e38, -3.3e38, 1e-38, -1e-38,
                            1e-40, -1e-40, 2.0 ** -60, -2.0 ** 60, 1.0, -1.0, 448.0], dtype=BF16)
    rows = special.repeat(4).view(1, 1, 64)
    scales = torch.tensor([scale])
    cache = [torch.zeros((1, 256, 1, 64), device="cuda").to(E4M3) for _ in range(2)]
    append_kv(None, rows.cuda(), rows.cuda(), None, None, *cache,
              torch.zeros(1, dtype=torch.int32, device="cuda"), k_scale=scales.cuda(),
              v_scale=scales.cuda())
    want = O.stored(rows.float(), scales, E4M3)[0, 0]
    for c in cache:
        got = c.cpu()[0, 0, 0]
        nan = want.float().isnan()
        assert torch.equal(got.float().isnan(), nan)
        assert torch.equal(bits(got)[~nan], bits(want)[~nan])


def test_no_rows_have_no_bounds():
    x = torch.zeros((2, 256, 2, 64), dtype=BF16, device="cuda")
    bounds = torch.full_like(allocate_bounds(x), 7.0)
    block_bounds(x, torch.zeros(0, dtype=torch.int32, device="cuda"), bounds)
    assert (bounds == 7.0).all()


def test_gradients_are_refused():
    x = make([700, 90], 8, 2, 128, E4M3, seed=61)
    g = dev(x)
    dense = allocate_block_resources(spec_of(x), "cuda")
    listed = allocate_block_resources(spec_of(x), "cuda", kept=3)
    blocks = torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda")
    bounds = bounds_of(x, 61).cuda()
    q = g["q"].clone().requires_grad_()
    keys = g["k"].bfloat16().requires_grad_()
    calls = [lambda: attend(x, dict(g, q=q), dense),
             lambda: attend(x, dict(g, q=q), listed, blocks),
             lambda: attend(x, dict(g, k=keys, v=g["v"].bfloat16(), k_scale=None, v_scale=None),
                            listed, blocks),
             lambda: select_blocks(q, bounds, g["tables"], g["lengths"], resources=listed)]
    for call in calls:
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("heads", [1, 4])
def test_one_row_of_any_stride(heads, kind):
    """A dimension of one entry has a stride that nothing reads."""
    x = make([700], heads, 1, 128, kind, seed=62)
    g = dev(x)
    strides = (3, 128 if heads > 1 else 5, 1)
    res = allocate_block_resources(spec_of(x), "cuda", kept=9)
    blocks = torch.arange(9, dtype=torch.int32, device="cuda").view(1, 1, 9)
    bounds = bounds_of(x, 62).cuda()
    plain = [attend(x, g, res, blocks).clone(),
             select_blocks(g["q"], bounds, g["tables"], g["lengths"], resources=res).clone()]
    g["q"] = torch.as_strided(g["q"], g["q"].shape, strides)
    assert torch.equal(attend(x, g, res, blocks), plain[0])
    assert torch.equal(select_blocks(g["q"], bounds, g["tables"], g["lengths"], resources=res),
                       plain[1])
    if kind == E4M3:
        check(attend(x, g, allocate_block_resources(spec_of(x), "cuda")), x)


def test_choices_and_dense_attention_have_their_bits_in_every_batch_of_a_bucket():
    """Five rows of eight, as a padded step has them: the rows' own bits, in every order."""
    lengths = [700, 90, 5000, 64, 0, 3333, 1, 4097]
    x = make(lengths, 8, 2, 128, E4M3, seed=44)
    g = dev(x)
    spec = DecodeSpec(8, 8, 2, 128, 5120)
    dense = allocate_block_resources(spec, "cuda")
    listed = allocate_block_resources(spec, "cuda", kept=9)
    bounds = bounds_of(x, 44).cuda()

    def step(rows):
        part = {n: t[rows] if n in ("q", "tables", "lengths") else t for n, t in g.items()}
        return (attend(x, part, dense).clone(),
                select_blocks(part["q"], bounds, part["tables"], part["lengths"],
                              resources=listed).clone())

    whole = step(list(range(8)))
    for rows in ([0, 1, 2, 3, 4], [7, 2, 5, 0, 4, 1], [6, 5, 4, 3, 2, 1, 0]):
        for got, want in zip(step(rows), whole):
            assert torch.equal(got, want[rows])


def test_select_beside_pages_outside_the_cache():
    """Blocks of a page that the cache does not have rank below all others, the lowest first."""
    gen = torch.Generator().manual_seed(6)
    bounds = torch.randn((3, 4, 1, 1, 64), generator=gen).expand(3, 4, 1, 2, 64).bfloat16()
    q = torch.randn((2, 4, 64), generator=gen).bfloat16()
    lengths = torch.full((2,), 64 * 12, dtype=torch.int32)
    for outside in (-5, 3, 2 ** 31 - 1):
        tables = torch.tensor([[0, outside, 2], [1, outside, 0]], dtype=torch.int32)
        known = torch.tensor([[0, 1, 2], [1, 2, 0]], dtype=torch.int32)
        for kept in (5, 8, 10):
            res = allocate_block_resources(DecodeSpec(2, 4, 1, 64, 768), "cuda", kept=kept)
            got = select_blocks(q.cuda(), bounds.contiguous().cuda(), tables.cuda(), lengths.cuda(),
                                resources=res).cpu()
            for b in range(2):
                j = torch.tensor([i for i in range(1, 11) if not 4 <= i < 8])
                s = O.scores(q[b], bounds[known[b, j // 4].long(), j % 4][:, 0])
                order = j[torch.sort(s, descending=True, stable=True).indices].tolist() + [4, 5, 6, 7]
                assert got[b, 0].tolist() == sorted([0, *order[:kept - 2], 11])
