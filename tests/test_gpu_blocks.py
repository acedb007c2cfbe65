"""fp8_decode, select_blocks and sparse_decode against the plain forms in 64 bits
(oracle/blocks.py: bounds derived from float32 arithmetic and one bf16 rounding)."""
import numpy as np
import pytest
import torch

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X GPU", allow_module_level=True)

from oracle import blocks as O
from paged_decode.block_decode import (allocate_block_resources, fp8_decode, select_blocks,
                                       sparse_decode)
from paged_decode.kv_append import allocate_bounds, append_kv, rope_cache
from paged_decode.spec import DecodeSpec

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
KINDS = [torch.bfloat16, E4M3]
IDS = ["bf16", "e4m3"]


def make(lengths, hq, hkv, d, kind, seed, spare=2, scales=True):
    """A paged cache whose slots behind the lengths hold NaN, its tables -1 behind the pages."""
    gen = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    counts = [-(-n // 256) for n in lengths]
    width = max(1, *counts)
    order = rng.permutation(sum(counts) + spare).astype(np.int32).tolist()
    tables = torch.tensor([[order.pop() for _ in range(c)] + [-1] * (width - c) for c in counts],
                          dtype=torch.int32)
    k, v = (torch.randn((sum(counts) + spare, 256, hkv, d), generator=gen).to(kind)
            for _ in range(2))
    nan = torch.zeros(k.shape[:2], dtype=torch.bool)
    nan[:] = True
    for table, n in zip(tables, lengths):
        for t0 in range(0, n, 256):
            nan[table[t0 // 256], :n - t0] = False
    for c in (k, v):
        c.view(torch.uint8 if kind == E4M3 else torch.int16)[nan] = 0x7F if kind == E4M3 else 0x7FC0
    q = torch.randn((len(lengths), hq, d), generator=gen).to(torch.bfloat16)
    scale = [torch.rand(hkv, generator=gen) + 0.5 if kind == E4M3 and scales else None
             for _ in range(2)]
    return dict(q=q, k=k, v=v, tables=tables, lengths=torch.tensor(lengths, dtype=torch.int32),
                k_scale=scale[0], v_scale=scale[1])


def dev(x):
    return {n: None if t is None else t.cuda() for n, t in x.items()}


def spec_of(x, capacity=None):
    b, hq, d = x["q"].shape
    return DecodeSpec(b, hq, x["k"].shape[2], d, capacity or x["tables"].shape[1] * 256)


def attend(x, g, resources, blocks=None):
    if blocks is None:
        return fp8_decode(g["q"], g["k"], g["v"], g["tables"], g["lengths"], resources=resources,
                          k_scale=g["k_scale"], v_scale=g["v_scale"])
    return sparse_decode(g["q"], g["k"], g["v"], g["tables"], g["lengths"], blocks,
                         resources=resources, k_scale=g["k_scale"], v_scale=g["v_scale"])


def check(got, x, blocks=None, **more):
    exact, bound = O.attention(x["q"], x["k"], x["v"], x["tables"], x["lengths"], blocks,
                               k_scale=x["k_scale"], v_scale=x["v_scale"], **more)
    ok = O.bf16_close(got.cpu(), exact, bound)
    assert ok.all(), (int((~ok).sum()), float((got.cpu().double() - exact).abs().max()))


LENGTHS = [[1], [0, 1, 31, 32, 33, 63, 64, 65, 127, 255, 256, 257], [700, 0, 2064, 1500],
           [5000], [64 * 97]]
HEADS = [(16, 4, 256), (32, 8, 128), (16, 16, 64), (8, 2, 128), (4, 4, 256), (17, 1, 64),
         (40, 2, 128), (16, 1, 256), (6, 3, 64)]


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_fp8_decode(lengths, hq, hkv, d):
    x = make(lengths, hq, hkv, d, E4M3, seed=hq + d + len(lengths), scales=hq != 8)
    g = dev(x)
    check(attend(x, g, allocate_block_resources(spec_of(x), "cuda")), x)


def random_blocks(x, kept, seed):
    """Random ascending choices, some rows shorter than kept, one listing nothing."""
    rng = np.random.default_rng(seed)
    b, hkv = x["q"].shape[0], x["k"].shape[2]
    out = torch.full((b, hkv, kept), -1, dtype=torch.int32)
    for i in range(b):
        n = -(-int(x["lengths"][i]) // 64)
        for g in range(hkv):
            take = min(n, kept if (i + g) % 3 else rng.integers(0, kept + 1))
            out[i, g, :take] = torch.from_numpy(np.sort(rng.permutation(n)[:take]))
    return out


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lengths,kept", [([1], 1), (LENGTHS[1], 3), ([700, 0, 2064, 1500], 9),
                                          ([5000], 37)], ids=str)
def test_sparse_decode(lengths, kept, hq, hkv, d, kind):
    x = make(lengths, hq, hkv, d, kind, seed=hq + d + kept)
    g = dev(x)
    blocks = random_blocks(x, kept, seed=kept)
    res = allocate_block_resources(spec_of(x), "cuda", kept=kept)
    check(attend(x, g, res, blocks.cuda()), x, blocks)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_lists_in_any_order_repeated_and_past_the_length(kind):
    x = make([300, 1000, 64], 8, 2, 128, kind, seed=21)
    g = dev(x)
    blocks = torch.tensor([[[4, 0, 4, -1, 2], [99, 5, -3, 1, 0]],
                           [[15, 15, 15, 15, 15], [0, 16, 3, 2 ** 31 - 1, 1]],
                           [[-1, -1, -1, -1, -1], [7, 8, 9, 10, 11]]], dtype=torch.int32)
    res = allocate_block_resources(spec_of(x), "cuda", kept=8)
    out = attend(x, g, res, blocks.cuda())
    check(out, x, blocks)
    assert not out[2].any()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_pages_outside_the_cache_have_no_tokens(kind):
    x = make([700, 600], 8, 2, 128, kind, seed=22)
    x["tables"][0, 1], x["tables"][1, 0] = -5, x["k"].shape[0]
    g = dev(x)
    blocks = torch.arange(11, dtype=torch.int32).expand(2, 2, 11).contiguous()
    res = allocate_block_resources(spec_of(x), "cuda", kept=11)
    check(attend(x, g, res, blocks.cuda()), x, blocks)


def test_infinite_and_nan_keys_and_values_stay_in_their_rows():
    x = make([200, 200, 200], 4, 2, 64, torch.bfloat16, seed=23)
    page = [int(x["tables"][b, 0]) for b in range(3)]
    x["v"][page[0], 199, 0, 5] = float("inf")
    x["v"][page[1], 10, 1, 7] = float("nan")
    x["k"][page[2], 3, 0, 0] = float("nan")
    g = dev(x)
    blocks = torch.arange(4, dtype=torch.int32).expand(3, 2, 4).contiguous()
    res = allocate_block_resources(spec_of(x), "cuda", kept=4)
    out = attend(x, g, res, blocks.cuda()).cpu().float()
    assert (out[0, :2, 5] == float("inf")).all() and out[1, 2:, 7].isnan().all()
    assert out[2, :2].isnan().all()
    odd = torch.zeros_like(out, dtype=torch.bool)
    odd[0, :2, 5] = odd[1, 2:, 7] = odd[2, :2] = True
    assert out[~odd].isfinite().all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_an_infinite_value_of_probability_one(d):
    """Probabilities that a bf16 holds exactly: one, and a half and a quarter of equal scores."""
    x = make([1, 2, 4], 4, 1, d, torch.bfloat16, seed=25)
    for b in range(3):
        x["k"][int(x["tables"][b, 0])] = 0.0
        x["v"][int(x["tables"][b, 0]), 0, 0, 1] = float("inf")
        x["v"][int(x["tables"][b, 0]), 0, 0, d - 1] = -float("inf")
    g = dev(x)
    blocks = torch.zeros((3, 1, 1), dtype=torch.int32)
    out = attend(x, g, allocate_block_resources(spec_of(x), "cuda", kept=1), blocks.cuda()).cpu()
    assert (out[..., 1] == float("inf")).all() and (out[..., d - 1] == -float("inf")).all()
    assert out[..., 2:d - 1].isfinite().all() and out[..., 0].isfinite().all()


def test_scores_of_large_magnitude():
    """Maxima far from zero and far apart: the running maximum moves at every tile."""
    x = make([900, 900], 4, 1, 128, torch.bfloat16, seed=24)
    ramp = torch.linspace(-30, 30, 900)
    for b in range(2):
        for t in range(900):
            x["k"][x["tables"][b, t // 256], t % 256] *= float(ramp[t if b else 899 - t])
    g = dev(x)
    blocks = torch.arange(15, dtype=torch.int32).expand(2, 1, 15).contiguous()
    res = allocate_block_resources(spec_of(x), "cuda", kept=15)
    check(attend(x, g, res, blocks.cuda()), x, blocks)


def bounds_of(x, seed, integers=False):
    gen = torch.Generator().manual_seed(seed)
    pages, _, hkv, d = x["k"].shape
    shape = (pages, 4, hkv, 1, d)
    if integers:
        low = torch.randint(-2, 1, shape, generator=gen).float()
        return torch.cat([low, low + torch.randint(0, 2, shape, generator=gen)], 3).bfloat16()
    middle, spread = torch.randn(shape, generator=gen), torch.rand(shape, generator=gen) + 1
    return torch.cat([middle - spread, middle + spread], 3).bfloat16()


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lengths,kept,first,last", [
    ([1], 1, 0, 1), ([1, 0, 64, 65, 256, 257, 300], 3, 1, 1), ([700, 0, 2064, 1500], 9, 1, 1),
    ([5000], 7, 0, 3), ([5000, 4000], 40, 2, 1), ([6208], 2, 1, 1), ([640, 641], 10, 1, 1)],
    ids=str)
def test_select_blocks(lengths, kept, first, last, hq, hkv, d):
    x = make(lengths, hq, hkv, d, torch.bfloat16, seed=hq + kept)
    for integers in (False, True):     # True: scores of small integers, ties everywhere
        q = x["q"].float().round().bfloat16() if integers else x["q"]
        bounds = bounds_of(x, kept + hq, integers)
        res = allocate_block_resources(spec_of(x), "cuda", kept=kept)
        got = select_blocks(q.cuda(), bounds.cuda(), x["tables"].cuda(), x["lengths"].cuda(),
                            resources=res, first=first, last=last)
        assert torch.equal(got.cpu(), O.select(q, bounds, x["tables"], x["lengths"], kept, first,
                                               last))


def test_select_odd_scores():
    x = make([3000, 3000, 3000], 4, 2, 64, torch.bfloat16, seed=31)
    bounds = bounds_of(x, 31)
    at = lambda b, j: (int(x["tables"][b, j // 4]), j % 4)  # noqa: E731
    bounds[at(0, 30)][0, 1, 3] = float("nan")
    bounds[at(0, 7)][1, 0] = -float("inf")
    bounds[at(0, 9)][0, 1] = float("inf")
    x["q"][1] = 0.0                                   # every score equal: the first blocks
    x["q"][2, 0, 0] = float("nan")                    # every score of kv head 0 infinite
    x["q"][2, 3, 9] = -float("inf")                   # and of kv head 1
    res = allocate_block_resources(spec_of(x), "cuda", kept=6)
    got = select_blocks(x["q"].cuda(), bounds.cuda(), x["tables"].cuda(), x["lengths"].cuda(),
                        resources=res).cpu()
    assert torch.equal(got, O.select(x["q"], bounds, x["tables"], x["lengths"], 6))
    assert {9, 30} <= set(got[0, 0].tolist()) and 7 in got[0, 1].tolist()
    assert got[1, 0].tolist() == [0, 1, 2, 3, 4, 46] == got[2, 0].tolist() == got[2, 1].tolist()


def test_select_from_a_long_table():
    """70,000 tokens a sequence, most of one score, more blocks than a workgroup's threads."""
    x = dict(q=torch.ones((2, 4, 64), dtype=torch.bfloat16))
    pages = 274
    tables = torch.from_numpy(np.random.default_rng(1).permutation(2 * pages).astype(np.int32)
                              .reshape(2, pages))
    gen = torch.Generator().manual_seed(32)
    bounds = torch.randint(0, 2, (2 * pages, 4, 2, 1, 64), generator=gen).float()
    bounds = torch.cat([bounds, bounds], 3).bfloat16()
    lengths = torch.tensor([70001, 69000], dtype=torch.int32)
    res = allocate_block_resources(DecodeSpec(2, 4, 2, 64, pages * 256), "cuda", kept=500)
    got = select_blocks(x["q"].cuda(), bounds.cuda(), tables.cuda(), lengths.cuda(), resources=res)
    assert torch.equal(got.cpu(), O.select(x["q"], bounds, tables, lengths, 500))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_strided_queries_narrow_tables_and_part_batches(kind):
    x = make([700, 90, 1400], 8, 2, 128, kind, seed=41)
    g = dev(x)
    wide = torch.zeros((3, 10, 2, 8, 128), dtype=torch.bfloat16, device="cuda")
    wide[:, 3, 1] = g["q"]
    tables = torch.full((3, 30), 10 ** 6, dtype=torch.int32, device="cuda")
    tables[:, 4:4 + g["tables"].shape[1]] = g["tables"]
    g = dict(g, q=wide[:, 3, 1], tables=tables[:, 4:4 + g["tables"].shape[1]])
    blocks = random_blocks(x, 9, seed=41)
    res = allocate_block_resources(DecodeSpec(5, 8, 2, 128, 4096), "cuda", kept=9)
    res.out.fill_(7.0)
    res.blocks.fill_(-9)
    out = attend(x, g, res, blocks.cuda())
    check(out, x, blocks)
    assert (res.out[3:] == 7.0).all()
    bounds = bounds_of(x, 41)
    got = select_blocks(g["q"], bounds.cuda(), g["tables"], g["lengths"], resources=res)
    assert torch.equal(got.cpu(), O.select(x["q"], bounds, x["tables"], x["lengths"], 9))
    assert (res.blocks[3:] == -9).all()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_a_sequence_has_its_bits_in_every_batch_of_a_bucket(kind):
    lengths = [700, 90, 5000, 64, 0, 333]
    x = make(lengths, 8, 2, 128, kind, seed=42)
    g = dev(x)
    res = allocate_block_resources(DecodeSpec(8, 8, 2, 128, 5120), "cuda", kept=20)
    blocks = random_blocks(x, 20, seed=42).cuda()
    whole = attend(x, g, res, blocks).clone()
    part = {n: t[:5] if n in ("q", "tables", "lengths") else t for n, t in g.items()}
    assert torch.equal(attend(x, part, res, blocks[:5]), whole[:5])


def test_cache_offsets_past_32_bits():
    """The last pages of a cache of more than 2^32 bytes."""
    pages = 2 ** 32 // (256 * 8 * 256) + 8
    k, v = (torch.empty((pages, 256, 8, 256), dtype=torch.uint8, device="cuda").view(E4M3)
            for _ in range(2))
    x = make([700], 16, 8, 256, E4M3, seed=43, spare=0)
    for c, small in ((k, x["k"]), (v, x["v"])):
        c.view(torch.uint8)[-3:] = small.view(torch.uint8).cuda()
    g = dev({n: t for n, t in x.items() if n not in ("k", "v")})
    g.update(k=k, v=v, tables=g["tables"] + (pages - 3))
    check(attend(x, g, allocate_block_resources(spec_of(x), "cuda")), x)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_prompt_and_steps_through_append_select_and_attend(kind):
    """A serving loop: two prompts appended, then captured steps (append, select, attend) whose
    outputs and choices equal the plain forms' on the cache as it then is."""
    hq, hkv, d, half, kept = 8, 2, 128, 32, 6
    gen = torch.Generator().manual_seed(51)
    tables = torch.tensor([[4, 0, 5], [1, 3, 2]], dtype=torch.int32, device="cuda")
    cache = [torch.full((6, 256, hkv, d), float("nan"), device="cuda").to(kind) for _ in range(2)]
    bounds = allocate_bounds(cache[0])
    rope = rope_cache(768, 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half))
    scales = dict(k_scale=torch.tensor([0.01, 0.02], device="cuda"),
                  v_scale=torch.tensor([0.012, 0.009], device="cuda")) if kind == E4M3 else {}
    lens = [510, 637]

    def rows(n):
        fused = torch.randn((n, (hq + 2 * hkv) * d), generator=gen).bfloat16().cuda()
        return [t.view(n, -1, d) for t in fused.split([hq * d, hkv * d, hkv * d], 1)]

    def slots(b, at):
        return tables[b, at // 256] * 256 + (at % 256).int()

    for b, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        append_kv(*rows(n), at, rope, *cache, slots(b, at), bounds=bounds, **scales)
    res = allocate_block_resources(DecodeSpec(2, hq, hkv, d, 768), "cuda", kept=kept)
    x = dict(zip("qkv", rows(2)), positions=torch.zeros(2, dtype=torch.long, device="cuda"),
             slots=torch.full((2,), -1, dtype=torch.int32, device="cuda"),
             lengths=torch.zeros(2, dtype=torch.int32, device="cuda"))

    def step():
        q = append_kv(x["q"], x["k"], x["v"], x["positions"], rope, *cache, x["slots"],
                      bounds=bounds, **scales)
        blocks = select_blocks(q, bounds, tables, x["lengths"], resources=res)
        return q, blocks, sparse_decode(q, *cache, tables, x["lengths"], blocks, resources=res,
                                        **scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, blocks, out = step()
    for i in range(5):
        new = rows(2)
        for name, t in zip("qkv", new):
            x[name].copy_(t)
        at = torch.tensor(lens, device="cuda") + i
        x["positions"].copy_(at)
        x["slots"].copy_(slots(torch.arange(2, device="cuda"), at))
        x["lengths"].copy_(at + 1)
        graph.replay()
        torch.cuda.synchronize()
        full = (at + 1) // 64
        for b in range(2):
            for j in range(int(full[b])):
                page, part = int(tables[b, j // 4]), j % 4
                assert torch.equal(bounds[page, part].cpu(), O.block_bounds(
                    cache[0][page, 64 * part:64 * part + 64].cpu()))
        host = dict(q=q.cpu(), k=cache[0].cpu(), v=cache[1].cpu(), tables=tables.cpu(),
                    lengths=x["lengths"].cpu(),
                    k_scale=scales["k_scale"].cpu() if scales else None,
                    v_scale=scales["v_scale"].cpu() if scales else None)
        assert torch.equal(blocks.cpu(), O.select(host["q"], bounds.cpu(), host["tables"],
                                                  host["lengths"], kept))
        check(out, host, blocks.cpu())


def test_other_streams_and_refused_arguments():
    x = make([700, 90], 8, 2, 128, E4M3, seed=61)
    g = dev(x)
    res = allocate_block_resources(spec_of(x), "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = attend(x, g, res)
    torch.cuda.current_stream().wait_stream(side)
    check(out, x)
    blocks = torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda")
    listed = allocate_block_resources(spec_of(x), "cuda", kept=3)
    bad = [(dict(g, q=g["q"].float()), None, "BF16 Q"), (dict(g, k=g["k"].float()), None, "float8"),
           (dict(g, v=g["v"].view(torch.uint8)), None, "caches"),
           (dict(g, lengths=g["lengths"].long()), None, "int32"),
           (dict(g, q=g["q"][:, :4]), None, "query_heads"),
           (dict(g, k_scale=torch.ones(3, device="cuda")), None, "scales"),
           (dict(g, k_scale=torch.ones(2)), None, "scales"),
           (dict(g, tables=g["tables"].t().contiguous().t()), None, "contiguous rows"),
           (g, blocks.long(), "int32"), (g, blocks.expand(2, 2, 3)[:, :1], "blocks"),
           (g, torch.zeros((2, 2, 4), dtype=torch.int32, device="cuda"), "at most kept")]
    for args, chosen, message in bad:
        with pytest.raises(ValueError, match=message):
            attend(x, args, res if chosen is None else listed, chosen)
    with pytest.raises(ValueError, match="sized for a list"):
        attend(x, g, listed)
    with pytest.raises(ValueError, match="kept="):
        attend(x, g, res, blocks)
    bounds = torch.zeros((g["k"].shape[0], 4, 2, 2, 128), dtype=torch.bfloat16, device="cuda")
    for first, last, kept in ((0, 0, 3), (2, 2, 3), (-1, 1, 3)):
        with pytest.raises(ValueError, match="kept blocks"):
            select_blocks(g["q"], bounds, g["tables"], g["lengths"], resources=listed, first=first,
                          last=last)
    with pytest.raises(ValueError, match="bounds"):
        select_blocks(g["q"], bounds.float(), g["tables"], g["lengths"], resources=listed)
    with pytest.raises(ValueError, match="finite"):
        fp8_decode(g["q"], g["k"], g["v"], g["tables"], g["lengths"], resources=res,
                   scale=float("inf"))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 8, 9, 16, 17, 33, 64, 100, 128])
def test_every_split_count_gives_the_same_attention(splits, kind):
    """Splits set by hand: more than the plan's and fewer, so that a wavefront's tiles are none,
    one, or more than it looks up at once (64)."""
    lengths = [0, 1, 33, 700, 9300]
    x = make(lengths, 8, 2, 128, kind, seed=71)
    g = dev(x)
    kept = 146
    blocks = torch.arange(kept, dtype=torch.int32).expand(5, 2, kept).contiguous()
    res = allocate_block_resources(spec_of(x), "cuda", kept=kept)
    res._splits[5, kind] = splits
    res.partials = torch.full((5 * 8 * splits * 128,), float("nan"), device="cuda")
    res.sums = torch.full((5 * 8 * splits * 2,), float("nan"), device="cuda")
    check(attend(x, g, res, blocks.cuda()), x, blocks)


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.3])
def test_scales_of_the_scores(scale):
    x = make([500, 70], 8, 2, 128, E4M3, seed=72)
    g = dev(x)
    res = allocate_block_resources(spec_of(x), "cuda")
    out = fp8_decode(g["q"], g["k"], g["v"], g["tables"], g["lengths"], resources=res, scale=scale,
                     k_scale=g["k_scale"], v_scale=g["v_scale"])
    check(out, x, scale=scale)


def test_select_from_more_blocks_than_a_workgroup_holds():
    pages = 590
    tables = torch.from_numpy(np.random.default_rng(2).permutation(pages).astype(np.int32)[None])
    gen = torch.Generator().manual_seed(73)
    lengths = torch.tensor([150_001], dtype=torch.int32)
    res = allocate_block_resources(DecodeSpec(1, 4, 2, 64, pages * 256), "cuda", kept=300)
    for integers in (False, True):
        shape = (pages, 4, 2, 1, 64)
        low = torch.randint(-2, 2, shape, generator=gen).float() if integers \
            else torch.randn(shape, generator=gen)
        bounds = torch.cat([low, low + torch.rand(shape, generator=gen).round()], 3).bfloat16()
        q = torch.randn((1, 4, 64), generator=gen)
        q = (q.round() if integers else q).bfloat16()
        got = select_blocks(q.cuda(), bounds.cuda(), tables.cuda(), lengths.cuda(), resources=res)
        assert torch.equal(got.cpu(), O.select(q, bounds, tables, lengths, 300))


def test_two_graphs_share_their_resources():
    """Captured with the same workspaces, replayed in turn on one stream."""
    x = make([3000, 1200], 8, 2, 128, torch.bfloat16, seed=74)
    g = dev(x)
    bounds = bounds_of(x, 74).cuda()
    res = allocate_block_resources(spec_of(x), "cuda", kept=8)
    graphs = []
    for i in range(2):
        q = g["q"].clone() if i else g["q"].neg()
        args = dict(g, q=q)

        def step():
            blocks = select_blocks(q, bounds, g["tables"], g["lengths"], resources=res)
            return blocks.clone(), attend(x, args, res, blocks).clone()

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        want = [t.clone() for t in want]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got, want, q))      # the graph reads q
    assert not torch.equal(graphs[0][2][0], graphs[1][2][0])
    for i in (0, 1, 1, 0, 0, 1):
        graph, got, want, _ = graphs[i]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
