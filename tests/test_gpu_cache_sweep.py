"""Seeded random calls of the cache operators: any head layout, lengths, table widths, list
lengths, splits of a capacity far above the lengths, page sizes and row orders."""
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
from test_gpu_append import bits, expected
from test_gpu_blocks import bounds_of, check, dev, make

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("seed", range(40))
def test_random_steps(seed):
    rng = np.random.default_rng([7, seed])
    hkv, dim = int(rng.integers(1, 6)), int(rng.choice([64, 128, 256]))
    hq = hkv * int(rng.choice([1, 2, 3, 4, 5, 8, 16, 17, 20]))
    kind = E4M3 if rng.random() < 0.5 else torch.bfloat16
    batch, high = int(rng.integers(1, 7)), int(np.exp(rng.uniform(0, np.log(6000))))
    lengths = [int(n) for n in rng.integers(0, high + 1, batch)]
    x = make(lengths, hq, hkv, dim, kind, seed=seed, spare=int(rng.integers(1, 4)),
             scales=rng.random() < 0.8)
    g = dev(x)
    capacity = x["tables"].shape[1] * 256 * int(rng.choice([1, 1, 3, 40]))
    spec = DecodeSpec(batch + int(rng.integers(0, 3)), hq, hkv, dim, capacity)
    print(f"seed {seed}: Hq {hq} Hkv {hkv} D {dim} {kind} capacity {capacity} {lengths}", flush=True)
    scale = dim ** -0.5 * float(rng.choice([1.0, 0.25, 4.0]))
    args = (g["q"], g["k"], g["v"], g["tables"], g["lengths"])
    more = dict(scale=scale, k_scale=g["k_scale"], v_scale=g["v_scale"])
    if kind == E4M3:
        out = fp8_decode(*args, resources=allocate_block_resources(spec, "cuda"), **more)
        check(out, x, scale=scale)
    kept = int(rng.integers(1, 60))
    first = int(rng.integers(0, min(3, kept)))
    last = int(rng.integers(1, min(3, kept - first) + 1))
    bounds = bounds_of(x, seed, integers=rng.random() < 0.5)
    res = allocate_block_resources(spec, "cuda", kept=kept)
    blocks = select_blocks(g["q"], bounds.cuda(), g["tables"], g["lengths"], resources=res,
                           first=first, last=last)
    assert torch.equal(blocks.cpu(), O.select(x["q"], bounds, x["tables"], x["lengths"], kept,
                                              first, last))
    listed = blocks.clone()
    if rng.random() < 0.5:
        listed = listed[:, :, torch.from_numpy(rng.permutation(kept)).cuda()].contiguous()
    out = sparse_decode(*args, listed, resources=res, **more)
    check(out, x, listed.cpu(), scale=scale)


@pytest.mark.parametrize("seed", range(40))
def test_random_appends(seed):
    rng = np.random.default_rng([8, seed])
    hkv, dim = int(rng.integers(1, 6)), int(rng.choice([64, 128, 256]))
    hq = int(rng.integers(0, 20))
    kind = E4M3 if rng.random() < 0.5 else torch.bfloat16
    half = 8 * int(rng.integers(0, dim // 16 + 1))
    interleaved = bool(rng.random() < 0.4)
    with_bounds = rng.random() < 0.7
    page = 64 * int(rng.integers(1, 5)) if with_bounds else int(rng.integers(1, 300))
    pages = -(-1200 // page)
    n = int(np.exp(rng.uniform(0, np.log(1000))))
    start = int(rng.integers(0, pages * page - n + 1))
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen).bfloat16().cuda()  # noqa: E731
    fused = normal(n, (hq + 2 * hkv) * dim + 8)[:, :-8]
    q, k, v = (t.view(n, -1, dim) for t in fused.split([hq * dim, hkv * dim, hkv * dim], 1))
    order = np.arange(start, start + n) if rng.random() < 0.5 else \
        rng.permutation(pages * page)[:n]
    order[rng.random(n) < 0.05] = -1
    scale = [(torch.rand(hkv, generator=gen) * 0.02 + 0.004).cuda()
             if kind == E4M3 and rng.random() < 0.8 else None for _ in range(2)]
    x = dict(q=q, k=k, v=v, positions=torch.from_numpy(rng.integers(0, 600, n)).cuda(),
             rope=rope_cache(600, 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half))
             if half else None, slots=torch.from_numpy(order.astype(np.int32)).cuda(),
             k_scale=scale[0], v_scale=scale[1],
             k_cache=normal(pages, page, hkv, dim).to(kind),
             v_cache=normal(pages, page, hkv, dim).to(kind))
    print(f"seed {seed}: N {n} Hq {hq} Hkv {hkv} D {dim} {kind} half {half} page {page}", flush=True)
    want_q, k_bits, v_bits, _ = expected(x, interleaved)
    bounds = torch.full_like(allocate_bounds(x["k_cache"]), 7.0) if with_bounds else None
    out = append_kv(q if hq else None, k, v, x["positions"], x["rope"], x["k_cache"], x["v_cache"],
                    x["slots"], interleaved=interleaved, k_scale=scale[0], v_scale=scale[1],
                    bounds=bounds)
    if hq:
        assert torch.equal(bits(out), bits(want_q))
    assert torch.equal(bits(x["k_cache"]), k_bits) and torch.equal(bits(x["v_cache"]), v_bits)
    if with_bounds:
        keys = x["k_cache"].cpu().view(-1, 64, hkv, dim)
        want = torch.full((len(keys), hkv, 2, dim), 7.0)
        for slot in order.tolist():
            if slot >= 0 and slot % 64 == 63:
                want[slot // 64] = O.block_bounds(keys[slot // 64]).float()
        assert torch.equal(bounds.cpu().view(want.shape).float(), want)
