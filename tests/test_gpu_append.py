"""append_kv and block_bounds against the plain form in float32 with every operation rounded
by itself (the kernel's outputs are the same bits) and in 64 bits (half a step of the output's
type, plus the three float32 roundings before it)."""
import numpy as np
import pytest
import torch

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X GPU", allow_module_level=True)

from oracle import blocks as O
from paged_decode.kv_append import allocate_bounds, append_kv, block_bounds, rope_cache

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
KINDS = [torch.bfloat16, E4M3]


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, dtype=torch.float32).to(torch.bfloat16)


def bits(t):
    return t.contiguous().view(torch.uint8 if t.dtype == E4M3 else torch.int16).cpu()


def make(n, hq, hkv, d, half, kind, seed, pages=3, page=256, start=None):
    """A fused projection's rows, positions and slots in order from `start` (random: None)."""
    gen = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    fused = normal(gen, n, (hq + 2 * hkv) * d)
    q, k, v = (t.view(n, -1, d) for t in fused.cuda().split([hq * d, hkv * d, hkv * d], 1))
    slots = (rng.permutation(pages * page)[:n] if start is None
             else np.arange(start, start + n)).astype(np.int32)
    rope = rope_cache(600, 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)) \
        if half else None
    scale = [(torch.rand(hkv, generator=gen) * 0.02 + 0.004).cuda() if kind == E4M3 else None
             for _ in range(2)]
    caches = [normal(gen, pages, page, hkv, d).to(kind).cuda() for _ in range(2)]
    return dict(q=q, k=k, v=v, positions=torch.from_numpy(rng.integers(0, 600, n)).cuda(),
                rope=rope, slots=torch.from_numpy(slots).cuda(), k_scale=scale[0],
                v_scale=scale[1], k_cache=caches[0], v_cache=caches[1])


def call(x, **more):
    return append_kv(x["q"], x["k"], x["v"], x["positions"], x["rope"], x["k_cache"], x["v_cache"],
                     x["slots"], k_scale=x["k_scale"], v_scale=x["v_scale"], **more)


def host(x):
    return {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in x.items()}


def expected(x, interleaved=False):
    """(q, k_cache, v_cache, rotated keys in 64 bits) from the inputs, on the host."""
    h = host(x)
    turn = lambda t, kind: (t.to(kind) if h["rope"] is None else  # noqa: E731
                            O.rotated(t, h["positions"], h["rope"], interleaved, kind))
    live = (h["slots"] >= 0) & (h["slots"] < h["k_cache"].shape[0] * h["k_cache"].shape[1])
    caches = []
    for name, rows in (("k", turn(h["k"], torch.float32)), ("v", h["v"].float())):
        cache = h[name + "_cache"].clone()
        flat = bits(cache).view(-1, *cache.shape[2:])
        flat[h["slots"][live].long()] = bits(O.stored(rows, h[name + "_scale"], cache.dtype))[live]
        caches.append(flat.view(cache.shape))
    return turn(h["q"], torch.float32).to(torch.bfloat16), *caches, turn(h["q"], torch.float64)


@pytest.mark.parametrize("kind", KINDS, ids=["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,d,half,interleaved", [
    (16, 4, 256, 32, False), (32, 8, 128, 64, False), (16, 16, 64, 32, True),
    (5, 1, 128, 8, True), (8, 2, 256, 128, True), (3, 3, 64, 8, False), (34, 2, 64, 24, False)])
@pytest.mark.parametrize("n", [1, 3, 37, 300])
def test_rotated_append(n, hq, hkv, d, half, interleaved, kind):
    x = make(n, hq, hkv, d, half, kind, seed=n + d + hq)
    q, k_bits, v_bits, exact = expected(x, interleaved)
    out = call(x, interleaved=interleaved)
    assert torch.equal(bits(out), bits(q))
    assert torch.equal(bits(x["k_cache"]), k_bits) and torch.equal(bits(x["v_cache"]), v_bits)
    # Against 64 bits: two float32 products and their sum, then the rounding to bf16.
    size = host(x)["q"].double().abs().amax(-1, keepdim=True) * 2
    assert ((out.cpu().double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 2.0 ** -22 * size).all()


@pytest.mark.parametrize("kind", KINDS, ids=["bf16", "e4m3"])
def test_skipped_slots_and_positions_outside_the_table(kind):
    x = make(64, 8, 2, 128, 32, kind, seed=5)
    x["slots"][[0, 9, 63]] = torch.tensor([-1, -7, 3 * 256], dtype=torch.int32, device="cuda")
    q, k_bits, v_bits, _ = expected(x)
    out = call(x)
    assert torch.equal(bits(out), bits(q))
    assert torch.equal(bits(x["k_cache"]), k_bits) and torch.equal(bits(x["v_cache"]), v_bits)
    y = make(64, 8, 2, 128, 32, kind, seed=6)
    far = [3, 40]
    y["positions"][far[0]], y["positions"][far[1]] = -1, 600
    h = dict(y, positions=y["positions"].clamp(0, 599), slots=y["slots"].clone())
    h["slots"][far] = -1
    q, k_bits, v_bits, _ = expected(h)
    out = call(y).cpu()
    assert out[far][..., :64].isnan().all() and torch.equal(out[far][..., 64:], q[far][..., 64:])
    rest = [i for i in range(64) if i not in far]
    assert torch.equal(bits(out[rest]), bits(q[rest]))
    assert torch.equal(bits(y["k_cache"]), k_bits) and torch.equal(bits(y["v_cache"]), v_bits)


@pytest.mark.parametrize("kind", KINDS, ids=["bf16", "e4m3"])
def test_values_at_the_ends_of_the_range(kind):
    x = make(32, 2, 2, 64, 0, kind, seed=8)
    special = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 3.0e38, -3.0e38,
                            1e-38, 2.0 ** -9, 3 * 2.0 ** -10, 2.0 ** -10, 448.0, 464.0, 465.0,
                            -447.9, 17.0, 19.0], dtype=torch.bfloat16, device="cuda")
    x["k_scale"] = x["v_scale"] = torch.ones(2, device="cuda") if kind == E4M3 else None
    for name in ("q", "k", "v"):
        x[name] = x[name].clone()
        x[name][:17, 0, 0] = special
        x[name][:17, 1, 33] = special.flip(0)
    q, k_bits, v_bits, _ = expected(x)
    out = call(x)
    nan = q.isnan()
    assert torch.equal(out.cpu().isnan(), nan) and torch.equal(bits(out)[~nan], bits(q)[~nan])
    for got, want in ((x["k_cache"], k_bits), (x["v_cache"], v_bits)):
        got, want = got.cpu(), want.view(kind)
        nan = want.float().isnan()
        assert torch.equal(got.float().isnan(), nan)
        assert torch.equal(bits(got)[~nan], bits(want)[~nan])


def test_without_queries_without_rotation_and_in_place():
    x = make(70, 8, 2, 128, 64, torch.bfloat16, seed=9)
    q, k_bits, v_bits, _ = expected(x)
    assert append_kv(None, x["k"], x["v"], x["positions"], x["rope"], x["k_cache"], x["v_cache"],
                     x["slots"]) is None
    assert torch.equal(bits(x["k_cache"]), k_bits) and torch.equal(bits(x["v_cache"]), v_bits)
    out = call(x, out=x["q"])       # rows of the fused projection, rotated where they are
    assert out is x["q"] and torch.equal(bits(out), bits(q))
    y = make(70, 8, 2, 128, 0, E4M3, seed=10)
    _, k_bits, v_bits, _ = expected(y)
    out = append_kv(y["q"], y["k"], y["v"], None, None, y["k_cache"], y["v_cache"], y["slots"],
                    k_scale=y["k_scale"], v_scale=y["v_scale"])
    assert torch.equal(bits(out), bits(y["q"]))
    assert torch.equal(bits(y["k_cache"]), k_bits) and torch.equal(bits(y["v_cache"]), v_bits)
    empty = append_kv(y["q"][:0], y["k"][:0], y["v"][:0], None, None, y["k_cache"], y["v_cache"],
                      y["slots"][:0], bounds=allocate_bounds(y["k_cache"]))
    assert empty.shape == (0, 8, 128)


@pytest.mark.parametrize("kind", KINDS, ids=["bf16", "e4m3"])
@pytest.mark.parametrize("hkv,d", [(1, 64), (3, 128), (2, 256), (8, 64)])
@pytest.mark.parametrize("n,start", [(1, 62), (1, 63), (1, 64), (64, 0), (63, 65), (500, 130)])
def test_bounds_of_full_blocks(n, start, hkv, d, kind):
    x = make(n, 4 * hkv, hkv, d, d // 4, kind, seed=n + start + d, start=start)
    bounds = torch.full_like(allocate_bounds(x["k_cache"]), 77.0)
    call(x, bounds=bounds)
    keys = x["k_cache"].cpu().view(-1, 64, hkv, d)
    want = torch.full((len(keys), hkv, 2, d), 77.0, dtype=torch.bfloat16)
    for j in range(len(keys)):
        if start <= 64 * j + 63 < start + n:
            want[j] = O.block_bounds(keys[j])
    assert torch.equal(bounds.cpu().view(want.shape).float(), want.float())
    again = torch.full_like(bounds, 77.0)
    block_bounds(x["k_cache"], x["slots"], again)
    assert torch.equal(bits(again), bits(bounds))


@pytest.mark.parametrize("kind", KINDS, ids=["bf16", "e4m3"])
def test_bounds_of_many_ends_at_once_and_of_nan_keys(kind):
    x = make(12 * 4, 4, 2, 128, 16, kind, seed=3, pages=12)
    ends = torch.from_numpy(np.random.default_rng(3).permutation(48).astype(np.int32)).cuda()
    x["slots"] = ends * 64 + 63
    x["k"] = x["k"].clone()
    x["k"][5, 1, 100] = float("nan")
    x["k"][6, 0, 0] = float("inf")
    bounds = allocate_bounds(x["k_cache"])
    call(x, bounds=bounds)
    keys = x["k_cache"].cpu().view(-1, 64, 2, 128)
    want = torch.stack([O.block_bounds(block) for block in keys]).float()
    got = bounds.cpu().view(want.shape).float()
    assert torch.equal(got.isnan(), want.isnan()) and want.isnan().sum() == 2
    assert torch.equal(got.nan_to_num(1.25), want.nan_to_num(1.25))


def test_slots_past_two_gigabytes_of_cache():
    """Slot offsets pass 32 bits."""
    pages = 2 ** 31 // (256 * 8 * 256) + 2                # elements past 2^31
    cache = [torch.zeros((pages, 256, 8, 256), dtype=torch.bfloat16, device="cuda")
             for _ in range(2)]
    x = make(3, 8, 8, 256, 32, torch.bfloat16, seed=4)
    last = pages * 256
    x.update(k_cache=cache[0], v_cache=cache[1],
             slots=torch.tensor([last - 1, last - 2, 0], dtype=torch.int32, device="cuda"))
    bounds = allocate_bounds(cache[0])
    call(x, bounds=bounds)
    small = dict(x, k_cache=torch.zeros_like(cache[0][:1]), v_cache=torch.zeros_like(cache[1][:1]),
                 slots=torch.tensor([255, 254, 0], dtype=torch.int32, device="cuda"))
    call(small)
    for a, b in ((cache[0], small["k_cache"]), (cache[1], small["v_cache"])):
        assert torch.equal(a[-1, 254:], b[0, 254:]) and torch.equal(a[0, 0], b[0, 0])
        assert int(torch.count_nonzero(a[1:-1])) == 0
    assert torch.equal(bounds[-1, 3].cpu(), O.block_bounds(cache[0][-1, 192:].cpu()))


@pytest.mark.parametrize("kind", KINDS, ids=["bf16", "e4m3"])
def test_captured_steps_replay_with_new_rows(kind):
    x = make(48, 8, 2, 128, 64, kind, seed=11, pages=2)
    bounds = allocate_bounds(x["k_cache"])
    out = torch.empty_like(x["q"].contiguous())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(x, bounds=bounds, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(x, bounds=bounds, out=out)
    for seed in range(12, 16):
        y = make(48, 8, 2, 128, 64, kind, seed=seed, pages=2, start=None if seed % 2 else 80)
        for name in ("q", "k", "v", "positions", "slots"):
            x[name].copy_(y[name])
        y.update(k_cache=x["k_cache"].clone(), v_cache=x["v_cache"].clone(),
                 k_scale=x["k_scale"], v_scale=x["v_scale"])
        eager_bounds = bounds.clone()
        graph.replay()
        torch.cuda.synchronize()
        eager = call(y, bounds=eager_bounds)
        assert torch.equal(bits(out), bits(eager))
        assert torch.equal(bits(x["k_cache"]), bits(y["k_cache"]))
        assert torch.equal(bits(x["v_cache"]), bits(y["v_cache"]))
        assert torch.equal(bits(bounds), bits(eager_bounds))


@pytest.mark.parametrize("kind", KINDS, ids=["bf16", "e4m3"])
@pytest.mark.parametrize("half,interleaved", [(0, False), (32, False), (64, True)])
@pytest.mark.parametrize("n", [200, 513, 700])
def test_bounds_of_rows_in_any_order(n, half, interleaved, kind):
    """Whole and part blocks with their rows permuted, some rows not written: padded slots and
    positions outside the table, whose keys stay the cache's own."""
    x = make(n, 8, 2, 128, half, kind, seed=n + half, start=70)
    order = torch.from_numpy(np.random.default_rng(n).permutation(n)).cuda()
    for name in ("q", "k", "v", "positions", "slots"):
        x[name] = x[name][order]
    x["slots"][5] = -1
    if half:
        x["positions"][[17, 30]] = torch.tensor([-1, 600], device="cuda")
    bounds = torch.full_like(allocate_bounds(x["k_cache"]), 77.0)
    call(x, bounds=bounds, interleaved=interleaved)
    torch.cuda.synchronize()
    keys = x["k_cache"].cpu().view(-1, 64, 2, 128)
    want = torch.full((len(keys), 2, 2, 128), 77.0, dtype=torch.bfloat16)
    for slot in x["slots"].tolist():
        if slot >= 0 and slot % 64 == 63:
            want[slot // 64] = O.block_bounds(keys[slot // 64])
    assert torch.equal(bounds.cpu().view(want.shape).float(), want.float())


def test_one_row_of_any_stride():
    x = make(1, 8, 2, 128, 64, torch.bfloat16, seed=31)
    q, k_bits, v_bits, _ = expected(x)
    for name in ("q", "k", "v"):
        x[name] = torch.as_strided(x[name].contiguous(), x[name].shape, (3, 128, 1))
    out = call(x)
    assert torch.equal(bits(out), bits(q))
    assert torch.equal(bits(x["k_cache"]), k_bits) and torch.equal(bits(x["v_cache"]), v_bits)


def test_refused_tensors():
    x = make(4, 8, 2, 128, 64, E4M3, seed=32)
    bounds = allocate_bounds(x["k_cache"])
    cases = [(dict(k=x["k"].float()), "BF16"), (dict(v=x["v"][:3]), "shape"),
             (dict(q=x["q"].transpose(1, 2)), "head_dim|heads"), (dict(q=x["q"].float()), "BF16"),
             (dict(k=x["k"].transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
             (dict(slots=x["slots"].long()), "int32"), (dict(slots=x["slots"][:3]), "one entry"),
             (dict(positions=x["positions"].int()), "int64"), (dict(slots=x["slots"].cpu()), "device"),
             (dict(rope=x["rope"].double()), "rope"), (dict(rope=x["rope"].transpose(0, 1)), "rope"),
             (dict(k_cache=x["k_cache"].float()), "float8"),
             (dict(k_cache=x["k_cache"].view(torch.uint8)), "float8"),
             (dict(k_cache=x["k_cache"][:, :, :1]), "heads"), (dict(v_cache=x["v_cache"][:1]), "heads"),
             (dict(k_scale=torch.ones(3, device="cuda")), "scales"),
             (dict(v_scale=torch.ones(2)), "scales"),
             (dict(k_cache=x["k_cache"].bfloat16(), v_cache=x["v_cache"].bfloat16()), "scales")]
    for change, message in cases:
        with pytest.raises(ValueError, match=message):
            call(dict(x, **change))
    for bad in (bounds.float(), bounds[:2], bounds.transpose(2, 3)):
        with pytest.raises(ValueError, match="bounds"):
            call(x, bounds=bad)
    with pytest.raises(ValueError, match="rows"):
        call(x, out=torch.empty((3, 8, 128), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="needs a query"):
        call(dict(x, q=None), out=x["q"])
    with pytest.raises(ValueError, match="no gradient"):
        call(dict(x, k=x["k"].clone().requires_grad_()))
    with pytest.raises(ValueError, match="multiple of 8"):
        call(dict(x, rope=x["rope"][:, :12].contiguous()))
    with pytest.raises(ValueError, match="needs positions"):
        call(dict(x, positions=None))


def test_quotients_at_the_midpoints_of_e4m3():
    """The stored value is the rounded division's: products of a scale with the midpoints and
    values of e4m3, and the floats next to them, through a rotation by (cos, 0)."""
    n, d = 512, 64
    rng = np.random.default_rng(33)
    grid = torch.arange(127, dtype=torch.uint8).view(E4M3).float()
    grid = torch.cat([grid, (grid[1:] + grid[:-1]) / 2])
    scale = torch.tensor([0.0123, 3.0, 1e-6, 7.7e8], dtype=torch.float32)
    pick = grid[torch.from_numpy(rng.integers(0, len(grid), (4, n, d // 2)))]
    near = torch.from_numpy(rng.integers(-2, 3, (4, n, d // 2)).astype(np.int32))
    for h in range(4):                 # one scale at a time, as every head's keys are one
        x = pick[h] * scale[h]
        x = (x.view(torch.int32) + near[h] * (x > 0)).view(torch.float32)
        rope = torch.stack([x, torch.zeros_like(x)], -1).cuda()              # [n, d / 2, 2]
        ones = torch.cat([torch.ones(n, 1, d // 2), torch.zeros(n, 1, d // 2)], 2)
        k = ones.bfloat16().cuda()
        cache = [torch.zeros((2, 256, 1, d), device="cuda").to(E4M3) for _ in range(2)]
        at = torch.arange(n, device="cuda")
        append_kv(None, k, k, at, rope, *cache, at.int(), k_scale=scale[h:h + 1].cuda())
        want = O.stored(x[:, None], scale[h:h + 1], E4M3)
        assert torch.equal(bits(cache[0]).view(n, d)[:, :d // 2], bits(want)[:, 0])
