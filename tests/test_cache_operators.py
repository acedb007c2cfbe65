"""Host side of the cache operators without a GPU: refusals before any launch, plans, and the
64-bit forms on small cases worked out by hand."""
import math

import pytest
import torch

from oracle import blocks as O
from paged_decode import _native
from paged_decode.block_decode import allocate_block_resources
from paged_decode.kv_append import allocate_bounds, append_kv, block_bounds, rope_cache
from paged_decode.spec import DecodeSpec

BF16 = torch.bfloat16


def test_host_tensors_are_refused():
    rows, cache = torch.zeros((3, 2, 64), dtype=BF16), torch.zeros((2, 256, 2, 64), dtype=BF16)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        append_kv(rows, rows, rows, None, None, cache, cache.clone(), slots)
    with pytest.raises(ValueError, match="CUDA device"):
        block_bounds(cache, slots, allocate_bounds(cache))
    with pytest.raises(ValueError, match="CUDA"):
        allocate_block_resources(DecodeSpec(1, 8, 2, 64, 256), "cpu")
    with pytest.raises(ValueError, match="whole blocks"):
        allocate_bounds(torch.zeros((2, 100, 2, 64), dtype=BF16))


@pytest.mark.parametrize("change,message", [
    (dict(head_dim=96), b"head_dim"), (dict(kv_heads=0), b"heads"), (dict(half=12), b"multiple of 8"),
    (dict(half=40), b"at most head_dim"), (dict(half=-8), b"multiple of 8"),
    (dict(cache_type=2), b"cache type"), (dict(slots=0), b"2^31 slots"),
    (dict(slots=2 ** 31 + 1), b"2^31 slots"), (dict(slots=100, bounds=64), b"whole blocks"),
    (dict(rows=-1), b"non-negative"), (dict(k=0), b"null"), (dict(rope=0), b"null"),
    (dict(q_out=0), b"null"), (dict(k=24), b"aligned"), (dict(k_stride=4), b"strides"),
    (dict(q_out_stride=64), b"strides"), (dict(rows=2 ** 30), b"grid")])
def test_append_arguments(change, message):
    x = dict(q=64, q_stride=512, k=64, k_stride=128, v=64, v_stride=128, positions=64, rope=64,
             max_positions=10, half=32, interleaved=0, q_out=64, q_out_stride=512, k_cache=64,
             v_cache=64, cache_type=0, slots=256, mapping=64, k_scale=0, v_scale=0, bounds=0, rows=4,
             heads=8, kv_heads=2, head_dim=64, stream=0)
    x.update(change)
    assert _native.lib().pd_append_kv(*x.values()) == _native.PD_EINVAL
    assert message in _native.lib().pd_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(head_dim=80), b"head_dim"), (dict(heads=9), b"divisible"), (dict(width=0), b"table width"),
    (dict(pages=0), b"page pool"), (dict(last=0), b"at least one last"),
    (dict(first=3), b"at least one last"), (dict(first=-1), b"at least one last"), (dict(keys=0), b"present"),
    (dict(q=8), b"aligned"), (dict(q_stride_b=4), b"aligned"), (dict(batch=70000), b"grid")])
def test_select_arguments(change, message):
    x = dict(q=64, q_stride_b=512, q_stride_h=64, bounds=64, pages=9, table=64, table_stride=4,
             width=4, lengths=64, keys=64, blocks=64, kept=3, first=1, last=1, batch=2, heads=8,
             kv_heads=2, head_dim=64, stream=0)
    x.update(change)
    assert _native.lib().pd_select_blocks(*x.values()) == _native.PD_EINVAL
    assert message in _native.lib().pd_last_error()


@pytest.mark.parametrize("change,message", [
    (dict(head_dim=80), b"head_dim"), (dict(heads=9), b"divisible"), (dict(pages=0), b"page pool"),
    (dict(cache_type=-1), b"cache type"), (dict(kept=0), b"at least one block"),
    (dict(splits=0), b"splits"), (dict(splits=129), b"splits"), (dict(part_o=0), b"present"),
    (dict(out=0), b"present"), (dict(k=8), b"aligned"), (dict(batch=2 ** 30), b"grid"),
    (dict(kv_heads=2 ** 15, heads=2 ** 15, head_dim=256), b"2 GiB")])
def test_decode_arguments(change, message):
    x = dict(q=64, q_stride_b=512, q_stride_h=64, k=64, v=64, cache_type=1, pages=9, table=64,
             table_stride=4, width=4, lengths=64, blocks=64, kept=3, k_scale=0, v_scale=0, part_o=64,
             part_ml=64, splits=2, out=64, batch=2, heads=8, kv_heads=2, head_dim=64, scale=0.1,
             stream=0)
    x.update(change)
    assert _native.lib().pd_block_decode(*x.values()) == _native.PD_EINVAL
    assert message in _native.lib().pd_last_error()


@pytest.mark.parametrize("dtype", [BF16, torch.float8_e4m3fn], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_splits(dim, dtype):
    for batch, heads, hkv, entries in ((1, 16, 4, 33), (128, 16, 16, 64), (64, 32, 8, 512),
                                       (3, 40, 2, 100000), (65535, 8, 8, 1)):
        for listed in (False, True):
            s = _native.block_splits(batch, heads, hkv, dim, dtype, entries, listed, 256)
            assert 1 <= s <= min(_native.MAX_BLOCK_SPLITS, entries)
            bucket = 1 << (batch - 1).bit_length()
            assert s == _native.block_splits(bucket, heads, hkv, dim, dtype, entries, listed, 256)
    with pytest.raises(ValueError, match="positive"):
        _native.block_splits(0, 8, 2, dim, dtype, 4, False, 256)
    with pytest.raises(ValueError, match="positive"):
        _native.block_splits(1, 9, 2, dim, dtype, 4, False, 256)
    with pytest.raises(ValueError, match="head_dim"):
        _native.block_splits(1, 8, 2, 80, dtype, 4, False, 256)


def test_rotation_table_holds_far_positions():
    table = rope_cache(70000, [1.0, 0.1], device="cpu")
    assert table.shape == (70000, 2, 2) and table.dtype == torch.float32
    assert abs(float(table[69999, 0, 0]) - math.cos(69999.0)) <= 2.0 ** -24
    assert abs(float(table[69999, 1, 1]) - math.sin(69999 * 0.1)) <= 2.0 ** -24 + 1e-10
    with pytest.raises(ValueError, match="positions"):
        rope_cache(0, [1.0], device="cpu")


def test_plain_forms_on_small_cases():
    # A quarter turn takes (a, b) to (-b, a), halves or neighbours.
    x = torch.arange(1.0, 9.0).view(1, 1, 8)
    rope = torch.tensor([[[0.0, 1.0], [0.0, 1.0]]])
    at = torch.zeros(1, dtype=torch.long)
    assert O.rotated(x, at, rope, False)[0, 0].tolist() == [-3, -4, 1, 2, 5, 6, 7, 8]
    assert O.rotated(x, at, rope, True)[0, 0].tolist() == [-2, 1, -4, 3, 5, 6, 7, 8]
    assert O.stored(torch.tensor([[[900.0, 17.0]]]), torch.tensor([0.5]),
                    torch.float8_e4m3fn).float().tolist() == [[[448.0, 32.0]]]  # 34 to even
    # Scores: the better corner of each channel; ties to the lowest block, ends always in.
    bounds = torch.zeros((2, 4, 1, 2, 64), dtype=BF16)
    bounds[0, 2, 0, 1, 0] = bounds[1, 1, 0, 1, 0] = 5.0
    bounds[1, 0, 0, 0, 1] = -7.0
    q = torch.zeros((1, 2, 64), dtype=BF16)
    q[0, 0, 0], q[0, 1, 1] = 1.0, -1.0
    tables = torch.tensor([[0, 1]], dtype=torch.int32)
    pick = lambda kept: O.select(q, bounds, tables, torch.tensor([500]), kept)[0, 0].tolist()  # noqa: E731
    assert pick(3) == [0, 4, 7] and pick(4) == [0, 2, 4, 7] and pick(6) == [0, 1, 2, 4, 5, 7]
    assert pick(9) == [0, 1, 2, 3, 4, 5, 6, 7, -1]
    # Two tokens of equal score average; a block listed twice weighs twice.
    k, v = torch.zeros((1, 256, 1, 64)), torch.zeros((1, 256, 1, 64))
    v[0, 64] = 3.0
    out, _ = O.attention(q, k, v, torch.zeros((1, 1), dtype=torch.int32), torch.tensor([65]),
                         torch.tensor([[[1, 0]]]))
    assert out[0, 0, 0] == pytest.approx(3 / 65)
    out, _ = O.attention(q, k, v, torch.zeros((1, 1), dtype=torch.int32), torch.tensor([65]),
                         torch.tensor([[[1, 1, 0]]]))
    assert out[0, 0, 0] == pytest.approx(6 / 66)


def test_a_launch_runs_on_the_device_of_its_tensors(monkeypatch):
    seen, inside = [], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            inside.append(self.index)

        def __exit__(self, *error):
            inside.pop()

    def function(*args):
        seen.append((args, tuple(inside)))
        return _native.PD_OK

    monkeypatch.setattr(_native, "_current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_native, "_raw_stream", lambda index: 100 + index)
    _native.launch(0, function, 7)
    _native.launch(1, function, 8)
    assert seen == [((7, 100), ()), ((8, 101), (1,))]
