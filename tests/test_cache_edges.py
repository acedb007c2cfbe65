"""Arguments of the cache operators at the C boundary, without a GPU: the smallest calls, and
combinations that would be computed otherwise than they read."""
import shutil
import subprocess

import pytest

from paged_decode import _native


def bounds_call(**change):
    x = dict(k_cache=64, cache_type=0, slots=256, mapping=64, rows=4, bounds=64, kv_heads=2,
             head_dim=64, stream=0)
    x.update(change)
    return _native.lib().pd_block_bounds(*x.values())


def test_bounds_of_no_rows():
    """An empty tensor has no address."""
    assert bounds_call(rows=0, mapping=0) == _native.PD_OK
    for change, message in ((dict(mapping=0), b"present"), (dict(bounds=0), b"present"),
                            (dict(k_cache=8), b"aligned"), (dict(rows=0, slots=100), b"whole blocks"),
                            (dict(rows=-1), b"non-negative"), (dict(rows=0, head_dim=80), b"head_dim")):
        assert bounds_call(**change) == _native.PD_EINVAL
        assert message in _native.lib().pd_last_error()


@pytest.mark.parametrize("scale", ["k_scale", "v_scale"])
def test_scales_of_a_bf16_cache(scale):
    x = dict(q=64, q_stride=512, k=64, k_stride=128, v=64, v_stride=128, positions=64, rope=64,
             max_positions=10, half=32, interleaved=0, q_out=64, q_out_stride=512, k_cache=64,
             v_cache=64, cache_type=0, slots=256, mapping=64, k_scale=0, v_scale=0, bounds=0, rows=0,
             heads=8, kv_heads=2, head_dim=64, stream=0)
    assert _native.lib().pd_append_kv(*x.values()) == _native.PD_OK
    assert _native.lib().pd_append_kv(*dict(x, cache_type=1, **{scale: 64}).values()) == _native.PD_OK
    assert _native.lib().pd_append_kv(*dict(x, **{scale: 64}).values()) == _native.PD_EINVAL
    assert b"scales belong" in _native.lib().pd_last_error()
    x = dict(q=64, q_stride_b=512, q_stride_h=64, k=64, v=64, cache_type=0, pages=9, table=64,
             table_stride=4, width=4, lengths=64, blocks=64, kept=3, k_scale=0, v_scale=0, part_o=64,
             part_ml=64, splits=2, out=64, batch=2 ** 30, heads=8, kv_heads=2, head_dim=64, scale=0.1,
             stream=0)                  # a batch past the grid: nothing is launched either way
    for cache_type, message in ((0, b"scales belong"), (1, b"grid")):
        call = dict(x, cache_type=cache_type, **{scale: 64})
        assert _native.lib().pd_block_decode(*call.values()) == _native.PD_EINVAL
        assert message in _native.lib().pd_last_error()


@pytest.mark.parametrize("batch,heads,stride_b,stride_h", [
    (2, 8, 516, 64), (1, 8, 3, 68), (2, 1, 3, 5), (2, 8, 512, 68)])
def test_strides_of_queries(batch, heads, stride_b, stride_h):
    """The strides that a call uses are multiples of 8."""
    x = dict(q=64, q_stride_b=stride_b, q_stride_h=stride_h, bounds=64, pages=9, table=64,
             table_stride=4, width=4, lengths=64, keys=64, blocks=64, kept=3, first=1, last=1,
             batch=batch, heads=heads, kv_heads=1, head_dim=64, stream=0)
    assert _native.lib().pd_select_blocks(*x.values()) == _native.PD_EINVAL
    assert b"aligned" in _native.lib().pd_last_error()
    x = dict(q=64, q_stride_b=stride_b, q_stride_h=stride_h, k=64, v=64, cache_type=1, pages=9,
             table=64, table_stride=4, width=4, lengths=64, blocks=64, kept=3, k_scale=0, v_scale=0,
             part_o=64, part_ml=64, splits=2, out=64, batch=batch, heads=heads, kv_heads=1,
             head_dim=64, scale=0.1, stream=0)
    assert _native.lib().pd_block_decode(*x.values()) == _native.PD_EINVAL
    assert b"aligned" in _native.lib().pd_last_error()


def test_the_library_exports_its_own_names_only():
    """A function of another name could be replaced by a program's own of that name."""
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("needs nm")
    listed = subprocess.run([nm, "-D", "-C", "--defined-only", _native.lib()._name], check=True,
                            capture_output=True, text=True).stdout
    names = [line.split(None, 2)[2] for line in listed.splitlines() if " T " in line]
    assert "pd_block_decode" in names
    assert [n for n in names if not n.startswith(("pd_", "pd::"))] == []
