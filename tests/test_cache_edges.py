"""Arguments of the cache operators at the C boundary, without a GPU: the smallest calls, and
combinations that would be computed otherwise than they read."""
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
