"""Keys and values of new tokens into a paged cache, rotated on the way.

``append_kv`` takes the place of a rotary embedding's launches and of ``store_kvcache``
behind them: one pass over a step's rows rotates the queries and keys and writes keys and
values to their cache slots, for prompts and for decode steps.  The cache is bf16, or e4m3
(torch.float8_e4m3fn) with one float32 scale per kv head for the keys and one for the values:
half the bytes, read by ``block_decode.fp8_decode`` and ``sparse_decode``.

``bounds`` are what ``block_decode.select_blocks`` scores: the smallest and largest stored key
per channel of every full block of 64 slots.  ``append_kv`` updates them for the blocks whose
last slot it wrote, ``block_bounds`` for a cache that was written otherwise.  A block is
expected to be written in order, its last slot last; a block that is not full has no bounds.

Nothing here synchronizes or reads device memory on the host, so a step can be captured in a
hipGraph.  Inference only.
"""
import torch

from . import _native
from .kv_write import _require

BLOCK = _native.BLOCK


def rope_cache(max_positions, inv_freq, device="cuda"):
    """float32 [max_positions, half, 2]: (cos, sin) of position x inv_freq [half], the angles
    in float64 (a float32 angle is off by 0.004 at position 65536)."""
    inv = torch.as_tensor(inv_freq, dtype=torch.float64, device=device)
    _require(inv.dim() == 1 and type(max_positions) is int and max_positions > 0,
             "rope_cache needs positions and inv_freq [half]")
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def allocate_bounds(k_cache):
    """bf16 [pages, page_size // 64, Hkv, 2, D] (smallest, largest) for a key cache, zeros."""
    pages, size, hkv, dim = k_cache.shape
    _require(size % BLOCK == 0, "bounds need pages of whole blocks of 64 slots")
    return torch.zeros((pages, size // BLOCK, hkv, 2, dim), dtype=torch.bfloat16,
                       device=k_cache.device)


def _check_cache(k_cache, bounds, device):
    _require(k_cache.dim() == 4 and k_cache.is_contiguous(),
             "caches must be contiguous [blocks, block_size, kv_heads, head_dim]")
    _require(k_cache.dtype in _native.CACHE_TYPES, "caches must be BF16 or float8_e4m3fn")
    if bounds is not None:
        pages, size, hkv, dim = k_cache.shape
        _require(size % BLOCK == 0 and bounds.shape == (pages, size // BLOCK, hkv, 2, dim)
                 and bounds.dtype == torch.bfloat16 and bounds.is_contiguous()
                 and bounds.get_device() == device,
                 "bounds must be contiguous BF16 [pages, page_size // 64, kv_heads, 2, head_dim] "
                 "on the cache's device")


def _check_rows(t, n, dim, device, what):
    _require(t.dim() == 3 and t.shape[0] == n and t.shape[2] == dim,
             f"{what} must be [N, heads, head_dim]")
    _require(t.dtype == torch.bfloat16, "BF16 query/key/value required")
    _require(t.stride(2) == 1 and (t.stride(1) == dim or t.shape[1] == 1),
             f"{what} heads must be contiguous")
    _require(t.get_device() == device, "all tensors must be on one CUDA device")


def _check_index(t, n, dtype, device, what):
    _require(t.dim() == 1 and t.shape[0] == n and t.dtype == dtype and t.is_contiguous(),
             f"{what} must be contiguous {str(dtype)[6:]} with one entry per token")
    _require(t.get_device() == device, "all tensors must be on one CUDA device")


def check_scales(k_scale, v_scale, dtype, hkv, device):
    for t in (k_scale, v_scale):
        if t is not None:
            _require(dtype == torch.float8_e4m3fn, "scales belong to a float8_e4m3fn cache")
            _require(t.shape == (hkv,) and t.dtype == torch.float32 and t.is_contiguous()
                     and t.get_device() == device,
                     "scales must be contiguous float32 [kv_heads] on the cache's device")


def append_kv(q, k, v, positions, rope, k_cache, v_cache, slot_mapping, *, interleaved=False,
              k_scale=None, v_scale=None, bounds=None, out=None):
    """Rotated queries [N, Hq, D]; keys (rotated) and values written to their slots.

    q [N, Hq, D] (or None: returns None), k and v [N, Hkv, D] bf16, heads contiguous; rows may be slices of a
    fused projection.  ``rope`` float32 [M, half, 2] (``rope_cache``) and ``positions`` int64
    [N]: element pairs (j, j + half), or (2j, 2j + 1) with ``interleaved``, of the leading
    2 half elements are rotated, half a multiple of 8; rope None rotates nothing.
    Caches [blocks, block_size, Hkv, D] bf16 or float8_e4m3fn, which holds x / scale, clamped
    to +-448; ``slot_mapping`` int32 [N], a negative slot (or one past the cache) writes
    nothing, slots of one call must differ.  A position outside the table writes nothing and
    gives its query NaN.  ``out``: where the queries go (q itself: in place).
    """
    _require(k.dim() == 3 and k.is_cuda, "key must be [N, kv_heads, head_dim] on a CUDA device")
    n, hkv, dim = k.shape
    device = k.get_device()
    _check_rows(k, n, dim, device, "key")
    _check_rows(v, n, dim, device, "value")
    _require(v.shape == k.shape, "value must have the key's shape")
    _check_cache(k_cache, bounds, device)
    _require(v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype
             and v_cache.is_contiguous() and k_cache.shape[2:] == (hkv, dim),
             "caches must have one shape and type, and the key's heads")
    _require(k_cache.get_device() == device and v_cache.get_device() == device,
             "all tensors must be on one CUDA device")
    _check_index(slot_mapping, n, torch.int32, device, "slot_mapping")
    check_scales(k_scale, v_scale, k_cache.dtype, hkv, device)
    if rope is not None:
        _require(rope.dim() == 3 and rope.shape[2] == 2 and rope.dtype == torch.float32
                 and rope.is_contiguous() and rope.get_device() == device,
                 "rope must be contiguous float32 [positions, half, 2] on the key's device")
        _check_index(positions, n, torch.int64, device, "positions")
    if q is not None:
        _check_rows(q, n, dim, device, "query")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _require(out.shape == q.shape, "out must have the query's shape")
            _check_rows(out, n, dim, device, "out")
    else:
        _require(out is None, "out needs a query")
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad
                                    or (q is not None and q.requires_grad)):
        raise ValueError("append_kv has no gradient: call it under torch.no_grad()")
    _native.append_kv(q, k, v, positions if rope is not None else None, rope, interleaved, out,
                      k_cache, v_cache, slot_mapping, k_scale, v_scale, bounds)
    return out


def block_bounds(k_cache, slot_mapping, bounds):
    """Sets the bounds of every block whose last slot is in ``slot_mapping`` (int32 [N]) from
    the keys in the cache: for blocks that ``append_kv`` did not write."""
    _require(k_cache.is_cuda, "the cache must be on a CUDA device")
    device = k_cache.get_device()
    _check_cache(k_cache, bounds, device)
    _require(bounds is not None and slot_mapping.dim() == 1, "bounds and slots are required")
    _check_index(slot_mapping, slot_mapping.shape[0], torch.int32, device, "slot_mapping")
    _native.block_bounds(k_cache, slot_mapping, bounds)
