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

BLOCK = _native.BLOCK


def rope_cache(max_positions, inv_freq, device="cuda"):
    """float32 [max_positions, half, 2]: (cos, sin) of position x inv_freq [half], the angles
    in float64 (a float32 angle is off by 0.004 at position 65536)."""
    inv = torch.as_tensor(inv_freq, dtype=torch.float64, device=device)
    if inv.dim() != 1 or type(max_positions) is not int or max_positions < 1:
        raise ValueError("rope_cache needs positions and inv_freq [half]")
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def allocate_bounds(k_cache):
    """bf16 [pages, page_size // 64, Hkv, 2, D] (smallest, largest) for a key cache, zeros."""
    pages, size, hkv, dim = k_cache.shape
    if size % BLOCK:
        raise ValueError("bounds need pages of whole blocks of 64 slots")
    return torch.zeros((pages, size // BLOCK, hkv, 2, dim), dtype=torch.bfloat16,
                       device=k_cache.device)


def _refuse(message):
    raise ValueError(message)


def _pointer(t):
    return None if t is None else t.data_ptr()


def _row_stride(t, rows, heads, dim, device, what):
    """Elements between the rows of t [rows, heads or any number (None), dim]."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[0] != rows or shape[2] != dim or heads not in (None, shape[1]):
        _refuse(f"{what} must be [N, heads, head_dim] with the key's rows")
    if t.dtype != torch.bfloat16:
        _refuse("BF16 query/key/value required")
    if stride[2] != 1 or (stride[1] != dim and shape[1] != 1):
        _refuse(f"{what} heads must be contiguous")
    if t.get_device() != device:
        _refuse("all tensors must be on one CUDA device")
    return stride[0]


def _check_index(t, n, dtype, device, what):
    if t.shape != (n,) or t.dtype != dtype or not t.is_contiguous() or t.get_device() != device:
        _refuse(f"{what} must be contiguous {str(dtype)[6:]} with one entry per token, on the "
                "cache's device")


def _check_bounds(bounds, cache_shape, device):
    pages, size, hkv, dim = cache_shape
    if (size % BLOCK or bounds.shape != (pages, size // BLOCK, hkv, 2, dim)
            or bounds.dtype != torch.bfloat16 or not bounds.is_contiguous()
            or bounds.get_device() != device):
        _refuse("bounds must be contiguous BF16 [pages, page_size // 64, kv_heads, 2, head_dim] "
                "on the cache's device")


def check_scales(k_scale, v_scale, dtype, hkv, device):
    for t in (k_scale, v_scale):
        if t is None:
            continue
        if dtype != torch.float8_e4m3fn:
            _refuse("scales belong to a float8_e4m3fn cache")
        if (t.shape != (hkv,) or t.dtype != torch.float32 or not t.is_contiguous()
                or t.get_device() != device):
            _refuse("scales must be contiguous float32 [kv_heads] on the cache's device")


def append_kv(q, k, v, positions, rope, k_cache, v_cache, slot_mapping, *, interleaved=False,
              k_scale=None, v_scale=None, bounds=None, out=None):
    """Rotated queries [N, Hq, D]; keys (rotated) and values written to their slots.

    q [N, Hq, D] (or None: returns None), k and v [N, Hkv, D] bf16, heads contiguous; rows may
    be slices of a fused projection.  ``rope`` float32 [M, half, 2] (``rope_cache``) and
    ``positions`` int64 [N]: element pairs (j, j + half), or (2j, 2j + 1) with ``interleaved``,
    of the leading 2 half elements are rotated, half a multiple of 8; rope None rotates nothing.
    Caches [blocks, block_size, Hkv, D] bf16 or float8_e4m3fn, which holds x / scale (scales
    positive and finite, float32 [Hkv], None: 1), clamped to +-448; ``slot_mapping`` int32
    [N], a negative slot (or one past the cache) writes nothing, slots of one call must differ.
    A position outside the table writes nothing and gives its query NaN.  ``out``: where the
    queries go (q itself: in place).
    """
    shape, device = k.shape, k.get_device()
    if len(shape) != 3 or device < 0:
        _refuse("key must be [N, kv_heads, head_dim] on a CUDA device")
    n, hkv, dim = shape
    k_stride, v_stride = k.stride(), v.stride()
    if v.shape != shape:
        _refuse("value must have the key's shape")
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        _refuse("BF16 query/key/value required")
    if (k_stride[2] != 1 or v_stride[2] != 1
            or (hkv != 1 and (k_stride[1] != dim or v_stride[1] != dim))):
        _refuse("key and value heads must be contiguous")
    cache, kind = k_cache.shape, k_cache.dtype
    cache_type = _native.CACHE_TYPES.get(kind)
    if cache_type is None or v_cache.dtype != kind:
        _refuse("caches must both be BF16 or float8_e4m3fn")
    if (len(cache) != 4 or cache[2] != hkv or cache[3] != dim or v_cache.shape != cache
            or not k_cache.is_contiguous() or not v_cache.is_contiguous()):
        _refuse("caches must be contiguous [blocks, block_size, kv_heads, head_dim] with the "
                "key's heads")
    if not k_cache.get_device() == v_cache.get_device() == v.get_device() == device:
        _refuse("all tensors must be on one CUDA device")
    _check_index(slot_mapping, n, torch.int32, device, "slot_mapping")
    if k_scale is not None or v_scale is not None:
        check_scales(k_scale, v_scale, kind, hkv, device)
    if bounds is not None:
        _check_bounds(bounds, cache, device)
    table = (None, None, 0, 0)
    if rope is not None:
        form = rope.shape
        if (len(form) != 3 or form[2] != 2 or rope.dtype != torch.float32
                or not rope.is_contiguous() or rope.get_device() != device):
            _refuse("rope must be contiguous float32 [positions, half, 2] on the key's device")
        if positions is None:
            _refuse("rope needs positions")
        _check_index(positions, n, torch.int64, device, "positions")
        table = (positions.data_ptr(), rope.data_ptr(), form[0], form[1])
    heads = q_stride = out_stride = 0
    if q is not None:
        q_stride, heads = _row_stride(q, n, None, dim, device, "query"), q.shape[1]
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            out_stride = heads * dim
        else:
            out_stride = _row_stride(out, n, heads, dim, device, "out")
    elif out is not None:
        _refuse("out needs a query")
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad
                                    or (q is not None and q.requires_grad)):
        _refuse("append_kv has no gradient: call it under torch.no_grad()")
    _native.launch(device, _native.lib().pd_append_kv, _pointer(q), q_stride, k.data_ptr(),
                   k_stride[0], v.data_ptr(), v_stride[0], *table, interleaved, _pointer(out),
                   out_stride, k_cache.data_ptr(), v_cache.data_ptr(), cache_type,
                   cache[0] * cache[1], slot_mapping.data_ptr(), _pointer(k_scale),
                   _pointer(v_scale), _pointer(bounds), n, heads, hkv, dim)
    return out


def block_bounds(k_cache, slot_mapping, bounds):
    """Sets the bounds of every block whose last slot is in ``slot_mapping`` (int32 [N]) from
    the keys in the cache: for blocks that ``append_kv`` did not write."""
    shape, device = k_cache.shape, k_cache.get_device()
    if len(shape) != 4 or device < 0 or not k_cache.is_contiguous():
        _refuse("the cache must be contiguous [blocks, block_size, kv_heads, head_dim] on a CUDA "
                "device")
    if k_cache.dtype not in _native.CACHE_TYPES:
        _refuse("caches must be BF16 or float8_e4m3fn")
    _check_bounds(bounds, shape, device)
    n = slot_mapping.numel()
    _check_index(slot_mapping, n, torch.int32, device, "slot_mapping")
    _native.launch(device, _native.lib().pd_block_bounds, k_cache.data_ptr(),
                   _native.CACHE_TYPES[k_cache.dtype], shape[0] * shape[1], slot_mapping.data_ptr(),
                   n, bounds.data_ptr(), shape[2], shape[3])
