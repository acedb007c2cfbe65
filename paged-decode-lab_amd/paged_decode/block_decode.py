"""Decode attention over an e4m3 cache, and over the blocks of a cache that matter.

``fp8_decode``     one query token per sequence over its whole e4m3 cache
                   (``kv_append.append_kv`` writes it), half the bytes of a bf16 one;
``select_blocks``  per sequence and kv head the blocks of 64 tokens whose keys can score
                   highest for the group's queries, by the bounds that append_kv keeps;
``sparse_decode``  one query token per sequence over the listed blocks, bf16 or e4m3.

Contract as of ``runtime.paged_decode``: outputs and workspaces belong to the resources and
are overwritten by the next call with them, two streams may not use them at once, contents
are not checked, nothing allocates, synchronizes or reads device memory on the host (a step
can be captured in a hipGraph).  Lengths past the table count as its capacity; a page outside
the cache is read as having no tokens.  A sequence's output depends on the batch through its
next power of two alone, so a padded graph bucket gives the bits of the eager call.
Inference only: a query, cache or bounds that ask for a gradient are refused.
"""
from dataclasses import dataclass, field
import math

import torch

from . import _native
from .kv_append import check_scales
from .runtime import _device_cus

BLOCK = _native.BLOCK
_PER_PAGE = 256 // BLOCK
E4M3 = torch.float8_e4m3fn


@dataclass
class BlockResources:
    spec: object
    kept: int                       # blocks listed per sequence and kv head, 0: every block
    out: torch.Tensor
    partials: torch.Tensor          # float32, flat: [B, Hq, splits, D] of a call
    sums: torch.Tensor              # float32, flat: [B, Hq, splits, 2]
    blocks: torch.Tensor | None = None
    keys: torch.Tensor | None = None
    sm_count: int = 0
    _splits: dict = field(default_factory=dict, repr=False, compare=False)

    def splits(self, batch, dtype):
        found = self._splits.get((batch, dtype))
        if found is None:
            spec = self.spec
            found = self._splits[batch, dtype] = _native.block_splits(
                batch, spec.num_heads, spec.num_kv_heads, spec.head_dim, dtype,
                self.kept or spec.table_width * _PER_PAGE, self.kept > 0, self.sm_count)
        return found


def allocate_block_resources(spec, device, *, kept=0):
    """Output and workspace of ``fp8_decode`` (kept 0), or of ``select_blocks`` and
    ``sparse_decode`` with ``kept`` blocks of 64 tokens per sequence and kv head."""
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("block resources require CUDA")
    if type(kept) is not int or kept < 0:
        raise ValueError("kept must be a non-negative integer")
    make = lambda *shape, dtype=torch.float32: torch.empty(shape, device=device, dtype=dtype)  # noqa: E731
    heads, hkv, dim = spec.num_heads, spec.num_kv_heads, spec.head_dim
    out = make(spec.max_batch, heads, dim, dtype=torch.bfloat16)
    result = BlockResources(spec, kept, out, out, out, sm_count=_device_cus(device))
    rows, batch = 0, 1
    while batch < 2 * spec.max_batch:
        batch = min(batch, spec.max_batch)
        splits = max(result.splits(batch, dtype) for dtype in _native.CACHE_TYPES)
        rows = max(rows, batch * heads * splits if splits > 1 else 0)
        batch *= 2
    result.partials, result.sums = make(rows * dim), make(rows * 2)
    if kept:
        result.blocks = make(spec.max_batch, hkv, kept, dtype=torch.int32)
        result.keys = make(spec.max_batch, hkv, spec.table_width * _PER_PAGE, dtype=torch.int64)
    return result


def _check_step(q, tables, lengths, resources):
    """(batch, device, Q's strides, the table's row stride and width)."""
    spec, shape, stride = resources.spec, q.shape, q.stride()
    device = q.get_device()
    if device < 0 or not (tables.get_device() == lengths.get_device()
                          == resources.out.get_device() == device):
        raise ValueError("all tensors must be on the same CUDA device")
    if q.dtype != torch.bfloat16:
        raise ValueError("BF16 Q required")
    if len(shape) != 3 or shape[1] != spec.num_heads or shape[2] != spec.head_dim:
        raise ValueError("Q must have shape [batch, query_heads, head_dim]")
    batch = shape[0]
    if not 0 < batch <= spec.max_batch or stride[2] != 1:
        raise ValueError("Q batch exceeds capacity or innermost dimension is not contiguous")
    form, step = tables.shape, tables.stride()
    if len(form) != 2 or form[0] != batch or step[1] != 1:
        raise ValueError("block table must have shape [batch,capacity] and contiguous rows")
    if not 0 < form[1] <= spec.table_width:
        raise ValueError("block table width outside configured capacity")
    if lengths.shape != (batch,) or not lengths.is_contiguous():
        raise ValueError("context lengths must be a contiguous [batch] tensor")
    if tables.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise ValueError("block tables and context lengths must be int32")
    return batch, device, stride[0], stride[1], step[0], form[1]


def _attend(q, k, v, tables, lengths, blocks, resources, scale, k_scale, v_scale):
    batch, device, stride_b, stride_h, table_stride, width = _check_step(q, tables, lengths,
                                                                         resources)
    spec, shape, kind = resources.spec, k.shape, k.dtype
    cache_type = _native.CACHE_TYPES.get(kind)
    if cache_type is None or v.dtype != kind:
        raise ValueError("caches must both be BF16 or float8_e4m3fn")
    hkv, dim = spec.num_kv_heads, spec.head_dim
    if len(shape) != 4 or shape[1] != 256 or shape[2] != hkv or shape[3] != dim:
        raise ValueError("KV must use NHD pages [pages,256,kv_heads,head_dim]")
    if v.shape != shape or not k.is_contiguous() or not v.is_contiguous() or shape[0] == 0:
        raise ValueError("K/V must have matching nonempty contiguous storage")
    if k.get_device() != device or v.get_device() != device:
        raise ValueError("all tensors must be on the same CUDA device")
    if k_scale is not None or v_scale is not None:
        check_scales(k_scale, v_scale, kind, hkv, device)
    scale = dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        raise ValueError("decode attention has no gradient: call it under torch.no_grad()")
    out = resources.out
    _native.launch(device, _native.lib().pd_block_decode, q.data_ptr(), stride_b, stride_h,
                   k.data_ptr(), v.data_ptr(), cache_type, shape[0], tables.data_ptr(), table_stride,
                   width, lengths.data_ptr(), None if blocks is None else blocks.data_ptr(),
                   0 if blocks is None else blocks.shape[2],
                   None if k_scale is None else k_scale.data_ptr(),
                   None if v_scale is None else v_scale.data_ptr(), resources.partials.data_ptr(),
                   resources.sums.data_ptr(), resources.splits(batch, kind), out.data_ptr(), batch,
                   spec.num_heads, hkv, dim, scale)
    return out if batch == spec.max_batch else out[:batch]


def fp8_decode(q, k, v, tables, lengths, *, resources, scale=None, k_scale=None, v_scale=None):
    """Attention of q [B, Hq, D] bf16 over e4m3 pages k, v [pages, 256, Hkv, D], whose values
    are the stored ones times ``k_scale`` and ``v_scale`` (float32 [Hkv], None: 1); returns
    ``resources.out[:B]``.  An empty sequence gives zeros."""
    if k.dtype != E4M3:
        raise ValueError("fp8_decode reads a float8_e4m3fn cache; paged_decode reads a BF16 one")
    if resources.kept:
        raise ValueError("these resources are sized for a list of blocks")
    return _attend(q, k, v, tables, lengths, None, resources, scale, k_scale, v_scale)


def select_blocks(q, bounds, tables, lengths, *, resources, first=1, last=1):
    """int32 [B, Hkv, kept]: the blocks that ``sparse_decode`` should read, ascending, -1 behind
    a sequence of fewer.

    Of a sequence's ceil(length / 64) blocks the first ``first`` and last ``last`` are always
    in; the others by score, the largest of the group's query heads' sums over the channels of
    max(q, 0) high + min(q, 0) low, computed in 64 bits; ties go to the lowest block.
    ``bounds`` as of ``kv_append``, of the keys as they are stored (a scale per kv head moves
    no block).  ``last`` is at least 1: the block being filled has no bounds.  A NaN score, an
    infinite query's too, counts as infinite."""
    batch, device, stride_b, stride_h, table_stride, width = _check_step(q, tables, lengths,
                                                                         resources)
    spec, blocks = resources.spec, resources.blocks
    if not resources.kept:
        raise ValueError("these resources hold no list of blocks: allocate them with kept=")
    if first < 0 or last < 1 or first + last > resources.kept:
        raise ValueError("kept blocks must hold the first ones and at least one last")
    hkv, dim, shape = spec.num_kv_heads, spec.head_dim, bounds.shape
    if (shape[1:] != (_PER_PAGE, hkv, 2, dim) or bounds.dtype != torch.bfloat16
            or not bounds.is_contiguous() or bounds.get_device() != device or shape[0] == 0):
        raise ValueError("bounds must be contiguous BF16 [pages, 4, kv_heads, 2, head_dim]")
    if torch.is_grad_enabled() and (q.requires_grad or bounds.requires_grad):
        raise ValueError("select_blocks has no gradient: call it under torch.no_grad()")
    _native.launch(device, _native.lib().pd_select_blocks, q.data_ptr(), stride_b, stride_h,
                   bounds.data_ptr(), shape[0], tables.data_ptr(), table_stride, width,
                   lengths.data_ptr(), resources.keys.data_ptr(), blocks.data_ptr(), resources.kept,
                   first, last, batch, spec.num_heads, hkv, dim)
    return blocks if batch == spec.max_batch else blocks[:batch]


def sparse_decode(q, k, v, tables, lengths, blocks, *, resources, scale=None, k_scale=None,
                  v_scale=None):
    """Attention of q [B, Hq, D] bf16 over the tokens below the length of the listed blocks,
    int32 [B, Hkv, listed <= kept] (``select_blocks``, or any choice); pages bf16 or
    float8_e4m3fn as in ``fp8_decode``; returns ``resources.out[:B]``.  Entries below 0 or past
    the length have no tokens, an entry listed twice counts twice, no token gives zeros."""
    if not resources.kept:
        raise ValueError("these resources hold no list of blocks: allocate them with kept=")
    form = blocks.shape
    if (len(form) != 3 or form[0] != q.shape[0] or form[1] != resources.spec.num_kv_heads
            or not 0 < form[2] <= resources.kept or blocks.dtype != torch.int32
            or not blocks.is_contiguous() or blocks.get_device() != q.get_device()):
        raise ValueError("blocks must be contiguous int32 [batch, kv_heads, listed], at most kept")
    return _attend(q, k, v, tables, lengths, blocks, resources, scale, k_scale, v_scale)
