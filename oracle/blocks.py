"""Plain 64-bit forms of the cache operators (paged_decode.kv_append, .block_decode), torch on
the CPU: written from the formulas, one sequence and kv head at a time."""
import math

import torch

BLOCK, PER_PAGE = 64, 4
E4M3_MAX = 448.0


def rotated(x, positions, rope, interleaved, dtype=torch.float64):
    """x [N, H, D] with the leading 2 half elements of every head rotated; with float32 each
    product and sum is rounded by itself."""
    out, half = x.to(dtype).clone(), rope.shape[1]
    cos, sin = rope[positions].to(dtype)[:, None].unbind(-1)
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = out[..., first].clone(), out[..., second].clone()
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    return out


def stored(x, scale, kind):
    """float32 rows [N, Hkv, D] as a cache of type `kind` holds them."""
    if kind == torch.float8_e4m3fn:
        if scale is not None:
            x = x / scale[:, None]
        x = x.clamp(-E4M3_MAX, E4M3_MAX)
    return x.to(kind)


def block_bounds(keys):
    """(smallest, largest) [Hkv, 2, D] of one block's stored keys [64, Hkv, D]."""
    keys = keys.float()
    return torch.stack([keys.amin(0), keys.amax(0)], 1).to(torch.bfloat16)


def scores(q, bounds):
    """float64 [blocks] of q [G, D] and bounds [blocks, 2, D]."""
    q, bounds = q.double(), bounds.double()
    q = torch.where(q.isinf(), math.nan, q)
    each = q.clamp(min=0) @ bounds[:, 1].T + q.clamp(max=0) @ bounds[:, 0].T      # [G, blocks]
    return torch.where(each.isnan(), math.inf, each).amax(0)


def select(q, bounds, tables, lengths, kept, first=1, last=1):
    batch, heads, _ = q.shape
    hkv = bounds.shape[2]
    out = torch.full((batch, hkv, kept), -1, dtype=torch.int32)
    for b in range(batch):
        n = -(-int(lengths[b]) // BLOCK)
        if n <= kept:
            out[b, :, :n] = torch.arange(n, dtype=torch.int32)
            continue
        j = torch.arange(first, n - last)
        found = bounds[tables[b, j // PER_PAGE].long(), j % PER_PAGE]
        for g in range(hkv):
            s = scores(q[b].view(hkv, heads // hkv, -1)[g], found[:, g])
            order = sorted(range(len(s)), key=lambda i: (-float(s[i]), i))[:kept - first - last]
            out[b, g] = torch.tensor([*range(first), *sorted(int(j[i]) for i in order),
                                      *range(n - last, n)], dtype=torch.int32)
    return out


def attention(q, k, v, tables, lengths, blocks=None, scale=None, k_scale=None, v_scale=None):
    """(out, bound) float64 [B, Hq, D]; `bound` is how far float32 arithmetic may move an output
    before its own rounding:

    * a score is a float32 sum of D exact products: (D + 2) 2^-24 sum |q k|, and its product
      with the scales two more roundings; a probability's relative error is that times the
      scale, twice (its own and the maximum's), and 2^-22 of the exponential;
    * the sums over n tokens add n 2^-24 each, numerator and denominator.
    """
    batch, heads, dim = q.shape
    hkv = k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros((batch, heads, dim), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b in range(batch):
        n = int(lengths[b])
        for g in range(hkv):
            tokens = torch.arange(n)
            if blocks is not None:
                each = [int(j) for j in blocks[b, g] if j >= 0]
                tokens = torch.cat([torch.arange(j * BLOCK, min(n, (j + 1) * BLOCK)) for j in each
                                    if j * BLOCK < n] or [torch.arange(0)])
            pages = tables[b, tokens // 256].long()
            tokens, pages = tokens[(pages >= 0) & (pages < k.shape[0])], \
                pages[(pages >= 0) & (pages < k.shape[0])]
            if not len(tokens):
                continue
            keys, values = (c[pages, tokens % 256, g].double() for c in (k.float(), v.float()))
            rows = q[b].view(hkv, heads // hkv, dim)[g].double()
            factor = scale * (1.0 if k_scale is None else float(k_scale[g]))
            s = rows @ keys.T * factor
            p = torch.softmax(s, -1)
            at = slice(g * (heads // hkv), (g + 1) * (heads // hkv))
            by = 1.0 if v_scale is None else float(v_scale[g])
            out[b, at] = p @ values * by
            spread = ((dim + 4) * 2.0 ** -24 * abs(factor)
                      * (rows.abs() @ keys.abs().T).amax(-1, keepdim=True))
            relative = 2 * spread + 2.0 ** -21 + 2 * (len(tokens) + 64) * 2.0 ** -24
            bound[b, at] = relative * (p @ values.abs() * abs(by))
    return out, bound


def bf16_close(got, exact, bound):
    """Within the float32 bound and half a bf16 step of the exact output (2^-8 of it)."""
    return (got.double() - exact).abs() <= bound + 2.0 ** -8 * (exact.abs() + bound) + 2.0 ** -126
