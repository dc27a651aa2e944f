"""The 8-bit cache in 64 bits, a block at a time: what the kernels' tests compare with."""
import math

import torch

F64 = torch.float64


def block_scale(largest: float) -> float:
    """2^e with the least e in -80..121 that has largest <= 127 * 2^e; NaN where it is not finite."""
    if not math.isfinite(largest):
        return math.nan
    return next((2.0 ** e for e in range(-80, 121) if largest <= 127.0 * 2.0 ** e), 2.0 ** 121)


def rotate(x, pos, rotary):
    """[heads, width] of one token, the first columns rotated in halves, 64 bits."""
    x = x.double().clone()
    if rotary is None:
        return x
    cos, sin, rot = rotary
    half = rot // 2
    c, s = cos[pos].double().cpu(), sin[pos].double().cpu()
    a, b = x[:, :half].clone(), x[:, half:rot].clone()
    x[:, :half], x[:, half:rot] = a * c - b * s, b * c + a * s
    return x


def append(codes, scales, rows, before, table, page_size):
    """Appends ``rows`` [tokens, heads, width] (64 bits) of one request behind its first ``before`` positions: ``codes`` (float64) and
    ``scales`` (float64) are changed in place."""
    n = rows.shape[0]
    at = before
    while at < before + n:
        lp, first = at // page_size, at % page_size
        last = min(page_size, first + before + n - at)
        page = int(table[lp]) if lp < len(table) else -1
        new = rows[at - before:at - before + last - first]
        at += last - first
        if not 0 <= page < codes.shape[0]:
            continue
        for h in range(codes.shape[1]):
            need, old = block_scale(new[:, h].abs().max().item()), scales[page, h].item()
            if torch.isnan(new[:, h]).any():
                need = math.nan
            s = need
            if first > 0:
                s = math.nan if math.isnan(old) or math.isnan(need) else max(old, need)
                if s > old:
                    codes[page, h, :first] = torch.round(codes[page, h, :first] * (old / s))
            codes[page, h, first:last] = torch.round(new[:, h] / s).clamp(-127, 127)
            scales[page, h] = s


def values(codes, scales):
    return codes.double() * scales.double()[:, :, None, None]


def attend(q, keys, vals, v_scales, table, page_size, position, scale, window, kv_heads):
    """One token's attention in 64 bits: q [heads, width], keys and vals [pages, kv heads, slots, width] as values, value scales [pages, kv
    heads]. Returns the row, sum_j w_j |v_j|, which roundings of the weights are relative to, and n 127 sum_j w_j s_j + n 2^-101 max |v|,
    2^-25 of which weights too small for a 16-bit number may lose (see the tests)."""
    heads, d = q.shape
    lo = max(0, position - window + 1) if window else 0
    j = torch.arange(lo, position + 1)
    pages, slots = torch.tensor([int(table[p]) for p in (j // page_size).tolist()]), j % page_size
    out, size, small = torch.empty(heads, d, dtype=F64), torch.empty(heads, d, dtype=F64), torch.empty(heads, 1, dtype=F64)
    for h in range(heads):
        g = h // (heads // kv_heads)
        k, v = keys[pages, g, slots], vals[pages, g, slots]
        w = torch.softmax(k @ q[h].double() * scale, dim=0)
        out[h], size[h] = w @ v, w @ v.abs()
        small[h] = j.numel() * (127 * (w @ v_scales[pages, g].double()) + 2.0 ** -101 * v.abs().max())
    return out, size, small
