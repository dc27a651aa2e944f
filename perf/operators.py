"""What is timed of the operators in few bits: the 8-bit cache of keys and values, and products with 4-bit weights.

Three kinds of case, each a dict of plain values; ``run`` takes one pass through one operator:

* ``append``: the keys and values of a step's tokens go into an 8-bit paged cache, rotated by their positions on the way.
  A block is the ``page`` tokens of one page and one kv head; its scale is a power of two, held as a float. With ``n0`` the
  slots of the page that were held before the step and ``a`` the largest magnitude among the step's elements in the block:
  ``e`` is the least integer, not below -80 and at most 121, with ``a <= 127 * 2^e``; the new scale is ``2^e`` where the
  page is fresh (``n0`` = 0, or scale 0) and else the larger one of the old scale and ``2^e``; codes held before become
  ``rint(code * old / new)``, new ones are ``rint(x / new)`` within -127..127. Back come the rotated queries, the scales and
  the values that the pools' codes stand for.
* ``attend``: attention of a step's tokens over such a cache, the step's own tokens included: softmax over the keys at
  positions ``lo..own`` of ``scale * q . (code * key scale)``, weighted sum of ``code * value scale``. Back come the rows.
* ``product``: ``x . w^T`` with ``w[n, k] = (code[n, k] - 8) * scale[n, k // group]``, codes of 4 bits, bfloat16 scales;
  ``mode`` "store" rounds to the type of x, "f32" does not, "swiglu" is ``silu(gate) * up`` of two such products.

``spread`` makes a batch ragged: request i of n has ``1 - spread * i / n`` of the largest length. Head layouts and widths
are those of the Qwen2.5 shapes that the benchmark serves and of its designs of equal size. Pages lie in the pool in random
order. A pass can be repeated on the same state: the append writes the same slots again.
"""
import math

import torch

own = False

# heads, kv heads, head width
_HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128), "1k": (16, 2, 64), "2k": (16, 2, 128)}
# hidden width, rows of q/k/v, width of the feed-forward
_WIDTHS = {"0.5b": (896, 1152, 4864), "1.5b": (1536, 2048, 8960), "7b": (3584, 4608, 18944)}
_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
_BASE = 1000000.0


def listed():
    return [
        # one user's chat, a token at a time: nothing but latency
        _append("append_1", "0.5b", requests=1, tokens=1, past=776),
        # a loaded server's decode step: sixty-four users at very different places
        _append("append_64_ragged", "0.5b", requests=64, tokens=1, past=4000, spread=0.95),
        # two long prompts' portions at the widths of the largest shape, ends inside a page
        _append("append_prompts_2x2048", "7b", requests=2, tokens=2048, past=1001, spread=0.3),
        # one user's chat
        _attend("attend_1", "0.5b", requests=1, tokens=1, past=776),
        # the benchmark's headline: eight users at a context of 4,096
        _attend("attend_8_ctx4096", "0.5b", requests=8, tokens=1, past=4095),
        # a loaded server, heads of 128
        _attend("attend_64_ragged", "1.5b", requests=64, tokens=1, past=4000, spread=0.95),
        # what an 8-bit cache is bought for: eight long documents
        _attend("attend_8_ctx32k", "7b", requests=8, tokens=1, past=32767),
        # the last portion of a long document
        _attend("attend_prompt_2048_after_14k", "1.5b", requests=1, tokens=2048, past=14336),
        # the 32-bit mode, a few users
        _attend("attend_4_f32", "0.5b", requests=4, tokens=1, past=300, spread=0.5, dtype="float32"),
        # one user's output projection, the smallest matrix of a decode step
        _product("product_1_out", "0.5b", "out", tokens=1),
        # eight users' gate and up projections of the largest shape
        _product("product_8_gate_up", "7b", "gate_up", tokens=8),
        # the down projection of a prompt's portion
        _product("product_601_down", "1.5b", "down", tokens=601),
    ]


def _append(name, heads, requests, tokens, past, spread=0.0, dtype="bfloat16", page=16, rot=1.0):
    return {"name": name, "kind": "append", "heads": heads, "dtype": dtype, "requests": requests, "tokens": tokens, "past": past,
            "spread": spread, "page": page, "rot": rot}


def _attend(name, heads, requests, tokens, past, spread=0.0, dtype="bfloat16", page=16, window=0):
    return {"name": name, "kind": "attend", "heads": heads, "dtype": dtype, "requests": requests, "tokens": tokens, "past": past,
            "spread": spread, "page": page, "window": window}


def _product(name, widths, what, tokens, group=64, mode=None):
    return {"name": name, "kind": "product", "widths": widths, "what": what, "tokens": tokens, "group": group,
            "mode": mode or ("swiglu" if what == "gate_up" else "store")}


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    spread = round(rng.choice([0.0, rng.uniform(0.0, 0.95)]), 3)
    page = rng.choice([16, 16, 8, 32, 64])
    dtype = rng.choice(["bfloat16"] * 5 + ["float32"])
    what = rng.choice(["append", "append", "decode", "decode", "decode", "prompt", "product", "product", "product"])
    if what == "append":
        heads = rng.choice(sorted(_HEADS))
        if rng.random() < 0.5:
            c = _append("", heads, log(1, 64), 1, log(1, 8000), spread, dtype, page, rng.choice([1.0, 1.0, 0.5]))
        else:
            n = rng.choice([1, 2, 3])
            c = _append("", heads, n, log(2, 4096 // n), rng.choice([0, log(1, 8000)]), spread, dtype, page, rng.choice([1.0, 1.0, 0.5]))
    elif what == "decode":
        heads = rng.choice(sorted(_HEADS))
        if dtype == "float32":
            c = _attend("", heads, log(1, 8), 1, log(1, 1000), spread, dtype, page)
        else:
            n = log(1, 64)
            c = _attend("", heads, n, 1, log(1, min(32767, 200000 // n)), spread, dtype, page, rng.choice([0, 0, 0, log(64, 4096)]))
    elif what == "prompt":
        heads = rng.choice(["0.5b", "1.5b", "1k", "2k"])
        n = rng.choice([1, 1, 2, 3])
        if dtype == "float32":
            c = _attend("", heads, n, log(2, 200 // n), rng.choice([0, log(1, 500)]), spread, dtype, page)
        else:
            c = _attend("", heads, n, log(2, 2048 // n), rng.choice([0, 0, log(1, 8000)]), spread, dtype, page, rng.choice([0, 0, 0, log(64, 4096)]))
    else:
        widths, matrix = rng.choice(sorted(_WIDTHS)), rng.choice(["qkv", "out", "gate_up", "down"])
        tokens = rng.choice([log(1, 16), log(1, 64), log(1, 601)])
        if widths == "7b":
            tokens = min(tokens, 128)
        mode = "swiglu" if matrix == "gate_up" else rng.choice(["store", "f32"])
        c = _product("", widths, matrix, tokens, rng.choice([64, 64, 32, 128]), mode)
    c.pop("name", None)
    return c


# ---- sizes ---------------------------------------------------------------------------------------------------
def _share(n, largest, spread, least):
    return [max(least, int(round(largest * (1.0 - spread * i / n)))) for i in range(n)]


def _lengths(case):
    """(new tokens, tokens held before) of every request."""
    n, spread = case["requests"], case["spread"]
    new = _share(n, case["tokens"], spread if case["tokens"] > 1 else 0.0, 1)
    past = [0] * n if case["past"] == 0 else _share(n, case["past"], spread, 1)
    return new, past


def _matrix(case):
    """(rows of one product, k)."""
    hidden, qkv, ff = _WIDTHS[case["widths"]]
    return {"qkv": (qkv, hidden), "out": (hidden, hidden), "gate_up": (ff, hidden), "down": (hidden, ff)}[case["what"]]


def work(case):
    if case["kind"] == "product":
        n, k = _matrix(case)
        twice = 2 if case["mode"] == "swiglu" else 1
        m, out = case["tokens"], (4 if case["mode"] == "f32" else 2)
        rows = n * twice
        return {"bytes": rows * k / 2 + 2 * rows * k / case["group"] + 2 * m * k + out * m * n, "flops": 2.0 * m * rows * k}
    h, kv, d = _HEADS[case["heads"]]
    new, past = _lengths(case)
    size = 4 if case["dtype"] == "float32" else 2
    m = sum(new)
    if case["kind"] == "append":
        return {"bytes": size * m * (2 * h + 2 * kv) * d + 2.0 * m * kv * d, "flops": 3.0 * m * (h + kv) * d + 4.0 * m * kv * d}
    window = case["window"]
    keys = pairs = 0
    for n, p in zip(new, past):
        first = max(0, p + 1 - window) if window else 0
        keys += p + n - first
        pairs += sum(min(p + i + 1, window) for i in range(n)) if window else n * p + n * (n + 1) // 2
    return {"bytes": 2.0 * keys * kv * d + 2.0 * size * m * h * d, "flops": 4.0 * pairs * h * d}


# ---- what a program has in hand ---------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 17)
    return g


def _pow2(e):
    """2^e exactly, as 64-bit numbers (a library's power may be off by a rounding, which moves values that lie between two codes)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _pow2_at_least(largest):
    """2^e with the least integer e, -80 <= e <= 121, so that largest <= 127 * 2^e (64-bit in, 64-bit out)."""
    _, e = torch.frexp(largest / 127.0)                 # largest / 127 = f * 2^e, 1/2 <= f < 1
    e = torch.where(largest > 127.0 * _pow2(e - 1), e, e - 1)            # (the quotient is 1/2 or rounded up to it)
    return _pow2(torch.where(largest > 0, e, -80).clamp(-80, 121))


def _quantize_pages(x):
    """[pages, heads, slots, width] -> codes and scales, a block at a time."""
    s = _pow2_at_least(x.double().abs().amax(dim=(2, 3)))
    codes = torch.round(x.double() / s[:, :, None, None]).clamp(-127, 127).to(torch.int8)
    return codes, s.float()


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "product":
        return _prepare_product(case, g)
    h, kv, d = _HEADS[case["heads"]]
    dtype, page = _TYPES[case["dtype"]], case["page"]
    new, past = _lengths(case)
    n, m = len(new), sum(new)
    dev = "cuda"
    total = [p + t for p, t in zip(past, new)]
    held = [-(-t // page) for t in total]
    first = [0] * n             # first page that the pool holds
    if case["kind"] == "append":
        first = [p // page for p in past]
    elif case["window"]:
        first = [max(0, p + 1 - case["window"]) // page for p in past]
    pages = sum(b - a for a, b in zip(first, held)) + 3
    order = torch.randperm(pages, generator=g, device=dev).tolist()
    table = torch.full((n, max(held)), -1, dtype=torch.int32)
    at = 0
    for i in range(n):
        count = held[i] - first[i]
        table[i, first[i]:held[i]] = torch.tensor(order[at:at + count], dtype=torch.int32)
        at += count
    # keys have a few large columns, as rotated keys of trained models do; values are plain
    column = torch.exp(0.6 * torch.randn(kv, 1, d, generator=g, device=dev))
    key_pool = torch.randn(pages, kv, page, d, generator=g, device=dev) * column
    k_codes, k_scales = _quantize_pages(key_pool)
    del key_pool
    v_codes, v_scales = _quantize_pages(torch.randn(pages, kv, page, d, generator=g, device=dev))
    qkv = torch.randn(m, h + 2 * kv, d, generator=g, device=dev)
    qkv[:, h:h + kv] *= column.reshape(1, kv, d)
    starts = [0]
    for t in new:
        starts.append(starts[-1] + t)
    positions = torch.cat([torch.arange(p, p + t) for p, t in zip(past, new)]).to(torch.int32)
    state = {
        "kind": case["kind"], "heads": (h, kv, d), "page": page, "dtype": dtype, "new": new, "past": past, "starts": starts,
        "qkv": qkv.reshape(m, -1).to(dtype), "table": table.to(dev), "positions": positions.to(dev),
        "req_index": torch.repeat_interleave(torch.arange(n), torch.tensor(new)).to(torch.int32).to(dev),
        "q_start": torch.tensor(starts, dtype=torch.int32, device=dev), "ctx_lens": torch.tensor(total, dtype=torch.int32, device=dev),
        "k_codes": k_codes, "v_codes": v_codes, "k_scales": k_scales, "v_scales": v_scales, "scale": d ** -0.5,
        "window": case.get("window", 0),
    }
    if case["kind"] == "append":
        rot = int(d * case["rot"])
        angle = torch.arange(max(total), device=dev, dtype=torch.float64)[:, None] \
            * (1.0 / _BASE ** (2.0 * torch.arange(rot // 2, device=dev, dtype=torch.float64) / rot))[None, :]
        state["rotary"] = (angle.cos().float(), angle.sin().float(), rot)
    if own:
        from nanoinfer_b200.csrc.lib import load_kernels
        from nanoinfer_b200.parts.base import HostBatch, StepContext
        state["ops"] = load_kernels()
        state["ctx"] = StepContext(num_tokens=m, token_ids=state["positions"], positions=state["positions"], req_index=state["req_index"],
                                   q_start=state["q_start"], ctx_lens=state["ctx_lens"], state_slots=state["ctx_lens"],
                                   host=HostBatch(list(new), list(total), [0] * n))
    return state


def _prepare_product(case, g):
    n, k = _matrix(case)
    rows = n * (2 if case["mode"] == "swiglu" else 1)
    dev = "cuda"
    group, m = case["group"], case["tokens"]
    w = torch.randn(rows, k // group, group, generator=g, device=dev) * (k ** -0.5)
    scales = (w.abs().amax(dim=2) / 7.0).to(torch.bfloat16)
    codes = (torch.round(w / scales.float()[:, :, None]).clamp(-8, 7) + 8).to(torch.uint8).reshape(rows, k)
    del w
    state = {"kind": "product", "x": torch.randn(m, k, generator=g, device=dev).to(torch.bfloat16), "mode": case["mode"],
             "codes": codes, "scales": scales, "group": group, "n": n}
    if own:
        from nanoinfer_b200.csrc.lib import load_kernels
        from nanoinfer_b200.weights.int4 import Int4Matrix
        state["ops"] = load_kernels()
        state["w"] = Int4Matrix.from_codes(codes, scales, group)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    kind = state["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "product": _own_product}[kind](state)
    return {"append": _plain_append, "attend": _plain_attend, "product": _plain_product}[kind](state)


def _own_append(s):
    ops, (h, kv, d) = s["ops"], s["heads"]
    q = torch.empty((s["qkv"].shape[0], h * d), dtype=s["dtype"], device="cuda")
    ops.rope_store_int8(s["qkv"], q, h, kv, d, s["ctx"], s["rotary"], s["table"], s["page"], s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
    keys = torch.empty(s["k_codes"].shape, dtype=s["dtype"], device="cuda")
    values = torch.empty_like(keys)
    ops.unpack_int8(s["k_codes"], s["k_scales"], keys)
    ops.unpack_int8(s["v_codes"], s["v_scales"], values)
    return {"q": q, "keys": keys, "values": values, "key_scales": s["k_scales"], "value_scales": s["v_scales"]}


def _own_attend(s):
    ops, (h, kv, d) = s["ops"], s["heads"]
    out = torch.empty((s["qkv"].shape[0], h * d), dtype=s["dtype"], device="cuda")
    ops.attention_int8(s["qkv"], out, h, kv, d, s["scale"], s["window"], s["ctx"], s["table"], s["page"], s["k_codes"], s["v_codes"],
                       s["k_scales"], s["v_scales"])
    return out


def _own_product(s):
    out = torch.empty((s["x"].shape[0], s["n"]), dtype=torch.float32 if s["mode"] == "f32" else s["x"].dtype, device="cuda")
    if s["mode"] == "swiglu":
        s["ops"].linear_swiglu(s["x"], s["w"], out)
    else:
        s["ops"].linear(s["x"], s["w"], None, out, s["mode"])
    return out


def _rotated(x, cos, sin, rot):
    """[tokens, heads, width] with the first ``rot`` columns rotated in halves, in the type of x."""
    half = rot // 2
    a, b = x[..., :half], x[..., half:rot]
    c, s = cos[:, None, :].to(x.dtype), sin[:, None, :].to(x.dtype)
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], dim=-1)


def _plain_append(s):
    h, kv, d = s["heads"]
    page = s["page"]
    cos, sin, rot = s["rotary"]
    pos = s["positions"].long()
    rows = s["qkv"].reshape(-1, h + 2 * kv, d)
    cos, sin = cos[pos], sin[pos]
    q = _rotated(rows[:, :h].float(), cos, sin, rot).to(s["dtype"])
    # a code is a rounding to whole steps: the angle's products are taken in 64 bits, so that no value changes its side
    keys = _rotated(rows[:, h:h + kv].double(), cos, sin, rot)
    values = rows[:, h + kv:].double()
    where = s["table"].long()[s["req_index"].long(), pos // page]
    slot = pos % page
    before = torch.full((s["k_codes"].shape[0],), page, dtype=torch.long, device=pos.device)
    before.scatter_reduce_(0, where, slot, "amin")            # slots held before the step's first token of the page
    touched = torch.zeros(before.shape, dtype=torch.bool, device=pos.device)
    touched[where] = True
    held = torch.arange(page, device=pos.device)[None, :] < before[:, None]
    out = {"q": q.reshape(q.shape[0], -1)}
    for name, x, codes, scales in (("key", keys, s["k_codes"], s["k_scales"]), ("value", values, s["v_codes"], s["v_scales"])):
        largest = torch.zeros(scales.shape, dtype=torch.float64, device=pos.device)
        largest.scatter_reduce_(0, where[:, None].expand(-1, kv), x.abs().amax(dim=2), "amax")
        need = _pow2_at_least(largest)
        old = scales.double()
        fresh = (before == 0)[:, None] | (old == 0)
        new = torch.where(touched[:, None], torch.where(fresh, need, torch.maximum(old, need)), old)
        moved = torch.round(codes.double() * (old / new)[:, :, None, None])
        stored = torch.where((touched[:, None] & held)[:, None, :, None], moved, codes.double())
        stored[where, :, slot] = torch.round(x / new[where][:, :, None]).clamp(-127, 127)
        out[name + "s"] = (stored * new[:, :, None, None]).to(s["dtype"])
        out[name + "_scales"] = new.float()
    return {k: out[k] for k in ("q", "keys", "values", "key_scales", "value_scales")}


def _gathered(s, i, end):
    """Keys and values of request i at positions 0..end-1 as 32-bit numbers, [kv heads, end, width]; pages not held are zero."""
    page = s["page"]
    kv, d = s["heads"][1:]
    ids = s["table"][i, :-(-end // page)].long().clamp(min=0)
    out = []
    for codes, scales in ((s["k_codes"], s["k_scales"]), (s["v_codes"], s["v_scales"])):
        x = codes[ids].float() * scales[ids][:, :, None, None]
        out.append(x.permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :end])
    return out


def _plain_attend(s):
    h, kv, d = s["heads"]
    rep = h // kv
    out = torch.empty((s["qkv"].shape[0], h * d), dtype=s["dtype"], device=s["qkv"].device)
    for i, (n, p) in enumerate(zip(s["new"], s["past"])):
        keys, values = _gathered(s, i, p + n)
        begin = s["starts"][i]
        q = s["qkv"][begin:begin + n, :h * d].float().reshape(n, kv, rep, d).permute(1, 2, 0, 3)
        at = torch.arange(p, p + n, device=q.device)[:, None]
        key = torch.arange(p + n, device=q.device)[None, :]
        hidden = key > at
        if s["window"]:
            hidden = hidden | (key <= at - s["window"])
        for j in range(kv):     # (a head group at a time: the scores of a long prompt fill the memory otherwise)
            score = (q[j].reshape(rep * n, d) @ keys[j].T).reshape(rep, n, -1) * s["scale"]
            score = score.masked_fill(hidden, float("-inf"))
            weight = torch.exp(score - score.amax(dim=-1, keepdim=True))
            row = (weight.reshape(rep * n, -1) @ values[j]).reshape(rep, n, d) / weight.sum(dim=-1, keepdim=True)
            out[begin:begin + n].view(n, kv, rep, d)[:, j] = row.permute(1, 0, 2).to(s["dtype"])
    return out


def _plain_product(s):
    group = s["group"]
    rows, k = s["codes"].shape
    w = (s["codes"].float() - 8.0).reshape(rows, k // group, group) * s["scales"].float()[:, :, None]
    y = s["x"].float() @ w.reshape(rows, k).T
    if s["mode"] == "f32":
        return y
    if s["mode"] == "swiglu":
        gate, up = y[:, :s["n"]], y[:, s["n"]:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(s["x"].dtype)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    """The same outputs in 64 bits, a request, a page or a block of rows at a time."""
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "product": _exact_product}[case["kind"]](s)


def _exact_append(s):
    h, kv, d = s["heads"]
    page, (cos, sin, rot) = s["page"], s["rotary"]
    x = s["qkv"].double().reshape(-1, h + 2 * kv, d)
    turned = x[:, :h + kv].clone()
    c, sn = cos.double()[s["positions"].long()].unsqueeze(1), sin.double()[s["positions"].long()].unsqueeze(1)
    left, right = x[:, :h + kv, :rot // 2], x[:, :h + kv, rot // 2:rot]
    turned[:, :, :rot // 2] = left * c - right * sn
    turned[:, :, rot // 2:rot] = right * c + left * sn
    result = {"q": turned[:, :h].reshape(-1, h * d)}
    table = s["table"].tolist()
    sources = {"key": (turned[:, h:], s["k_codes"], s["k_scales"]), "value": (x[:, h + kv:], s["v_codes"], s["v_scales"])}
    for name, (rows, codes, scales) in sources.items():
        meant = codes.double() * scales.double()[:, :, None, None]
        final = scales.double().clone()
        for i, (n, p) in enumerate(zip(s["new"], s["past"])):
            at = p
            while at < p + n:
                begin, end = at % page, min(page, at % page + p + n - at)
                b = table[i][at // page]
                mine = rows[s["starts"][i] + at - p:s["starts"][i] + at - p + end - begin].permute(1, 0, 2)      # [kv, slots, d]
                top = mine.abs().amax(dim=(1, 2))
                step = torch.tensor([next((2.0 ** e for e in range(-80, 121) if a <= 127.0 * 2.0 ** e), 2.0 ** 121) for a in top.tolist()],
                                    dtype=torch.float64, device="cuda")
                before = final[b]
                if begin > 0:
                    step = torch.where(before > step, before, step)
                old = codes[b].double()
                old[:, :begin] = torch.round(old[:, :begin] * (before / step)[:, None, None])
                old[:, begin:end] = torch.round(mine / step[:, None, None]).clamp(-127, 127)
                meant[b] = old * step[:, None, None]
                final[b] = step
                at += end - begin
        result[name + "s"] = meant
        result[name + "_scales"] = final
    return {k: result[k] for k in ("q", "keys", "values", "key_scales", "value_scales")}


def _exact_attend(s):
    h, kv, d = s["heads"]
    rep, page = h // kv, s["page"]
    result = torch.zeros((s["qkv"].shape[0], h, d), dtype=torch.float64, device="cuda")
    for i, (n, p) in enumerate(zip(s["new"], s["past"])):
        lowest = max(0, p + 1 - s["window"]) if s["window"] else 0
        j = torch.arange(lowest, p + n, device="cuda")
        b, slot = s["table"][i].long()[j // page], j % page
        rows = s["qkv"][s["starts"][i]:s["starts"][i] + n, :h * d].double().reshape(n, h, d)
        visible = j[None, :] <= (p + torch.arange(n, device="cuda"))[:, None]
        if s["window"]:
            visible &= j[None, :] > (p + torch.arange(n, device="cuda"))[:, None] - s["window"]
        for g in range(kv):
            k = s["k_codes"][b, g, slot].double() * s["k_scales"][b, g].double()[:, None]
            v = s["v_codes"][b, g, slot].double() * s["v_scales"][b, g].double()[:, None]
            for head in range(g * rep, (g + 1) * rep):
                score = torch.where(visible, rows[:, head] @ k.T * s["scale"], -math.inf)
                result[s["starts"][i]:s["starts"][i] + n, head] = torch.softmax(score, dim=1) @ v
    return result.reshape(-1, h * d)


def _exact_product(s):
    group, parts = s["group"], []
    x = s["x"].double()
    for begin in range(0, s["codes"].shape[0], 4096):
        c = s["codes"][begin:begin + 4096].double() - 8.0
        c *= torch.repeat_interleave(s["scales"][begin:begin + 4096].double(), group, dim=1)
        parts.append(torch.matmul(x, c.T))
    y = torch.cat(parts, dim=1)
    if s["mode"] == "swiglu":
        gate = y[:, :s["n"]]
        y = gate * torch.sigmoid(gate) * y[:, s["n"]:]
    return y
