"""The 8-bit cache of keys and values: appending with the rotation, reading back, attention over it."""
import math

import pytest
import torch

import int8_cache_ref as ref
from gpu_util import make_paged_batch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops():
    from nanoinfer_b200.csrc.lib import load_kernels
    return load_kernels(verbose=False)


def rotary_tables(positions, rot, base=10000.0):
    if rot == 0:
        return None
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * (1.0 / base ** (2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot))
    return angle.cos().float().cuda(), angle.sin().float().cuda(), rot


def filled_pool(pages, kv, page, d, g, spread=1.0):
    """Codes and scales of a pool in which every slot is held."""
    x = torch.randn(pages, kv, page, d, generator=g, dtype=torch.float64) * torch.exp(spread * torch.randn(pages, kv, 1, 1, generator=g, dtype=torch.float64))
    s = torch.tensor([[ref.block_scale(b.abs().max().item()) for b in p] for p in x], dtype=torch.float64)
    return torch.round(x / s[:, :, None, None]).clamp(-127, 127), s


class Batch:
    """A step over a pool: inputs on the device, the pool's 64-bit copy here."""

    def __init__(self, heads, kv, d, rot, page, q_lens, before, dtype, seed=0, pages=None, held=True):
        g = torch.Generator().manual_seed(seed)
        need = sum(-(-(b + n) // page) for b, n in zip(before, q_lens))
        pages = pages or need + 2
        self.heads, self.kv, self.d, self.page, self.dtype, self.q_lens, self.before = heads, kv, d, page, dtype, q_lens, before
        self.ctx, self.table = make_paged_batch(q_lens, before, page, pages, "cuda", seed=seed)
        self.codes, self.scales = zip(*(filled_pool(pages, kv, page, d, g) for _ in range(2)))
        m = sum(q_lens)
        self.rows = (torch.randn(m, heads + 2 * kv, d, generator=g) * torch.exp(torch.randn(m, heads + 2 * kv, 1, generator=g))).to(dtype)
        self.qkv = self.rows.reshape(m, -1).cuda()
        self.rotary = rotary_tables(max(b + n for b, n in zip(before, q_lens)), rot)
        self.pools = [c.to(torch.int8).cuda() for c in self.codes]
        self.pool_scales = [s.float().cuda() for s in self.scales]

    def append(self, ops, q_out=None):
        q = q_out if q_out is not None else torch.full((self.qkv.shape[0], self.heads * self.d), float("nan"), dtype=self.dtype, device="cuda")
        ops.rope_store_int8(self.qkv, q, self.heads, self.kv, self.d, self.ctx, self.rotary, self.table, self.page, *self.pools, *self.pool_scales)
        return q

    def expected(self):
        """(rotated queries, key codes, value codes, key scales, value scales) in 64 bits."""
        codes, scales = [c.clone() for c in self.codes], [s.clone() for s in self.scales]
        turned, at = [], 0
        tables = self.table.cpu().tolist()
        for i, (n, b) in enumerate(zip(self.q_lens, self.before)):
            rows = self.rows[at:at + n]
            at += n
            qk = torch.stack([ref.rotate(rows[t, :self.heads + self.kv], b + t, self.rotary) for t in range(n)])
            turned.append(qk[:, :self.heads])
            for j, x in enumerate((qk[:, self.heads:], rows[:, self.heads + self.kv:].double())):
                ref.append(codes[j], scales[j], x, b, tables[i], self.page)
        return torch.cat(turned), codes[0], codes[1], scales[0], scales[1]


def check_append(ops, b):
    q = b.append(ops)
    want_q, *want = b.expected()
    # two products and a sum in 32 bits, and one rounding to the stored type
    size = b.rows[:, :b.heads].double().abs().amax(dim=2, keepdim=True)
    bound = HALF_STEP[b.dtype] * want_q.abs() + 4 * 2.0 ** -24 * size
    assert ((q.cpu().double().reshape(want_q.shape) - want_q).abs() <= bound).all()
    for got, w in zip(b.pools + b.pool_scales, want):
        assert torch.equal(got.cpu().double(), w)


SHAPES = [(14, 2, 64, 64, 16), (28, 4, 128, 128, 16), (4, 2, 64, 32, 8), (6, 3, 128, 64, 32), (4, 4, 32, 32, 5), (4, 1, 80, 80, 24), (2, 2, 18, 6, 3),
          (3, 1, 64, 0, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,d,rot,page", SHAPES)
def test_append_follows_the_definition(ops, heads, kv, d, rot, page, dtype):
    check_append(ops, Batch(heads, kv, d, rot, page, [1], [0], dtype, seed=1))
    check_append(ops, Batch(heads, kv, d, rot, page, [1, 1, 1, 1], [7, page - 1, page, 4 * page + 2], dtype, seed=2))
    check_append(ops, Batch(heads, kv, d, rot, page, [3 * page + 1, 1, page, 2], [0, 2 * page - 1, page + 1, page - 1], dtype, seed=3))


def test_append_of_more_requests_than_a_warp_has_lanes(ops):
    lens = [1 + (5 * i) % 23 for i in range(75)]
    check_append(ops, Batch(4, 2, 64, 64, 16, lens, [(7 * i) % 40 for i in range(75)], torch.bfloat16, seed=4))


def test_append_token_by_token_and_all_at_once_differ_by_less_than_a_step(ops):
    n, page = 50, 16
    whole = Batch(2, 2, 64, 64, page, [n], [0], torch.bfloat16, seed=5)
    whole.append(ops)
    single = Batch(2, 2, 64, 64, page, [n], [0], torch.bfloat16, seed=5)
    for t in range(n):
        step = Batch(2, 2, 64, 64, page, [1], [t], torch.bfloat16, seed=5)
        step.pools, step.pool_scales, step.rotary = single.pools, single.pool_scales, single.rotary
        step.table, step.qkv = single.table, single.qkv[t:t + 1].contiguous()
        step.append(ops)
    for j in range(2):
        # the last scale of a block is that of its largest token either way
        assert torch.equal(whole.pool_scales[j], single.pool_scales[j])
        a, b = (ref.values(x.pools[j].cpu(), x.pool_scales[j].cpu()) for x in (whole, single))
        for lp in range(-(-n // page)):
            p = int(whole.table[0, lp])
            held = min(page, n - lp * page)
            assert ((a - b)[p, :, :held].abs() <= whole.pool_scales[j].cpu().double()[p][:, None, None]).all()


def test_append_in_place_strided_rows_and_a_padding_row(ops):
    b = Batch(6, 2, 64, 64, 16, [1, 4], [20, 13], torch.bfloat16, seed=6)
    want_q, *want = b.expected()
    wide = torch.zeros(5, 10 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, 4:-4] = b.qkv
    b.qkv = wide[:, 4:-4]           # rows that begin in the middle of 16 bytes
    kept = wide[:, 4 + 6 * 64:].clone()
    q = b.append(ops, q_out=wide[:, 4:4 + 6 * 64])
    assert torch.equal(wide[:, 4 + 6 * 64:], kept) and (wide[:, :4] == 0).all()
    assert ((q.cpu().double().reshape(want_q.shape) - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 1e-5 * b.rows.double().abs().max()).all()
    for got, w in zip(b.pools + b.pool_scales, want):
        assert torch.equal(got.cpu().double(), w)
    # a row of a request that holds nothing writes nothing
    b.ctx.ctx_lens.fill_(0)
    b.ctx.ctx_lens[1] = 17
    before = [t.clone() for t in b.pools]
    b.qkv = torch.randn_like(b.qkv)
    b.append(ops)
    own = int(b.table[0, 1])
    assert torch.equal(b.pools[0][own], before[0][own]) and not torch.equal(b.pools[0], before[0])


def test_append_where_pages_are_not_held_or_lie_outside_the_pool_writes_nothing_there(ops):
    b = Batch(2, 1, 64, 64, 8, [9, 9], [4, 0], torch.bfloat16, seed=7)
    b.table[0, 0] = -1
    b.table[1, 1] = 1 << 20
    check_append(ops, b)


def test_append_keeps_zero_blocks_and_extreme_magnitudes(ops):
    for factor in (0.0, 2.0 ** -120, 2.0 ** 120, 1e-30):
        b = Batch(2, 2, 64, 64, 16, [5, 1], [3, 16], torch.float32, seed=8)
        b.rows = (b.rows.double() * factor).float()
        b.qkv = b.rows.reshape(6, -1).cuda()
        b.append(ops)
        _, *want = b.expected()
        for got, w in zip(b.pools + b.pool_scales, want):
            assert torch.equal(got.cpu().double(), w)


def test_append_of_undefined_values_marks_their_block_and_no_other(ops):
    for bad in (float("nan"), float("inf"), -float("inf")):
        b = Batch(2, 2, 64, 64, 16, [20, 1], [3, 40], torch.bfloat16, seed=9)
        b.qkv[2, (2 + 2 + 1) * 64 + 5] = bad            # a value of kv head 1, position 5
        b.qkv[20, 2 * 64 + 3] = bad                     # a key of kv head 0, position 40
        before = [t.clone() for t in b.pool_scales]
        b.append(ops)
        v_page, k_page = int(b.table[0, 0]), int(b.table[1, 2])
        assert torch.isnan(b.pool_scales[1][v_page, 1]) and torch.isnan(b.pool_scales[0][k_page, 0])
        for j, at in ((0, (k_page, 0)), (1, (v_page, 1))):
            rest = torch.ones_like(before[j], dtype=torch.bool)
            rest[at] = False
            assert torch.isfinite(b.pool_scales[j][rest]).all()
        # the mark stays until the page begins anew
        c = Batch(2, 2, 64, 64, 16, [1], [41], torch.bfloat16, seed=10)
        c.pools, c.pool_scales, c.table = b.pools, b.pool_scales, b.table[1:].contiguous()
        c.append(ops)
        assert torch.isnan(b.pool_scales[0][k_page, 0])
        d = Batch(2, 2, 64, 64, 16, [1], [32], torch.bfloat16, seed=10)
        d.pools, d.pool_scales, d.table = b.pools, b.pool_scales, b.table[1:].contiguous()
        d.append(ops)
        assert torch.isfinite(b.pool_scales[0][k_page, 0])


def test_append_a_scale_that_was_never_set_stands_for_zeros(ops):
    b = Batch(2, 1, 64, 64, 16, [2], [3], torch.bfloat16, seed=11)
    page = int(b.table[0, 0])
    for j in range(2):
        b.scales[j][page] = 0.0
        b.pool_scales[j][page] = 0.0
    check_append(ops, b)
    assert (b.pools[0][page, :, :3] == 0).all()


def test_append_of_a_position_behind_the_tables_is_undefined_and_reads_nothing_else(ops):
    b = Batch(2, 1, 64, 64, 16, [1, 1], [5, 9], torch.bfloat16, seed=12)
    cos, sin, rot = b.rotary
    b.rotary = (cos[:6].contiguous(), sin[:6].contiguous(), rot)
    q = b.append(ops)
    assert torch.isfinite(q[0]).all() and torch.isnan(q[1]).all()
    assert torch.isnan(b.pool_scales[0][int(b.table[1, 0]), 0]) and torch.isfinite(b.pool_scales[1]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(7, 2, 16, 64), (3, 1, 5, 18), (1, 1, 1, 1)])
def test_unpack_is_exact(ops, shape, dtype):
    codes, scales = filled_pool(*shape, torch.Generator().manual_seed(13))
    out = torch.empty(shape, dtype=dtype, device="cuda")
    ops.unpack_int8(codes.to(torch.int8).cuda(), scales.float().cuda(), out)
    assert torch.equal(out.cpu().double(), ref.values(codes, scales))


# ---- attention --------------------------------------------------------------------------------------------------------
def check_attention(ops, b, window=0, scale=None):
    """The weights are rounded to 16 bits where a tensor core multiplies them with the values (half a step of bfloat16, relative to
    sum w |v|), a bfloat16 row once more; 32-bit sums of some thousand terms lose a few steps of 2^-24 of the same size, and the
    exponent of a score s loses |s| 2^-23, for which 2^-14 is ample.

    A weight that is small beside the largest one is rounded to a multiple of the smallest 16-bit number: with p_j = 2^(t_j - M), t_j the
    score plus the logarithm of the value scale s_j and M at most max t, that is off by at most 2^-25 each, which moves the row by at most
    2^-25 sum_j 127 2^M / sum_j 2^(score_j) <= 2^-25 n 127 sum_j w_j s_j. One below 2^-126 of the largest is nothing in 32 bits."""
    scale = b.d ** -0.5 if scale is None else scale
    out = torch.full((b.qkv.shape[0], b.heads * b.d), float("nan"), dtype=b.dtype, device="cuda")
    ops.attention_int8(b.qkv, out, b.heads, b.kv, b.d, scale, window, b.ctx, b.table, b.page, *b.pools, *b.pool_scales)
    keys, vals = (ref.values(c.cpu(), s.cpu()) for c, s in zip(b.pools, b.pool_scales))
    tables, at = b.table.cpu().tolist(), 0
    rounding = (2.0 ** -8 if b.dtype == torch.bfloat16 else 0.0) + 2.0 ** -14
    for i, (n, p) in enumerate(zip(b.q_lens, b.before)):
        for t in range(n):
            q = b.rows[at, :b.heads]
            want, size, small = ref.attend(q, keys, vals, b.pool_scales[1].cpu(), tables[i], b.page, p + t, scale, window, b.kv)
            got = out[at].cpu().double().reshape(b.heads, b.d)
            assert ((got - want).abs() <= HALF_STEP[b.dtype] * want.abs() + rounding * size + 2.0 ** -25 * small).all(), (i, t)
            at += 1
    return out


ATTENTION_SHAPES = [(14, 2, 64, 16), (12, 2, 128, 16), (28, 4, 128, 32), (16, 1, 64, 8), (12, 1, 128, 64), (32, 2, 64, 64), (3, 3, 64, 16),
                    (6, 2, 32, 16), (4, 2, 80, 24), (20, 1, 64, 16), (4, 2, 64, 5), (2, 1, 18, 3)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,d,page", ATTENTION_SHAPES)
def test_attention_of_single_tokens(ops, heads, kv, d, page, dtype):
    check_attention(ops, Batch(heads, kv, d, 0, page, [1], [0], dtype, seed=20))
    check_attention(ops, Batch(heads, kv, d, 0, page, [1, 1, 1, 1, 1], [1, 15, 16, 200, 517], dtype, seed=21))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,d,page", ATTENTION_SHAPES)
def test_attention_of_portions_and_mixed_steps(ops, heads, kv, d, page, dtype):
    check_attention(ops, Batch(heads, kv, d, 0, page, [1, 1, 37, 2, 70], [130, 0, 0, 63, 61], dtype, seed=22))


@pytest.mark.parametrize("window", [1, 7, 16, 64, 100, 1000])
def test_attention_within_a_window_whose_first_pages_are_given_back(ops, window):
    for heads, kv, d, page in ((14, 2, 64, 16), (12, 2, 128, 8), (4, 2, 32, 16)):
        b = Batch(heads, kv, d, 0, page, [1, 1, 1, 9, 80], [300, 4, 63, 150, 40], torch.bfloat16, seed=23)
        for i, p in enumerate(b.before):
            b.table[i, :max(0, p + 1 - window) // page] = -1
        check_attention(ops, b, window=window)


def test_attention_of_a_long_context_over_many_ctas(ops):
    for heads, kv, d, before in ((14, 2, 64, [9000]), (4, 1, 128, [20011, 3]), (2, 2, 64, [4095, 4096, 2047, 1])):
        check_attention(ops, Batch(heads, kv, d, 0, 16, [1] * len(before), before, torch.bfloat16, seed=24))


def test_attention_rows_that_see_nothing_are_zero_and_masked_blocks_do_not_count(ops):
    for dtype in (torch.bfloat16, torch.float32):
        b = Batch(6, 2, 64, 0, 16, [1, 1], [40, 70], dtype, seed=25)
        # undefined blocks that no token sees: behind the window's end, and slots behind a request's last token
        window = 20
        for t in b.pool_scales:
            t[int(b.table[1, 0])] = float("nan")
        got = attention_rows(ops, b, window)
        assert torch.isfinite(got).all()
        b.ctx.ctx_lens[0] = 0
        b.table[0] = -1
        out = torch.full((2, 6 * 64), float("nan"), dtype=dtype, device="cuda")
        ops.attention_int8(b.qkv, out, 6, 2, 64, 0.125, window, b.ctx, b.table, 16, *b.pools, *b.pool_scales)
        assert (out[0] == 0).all() and torch.equal(out[1], got[1])


def attention_rows(ops, b, window=0):
    out = torch.empty(b.qkv.shape[0], b.heads * b.d, dtype=b.dtype, device="cuda")
    ops.attention_int8(b.qkv, out, b.heads, b.kv, b.d, b.d ** -0.5, window, b.ctx, b.table, b.page, *b.pools, *b.pool_scales)
    return out


def test_attention_of_undefined_blocks_is_undefined(ops):
    for j in range(2):
        for dtype in (torch.bfloat16, torch.float32):
            b = Batch(4, 2, 64, 0, 16, [1, 1], [40, 70], dtype, seed=26)
            b.pool_scales[j][int(b.table[0, 1]), 1] = float("nan")
            got = attention_rows(ops, b).reshape(2, 4, 64)
            assert torch.isnan(got[0, 2:]).all() and torch.isfinite(got[0, :2]).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("exponents", [(-80, 121), (-60, 60), (-20, 20), (-80, -70), (100, 119)])
def test_attention_over_blocks_of_very_different_sizes(ops, exponents):
    """Value scales that differ by any power of two: the rows are still right to their own size."""
    lo, hi = exponents
    b = Batch(6, 2, 64, 0, 16, [1, 1], [90, 170], torch.bfloat16, seed=27)
    g = torch.Generator().manual_seed(28)
    b.pool_scales[1].copy_(torch.pow(2.0, torch.randint(lo, hi + 1, b.scales[1].shape, generator=g).double()).float())
    check_attention(ops, b)


def test_attention_of_queries_of_very_different_sizes(ops):
    for factor in (2.0 ** -100, 2.0 ** -20, 2.0 ** 14, 2.0 ** 40):
        b = Batch(6, 2, 128, 0, 16, [1, 1], [90, 170], torch.bfloat16, seed=29)
        b.rows = (b.rows.float() * factor).to(torch.bfloat16)
        b.qkv = b.rows.reshape(2, -1).cuda()
        check_attention(ops, b, scale=128 ** -0.5 / factor)


def test_append_and_attention_run_together_as_a_model_calls_them(ops):
    """A prompt in two portions, then tokens one at a time, all requests at different places: every row is the attention of the
    cache as it is then."""
    heads, kv, d, page = 14, 2, 64, 16
    pages = 64
    first = Batch(heads, kv, d, d, page, [33, 20], [0, 0], torch.bfloat16, seed=30, pages=pages)
    pools, scales, table = first.pools, first.pool_scales, torch.full((2, 16), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(31)).tolist()
    lengths = [0, 0]
    rotary = rotary_tables(256, d)
    for step, lens in enumerate([[33, 20], [1, 31], [40, 1], [1, 1], [1, 1], [1, 1]]):
        b = Batch(heads, kv, d, d, page, lens, list(lengths), torch.bfloat16, seed=40 + step, pages=pages)
        for i in range(2):
            for lp in range(-(-(lengths[i] + lens[i]) // page)):
                if int(table[i, lp]) < 0:
                    table[i, lp] = order.pop()
        b.pools, b.pool_scales, b.table, b.rotary = pools, scales, table, rotary
        q = b.append(ops)
        out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
        ops.rope_store_int8(b.qkv, q, heads, kv, d, b.ctx, rotary, table, page, *pools, *scales)        # (again: the same codes)
        ops.attention_int8(q, out, heads, kv, d, d ** -0.5, 0, b.ctx, table, page, *pools, *scales, earlier_complete=True)
        b.rows[:, :heads] = q.reshape(-1, heads, d).cpu()
        b.qkv = q
        assert torch.equal(out, check_attention(ops, b))
        lengths = [a + n for a, n in zip(lengths, lens)]


def test_rows_and_results_off_16_bytes(ops):
    """Strided rows, and memory that begins in the middle of what a kernel likes to read at a time: the same values."""
    for heads, kv, d, page in ((14, 2, 64, 16), (4, 2, 128, 8)):
        b = Batch(heads, kv, d, 0, page, [1, 1, 30], [40, 9, 20], torch.bfloat16, seed=60)
        want = attention_rows(ops, b)
        m = b.qkv.shape[0]
        for lead, width in ((1, b.qkv.shape[1] + 1), (2, b.qkv.shape[1] + 6), (8, b.qkv.shape[1] + 8)):
            wide = torch.zeros(m, width + lead, dtype=torch.bfloat16, device="cuda")
            wide[:, lead:lead + b.qkv.shape[1]] = b.qkv
            room = torch.zeros(m * heads * d + 8, dtype=torch.bfloat16, device="cuda")
            out = room[lead:lead + m * heads * d].view(m, heads * d)
            ops.attention_int8(wide[:, lead:lead + b.qkv.shape[1]], out, heads, kv, d, d ** -0.5, 0, b.ctx, b.table, page, *b.pools, *b.pool_scales)
            # another kernel takes some of them: its weights are not rounded to 16 bits
            assert (out.double() - want.double()).abs().max() <= 2.0 ** -6 * want.double().abs().max()
            assert (room[:lead] == 0).all() and (room[lead + m * heads * d:] == 0).all()
        pools = [torch.zeros(p.numel() + 16, dtype=torch.int8, device="cuda")[8:8 + p.numel()].view(p.shape).copy_(p) for p in b.pools]
        out = torch.empty_like(want)
        ops.attention_int8(b.qkv, out, heads, kv, d, d ** -0.5, 0, b.ctx, b.table, page, *pools, *b.pool_scales)
        assert (out.double() - want.double()).abs().max() <= 2.0 ** -6 * want.double().abs().max()


def test_pools_of_more_than_2_to_the_31_codes(ops):
    heads, kv, d, page, pages = 8, 8, 128, 64, 36000          # 2.4e9 codes
    b = Batch(heads, kv, d, d, page, [1, 70], [130, 60], torch.bfloat16, seed=61)
    small = b.pools[0].shape[0]
    pools = [torch.zeros(pages, kv, page, d, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, kv, dtype=torch.float32, device="cuda") for _ in range(2)]
    for j in range(2):
        pools[j][-small:] = b.pools[j]
        scales[j][-small:] = b.pool_scales[j]
    table = torch.where(b.table >= 0, b.table + pages - small, b.table)
    q, q2 = (torch.empty(71, heads * d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.rope_store_int8(b.qkv, q, heads, kv, d, b.ctx, b.rotary, table, page, *pools, *scales)
    b.append(ops, q_out=q2)
    for j in range(2):
        assert torch.equal(pools[j][-small:], b.pools[j]) and torch.equal(scales[j][-small:], b.pool_scales[j]) and (pools[j][:-small] == 0).all()
    b.qkv = q2
    want, out = attention_rows(ops, b), torch.empty_like(q)
    ops.attention_int8(q, out, heads, kv, d, d ** -0.5, 0, b.ctx, table, page, *pools, *scales)
    assert torch.equal(q, q2) and torch.equal(out, want)


def test_two_streams_at_once_and_a_replayed_graph(ops):
    """Calls on two streams share nothing; a captured pair of calls follows its inputs' contents."""
    batches = [Batch(14, 2, 64, 64, 16, [1] * n, [300 + 700 * i for i in range(n)], torch.bfloat16, seed=70 + n) for n in (3, 5)]
    want = []
    for b in batches:
        q = b.append(ops)
        want.append(attention_of(ops, b, q))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, (b, st) in enumerate(zip(batches, streams)):
            with torch.cuda.stream(st):
                got[i].append(attention_of(ops, b, b.append(ops)))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    b = batches[1]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        out = attention_of(ops, b, b.append(ops))
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    b.qkv.copy_(b.qkv.flip(0))
    b.ctx.ctx_lens.sub_(1)
    b.ctx.positions.sub_(1)
    graph.replay()
    replayed = out.clone()
    assert torch.equal(replayed, attention_of(ops, b, b.append(ops))) and not torch.equal(replayed, want[1])


def attention_of(ops, b, q):
    out = torch.empty_like(q)
    ops.attention_int8(q, out, b.heads, b.kv, b.d, b.d ** -0.5, 0, b.ctx, b.table, b.page, *b.pools, *b.pool_scales)
    return out


def test_every_way_of_cutting_the_keys_gives_the_row(ops):
    """Clusters of one to eight CTAs, and shares: against 64 bits."""
    for heads, kv, d, dtype in ((14, 2, 64, torch.bfloat16), (20, 2, 128, torch.bfloat16), (4, 2, 32, torch.bfloat16), (6, 3, 64, torch.float32)):
        b = Batch(heads, kv, d, 0, 16, [1, 1, 1, 1], [700, 3, 1500, 64], dtype, seed=80)
        b.ctx.ctx_lens[3] = 0           # a padding row
        for splits in (1, 2, 4, 8, 9, 40, 200):
            check_attention_rows(ops.with_options(fixed_decode_splits=splits), b, skip=3)


def check_attention_rows(ops, b, skip):
    out = torch.full((b.qkv.shape[0], b.heads * b.d), float("nan"), dtype=b.dtype, device="cuda")
    ops.attention_int8(b.qkv, out, b.heads, b.kv, b.d, b.d ** -0.5, 0, b.ctx, b.table, b.page, *b.pools, *b.pool_scales)
    keys, vals = (ref.values(c.cpu(), s.cpu()) for c, s in zip(b.pools, b.pool_scales))
    rounding = (2.0 ** -8 if b.dtype == torch.bfloat16 else 0.0) + 2.0 ** -14
    for i, p in enumerate(b.before):
        if i == skip:
            assert (out[i] == 0).all()
            continue
        want, size, small = ref.attend(b.rows[i, :b.heads], keys, vals, b.pool_scales[1].cpu(), b.table.cpu().tolist()[i], b.page, p, b.d ** -0.5, 0, b.kv)
        assert ((out[i].cpu().double().reshape(b.heads, b.d) - want).abs() <= HALF_STEP[b.dtype] * want.abs() + rounding * size + 2.0 ** -25 * small).all(), i


def test_contexts_of_one_token_and_many_requests(ops):
    check_attention(ops, Batch(4, 2, 64, 0, 16, [1] * 130, [(37 * i) % 90 for i in range(130)], torch.bfloat16, seed=81))
    check_attention(ops, Batch(4, 2, 128, 0, 16, [1] * 70, [(i % 3) * 17 for i in range(70)], torch.bfloat16, seed=82))


def test_refusals(ops):
    from nanoinfer_b200.csrc.lib import KernelError
    b = Batch(4, 2, 64, 64, 16, [1, 3], [5, 25], torch.bfloat16, seed=50)      # (a table of two columns: one of one column is dense turned over, too)
    q = torch.empty(4, 256, dtype=torch.bfloat16, device="cuda")

    def append(**change):
        a = dict(qkv=b.qkv, q_out=q, heads=4, kv_heads=2, head_dim=64, ctx=b.ctx, rotary=b.rotary, block_table=b.table, page_size=16,
                 k_pages=b.pools[0], v_pages=b.pools[1], k_scales=b.pool_scales[0], v_scales=b.pool_scales[1])
        a.update(change)
        ops.rope_store_int8(**a)

    def attend(**change):
        a = dict(qkv=b.qkv, out=q, heads=4, kv_heads=2, head_dim=64, scale=0.125, window=0, ctx=b.ctx, block_table=b.table, page_size=16,
                 k_pages=b.pools[0], v_pages=b.pools[1], k_scales=b.pool_scales[0], v_scales=b.pool_scales[1])
        a.update(change)
        ops.attention_int8(**a)

    for call in (append, attend):
        call()
        for change in (dict(k_pages=b.pools[0].to(torch.uint8)), dict(v_pages=b.pools[1].cpu()), dict(v_pages=b.pools[1][:-1].contiguous()),
                       dict(k_scales=b.pool_scales[0].double()), dict(v_scales=b.pool_scales[1][:-1].contiguous()), dict(page_size=8),
                       dict(kv_heads=1), dict(head_dim=32), dict(block_table=b.table.long()), dict(block_table=b.table[:1]),
                       dict(block_table=b.table.t().contiguous().t()), dict(qkv=b.qkv[:3]), dict(qkv=b.qkv.half())):
            with pytest.raises(KernelError):
                call(**change)
    for change in (dict(q_out=q[:, :128]), dict(q_out=q.float()), dict(rotary=(b.rotary[0], b.rotary[1], 32)), dict(rotary=(b.rotary[0].cpu(), b.rotary[1], 64))):
        with pytest.raises(KernelError):
            append(**change)
    for change in (dict(out=q.float()), dict(out=q[:3]), dict(window=-1), dict(heads=3)):
        with pytest.raises(KernelError):
            attend(**change)
    with pytest.raises(KernelError):
        ops.unpack_int8(b.pools[0], b.pool_scales[0], torch.empty(b.pools[0].shape, dtype=torch.float16, device="cuda"))
    with pytest.raises(KernelError):
        ops.unpack_int8(b.pools[0], b.pool_scales[0], torch.empty(2, 2, dtype=torch.float32, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_lens,before", [([0, 2], [7, 15]), ([2, 0], [31, 5]), ([1, 0], [40, 9]), ([0, 1, 0, 1, 3], [3, 16, 0, 33, 14]),
                                           ([0, 70, 0, 5], [1, 11, 130, 60])])
def test_requests_that_bring_no_token(ops, q_lens, before, dtype):
    """Their pages stay as they are, and the other requests' rows are theirs."""
    b = Batch(4, 2, 64, 64, 16, q_lens, before, dtype, seed=90)
    codes, scales = [c.clone() for c in b.codes], [s.clone() for s in b.scales]
    tables, at, turned = b.table.cpu().tolist(), 0, []
    for i, (n, p) in enumerate(zip(q_lens, before)):
        rows = b.rows[at:at + n]
        at += n
        for t in range(n):
            turned.append(ref.rotate(rows[t, :b.heads + b.kv], p + t, b.rotary))
        if n:
            ref.append(codes[0], scales[0], torch.stack(turned[-n:])[:, b.heads:], p, tables[i], b.page)
            ref.append(codes[1], scales[1], rows[:, b.heads + b.kv:].double(), p, tables[i], b.page)
    q = b.append(ops)
    assert torch.isfinite(q).all()
    for got, want in zip(b.pools + b.pool_scales, codes + scales):
        assert torch.equal(got.cpu().double(), want)
    b.qkv, b.rows = q, q.reshape(-1, b.heads, b.d).cpu()
    check_attention(ops, b)


@pytest.mark.parametrize("q_lens,before", [([300], [50]), ([1, 1, 90], [700, 33, 0]), ([1, 1], [515, 90])])
def test_rows_that_the_kernel_before_makes(ops, q_lens, before):
    """Product, append and attention launched one behind the other, many times over the same buffers with other inputs each time: what each
    leaves is what it leaves when every kernel before it has ended."""
    heads, kv, d, hidden = 14, 2, 64, 896
    b = Batch(heads, kv, d, d, 16, q_lens, before, torch.bfloat16, seed=100)
    m = sum(q_lens)
    g = torch.Generator().manual_seed(101)
    w = (torch.randn((heads + 2 * kv) * d, hidden, generator=g) * hidden ** -0.5).to(torch.bfloat16).cuda()
    inputs = [(torch.randn(m, hidden, generator=g) * 2.0 ** i).to(torch.bfloat16).cuda() for i in range(4)]
    start = [t.clone() for t in b.pools + b.pool_scales]
    q, out = (torch.empty(m, heads * d, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    product = ops.with_options(tc_splits=1)          # (parts of K would add up as they come)

    def run(x, wait):
        for step in (lambda: product.linear(x, w, None, b.qkv, "store"), lambda: b.append(ops, q_out=q),
                     lambda: ops.attention_int8(q, out, heads, kv, d, d ** -0.5, 0, b.ctx, b.table, 16, *b.pools, *b.pool_scales)):
            step()
            if wait:
                torch.cuda.synchronize()
        return out.clone(), [t.clone() for t in b.pools + b.pool_scales]

    def runs(wait):
        for t, s in zip(b.pools + b.pool_scales, start):
            t.copy_(s)
        torch.cuda.synchronize()
        return [run(inputs[i % 4], wait) for i in range(20)]

    for (row, pools), (want, want_pools) in zip(runs(False), runs(True)):
        assert torch.equal(row, want) and all(torch.equal(x, y) for x, y in zip(pools, want_pools))


@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 16), (14, 2, 64, 8), (16, 4, 64, 64), (28, 4, 128, 16), (12, 2, 128, 8), (24, 2, 128, 32)])
def test_pages_that_are_sent_for_ahead_of_the_wait(ops, heads, kv, d, page):
    """Decoding as an engine does it: a copy of the step's lengths, the product that makes the rows, append, attention with the promise that
    earlier pages are complete. The requests' pages follow one another, so that scales of earlier pages lie beside the one that
    the append writes, and every token is larger than the one before: its page's scale grows. The rows are those without the
    promise, bit for bit, launched and replayed, and those of 64 bits."""
    before, steps, hidden = [130, 255, 64, 1041, 5000, 3], 6, 256
    n = len(before)
    total = [p + steps for p in before]
    pages = sum(-(-t // page) for t in total) + 1
    b = Batch(heads, kv, d, d, page, [1] * n, total, torch.bfloat16, seed=110, pages=sum(-(-(t + 1) // page) for t in total) + 2)
    table, at = torch.full_like(b.table, -1), 0
    for i, t in enumerate(total):
        held = -(-t // page)
        table[i, :held] = torch.arange(at, at + held, dtype=torch.int32, device="cuda")
        at += held
    assert at < pages
    b.table = table
    g = torch.Generator().manual_seed(111)
    w = (torch.randn((heads + 2 * kv) * d, hidden, generator=g) * hidden ** -0.5).to(torch.bfloat16).cuda()
    x = [(torch.randn(n, hidden, generator=g) * 1.5 ** t).to(torch.bfloat16).cuda() for t in range(steps)]
    lens = [torch.tensor([p + t + 1 for p in before], dtype=torch.int32, device="cuda") for t in range(steps)]
    start = [t.clone() for t in b.pools + b.pool_scales]
    feed = torch.empty_like(x[0])
    rows, q, out = b.qkv, *(torch.empty(n, heads * d, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def step(ops, early):
        ops.linear(feed, w, None, rows, "store")
        b.append(ops, q_out=q)
        ops.attention_int8(q, out, heads, kv, d, d ** -0.5, 0, b.ctx, b.table, page, *b.pools, *b.pool_scales, earlier_complete=early)

    def decode(one_step):
        for t, s in zip(b.pools + b.pool_scales, start):
            t.copy_(s)
        got = []
        for t in range(steps):
            feed.copy_(x[t])
            b.ctx.positions.copy_(lens[t] - 1)
            b.ctx.ctx_lens.copy_(lens[t])
            one_step()
            got.append(out.clone())
        return got

    for splits in (0, 1, 4, 8, 40):
        k = ops.with_options(fixed_decode_splits=splits)
        want = decode(lambda: step(k, False))
        grown = [(t != s).sum().item() for t, s in zip(b.pool_scales, start[2:])]
        assert min(grown) > 0
        for i in range(3):
            assert all(torch.equal(a, c) for a, c in zip(decode(lambda: step(k, True)), want)), (splits, i)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.capture_begin()
            step(k, True)
            graph.capture_end()
        torch.cuda.current_stream().wait_stream(side)
        for i in range(3):
            assert all(torch.equal(a, c) for a, c in zip(decode(graph.replay), want)), (splits, i)
    # the last step's rows
    keys, vals = (ref.values(c.cpu(), s.cpu()) for c, s in zip(b.pools, b.pool_scales))
    tables, q64 = b.table.cpu().tolist(), q.cpu().reshape(n, heads, d)
    for i, p in enumerate(total):
        want, size, small = ref.attend(q64[i], keys, vals, b.pool_scales[1].cpu(), tables[i], page, p - 1, d ** -0.5, 0, kv)
        bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size + 2.0 ** -25 * small
        assert ((out[i].cpu().double().reshape(heads, d) - want).abs() <= bound).all(), i


@pytest.mark.parametrize("heads,kv,d", [(14, 2, 64), (6, 2, 128), (24, 2, 128)])
@pytest.mark.parametrize("below", [(42, 75), (70, 78)])
def test_one_sharp_key_before_tens_of_thousands_that_weigh_little(ops, heads, kv, d, below):
    """Keys 15 to 27, and 25 to 28, octaves below the largest, whose values are all of a sign and are all that some dims of the row consist of. Their weights
    are 16-bit numbers as the largest one's is, and the denominator holds them in 32 bits: what is lost of one is half a step of it (2^-11) or
    2^-34 of the reference (2^-25, half of the smallest 16-bit number, which stands 2^9 above the row's reference); the row's rounding
    to bfloat16 and 32-bit sums come on top."""
    before = [40000, 9000, 700]
    b = Batch(heads, kv, d, 0, 16, [1] * 3, before, torch.bfloat16, seed=120)
    g = torch.Generator().manual_seed(121)
    codes = [torch.zeros_like(c) for c in b.codes]
    codes[0][..., 0] = torch.randint(100 - below[1], 101 - below[0], codes[0][..., 0].shape, generator=g).double()       # a quarter each
    codes[1][:] = torch.randint(60, 128, codes[1].shape, generator=g).double()
    for i, p in enumerate(before):
        at = 5 + 37 * i
        page, slot = int(b.table[i, at // 16]), at % 16
        codes[0][page, :, slot, 0] = 100
        codes[1][page, :, slot, ::2] = 0
    for t, c in zip(b.pools, codes):
        t.copy_(c)
    b.pool_scales[0].fill_(0.25)
    b.pool_scales[1].fill_(2.0 ** -3)
    b.rows[:, :heads] = 0
    b.rows[:, :heads, 0] = 1
    b.qkv.copy_(b.rows.reshape(3, -1))
    keys, vals = (ref.values(c, s.cpu()) for c, s in zip(codes, b.pool_scales))
    tables = b.table.cpu().tolist()
    want = [ref.attend(b.rows[i, :heads], keys, vals, b.pool_scales[1].cpu(), tables[i], 16, p, 1.0, 0, kv) for i, p in enumerate(before)]
    for splits in (0, 1, 8, 40):
        out = torch.empty(3, heads * d, dtype=torch.bfloat16, device="cuda")
        ops.with_options(fixed_decode_splits=splits).attention_int8(b.qkv, out, heads, kv, d, 1.0, 0, b.ctx, b.table, 16, *b.pools, *b.pool_scales)
        for i, (row, size, small) in enumerate(want):
            err = (out[i].cpu().double().reshape(heads, d) - row).abs()
            assert (err <= 2.0 ** -8 * row.abs() + (2.0 ** -11 + 2.0 ** -14) * size + 2.0 ** -34 * small).all(), (splits, i)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,d,page", [(4, 2, 64, 16), (4, 2, 128, 8), (4, 2, 32, 16)])
def test_an_undefined_block_is_undefined_however_little_it_weighs(ops, heads, kv, d, page, dtype):
    """0 times an undefined value is undefined, in the middle of the keys and among the last ones alike; behind the last key, and before a
    window, it is nobody's."""
    for n, at in ((300, 1), (300, 290 // page), (41, 40 // page), (41, 0)):
        b = Batch(heads, kv, d, 0, page, [1, 1], [n - 1, n - 1], dtype, seed=130)
        b.rows[:, :heads] = 0
        b.rows[:, :heads, 0] = 1
        b.qkv.copy_(b.rows.reshape(2, -1))
        for t in b.pools[0]:
            t[..., 0] = 100
        b.pool_scales[0].fill_(4.0)
        bad = int(b.table[0, at])
        b.pools[0][bad, :, :, 0] = -100             # 800 below the others: 2^-1154 of their weight
        b.pool_scales[1][bad, 1] = float("nan")
        out = torch.empty(2, heads * d, dtype=dtype, device="cuda")
        ops.attention_int8(b.qkv, out, heads, kv, d, 1.0, 0, b.ctx, b.table, page, *b.pools, *b.pool_scales)
        rows = out.reshape(2, kv, heads // kv, d)
        assert torch.isnan(rows[0, 1]).all() and torch.isfinite(rows[0, 0]).all() and torch.isfinite(rows[1]).all(), (n, at)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,d,page", [(4, 2, 64, 16), (12, 2, 128, 16), (4, 2, 32, 8)])
def test_undefined_blocks_in_portions_are_their_tokens_alone(ops, heads, kv, d, page, dtype):
    """A portion's tokens that see an undefined block are undefined; those before it, those whose window has left it, the other kv head's and
    the other request's are what they are without it."""
    for j in range(2):
        for window in (0, 50):
            b = Batch(heads, kv, d, 0, page, [150, 20], [40, 9], dtype, seed=140)
            want = attention_rows(ops, b, window).reshape(-1, kv, heads // kv, d)
            first = 4 * page                    # position of the block's first token
            b.pool_scales[j][int(b.table[0, 4]), 1] = float("nan")
            got = attention_rows(ops, b, window).reshape(-1, kv, heads // kv, d)
            sees = torch.zeros(170, dtype=torch.bool)
            for t in range(150):
                lo = max(0, 40 + t - window + 1) if window else 0
                sees[t] = 40 + t >= first and lo < first + page
            assert torch.isnan(got[sees, 1]).all() and torch.equal(got[~sees], want[~sees]) and torch.equal(got[:, 0], want[:, 0]), (j, window)


@pytest.mark.parametrize("window", [0, 100])
def test_scratch_of_portions_follows_what_they_see(ops, window):
    """Sixty short prompts, and one portion behind 30,000 positions, beside a decoded token at 40,000: by the table's width it would be 61 times
    40,000 positions (2.5 GB), by what the requests' tokens see it is some thousand (and the one that sees 30,070 of them without a window)."""
    heads, kv, d, page = 12, 2, 128, 16
    q_lens, before = [1] + [40] * 60 + [70], [40000] + [(7 * i) % 30 for i in range(60)] + [30000]
    b = Batch(heads, kv, d, 0, page, q_lens, before, torch.bfloat16, seed=150)
    out = torch.empty(sum(q_lens), heads * d, dtype=torch.bfloat16, device="cuda")

    def call():
        ops.attention_int8(b.qkv, out, heads, kv, d, d ** -0.5, window, b.ctx, b.table, page, *b.pools, *b.pool_scales)

    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    call()
    seen = sum(-(-(n + p) // 64) for n, p in zip(q_lens[1:], before[1:])) if not window else 60 * 2 + 4       # pages of 64
    bound = seen * 64 * kv * d * 2 * 2 + 62 * 4 * -(-40001 // 64) + (8 << 20)            # keys and values, the table, queries and the token's parts
    assert torch.cuda.max_memory_allocated() - held <= bound
    keys, vals = (ref.values(c, s.cpu()) for c, s in zip(b.codes, b.pool_scales))
    tables, at = b.table.cpu().tolist(), 0
    for i, (n, p) in enumerate(zip(q_lens, before)):
        for t in (0, n // 2, n - 1) if i % 7 in (0, 5) else ():
            want, size, small = ref.attend(b.rows[at + t, :heads], keys, vals, b.pool_scales[1].cpu(), tables[i], page, p + t, d ** -0.5, window, kv)
            err = (out[at + t].cpu().double().reshape(heads, d) - want).abs()
            assert (err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * size + 2.0 ** -25 * small).all(), (i, t)
        at += n


@pytest.mark.parametrize("bounds", [None, [512, 256, 1024]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_portions_of_a_captured_call_may_be_longer_at_a_replay(ops, dtype, bounds):
    """The same portions further on in their requests: a table of 1,024 positions, lengths up to it or up to what the call was told."""
    heads, kv, d, page, q_lens = 4, 2, 64, 16, [1, 70, 33]
    b = Batch(heads, kv, d, 0, page, q_lens, [400, 180, 980], dtype, seed=160)
    lens = [[0, 0, 0], [100, 30, 700], [400, 180, 980], [17, 186, 5]]         # held before the step
    b.ctx.host.ctx_lens = [n for n in q_lens]
    b.ctx.host.ctx_bounds = bounds

    def inputs(before):
        b.ctx.ctx_lens.copy_(torch.tensor([n + p for n, p in zip(q_lens, before)], dtype=torch.int32))
        b.ctx.positions.copy_(torch.cat([torch.arange(p, p + n) for n, p in zip(q_lens, before)]).to(torch.int32))

    inputs(lens[0])
    k = ops.with_options(fixed_decode_splits=2)
    graph, side, out = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.empty(104, heads * d, dtype=dtype, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        k.attention_int8(b.qkv, out, heads, kv, d, d ** -0.5, 0, b.ctx, b.table, page, *b.pools, *b.pool_scales)
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for before in lens:
        inputs(before)
        out.fill_(float("nan"))
        graph.replay()
        b.ctx.host.ctx_lens, b.ctx.host.ctx_bounds = [n + p for n, p in zip(q_lens, before)], None
        assert torch.equal(out, attention_rows(k, b)), before


def test_rows_further_apart_than_32_bits_are_refused(ops):
    """Strides go to the kernels in 32 bits. (One row each: nothing lies at the stride's end.)"""
    from nanoinfer_b200.csrc.lib import KernelError
    far = 2 ** 31
    for q_lens, before in (([1], [5]), ([40], [5])):
        b = Batch(4, 2, 64, 64, 16, q_lens, before, torch.bfloat16, seed=170)
        m = q_lens[0]
        q = torch.empty(m, 256, dtype=torch.bfloat16, device="cuda")
        b.append(ops, q_out=q)
        one = m == 1
        rows = b.qkv.as_strided(b.qkv.shape, (far, 1)) if one else b.qkv
        out = q.as_strided(q.shape, (far, 1)) if one else q
        table = b.table.as_strided(b.table.shape, (far, 1))
        for change in [dict(block_table=table)] + ([dict(qkv=rows), dict(q_out=out)] if one else []):
            a = dict(qkv=b.qkv, q_out=q, heads=4, kv_heads=2, head_dim=64, ctx=b.ctx, rotary=b.rotary, block_table=b.table, page_size=16,
                     k_pages=b.pools[0], v_pages=b.pools[1], k_scales=b.pool_scales[0], v_scales=b.pool_scales[1])
            with pytest.raises(KernelError):
                ops.rope_store_int8(**{**a, **change})
        for change in [dict(block_table=table), dict(window=far)] + ([dict(qkv=rows)] if one else []):
            a = dict(qkv=b.qkv, out=q, heads=4, kv_heads=2, head_dim=64, scale=0.125, window=0, ctx=b.ctx, block_table=b.table, page_size=16,
                     k_pages=b.pools[0], v_pages=b.pools[1], k_scales=b.pool_scales[0], v_scales=b.pool_scales[1])
            with pytest.raises(KernelError):
                ops.attention_int8(**{**a, **change})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_portions_of_dense_rows_of_odd_width(ops, dtype):
    for heads, kv, d in ((4, 2, 64), (12, 2, 128), (3, 1, 33)):
        b = Batch(heads, kv, d, 0, 16, [1, 40, 2], [30, 20, 9], dtype, seed=171)
        want = attention_rows(ops, b)
        wide = torch.zeros(43, b.qkv.shape[1] + 1 + b.qkv.shape[1] % 2, dtype=dtype, device="cuda")
        assert wide.shape[1] % 2 and wide.is_contiguous()
        wide[:, :b.qkv.shape[1]] = b.qkv
        out = torch.empty_like(want)
        ops.attention_int8(wide, out, heads, kv, d, d ** -0.5, 0, b.ctx, b.table, 16, *b.pools, *b.pool_scales)
        # a decoded token whose rows lie off 4 bytes goes to another kernel, whose weights are not rounded to 16 bits
        assert (out[0].double() - want[0].double()).abs().max() <= 2.0 ** -6 * want[0].double().abs().max() and torch.equal(out[1:], want[1:])


def test_more_keys_than_a_launch_counts_are_refused(ops):
    """Chunks of all rows are counted in 32 bits: a table of 2^20 pages of 64 for each of 600 tokens may have more."""
    from nanoinfer_b200.csrc.lib import KernelError
    b = Batch(4, 2, 64, 0, 64, [1] * 600, [3] * 600, torch.bfloat16, seed=180)
    table = torch.zeros(1, 1 << 20, dtype=torch.int32, device="cuda").expand(600, 1 << 20)
    out, k = torch.empty(600, 256, dtype=torch.bfloat16, device="cuda"), ops.with_options(fixed_decode_splits=40)
    with pytest.raises(KernelError, match="too many keys"):
        k.attention_int8(b.qkv, out, 4, 2, 64, 0.125, 0, b.ctx, table, 64, *b.pools, *b.pool_scales)
    k.attention_int8(b.qkv, out, 4, 2, 64, 0.125, 0, b.ctx, table[:, :1 << 16], 64, *b.pools, *b.pool_scales)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [64, 65, 1536, 1537])
def test_queries_in_the_keys_launch_and_in_one_of_their_own(ops, m, dtype):
    """On both sides of where the launches part."""
    check_append(ops, Batch(6, 2, 64, 64, 16, [1, m - 1], [20, 37], dtype, seed=190))
