"""Products with 4-bit weights against 64 bits."""
import pytest
import torch

from nanoinfer_b200.weights.int4 import Int4Matrix

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from nanoinfer_b200.csrc.lib import load_kernels
    return load_kernels(verbose=False)


def matrix(n, k, group, seed, narrow=False):
    """(on the device, in 64 bits): random codes, scales of 8 significant bits or of 5."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g).to(torch.uint8)
    scales = (torch.exp(torch.randn(n, k // group, generator=g)) * k ** -0.5 / 4).to(torch.bfloat16)
    if narrow:
        scales = (scales.view(torch.int16) & ~7).view(torch.bfloat16)
    w = Int4Matrix.from_codes(codes.cuda(), scales.cuda(), group)
    assert w.bf16_exact == narrow
    return w, (codes.double() - 8) * scales.double().repeat_interleave(group, dim=1)


def rows(m, k, dtype, seed):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).to(dtype)


def bounds(x, w, weights_rounded):
    """What 32-bit sums of k products lose, in any order: k 2^-24 of the sum of magnitudes at most; and half a step of bfloat16 of
    every weight, where weights are rounded."""
    size = x.double().abs() @ w.abs().T
    return size * (x.shape[1] * 2.0 ** -24 + (2.0 ** -8 if weights_rounded else 0.0))


def check(ops, n, k, group, m, mode, bias=False, narrow=False, dtype=torch.bfloat16, seed=0):
    w, w64 = matrix(n, k, group, seed, narrow)
    x = rows(m, k, dtype, seed + 1)
    b = torch.randn(n, generator=torch.Generator().manual_seed(seed + 2)) if bias else None
    want = x.double() @ w64.T + (0 if b is None else b.double())
    out = torch.full((m, n), 0.5, dtype=torch.float32 if mode in ("add", "f32") else dtype, device="cuda")
    ops.linear(x.cuda(), w, None if b is None else b.cuda(), out, mode)
    if mode == "add":
        want = want + 0.5
    bound = bounds(x, w64, dtype == torch.bfloat16 and mode == "store" and m > 64 and not narrow) + 2.0 ** -23 * (want.abs() + 1)
    if mode == "store" and dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * want.abs()
    assert ((out.cpu().double() - want).abs() <= bound).all(), (n, k, group, m, mode)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(16, 128), (40, 384), (896, 896), (1152, 896), (33, 4864 // 128 * 128)])
def test_products_of_few_tokens(ops, n, k, group):
    for i, m in enumerate((1, 2, 7, 8, 9, 16, 17, 31, 33, 64)):
        check(ops, n, k, group, m, ("store", "f32", "add")[i % 3], bias=i % 2 == 0, seed=10 * i)


def test_products_of_few_tokens_whose_columns_are_half_a_tile(ops):
    for k in (32, 96, 160, 1056):
        for m in (1, 5, 20):
            check(ops, 100, k, 32, m, "f32", bias=True, seed=k + m)


def test_products_of_many_rows(ops):
    for m in (1, 8, 30, 64):
        check(ops, 152 * 256 + 5, 256, 64, m, "f32", seed=m)


def test_products_of_few_tokens_with_many_weights(ops):
    for n, k, group in ((2080, 4128, 32), (2050, 4096, 64), (2064, 4352, 128)):
        for i, m in enumerate((1, 3, 8, 9, 16, 24, 40, 64)):
            check(ops, n, k, group, m, ("f32", "store", "add")[i % 3], bias=i % 2 == 0, seed=m)


def large(n, k, group, seed):
    """As ``matrix``, made and kept on the device."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda").to(torch.uint8)
    scales = (torch.exp(torch.randn(n, k // group, generator=g, device="cuda")) * k ** -0.5 / 4).to(torch.bfloat16)
    return Int4Matrix.from_codes(codes, scales, group), (codes.double() - 8) * scales.double().repeat_interleave(group, dim=1)


@pytest.mark.parametrize("n,k,group", [(25610, 4128, 32), (24600, 4096, 64), (24600, 4096, 128)])
def test_products_whose_activations_are_prepared(ops, n, k, group):
    """From 48 MB of codes on, up to 16 tokens. A token's own size does not matter (its largest element takes a power of two to 2^13),
    nor do elements far below the largest: what 16 bits lose of them is 2^-38 of the largest."""
    w, w64 = large(n, k, group, 3)
    assert w.packed.numel() >= 48 << 20
    g = torch.Generator().manual_seed(4)
    for m in (1, 8, 9, 16):
        x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-20, 21, (m, k), generator=g).float())
        x *= torch.exp2(torch.randint(-100, 81, (m, 1), generator=g).float())
        x[m // 2] = torch.randn(k, generator=g) if m > 1 else x[0]
        x = x.to(torch.bfloat16).cuda()
        if m == 9:
            x[8] = 0.0
        out = torch.empty(m, n, dtype=torch.float32, device="cuda")
        ops.linear(x, w, None, out, "f32")
        bound = bounds(x, w64, False) + x.double().abs().amax(dim=1, keepdim=True) * 2.0 ** -38 * w64.abs().sum(dim=1)[None]
        assert ((out.double() - x.double() @ w64.T).abs() <= bound).all(), m
        half = torch.empty(m, n // 2, dtype=torch.bfloat16, device="cuda")
        if n // 2 % 16 == 0:
            y = x[m // 2:m // 2 + 1].contiguous()
            ops.linear_swiglu(y, w, half[:1])
            v = y.double() @ w64.T
            want, e = torch.nn.functional.silu(v[:, :n // 2]) * v[:, n // 2:], bounds(y, w64, False)
            slope = 1.2 * (v[:, :n // 2].abs() + v[:, n // 2:].abs() + 2)
            assert ((half[:1].double() - want).abs() <= slope * (e[:, :n // 2] + e[:, n // 2:] + 2.0 ** -19) + 2.0 ** -8 * want.abs()).all()
    x = torch.randn(3, k, generator=g).to(torch.bfloat16).cuda()
    clean, out = (torch.empty(3, n, dtype=torch.float32, device="cuda") for _ in range(2))
    ops.linear(x, w, None, clean, "f32")
    x[1, 7] = float("inf")
    ops.linear(x, w, None, out, "f32")
    assert not torch.isfinite(out[1]).any() and torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])


@pytest.mark.parametrize("narrow", [False, True])
@pytest.mark.parametrize("mode", ["store", "f32", "add"])
def test_products_of_many_tokens(ops, mode, narrow):
    for n, k, group, m in ((896, 896, 64, 65), (1152, 896, 128, 300), (100, 96, 32, 129), (2048, 1536, 64, 601)):
        check(ops, n, k, group, m, mode, bias=True, narrow=narrow, seed=m)


def test_products_of_32_bit_rows(ops):
    for m in (1, 9, 70):
        for mode in ("store", "f32", "add"):
            check(ops, 96, 192, 64, m, mode, bias=True, dtype=torch.float32, seed=m)


def gated(x, w64, n, act, glu):
    y = x.double() @ w64.T
    g, u = y[:, :n], y[:, n:]
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(g, approximate="tanh") * u
    if glu is not None:
        g, u = g.clamp(max=glu[1]), u.clamp(-glu[1], glu[1])
        return g * torch.sigmoid(glu[0] * g) * (u + glu[2])
    return g * torch.sigmoid(g) * u


@pytest.mark.parametrize("act,glu", [("silu", None), ("gelu_tanh", None), ("silu", (1.702, 7.0, 1.0))])
@pytest.mark.parametrize("n,k,group", [(64, 128, 64), (304, 384, 32), (40, 128, 128), (1056, 4096, 64), (1056, 4128, 32)])
def test_gated_products(ops, n, k, group, act, glu):
    """40 rows are no whole row tiles: they go the way of many tokens. |d gated / d gate| and |d / d up| are at most 1.13 |up| + |shift|
    and |gate| + ...: both sums' errors are scaled by at most 1.2 (|gate| + |up| + 1); fast exponential and division add some 2^-21."""
    for m in (1, 8, 13, 40, 64, 65, 200):
        w, w64 = matrix(2 * n, k, group, m)
        x = rows(m, k, torch.bfloat16, m + 1)
        out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
        ops.linear_swiglu(x.cuda(), w, out, glu, act)
        want = gated(x, w64, n, act, glu)
        y = x.double() @ w64.T
        e = bounds(x, w64, m > 64 or n % 16 != 0)
        slope = 1.2 * (y[:, :n].abs() + y[:, n:].abs() + 2)
        bound = slope * (e[:, :n] + e[:, n:]) + 2.0 ** -8 * want.abs() + 2.0 ** -19 * slope
        assert ((out.cpu().double() - want).abs() <= bound).all(), m


def test_strided_and_misaligned_rows(ops):
    w, w64 = matrix(96, 128, 64, 5)
    wide = rows(12, 160, torch.bfloat16, 6).cuda()
    for cut in (wide[:, 8:136], wide[:, 3:131]):           # rows on and off 16 bytes
        out = torch.full((12, 100), -1.0, dtype=torch.float32, device="cuda")
        ops.linear(cut, w, None, out[:, 2:98], "f32")
        want = cut.cpu().double() @ w64.T
        assert ((out[:, 2:98].cpu().double() - want).abs() <= bounds(cut.cpu(), w64, False) + 1e-6).all()
        assert (out[:, :2] == -1).all() and (out[:, 98:] == -1).all()


def test_undefined_activations_stay_in_their_token(ops):
    for (n, k), m in [(s, m) for s in ((64, 128), (2080, 4096)) for m in (3, 20, 70)]:
        w, w64 = matrix(n, k, 64, 7)
        x = rows(m, k, torch.bfloat16, 8).cuda()
        clean = torch.empty(m, n, dtype=torch.float32, device="cuda")
        ops.linear(x, w, None, clean, "f32")
        x[1, 5] = float("nan")
        out = torch.empty_like(clean)
        ops.linear(x, w, None, out, "f32")
        assert torch.isnan(out[1]).all()
        rest = torch.arange(m) != 1
        # the same sums in the same order; those of many tokens may be split and added up as they come: two orders' errors
        slack = 2 * bounds(x.cpu()[rest], w64, False) if m > 64 else 0.0
        assert ((out[rest] - clean[rest]).cpu().double().abs() <= slack).all()


def test_weights_packed_just_before_and_replayed_from_a_graph(ops):
    x = rows(8, 896, torch.bfloat16, 9).cuda()
    outs = []
    for i in range(4):
        w, w64 = matrix(896, 896, 64, i)
        out = torch.empty(8, 896, dtype=torch.float32, device="cuda")
        ops.linear(x, w, None, out, "f32")
        outs.append((out, w64, w))
    for out, w64, _ in outs:
        assert ((out.cpu().double() - x.cpu().double() @ w64.T).abs() <= bounds(x.cpu(), w64, False) + 1e-6).all()
    graph, got = torch.cuda.CUDAGraph(), torch.empty(8, 896, dtype=torch.float32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        ops.linear(x, outs[0][2], None, got, "f32")
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    x.copy_(rows(8, 896, torch.bfloat16, 10))
    graph.replay()
    again = torch.empty_like(got)
    ops.linear(x, outs[0][2], None, again, "f32")
    assert torch.equal(got, again)


def test_refusals(ops):
    from nanoinfer_b200.csrc.lib import KernelError
    w, _ = matrix(64, 128, 64, 11)
    x, out = rows(4, 128, torch.bfloat16, 12).cuda(), torch.empty(4, 64, dtype=torch.bfloat16, device="cuda")
    ops.linear(x, w, None, out, "store")
    for bad in ((x[:, :64], w, None, out, "store"), (x.half(), w, None, out, "store"), (x.cpu(), w, None, out, "store"),
                (x, w, None, out.float(), "store"), (x, w, None, out, "f32"), (x, w, None, out[:, :32], "store"), (x, w, None, out[:2], "store"),
                (x, w, torch.zeros(63, device="cuda"), out, "store"), (x, w, torch.zeros(64, dtype=torch.bfloat16, device="cuda"), out, "store"),
                (x.t().contiguous().t(), w, None, out, "store")):
        with pytest.raises(KernelError):
            ops.linear(*bad)
    half = torch.empty(4, 32, dtype=torch.bfloat16, device="cuda")
    ops.linear_swiglu(x, w, half)
    for bad in ((x, w, out), (x, w, half.float()), (x, w, half, None, "relu"), (x, w, half, (1.0, 2.0, 3.0), "gelu_tanh")):
        with pytest.raises(KernelError):
            ops.linear_swiglu(*bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [5, 70, 300])
def test_rows_of_wider_tensors_in_every_mode(ops, m, dtype):
    """Rows of activations and results that begin on and off 16 bytes, at strides that are and are not a multiple of them."""
    w, w64 = matrix(96, 128, 64, 21, narrow=True)
    for width, lead in ((160, 8), (161, 3), (160, 1)):
        x = rows(m, width, dtype, 22).cuda()[:, lead:lead + 128]
        want = x.cpu().double() @ w64.T
        bound = bounds(x.cpu(), w64, False) + 2.0 ** -23 * (want.abs() + 1)
        for mode in ("store", "f32", "add"):
            out = torch.full((m, 101), 0.5, dtype=dtype if mode == "store" else torch.float32, device="cuda")
            ops.linear(x, w, None, out[:, 3:99], mode)
            extra = 2.0 ** -8 * want.abs() if mode == "store" and dtype == torch.bfloat16 else 0.0
            assert ((out[:, 3:99].cpu().double() - want - (0.5 if mode == "add" else 0.0)).abs() <= bound + extra).all(), (width, lead, mode)
            assert (out[:, :3] == 0.5).all() and (out[:, 99:] == 0.5).all()


@pytest.mark.parametrize("m", [5, 70])
def test_codes_and_scales_off_their_words_are_refused(ops, m):
    from nanoinfer_b200.csrc.lib import KernelError
    w, _ = matrix(64, 128, 64, 23)
    x, out = rows(m, 128, torch.bfloat16, 24).cuda(), torch.empty(m, 64, dtype=torch.bfloat16, device="cuda")
    for lead_codes, lead_scales in ((8, 0), (0, 1)):
        codes = torch.empty(w.packed.numel() + 16, dtype=torch.uint8, device="cuda")[lead_codes:lead_codes + w.packed.numel()].copy_(w.packed)
        scales = torch.empty(w.scales.numel() + 2, dtype=torch.bfloat16, device="cuda")[lead_scales:lead_scales + w.scales.numel()].copy_(w.scales.reshape(-1))
        with pytest.raises(KernelError):
            ops.linear(x, Int4Matrix(codes, scales, w.shape, w.group, w.bf16_exact), None, out, "store")


def test_rows_further_apart_than_32_bits_are_refused(ops):
    from nanoinfer_b200.csrc.lib import KernelError
    w, _ = matrix(64, 128, 64, 25)
    for dtype in (torch.bfloat16, torch.float32):
        x, out = rows(1, 128, dtype, 26).cuda(), torch.empty(1, 64, dtype=dtype, device="cuda")
        ops.linear(x, w, None, out, "store")
        for bad in ((x.as_strided((1, 128), (2 ** 31, 1)), out), (x, out.as_strided((1, 64), (2 ** 31, 1)))):
            with pytest.raises(KernelError):
                ops.linear(bad[0], w, None, bad[1], "store")
