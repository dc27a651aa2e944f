"""Matrices of 4-bit weights on the host: layout, quantization, refusals."""
import pytest
import torch

from nanoinfer_b200.weights.int4 import Int4Matrix


def unpacked(w: Int4Matrix) -> torch.Tensor:
    """The weights by the layout as csrc/gemm_int4.cu states it, a nibble at a time."""
    n, k = w.shape
    k_tiles = -(-k // 64)
    out = torch.empty(n, k, dtype=torch.float64)
    words = w.packed.cpu().reshape(-1, 4).to(torch.int64)
    words = words[:, 0] | (words[:, 1] << 8) | (words[:, 2] << 16) | (words[:, 3] << 24)
    scales = w.scales.double().cpu()
    order = [(0, 0), (1, 0), (0, 2), (1, 2), (0, 1), (1, 1), (0, 3), (1, 3)]        # (half, e) of every nibble
    nibble = {v: i for i, v in enumerate(order)}
    for row in range(n):
        for col in range(k):
            rt, half, g = row // 16, row % 16 // 8, row % 8
            kt, b, t, j, e = col // 64, col % 64 // 32, col % 32 // 8, col % 8 // 4, col % 4
            word = int(words[((rt * k_tiles + kt) * 32 + g * 4 + t) * 4 + 2 * b + j])
            code = word >> (4 * nibble[(half, e)]) & 15
            out[row, col] = (code - 8) * scales[rt, col // w.group, g, half]
    return out


@pytest.mark.parametrize("n,k,group", [(16, 64, 64), (5, 32, 32), (33, 96, 32), (17, 128, 128), (20, 192, 64)])
def test_layout_of_codes_and_scales(n, k, group):
    g = torch.Generator().manual_seed(n)
    codes = torch.randint(0, 16, (n, k), generator=g).to(torch.uint8)
    scales = torch.rand(n, k // group, generator=g).to(torch.bfloat16)
    w = Int4Matrix.from_codes(codes, scales, group)
    want = (codes.double() - 8) * scales.double().repeat_interleave(group, dim=1)
    assert torch.equal(unpacked(w), want)
    assert w.shape == (n, k) and w.nbytes() == (-(-n // 16)) * 16 * ((-(-k // 64)) * 32 + 2 * (k // group))


def test_quantize_is_within_half_a_step_and_exact_in_bfloat16():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(24, 128, generator=g) * torch.exp(2 * torch.randn(24, 1, generator=g))
    x[3] = 0.0
    x[4] *= 1e-36
    for dtype in (torch.float32, torch.bfloat16):
        w = Int4Matrix.quantize(x.to(dtype), 32)
        got = unpacked(w)
        assert w.bf16_exact and torch.equal(got, got.to(torch.bfloat16).double())
        largest = x.to(dtype).double().reshape(24, 4, 32).abs().amax(dim=2).repeat_interleave(32, dim=1)
        # a scale is the largest magnitude / 7, up to 1/16 more (5 significant bits); half a step of it
        assert ((got - x.to(dtype).double()).abs() <= largest / 7 * (1 + 2.0 ** -4) / 2 + 2.0 ** -117).all()


def test_scales_of_more_bits_are_told_apart():
    codes = torch.full((16, 64), 15, dtype=torch.uint8)
    assert Int4Matrix.from_codes(codes, torch.full((16, 1), 1.9375, dtype=torch.bfloat16), 64).bf16_exact
    assert not Int4Matrix.from_codes(codes, torch.full((16, 1), 1.96875, dtype=torch.bfloat16), 64).bf16_exact


def test_refusals():
    codes, scales = torch.zeros(16, 64, dtype=torch.uint8), torch.ones(16, 1, dtype=torch.bfloat16)
    for bad in ((codes, scales, 48), (codes, scales, 128), (codes.int(), scales, 64), (codes, scales.float(), 64), (codes, scales[:8], 64),
                (codes[:, :32], scales, 64), (codes[0], scales, 64), (codes + 16, scales, 64), (codes[:0], scales[:0], 64)):
        with pytest.raises(ValueError):
            Int4Matrix.from_codes(*bad)
    for bad in ((codes, 64), (scales, 64), (torch.randn(4, 64), 16), (torch.randn(64), 64), (torch.full((4, 64), float("nan")), 64),
                (torch.full((4, 64), float("inf")), 32)):
        with pytest.raises(ValueError):
            Int4Matrix.quantize(*bad)


def test_a_matrix_whose_parts_do_not_fit_its_shape_is_refused():
    """The kernels read codes and scales by the shape: anything shorter, or of another type, would be read beyond its end."""
    w = Int4Matrix.from_codes(torch.zeros(40, 192, dtype=torch.uint8), torch.ones(40, 3, dtype=torch.bfloat16), 64)
    again = Int4Matrix(w.packed, w.scales, w.shape, w.group, w.bf16_exact)
    assert again.shape == (40, 192) and torch.equal(unpacked(again), unpacked(w))
    for bad in ((w.packed[:-512], w.scales, w.shape, 64), (w.packed, w.scales[:-1], w.shape, 64), (w.packed, w.scales, (64, 192), 64), (w.packed, w.scales, (40, 256), 64),
                (w.packed, w.scales, w.shape, 32), (w.packed, w.scales, w.shape, 48), (w.packed, w.scales, (0, 192), 64), (w.packed, w.scales, (40, 160), 64),
                (w.packed.to(torch.int8), w.scales, w.shape, 64), (w.packed, w.scales.float(), w.shape, 64), (w.packed.repeat(2)[::2], w.scales, w.shape, 64),
                (w.packed, w.scales.to("meta"), w.shape, 64), (w.packed, w.scales, (40,), 64)):
        with pytest.raises(ValueError):
            Int4Matrix(*bad, True)
