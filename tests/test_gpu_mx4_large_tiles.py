"""The 4-bit product's 256 x 256 tiles at every kind of stage count they are taken for."""
import pytest

# rows, columns, features: 9, 13 and 43 stages of 256 columns (odd counts, whole and cut ones), 8 and 20 (even), rows and
# features that end inside a tile
SIZES = [(8100, 2300, 8192), (4000, 3300, 4090), (4096, 11000, 4096), (8192, 1800, 8192), (8000, 5000, 8189)]
LARGE, TWO_PER_CU = 3, 2


@pytest.mark.parametrize("rows,cols,out", SIZES)
def test_the_sizes_take_large_tiles(rows, cols, out):
    """Or the test below checks another kernel."""
    from alphazero_amd import _lib
    assert _lib.load().nnb_debug_mx4_form(rows, cols, out, 2) == LARGE


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,out", SIZES)
def test_large_tiles_against_float64(rows, cols, out):
    """Rows from the start, the middle and the end against float64 sums of the rounded operands.  Products are exact; a sum
    passes through one accumulation per 128 columns at most, 32 additions within a step and the bias, each off by at most 2^-23
    of the running absolute sum, and is rounded once: half a step."""
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X (torch.cuda.is_available() is False)")
    from alphazero_amd import mx4
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, w = torch.randn(rows, cols, generator=g, device="cuda"), torch.randn(out, cols, generator=g, device="cuda")
    bias = torch.randn(out, generator=g, device="cuda")
    rounded, weight = mx4.quantize(x), mx4.quantize(w)
    y = mx4.linear(x, weight, bias=bias, out_dtype=torch.bfloat16)
    assert y.shape == (rows, out) and torch.equal(y, mx4.linear(rounded, weight, bias=bias, out_dtype=torch.bfloat16))
    xq, wq, b = rounded.dequantize(), weight.dequantize().double().t().contiguous(), bias.double()
    steps = -(-cols // 128) + 32 + 1
    for first in (0, rows // 2 - 40, rows - 130):
        part = xq[first:first + 130].double()
        want, size = part @ wq + b, part.abs() @ wq.abs() + b.abs()
        assert ((y[first:first + 130].double() - want).abs() <= steps * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all()
