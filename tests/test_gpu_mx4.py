"""4-bit floats with shared scales against their definition in 64 bits: quantisation exactly, the linear layer within
the rounding of its float32 sums."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantized(x):
    """x float64 [rows, cols] -> the values it stands for: the nearest of VALUES times the block's scale, the even code on
    ties, by comparing distances."""
    rows, cols = x.shape
    padded = np.zeros((rows, -(-cols // 32) * 32))
    padded[:, :cols] = x
    v = padded.reshape(rows, padded.shape[1] // 32, 32)
    bad = ~np.isfinite(v).all(axis=2)
    top = np.abs(np.where(np.isfinite(v), v, 0.0)).max(axis=2)
    exponent = np.frexp(top)[1] - 3
    scale = np.ldexp(1.0, np.maximum(np.where(top > 0, exponent, 0), -127))
    y = np.abs(np.where(np.isfinite(v), v, 0.0)) / scale[..., None]
    y = np.minimum(y, 6.0)
    order = [0, 2, 4, 6, 1, 3, 5, 7]                                   # argmin takes the first: even codes win ties
    dist = np.abs(y[..., None] - VALUES[order])
    code = np.array(order)[dist.argmin(axis=-1)]
    out = np.copysign(VALUES[code], v) * scale[..., None]
    out[bad] = np.nan
    return out.reshape(padded.shape)[:, :cols]


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X (torch.cuda.is_available() is False)")
    return torch


def _same(got, want):
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64)
    assert got.shape == want.shape
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.nan_to_num(got), np.nan_to_num(want))


SHAPES = [(1, 1), (1, 31), (1, 33), (2, 32), (3, 128), (5, 129), (17, 255), (4, 257), (3, 511), (9, 513), (2, 1000), (7, 11520),
          (333, 1001), (1000, 40)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_equals_its_definition(shape, dtype):
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(shape[0] * 7919 + shape[1])
    x = (torch.randn(shape, generator=g) * torch.exp(3 * torch.randn(shape[0], 1, generator=g))).to(getattr(torch, dtype))
    q = mx4.quantize(x.cuda())
    _same(q.dequantize().cpu(), quantized(x.double().numpy()))
    units = (-(-shape[0] // 32), -(-shape[1] // 256))
    assert q.codes.shape == units + (4096,) and q.scales.shape == units + (256,)
    # padding multiplies as zero: [unit, 2 k-steps of 64.., half, row, 16 bytes] back to rows
    full = q.codes.reshape(units + (4, 2, 32, 16)).permute(0, 4, 1, 2, 3, 5).reshape(units[0] * 32, units[1] * 128).cpu()
    assert not full[shape[0]:].any() and not full[:, -(-shape[1] // 32) * 16:].any()


def test_quantize_every_half_and_every_bfloat16():
    torch = _torch()
    from alphazero_amd import mx4
    for dtype in (torch.float16, torch.bfloat16):
        bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
        x = bits.view(dtype).reshape(-1, 32)                           # neighbours share a block
        _same(mx4.quantize(x.cuda()).dequantize().cpu(), quantized(x.double().numpy()))
        # every value under the scale of a fixed neighbour: all alignments of value and scale
        finite = x.reshape(-1)[torch.isfinite(x.reshape(-1).float())]
        for top in (1.0, 1.5, 2.0 ** -10, 0.0):
            y = torch.zeros(finite.numel(), 32, dtype=dtype)
            y[:, 7] = finite
            y[:, 20] = top
            _same(mx4.quantize(y.cuda()).dequantize().cpu(), quantized(y.double().numpy()))


def test_quantize_ties_saturation_and_extreme_scales():
    torch = _torch()
    from alphazero_amd import mx4
    borders = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.0, 7.5, 7.999]
    row = []
    for b in borders:
        row += [b, -b, np.nextafter(np.float32(b), np.float32(0)), np.nextafter(np.float32(b), np.float32(9))]
    base = np.zeros((40, 64), dtype=np.float32)
    base[:, :len(row)] = row
    base[:, 31] = base[:, 63] = 4.0                                    # both blocks have the scale 1
    exps = np.array([0, 1, -1, 20, -20, 100, 125, -100, -120, -124, -125, -126, -127, -128, -130, -140, -149] + [0] * 23)
    with np.errstate(over="ignore"):
        x = np.ldexp(base, exps[:, None]).astype(np.float32)
    x[20] = 0.0
    x[21, 3], x[22, 40], x[23, 5] = np.nan, np.inf, -np.inf
    x[24] = -0.0
    t = torch.from_numpy(x)
    _same(mx4.quantize(t.cuda()).dequantize().cpu(), quantized(x.astype(np.float64)))


def test_quantize_strided_views():
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(5)
    base = torch.randn(70, 200, generator=g).cuda()
    views = [base.t(), base[:, 3:150], base[::2, ::3], base[:1].expand(6, 200), base[:, :1].expand(70, 64), base.flip(0),
             base[5], base.view(7, 10, 200), base.view(7, 10, 200).transpose(0, 1), base[:0], base.half()[:, 8:136],
             base.bfloat16()[:, 1:]]
    for v in views:
        q = mx4.quantize(v)
        assert q.shape == v.shape
        _same(q.dequantize().cpu().reshape(-1, v.shape[-1]), quantized(v.cpu().double().reshape(-1, v.shape[-1]).numpy()))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_dequantize_rounds_once(dtype):
    torch = _torch()
    from alphazero_amd import mx4
    x = torch.randn(5, 77, generator=torch.Generator().manual_seed(1)) * torch.tensor([[1.0], [1e-9], [1e4], [1e-7], [1e30]])
    q = mx4.quantize(x.cuda())
    want = torch.from_numpy(quantized(x.double().numpy())).to(getattr(torch, dtype))
    _same(q.dequantize(getattr(torch, dtype)).double().cpu(), want.double())


def _linear_reference(x, w, bias, relu):
    """float64 result and the sum of absolute products that bounds its rounding."""
    xq, wq = quantized(x.double().cpu().reshape(-1, x.shape[-1]).numpy()), quantized(w.double().cpu().numpy())
    y, size = xq @ wq.T, np.abs(xq) @ np.abs(wq).T
    if bias is not None:
        y, size = y + bias.double().cpu().numpy(), size + np.abs(bias.double().cpu().numpy())
    return np.where(y < 0, 0.0, y) if relu else y, size


def _check_linear(got, x, w, bias, relu):
    """Products are exact.  A sum passes through one accumulation per 128 elements, at most 32 additions within such a
    step, 16 joins of partial sums and the bias: each costs at most 2^-23 of the running absolute sum (a truncated
    float32 addition).  The result is rounded once to its own type: half a step."""
    want, size = _linear_reference(x, w, bias, relu)
    steps = -(-x.shape[-1] // 128) + 32 + 16 + 1
    half_step = {"torch.float32": 2.0 ** -24, "torch.float16": 2.0 ** -11, "torch.bfloat16": 2.0 ** -8}[str(got.dtype)]
    tol = steps * 2.0 ** -23 * size + half_step * np.abs(want) + 2.0 ** -25 * (got.element_size() == 2)
    g = got.double().cpu().reshape(want.shape).numpy()
    np.testing.assert_array_equal(np.isnan(g), np.isnan(want))
    bad = np.abs(np.nan_to_num(g - want)) > np.nan_to_num(tol)
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(np.nan_to_num(g - want)).max())


ROWS = [1, 2, 7, 16, 17, 33, 64, 65, 130, 300]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("cols,out", [(1, 1), (32, 16), (129, 63), (500, 200), (1500, 97), (11520, 40), (2048, 300)])
def test_linear_against_float64(rows, cols, out):
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(rows * 100003 + cols * 17 + out)
    x, w, b = torch.randn(rows, cols, generator=g), torch.randn(out, cols, generator=g), torch.randn(out, generator=g)
    weight = mx4.quantize(w.cuda())
    for dtype, bias, relu, out_dtype in ((torch.float32, b, True, torch.float32), (torch.bfloat16, None, False, torch.bfloat16),
                                         (torch.float16, b.half(), False, torch.float32)):
        xi = x.to(dtype)
        got = mx4.linear(xi.cuda(), weight, bias=None if bias is None else bias.cuda(), relu=relu, out_dtype=out_dtype)
        assert got.shape == (rows, out) and got.dtype == out_dtype
        _check_linear(got, xi, w, bias, relu)


@pytest.mark.parametrize("rows,cols,out", [(1000, 1024, 1024), (517, 11520, 1024), (2500, 640, 777), (300, 4096, 4100)])
def test_linear_large(rows, cols, out):
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(rows + cols + out)
    x, w, b = torch.randn(rows, cols, generator=g).half(), torch.randn(out, cols, generator=g), torch.randn(out, generator=g)
    got = mx4.linear(x.cuda(), mx4.quantize(w.cuda()), bias=b.cuda(), relu=True, out_dtype=torch.float32)
    _check_linear(got, x, w, b, True)


def test_linear_on_quantized_rows_equals_linear_on_numbers():
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(3)
    for rows in (1, 3, 20, 200, 700):
        x, w = torch.randn(rows, 700, generator=g).cuda(), torch.randn(150, 700, generator=g).cuda()
        weight = mx4.quantize(w)
        a, b = mx4.linear(x, weight), mx4.linear(mx4.quantize(x), weight)
        assert torch.equal(a, b)
        assert torch.equal(a, mx4.linear(x, weight))                   # the same call gives the same bits


def test_linear_does_not_depend_on_the_other_rows():
    """A row's outputs are the same bits in a call of one kernel form whatever rows stand beside it."""
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(4)
    x, weight = torch.randn(600, 1000, generator=g).cuda(), mx4.quantize(torch.randn(200, 1000, generator=g).cuda())
    y = mx4.linear(x, weight)
    z = mx4.linear(x.flip(0), weight).flip(0)
    assert torch.equal(y, z)


def test_linear_shapes_strides_and_out():
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(6)
    w = torch.randn(50, 96, generator=g)
    weight = mx4.quantize(w.cuda())
    base = torch.randn(96, 24, generator=g)
    for x in (base.t(), base.t()[::2], base.t().reshape(2, 3, 4, 96), base.t()[3], base.t()[:0], base.t()[:1].expand(5, 96)):
        got = mx4.linear(x.cuda() if x.numel() else x.cuda(), weight)
        assert got.shape == tuple(x.shape[:-1]) + (50,)
        if x.numel():
            _check_linear(got, x, w, None, False)
    wide = torch.full((24, 64), 7.0, device="cuda")
    got = mx4.linear(base.t().cuda(), weight, out=wide[:, 5:55])
    _check_linear(got, base.t(), w, None, False)
    assert (wide[:, :5] == 7).all() and (wide[:, 55:] == 7).all()      # columns beside the output are left alone
    empty = mx4.quantize(torch.zeros(0, 96, device="cuda"))
    assert mx4.linear(base.t().cuda(), empty).shape == (24, 0)


def test_linear_infinities_and_nan_reach_the_output():
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(8)
    for rows in (5, 300):
        x, w = torch.randn(rows, 200, generator=g), torch.randn(70, 200, generator=g)
        x[2, 150], x[4, 10] = float("nan"), float("inf")
        w[33, 7] = float("-inf")
        for relu in (False, True):
            got = mx4.linear(x.cuda(), mx4.quantize(w.cuda()), relu=relu)
            _check_linear(got, x, w, None, relu)
            assert got[2].isnan().all() and got[4].isnan().all() and got[:, 33].isnan().all()


def test_linear_small_and_large_scales():
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(9)
    for rows in (3, 200):
        for sx, sw in ((1e-30, 1e25), (1e20, 1e-35), (1e-38, 1.0), (1e18, 1e18)):
            x = (torch.randn(rows, 320, generator=g).double() * sx).float()
            w = (torch.randn(33, 320, generator=g).double() * sw).float()
            got = mx4.linear(x.cuda(), mx4.quantize(w.cuda()))
            want, size = _linear_reference(x, w, None, False)
            # results below the normal range may lose what lies under it: one smallest step per accumulation
            tol = (320 // 128 + 50) * (2.0 ** -23 * size + 2.0 ** -126)
            assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


def test_streams_and_graph():
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator().manual_seed(10)
    x, w, b = torch.randn(100, 600, generator=g).cuda(), torch.randn(300, 600, generator=g).cuda(), torch.randn(300, generator=g).cuda()
    want = mx4.linear(x, mx4.quantize(w), bias=b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mx4.linear(x, mx4.quantize(w), bias=b)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    xs, ws = x.clone(), w.clone()
    with torch.cuda.graph(graph):
        out = mx4.linear(xs, mx4.quantize(ws), bias=b)
    for k in range(4):
        xs.copy_(x * (k + 1))
        ws.copy_(w.roll(k, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mx4.linear(x * (k + 1), mx4.quantize(w.roll(k, 0)), bias=b))


def test_large_offsets():
    """More than 2^31 elements in x: rows behind that border are read from the right place."""
    torch = _torch()
    from alphazero_amd import mx4
    cols = 65536
    x = torch.zeros(32769 + 3, cols, dtype=torch.float16, device="cuda")
    g = torch.Generator().manual_seed(11)
    tail = torch.randn(4, cols, generator=g).half()
    x[-4:] = tail.cuda()
    w = torch.randn(20, cols, generator=g)
    got = mx4.linear(x, mx4.quantize(w.cuda()), out_dtype=torch.float32)
    assert not got[:-4].any()
    _check_linear(got[-4:], tail, w, None, False)


@pytest.mark.parametrize("rows,cols,out", [(32768, 200, 32800), (20000, 500, 30000), (5000, 4096, 5001), (6000, 11000, 6100)])
def test_linear_largest_tiles(rows, cols, out):
    """Sizes at which 256 x 256 tiles multiply, with one stage of K, two, many and an odd number.  Rows from the start, the
    middle and the end against float64 sums of the rounded operands, with the bounds of the smaller cases."""
    torch = _torch()
    from alphazero_amd import mx4
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, w = torch.randn(rows, cols, generator=g, device="cuda"), torch.randn(out, cols, generator=g, device="cuda")
    rounded, weight = mx4.quantize(x), mx4.quantize(w)
    y = mx4.linear(x, weight, out_dtype=torch.bfloat16)
    xq, wq = rounded.dequantize(), weight.dequantize().double().t().contiguous()
    steps = -(-cols // 128) + 32 + 16 + 1
    for first in (0, rows // 2 - 40, rows - 130):
        part = xq[first:first + 130].double()
        want, size = part @ wq, part.abs() @ wq.abs()
        assert ((y[first:first + 130].double() - want).abs() <= steps * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all()
