"""What the training and low-precision operators are timed on, and their plain forms.

Four operators:

  orthogonalize  a matrix (or a batch of them) pushed towards the nearest orthogonal one by a few Newton-Schulz
                 products, what an orthogonalised-momentum optimiser does to its updates
  muon           one optimiser step on a list of matrices: momentum, orthogonalisation, weight update
  quantize       rows of numbers to 4-bit floats (e2m1) with a power-of-two scale for every 32, and back
  linear         a linear layer with weights kept in that form: the rows are quantised on the way in, the products
                 are formed in 4 bits and summed in float32, bias and ReLU follow

`run` computes them with elementary torch operations where `own` is false and calls the package where it is true.
"""
import math

import torch

own = False

F32, F16, BF16 = "float32", "float16", "bfloat16"
BLOCK = 32                                     # values that share a scale
COEFFICIENTS = (3.4445, -4.7750, 2.0315)       # the quintic of one Newton-Schulz step
STEPS = 5
EPS = 1e-7
LR, MOMENTUM, WEIGHT_DECAY = 0.02, 0.95, 0.01

# Connect4Net's weight tensors as matrices (output channels x everything else): its three convolutions and its
# linear layer.  The heads and the biases are not orthogonalised.
CONNECT4NET = "128x32,128x2048,128x2048,1024x11520"


def _matrices(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def listed():
    return [
        # the first convolution's weights: the smallest call, bound by latency
        dict(name="orthogonalize_conv0", op="orthogonalize", batch=1, rows=128, cols=32, dtype=F32, layout="rows"),
        # the two 128 -> 128 convolutions together
        dict(name="orthogonalize_conv_pair", op="orthogonalize", batch=2, rows=128, cols=2048, dtype=F32, layout="rows"),
        # the linear layer, nine tenths of the network's weights
        dict(name="orthogonalize_fc", op="orthogonalize", batch=1, rows=1024, cols=11520, dtype=F32, layout="rows"),
        # sizes that fit no tile, in bfloat16, columns the longer side of a transposed view
        dict(name="orthogonalize_ragged", op="orthogonalize", batch=3, rows=1501, cols=777, dtype=BF16, layout="columns"),
        # one optimiser step of the whole network, as training makes it
        dict(name="muon_network", op="muon", shapes=CONNECT4NET, dtype=F32, nesterov=True),
        # a handful of odd matrices kept in bfloat16
        dict(name="muon_odd", op="muon", shapes="7x1024,65x130,300x211,33x33,515x129", dtype=BF16, nesterov=False),
        # what the convolutions hand the linear layer for a full leaf batch
        dict(name="quantize_activations", op="quantize", rows=4096, cols=11520, dtype=F16, values="relu"),
        # few short rows whose last block is cut
        dict(name="quantize_ragged", op="quantize", rows=333, cols=1001, dtype=BF16, values="normal"),
        # one position: the linear layer of a single evaluation
        dict(name="linear_one_row", op="linear", rows=1, cols=11520, out=1024, dtype=F32, out_dtype=F32, bias=True,
             relu=True, values="relu"),
        # a full leaf batch
        dict(name="linear_leaf_batch", op="linear", rows=4096, cols=11520, out=1024, dtype=F16, out_dtype=F32, bias=True,
             relu=True, values="relu"),
        # sizes that fit no tile
        dict(name="linear_ragged", op="linear", rows=77, cols=1500, out=2111, dtype=BF16, out_dtype=BF16, bias=True,
             relu=False, values="normal"),
        # the largest: a wide layer over many rows
        dict(name="linear_wide", op="linear", rows=8192, cols=8192, out=8192, dtype=BF16, out_dtype=BF16, bias=False,
             relu=False, values="normal"),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _orthogonalize_flops(rows, cols):
    """Newton-Schulz can run on the small Gram matrix: one symmetric product over the long side, one product to
    apply the result, and per step products of symmetric matrices (half of each computed)."""
    m, n = min(rows, cols), max(rows, cols)
    return 3.0 * m * m * n + (4 * STEPS - 3) * float(m) ** 3


def draw(rng):
    op = rng.choice(["orthogonalize", "muon", "quantize", "linear", "linear"])
    dtype = rng.choice([F32, F16, BF16])
    if op == "orthogonalize":
        while True:
            batch, rows, cols = _spread(rng, 1, 16), _spread(rng, 1, 2048), _spread(rng, 1, 11520)
            if batch * _orthogonalize_flops(rows, cols) <= _orthogonalize_flops(1024, 11520):
                break
        if rng.random() < 0.3:
            rows, cols = cols, rows
        return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=dtype, layout=rng.choice(["rows", "columns", "padded"]))
    if op == "muon":
        shapes, flops = [], 0.0
        for _ in range(rng.randint(1, 12)):
            rows, cols = _spread(rng, 1, 1024), _spread(rng, 1, 4096)
            if rng.random() < 0.3:
                rows, cols = cols, rows
            flops += _orthogonalize_flops(rows, cols)
            if flops <= _orthogonalize_flops(1024, 11520):
                shapes.append("%dx%d" % (rows, cols))
        return dict(op=op, shapes=",".join(shapes or ["64x96"]), dtype=rng.choice([F32, BF16]), nesterov=rng.random() < 0.5)
    if op == "quantize":
        while True:
            rows, cols = _spread(rng, 1, 16384), _spread(rng, 1, 16384)
            if rows * cols <= 4096 * 11520:
                break
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, values=rng.choice(["relu", "normal"]))
    while True:
        rows, cols, out = _spread(rng, 1, 8192), _spread(rng, 1, 16384), _spread(rng, 1, 8192)
        if rows * cols * out <= 8192 ** 3:
            break
    return dict(op=op, rows=rows, cols=cols, out=out, dtype=dtype, out_dtype=rng.choice([F32, dtype]),
                bias=rng.random() < 0.5, relu=rng.random() < 0.5, values=rng.choice(["relu", "normal"]))


# ---------------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _gradient(g, rows, cols, batch=()):
    """Like a gradient: rows and columns of different sizes, a thousandth in scale."""
    x = torch.randn(*batch, rows, cols, generator=g, device="cuda")
    r = torch.exp(0.5 * torch.randn(*batch, rows, 1, generator=g, device="cuda"))
    c = torch.exp(0.5 * torch.randn(*batch, 1, cols, generator=g, device="cuda"))
    return x.mul_(r).mul_(c).mul_(1e-3)


def _rows_of(g, case):
    """Layer inputs: normal with sizes that differ by feature, or the same behind a ReLU."""
    x = torch.randn(case["rows"], case["cols"], generator=g, device="cuda")
    x.mul_(torch.exp(0.7 * torch.randn(1, case["cols"], generator=g, device="cuda")))
    if case["values"] == "relu":
        x.clamp_(min=0.0)
    return x.to(getattr(torch, case["dtype"]))


def prepare(case, seed):
    g = _generator(seed)
    dtype = getattr(torch, case["dtype"])
    state = dict(case=case)
    if case["op"] == "orthogonalize":
        x = _gradient(g, case["rows"], case["cols"], (case["batch"],)).to(dtype)
        if case["layout"] == "columns":                       # a transposed view of row-major memory
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif case["layout"] == "padded":                      # columns of a wider buffer
            wide = torch.zeros(case["batch"], case["rows"], case["cols"] + 9, dtype=dtype, device="cuda")
            wide[:, :, 5:5 + case["cols"]] = x
            x = wide[:, :, 5:5 + case["cols"]]
        state["x"] = x
    elif case["op"] == "muon":
        state["grads"], state["weights"], state["momenta"] = [], [], []
        for rows, cols in _matrices(case):
            state["grads"].append(_gradient(g, rows, cols).to(dtype))
            w = torch.empty(rows, cols, device="cuda").uniform_(-1.0, 1.0, generator=g).mul_(1.0 / math.sqrt(cols))
            state["weights"].append(w.to(dtype))
            state["momenta"].append(_gradient(g, rows, cols).mul_(4.0))
    else:
        state["x"] = _rows_of(g, case)
        if case["op"] == "linear":
            w = torch.randn(case["out"], case["cols"], generator=g, device="cuda").mul_(1.0 / math.sqrt(case["cols"]))
            w = w.to(dtype)
            state["bias"] = torch.randn(case["out"], generator=g, device="cuda").mul_(0.1) if case["bias"] else None
            if own:
                from alphazero_amd import mx4
                state["weight"] = mx4.quantize(w)
            else:
                state["weight"] = _quantized_values(w)        # the values the 4-bit weights stand for
    return state


# ----------------------------------------------------------------------------------------------- plain forms

def _newton_schulz(x):
    """x float32 [..., rows, cols]."""
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2).contiguous()
    norm = torch.sqrt((x.double() * x.double()).sum(dim=(-2, -1), keepdim=True)) + EPS
    x = x / norm.float()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2) if tall else x


def _quantized_values(x):
    """The values x [rows, cols] stands for after quantisation, float32: blocks of 32 along the columns share the
    scale 2^(floor(log2 max|x|) - 2); an element over its scale goes to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6
    (ties to the even code, larger ones to 6)."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).reshape(rows, -1, BLOCK)
    exponent = torch.frexp(v.abs().amax(dim=2, keepdim=True)).exponent - 3
    exponent = exponent.clamp(min=-127)
    y = torch.ldexp(v, -exponent)
    size = y.abs().clamp(max=6.0)
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0))
    size = torch.round(size / step) * step                     # round() takes ties to even
    return torch.ldexp(torch.copysign(size, y), exponent).reshape(rows, -1)[:, :cols]


def _muon_scale(rows, cols):
    return math.sqrt(max(1.0, rows / cols))


def _run_plain(state):
    case = state["case"]
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "orthogonalize":
        return _newton_schulz(state["x"].float()).to(dtype)
    if case["op"] == "muon":
        weights, momenta = [], []
        for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
            g = g.float()
            m = MOMENTUM * m + g
            u = _newton_schulz(g + MOMENTUM * m if case["nesterov"] else m)
            w = w.float() * (1.0 - LR * WEIGHT_DECAY) - (LR * _muon_scale(*w.shape)) * u
            weights.append(w.to(dtype))
            momenta.append(m)
        return dict(weights=weights, momenta=momenta)
    if case["op"] == "quantize":
        return _quantized_values(state["x"])
    y = _quantized_values(state["x"]) @ state["weight"].t()
    if state["bias"] is not None:
        y = y + state["bias"]
    if case["relu"]:
        y = torch.relu(y)
    return y.to(getattr(torch, case["out_dtype"]))


def _run_own(state):
    from alphazero_amd import mx4, optim
    case = state["case"]
    if case["op"] == "orthogonalize":
        return optim.orthogonalize(state["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    if case["op"] == "muon":
        weights, momenta = optim.muon_update(state["weights"], state["grads"], state["momenta"], lr=LR, momentum=MOMENTUM,
                                             nesterov=case["nesterov"], weight_decay=WEIGHT_DECAY, steps=STEPS,
                                             coefficients=COEFFICIENTS, eps=EPS, inplace=False)
        return dict(weights=weights, momenta=momenta)
    if case["op"] == "quantize":
        return mx4.quantize(state["x"]).dequantize()
    return mx4.linear(state["x"], state["weight"], bias=state["bias"], relu=case["relu"],
                      out_dtype=getattr(torch, case["out_dtype"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------- exact

def _exact_polar_steps(x):
    """The same polynomial in float64, x [rows, cols]: a x + b (x x') x + c (x x')^2 x, five times."""
    x = x / (torch.linalg.vector_norm(x) + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        if x.shape[0] <= x.shape[1]:
            g = x.mm(x.t())
            y = g.mm(x)
            x = a * x + b * y + c * g.mm(y)
        else:
            g = x.t().mm(x)
            y = x.mm(g)
            x = a * x + b * y + c * y.mm(g)
    return x


def _exact_quantized(x):
    """Nearest representable value by comparing with the borders between them, float64."""
    rows, cols = x.shape
    padded = torch.zeros(rows, -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    padded[:, :cols] = x
    v = padded.view(rows, -1, BLOCK)
    top = v.abs().max(dim=2, keepdim=True).values
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -127))) - 2.0).clamp(min=2.0 ** -127)
    # a logarithm can land on the wrong side of a power of two
    scale = torch.where(scale * 8.0 <= top, scale * 2.0, scale)
    scale = torch.where((scale * 4.0 > top) & (scale > 2.0 ** -127), scale * 0.5, scale)
    size = (v / scale).abs()
    # values 0 0.5 1 1.5 2 3 4 6; a border belongs to the neighbour with the even code: 0, 1, 2, 4
    out = torch.zeros_like(size)
    for value, border, upper in ((0.5, 0.25, False), (1.0, 0.75, True), (1.5, 1.25, False), (2.0, 1.75, True),
                                 (3.0, 2.5, False), (4.0, 3.5, True), (6.0, 5.0, False)):
        out = torch.where((size >= border) if upper else (size > border), value, out)
    return (out * torch.sign(v) * scale).view(rows, -1)[:, :cols]


def exact(case, seed):
    if case["op"] == "orthogonalize":
        x = prepare(case, seed)["x"].double()
        return torch.stack([_exact_polar_steps(x[i]) for i in range(case["batch"])])
    if case["op"] == "muon":
        state = prepare(case, seed)
        weights, momenta = [], []
        for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
            m = m.double() * MOMENTUM + g.double()
            u = m * MOMENTUM + g.double() if case["nesterov"] else m
            scale = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
            weights.append((1.0 - LR * WEIGHT_DECAY) * w.double() - LR * scale * _exact_polar_steps(u))
            momenta.append(m)
        return dict(weights=weights, momenta=momenta)
    if case["op"] == "quantize":
        return _exact_quantized(prepare(case, seed)["x"].double())
    g = _generator(seed)
    x = _rows_of(g, case)
    w = torch.randn(case["out"], case["cols"], generator=g, device="cuda").mul_(1.0 / math.sqrt(case["cols"]))
    w = w.to(x.dtype)
    bias = torch.randn(case["out"], generator=g, device="cuda").mul_(0.1) if case["bias"] else None
    y = torch.mm(_exact_quantized(x.double()), _exact_quantized(w.double()).t())
    if bias is not None:
        y += bias.double()
    return y.clamp(min=0.0) if case["relu"] else y


# ------------------------------------------------------------------------------------------------------ work

def _size(dtype):
    return 4 if dtype == F32 else 2


def work(case):
    s = _size(case["dtype"])
    if case["op"] == "orthogonalize":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * s * n, "flops": case["batch"] * _orthogonalize_flops(case["rows"], case["cols"])}
    if case["op"] == "muon":
        n = sum(r * c for r, c in _matrices(case))
        # gradient, weight and momentum in; weight and momentum out
        return {"bytes": (3 * s + 8) * n, "flops": sum(_orthogonalize_flops(r, c) for r, c in _matrices(case))}
    n = case["rows"] * case["cols"]
    packed = lambda rows, cols: rows * -(-cols // BLOCK) * (BLOCK // 2 + 1)
    if case["op"] == "quantize":
        # the packed form is written and read on the way to the values
        return {"bytes": s * n + 2 * packed(case["rows"], case["cols"]) + 4 * n, "flops": 4.0 * n}
    o = _size(case["out_dtype"])
    return {"bytes": s * n + packed(case["out"], case["cols"]) + o * case["rows"] * case["out"]
            + (4 * case["out"] if case["bias"] else 0), "flops": 2.0 * n * case["out"]}
