"""Orthogonalised-momentum optimiser (Muon) on hand-written kernels.

A weight matrix's update is its momentum pushed towards the nearest orthogonal matrix by a few Newton-Schulz products,
so that all its directions are learned at one rate.  `Muon` is a torch optimiser for matrices (a convolution's weight
counts as output channels x everything else); biases, heads and embeddings belong to another optimiser.

    matrices, rest = optim.split_parameters(agent.model)
    muon, adam = optim.Muon(matrices, lr=0.02), torch.optim.Adam(rest)

The kernels run on the tensors' device, on torch's current stream there, and wait for nothing.  They can be captured into
a graph, which then keeps the learning rate and the other numbers of the call it recorded; `Muon` makes its momenta in its
first step, which has to come before the capture.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Sequence

import torch

from . import _lib
from ._lib import NS_MAX_STEPS, MuonMatrix, MuonParams, NewtonSchulz, NnbError, check
from ._tensors import dtype_code, no_grad, no_tangent, on_device, overlaps_itself, ptr, resolved, share_memory, stream_of, writable

QUINTIC = (3.4445, -4.7750, 2.0315)


def _newton_schulz(steps: int, coefficients, eps: float) -> NewtonSchulz:
    steps = int(steps)
    if not 1 <= steps <= NS_MAX_STEPS:
        raise ValueError(f"steps must be in [1, {NS_MAX_STEPS}], got {steps}")
    rows = list(coefficients)
    if rows and not hasattr(rows[0], "__len__"):
        rows = [rows] * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError("coefficients must be one triple (a, b, c) or one for every step")
    ns = NewtonSchulz(steps=steps, eps=float(eps))
    for i, row in enumerate(rows):
        for j in range(3):
            ns.coefficients[i][j] = float(row[j])
    return ns


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def orthogonalize(x: torch.Tensor, steps: int = 5, coefficients=QUINTIC, eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., rows, cols] (float32, float16 or bfloat16, any strides) divided by its Frobenius norm (+ eps), then `steps`
    times X <- a X + b (X X^T) X + c (X X^T)^2 X: the singular values go towards 1, the singular vectors stay.

    float32-faithful inside whatever the type, one rounding at the end.  A matrix with a NaN or an infinity gives NaN.
    `out` (same shape and type; x itself, or no element in common with it) is written instead of a new tensor when given.
    No derivatives."""
    code = dtype_code(x, "x")
    no_grad("optim.orthogonalize", x, out)
    if x.dim() < 2:
        raise ValueError(f"x of shape {tuple(x.shape)} is no matrix")
    ns = _newton_schulz(steps, coefficients, eps)
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype or out.device != x.device):
        raise ValueError(f"out is {out.dtype} {tuple(out.shape)} on {out.device}, expected {x.dtype} {tuple(x.shape)} on {x.device}")
    given = out
    if out is not None:
        writable(out, "out")
        if overlaps_itself(out):
            raise ValueError("out has elements that share memory")
    if out is not None and not (out.data_ptr() == x.data_ptr() and out.stride() == x.stride()) and share_memory(out, x):
        raise ValueError("out shares memory with x but is not x")
    with on_device(x):
        x = resolved(x.detach())
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        rows, cols = x.shape[-2:]
        xb = x if x.dim() == 3 else x.reshape((-1, rows, cols) if x.numel() else (0, rows, cols))
        try:
            ob = out if out.dim() == 3 else out.view((-1, rows, cols) if x.numel() else (0, rows, cols))
        except RuntimeError:
            raise ValueError(f"out of shape {tuple(out.shape)}, strides {out.stride()} is no evenly spaced batch of matrices") from None
        lib = _lib.load()
        nbytes = C.c_size_t()
        check(lib.nnb_orthogonalize_workspace_bytes(xb.shape[0], rows, cols, C.byref(nbytes)), "nnb_orthogonalize_workspace_bytes")
        workspace = _workspace(nbytes.value, x.device)
        strides = C.c_int64 * 3
        check(lib.nnb_orthogonalize(stream_of(x), code, xb.shape[0], rows, cols, ptr(xb), strides(*xb.stride()), ptr(ob),
                                    strides(*ob.stride()), C.byref(ns), ptr(workspace), nbytes.value), "nnb_orthogonalize")
    if given is not None:
        torch.autograd.graph.increment_version(given)             # the kernels write behind torch's back
    return out


def _as_matrix(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() < 2:
        raise ValueError(f"{name} of shape {tuple(t.shape)} is no matrix")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return resolved(t.detach())


@torch.no_grad()
def muon_update(weights: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], lr: float,
                momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                coefficients=QUINTIC, eps: float = 1e-7, inplace: bool = True):
    """One optimiser step on a list of matrices (a tensor [n, ...] counts as n rows), all together:

        m' = momentum m + g;   u = g + momentum m' (nesterov) or m'
        w' = w (1 - lr weight_decay) - lr max(1, rows / cols)^(1/2) orthogonalize(u)

    A matrix's precision goes by its own size; what else is in the call can only change the order of its sums.

    weights and grads of one type (float32, float16, bfloat16), momenta float32, all contiguous on one device, without
    elements in common.  Returns
    (weights, momenta): the given tensors, updated, or new ones with inplace=False."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    if not len(weights) == len(grads) == len(momenta):
        raise ValueError(f"{len(weights)} weights, {len(grads)} gradients and {len(momenta)} momenta")
    ns = _newton_schulz(steps, coefficients, eps)
    if not weights:
        return weights, momenta
    first = weights[0]
    code = dtype_code(first, "weights[0]")
    no_tangent("optim.muon_update", *weights, *grads, *momenta)
    for i, (w, g, m) in enumerate(zip(weights, grads, momenta)):
        if w.dtype != first.dtype or g.dtype != first.dtype or m.dtype != torch.float32:
            raise ValueError(f"matrix {i}: weight {w.dtype}, gradient {g.dtype}, momentum {m.dtype}; expected {first.dtype}, "
                             f"{first.dtype}, torch.float32")
        if w.shape != g.shape or w.shape != m.shape:
            raise ValueError(f"matrix {i}: weight {tuple(w.shape)}, gradient {tuple(g.shape)}, momentum {tuple(m.shape)}")
        if any(t.device != first.device for t in (w, g, m)):
            raise ValueError(f"matrix {i}: all tensors must be on {first.device}")
    if inplace:
        for name, ts in (("weights", weights), ("momenta", momenta)):
            for i, t in enumerate(ts):
                writable(t, f"{name}[{i}]")
        used = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), written)
                      for ts, written in ((weights, True), (momenta, True), (grads, False)) for t in ts if t.numel())
        any_end = written_end = 0                     # how far the ranges so far reach, and the written ones among them
        for start, end, written in used:
            if start < written_end or (written and start < any_end):
                raise ValueError("a weight or momentum shares memory with another tensor of the call")
            any_end = max(any_end, end)
            if written:
                written_end = max(written_end, end)
    with on_device(first):
        wv = [_as_matrix(t, f"weights[{i}]") for i, t in enumerate(weights)]
        gv = [_as_matrix(t, f"grads[{i}]") for i, t in enumerate(grads)]
        mv = [_as_matrix(t, f"momenta[{i}]") for i, t in enumerate(momenta)]
        w_out = weights if inplace else [torch.empty_like(t) for t in wv]
        m_out = momenta if inplace else [torch.empty_like(t) for t in mv]
        items = (MuonMatrix * len(wv))()
        for it, w, g, m, wo, mo in zip(items, wv, gv, mv, w_out, m_out):
            it.weight, it.grad, it.momentum = w.data_ptr(), g.data_ptr(), m.data_ptr()
            it.weight_out, it.momentum_out = wo.data_ptr(), mo.data_ptr()
            it.rows = w.shape[0]
            it.cols = w.numel() // w.shape[0] if w.shape[0] else 0
        params = MuonParams(lr=float(lr), momentum=float(momentum), weight_decay=float(weight_decay),
                            nesterov=int(bool(nesterov)), ns=ns)
        lib = _lib.load()
        nbytes = C.c_size_t()
        check(lib.nnb_muon_workspace_bytes(len(wv), items, C.byref(nbytes)), "nnb_muon_workspace_bytes")
        workspace = _workspace(nbytes.value, first.device)
        check(lib.nnb_muon_step(stream_of(first), code, len(wv), items, C.byref(params), ptr(workspace), nbytes.value),
              "nnb_muon_step")
    if inplace:
        # the kernels write behind torch's back: whoever watches the version counters (saved tensors, the agent's engine)
        # has to see the change
        for t in weights + momenta:
            torch.autograd.graph.increment_version(t)
    return w_out, m_out


class Muon(torch.optim.Optimizer):
    """Orthogonalised-momentum optimiser for matrices, state "momentum" float32 per parameter (see muon_update)."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients=QUINTIC, eps: float = 1e-7):
        if lr < 0.0 or weight_decay < 0.0 or not 0.0 <= momentum < 1.0:
            raise ValueError(f"lr {lr} and weight_decay {weight_decay} must be >= 0, momentum {momentum} in [0, 1)")
        _newton_schulz(steps, coefficients, eps)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() < 2:
                    raise ValueError(f"a parameter of shape {tuple(p.shape)} is no matrix: give it to another optimiser")
                if p.is_sparse or not p.is_contiguous():
                    raise ValueError(f"a parameter of shape {tuple(p.shape)} is not dense and contiguous")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            batches = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if "momentum" not in self.state[p]:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise NnbError("a new momentum's zeros would be part of the graph: make one step before it is captured")
                    self.state[p]["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                batches.setdefault((p.device, p.dtype), []).append(p)
            for params in batches.values():
                muon_update(params, [p.grad.contiguous() for p in params], [self.state[p]["momentum"] for p in params],
                            lr=group["lr"], momentum=group["momentum"], nesterov=group["nesterov"],
                            weight_decay=group["weight_decay"], steps=group["steps"], coefficients=group["coefficients"],
                            eps=group["eps"])
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but the momentum stays float32: the base class casts state to the parameter's type."""
        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for key, p in zip(saved["params"], group["params"]):
                if "momentum" in state_dict["state"].get(key, {}):
                    self.state[p]["momentum"] = state_dict["state"][key]["momentum"].to(
                        device=p.device, dtype=torch.float32, copy=True).contiguous()


def split_parameters(model: torch.nn.Module) -> tuple:
    """(matrices for Muon, the rest): Connect4Net's hidden weights are orthogonalised, its heads (policy_head,
    value_head) and all biases are not."""
    matrices: List[torch.nn.Parameter] = []
    rest: List[torch.nn.Parameter] = []
    for name, p in model.named_parameters():
        (rest if p.dim() < 2 or "head" in name else matrices).append(p)
    return matrices, rest
