"""Orthogonalised updates for the matrices beside the table: adapter factors and projections.

`OverlayAdam` steps table rows, each on its own.  A matrix that maps one space
to another is better stepped as a whole: `orthogonalize` moves all singular
values of an update toward 1 by Newton-Schulz products, `muon_step` is one
optimizer step with it (momentum, Nesterov's update, its orthogonalisation,
the parameter), and `Muon` the torch.optim.Optimizer of it, a matrix or a stack
of matrices (the factors of all loaded adapters) a parameter.  The update rule
and the defaults are those of torch.optim.Muon with its "original" learning-rate
adjustment.  Its products run in more than bf16: matrices with a side of up to 64
are summed in 64 bits, larger ones in operands of 22 bits, within some 1e-4 of
the orthogonalised update's norm (4e-6 in plain fp32); a bf16 update given to
`orthogonalize` takes operands of 11 bits, within 2^-8.  The reference has no
counterpart: its descent trains rows only.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib as L

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_DTYPES = {torch.float32: L.DTYPE_F32, torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_F16}


@functools.lru_cache(maxsize=64)
def _table(coefficients: tuple, steps: int):
    if not coefficients:
        raise ValueError("coefficients: none given")
    rows = coefficients if isinstance(coefficients[0], (tuple, list)) else (coefficients,) * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError(f"coefficients: expected 3 numbers, or 3 for each of the {steps} steps")
    return (C.c_double * (3 * steps))(*[float(v) for r in rows for v in r])


def _coefficients(coefficients, steps: int):
    if not 1 <= steps <= 32:
        raise ValueError(f"steps: {steps}, expected 1 to 32")
    if coefficients is COEFFICIENTS:
        return _table(coefficients, steps)
    return _table(tuple(tuple(c) if isinstance(c, (tuple, list)) else float(c) for c in coefficients), int(steps))


def _stack(x: torch.Tensor, name: str) -> tuple[int, int, int]:
    if not x.is_cuda or x.dtype not in _DTYPES or x.dim() not in (2, 3) or not x.is_contiguous():
        raise ValueError(f"{name}: needs a contiguous float32, bfloat16 or float16 CUDA matrix or stack of matrices "
                         f"(got {x.dtype} {tuple(x.shape)}, strides {tuple(x.stride())}, on {x.device})")
    stack = x.shape[0] if x.dim() == 3 else 1
    rows, cols = x.shape[-2:]
    return (0 if rows == 0 or cols == 0 else stack), max(rows, 1), max(cols, 1)


def _same(x: torch.Tensor, like: torch.Tensor, name: str, dtype=None) -> None:
    if x.shape != like.shape or x.device != like.device or not x.is_contiguous() or x.dtype != (dtype or like.dtype):
        raise ValueError(f"{name}: needs a contiguous {dtype or like.dtype} tensor {tuple(like.shape)} on {like.device} "
                         f"(got {x.dtype} {tuple(x.shape)}, strides {tuple(x.stride())}, on {x.device})")


@functools.lru_cache(maxsize=256)
def _workspace_bytes(code, stack, rows, cols) -> int:
    size = L.load().engram_orthogonalize_workspace_bytes(code, stack, rows, cols)
    L.check(min(size, 0), "engram_orthogonalize_workspace_bytes")
    return max(size, 1)


def orthogonalize(update: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Each matrix of update [rows, cols] or [stack, rows, cols], divided by its
    Frobenius norm (at least eps) and taken through `steps` steps
    X <- c0 X + (c1 G + c2 G G) X, G = X X^T over the shorter side.
    coefficients: (c0, c1, c2), or one such triple a step.  A zero matrix stays
    zero.  out (update itself, or no part of it): where to write.  Not differentiable."""
    stack, rows, cols = _stack(update, "update")
    table = _coefficients(coefficients, steps)
    if out is None:
        out = torch.empty_like(update)
    else:
        _same(out, update, "out")
    code = _DTYPES[update.dtype]
    size = _workspace_bytes(code, stack, rows, cols)
    ws = torch.empty(size, dtype=torch.uint8, device=update.device)
    st = L.on_device(update.device, lambda stream: L.load().engram_orthogonalize(
        code, update.data_ptr(), stack, rows, cols, steps, table, eps, out.data_ptr(), ws.data_ptr(), size, stream))
    L.check(st, "engram_orthogonalize")
    torch.autograd.graph.increment_version(out)
    return out


def muon_step(param: torch.Tensor, grad: torch.Tensor, momentum: torch.Tensor, lr: float, beta: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5, coefficients=COEFFICIENTS,
              eps: float = 1e-7, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """One step of a matrix or a stack of matrices, each by itself:
        momentum <- momentum + (1 - beta) (grad - momentum)
        u = grad + beta (momentum - grad) if nesterov else momentum
        param <- (1 - lr weight_decay) param - lr sqrt(max(1, rows / cols)) orthogonalize(u)
    param and momentum: float32, updated in place, or written to out = (param,
    momentum); grad: float32, bfloat16 or float16.  param, grad and momentum must
    not overlap one another (an output and its own input may be one).  Returns (param, momentum)."""
    stack, rows, cols = _stack(grad, "grad")
    _same(param, grad, "param", torch.float32)
    _same(momentum, grad, "momentum", torch.float32)
    table = _coefficients(coefficients, steps)
    p_out, m_out = (param, momentum) if out is None else out
    if out is not None:
        _same(p_out, grad, "out[0]", torch.float32)
        _same(m_out, grad, "out[1]", torch.float32)
    size = _workspace_bytes(L.DTYPE_F32, stack, rows, cols)
    ws = torch.empty(size, dtype=torch.uint8, device=grad.device)
    st = L.on_device(grad.device, lambda stream: L.load().engram_muon_step(
        _DTYPES[grad.dtype], param.data_ptr(), grad.data_ptr(), momentum.data_ptr(), p_out.data_ptr(), m_out.data_ptr(),
        stack, rows, cols, lr, beta, int(nesterov), weight_decay, steps, table, eps, ws.data_ptr(), size, stream))
    L.check(st, "engram_muon_step")
    torch.autograd.graph.increment_version((p_out, m_out))
    return p_out, m_out


class Muon(torch.optim.Optimizer):
    """muon_step over parameters that are matrices or stacks of matrices
    (contiguous float32 CUDA tensors); state: the momentum."""

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95,
                 nesterov: bool = True, ns_coefficients=COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5):
        if lr < 0 or weight_decay < 0 or not 0 <= momentum < 1 or eps <= 0:
            raise ValueError(f"invalid Muon hyper-parameters lr={lr} weight_decay={weight_decay} momentum={momentum} "
                             f"eps={eps}")
        _coefficients(ns_coefficients, ns_steps)
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() not in (2, 3):
                    raise ValueError(f"Muon steps matrices and stacks of them, not {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = self.state[p]
                if not st:
                    st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                muon_step(p, p.grad.contiguous(), st["momentum_buffer"], float(group["lr"]), float(group["momentum"]),
                          bool(group["nesterov"]), float(group["weight_decay"]), int(group["ns_steps"]),
                          group["ns_coefficients"], float(group["eps"]))
        return loss
