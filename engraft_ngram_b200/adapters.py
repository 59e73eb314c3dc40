"""Low-rank adapters of many requests at once, beside a shared projection.

A request may carry an adapter of its own: a pair of factors a [rank, K] and
b [N, rank] that changes a projection y = W x into y + scale * b (a x).  The
factors of all loaded adapters stand in two stacks, and index says which one
each position uses (-1: none):

    out[t] = base[t] + scale[i] * b[i] @ (a[i] @ x[t]),   i = index[t]

so positions of any number of requests share one call: one new token of each
of many sequences in slot order, or packed prompts.  `adapter_add` is the
product (differentiable in base, x, a and b), `adapter_gradients` its
gradients as tensors, and `PleAdapters` hands adapters to `ple_forward`, which
applies them to the PLE block's key and value projections.  The reference has
no adapters: its descent trains table rows only.

float32, bfloat16 and float16; sums in fp32, results rounded once and, for the
same inputs, the same bits.  Infinities and NaN stay in the rows and gradients of
the positions' own adapters.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L

_DTYPES = {torch.float32: L.DTYPE_F32, torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_F16}
MAX_RANK, MAX_ADAPTERS = 128, 16384


@dataclass
class PleAdapters:
    """Adapters of the PLE block's projections: a [n, rank, n_embd] and
    b [n, hc*n_embd + n_embd, rank] (key columns, then value columns, as the
    stacked projection [w_key; w_value] has its rows), index int32 [T] of the
    positions' adapters, scale float32 [n] or None (1).  The block computes in
    float32, so a and b are float32; 16-bit adapters are for adapter_add beside
    a caller's own projection."""
    a: torch.Tensor
    b: torch.Tensor
    index: torch.Tensor
    scale: torch.Tensor | None = None


def _rows(x: torch.Tensor, name: str, T: int, width: int, like: torch.Tensor) -> int:
    """The row stride of a [T, width] operand (its elements of a row consecutive)."""
    if x.dtype != like.dtype or x.device != like.device:
        raise ValueError(f"{name}: {x.dtype} on {x.device}, but x is {like.dtype} on {like.device}")
    if x.shape != (T, width):
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {(T, width)}")
    rows, columns = x.stride()
    ld = rows if T > 1 else width
    if (width > 1 and columns != 1) or ld < width:
        raise ValueError(f"{name}: strides {(rows, columns)}: the elements of a row have to be consecutive "
                         "and its rows apart")
    return ld


@functools.lru_cache(maxsize=256)
def _plan(dtype, x_shape, a_shape, b_shape, backward: int):
    """(dtype code, T, K, N, rank, adapters, workspace bytes) of a call's types and shapes."""
    code = _DTYPES.get(dtype)
    if code is None or len(x_shape) != 2:
        raise ValueError(f"x: needs a [T, K] float32, bfloat16 or float16 CUDA tensor (got {dtype} {tuple(x_shape)})")
    if len(a_shape) != 3 or len(b_shape) != 3 or a_shape[0] != b_shape[0] or a_shape[1] != b_shape[2]:
        raise ValueError(f"a {tuple(a_shape)}, b {tuple(b_shape)}: expected [adapters, rank, K] and [adapters, N, rank]")
    T, K = x_shape
    n, rank, N = a_shape[0], a_shape[1], b_shape[1]
    if a_shape[2] != K:
        raise ValueError(f"a {tuple(a_shape)}: its last dimension has to be x's {K}")
    if not 1 <= rank <= MAX_RANK or n > MAX_ADAPTERS or K < 1 or N < 1:
        raise ValueError(f"rank {rank}, {n} adapters, {K} -> {N}: ranks are 1 to {MAX_RANK}, at most {MAX_ADAPTERS} "
                         "adapters, widths at least 1")
    size = L.load().engram_adapter_workspace_bytes(T, n, rank, K, N, backward)
    L.check(min(size, 0), "engram_adapter_workspace_bytes")
    return code, T, K, N, rank, n, max(size, 1)


def _check(x, a, b, index, scale, backward: int):
    if not x.is_cuda:
        raise ValueError(f"x: needs a CUDA tensor (got {x.dtype} on {x.device})")
    plan = _plan(x.dtype, x.shape, a.shape, b.shape, backward)
    dtype, dev = x.dtype, x.device
    if a.dtype != dtype or b.dtype != dtype or a.device != dev or b.device != dev or not a.is_contiguous() \
            or not b.is_contiguous():
        for name, f in (("a", a), ("b", b)):
            if f.dtype != dtype or f.device != dev or not f.is_contiguous():
                raise ValueError(f"{name}: needs a contiguous {dtype} tensor on {dev} (got {f.dtype} on {f.device}, "
                                 f"strides {tuple(f.stride())})")
    if index.dtype != torch.int32 or index.device != dev or index.shape != (plan[1],) or not index.is_contiguous():
        raise ValueError(f"index: needs a contiguous int32 [{plan[1]}] tensor on {dev} (got {index.dtype} "
                         f"{tuple(index.shape)} on {index.device})")
    if scale is not None and (scale.dtype != torch.float32 or scale.device != dev or scale.shape != (plan[5],)
                              or not scale.is_contiguous()):
        raise ValueError(f"scale: needs a contiguous float32 [{plan[5]}] tensor on {dev} (got {scale.dtype} "
                         f"{tuple(scale.shape)} on {scale.device})")
    return plan


def forward_into(out, base, x, a, b, index, scale) -> torch.Tensor:
    """out (None: a new tensor) = base (None: zeros) + the adapters' product; no autograd.  out may be base."""
    code, T, K, N, rank, n, ws_bytes = _check(x, a, b, index, scale, 0)
    dev = x.device
    given = out is not None
    if not given:
        out = x.new_empty((T, N))
    ldx = _rows(x, "x", T, K, x)
    ldout = _rows(out, "out", T, N, x) if given else N
    ldbase = _rows(base, "base", T, N, x) if base is not None else 0
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    st = L.on_device(dev, lambda stream: L.load().engram_adapter_forward(
        code, x.data_ptr(), ldx, a.data_ptr(), b.data_ptr(), index.data_ptr(), None if scale is None else scale.data_ptr(),
        T, n, rank, K, N, None if base is None else base.data_ptr(), ldbase, out.data_ptr(), ldout, ws.data_ptr(),
        ws_bytes, stream))
    L.check(st, "engram_adapter_forward")
    if given:
        torch.autograd.graph.increment_version(out)
    return out


def backward_into(grad, x, a, b, index, scale, dx=None, dx_base=None, da=None, db=None) -> None:
    """The gradients wanted (dx, da, db given) of the adapters' product; dx = dx_base (None: zeros) + its own
    part, and dx_base may be dx.  Otherwise no output may overlap another one or an input."""
    code, T, K, N, rank, n, ws_bytes = _check(x, a, b, index, scale, 1)
    dev = x.device
    ldx, ldg = _rows(x, "x", T, K, x), _rows(grad, "grad", T, N, x)
    lddx = _rows(dx, "dx", T, K, x) if dx is not None else 0
    ldbase = _rows(dx_base, "dx_base", T, K, x) if dx_base is not None else 0
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    st = L.on_device(dev, lambda stream: L.load().engram_adapter_backward(
        code, grad.data_ptr(), ldg, x.data_ptr(), ldx, a.data_ptr(), b.data_ptr(), index.data_ptr(), L.ptr(scale), T, n,
        rank, K, N, L.ptr(dx_base), ldbase, L.ptr(dx), lddx, L.ptr(da), L.ptr(db), ws.data_ptr(), ws_bytes, stream))
    L.check(st, "engram_adapter_backward")


def refuse_scale_gradient(scale) -> None:
    """No gradient of scale is built: an error where one would be lost."""
    if scale is not None and scale.requires_grad and torch.is_grad_enabled():
        raise ValueError("scale requires grad, but adapters have no gradient of it: pass scale.detach(), or train it "
                         "inside b")


def adapter_gradients(grad: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor,
                      scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, da, db): the gradients of x, a and b from grad [T, N], the gradient
    of adapter_add's result (base's own gradient is grad itself).  A position
    without an adapter gets dx = 0, an adapter that no position uses da = db = 0.
    The results carry no graph, whatever the inputs require."""
    grad, x, a, b = grad.detach(), x.detach(), a.detach(), b.detach()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    da = torch.empty_like(a, memory_format=torch.contiguous_format)
    db = torch.empty_like(b, memory_format=torch.contiguous_format)
    backward_into(grad, x, a, b, index, scale, dx, None, da, db)
    return dx, da, db


class _AdapterFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, base, x, a, b, index, scale):
        out = forward_into(None, base, x, a, b, index, scale)
        ctx.save_for_backward(x, a, b, index, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, a, b, index, scale = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want[1] else None
        da = torch.empty_like(a) if want[2] else None
        db = torch.empty_like(b) if want[3] else None
        if want[1] or want[2] or want[3]:
            backward_into(grad.contiguous(), x, a, b, index, scale, dx, None, da, db)
        return grad if want[0] else None, dx, da, db, None, None


def adapter_add(base: torch.Tensor | None, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index: torch.Tensor,
                scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """out [T, N] = base [T, N] (None: zeros) + scale[i] * b[i] @ (a[i] @ x[t]), i = index[t].

    x [T, K] and base: row-strided views are taken as they are; a [n, rank, K]
    and b [n, N, rank]: contiguous, ranks up to 128; index: int32 [T], outside
    [0, n) for a position without an adapter (its row is base's); scale:
    float32 [n], not differentiable (refused where it requires grad), or None
    (1).  out: where to write (base itself adds in place); only for calls that
    need no gradients, and it must not overlap x, a or b, nor base in any other
    way."""
    refuse_scale_gradient(scale)
    if torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad
                                    or (base is not None and base.requires_grad)):
        if out is not None:
            raise ValueError("adapter_add: out= is for calls that need no gradients")
        return _AdapterFn.apply(base, x, a, b, index, scale)
    if out is not None and out.requires_grad and torch.is_grad_enabled():
        raise ValueError("adapter_add: out requires grad")
    return forward_into(out, base, x, a, b, index, scale)
