"""Operators on rows chosen by an index that the model makes, on torch CUDA tensors.

    embedding(table, tokens, scale=1.0)            rows of a table by token, scaled
    embedding_grad(grad, tokens, rows, ...)        the table's gradient, summed by sorted tokens
    route(logits, top_k, normalize=True)           softmax and top-k of a router: (weights, chosen)
    route_grad(grad, logits, weights, chosen)      its gradient for the logits
    dispatch(x, chosen, num_experts, align=1)      tokens in the order of their experts: (rows, plan)
    dispatch_grad(grad_rows, plan)                 its gradient
    combine(y, plan, weights=None, add=None)       the experts' rows back, weighted and summed
    combine_grad(grad, y, plan, weights)           its gradients for the rows and the weights

Matrices are float32, bfloat16 or float16 tensors whose rows are contiguous (any row
stride of at least the width); indices are int32 or int64.  ``stream`` is a torch
stream or a raw handle; without it a call runs on PyTorch's current stream of the
tensors' device, which need not be the current device.  With it, outputs and scratch
that the call allocates belong to that stream, and ordering the inputs before it and
other uses of the outputs after it is the caller's part, as with SpMM.  Nothing here
waits for the device, and every call can be captured into a CUDA graph.

The C entry points and their exact contracts are in ``include/powersparse_b200.h``.
``powersparse_b200.torch_ops`` registers the same operators, with autograd, as
``torch.ops.powersparse.*``.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional

import torch

from . import _check, load_library

__all__ = ["embedding", "embedding_grad", "route", "route_grad", "DispatchPlan", "dispatch_rows", "dispatch", "dispatch_grad",
           "combine", "combine_grad"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INDICES = {torch.int32: 0, torch.int64: 1}
_MAX_WIDTH, _MAX_ROWS = 1 << 24, (1 << 31) - 1  # what the C entry points take (and what fits their int arguments)


def _matrix(t, name: str, device=None, dtype=None, shape=None) -> int:
    """Checks a matrix with contiguous rows; its row stride in elements."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dim() != 2 or t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be a matrix of float32, bfloat16 or float16")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    rows, width = t.shape
    if shape is not None and (rows, width) != tuple(shape):
        raise ValueError(f"{name} must have the shape {tuple(shape)}, not {(rows, width)}")
    if not 1 <= width <= _MAX_WIDTH or rows > _MAX_ROWS:
        raise ValueError(f"{name} must have rows of 1 to 2^24 elements, and below 2^31 of them")
    if width > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have contiguous rows")
    if rows <= 1:
        return width
    stride = t.stride(0)
    if stride < width:
        raise ValueError(f"{name} has rows that overlap")
    return stride


def _packed(t, name: str, dtypes, device, shape=None):
    """Checks a contiguous tensor of one of ``dtypes``."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have the shape {tuple(shape)}, not {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


@contextlib.contextmanager
def _entered(device, stream):
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream(device).cuda_stream
        else:
            s = torch.cuda.ExternalStream(stream, device) if isinstance(stream, int) else stream
            with torch.cuda.stream(s):
                yield s.cuda_stream


class _Here:
    """The common case of ``_entered``: the current device and its current stream."""

    __slots__ = ("handle",)

    def __init__(self, handle):
        self.handle = handle

    def __enter__(self):
        return self.handle

    def __exit__(self, *exc):
        return False


def _on(device, stream):
    """Context in which allocations and the launch belong to ``stream`` on ``device``; gives the stream's handle."""
    if stream is None and torch.cuda.current_device() == device.index:
        return _Here(torch.cuda.current_stream(device).cuda_stream)
    if stream is not None and not isinstance(stream, int) and stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    return _entered(device, stream)


def embedding(table, tokens, scale: float = 1.0, out=None, stream=None):
    """``out[i] = scale * table[tokens[i]]`` (ps_embedding): a tensor of ``tokens``' shape and the table's width.

    A token outside ``[0, len(table))`` gives a row of zeros.  ``out``: a matrix of ``tokens.numel()`` rows.
    """
    stride = _matrix(table, "table")
    device = table.device
    _packed(tokens, "tokens", _INDICES, device)
    n, width = tokens.numel(), table.shape[1]
    if table.shape[0] < 1:
        raise ValueError("the table has no rows")
    if out is not None:
        out_stride = _matrix(out, "out", device, table.dtype, (n, width))
    with _on(device, stream) as s:
        if out is None:
            out = torch.empty((*tokens.shape, width), dtype=table.dtype, device=device)
            out_stride = width
        _check(load_library().ps_embedding(table.data_ptr(), _DTYPES[table.dtype], table.shape[0], width, stride, tokens.data_ptr(),
                                           _INDICES[tokens.dtype], n, scale, out.data_ptr(), out_stride, s))
    return out


def embedding_grad(grad, tokens, rows: int, scale: float = 1.0, padding: Optional[int] = None, dtype=None, out=None,
                   accumulate: bool = False, stream=None):
    """Gradient of ``embedding`` for a table of ``rows`` rows (ps_embedding_grad).

    ``grad``: ``[tokens.numel(), width]`` (or ``tokens``' shape and the width).  ``padding``: a token that takes no
    part, besides those outside the table.  ``dtype``: ``grad``'s (default) or float32.  ``out``: a matrix
    ``[rows, width]``, overwritten, or with ``accumulate`` added to.
    """
    if isinstance(grad, torch.Tensor) and grad.dim() != 2 and isinstance(tokens, torch.Tensor) \
            and grad.shape[:-1] == tokens.shape:
        if not grad.is_contiguous():
            raise ValueError("grad must be a matrix with contiguous rows, or contiguous")
        grad = grad.view(tokens.numel(), grad.shape[-1])
    stride = _matrix(grad, "grad")
    device = grad.device
    _packed(tokens, "tokens", _INDICES, device)
    n, width = tokens.numel(), grad.shape[1]
    if grad.shape[0] != n:
        raise ValueError(f"grad has {grad.shape[0]} rows for {n} tokens")
    if not 1 <= rows < _MAX_ROWS:
        raise ValueError("the table's rows must be in [1, 2^31 - 2]")
    if padding is not None and not 0 <= padding < rows:
        raise ValueError("padding must be a row of the table")
    if accumulate and out is None:
        raise ValueError("accumulate needs the gradient to add to (out)")
    dtype = dtype or (out.dtype if out is not None else grad.dtype)
    if dtype not in (grad.dtype, torch.float32):
        raise ValueError(f"the gradient of the table is {grad.dtype} or torch.float32, not {dtype}")
    if out is not None:
        out_stride = _matrix(out, "out", device, dtype, (rows, width))
    lib = load_library()
    need = lib.ps_embedding_grad_workspace(n, rows, width)
    if need < 0:
        raise ValueError("the number of tokens must be below 2^31")
    with _on(device, stream) as s:
        if out is None:
            out = torch.empty((rows, width), dtype=dtype, device=device)
            out_stride = width
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=device)
        _check(lib.ps_embedding_grad(grad.data_ptr(), _DTYPES[grad.dtype], stride, tokens.data_ptr(), _INDICES[tokens.dtype], n,
                                     scale, -1 if padding is None else padding, int(accumulate), out.data_ptr(), _DTYPES[dtype],
                                     out_stride, rows, width, workspace.data_ptr(), workspace.numel(), s))
    return out


def route(logits, top_k: int, normalize: bool = True, stream=None):
    """``(weights, chosen)`` of a router's scores ``[tokens, experts]`` (ps_route).

    float32 weights and int32 experts, ``[tokens, top_k]``, in descending order of score, of equal scores the lower
    index first.  The weights are softmax shares of the chosen experts, or with ``normalize=False`` of all.  A score
    of -inf switches an expert off; choices that are left over are -1 with weight 0.
    """
    stride = _matrix(logits, "logits")
    device = logits.device
    tokens, experts = logits.shape
    if not 1 <= top_k <= min(experts, 32):
        raise ValueError(f"top_k must be in [1, min({experts}, 32)]")
    with _on(device, stream) as s:
        weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
        chosen = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
        _check(load_library().ps_route(logits.data_ptr(), _DTYPES[logits.dtype], stride, tokens, experts, top_k, int(normalize),
                                       weights.data_ptr(), chosen.data_ptr(), s))
    return weights, chosen


def route_grad(grad, logits, weights, chosen, normalize: bool = True, out=None, stream=None):
    """Gradient of ``route`` for the logits, from the gradient of its weights and its outputs (ps_route_grad)."""
    stride = _matrix(logits, "logits")
    device = logits.device
    tokens, experts = logits.shape
    _packed(chosen, "chosen", (torch.int32,), device)
    if chosen.dim() != 2 or chosen.shape[0] != tokens:
        raise ValueError(f"chosen must be [{tokens}, top_k]")
    _packed(weights, "weights", (torch.float32,), device, chosen.shape)
    _packed(grad, "grad", (torch.float32,), device, chosen.shape)
    if out is not None:
        out_stride = _matrix(out, "out", device, logits.dtype, logits.shape)
    with _on(device, stream) as s:
        if out is None:
            out = torch.empty((tokens, experts), dtype=logits.dtype, device=device)
            out_stride = experts
        _check(load_library().ps_route_grad(grad.data_ptr(), logits.data_ptr(), _DTYPES[logits.dtype], stride, weights.data_ptr(),
                                            chosen.data_ptr(), tokens, experts, chosen.shape[1], int(normalize), out.data_ptr(),
                                            out_stride, s))
    return out


class DispatchPlan(NamedTuple):
    """Where ``dispatch`` put the tokens: what ``combine`` and the experts' products need.

    ``position`` int32 [tokens, top_k]: row of each choice (-1: dropped); ``offsets`` int32 [experts + 1]: first row
    of each expert, and the end; ``counts`` int32 [experts]: tokens of each expert.
    """

    position: torch.Tensor
    offsets: torch.Tensor
    counts: torch.Tensor


def _plan(plan, device):
    position, offsets, counts = plan
    _packed(position, "plan.position", (torch.int32,), device)
    if position.dim() != 2 or not 1 <= position.shape[1] <= 32:
        raise ValueError("plan.position must be [tokens, top_k] with top_k in [1, 32]")
    _packed(counts, "plan.counts", (torch.int32,), device)
    if counts.dim() != 1 or not 1 <= counts.shape[0] <= 1024:
        raise ValueError("plan.counts must be [experts] with 1 to 1024 experts")
    _packed(offsets, "plan.offsets", (torch.int32,), device, (counts.shape[0] + 1,))
    return position, offsets, counts


def dispatch_rows(slots: int, num_experts: int, align: int = 1) -> int:
    """Rows that ``slots`` = tokens * top_k choices can fill at the most (ps_dispatch_rows)."""
    if not (0 <= slots <= _MAX_ROWS and 1 <= num_experts <= 1024 and 1 <= align <= 65536):
        raise ValueError("slots must be in [0, 2^31), the number of experts in [1, 1024] and align in [1, 65536]")
    return load_library().ps_dispatch_rows(slots, num_experts, align)


def dispatch(x, chosen, num_experts: int, align: int = 1, out=None, stream=None):
    """``(rows, plan)``: the tokens ``x`` copied into the order of their experts ``chosen`` [tokens, top_k] (ps_dispatch).

    Each expert's rows begin at a multiple of ``align``; the rows between its tokens and the next expert are zeros.
    A choice outside ``[0, num_experts)`` is dropped.  ``out``: at least ``dispatch_rows(...)`` rows, of which those
    from ``plan.offsets[-1]`` on stay as they were; in a tensor that the call allocates they are zeros.
    """
    stride = _matrix(x, "x")
    device = x.device
    tokens, width = x.shape
    _packed(chosen, "chosen", _INDICES, device)
    if chosen.dim() != 2 or chosen.shape[0] != tokens or not 1 <= chosen.shape[1] <= 32:
        raise ValueError(f"chosen must be [{tokens}, top_k] with top_k in [1, 32]")
    top_k = chosen.shape[1]
    need = dispatch_rows(tokens * top_k, num_experts, align)
    fresh = out is None
    if not fresh:
        out_stride = _matrix(out, "out", device, x.dtype)
        if out.shape[0] < need or out.shape[1] != width:
            raise ValueError(f"out must have at least {need} rows of {width}")
    with _on(device, stream) as s:
        if fresh:
            out = torch.empty((need, width), dtype=x.dtype, device=device)
            out_stride = width
        position = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
        offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
        counts = torch.empty(num_experts, dtype=torch.int32, device=device)
        _check(load_library().ps_dispatch(x.data_ptr(), _DTYPES[x.dtype], stride, chosen.data_ptr(), _INDICES[chosen.dtype], tokens,
                                          top_k, num_experts, align, width, out.data_ptr(), out_stride, out.shape[0],
                                          int(fresh), position.data_ptr(), offsets.data_ptr(), counts.data_ptr(), s))
    return out, DispatchPlan(position, offsets, counts)


def combine(y, plan, weights=None, add=None, out=None, stream=None):
    """``out[t] = add[t] + sum_j weights[t, j] * y[plan.position[t, j]]`` (ps_combine); dropped choices are skipped.

    ``weights``: float32 [tokens, top_k], default ones; ``add``: a matrix [tokens, width], default zeros; it may be
    ``out`` itself.
    """
    stride = _matrix(y, "y")
    device, width = y.device, y.shape[1]
    position, _, _ = _plan(plan, device)
    tokens, top_k = position.shape
    if weights is not None:
        _packed(weights, "weights", (torch.float32,), device, position.shape)
    add_stride = _matrix(add, "add", device, y.dtype, (tokens, width)) if add is not None else width
    if out is not None:
        out_stride = _matrix(out, "out", device, y.dtype, (tokens, width))
    with _on(device, stream) as s:
        if out is None:
            out = torch.empty((tokens, width), dtype=y.dtype, device=device)
            out_stride = width
        _check(load_library().ps_combine(y.data_ptr(), _DTYPES[y.dtype], stride, y.shape[0], position.data_ptr(),
                                         None if weights is None else weights.data_ptr(), None if add is None else add.data_ptr(),
                                         add_stride, tokens, top_k, width, out.data_ptr(), out_stride, s))
    return out


def dispatch_grad(grad_rows, plan, out=None, stream=None):
    """Gradient of ``dispatch`` for the tokens: each token's rows summed (``combine`` without weights)."""
    return combine(grad_rows, plan, out=out, stream=stream)


def combine_grad(grad, y, plan, weights, out=None, stream=None):
    """``(grad_y, grad_weights)`` of ``combine`` (ps_combine_grad).

    Rows of ``grad_y`` that no token has are zeros.  ``out``: the tensor for ``grad_y``, [len(y), width], of which
    the rows from ``plan.offsets[-1]`` on stay as they were.
    """
    stride = _matrix(y, "y")
    device, (rows, width) = y.device, y.shape
    position, offsets, counts = _plan(plan, device)
    tokens, top_k = position.shape
    grad_stride = _matrix(grad, "grad", device, y.dtype, (tokens, width))
    _packed(weights, "weights", (torch.float32,), device, position.shape)
    fresh = out is None
    if not fresh:
        out_stride = _matrix(out, "out", device, y.dtype, (rows, width))
    with _on(device, stream) as s:
        if fresh:
            out = torch.empty((rows, width), dtype=y.dtype, device=device)
            out_stride = width
        grad_weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
        _check(load_library().ps_combine_grad(grad.data_ptr(), _DTYPES[y.dtype], grad_stride, y.data_ptr(), stride, rows,
                                              position.data_ptr(), offsets.data_ptr(), counts.data_ptr(), counts.shape[0],
                                              weights.data_ptr(), tokens, top_k, width, out.data_ptr(), out_stride,
                                              int(fresh), grad_weights.data_ptr(), s))
    return out, grad_weights
