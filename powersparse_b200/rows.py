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
stride of at least the width); indices are int32 or int64, and they, weights and plans are
contiguous.  ``stream`` is a torch
stream or a raw handle; without it a call runs on PyTorch's current stream of the
tensors' device, which need not be the current device.  With it, outputs and scratch
that the call allocates belong to that stream, and ordering the inputs before it and
other uses of the outputs after it is the caller's part, as with SpMM.  An ``out`` must
not overlap the inputs but where its function says so.  Nothing here waits for the
device, and every call can be captured into a CUDA graph.  These functions take no part
in autograd, but a tensor given as ``out`` counts as changed in place there.

The C entry points and their exact contracts are in ``include/powersparse_b200.h``.
``powersparse_b200.torch_ops`` registers the same operators, with autograd, as
``torch.ops.powersparse.*``.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import sysconfig
from typing import NamedTuple, Optional

import torch

from . import PKG, load_library

__all__ = ["embedding", "embedding_grad", "route", "route_grad", "DispatchPlan", "dispatch_rows", "dispatch", "dispatch_grad",
           "combine", "combine_grad"]

_MODULE_PATH = os.path.join(PKG, "lib", "_rows.so")
# Beside the module: what it was built for, since its layout of torch's and Python's objects is theirs.
_BUILT_FOR_PATH = _MODULE_PATH + ".built_for"
_THIS_TORCH = f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}"
# The entry points that the native module calls, in the order in which its bind() takes them.
_ENTRY_POINTS = ("ps_last_error", "ps_embedding", "ps_embedding_grad_workspace", "ps_embedding_grad", "ps_route", "ps_route_grad",
                 "ps_dispatch_rows", "ps_dispatch", "ps_combine", "ps_combine_grad")
_DTYPES = {None: -1, torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _load_native():
    """The native module (csrc/python/rows_module.cpp), bound to the library that the package has loaded."""
    if not os.path.exists(_MODULE_PATH):
        raise RuntimeError(f"{_MODULE_PATH} is missing: build it with `python -m powersparse_b200.build`")
    if os.path.exists(_BUILT_FOR_PATH):
        with open(_BUILT_FOR_PATH) as f:
            built_for = f.read()
        if built_for != _THIS_TORCH:
            raise RuntimeError(f"{_MODULE_PATH} was built for {built_for}, this is {_THIS_TORCH}: "
                               "build it again with `python -m powersparse_b200.build`")
    name = "powersparse_b200._rows"
    loader = importlib.machinery.ExtensionFileLoader(name, _MODULE_PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_file_location(name, _MODULE_PATH, loader=loader))
    loader.exec_module(module)
    lib = load_library()
    module.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ENTRY_POINTS))
    return module


class _Unloaded:
    """Stands for the native module until its first use."""

    def __getattr__(self, name):
        global _native
        _native = _load_native()
        return getattr(_native, name)


_native = _Unloaded()


def _handle(stream, tensor):
    """The stream's handle; a torch stream must be one of the tensor's device."""
    if stream is None or isinstance(stream, int):
        return stream
    if isinstance(tensor, torch.Tensor) and stream.device != tensor.device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {tensor.device}")
    return stream.cuda_stream


def embedding(table, tokens, scale: float = 1.0, out=None, stream=None):
    """``out[i] = scale * table[tokens[i]]`` (ps_embedding): a tensor of ``tokens``' shape and the table's width.

    A token outside ``[0, len(table))`` gives a row of zeros.  ``out``: a matrix of ``tokens.numel()`` rows.
    """
    return _native.embedding(table, tokens, scale, out, _handle(stream, table))


def embedding_grad(grad, tokens, rows: int, scale: float = 1.0, padding: Optional[int] = None, dtype=None, out=None,
                   accumulate: bool = False, stream=None):
    """Gradient of ``embedding`` for a table of ``rows`` rows (ps_embedding_grad).

    ``grad``: ``[tokens.numel(), width]`` (or ``tokens``' shape and the width).  ``padding``: a token that takes no
    part, besides those outside the table.  ``dtype``: ``grad``'s (default) or float32.  ``out``: a matrix
    ``[rows, width]``, overwritten, or with ``accumulate`` added to.
    """
    if dtype not in _DTYPES:
        raise ValueError(f"the gradient of the table has the type of grad or torch.float32, not {dtype}")
    return _native.embedding_grad(grad, tokens, rows, scale, padding, _DTYPES[dtype], out, accumulate, _handle(stream, grad))


def route(logits, top_k: int, normalize: bool = True, stream=None):
    """``(weights, chosen)`` of a router's scores ``[tokens, experts]`` (ps_route).

    float32 weights and int32 experts, ``[tokens, top_k]``, in descending order of score, of equal scores the lower
    index first.  The weights are softmax shares of the chosen experts, or with ``normalize=False`` of all.  A score
    of -inf switches an expert off; choices that are left over are -1 with weight 0.  A NaN is never chosen and makes
    all weights of its row NaN, as +inf does.
    """
    return _native.route(logits, top_k, normalize, _handle(stream, logits))


def route_grad(grad, logits, weights, chosen, normalize: bool = True, out=None, stream=None):
    """Gradient of ``route`` for the logits, from the gradient of its weights and its outputs (ps_route_grad)."""
    return _native.route_grad(grad, logits, weights, chosen, normalize, out, _handle(stream, logits))


class DispatchPlan(NamedTuple):
    """Where ``dispatch`` put the tokens: what ``combine`` and the experts' products need.

    ``position`` int32 [tokens, top_k]: row of each choice (-1: dropped); ``offsets`` int32 [experts + 1]: first row
    of each expert, and the end; ``counts`` int32 [experts]: tokens of each expert.
    """

    position: torch.Tensor
    offsets: torch.Tensor
    counts: torch.Tensor


def dispatch_rows(slots: int, num_experts: int, align: int = 1) -> int:
    """Rows that ``slots`` = tokens * top_k choices can fill at the most (ps_dispatch_rows)."""
    return _native.dispatch_rows(slots, num_experts, align)


def dispatch(x, chosen, num_experts: int, align: int = 1, out=None, stream=None):
    """``(rows, plan)``: the tokens ``x`` copied into the order of their experts ``chosen`` [tokens, top_k] (ps_dispatch).

    Each expert's rows begin at a multiple of ``align``; the rows between its tokens and the next expert are zeros.
    A choice outside ``[0, num_experts)`` is dropped.  ``out``: at least ``dispatch_rows(...)`` rows, of which those
    from ``plan.offsets[-1]`` on stay as they were; in a tensor that the call allocates they are zeros.
    """
    rows, *plan = _native.dispatch(x, chosen, num_experts, align, out, _handle(stream, x))
    return rows, DispatchPlan(*plan)


def combine(y, plan, weights=None, add=None, out=None, stream=None):
    """``out[t] = add[t] + sum_j weights[t, j] * y[plan.position[t, j]]`` (ps_combine); dropped choices are skipped.

    ``weights``: float32 [tokens, top_k], default ones; ``add``: a matrix [tokens, width], default zeros; it may be
    ``out`` itself.
    """
    return _native.combine(y, *plan, weights, add, out, _handle(stream, y))


def dispatch_grad(grad_rows, plan, out=None, stream=None):
    """Gradient of ``dispatch`` for the tokens: each token's rows summed (``combine`` without weights)."""
    return combine(grad_rows, plan, out=out, stream=stream)


def combine_grad(grad, y, plan, weights, out=None, stream=None):
    """``(grad_y, grad_weights)`` of ``combine`` (ps_combine_grad).

    Rows of ``grad_y`` that no token has are zeros.  ``out``: the tensor for ``grad_y``, [len(y), width], of which
    the rows from ``plan.offsets[-1]`` on stay as they were; it may be ``y`` itself.
    """
    return _native.combine_grad(grad, y, *plan, weights, out, _handle(stream, y))
