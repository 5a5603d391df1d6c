"""PowerSparse operators registered with PyTorch: ``torch.ops.powersparse.*``.

For GNN code that calls operators through the dispatcher.  The ops take the integer
handle of a ``PowerSparseMatrixGPU`` (``matrix.handle``) and CUDA tensors, run on
PyTorch's current stream and copy nothing (the C ABI reads the tensors in place):

    spmm(handle, B) -> C                     C = A·B, fresh [rows, N] tensor
    spmm_(handle, B, C) -> ()                C (+)= A·B in place (the reference's contract)
    sddmm_csr(handle, lhs, rhs) -> out       out[p] = A_p·<lhs[row(p)], rhs[col(p)]>, CSR order
    sddmm_(handle, lhs, rhs, outs) -> ()     per-workset outputs in workset order, in place

and the operators on rows chosen by an index (``powersparse_b200.rows``), differentiable:

    embedding(table, tokens, scale, padding) -> rows           padding: a token without a gradient
    route(logits, top_k, normalize) -> (weights, chosen)
    dispatch(x, chosen, num_experts, align) -> (rows, position, offsets, counts)
    combine(y, position, offsets, counts, weights, add) -> out

with their gradients as ops of their own (embedding_grad, route_grad, combine_grad).
An op costs its caller about 10 us more than the function of ``rows`` behind it, and 24
more where a gradient is wanted; outputs are always new tensors, zeros behind the last
expert's rows included.  A gradient has the type of its input.

Fake (meta) implementations give shapes for tracing; they read the matrix's
dimensions through the C ABI.  Importing this module registers the ops once.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import SDDMM, SDDMM_csr, SpMM, load_library, rows

__all__ = ["spmm", "spmm_", "sddmm_csr", "sddmm_", "embedding", "embedding_grad", "route", "route_grad", "dispatch", "combine",
           "combine_grad"]


def _dims(handle: int):
    lib = load_library()
    return lib.ps_matrix_row(handle), lib.ps_matrix_col(handle), lib.ps_matrix_nnz(handle)


class _Handle:
    """Minimal stand-in for a matrix object: the module-level functions want ``.handle``."""

    def __init__(self, handle: int):
        self.handle = handle

    def GroupTypeNum(self) -> int:
        return load_library().ps_matrix_group_type_num(self.handle)


def _require(t: torch.Tensor, name: str):
    if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 CUDA tensor")


@torch.library.custom_op("powersparse::spmm_", mutates_args=("C",))
def spmm_(handle: int, B: torch.Tensor, C: torch.Tensor) -> None:
    _require(B, "B")
    _require(C, "C")
    SpMM(_Handle(handle), B.shape[1], B, C, torch.cuda.current_stream(B.device))


@torch.library.custom_op("powersparse::spmm", mutates_args=())
def spmm(handle: int, B: torch.Tensor) -> torch.Tensor:
    _require(B, "B")
    rows, _, _ = _dims(handle)
    C = torch.zeros((rows, B.shape[1]), dtype=torch.float32, device=B.device)
    SpMM(_Handle(handle), B.shape[1], B, C, torch.cuda.current_stream(B.device))
    return C


@spmm.register_fake
def _(handle: int, B: torch.Tensor) -> torch.Tensor:
    rows, _, _ = _dims(handle)
    return B.new_empty((rows, B.shape[1]))


@torch.library.custom_op("powersparse::sddmm_csr", mutates_args=())
def sddmm_csr(handle: int, lhs: torch.Tensor, rhs: torch.Tensor) -> torch.Tensor:
    _require(lhs, "lhs")
    _require(rhs, "rhs")
    _, _, nnz = _dims(handle)
    out = torch.empty(nnz, dtype=torch.float32, device=lhs.device)
    SDDMM_csr(_Handle(handle), lhs.shape[1], lhs, rhs, out, torch.cuda.current_stream(lhs.device))
    return out


@sddmm_csr.register_fake
def _(handle: int, lhs: torch.Tensor, rhs: torch.Tensor) -> torch.Tensor:
    _, _, nnz = _dims(handle)
    return lhs.new_empty((nnz,))


@torch.library.custom_op("powersparse::sddmm_", mutates_args=("outs",))
def sddmm_(handle: int, lhs: torch.Tensor, rhs: torch.Tensor, outs: List[torch.Tensor]) -> None:
    _require(lhs, "lhs")
    _require(rhs, "rhs")
    SDDMM(_Handle(handle), lhs.shape[1], lhs, rhs, list(outs), torch.cuda.current_stream(lhs.device))


# -- rows chosen by an index: the operators of powersparse_b200.rows with autograd.  A
# gradient that autograd hands over may be an expanded or strided view, so it is made
# contiguous first (free where it is already).


def _require_padding(table_rows: int, padding: Optional[int]) -> None:
    """Only the gradient looks at the padding; a bad one is refused before the forward pass."""
    if padding is not None and not 0 <= padding < table_rows:
        raise ValueError(f"padding must be a row of the table, in [0, {table_rows})")


@torch.library.custom_op("powersparse::embedding", mutates_args=())
def embedding(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0, padding: Optional[int] = None) -> torch.Tensor:
    _require_padding(table.shape[0], padding)
    return rows.embedding(table, tokens, scale)


@embedding.register_fake
def _(table, tokens, scale=1.0, padding=None):
    _require_padding(table.shape[0], padding)
    return table.new_empty((*tokens.shape, table.shape[1]))


@torch.library.custom_op("powersparse::embedding_grad", mutates_args=())
def embedding_grad(grad: torch.Tensor, tokens: torch.Tensor, table_rows: int, scale: float = 1.0,
                   padding: Optional[int] = None) -> torch.Tensor:
    return rows.embedding_grad(grad, tokens, table_rows, scale, padding)


@embedding_grad.register_fake
def _(grad, tokens, table_rows, scale=1.0, padding=None):
    return grad.new_empty((table_rows, grad.shape[-1]))


def _embedding_context(ctx, inputs, output):
    table, tokens, ctx.scale, ctx.padding = inputs
    ctx.table_rows = table.shape[0]
    ctx.save_for_backward(tokens)


def _embedding_backward(ctx, grad):
    (tokens,) = ctx.saved_tensors
    return embedding_grad(grad.contiguous(), tokens, ctx.table_rows, ctx.scale, ctx.padding), None, None, None


embedding.register_autograd(_embedding_backward, setup_context=_embedding_context)


@torch.library.custom_op("powersparse::route", mutates_args=())
def route(logits: torch.Tensor, top_k: int, normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    return rows.route(logits, top_k, normalize)


@route.register_fake
def _(logits, top_k, normalize=True):
    shape = (logits.shape[0], top_k)
    return logits.new_empty(shape, dtype=torch.float32), logits.new_empty(shape, dtype=torch.int32)


@torch.library.custom_op("powersparse::route_grad", mutates_args=())
def route_grad(grad: torch.Tensor, logits: torch.Tensor, weights: torch.Tensor, chosen: torch.Tensor,
               normalize: bool = True) -> torch.Tensor:
    return rows.route_grad(grad, logits, weights, chosen, normalize)


@route_grad.register_fake
def _(grad, logits, weights, chosen, normalize=True):
    return logits.new_empty(logits.shape)


def _route_context(ctx, inputs, output):
    logits, _, ctx.normalize = inputs
    ctx.save_for_backward(logits, *output)


def _route_backward(ctx, grad, _):
    logits, weights, chosen = ctx.saved_tensors
    return route_grad(grad.contiguous(), logits, weights, chosen, ctx.normalize), None, None


route.register_autograd(_route_backward, setup_context=_route_context)


@torch.library.custom_op("powersparse::dispatch", mutates_args=())
def dispatch(x: torch.Tensor, chosen: torch.Tensor, num_experts: int,
             align: int = 1) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    out, plan = rows.dispatch(x, chosen, num_experts, align)
    return (out, *plan)


@dispatch.register_fake
def _(x, chosen, num_experts, align=1):
    slots = chosen.shape[0] * chosen.shape[1]
    filled = (slots + min(num_experts, slots) * (align - 1)) // align * align
    return (x.new_empty((filled, x.shape[1])), x.new_empty(chosen.shape, dtype=torch.int32),
            x.new_empty(num_experts + 1, dtype=torch.int32), x.new_empty(num_experts, dtype=torch.int32))


def _dispatch_context(ctx, inputs, output):
    ctx.save_for_backward(*output[1:])


def _dispatch_backward(ctx, grad, *_):
    return combine(grad.contiguous(), *ctx.saved_tensors), None, None, None


dispatch.register_autograd(_dispatch_backward, setup_context=_dispatch_context)


@torch.library.custom_op("powersparse::combine", mutates_args=())
def combine(y: torch.Tensor, position: torch.Tensor, offsets: torch.Tensor, counts: torch.Tensor,
            weights: Optional[torch.Tensor] = None, add: Optional[torch.Tensor] = None) -> torch.Tensor:
    return rows.combine(y, rows.DispatchPlan(position, offsets, counts), weights, add)


@combine.register_fake
def _(y, position, offsets, counts, weights=None, add=None):
    return y.new_empty((position.shape[0], y.shape[1]))


@torch.library.custom_op("powersparse::combine_grad", mutates_args=())
def combine_grad(grad: torch.Tensor, y: torch.Tensor, position: torch.Tensor, offsets: torch.Tensor, counts: torch.Tensor,
                 weights: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return rows.combine_grad(grad, y, rows.DispatchPlan(position, offsets, counts), weights)


@combine_grad.register_fake
def _(grad, y, position, offsets, counts, weights):
    return y.new_empty(y.shape), weights.new_empty(weights.shape)


def _combine_context(ctx, inputs, output):
    y, position, offsets, counts, weights, add = inputs
    ctx.has_add = add is not None
    ctx.save_for_backward(y, position, offsets, counts, weights)


def _combine_backward(ctx, grad):
    y, position, offsets, counts, weights = ctx.saved_tensors
    grad = grad.contiguous()
    ones = weights if weights is not None else torch.ones(position.shape, dtype=torch.float32, device=y.device)
    grad_y, grad_weights = combine_grad(grad, y, position, offsets, counts, ones)
    return grad_y, None, None, None, None if weights is None else grad_weights, grad if ctx.has_add else None


combine.register_autograd(_combine_backward, setup_context=_combine_context)
