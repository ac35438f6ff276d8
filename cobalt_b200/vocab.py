"""The two dense ends of a compressed model: embedding lookup and softmax cross entropy against the head, with their gradients.

The recipe compresses the projections and leaves the embedding table and the head alone (the reference's sinq/patch_model.py:49), the largest
tensors of a model with a large vocabulary.  ``embed`` is what a decoder begins with; ``head_loss`` scores its last hidden states without
ever holding the logits.  Both are differentiable, so a head can be tuned after compression.  A table's gradient, and that of the hidden states, is the whole
one only where everything in between has a backward pass: compressed linears have none and end a graph without a word, so that of a model with compressed
blocks an embedding table (and a tied table's share from that end) would see what comes by the residual stream alone.
The kernels' contract is in ``include/cobalt_b200.h``.  There is no torch fallback: on a non-CUDA tensor every function raises.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable

from . import _lib
from .linear import _raw_stream

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_REDUCTIONS = ("none", "sum", "mean")
_WIDEST = 1 << 28                                            # columns of a table; larger sizes would not pass the C ABI's 32 bits


def _call(index: int, name: str, *args):
    """A library call on device ``index`` and its current stream (the last argument)."""
    fn = getattr(_lib.load(), name)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(name, rc)


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(index: int, name: str, *sizes: int) -> int:
    with torch.cuda.device(index):
        return getattr(_lib.load(), name)(*sizes)


def _gpu(name: str, t: torch.Tensor) -> int:
    index = t.get_device()
    if index < 0 or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor; there is no CPU path")
    return index


def _no_tangent(*tensors: torch.Tensor):
    for t in tensors:
        if fwAD.unpack_dual(t).tangent is not None:
            raise RuntimeError("there are no forward-mode derivatives: a tensor that carries a tangent is not taken")


def _check_status(status: Optional[torch.Tensor], t: torch.Tensor):
    if status is not None and (status.dtype is not torch.int32 or status.shape != (1,) or status.device != t.device):
        raise ValueError(f"status must be int32 [1] on {t.device}, got {status.dtype} {list(status.shape)} on {status.device}")


def _tokens(name: str, t: torch.Tensor, index: int) -> torch.Tensor:
    if t.dtype is not torch.int64:
        raise TypeError(f"{name} must be int64, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")
    return t if t.is_contiguous() else t.contiguous()


def _matrix(name: str, t: torch.Tensor, width: int, unit: int = 1):
    """``(rows, their distance)``: ``t [..., width]`` as rows that the kernels read where they lie, or a copy: neighbouring values, rows apart by
    a multiple of ``unit`` values that do not overlap (``unit`` > 1: on 16-byte boundaries)."""
    shape = t.shape
    if not shape or shape[-1] != width:
        raise ValueError(f"{name} must be [..., {width}], got {list(shape)}")
    if t.is_contiguous() and (unit == 1 or t.data_ptr() % 16 == 0):
        return t, width
    rows = t if len(shape) == 2 else t.reshape(-1, width)
    n, apart = rows.shape[0], rows.stride(0)
    if (rows.stride(1) != 1 and width > 1) or (n > 1 and (apart < width or apart % unit)) or (unit > 1 and rows.data_ptr() % 16):
        rows = rows.clone(memory_format=torch.contiguous_format)
        apart = width
    return rows, apart if n > 1 else width


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the bytes from the first value of ``a`` to its last meet those of ``b``."""
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in (a, b))
    return a0 < b1 and b0 < a1


# ----------------------------------------------------------------------------- embedding
def embed(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, out: Optional[torch.Tensor] = None,
          status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``table[ids] * scale``: rows of ``table [n_rows, width]`` (bf16, fp16 or fp32) for int64 ``ids`` of any shape, ``[*ids.shape, width]``.  The
    product is formed in fp32 and rounded once.  An id outside the table (-1: padding) reads zeros.  ``out`` (contiguous, apart from ``ids`` and
    ``table``) receives the result.  ``status`` (int32 ``[1]``, zero) becomes 8 if an id is beyond the table's end, which no padding is.  Differentiable in
    ``table`` (``embed_grad``)."""
    index = _gpu("table", table)
    shape, kind = table.shape, _TYPES.get(table.dtype)
    if kind is None:
        raise TypeError(f"table must be bfloat16, float16 or float32, got {table.dtype}")
    if len(shape) != 2 or 0 in shape or shape[1] > _WIDEST:
        raise ValueError(f"table must be [n_rows, width] with width at most {_WIDEST}, got {list(shape)}")
    ids = _tokens("ids", ids, index)
    _no_tangent(table)
    _check_status(status, table)
    grad = torch.is_grad_enabled() and table.requires_grad
    if out is not None:
        _no_tangent(out)
        if out.shape != (*ids.shape, shape[1]) or out.dtype is not table.dtype or out.get_device() != index or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {table.dtype} {[*ids.shape, shape[1]]} on {table.device}")
        if grad or (out.requires_grad and torch.is_grad_enabled()):
            raise RuntimeError("out cannot take a result that requires a gradient")
        if _overlap(out, table) or _overlap(out, ids):
            raise ValueError("out must not overlap table or ids")
    if grad:
        return _seen(_Embed.apply(ids, table, float(scale), status))
    return _embed(ids, table, float(scale), status, out)


def _embed(ids, table, scale, status, out=None):
    n_rows, width = table.shape
    rows, apart = _matrix("table", table, width)
    n, given = ids.numel(), out is not None
    if not given:
        out = table.new_empty((*ids.shape, width))
    if n:
        if given:
            torch.autograd.graph.increment_version(out)      # who saved what it held is told, as by an operation of torch
        _call(table.get_device(), "cobalt_embed_watched", ids.data_ptr(), n, rows.data_ptr(), apart, _TYPES[table.dtype], n_rows, width, scale, out.data_ptr(), width,
              None if status is None else status.data_ptr())
    return out


_STREAM = "cobalt_b200.stream"                               # in the metadata of a leaf's node: the stream that it was first seen on


def _leaf_nodes(fn):
    """The nodes of the leaves that ``fn`` takes, directly or behind casts and views (nodes with one input)."""
    for node, _ in fn.next_functions:
        while node is not None and type(node).__name__ != "AccumulateGrad":
            nexts = node.next_functions
            node = nexts[0][0] if len(nexts) == 1 else None
        if node is not None:
            yield node


def _seen(result: torch.Tensor) -> torch.Tensor:
    """``result`` of an operator's forward pass.  A leaf's node lives as long as any graph holds it, and what is written into it as long as itself."""
    stream = _raw_stream(result.get_device())
    for node in _leaf_nodes(result.grad_fn):
        node.metadata.setdefault(_STREAM, stream)
    return result


def _refuse_captured(name: str, fn, index: int):
    """A captured backward pass must not reach a leaf through a node that was made on another stream: torch would wait for that stream, which
    invalidates the capture (or ends the process, where nothing catches it).  Said before, as far as these functions saw the graph that holds the node."""
    if torch.cuda.is_current_stream_capturing():
        stream = _raw_stream(index)
        if any(node.metadata.get(_STREAM, stream) != stream for node in _leaf_nodes(fn)):
            raise RuntimeError(f"{name}: a graph of this leaf that was made on another stream is still alive; drop it before the capture, or capture "
                               "embed_grad / head_loss_and_grad, which need none")


def embed_grad(grad: torch.Tensor, ids: torch.Tensor, n_rows: int, scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``embed`` with respect to its table, dense ``[n_rows, width]`` of ``grad``'s type: ``scale`` times the sum of the rows of
    ``grad [*ids.shape, width]`` by token, in fp32 and in an order that ``ids`` alone decide (partial sums over up to 16 tokens each).  Tokens outside the table are left out.  No second
    derivatives: a ``grad`` that requires one is refused."""
    index, kind = _gpu("grad", grad), _TYPES.get(grad.dtype)
    if kind is None:
        raise TypeError(f"grad must be bfloat16, float16 or float32, got {grad.dtype}")
    ids = _tokens("ids", ids, index)
    shape = grad.shape
    if not shape or shape[:-1] != ids.shape or not 1 <= shape[-1] <= _WIDEST or n_rows < 1:
        raise ValueError(f"grad must be [*ids.shape, width] = {[*ids.shape, 'width']}, width at most {_WIDEST}, and n_rows at least 1, got {list(shape)} "
                         f"and {n_rows}")
    _no_tangent(grad)
    if grad.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("there are no second derivatives: grad must not require a gradient")
    width, n = shape[-1], ids.numel()
    if n == 0:
        return grad.new_zeros((n_rows, width))
    rows, apart = _matrix("grad", grad, width)
    out = grad.new_empty((n_rows, width))
    need = _scratch_bytes(index, "cobalt_embed_grad_scratch_bytes", n, width)
    scratch = out.new_empty(need, dtype=torch.uint8)         # per call, from the stream's own pool: overlapping calls never share one
    _call(index, "cobalt_embed_grad", ids.data_ptr(), n, rows.data_ptr(), apart, kind, n_rows, width, float(scale), out.data_ptr(), scratch.data_ptr(), need)
    return out


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, status):
        ctx.save_for_backward(ids)
        ctx.n_rows, ctx.scale = table.shape[0], scale
        return _embed(ids, table, scale, status)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_captured("embed", ctx, grad.get_device())
        return None, embed_grad(grad, ctx.saved_tensors[0], ctx.n_rows, ctx.scale), None, None


# ----------------------------------------------------------------------------- head loss
def head_loss(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, reduction: str = "mean", status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax cross entropy of the logits ``x @ weight.T``, which are never held: ``x [..., hidden]`` and ``weight [vocab, hidden]`` bf16 (hidden a
    multiple of 8), int64 ``targets`` of ``x``'s leading shape.  fp32 result: of every token (``"none"``), their ``"sum"``, or their ``"mean"`` over the
    tokens that count.  A target outside the vocabulary (-1, -100: padding, a prompt) does not count: loss and gradient zero, whatever
    its row holds.  If none counts, the mean is 0.  Differentiable in ``x`` and ``weight``; the backward pass forms the logits once more.
    ``status`` (int32 ``[1]``, zero) takes the code of a bounded wait that gave up, as ``head_loss_status`` tells it without one."""
    targets = _check_loss(x, weight, targets, reduction, status)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _seen(_HeadLoss.apply(x, weight, targets, reduction, status))
    return _head_loss(x, weight, targets, reduction, status, False)[0]


def head_loss_and_grad(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, reduction: str = "mean", grad: Optional[torch.Tensor] = None,
                       need_x: bool = True, need_weight: bool = True, status: Optional[torch.Tensor] = None):
    """``(loss, dx, dw)`` of ``head_loss`` without autograd, for captured steps and loops of one's own.  ``grad``: fp32 gradient of the result (of
    its shape; ones by default).  ``need_x`` and ``need_weight``: which gradients are formed (``None`` else)."""
    targets = _check_loss(x, weight, targets, reduction, status)
    shape = targets.shape if reduction == "none" else ()
    if grad is None:
        grad = x.new_ones((), dtype=torch.float32).expand(shape)
    elif grad.dtype is not torch.float32 or grad.shape != shape or grad.device != x.device:
        raise ValueError(f"grad must be float32 {list(shape)} on {x.device}, got {grad.dtype} {list(grad.shape)} on {grad.device}")
    _no_tangent(grad)
    with torch.no_grad():
        loss, stats = _head_loss(x, weight, targets, reduction, status, True)
        dx, dw = _head_loss_grad(x, weight, targets, stats, grad, reduction, status, need_x, need_weight) if need_x or need_weight else (None, None)
    return loss, dx, dw


def _check_loss(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, reduction: str, status: Optional[torch.Tensor]) -> torch.Tensor:
    """``targets`` as the kernels read them, if the arguments are in order."""
    index = _gpu("x", x)
    shape, head = x.shape, weight.shape
    if x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16:
        raise TypeError(f"x and weight must be bfloat16, got {x.dtype} and {weight.dtype}")
    if _gpu("weight", weight) != index:
        raise ValueError(f"weight is on {weight.device}, x on {x.device}")
    if len(head) != 2 or 0 in head or head[1] % 8:
        raise ValueError(f"weight must be [vocab, hidden] with hidden a multiple of 8, got {list(head)}")
    if not shape or shape[-1] != head[1]:
        raise ValueError(f"x must be [..., {head[1]}], got {list(shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    if targets.numel() >= 1 << 31:
        raise ValueError(f"{targets.numel()} tokens in one call")
    targets = _tokens("targets", targets, index)
    if targets.shape != shape[:-1]:
        raise ValueError(f"targets must be {list(shape[:-1])}, got {list(targets.shape)}")
    _no_tangent(x, weight)
    _check_status(status, x)
    return targets


def _head_loss(x, weight, targets, reduction, status, keep):
    """(result, what the gradient needs: ``[n, 2]`` if ``keep``)"""
    V, H = weight.shape
    n = targets.numel()
    each = reduction == "none"
    if n == 0:
        return x.new_zeros(targets.shape if each else (), dtype=torch.float32), x.new_empty((0, 2), dtype=torch.float32) if keep else None
    rows, apart = _matrix("x", x, H, 8)
    w, apart_w = _matrix("weight", weight, H, 8)
    index = x.get_device()
    result = x.new_empty(targets.shape if each else (), dtype=torch.float32)
    stats = x.new_empty((n, 2), dtype=torch.float32) if keep else None
    need = _scratch_bytes(index, "cobalt_head_loss_scratch_bytes", n, H, V)
    scratch = x.new_empty(need if each else need + 4 * n, dtype=torch.uint8)       # per call, from the stream's own pool: overlapping calls never share one
    at = scratch.data_ptr()
    # (the tokens' losses, where only their sum is asked for, go behind the scratch)
    _call(index, "cobalt_head_loss", rows.data_ptr(), apart, w.data_ptr(), apart_w, targets.data_ptr(), n, H, V, result.data_ptr() if each else at + need,
          None if stats is None else stats.data_ptr(), None if each else result.data_ptr(), 1 if reduction == "mean" else 0, at, need,
          None if status is None else status.data_ptr())
    return result, stats


def _head_loss_grad(x, weight, targets, stats, grad, reduction, status, want_x, want_w):
    V, H = weight.shape
    n = targets.numel()
    dx = x.new_empty(x.shape) if want_x else None
    dw = weight.new_empty((V, H)) if want_w else None
    if n == 0:
        return dx, None if dw is None else dw.zero_()
    rows, apart = _matrix("x", x, H, 8)
    w, apart_w = _matrix("weight", weight, H, 8)
    each = reduction == "none" and any(step for step, size in zip(grad.stride(), grad.shape) if size > 1)   # (a sum's gradient is one value, expanded)
    if each:
        grad = grad.contiguous()
    index = x.get_device()
    need = _scratch_bytes(index, "cobalt_head_loss_grad_scratch_bytes", n, H, V, 1 if want_x else 0, 1 if want_w else 0)
    scratch = x.new_empty(need, dtype=torch.uint8)
    _call(index, "cobalt_head_loss_grad", rows.data_ptr(), apart, w.data_ptr(), apart_w, targets.data_ptr(), stats.data_ptr(), grad.data_ptr(), 1 if each else 0,
          1 if reduction == "mean" else 0, n, H, V, None if dx is None else dx.data_ptr(), H, None if dw is None else dw.data_ptr(), H, scratch.data_ptr(), need,
          None if status is None else status.data_ptr())
    return dx, dw


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, reduction, status):
        result, stats = _head_loss(x, weight, targets, reduction, status, True)
        ctx.save_for_backward(x, weight, targets, stats)
        ctx.reduction, ctx.status = reduction, status      # (the word is no input of the result)
        return result

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _refuse_captured("head_loss", ctx, grad.get_device())
        want_x, want_w = ctx.needs_input_grad[:2]
        dx, dw = _head_loss_grad(*ctx.saved_tensors, grad, ctx.reduction, ctx.status, want_x, want_w) if want_x or want_w else (None, None)
        return dx, dw, None, None, None


def head_loss_status(device=None) -> int:
    """0, or the code of the first bounded wait of ``head_loss`` or its gradient on ``device`` that gave up since the last question, of
    those without a status word of their own; what it concerns is NaN.  Waits for the current stream."""
    word = ctypes.c_uint32(0)
    with torch.cuda.device(device):
        rc = _lib.load().cobalt_vocab_status(_raw_stream(torch.cuda.current_device()), ctypes.byref(word))
    if rc not in (0, _lib.ETIMEOUT):
        _lib.check("cobalt_vocab_status", rc)
    return int(word.value)
