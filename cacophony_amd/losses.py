"""Losses of a linear vocabulary head without its logits: cross entropy (caption likelihoods and their gradient) and distillation from
a teacher's top logits.  C ABI: caco_linear_ce / caco_linear_distill (include/caco_hip.h has the formulas).

The reference forms the logits [tokens, vocab] of its caption decoder (`decoder_proj`, src/caco_torch/text_models/roberta.py:371,
src/caco_torch/caco.py:212-240) and leaves what follows to its callers; at 256 captions of 32 tokens that matrix alone is 1.6 GB in fp32.
Here the rows' losses come out of the same pass that forms a tile of logits: losses alone take 16 MB at that size.  The gradients
of hidden states, weight and bias go through the gradient of the logits, in bf16 and for one piece of the vocabulary at a time, and
`piece_bytes` is what it may take: by default 2 GiB, which is the whole vocabulary at that size (1.59 ms, a workspace of 2.0 GB).
Smaller pieces trade time for memory: 1.85 ms in 750 MB (512 MiB of pieces), 3.2 in 450 (128), 8.4 in 346 (32).

Two forms of each loss:

* `linear_cross_entropy` / `linear_topk_distillation` take part in autograd, in reverse mode: tensors with a tangent are refused.
* `..._with_grad` return the loss and the gradients of one call: one preparation for both passes, no autograd state, and they may be
  captured into a graph.  (The autograd forms refuse to be captured with gradients on: a captured backward pass whose leaves still have
  an eager graph alive would wait for that graph's stream inside the capture.)

Tensors: hidden bf16 [..., dim], weight bf16 [vocab, dim], bias fp32 [vocab] or None; labels / teacher entries with hidden's leading
dimensions.  dim is a multiple of 8.  Any strides are taken; rows that do not start at multiples of 16 bytes are copied first.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .model import _ptr, _stream

Tensor = torch.Tensor

FORWARD, BACKWARD, LSE_PAIR = 1, 2, 4
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
# d logits of one piece of the vocabulary, bf16, by rows and by columns: 8192 tokens x 50265 words are one piece, with the rest 0.7 % of a card's memory
PIECE_BYTES = 2 << 30


class LinearLossGrads(NamedTuple):
    """What the `_with_grad` forms return.  `loss` is None for reduction "none", `d_bias` without a bias."""
    loss: Optional[Tensor]
    row_loss: Tensor
    d_hidden: Tensor
    d_weight: Tensor
    d_bias: Optional[Tensor]


class _Head:
    """The checked operands of a call."""

    def __init__(self, what: str, hidden: Tensor, weight: Tensor, bias: Optional[Tensor], reduction: str):
        if reduction not in _REDUCTIONS:
            raise ValueError(f"{what}: reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
        operands = [("hidden", hidden, torch.bfloat16), ("weight", weight, torch.bfloat16)] + ([] if bias is None else [("bias", bias, torch.float32)])
        for name, t, dt in operands:
            if not torch.is_tensor(t) or t.dtype != dt:
                raise ValueError(f"{what}: {name} must be a {dt} tensor, got {t.dtype if torch.is_tensor(t) else type(t)}")
        for name, t, _ in operands:
            if t.device.type != "cuda" or t.device != hidden.device:
                raise RuntimeError(f"{what}: hidden, weight and bias must be on the same GPU, {name} is on {t.device}")
        if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
            raise ValueError(f"{what}: expected hidden [..., dim] and weight [vocab, dim], got {tuple(hidden.shape)} and {tuple(weight.shape)}")
        if bias is not None and tuple(bias.shape) != (weight.shape[0],):
            raise ValueError(f"{what}: bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
        self.what, self.reduction_name, self.reduction = what, reduction, _REDUCTIONS[reduction]
        self.vocab, self.dim = int(weight.shape[0]), int(weight.shape[1])
        self.lead = tuple(hidden.shape[:-1])
        self.hidden, self.ld_h = _rows(hidden.detach().reshape(math.prod(self.lead), self.dim))
        self.weight, self.ld_w = _rows(weight.detach())
        self.bias = None if bias is None else bias.detach().contiguous()
        self.rows = int(self.hidden.shape[0])
        self.device = hidden.device

    def per_row(self, name: str, t: Tensor, tail: Tuple[int, ...] = ()) -> Tensor:
        if not torch.is_tensor(t):
            raise ValueError(f"{self.what}: {name} must be a tensor, got {type(t)}")
        if t.device != self.device:
            raise RuntimeError(f"{self.what}: {name} must be on {self.device}, is on {t.device}")
        if tuple(t.shape) != self.lead + tail:
            raise ValueError(f"{self.what}: {name} must be {list(self.lead + tail)}, got {list(t.shape)}")
        return t.detach().reshape((self.rows,) + tail)


def _rows(x: Tensor) -> Tuple[Tensor, int]:
    """[n, dim] whose rows start at multiples of 16 bytes, and their stride."""
    if x.stride(1) != 1 or x.data_ptr() % 16 or (x.shape[0] > 1 and (x.stride(0) < x.shape[1] or x.stride(0) % 8 or x.stride(0) >= 1 << 22)):
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x, int(x.stride(0)) if x.shape[0] > 1 else int(x.shape[1])


def _labels(head: _Head, labels: Tensor) -> dict:
    labels = head.per_row("labels", labels)
    if labels.dtype.is_floating_point or labels.dtype == torch.bool or labels.dtype.is_complex:
        raise ValueError(f"{head.what}: labels must be integers, got {labels.dtype}")
    return {"labels": labels.to(torch.int64).contiguous()}


def _teacher(head: _Head, logits: Tensor, indices: Tensor, temperature: float) -> dict:
    if not torch.is_tensor(logits) or logits.dim() < 1:
        raise ValueError(f"{head.what}: teacher_logits must be a tensor [..., k]")
    k = int(logits.shape[-1])
    logits, indices = head.per_row("teacher_logits", logits, (k,)), head.per_row("teacher_indices", indices, (k,))
    if not logits.dtype.is_floating_point:
        raise ValueError(f"{head.what}: teacher_logits must be floating point, got {logits.dtype}")
    if indices.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{head.what}: teacher_indices must be int32 or int64, got {indices.dtype}")
    return {"teacher": logits.to(torch.float32).contiguous(), "indices": indices.contiguous(), "temperature": float(temperature)}


def _call(head: _Head, target: dict, what: int, *, ignore_index: int = -100, reduction: Optional[int] = None, row_weight=None, grad_scale=None,
          row_loss=None, lse=None, loss=None, d_hidden=None, d_weight=None, d_bias=None, piece_bytes: int = PIECE_BYTES) -> None:
    lib = _lib.load()
    topk = int(target["teacher"].shape[1]) if "teacher" in target else 0
    if "teacher" in target and not 1 <= topk <= 128:
        raise ValueError(f"{head.what}: 1 to 128 teacher entries per row, got {topk}")
    if int(piece_bytes) <= 0:
        raise ValueError(f"{head.what}: piece_bytes must be positive, got {piece_bytes}")
    reduction = head.reduction if reduction is None else reduction
    with torch.cuda.device(head.device):
        need = int(lib.caco_linear_loss_workspace(head.rows, head.vocab, head.dim, topk, int(piece_bytes), what))
        if need < 0:
            _lib.check(need, head.what)
        ws = torch.empty(need, dtype=torch.uint8, device=head.device)
        first = (what, _ptr(head.hidden), head.ld_h, _ptr(head.weight), head.ld_w, _ptr(head.bias))
        last = (head.rows, head.vocab, head.dim, reduction, _ptr(row_weight), _ptr(grad_scale), _ptr(row_loss), _ptr(lse), _ptr(loss),
                _ptr(d_hidden), head.dim, _ptr(d_weight), head.dim, _ptr(d_bias), _ptr(ws), need, _stream())
        if topk:
            idx = target["indices"]
            _lib.check(lib.caco_linear_distill(*first, _ptr(target["teacher"]), topk, _ptr(idx), topk, idx.element_size(), topk,
                                               target["temperature"], *last), head.what)
        else:
            _lib.check(lib.caco_linear_ce(*first, _ptr(target["labels"]), int(ignore_index), *last), head.what)


def _forward(head: _Head, target: dict, ignore_index: int, keep_lse: bool):
    new = lambda *s: torch.empty(*s, dtype=torch.float32, device=head.device)
    row_loss = new(head.rows)
    lse = new(2, head.rows) if keep_lse else None      # with the rest that its rounding leaves: a confident row's gradient needs it
    loss = new(()) if head.reduction else None
    _call(head, target, FORWARD | LSE_PAIR, ignore_index=ignore_index, row_loss=row_loss, lse=lse, loss=loss)
    return (row_loss.reshape(head.lead) if loss is None else loss), lse


class _LinearLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, head, target, ignore_index, piece_bytes):
        out, lse = _forward(head, target, ignore_index, True)
        # All tensors that the backward pass reads are saved here and nowhere else: a change in place is an error (a detached tensor shares its
        # version), hooks on saved tensors see them, and they are free once the backward pass is over.
        names = tuple(k for k, t in target.items() if torch.is_tensor(t))
        ctx.save_for_backward(hidden, weight, bias, lse, *(target[k] for k in names))
        ctx.names, ctx.rest = names, {k: v for k, v in target.items() if k not in names}
        ctx.what, ctx.reduction, ctx.ignore_index, ctx.piece_bytes = head.what, head.reduction_name, ignore_index, piece_bytes
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        with torch.cuda.device(grad.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{ctx.what}: the autograd form cannot be captured into a graph; capture {ctx.what}_with_grad")
            hidden, weight, bias, lse, *tensors = ctx.saved_tensors
            head = _Head(ctx.what, hidden, weight, bias, ctx.reduction)
            target = {**dict(zip(ctx.names, tensors)), **ctx.rest}
            new = lambda n, t: torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and ctx.needs_input_grad[n] else None
            dh, dw, db = new(0, hidden), new(1, weight), new(2, bias)
            grad = grad.to(torch.float32).contiguous()
            kw = {"grad_scale": grad} if head.reduction else {"row_weight": grad.reshape(-1)}
            _call(head, target, BACKWARD | LSE_PAIR, ignore_index=ctx.ignore_index, lse=lse, d_hidden=dh, d_weight=dw, d_bias=db,
                  piece_bytes=ctx.piece_bytes, **kw)
        return dh, dw, db, None, None, None, None


def _reverse_mode_only(what: str, *tensors) -> None:
    for t in tensors:
        if torch.is_tensor(t) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what}: there is no forward-mode derivative; a tangent would be lost")


def _loss(head: _Head, target: dict, hidden, weight, bias, ignore_index: int, piece_bytes: int) -> Tensor:
    if int(piece_bytes) <= 0:
        raise ValueError(f"{head.what}: piece_bytes must be positive, got {piece_bytes}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (hidden, weight, bias)):
        with torch.cuda.device(head.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{head.what}: the autograd form cannot be captured into a graph; capture {head.what}_with_grad")
        return _LinearLoss.apply(hidden, weight, bias, head, target, ignore_index, piece_bytes)
    return _forward(head, target, ignore_index, False)[0]


def _with_grad(head: _Head, target: dict, ignore_index: int, row_weight: Optional[Tensor], piece_bytes: int) -> LinearLossGrads:
    if row_weight is not None:
        row_weight = head.per_row("row_weight", row_weight)
        if row_weight.dtype != torch.float32:
            raise ValueError(f"{head.what}: row_weight must be fp32, got {row_weight.dtype}")
        row_weight = row_weight.contiguous()
    new = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device=head.device)
    row_loss, loss = new(head.rows), new(()) if head.reduction else None
    dh, dw = new(head.rows, head.dim, dtype=torch.bfloat16), new(head.vocab, head.dim, dtype=torch.bfloat16)
    db = None if head.bias is None else new(head.vocab)
    _call(head, target, FORWARD | BACKWARD, ignore_index=ignore_index, row_weight=row_weight, row_loss=row_loss, loss=loss, d_hidden=dh, d_weight=dw,
          d_bias=db, piece_bytes=piece_bytes)
    return LinearLossGrads(loss, row_loss.reshape(head.lead), dh.reshape(head.lead + (head.dim,)), dw, db)


def linear_cross_entropy(hidden: Tensor, weight: Tensor, labels: Tensor, bias: Optional[Tensor] = None, *, ignore_index: int = -100,
                         reduction: str = "mean", piece_bytes: int = PIECE_BYTES) -> Tensor:
    """logsumexp(z) - z[label] with z = hidden @ weight.T + bias, fp32.  A row whose label is `ignore_index` or outside [0, vocab) has
    loss 0 and does not count for the mean (which is NaN, with zero gradients, when no row does).  reduction "none" gives the rows'
    losses - minus the log-likelihood of each token - in the shape of `labels`."""
    _reverse_mode_only("linear_cross_entropy", hidden, weight, bias)
    head = _Head("linear_cross_entropy", hidden, weight, bias, reduction)
    return _loss(head, _labels(head, labels), hidden, weight, bias, ignore_index, piece_bytes)


def linear_cross_entropy_with_grad(hidden: Tensor, weight: Tensor, labels: Tensor, bias: Optional[Tensor] = None, *, ignore_index: int = -100,
                                   reduction: str = "mean", row_weight: Optional[Tensor] = None, piece_bytes: int = PIECE_BYTES) -> LinearLossGrads:
    """The loss, the rows' losses and the gradients of sum(row_weight * row_loss), for "mean" divided by the number of rows that
    count.  row_weight fp32 in the shape of `labels`, None = 1."""
    head = _Head("linear_cross_entropy", hidden, weight, bias, reduction)
    return _with_grad(head, _labels(head, labels), ignore_index, row_weight, piece_bytes)


def linear_topk_distillation(hidden: Tensor, weight: Tensor, teacher_logits: Tensor, teacher_indices: Tensor, bias: Optional[Tensor] = None, *,
                             temperature: float = 1.0, reduction: str = "mean", piece_bytes: int = PIECE_BYTES) -> Tensor:
    """T^2 KL(q || softmax(z / T)) with z = hidden @ weight.T + bias and q = softmax(teacher_logits / T) over the entries a teacher gives
    per row: teacher_logits [..., k], teacher_indices int32 or int64 [..., k], k <= 128 (`retrieval.topk` or `torch.topk` of the teacher's
    logits).  An index outside [0, vocab) (`retrieval.topk` pads with -1) or a logit of -inf is no entry, entries of one token add up, a
    row without entries has loss 0 and does not count.  No gradient flows to the teacher.  temperature 2^-20 .. 2^20."""
    _reverse_mode_only("linear_topk_distillation", hidden, weight, bias)
    head = _Head("linear_topk_distillation", hidden, weight, bias, reduction)
    return _loss(head, _teacher(head, teacher_logits, teacher_indices, temperature), hidden, weight, bias, -100, piece_bytes)


def linear_topk_distillation_with_grad(hidden: Tensor, weight: Tensor, teacher_logits: Tensor, teacher_indices: Tensor, bias: Optional[Tensor] = None,
                                       *, temperature: float = 1.0, reduction: str = "mean", row_weight: Optional[Tensor] = None,
                                       piece_bytes: int = PIECE_BYTES) -> LinearLossGrads:
    """The distillation loss with its gradients in one call; see `linear_cross_entropy_with_grad`.  No gradient flows to the teacher."""
    head = _Head("linear_topk_distillation", hidden, weight, bias, reduction)
    return _with_grad(head, _teacher(head, teacher_logits, teacher_indices, temperature), -100, row_weight, piece_bytes)
