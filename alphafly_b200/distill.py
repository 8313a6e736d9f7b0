"""Distillation: training a network on another one's best moves (the targets' selection, the loss, the step).

The reference trains on the visit distributions of its own search (chessfly/train.py:105-132).  A network can
also learn from a slower one (more steps through the wiring, another checkpoint): ``top_logits`` keeps each
position's k best policy logits of the teacher, some 12 k bytes instead of a dense (4168,) row, and
``distillation_loss`` is the divergence of the student's distribution from the teacher's,

    loss = T^2 sum_c p_c (log p_c - log q_c)

with p = softmax(teacher / T) over the k named moves and, with ``rest``, one more outcome "any other move" of
the mass the teacher leaves to it, and q = softmax(student / T) over all moves or the legal ones.  Both run in
libafb (``afb_top_logits``, ``afb_distill_loss``); the loss and its gradient are one pass over the logits.

    top = teacher_targets(teacher, batch.x, 16, legal=(batch.moves, batch.valid))      # teacher.infer_heads = "int8"
    train_step(student, opt, batch, device, teacher=top)                               # alphafly_b200.train
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .int8 import TYPES


class TopLogits(NamedTuple):
    """A teacher's best moves per position: ``values`` (B, k) float32 logits, largest first, ``moves`` (B, k)
    int64 (-inf and -1 where a position has fewer), ``log_rest`` (B,) float32: log sum exp(logit / temperature)
    of the other moves, and the ``temperature`` it was taken at."""
    values: torch.Tensor
    moves: torch.Tensor
    log_rest: torch.Tensor
    temperature: float = 1.0


def _check_logits(logits: torch.Tensor, temperature: float) -> torch.Tensor:
    if logits.dim() != 2:
        raise ValueError(f"logits must be (B, moves), got {tuple(logits.shape)}")
    if logits.dtype not in TYPES:
        raise TypeError(f"logits must be float32, float16 or bfloat16, not {logits.dtype}")
    if not logits.is_cuda:
        raise RuntimeError("logits must be a CUDA tensor")
    if not temperature > 0:
        raise ValueError("the temperature must be positive")
    return logits if logits.stride(1) == 1 and logits.stride(0) >= logits.shape[1] else logits.contiguous()


def _matrix(t: torch.Tensor, shape: tuple, dtype: torch.dtype, device, name: str) -> torch.Tensor:
    if tuple(t.shape) != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} {shape} on the logits' device, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _legal(legal, logits: torch.Tensor):
    """(moves, valid, length) of the legal-move lists, or Nones."""
    if legal is None:
        return None, None, 0
    moves, valid = legal
    if moves.dim() != 2:
        raise ValueError(f"legal moves must be (B, K), got {tuple(moves.shape)}")
    shape = (logits.shape[0], moves.shape[1])
    moves = _matrix(moves, shape, torch.int64, logits.device, "legal moves")
    valid = _matrix(valid, shape, torch.bool, logits.device, "legal valid")
    if shape[1] == 0:                            # no entries have no address, and no address means all moves
        moves, valid = moves.new_zeros(shape[0], 1), valid.new_zeros(shape[0], 1)
    return moves, valid, moves.shape[1]


def _ptr(t: torch.Tensor | None):
    return t.data_ptr() if t is not None else None


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0, legal=None) -> TopLogits:
    """The k (at most 256) largest of each row of ``logits`` (B, moves), equal ones by the lower move, without gradients;
    -inf and NaN are never taken.  ``legal``: (moves (B, K) int64, valid (B, K) bool), as a ``train.Batch`` holds them, restricts
    a row to its listed moves; a row without any comes back as -inf / -1."""
    logits = _check_logits(logits, temperature)
    if not 1 <= k <= 256:
        raise ValueError("k must be between 1 and 256")
    b, n = logits.shape
    dev = logits.device
    moves, valid, listed = _legal(legal, logits)
    out = TopLogits(torch.empty(b, k, dtype=torch.float32, device=dev), torch.empty(b, k, dtype=torch.int64, device=dev),
                    torch.empty(b, dtype=torch.float32, device=dev), float(temperature))
    ld = logits.stride(0) if b > 1 else n        # a single row's stride says nothing: torch leaves any number there
    with _lib.on_device(dev):
        _lib.call("afb_top_logits", b, n, TYPES[logits.dtype], logits.data_ptr(), ld, k, float(temperature),
                  _ptr(moves), _ptr(valid), listed, out.values.data_ptr(), out.moves.data_ptr(), out.log_rest.data_ptr(),
                  _lib.stream_of(dev))
    return out


@torch.no_grad()
def teacher_targets(teacher, x: torch.Tensor, k: int, temperature: float = 1.0, legal=None) -> TopLogits:
    """``teacher`` (a ``FlyChessNet``) on the positions ``x`` (B, N_FEATURES), in inference: its ``top_logits``.  With
    ``teacher.infer_heads`` "int8" the readout runs in 8-bit integers."""
    modes = [(m, m.training) for m in teacher.modules()]         # a part may be frozen in a mode of its own
    teacher.eval()
    try:
        logits, _ = teacher(x)
    finally:
        for m, training in modes:
            m.training = training
    return top_logits(logits, k, temperature, legal)


class _Loss:
    """The arguments of one ``afb_distill_loss``, all but the student's logits."""

    def __init__(self, values, moves, log_rest, temperature, legal, weight, scale, differentiable):
        self.tensors = [t for t in (values, moves, log_rest, legal[0], legal[1], weight) if t is not None]   # for the backward
        self.versions = self.current_versions() if differentiable else None
        self.front = (values.shape[1], values.data_ptr(), moves.data_ptr(), _ptr(log_rest), temperature, _ptr(legal[0]),
                      _ptr(legal[1]), legal[2], _ptr(weight), scale)

    def current_versions(self) -> list:
        """What tells a change in place; tensors made in inference mode have no version."""
        return [None if t.is_inference() else t._version for t in self.tensors]

    def launch(self, logits, upstream, skip_ones, rows, total, grad) -> None:
        b, n = logits.shape
        dev = logits.device
        ld = logits.stride(0) if b > 1 else n    # as in top_logits
        with _lib.on_device(dev):
            _lib.call("afb_distill_loss", b, n, TYPES[logits.dtype], logits.data_ptr(), ld, *self.front,
                      _ptr(upstream), upstream.stride(0) if upstream is not None and upstream.dim() else 0, skip_ones, _ptr(rows),
                      _ptr(total), _ptr(grad), n, _lib.stream_of(dev))


class _Distillation(torch.autograd.Function):
    """The forward writes the gradient for an upstream gradient of 1 in the same pass over the logits.  The backward
    recomputes the rows whose upstream gradient, read on the device, is anything else (it rounds to the logits' type
    once, after the scaling); a second backward writes a gradient of its own."""

    @staticmethod
    def forward(ctx, logits, loss, reduction, differentiable):
        b = logits.shape[0]
        rows = torch.empty(b, dtype=torch.float32, device=logits.device)
        total = None if reduction == "none" else torch.empty((), dtype=torch.float32, device=logits.device)
        grad = None
        if differentiable:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            ctx.save_for_backward(logits)
            ctx.loss, ctx.grad = loss, grad
        loss.launch(logits, None, 0, rows, total, grad)
        return rows if total is None else total

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():
            raise RuntimeError("distillation_loss has no second derivative (create_graph)")
        logits, = ctx.saved_tensors
        if ctx.loss.current_versions() != ctx.loss.versions:
            raise RuntimeError("distillation_loss: a target or list was modified in place before the backward")
        grad, ctx.grad = ctx.grad, None
        skip = grad is not None
        if not skip:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        ctx.loss.launch(logits, g if g.dtype == torch.float32 else g.float(), int(skip), None, None, grad)
        return grad, None, None, None


def distillation_loss(logits: torch.Tensor, top: TopLogits, legal=None, rest: bool = False, weight: torch.Tensor | None = None,
                      reduction: str = "mean") -> torch.Tensor:
    """The divergence of the student's ``logits`` (B, moves) from the teacher's ``top`` (module docstring), with a
    gradient by ``logits``: float32, the mean over the B positions, their sum, or (B,) with ``reduction`` "none".
    ``legal``: the lists that restrict the student's softmax (as for ``top_logits``); a named move outside them is
    left out.  ``rest``: the moves the teacher does not name count as one outcome.  ``weight`` (B,) float32 scales
    the positions' losses (no gradient goes to it or to ``top``).  A position without a named move contributes zero."""
    logits = _check_logits(logits, top.temperature)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"unknown reduction {reduction!r}")
    b, dev = logits.shape[0], logits.device
    k = top.values.shape[1] if top.values.dim() == 2 else 0
    if not 1 <= k <= 256:
        raise ValueError("top must hold between 1 and 256 moves a position")
    values = _matrix(top.values, (b, k), torch.float32, dev, "top.values")
    moves = _matrix(top.moves, (b, k), torch.int64, dev, "top.moves")
    log_rest = _matrix(top.log_rest, (b,), torch.float32, dev, "top.log_rest") if rest else None
    if weight is not None:
        weight = _matrix(weight.detach(), (b,), torch.float32, dev, "weight")
    differentiable = torch.is_grad_enabled() and logits.requires_grad
    loss = _Loss(values, moves, log_rest, float(top.temperature), _legal(legal, logits), weight,
                 1.0 / b if reduction == "mean" and b else 1.0, differentiable)
    return _Distillation.apply(logits, loss, reduction, differentiable)
