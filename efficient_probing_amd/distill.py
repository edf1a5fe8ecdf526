"""Distillation from a teacher's stored top logits: the loss beside ``functional.cross_entropy`` for a probe that learns from a
fine-tuned or larger model's K best logits per image instead of (or beside) the labels.

    loss_rows, dlogits = topk_distillation(logits, teacher_values, teacher_index, targets, temperature=2.0, alpha=0.5)
    loss = distillation_loss(logits, teacher_values, teacher_index, ...)          # mean over rows, differentiable in logits
    values, index, tail = teacher_topk(teacher_logits, k, temperature)            # what a dump keeps of the teacher
    criterion = TopKDistillation.from_store(store, temperature=2.0, alpha=0.5)    # for engine_finetune.train_one_epoch

Per row, with y = logits / T and p = softmax of the teacher's listed logits / T (and, with ``teacher_tail``, of the mass of all
classes it does not list, as one more outcome on both sides):

    loss = alpha T^2 sum_k p_k (log p_k - log softmax(y)_k)  +  (1 - alpha) cross_entropy(logits, target)

The reference trains on labels alone (main_linprobe.py:589); there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from . import functional as F_

MAX_K = 1024
MAX_CLASSES = 1 << 20
_DT = {torch.float32: N.EP_DTYPE_F32, torch.bfloat16: N.EP_DTYPE_BF16, torch.float16: N.EP_DTYPE_F16}


def _check_temperature(T: float) -> None:
    if not 1e-15 <= T <= 1e15:                                  # (its square and its inverse times a logit stay within fp32)
        raise ValueError(f"temperature must lie within [1e-15, 1e15], got {T}")


def _check_alpha(alpha: float) -> None:
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"alpha must lie within [0, 1], got {alpha}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows with contiguous elements that do not overlap, as the kernels read them."""
    return t if t.stride(1) == 1 and (t.shape[0] == 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _int32(t: torch.Tensor, most: int) -> torch.Tensor:
    """Indices as the kernels read them: a 64-bit one beyond int32 stays out of range instead of wrapping into it."""
    return t if t.dtype == torch.int32 else t.to(torch.int64).clamp(-1, most).to(torch.int32)


def _call(lg, val, idx, tail, rows, tgt, temperature, alpha, grad_scale, grad_scale_dev, grad) -> torch.Tensor:
    B, C_ = lg.shape
    R, K = val.shape
    loss = val.new_empty((B,))
    lib = N.load()
    nbytes = lib.ep_distill_workspace_bytes(B, C_, K)
    ws = torch.empty(nbytes, device=lg.device, dtype=torch.uint8) if nbytes else None
    args = N.EPDistillArgs(lg.data_ptr(), _DT[lg.dtype], lg.stride(0), B, C_, K, R, val.data_ptr(), val.stride(0), idx.data_ptr(), idx.stride(0),
                           F_._ptr(tail), F_._ptr(rows), F_._ptr(tgt), temperature, alpha, grad_scale, F_._ptr(grad_scale_dev), loss.data_ptr(),
                           F_._ptr(grad), C_)
    with N.device_guard(lg.device):
        N.check(lib.ep_distill_topk(C.byref(args), F_._ptr(ws), nbytes, N.current_stream_ptr(lg.device)), "ep_distill_topk")
    return loss


def _checked(logits, teacher_values, teacher_index, targets, teacher_tail, teacher_rows, temperature, alpha):
    """The call's arguments as the kernels read them; raises on what they do not take."""
    N.require_gpu_tensor(logits, "logits")
    if logits.dim() != 2 or min(logits.shape) < 1:
        raise ValueError(f"logits must be (B, C), got {tuple(logits.shape)}")
    if logits.dtype not in _DT:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    B, C_ = logits.shape
    if teacher_values.dim() != 2 or teacher_values.shape != teacher_index.shape or min(teacher_values.shape) < 1:
        raise ValueError(f"teacher_values and teacher_index must be (rows, K), got {tuple(teacher_values.shape)} and {tuple(teacher_index.shape)}")
    R, K = teacher_values.shape
    if K > MAX_K or C_ > MAX_CLASSES:
        raise ValueError(f"at most {MAX_K} teacher entries and {MAX_CLASSES} classes, got {K} and {C_}")
    if teacher_index.dtype.is_floating_point or teacher_index.dtype == torch.bool:
        raise ValueError(f"teacher_index must hold integers, got {teacher_index.dtype}")
    _check_temperature(temperature)
    _check_alpha(alpha)
    if alpha < 1.0 and targets is None:
        raise ValueError("alpha < 1 needs targets")
    if targets is not None and tuple(targets.shape) != (B,):
        raise ValueError(f"targets must be ({B},), got {tuple(targets.shape)}")
    if targets is not None and (targets.dtype.is_floating_point or targets.dtype == torch.bool):
        raise ValueError(f"targets must hold integers, got {targets.dtype}")
    if teacher_tail is not None and tuple(teacher_tail.shape) != (R,):
        raise ValueError(f"teacher_tail must be ({R},), got {tuple(teacher_tail.shape)}")
    if teacher_rows is None:
        if R != B:
            raise ValueError(f"{R} teacher rows for {B} logit rows: give teacher_rows")
    elif teacher_rows.dtype != torch.int32 or tuple(teacher_rows.shape) != (B,) or not teacher_rows.is_contiguous():
        raise ValueError(f"teacher_rows must be a contiguous int32 vector of {B}")
    dev = logits.device
    for name, t in (("teacher_values", teacher_values), ("teacher_index", teacher_index), ("teacher_tail", teacher_tail), ("teacher_rows", teacher_rows),
                    ("targets", targets)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the logits on {dev}")
    lg = _rows(logits)
    val = _rows(teacher_values if teacher_values.dtype == torch.float32 else teacher_values.float())
    idx = _rows(_int32(teacher_index, MAX_CLASSES))
    tail = None if teacher_tail is None else teacher_tail.float().contiguous()
    tgt = None if targets is None else targets.to(torch.int64).contiguous()
    return lg, val, idx, tail, teacher_rows, tgt, float(temperature), float(alpha)


def topk_distillation(logits: torch.Tensor, teacher_values: torch.Tensor, teacher_index: torch.Tensor, targets: Optional[torch.Tensor] = None, *,
                      teacher_tail: Optional[torch.Tensor] = None, teacher_rows: Optional[torch.Tensor] = None, temperature: float = 1.0,
                      alpha: float = 1.0, grad_scale: float = 1.0, need_grad: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(loss of every row (B,) fp32, d(mean loss)/dlogits * grad_scale in the logits' type, or None without ``need_grad``).

    ``logits`` (B, C) fp32 / bf16 / fp16, any row stride.  ``teacher_values`` / ``teacher_index`` (R, K): the teacher's logits and their
    classes, in any order; entries with a negative class are skipped, a class listed twice counts as two entries (the loss sums
    p (log p - log q) of each, the gradient takes the sum of their p).  ``teacher_tail``
    (R,): log of the sum of exp(logit / temperature) over the classes not listed (-inf: none); without it the listed classes are
    the teacher's whole distribution.  ``teacher_rows`` (B,) int32: batch row b reads row ``teacher_rows[b]`` of the tables in place
    (a store's table and the batch's image_index); without it row b.  ``targets`` (B,) class indices for ``alpha`` < 1; a negative
    one takes no label term.  A row whose teacher lists nothing, and any row with ``alpha`` 0, has no distillation term.  A class, target or row out of range
    makes that row's loss and gradient NaN."""
    args = _checked(logits, teacher_values, teacher_index, targets, teacher_tail, teacher_rows, temperature, alpha)
    grad = torch.empty_like(logits, memory_format=torch.contiguous_format) if need_grad else None
    return _call(*args, float(grad_scale), None, grad), grad


def mean_rows(rows: torch.Tensor) -> torch.Tensor:
    """Mean of row losses, by sums of at most 65536 at a time: a library reduction over several workgroups clears its counters by a memset,
    which a captured graph does not repeat, and gives the first replay's mean ever after."""
    n = rows.shape[0]
    while rows.shape[0] > 65536:
        whole = rows.shape[0] // 1024 * 1024
        rows = torch.cat((rows[:whole].view(-1, 1024).sum(1), rows[whole:]))
    return rows.sum() / n


class _Distillation(torch.autograd.Function):
    """The backward pass runs the rows again with the incoming gradient as its scale: no second buffer of the logits' size is kept or
    rescaled, and a loss scale acts before the gradient is rounded to a 16-bit type."""

    @staticmethod
    def forward(ctx, logits, values, index, targets, tail, rows, temperature, alpha):
        args = _checked(logits, values, index, targets, tail, rows, temperature, alpha)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(*args[:6])
            ctx.t, ctx.alpha = args[6:]
        return mean_rows(_call(*args, 1.0, None, None))

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        lg = ctx.saved_tensors[0]
        grad = torch.empty(lg.shape, device=lg.device, dtype=lg.dtype)
        _call(*ctx.saved_tensors, ctx.t, ctx.alpha, 1.0, g.float().contiguous(), grad)
        return (grad,) + (None,) * 7


def distillation_loss(logits: torch.Tensor, teacher_values: torch.Tensor, teacher_index: torch.Tensor, targets: Optional[torch.Tensor] = None, *,
                      teacher_tail: Optional[torch.Tensor] = None, teacher_rows: Optional[torch.Tensor] = None, temperature: float = 1.0,
                      alpha: float = 1.0) -> torch.Tensor:
    """Mean of ``topk_distillation``'s row losses, differentiable in ``logits`` (the teacher takes no gradient)."""
    tail = None if teacher_tail is None else teacher_tail.detach()
    return _Distillation.apply(logits, teacher_values.detach(), teacher_index, targets, tail, teacher_rows, temperature, alpha)


@torch.no_grad()
def teacher_topk(logits: torch.Tensor, k: int, temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(values (R, k) fp32, index (R, k) int32, tail (R,) fp32) of a teacher's full logits (R, C): its k largest, and the log of the
    sum of exp(logit / temperature) over the others (-inf where k = C)."""
    if logits.dim() != 2 or not 1 <= k <= min(logits.shape[1], MAX_K):
        raise ValueError(f"logits must be (R, C) and k within [1, min(C, {MAX_K})], got {tuple(logits.shape)} and {k}")
    _check_temperature(temperature)
    lg = logits.float()
    values, index = lg.topk(k, dim=1)
    tail = (lg / temperature).scatter(1, index, float("-inf")).logsumexp(1)
    return values, index.to(torch.int32), tail


class TopKDistillation(torch.nn.Module):
    """``distillation_loss`` against a table of teacher rows, as a criterion: ``criterion(logits, targets, image_index)`` with batch row
    b's teacher in table row ``image_index[b]`` (without it: row b).  ``engine_finetune.train_one_epoch`` hands it the image_index of a
    resident store's batches.  The table is not part of ``state_dict()``; ``.to(device)`` moves it."""

    def __init__(self, teacher_values: torch.Tensor, teacher_index: torch.Tensor, teacher_tail: Optional[torch.Tensor] = None,
                 temperature: float = 1.0, alpha: float = 1.0):
        super().__init__()
        self.temperature, self.alpha = float(temperature), float(alpha)
        _check_temperature(self.temperature)
        _check_alpha(self.alpha)
        if teacher_values.dim() != 2 or teacher_values.shape != teacher_index.shape or min(teacher_values.shape) < 1:
            raise ValueError(f"teacher_values and teacher_index must be (rows, K), got {tuple(teacher_values.shape)} and {tuple(teacher_index.shape)}")
        if teacher_tail is not None and tuple(teacher_tail.shape) != (teacher_values.shape[0],):
            raise ValueError(f"teacher_tail must be ({teacher_values.shape[0]},), got {tuple(teacher_tail.shape)}")
        self.register_buffer("teacher_values", teacher_values.float(), persistent=False)
        if teacher_index.dtype.is_floating_point or teacher_index.dtype == torch.bool:
            raise ValueError(f"teacher_index must hold integers, got {teacher_index.dtype}")
        self.register_buffer("teacher_index", _int32(teacher_index, MAX_CLASSES), persistent=False)
        self.register_buffer("teacher_tail", None if teacher_tail is None else teacher_tail.float(), persistent=False)

    @classmethod
    def from_store(cls, store, temperature: Optional[float] = None, alpha: float = 1.0) -> "TopKDistillation":
        """The teacher that a store carries (``token_store``); the tail belongs to the temperature it was written for."""
        t = store.teacher
        if t is None:
            raise ValueError("this store carries no teacher logits")
        if temperature is None:
            temperature = t.temperature
        if t.tail is not None and temperature != t.temperature:
            raise ValueError(f"the store's tail was written for temperature {t.temperature}, not {temperature}")
        return cls(t.values, t.index, t.tail, temperature, alpha)

    def _rows(self, batch: int, image_index: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        if image_index is None and batch != self.teacher_values.shape[0]:
            raise ValueError(f"a batch of {batch} against a table of {self.teacher_values.shape[0]} teacher rows needs image_index "
                             "(batches of a token_store.ResidentTokenStore carry it)")
        return None if image_index is None else _int32(image_index, 2 ** 31 - 1).contiguous()

    def forward(self, logits: torch.Tensor, targets: Optional[torch.Tensor] = None, image_index: Optional[torch.Tensor] = None) -> torch.Tensor:
        return distillation_loss(logits, self.teacher_values, self.teacher_index, targets if self.alpha < 1.0 else None, teacher_tail=self.teacher_tail,
                                 teacher_rows=self._rows(logits.shape[0], image_index), temperature=self.temperature, alpha=self.alpha)

    def rows_and_gradient(self, logits: torch.Tensor, targets: Optional[torch.Tensor], image_index: Optional[torch.Tensor], grad_scale: float):
        """``topk_distillation`` of the batch: (row losses, gradient), no autograd graph."""
        return topk_distillation(logits, self.teacher_values, self.teacher_index, targets if self.alpha < 1.0 else None, teacher_tail=self.teacher_tail,
                                 teacher_rows=self._rows(logits.shape[0], image_index), temperature=self.temperature, alpha=self.alpha, grad_scale=grad_scale)
