"""Losses of the fine-tune loop (row f2 of SURVEY.md 8f) on MI355X, behind the names the reference uses:

    criterion = smp.losses.DiceLoss(smp.losses.MULTICLASS_MODE, classes=cls_idx, from_logits=True)
                                                                                    tools/ssl_finetune.py:287-288
    loss = (1 - lam) * criterion(context_logits_mask, masks[0]) + lam * criterion(target_logits_mask, masks[1])   :444-447

`segmentation_models_pytorch` is a third-party dependency outside the reference tree (absent from this image): its
published algorithm (losses/dice.py + losses/_functional.soft_dice_score) is restated -- parity unpinned.  The reduction,
the loss value and d loss / d logits are computed by the HIP kernels of csrc/unet.hip; there is no CPU path."""
from __future__ import annotations

from typing import List, NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import kernels as kn

BINARY_MODE, MULTICLASS_MODE, MULTILABEL_MODE = "binary", "multiclass", "multilabel"


class _DiceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, classes, eps, smooth):
        N, C1, H, W = logits.shape
        CP = (C1 + 7) // 8 * 8
        nhwc = torch.empty(N, H, W, CP, dtype=torch.float32, device=logits.device)
        kn.nchw_to_nhwc(logits.detach().float().contiguous(), nhwc, CP)
        loss = torch.zeros(1, dtype=torch.float64, device=logits.device)
        kn.dice_loss(nhwc, target, C1, classes, 1.0, loss, eps=eps, smooth=smooth)
        ctx.save_for_backward(nhwc, target)
        ctx.meta = (C1, classes, eps, smooth, logits.dtype)
        return loss[0].float()

    @staticmethod
    def backward(ctx, g):
        nhwc, target = ctx.saved_tensors
        C1, classes, eps, smooth, dt = ctx.meta
        dl = torch.empty_like(nhwc)
        scratch = torch.zeros(1, dtype=torch.float64, device=nhwc.device)
        kn.dice_loss(nhwc, target, C1, classes, 1.0, scratch, dlogits=dl, grad_scale=g.detach().float().reshape(1).contiguous(),
                     eps=eps, smooth=smooth)
        return kn.nhwc_to_nchw(dl, C1).to(dt), None, None, None, None


class DiceLoss(torch.nn.Module):
    """smp.losses.DiceLoss for mode="multiclass", from_logits=True (the reference's only use)"""

    def __init__(self, mode: str, classes: Optional[List[int]] = None, log_loss: bool = False, from_logits: bool = True,
                 smooth: float = 0.0, ignore_index: Optional[int] = None, eps: float = 1e-7):
        super().__init__()
        if mode != MULTICLASS_MODE or log_loss or not from_logits or ignore_index is not None:
            raise NotImplementedError("only DiceLoss(MULTICLASS_MODE, classes=..., from_logits=True) is used by MSF-WSI")
        self.mode, self.classes, self.smooth, self.eps = mode, classes, float(smooth), float(eps)

    def forward(self, y_pred: torch.Tensor, y_true: torch.Tensor) -> torch.Tensor:
        if not y_pred.is_cuda:
            raise _lib.MsfwsiHipError("DiceLoss runs only on a HIP device (no CPU path)")
        if y_true.size(0) != y_pred.size(0):
            raise AssertionError("y_true.size(0) == y_pred.size(0)")
        C1 = y_pred.shape[1]
        classes = list(range(C1)) if self.classes is None else list(self.classes)
        return _DiceFn.apply(y_pred, y_true.long().contiguous(), classes, self.eps, self.smooth)


class TopLogits(NamedTuple):
    """What a teacher's row of logits is kept as: its k largest logits (float32, descending), their class indices (int32; a
    negative one marks padding) and rest = log sum over all other classes of exp(logit / T) (None: the list is taken as the
    teacher's whole distribution).  The class dimension of values and indices lies where the logits had it."""

    values: torch.Tensor
    indices: torch.Tensor
    rest: Optional[torch.Tensor] = None


def _class_dim(logits: torch.Tensor, dim: int, what: str) -> int:
    """dim >= 0 of the classes: the last dimension, or 1"""
    kn._gpu(logits, what)
    kn._float(logits, what)
    nd = logits.dim()
    if nd == 0 or not -nd <= dim < nd:
        raise ValueError(f"{what}: no dimension {dim} in {tuple(logits.shape)}")
    dim = dim % nd
    if dim != nd - 1 and dim != 1:
        raise ValueError(f"{what}: the class dimension must be the last one or dimension 1")
    if logits.shape[dim] == 0:
        raise ValueError(f"{what}: no classes in {tuple(logits.shape)}")
    if logits.shape[dim] > kn.LOGITS_MAX_CLASSES:
        raise ValueError(f"{what}: {logits.shape[dim]} classes; at most {kn.LOGITS_MAX_CLASSES} are supported")
    return dim


def _logit_view(logits: torch.Tensor, dim: int) -> torch.Tensor:
    """[rows, C] where the classes are adjacent in memory (also a channels-last map), else [N, C, positions]"""
    nd = logits.dim()
    if dim == nd - 1:
        rows = logits if nd == 2 else logits.reshape(-1, logits.shape[-1])
    else:
        last = logits.movedim(dim, -1)
        if not last.is_contiguous():
            return logits.contiguous().flatten(2)
        rows = last.reshape(-1, last.shape[-1])
    if not rows.is_contiguous() and ((rows.shape[1] > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and rows.stride(0) < rows.shape[1])):
        rows = rows.contiguous()
    return rows


def _temperature(t: float) -> float:
    t = float(t)
    if not 1e-6 <= t <= 1e6:  # so that 1 / T and T^2 stay far inside float32
        raise ValueError(f"temperature must lie within 1e-6 ... 1e6, got {t}")
    return t


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0, dim: int = -1) -> TopLogits:
    """The k largest logits along `dim` (the last dimension, or 1 as in segmentation maps [N, C, H, W]) of a frozen teacher:
    descending, equal ones by ascending class index, NaN above every number.  k <= 64; not differentiable.  `rest` is taken
    at `temperature`, the one the loss will run at."""
    dim = _class_dim(logits, dim, "top_logits")
    view = _logit_view(logits.detach(), dim)
    t, k = _temperature(temperature), int(k)
    if not 1 <= k <= min(kn.TOP_LOGITS_MAX_K, view.shape[1]):
        raise ValueError(f"top_logits: k = {k} outside 1 ... {min(kn.TOP_LOGITS_MAX_K, view.shape[1])}")
    outer, inner = view.shape[0], view.shape[2:]
    values = torch.empty(outer, k, *inner, dtype=torch.float32, device=view.device)
    indices = torch.empty(outer, k, *inner, dtype=torch.int32, device=view.device)
    others = [n for i, n in enumerate(logits.shape) if i != dim]
    rest = torch.empty(others, dtype=torch.float32, device=view.device)
    kn.top_logits(view, k, t, values, indices, rest)
    if view.dim() == 3:
        shape = (outer, k) + tuple(logits.shape[2:])
        return TopLogits(values.view(shape), indices.view(shape), rest)
    if dim == logits.dim() - 1:
        return TopLogits(values.view(*others, k), indices.view(*others, k), rest)
    return TopLogits(values.view(*others, k).movedim(-1, dim), indices.view(*others, k).movedim(-1, dim), rest)


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, indices, rest, mask, dim, temperature, reduction):
        dim = _class_dim(logits, dim, "TopLogitDistillLoss")
        shape = logits.shape
        others = shape[:dim] + shape[dim + 1:]
        k = values.shape[dim] if values.dim() == len(shape) else 0
        if values.shape != indices.shape or values.shape != shape[:dim] + (k,) + shape[dim + 1:]:
            raise ValueError(f"teacher of shapes {tuple(values.shape)}, {tuple(indices.shape)} for logits {tuple(shape)}")
        if not 1 <= k <= kn.TOP_LOGITS_MAX_K:
            raise ValueError(f"the teacher lists {k} classes; 1 ... {kn.TOP_LOGITS_MAX_K} are supported")
        for name, t, dt in (("rest", rest, torch.float32), ("mask", mask, torch.bool)):
            if t is not None and (t.shape != others or t.dtype is not dt):
                raise ValueError(f"{name} must be {dt} of shape {tuple(others)}, got {t.dtype} {tuple(t.shape)}")
        view = _logit_view(logits, dim)
        if view.dim() == 2 and dim != len(shape) - 1:
            values, indices = values.movedim(dim, -1), indices.movedim(dim, -1)
        values, indices, rest, mask = (None if t is None else t.contiguous() for t in (values, indices, rest, mask))
        mean = reduction == "mean"
        row_loss, loss, saved = kn.distill_fwd(view, values, indices, rest, mask, k, temperature, mean, reduction == "none")
        ctx.save_for_backward(view, values, indices, rest, saved)
        ctx.meta = (shape, dim, k, temperature, mean)
        return loss if row_loss is None else row_loss.view(others)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        view, values, indices, rest, saved = ctx.saved_tensors
        shape, dim, k, temperature, mean = ctx.meta
        dz = torch.empty(view.shape, dtype=view.dtype, device=view.device)
        kn.distill_bwd(view, values, indices, rest, k, temperature, saved, mean, g.float().contiguous(), dz)
        if view.dim() == 2 and dim != len(shape) - 1:
            dz = dz.view(shape[:dim] + shape[dim + 1:] + (shape[dim],)).movedim(-1, dim)
        elif dz.shape != shape:
            dz = dz.view(shape)
        return dz, None, None, None, None, None, None, None


class TopLogitDistillLoss(torch.nn.Module):
    """Distillation of a student from the top logits of a frozen teacher: T^2 times the Kullback-Leibler divergence between
    the two softened distributions, with the classes outside the teacher's list taken as one.

        teacher = top_logits(teacher_logits, k, temperature=T)
        loss = TopLogitDistillLoss(temperature=T)(student_logits, teacher)

    Without `teacher.rest` the teacher's distribution is its list alone, renormalised.  reduction: "mean" over the rows that
    count, "sum", or "none" (one value per row).  A row does not count -- no loss, a zero gradient -- where `mask` (bool, the
    logits' shape without the class dimension) is False or the teacher's list and rest are empty (all indices negative or all
    values -inf); a mean over no rows is 0.  An index listed twice adds its shares; an index past the classes makes its row's
    loss and gradient NaN.  dim: the class dimension, the last or 1."""

    def __init__(self, temperature: float = 1.0, reduction: str = "mean", dim: int = -1):
        super().__init__()
        if reduction not in ("mean", "sum", "none"):
            raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
        self.temperature, self.reduction, self.dim = _temperature(temperature), reduction, int(dim)

    def forward(self, logits: torch.Tensor, teacher: TopLogits, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        values, indices, rest = teacher
        if (values.requires_grad or (rest is not None and rest.requires_grad)) and torch.is_grad_enabled():
            raise ValueError("the teacher is frozen: detach its values")
        return _DistillFn.apply(logits, values, indices, rest, mask, self.dim, self.temperature, self.reduction)
