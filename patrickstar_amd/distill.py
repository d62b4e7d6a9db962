"""A teacher's top logits, and the loss of a student against them.

``top_logits`` reduces a row of logits to its ``k`` largest, their places and the row's log-sum-exp: what a teacher has to
leave behind for its student.  ``distill_loss`` is the student's side, a loss whose gradient starts the backward pass that
``FP16Adam.step()`` ends.  The hand-written kernels are behind ``include/ps_ops.h``.

fp16 gradients of a softmax over a vocabulary need the loss scale: most of them are far below fp16's smallest number.  The
scale therefore has to be in the gradient before it is rounded.  ``grad_scale`` tells the forward pass what backward is going
to multiply by (``DynamicLossScaler.scale_tensor``, ``LossScaler.loss_scale``): it then makes the gradient while it has the
logits in registers, and backward hands it out if the factor was that one (decided on the device, without a
synchronisation) and makes it anew if not.
"""
import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .rotary import DTYPES

REDUCTIONS = ("mean", "sum", "none")
_REDUCTION_NUMBER = {name: i for i, name in enumerate(REDUCTIONS)}


class TopLogits(NamedTuple):
    """``values`` (of the logits' type) and ``ids`` (int32), largest first, ``[..., k]``; ``logsumexp`` (fp32), ``[...]``."""

    values: torch.Tensor
    ids: torch.Tensor
    logsumexp: torch.Tensor


def top_logits(logits, k, temperature=1.0):
    """The ``k`` largest of every row of ``logits`` ``[..., vocabulary]`` and ``logsumexp(logits / temperature)``.

    Equal logits are taken by their place, the lowest first; NaN counts as larger than every number.  fp16, bf16 or fp32 on
    the GPU, ``k`` up to 1024 (and the vocabulary).  Not differentiable: a teacher's logits are data.
    """
    ops = _lib.load().ops
    if ops is not None:
        out = ops.ops_top(logits, k, temperature)
        if out is not None:
            return TopLogits(*out)
    rows = _logit_rows("top_logits", logits)
    vocab = logits.shape[-1]
    if isinstance(k, bool) or not isinstance(k, int) or not 1 <= k <= min(vocab, _lib.PS_MAX_TOP):
        raise ValueError(f"top_logits: k must be 1 .. {min(vocab, _lib.PS_MAX_TOP)}, got {k!r}")
    _check_temperature("top_logits", temperature)
    lead, device = logits.shape[:-1], logits.device
    values = torch.empty((*lead, k), dtype=logits.dtype, device=device)
    ids = torch.empty((*lead, k), dtype=torch.int32, device=device)
    lse = torch.empty(lead, dtype=torch.float, device=device)
    c = _lib.ps_top_call()
    c.logits, c.values, c.ids, c.lse = rows.data_ptr(), values.data_ptr(), ids.data_ptr(), lse.data_ptr()
    c.rows, c.vocab, c.row_stride = rows.shape[0], vocab, rows.stride(0)
    c.k, c.dtype, c.temperature = k, DTYPES[logits.dtype], temperature
    with _lib.on_device(device):
        _lib.check(_lib.load().ps_top_logits(_lib.address(c), _lib.raw_stream(device)), "ps_top_logits")
    return TopLogits(values, ids, lse)


def distill_loss(logits, ids, teacher_logits, teacher_lse=None, labels=None, *, label_weight=0.0, temperature=1.0,
                 ignore_index=-100, reduction="mean", grad_scale=None):
    """Loss of ``logits`` ``[..., vocabulary]`` against a teacher's list ``ids``, ``teacher_logits`` ``[..., k]``; fp32.

    Every row's loss is ``(1 - label_weight) * temperature**2 * KL(teacher || student) + label_weight * cross_entropy``, with
    teacher and student at ``temperature`` and the cross entropy of ``labels`` at 1.

    Without ``teacher_lse`` the teacher's probabilities are the softmax of its list.  With it (``top_logits``' third result,
    at the same temperature) they are ``exp(teacher_logits / temperature - teacher_lse)``, and what they leave to 1 is
    compared, as one more outcome, with all that the student gives to tokens off the list.

    A negative id marks an entry that is not there; the other ids of a row must differ.  Rows whose label is
    ``ignore_index`` count for nothing, in the loss, the mean and the gradient; a mean over no rows is 0.  What cannot be
    checked without waiting for the GPU does not go unnoticed: an id that comes twice or lies beyond the vocabulary, or such
    a label, makes its row's loss and gradient NaN, which the scaler's overflow probe finds.

    ``grad_scale``: the factor that backward is going to arrive with (a number, or a tensor with one element on the GPU), if
    the caller knows it; the logits are then read once for loss and gradient, whose memory is taken in the forward pass.  Another factor
    is no error: the gradient is then made in the backward pass.  Not with ``reduction="none"``.
    """
    ops = _lib.load().ops
    if ops is not None:
        loss = ops.ops_distill(logits, ids, teacher_logits, teacher_lse, labels, label_weight, temperature, ignore_index,
                               _REDUCTION_NUMBER.get(reduction), grad_scale)
        if loss is not None:
            return loss
    rows = _logit_rows("distill_loss", logits)
    options = _checked_options(logits, ids, teacher_logits, teacher_lse, labels, label_weight, temperature, ignore_index, reduction,
                               grad_scale)
    k = ids.shape[-1]
    lists = (_rows_of(ids, k), _rows_of(teacher_logits.detach(), k), None if teacher_lse is None else teacher_lse.detach().reshape(-1),
             None if labels is None else labels.reshape(-1))
    if torch.is_grad_enabled() and logits.requires_grad:
        if isinstance(grad_scale, torch.Tensor):
            grad_scale = grad_scale.detach().float()
        loss = _DistillLoss.apply(rows, *lists, options, grad_scale)
    else:
        loss = _forward(rows, *lists, options)[0]
    return loss.view(logits.shape[:-1]) if reduction == "none" else loss


# -------------------------------------------------------------------------------------------------------------- checks


def _logit_rows(what, logits):
    if not logits.is_cuda:
        raise RuntimeError(f"{what}: logits must be a GPU tensor (got {logits.device})")
    if logits.dtype not in DTYPES:
        raise TypeError(f"{what}: logits must be float16, bfloat16 or float32, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be [..., vocabulary], got {tuple(logits.shape)}")
    return _rows_of(logits, logits.shape[-1])


def _rows_of(x, width):
    """[rows, width] with the elements of a row next to one another."""
    x = x.reshape(math.prod(x.shape[:-1]), width)
    return x if x.stride(1) == 1 or width == 1 else x.contiguous()


def _check_temperature(what, temperature):
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"{what}: temperature must be positive, got {temperature}")


def _checked_options(logits, ids, teacher_logits, teacher_lse, labels, label_weight, temperature, ignore_index, reduction, grad_scale):
    lead = tuple(logits.shape[:-1])
    given = [("ids", ids), ("teacher_logits", teacher_logits), ("teacher_lse", teacher_lse), ("labels", labels)]
    for name, x in given:
        if x is not None and x.device != logits.device:
            raise RuntimeError(f"distill_loss: logits are on {logits.device}, {name} on {x.device}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"distill_loss: ids must be int32 or int64, got {ids.dtype}")
    if teacher_logits.dtype not in DTYPES:
        raise TypeError(f"distill_loss: teacher_logits must be float16, bfloat16 or float32, got {teacher_logits.dtype}")
    if ids.dim() != logits.dim() or tuple(ids.shape[:-1]) != lead or ids.shape != teacher_logits.shape:
        raise ValueError(f"distill_loss: logits {tuple(logits.shape)}, ids {tuple(ids.shape)} and teacher_logits "
                         f"{tuple(teacher_logits.shape)} do not match")
    if not 1 <= ids.shape[-1] <= _lib.PS_MAX_TOP:
        raise ValueError(f"distill_loss: a list must have 1 .. {_lib.PS_MAX_TOP} entries, got {ids.shape[-1]}")
    if teacher_lse is not None:
        if teacher_lse.dtype != torch.float:
            raise TypeError(f"distill_loss: teacher_lse must be float32, got {teacher_lse.dtype}")
        if tuple(teacher_lse.shape) != lead:
            raise ValueError(f"distill_loss: teacher_lse must be {lead}, got {tuple(teacher_lse.shape)}")
    if labels is not None:
        if labels.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"distill_loss: labels must be int32 or int64, got {labels.dtype}")
        if tuple(labels.shape) != lead:
            raise ValueError(f"distill_loss: labels must be {lead}, got {tuple(labels.shape)}")
    if not 0.0 <= label_weight <= 1.0:
        raise ValueError(f"distill_loss: label_weight must be 0 .. 1, got {label_weight}")
    if label_weight > 0.0 and labels is None:
        raise ValueError("distill_loss: label_weight without labels")
    _check_temperature("distill_loss", temperature)
    if reduction not in REDUCTIONS:
        raise ValueError(f"distill_loss: reduction must be one of {REDUCTIONS}, got {reduction!r}")
    if grad_scale is not None:
        if reduction == "none":
            raise ValueError("distill_loss: grad_scale needs a loss that is one number")
        if isinstance(grad_scale, torch.Tensor) and (grad_scale.numel() != 1 or grad_scale.device != logits.device):
            raise ValueError(f"distill_loss: grad_scale must be one number on {logits.device}")
    return dict(label_weight=float(label_weight), temperature=float(temperature), ignore_index=int(ignore_index), reduction=reduction)


# --------------------------------------------------------------------------------------------------------------- calls


def _call(logits, ids, values, teacher_lse, labels, options):
    c = _lib.ps_distill_call()
    held = [ids, values]
    c.logits, c.ids, c.values = logits.data_ptr(), ids.data_ptr(), values.data_ptr()
    if teacher_lse is not None:
        teacher_lse = teacher_lse.contiguous()
        held.append(teacher_lse)
        c.teacher_lse = teacher_lse.data_ptr()
    if labels is not None:
        labels = labels.contiguous()
        held.append(labels)
        c.labels, c.labels_bytes = labels.data_ptr(), labels.element_size()
    c.rows, c.vocab = logits.shape
    c.row_stride, c.ids_stride, c.values_stride = logits.stride(0), ids.stride(0), values.stride(0)
    c.ignore_index, c.k = options["ignore_index"], ids.shape[1]
    c.dtype, c.values_dtype, c.ids_bytes = DTYPES[logits.dtype], DTYPES[values.dtype], ids.element_size()
    c.mean = options["reduction"] == "mean"
    c.temperature, c.label_weight = options["temperature"], options["label_weight"]
    return c, held


def _forward(logits, ids, values, teacher_lse, labels, options, backward=False, grad_scale=None):
    """Loss, and what backward needs: [stats of every row, denominator, factor of the gradient made here], that gradient."""
    c, held = _call(logits, ids, values, teacher_lse, labels, options)
    n, device = logits.shape[0], logits.device
    row_loss = torch.empty(n, dtype=torch.float, device=device)
    loss = row_loss if options["reduction"] == "none" else torch.empty((), dtype=torch.float, device=device)
    kept = torch.empty(4 * n + 2 if backward else 1, dtype=torch.float, device=device)
    c.row_loss, c.denominator = row_loss.data_ptr(), kept[-1:].data_ptr()
    if loss is not row_loss:
        c.loss = loss.data_ptr()
    grad = None
    if backward:
        c.stats = kept.data_ptr()
        if grad_scale is not None:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=device)
            c.grad, c.upstream_used = grad.data_ptr(), kept[-2:].data_ptr()
            if isinstance(grad_scale, torch.Tensor):
                c.upstream = grad_scale.data_ptr()
            else:
                c.upstream_value = grad_scale
    with _lib.on_device(device):
        _lib.check(_lib.load().ps_distill_loss(_lib.address(c), _lib.raw_stream(device)), "ps_distill_loss")
    return loss, kept, grad


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, values, teacher_lse, labels, options, grad_scale):
        loss, kept, ctx.grad = _forward(logits, ids, values, teacher_lse, labels, options, backward=True, grad_scale=grad_scale)
        ctx.save_for_backward(logits, ids, values, teacher_lse, labels, kept)
        ctx.options = options
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        logits, ids, values, teacher_lse, labels, kept = ctx.saved_tensors
        c, held = _call(logits, ids, values, teacher_lse, labels, ctx.options)
        # the gradient that forward made is handed out once: whoever gets it may write to it
        grad, ctx.grad = ctx.grad, None
        c.stats, c.denominator = kept.data_ptr(), kept[-1:].data_ptr()
        c.upstream = upstream.data_ptr()
        c.upstream_stride = upstream.stride(0) if upstream.dim() else 0
        if grad is None:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        else:
            c.upstream_used = kept[-2:].data_ptr()
        c.grad = grad.data_ptr()
        with _lib.on_device(logits.device):
            _lib.check(_lib.load().ps_distill_loss_backward(_lib.address(c), _lib.raw_stream(logits.device)), "ps_distill_loss_backward")
        return grad, None, None, None, None, None, None
