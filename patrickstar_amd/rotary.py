"""Positions and norms of queries and keys, in front of attention.

``rotate_qk`` turns every head's query and key by the token's position, on one axis (text) or several (time, height and
width of a video's or an image's patches).  ``norm_rotate_qk`` divides them by their root mean square first and multiplies
by a weight, in the same pass over memory.  Both are differentiable; the hand-written kernels are behind
``include/ps_ops.h``.

Pair ``i`` of a head is turned by the angle ``position * inv_freq[i]``.  A float cannot hold that angle for long
sequences (at position 10**6 its last bit is 0.06 radians), so a plan keeps how far ONE position turns a pair as a 64-bit
fraction of a whole turn: multiplying that by the position wraps around exactly where the angle does.
"""
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

DTYPES = {torch.half: _lib.PS_F16, torch.bfloat16: _lib.PS_BF16, torch.float: _lib.PS_F32}


class RotaryPlan:
    """Which elements of a head form pairs, what axis each pair follows and how far a position turns it.

    ``rotary_dim``: so many elements at the front of a head are rotated, the rest passes (even).
    ``base``: pair ``i`` turns by ``base ** (-2 i / rotary_dim)`` radians a position; ``inv_freq`` gives the
    ``rotary_dim / 2`` numbers themselves instead.
    ``sections``: how many pairs each axis has, for positions on several axes.  They follow one another in blocks; with
    ``cycled`` they are dealt to the axes in turn, an axis that has its number being passed over.
    ``interleaved``: pairs are neighbours ``(2 i, 2 i + 1)`` instead of ``(i, i + rotary_dim / 2)``.

    A plan is made once and used for every call; it belongs to one device (by default the current GPU).
    """

    def __init__(self, rotary_dim, base=10000.0, *, inv_freq=None, sections=None, cycled=False, interleaved=False, device=None):
        if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, int) or rotary_dim < 2 or rotary_dim % 2:
            raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim!r}")
        if rotary_dim > _lib.PS_MAX_HEAD_DIM:
            raise ValueError(f"rotary_dim = {rotary_dim} is more than {_lib.PS_MAX_HEAD_DIM}")
        pairs = rotary_dim // 2
        if inv_freq is None:
            if not (base > 0 and math.isfinite(base)):
                raise ValueError(f"base must be positive, got {base}")
            inv_freq = [float(base) ** (-2.0 * i / rotary_dim) for i in range(pairs)]
        else:
            inv_freq = [float(f) for f in inv_freq]
            if len(inv_freq) != pairs or not all(math.isfinite(f) for f in inv_freq):
                raise ValueError(f"inv_freq must hold {pairs} finite numbers")
        sections = (pairs,) if sections is None else tuple(int(n) for n in sections)
        if not sections or min(sections) < 0 or sum(sections) != pairs:
            raise ValueError(f"sections {sections} must hold the {pairs} pairs of rotary_dim = {rotary_dim}")
        self.rotary_dim = rotary_dim
        self.interleaved = bool(interleaved)
        self.sections = sections
        self.axes = len(sections)
        self.axis_of_pair = _dealt(sections) if cycled else [a for a, n in enumerate(sections) for _ in range(n)]
        self.steps = [_step(f) for f in inv_freq]
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        # one row a pair: step, axis
        self.table = torch.tensor([[s, a] for s, a in zip(self.steps, self.axis_of_pair)], dtype=torch.int64, device=device)

    @property
    def device(self):
        return self.table.device


def _step(inv_freq):
    """Radians -> units of 2**-64 of a turn, modulo one turn, as a signed 64-bit number."""
    turns = math.fmod(inv_freq / (2.0 * math.pi), 1.0)
    step = int(turns * 2.0**64) % (1 << 64)
    return step - (1 << 64) if step >= 1 << 63 else step


def _dealt(sections):
    left, out = list(sections), []
    while any(left):
        for axis in range(len(left)):
            if left[axis]:
                left[axis] -= 1
                out.append(axis)
    return out


def rotate_qk(q, k, positions, plan):
    """Turn queries and keys by their positions; returns ``(q, k)`` as new contiguous tensors.

    ``q``, ``k``: ``[tokens, heads, head_dim]`` or ``[batch, tokens, heads, head_dim]`` on the GPU, fp16, bf16 or fp32, with
    their own numbers of heads; any strides (views of one projection's output, say), except that a last dimension that is
    not contiguous is copied first.  ``k`` may be None.  ``positions``: int32 or int64, ``[batch, tokens]`` or what expands to
    it, with a dimension for the axes in front if the plan has several.
    """
    out = _compiled(q, k, None, None, positions, plan, False, 0.0)
    if out is not None:
        return out
    q, k, positions = _checked("rotate_qk", q, k, positions, plan)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotate.apply(q, k, positions, plan)
    return _rotate(q, k, positions, plan)


def norm_rotate_qk(q, k, q_weight, k_weight, positions, plan, eps=1e-6):
    """``rotate_qk`` of ``x / sqrt(mean(x ** 2) + eps) * weight`` of every head, in one pass.

    ``q_weight``, ``k_weight``: ``[head_dim]``, of the queries' type or fp32, or None for ones.  Sums and norms are held in
    32 bits and the result is rounded once.  Gradients: of queries, keys and weights, the latter summed over tokens and heads
    in an order that does not change from call to call.
    """
    out = _compiled(q, k, q_weight, k_weight, positions, plan, True, eps)
    if out is not None:
        return out
    q, k, positions = _checked("norm_rotate_qk", q, k, positions, plan)
    if not eps >= 0.0:
        raise ValueError(f"norm_rotate_qk: eps must not be negative, got {eps}")
    q_weight, k_weight = _checked_weights(q, k, q_weight, k_weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _NormRotate.apply(q, k, q_weight, k_weight, positions, plan, float(eps))
    return _rotate(q, k, positions, plan, weights=(q_weight, k_weight), eps=float(eps))


def _compiled(q, k, q_weight, k_weight, positions, plan, norm, eps):
    """The call as csrc/ps_ops_binding.cpp makes it, or None where it is not of the ordinary form."""
    if type(plan) is not RotaryPlan:
        return None
    ops = _lib.load().ops
    if ops is None:
        return None
    return ops.ops_heads(q, k, q_weight, k_weight, positions, plan.table, plan.axes, plan.rotary_dim, plan.interleaved, norm, eps)


# -------------------------------------------------------------------------------------------------------------- checks


def _checked(what, q, k, positions, plan):
    if not isinstance(plan, RotaryPlan):
        raise TypeError(f"{what}: plan must be a RotaryPlan, got {type(plan).__name__}")
    for name, x in (("q", q), ("k", k)):
        if x is None and name == "k":
            continue
        if not x.is_cuda:
            raise RuntimeError(f"{what}: {name} must be a GPU tensor (got {x.device})")
        if x.device != q.device:
            raise RuntimeError(f"{what}: q is on {q.device}, {name} on {x.device}")
        if x.dtype not in DTYPES:
            raise TypeError(f"{what}: {name} must be float16, bfloat16 or float32, got {x.dtype}")
        if x.dim() not in (3, 4):
            raise ValueError(f"{what}: {name} must be [tokens, heads, head_dim] or [batch, tokens, heads, head_dim], got {tuple(x.shape)}")
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError(f"{what}: q is {q.dtype}, k {k.dtype}")
        if k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
            raise ValueError(f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ in more than their heads")
    if not 1 <= q.shape[-1] <= _lib.PS_MAX_HEAD_DIM:
        raise ValueError(f"{what}: head_dim must be 1 .. {_lib.PS_MAX_HEAD_DIM}, got {q.shape[-1]}")
    if plan.rotary_dim > q.shape[-1]:
        raise ValueError(f"{what}: the plan rotates {plan.rotary_dim} elements, a head has {q.shape[-1]}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: positions must be int32 or int64, got {positions.dtype}")
    if positions.device != q.device or plan.device != q.device:
        raise RuntimeError(f"{what}: q is on {q.device}, positions on {positions.device}, the plan on {plan.device}")
    lead = tuple(q.shape[:-2])
    wanted = lead if plan.axes == 1 else (plan.axes, *lead)
    if tuple(positions.shape) != wanted:
        try:
            if plan.axes > 1 and (positions.dim() < 1 or positions.shape[0] != plan.axes):
                raise RuntimeError
            if positions.dim() < len(wanted) and plan.axes > 1:  # the axes stay in front
                positions = positions.reshape(plan.axes, *[1] * (len(wanted) - positions.dim()), *positions.shape[1:])
            positions = positions.expand(wanted)
        except RuntimeError:
            raise ValueError(f"{what}: positions {tuple(positions.shape)} do not expand to {wanted}") from None
    return q, k, positions


def _checked_weights(q, k, q_weight, k_weight):
    if k is None and k_weight is not None:
        raise ValueError("norm_rotate_qk: k_weight without k")
    given = [(name, w) for name, w in (("q_weight", q_weight), ("k_weight", k_weight)) if w is not None]
    for name, w in given:
        if w.device != q.device:
            raise RuntimeError(f"norm_rotate_qk: q is on {q.device}, {name} on {w.device}")
        if w.dtype not in (q.dtype, torch.float):
            raise TypeError(f"norm_rotate_qk: {name} must be {q.dtype} or float32, got {w.dtype}")
        if tuple(w.shape) != (q.shape[-1],):
            raise ValueError(f"norm_rotate_qk: {name} must have {q.shape[-1]} elements, got {tuple(w.shape)}")
    if len(given) == 2 and q_weight.dtype != k_weight.dtype:
        raise TypeError(f"norm_rotate_qk: q_weight is {q_weight.dtype}, k_weight {k_weight.dtype}")
    return q_weight, k_weight


# --------------------------------------------------------------------------------------------------------------- calls


def _rows(x):
    """The tensor as its kernel takes it (elements of a head next to one another), and its strides of batch, token, head."""
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    s = x.stride()
    return x, ((0, s[0], s[1]) if x.dim() == 3 else s[:3])


def _call(q, k, positions, plan, weights=(None, None), eps=0.0, norm=False, inverse=False):
    """The descriptor, and what has to live until the launch."""
    c = _lib.ps_heads_call()
    shape = q.shape if q is not None else k.shape
    held = []
    strides = []
    for which, x in enumerate((q, k)):
        if x is None:
            strides += [0, 0, 0]
            continue
        x, s = _rows(x)
        held.append(x)
        strides += s
        c.x[which] = x.data_ptr()
        c.heads[which] = x.shape[-2]
        w = weights[which]
        if w is not None:
            w = w.contiguous()
            held.append(w)
            c.weight[which] = w.data_ptr()
            c.weight_dtype = DTYPES[w.dtype]
    c.x_stride[:] = strides
    c.dtype = DTYPES[held[0].dtype]
    if weights[0] is None and weights[1] is None:
        c.weight_dtype = c.dtype
    c.positions = positions.data_ptr()
    c.plan = plan.table.data_ptr()
    p = positions.stride() if plan.axes > 1 else (0, *positions.stride())
    c.position_stride[:] = p if len(p) == 3 else (p[0], 0, p[1])
    c.batch, c.tokens = (1, shape[0]) if len(shape) == 3 else shape[:2]
    c.dim, c.rotary, c.axes = shape[-1], plan.rotary_dim, plan.axes
    c.position_bytes = positions.element_size()
    c.interleaved, c.inverse, c.norm, c.eps = plan.interleaved, inverse, norm, eps
    return c, held


def _outputs(c, q, k):
    out = [None if x is None else torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k)]
    for which, x in enumerate(out):
        if x is not None:
            c.out[which] = x.data_ptr()
    return out


def _rotate(q, k, positions, plan, weights=None, eps=0.0, inverse=False):
    c, held = _call(q, k, positions, plan, weights or (None, None), eps, norm=weights is not None, inverse=inverse)
    out = _outputs(c, q, k)
    device = held[0].device
    with _lib.on_device(device):
        _lib.check(_lib.load().ps_rotate_heads(_lib.address(c), _lib.raw_stream(device)), "ps_rotate_heads")
    return tuple(out)


class _Rotate(torch.autograd.Function):
    """The gradient of a rotation is the gradient, turned back: nothing of the inputs is kept."""

    @staticmethod
    def forward(ctx, q, k, positions, plan):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.plan = plan
        return _rotate(q, k, positions, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, q_grad, k_grad):
        if q_grad is None and k_grad is None:
            return None, None, None, None
        return (*_rotate(q_grad, k_grad, *ctx.saved_tensors, ctx.plan, inverse=True), None, None)


class _NormRotate(torch.autograd.Function):
    """Keeps the inputs only: the roots are made again from them."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, plan, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.plan, ctx.eps = plan, eps
        return _rotate(q, k, positions, plan, weights=(q_weight, k_weight), eps=eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, q_grad, k_grad):
        q, k, q_weight, k_weight, positions = ctx.saved_tensors
        if q_grad is None and k_grad is None:
            return (None,) * 7
        # (an output that went nowhere has no part in it)
        q, q_weight = (q, q_weight) if q_grad is not None else (None, None)
        k, k_weight = (k, k_weight) if k_grad is not None else (None, None)
        weights = (q_weight, k_weight)
        c, held = _call(q, k, positions, ctx.plan, weights, ctx.eps, norm=True)
        out = _outputs(c, q, k)
        weight_grads = [None, None]
        for which, (x, g) in enumerate(((q, q_grad), (k, k_grad))):
            if x is None:
                continue
            g, s = _rows(g)
            held.append(g)
            c.grad[which] = g.data_ptr()
            c.grad_stride[3 * which : 3 * which + 3] = s
            if weights[which] is not None and ctx.needs_input_grad[2 + which]:
                weight_grads[which] = torch.empty(weights[which].shape, dtype=weights[which].dtype, device=x.device)
                c.weight_grad[which] = weight_grads[which].data_ptr()
        device = held[0].device
        lib = _lib.load()
        at = _lib.address(c)
        with _lib.on_device(device):
            size = lib.ps_norm_rotate_heads_workspace_bytes(at)
            workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
            _lib.check(
                lib.ps_norm_rotate_heads_backward(at, workspace.data_ptr() if size else None, size, _lib.raw_stream(device)),
                "ps_norm_rotate_heads_backward",
            )
        return (*out, *weight_grads, None, None, None)
