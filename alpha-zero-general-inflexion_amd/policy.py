"""Operators over rows of policy logits (csrc/azg_policy.hip), beside the trainer's HeadsLoss
(wino_train.py) and the search's softmax heads:

  action_logprobs     log-probabilities of given actions, the policy's entropy and its top
                      alternatives; differentiable (policy-gradient losses, entropy bonus)
  distill_loss        KL(teacher || student) from a teacher's top alternatives; differentiable
  distill_loss_grad   the same loss with its gradient in one call (no autograd graph)

A teacher's `action_logprobs(..., top=k)` is what the student's distill_loss reads; a search's
visit counts are such a teacher too (ids of the visited actions, logarithms of their counts).

Logits are [..., V], f32, bf16 or f16 on a HIP device (no CPU fallback): leading dimensions are
rows, of any strides that fold into two (a padded buffer's rows, logits[:, :-1]; others are copied).
Statistics and losses are f32, gradients have the logits' type.  `mask` ([..., V] or anything that
broadcasts to it, bool or uint8) marks the legal actions: what stands at an illegal one is not read as a
number (infinities and NaN there do not matter), its probability and its gradient are 0.  A legal
logit of -inf is probability 0; a legal NaN or +inf makes its row's numbers NaN.  All work is queued on
the current stream of the logits' device; nothing synchronises, and results do not depend on the
order in which blocks run.  Gradients are those of reverse mode, once; a forward-mode tangent is refused."""
import functools
import math
import struct
from collections import namedtuple

import torch
from torch.autograd import forward_ad

from . import _lib

TOP_MAX = 128      # azg.h AZG_POLICY_TOP_MAX
VOCAB_MAX = 1 << 29
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # enum azg_dtype

ActionLogprobs = namedtuple("ActionLogprobs", "logp entropy lse top_logp top_ids")


# azg_logits and azg_teacher as bytes (the calls copy them): a fifth of what a ctypes.Structure costs to fill
_LOGITS = struct.Struct("PPqqqqqqqif").pack
_TEACHER = struct.Struct("PPiiii").pack
_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(i).cuda_stream without the Stream object


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(device, fn, *args):
    """fn(*args, stream) on the device of the logits, whichever is current."""
    i = device.index
    if torch.cuda.current_device() == i:
        _lib.check(fn(*args, _stream(i)))
    else:
        with torch.cuda.device(i):
            _lib.check(fn(*args, _stream(i)))


def _fold(shape, *strides):
    """The leading dimensions `shape` as (outer, inner) rows shared by every tensor of `strides`:
    (inner, [(outer stride, inner stride), ...]), or None if two levels do not hold them."""
    dims = []  # [size, [stride of each tensor]]
    for n, st in zip(shape, zip(*strides)):
        if n == 1:
            continue
        if dims and all(a == b * n for a, b in zip(dims[-1][1], st)):
            dims[-1][0] *= n
            dims[-1][1] = st
        else:
            dims.append([n, st])
    if len(dims) > 2:
        return None
    zero = (0,) * len(strides)
    while len(dims) < 2:
        dims.insert(0, [1, zero])
    return dims[1][0], list(zip(dims[0][1], dims[1][1]))


def _check_logits(name, logits, temperature):
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES:
        raise ValueError(f"{name}: logits must be a float32, bfloat16 or float16 tensor")
    if not logits.is_cuda:
        raise _lib.AzgError(f"{name} runs on a HIP device (no CPU fallback)")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= VOCAB_MAX:
        raise ValueError(f"{name}: logits need a last dimension of 1 to {VOCAB_MAX} actions, got "
                         f"{tuple(logits.shape)}")
    t = float(temperature)
    if not (1e-6 <= t <= 1e6):
        raise ValueError(f"{name}: temperature {temperature} (1e-6 to 1e6)")
    return t


def _check_tangents(name, *tensors):
    """The kernels read values alone: a tangent would be dropped."""
    if forward_ad._current_level < 0:  # outside of dual_level(), the usual case
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative")


def _check_mask(name, logits, mask):
    if mask is None:
        return None
    if mask.dtype is not torch.bool and mask.dtype is not torch.uint8:
        raise ValueError(f"{name}: mask must be bool or uint8, got {mask.dtype}")
    if mask.device != logits.device:
        raise ValueError(f"{name}: mask on {mask.device}, logits on {logits.device}")
    if mask.shape != logits.shape:
        try:
            mask = mask.expand(logits.shape)
        except RuntimeError:
            raise ValueError(f"{name}: mask {tuple(mask.shape)} does not broadcast to the logits' "
                             f"{tuple(logits.shape)}") from None
    return mask


def _rows(logits, mask, temperature):
    """(logits, mask, rows, azg_logits): copies only where the strides do not fold."""
    V = logits.shape[-1]
    n = logits.numel() // V
    if logits.is_contiguous() and (mask is None or mask.is_contiguous()):
        return logits, mask, n, _LOGITS(logits.data_ptr(), 0 if mask is None else mask.data_ptr(), n, max(n, 1), 0, V, 0,
                                        V, V, _DTYPES[logits.dtype], temperature)
    lead = logits.shape[:-1]
    if logits.stride(-1) != 1 and V > 1:
        logits = logits.contiguous()
    if mask is not None and mask.stride(-1) != 1 and V > 1:
        mask = mask.contiguous()
    both = (logits,) if mask is None else (logits, mask)
    f = _fold(lead, *(t.stride()[:-1] for t in both))
    if f is None:
        logits = logits.contiguous()
        both = (logits,) if mask is None else (logits, mask)
        f = _fold(lead, *(t.stride()[:-1] for t in both))
        if f is None:
            mask = mask.contiguous()
            f = _fold(lead, logits.stride()[:-1], mask.stride()[:-1])
    inner, st = f
    m = st[1] if mask is not None else (0, 0)
    return logits, mask, n, _LOGITS(logits.data_ptr(), _ptr(mask) or 0, n, inner, st[0][0], st[0][1], m[0], m[1], V,
                                    _DTYPES[logits.dtype], temperature)


def _check_ints(name, what, t, shape, device):
    if t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name}: {what} must be int64 or int32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: {what} on {t.device}, logits on {device}")
    if t.shape != shape:
        raise ValueError(f"{name}: {what} {tuple(t.shape)}, expected {tuple(shape)}")
    return t.contiguous()


def _spread(g):
    """(tensor, stride) of a per-row gradient or weight: an expanded scalar stays one value."""
    if g is None:
        return None, 0
    if g.dtype is not torch.float32:
        g = g.float()
    if g.numel() <= 1 or not any(g.stride()):
        return g, 0
    return g.contiguous(), 1


@functools.lru_cache(maxsize=1024)
def _logprobs_work(n, V, dtype, top):
    return _lib.lib().azg_logprobs_work(_LOGITS(1, 0, n, n, 0, 0, 0, 0, V, dtype, 1.0), top)


@functools.lru_cache(maxsize=1024)
def _distill_work(n, V, dtype, grad):
    return _lib.lib().azg_distill_work(_LOGITS(1, 0, n, n, 0, 0, 0, 0, V, dtype, 1.0), grad)


def _work(nbytes, device):
    if nbytes < 0:  # all else is checked by now
        raise ValueError("more than 2^35 rows, or 2^60 logits")
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _logprobs(logits, actions, top, t, mask, want_stats):
    lead, dev = logits.shape[:-1], logits.device
    logits, mask, n, L = _rows(logits, mask, t)
    logp = top_logp = top_ids = stats = None
    # One allocation, but tensors of their own: to autograd unsafe_chunk's results are no views, so they may be written
    # with what requires a gradient, and a write to one is none to the others (three allocations: 1.1 to 3.1 us more)
    c = 2 if actions is None else 3
    if lead:
        rows = torch.unsafe_chunk(torch.empty((c * lead[0], *lead[1:]), dtype=torch.float32, device=dev), c)
    else:
        rows = [torch.empty((), dtype=torch.float32, device=dev) for _ in range(c)]
    entropy, lse = rows[:2]
    if c == 3:
        logp = rows[2]
    if top:
        top_logp = torch.empty((*lead, top), dtype=torch.float32, device=dev)
        top_ids = torch.empty((*lead, top), dtype=torch.int64, device=dev)
    if want_stats:
        stats = torch.empty((n, 4), dtype=torch.float32, device=dev)
    if n:
        nb = _logprobs_work(n, logits.shape[-1], _DTYPES[logits.dtype], top)
        work = _work(nb, dev)
        _call(dev, _lib.lib().azg_logprobs_fwd, L, _ptr(actions), actions is not None and
              actions.dtype is torch.int64, top, _ptr(stats), _ptr(logp), entropy.data_ptr(), lse.data_ptr(),
              _ptr(top_logp), _ptr(top_ids), _ptr(work), nb)
    return logits, mask, (logp, entropy, lse, top_logp, top_ids), stats


class _ActionLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, top, t, mask):
        x, m, out, stats = _logprobs(logits, actions, top, t, mask, True)
        ctx.save_for_backward(x, m, actions, stats)
        ctx.t = t
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(o for o in out[3:] if o is not None))
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logp, g_entropy, g_lse, _a, _b):
        logits, mask, actions, stats = ctx.saved_tensors
        if g_logp is None and g_entropy is None and g_lse is None:
            return None, None, None, None, None
        _check_tangents("action_logprobs' gradient", g_logp, g_entropy, g_lse)
        logits, mask, n, L = _rows(logits, mask, ctx.t)
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if n:
            (a, sa), (e, se), (z, sz) = _spread(g_logp), _spread(g_entropy), _spread(g_lse)
            _call(logits.device, _lib.lib().azg_logprobs_bwd, L, _ptr(actions), actions is not None and
                  actions.dtype is torch.int64, stats.data_ptr(), _ptr(a), sa, _ptr(e), se, _ptr(z), sz, dx.data_ptr())
        return dx, None, None, None, None


def action_logprobs(logits, actions=None, *, top=0, temperature=1.0, mask=None):
    """Log-probabilities of given actions under softmax(logits / temperature) over the legal actions, with the
    policy's entropy and its `top` (at most 128, at most V) likeliest alternatives.

    actions [...] (int64 or int32; None: no logp): one per row; an action outside 0..V-1 (padding) has
    log-probability 0 and no gradient, an illegal one -inf.  Returns ActionLogprobs:
      logp, entropy, lse [...]   f32; lse = log sum exp(logits / temperature); differentiable; logp <= 0 <= entropy
      top_logp, top_ids [..., top]  f32 / int64 (None when top = 0), likeliest first, equal logits in
                                 the order of their indices; not differentiable
    A row with fewer than `top` legal actions of probability above 0 is filled up with -inf and -1; one without any
    has entropy 0, lse and logp -inf, and gradient 0."""
    t = _check_logits("action_logprobs", logits, temperature)
    if isinstance(top, bool) or not isinstance(top, int) or not 0 <= top <= min(TOP_MAX, logits.shape[-1]):
        raise ValueError(f"action_logprobs: top = {top!r} (an int from 0 to min({TOP_MAX}, V = {logits.shape[-1]}))")
    mask = _check_mask("action_logprobs", logits, mask)
    _check_tangents("action_logprobs", logits)
    if actions is not None:
        actions = _check_ints("action_logprobs", "actions", actions, logits.shape[:-1], logits.device)
    if logits.requires_grad and torch.is_grad_enabled():
        return ActionLogprobs(*_ActionLogprobs.apply(logits, actions, top, t, mask))
    return ActionLogprobs(*_logprobs(logits, actions, top, t, mask, False)[2])


def _check_teacher(name, logits, teacher_logp, teacher_ids):
    lead = logits.shape[:-1]
    if teacher_logp.dtype not in _DTYPES:
        raise ValueError(f"{name}: teacher_logp must be float32, bfloat16 or float16, got {teacher_logp.dtype}")
    if teacher_logp.dim() != len(lead) + 1 or teacher_logp.shape[:-1] != lead or \
            not 1 <= teacher_logp.shape[-1] <= TOP_MAX:
        raise ValueError(f"{name}: teacher_logp {tuple(teacher_logp.shape)}, expected {tuple(lead)} + (1 to {TOP_MAX},)")
    if teacher_logp.device != logits.device:
        raise ValueError(f"{name}: teacher_logp on {teacher_logp.device}, logits on {logits.device}")
    if teacher_logp.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: the teacher gets no gradient: detach teacher_logp")
    _check_tangents(name, logits, teacher_logp)
    ids = _check_ints(name, "teacher_ids", teacher_ids, teacher_logp.shape, logits.device)
    if teacher_logp.requires_grad:
        teacher_logp = teacher_logp.detach()
    return teacher_logp.contiguous(), ids


def _teacher(logp, ids, rest):
    return _TEACHER(logp.data_ptr(), ids.data_ptr(), _DTYPES[logp.dtype], ids.dtype is torch.int64, logp.shape[-1],
                    bool(rest))


def _distill(logits, mask, t, t_logp, t_ids, rest, weight, scale, want_stats, want_total, want_grad):
    """(row losses, total, gradient, stats) of scale sum_r weight_r KL_r."""
    lead, dev, shape = logits.shape[:-1], logits.device, logits.shape
    logits, mask, n, L = _rows(logits, mask, t)
    loss = torch.empty(lead, dtype=torch.float32, device=dev)
    total = torch.empty((), dtype=torch.float32, device=dev) if want_total else None
    dx = torch.empty(shape, dtype=logits.dtype, device=dev) if want_grad else None
    stats = torch.empty((n, 8), dtype=torch.float32, device=dev) if want_stats else None
    if n:
        w, ws = _spread(weight)
        nb = _distill_work(n, shape[-1], _DTYPES[logits.dtype], want_grad)
        work = _work(nb, dev)
        _call(dev, _lib.lib().azg_distill_fwd, L, _teacher(t_logp, t_ids, rest), _ptr(stats), loss.data_ptr(), _ptr(w),
              ws, scale, _ptr(total), _ptr(dx), _ptr(work), nb)
    elif want_total:
        total.zero_()
    return logits, mask, loss, total, dx, stats


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, t_logp, t_ids, t, mask, rest, reduction):
        n = logits.numel() // logits.shape[-1]
        ctx.scale = 1.0 / max(n, 1) if reduction == "mean" else 1.0
        x, m, loss, total, _, stats = _distill(logits, mask, t, t_logp, t_ids, rest, None, ctx.scale, True,
                                               reduction != "none", False)
        ctx.save_for_backward(x, m, t_logp, t_ids, stats)
        ctx.t, ctx.rest = t, rest
        return loss if reduction == "none" else total

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, mask, t_logp, t_ids, stats = ctx.saved_tensors
        _check_tangents("distill_loss's gradient", g)
        logits, mask, n, L = _rows(logits, mask, ctx.t)
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if n:
            w, ws = _spread(g)
            _call(logits.device, _lib.lib().azg_distill_bwd, L, _teacher(t_logp, t_ids, ctx.rest), stats.data_ptr(),
                  w.data_ptr(), ws, ctx.scale, dx.data_ptr())
        return dx, None, None, None, None, None, None


def distill_loss(logits, teacher_logp, teacher_ids, *, temperature=1.0, mask=None, rest=False, reduction="mean"):
    """KL(teacher || student) of each row, the teacher given by its top alternatives, the student by
    softmax(logits / temperature) over the legal actions.

    teacher_logp, teacher_ids [..., k], 1 <= k <= 128: log-probabilities (f32, bf16, f16; already at the
    temperature) and their actions (int64 or int32); an entry of -inf or with an id outside 0..V-1 is none, an
    action given twice counts with both its probabilities.
      rest=False  the teacher's probabilities are softmax(teacher_logp) over its entries (any constant per row
                  may be added: logits or log visit counts do)
      rest=True   they are exp(teacher_logp), and what they leave of 1 is compared with all the mass that
                  the student gives to actions outside the entries (left out where it has none to give)
    reduction: "mean" (over all rows), "sum" (both 0-dim) or "none" ([...], f32).  A row without an entry or
    without a legal action counts 0 and gets no gradient, whatever its logits are.  An entry at an action that the student cannot play (illegal, or a logit of
    -inf) makes its row's loss +inf; its gradient is that of the others.  The teacher gets no gradient."""
    t = _check_logits("distill_loss", logits, temperature)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"distill_loss: reduction {reduction!r} ('mean', 'sum' or 'none')")
    mask = _check_mask("distill_loss", logits, mask)
    t_logp, t_ids = _check_teacher("distill_loss", logits, teacher_logp, teacher_ids)
    if logits.requires_grad and torch.is_grad_enabled():
        return _DistillLoss.apply(logits, t_logp, t_ids, t, mask, bool(rest), reduction)
    n = logits.numel() // logits.shape[-1]
    _, _, loss, total, _, _ = _distill(logits, mask, t, t_logp, t_ids, rest, None,
                                       1.0 / max(n, 1) if reduction == "mean" else 1.0, False, reduction != "none",
                                       False)
    return loss if reduction == "none" else total


def distill_loss_grad(logits, teacher_logp, teacher_ids, *, temperature=1.0, mask=None, rest=False, weight=None):
    """(loss, gradient) of sum_r weight_r KL_r (distill_loss's rows) in one call: what a training step needs, with
    one pass over the logits less than autograd.  weight: a number, or a tensor [...] of one per row (any floating
    type, taken as f32); None: 1 / rows (the mean).  The loss is 0-dim f32, the gradient has the logits' shape and type (a new contiguous tensor):
    logits.backward(gradient).  No autograd graph is built: in a training step captured in a HIP graph, or with the
    loss scaled from outside (weight), this is the form to take."""
    t = _check_logits("distill_loss_grad", logits, temperature)
    mask = _check_mask("distill_loss_grad", logits, mask)
    t_logp, t_ids = _check_teacher("distill_loss_grad", logits, teacher_logp, teacher_ids)
    w, scale = None, 1.0
    if weight is None:
        scale = 1.0 / max(logits.numel() // logits.shape[-1], 1)
    elif isinstance(weight, torch.Tensor):
        if weight.device != logits.device or not weight.is_floating_point():
            raise ValueError("distill_loss_grad: weight must be a floating-point tensor on the logits' device")
        if weight.dim() and weight.shape != logits.shape[:-1]:
            raise ValueError(f"distill_loss_grad: weight {tuple(weight.shape)}, expected "
                             f"{tuple(logits.shape[:-1])} or one number")
        _check_tangents("distill_loss_grad", weight)
        w = weight.detach()
    else:
        scale = float(weight)
        if not math.isfinite(scale):
            raise ValueError(f"distill_loss_grad: weight {weight}")
    if logits.requires_grad:
        logits = logits.detach()
    _, _, _, total, dx, _ = _distill(logits, mask, t, t_logp, t_ids, rest, w, scale, False, True, True)
    return total, dx


__all__ = ["ActionLogprobs", "action_logprobs", "distill_loss", "distill_loss_grad"]
