"""``einpolicy``: clipped policy loss with a KL term, from logits.

For a token with logits ``z`` over the vocabulary axis, sampled id ``a``,
log-probability ``old`` under the policy that sampled it and advantage ``A``,

    lp   = z_a / T - log sum_j exp(z_j / T)
    r    = exp(lp - old)
    loss = -min(r A, clip(r, 1 - low, 1 + high) A) + kl * (exp(ref - lp) - (ref - lp) - 1)

reduced over the tokens that ``mask`` keeps.  Neither probabilities nor a 32-bit
copy of the logits is ever written: with gradients, the forward pass also writes
that of the logits (``csrc/policy.cu``), which backward hands out, so a training
step reads the logits once.  A token that the mask leaves out
has no loss and a gradient of exactly zero, whatever its logits, id and other
inputs hold.  A kept id outside the vocabulary makes the loss NaN.

CUDA logits of 16 and 32 bits run natively, everything else on torch.  An
extension of this framework.
"""

import math
from functools import lru_cache
from typing import NamedTuple

import torch

from ..notation.families import cached_expand_axis_families
from ..notation.parser import parse_sharding
from ..notation.spec import AxisGroup, EllipsisAxis
from . import _native

__all__ = ["PolicyLoss", "einpolicy"]

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_FLOATS = (*_TYPES, torch.float64)
_REDUCTIONS = {"mean": 0, "sequence": 1, "sum": 2}


class PolicyLoss(NamedTuple):
    """``loss`` (differentiable) with the KL term, ``kl`` and the share of ``clipped`` tokens under the same
    reduction, and ``logp`` of every token (0 where masked)."""

    loss: torch.Tensor
    logp: torch.Tensor
    kl: torch.Tensor
    clipped: torch.Tensor


def _on_kernels(x):
    if not x.is_cuda or x.dtype not in _TYPES:
        return False
    if _native.available():
        return True
    if _native.allow_fallback():
        return False
    _native.require()  # raises: native extension missing on a CUDA machine
    return False


def _torch_policy(logits, ids, mask, old, ref, adv, conf):
    length, low, high, kl_weight, temperature, reduction, weight = conf
    vocab = logits.shape[-1]
    logits = logits.reshape(-1, vocab)
    tokens = logits.shape[0]
    wide = torch.promote_types(logits.dtype, torch.float32)
    keep = torch.ones(tokens, dtype=torch.bool, device=logits.device) if mask is None else mask
    z = torch.where(keep[:, None], logits.to(wide), 0)
    z = (z - z.detach().amax(1, keepdim=True)) / temperature  # differences of very large logits stay what they are
    known = (ids >= 0) & (ids < vocab)
    lp = z.gather(1, torch.where(known, ids, 0)[:, None])[:, 0] - torch.logsumexp(z, 1)
    lp = torch.where(known | ~keep, lp, float("nan"))

    def kept(t, other=0):
        return torch.where(keep, t.to(wide), other)

    adv = kept(adv if adv.shape[0] == tokens else adv.repeat_interleave(length))
    ratio = torch.exp(lp - (lp.detach() if old is None else torch.where(keep, old.to(wide), lp.detach())))
    clip = ratio.clamp(1 - low, 1 + high)
    gain = torch.where((adv == 0) & ~torch.isnan(lp), 0, torch.minimum(ratio * adv, clip * adv))
    clipped = (ratio * adv > clip * adv).to(wide)
    if ref is None:
        kl = torch.zeros_like(lp)
    else:
        away = torch.where(keep, ref.to(wide), lp.detach()) - lp
        kl = torch.expm1(away) - away
    count = keep.view(-1, length).sum(1)

    def reduced(t):
        t = kept(t).view(-1, length).sum(1)
        if reduction == _REDUCTIONS["sum"]:
            return t.sum()
        if reduction == _REDUCTIONS["mean"]:
            return t.sum() / count.sum().clamp(min=1)
        return (t / count.clamp(min=1)).sum() / (count > 0).sum().clamp(min=1)

    loss = weight * reduced(-gain + kl_weight * kl)
    return loss, reduced(kl).detach(), reduced(clipped).detach(), kept(lp).detach()


@lru_cache(maxsize=1024)
def _vocabulary(shard, axis, rank):
    """The vocabulary's dimension."""
    spec = parse_sharding(f"{shard} -> {shard}")[0]
    if getattr(spec, "partials", ()):
        raise ValueError("einpolicy does not take partial sums")
    names = []
    for a in spec.axes:
        if isinstance(a, (AxisGroup, EllipsisAxis)):
            raise NotImplementedError("einpolicy needs every axis named, none factored")
        if not a.local():
            raise NotImplementedError(f"einpolicy needs axis {a.name!r} whole on every rank")
        if a.name in names:
            raise ValueError(f"Axis {a.name!r} appears more than once")
        names.append(a.name)
    if rank != len(names):
        raise ValueError(f"The logits have {rank} dimensions, {shard!r} names {len(names)} axes")
    if axis not in names:
        raise ValueError(f"Axis {axis!r} is not among the logits' axes")
    return names.index(axis)


def _token_input(t, name, shapes, logits):
    """A constant of the loss as contiguous fp32 (fp64 beside fp64 logits)."""
    if t.device != logits.device or not t.is_floating_point():
        raise ValueError(f"{name} must be floating-point on {logits.device}, not {t.dtype} on {t.device}")
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name} must have the shape {' or '.join(str(s) for s in shapes)}, not {tuple(t.shape)}")
    if t.requires_grad:
        raise ValueError(f"{name} is a constant of the loss: detach it")
    return _flat(t.to(torch.float64 if logits.dtype == torch.float64 else torch.float32).resolve_neg())


def _flat(t):
    """One contiguous row."""
    return t.reshape(-1).contiguous()


def einpolicy(shard, logits, ids, *, axis, advantages, old_logp=None, ref_logp=None, mask=None, clip=0.2, kl=0.0,
              temperature=1.0, reduction="mean", weight=1.0, families=None):
    """Clipped policy loss of ``logits`` (see the module docstring) as a :class:`PolicyLoss`.

    ``shard`` names the axes of the logits ("b s v"), ``axis`` the vocabulary.
    The last of the other axes runs along a sequence.  ``ids`` (integers),
    ``old_logp``, ``ref_logp`` and ``mask`` (truth values, True keeps) have
    those other axes; ``advantages`` too, or one value a sequence.  Without
    ``old_logp`` the ratio is 1 and its gradient that of ``lp`` (on-policy);
    without ``ref_logp`` there is no KL term.  ``clip`` is one margin or
    ``(low, high)``.  ``reduction``: "mean" over kept tokens, "sequence" (mean
    over the tokens of a sequence, then over sequences that keep any) or "sum";
    no kept token at all gives 0.  ``weight`` multiplies the loss (a share of
    accumulated steps): here it is free, where a factor outside makes backward
    form the gradient again."""
    if families is not None:
        shard, _ = cached_expand_axis_families(shard, families=families)
    if logits.dtype not in _FLOATS:
        raise TypeError(f"einpolicy takes floating-point logits, not {logits.dtype}")
    place = _vocabulary(shard, axis, logits.dim())
    shape = tuple(logits.shape[:place]) + tuple(logits.shape[place + 1:])
    vocab = logits.shape[place]
    if vocab == 0:
        raise ValueError(f"The vocabulary axis {axis!r} is empty")
    low, high = (clip, clip) if isinstance(clip, (int, float)) else clip
    if not (0 <= low <= 1 and high >= 0):
        raise ValueError(f"clip margins must be 0 <= low <= 1 and high >= 0, not {low} and {high}")
    if not (math.isfinite(kl) and kl >= 0):
        raise ValueError(f"kl must be finite and not negative, not {kl}")
    if kl > 0 and ref_logp is None:
        raise ValueError("a KL term needs ref_logp")
    if not (math.isfinite(temperature) and temperature > 0):
        raise ValueError(f"temperature must be finite and positive, not {temperature}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(map(repr, _REDUCTIONS))}, not {reduction!r}")
    if not math.isfinite(weight):
        raise ValueError(f"weight must be finite, not {weight}")
    if ids.dtype not in (torch.int64, torch.int32) or tuple(ids.shape) != shape or ids.device != logits.device:
        raise ValueError(f"ids must be integers of the shape {shape} on {logits.device}, not {ids.dtype}, "
                         f"{tuple(ids.shape)} on {ids.device}")
    if mask is not None and (mask.dtype != torch.bool or tuple(mask.shape) != shape or mask.device != logits.device):
        raise ValueError(f"mask must be truth values of the shape {shape} on {logits.device}, not {mask.dtype}, "
                         f"{tuple(mask.shape)} on {mask.device}")
    adv = _token_input(advantages, "advantages", [shape, shape[:-1]] if shape else [shape], logits)
    old = None if old_logp is None else _token_input(old_logp, "old_logp", [shape], logits)
    ref = None if ref_logp is None else _token_input(ref_logp, "ref_logp", [shape], logits)

    tokens = math.prod(shape)
    if tokens == 0:
        zero = logits.detach().new_zeros((), dtype=torch.promote_types(logits.dtype, torch.float32))
        return PolicyLoss(logits.sum(dtype=zero.dtype), zero.expand(shape), zero, zero)
    rows = logits.resolve_neg()  # the kernels read raw memory
    rows = rows if place == len(shape) else rows.movedim(place, -1)
    mask = None if mask is None else _flat(mask)
    conf = (max(shape[-1], 1) if shape else 1, float(low), float(high), float(kl), float(temperature),
            _REDUCTIONS[reduction], float(weight))
    args = (rows, _flat(ids.long()), mask, old, ref, adv, conf)
    if not _on_kernels(logits):
        loss, kl_value, clipped, logp = _torch_policy(*args)
        return PolicyLoss(loss, logp.view(shape), kl_value, clipped)
    _native.refuse_tangents("einpolicy", logits, adv, old, ref)
    if torch.is_grad_enabled() and rows.requires_grad:
        loss, kl_value, clipped, logp = _native.require().policy(*args[:-1], *conf)
    else:
        rows = rows.reshape(tokens, vocab)
        if rows.stride(1) != 1 and vocab > 1:
            rows = rows.contiguous()
        loss, kl_value, clipped, logp, *_ = _native.require().policy_forward(rows, *args[1:-1], *conf, False)
    return PolicyLoss(loss, logp.view(shape), kl_value, clipped)
