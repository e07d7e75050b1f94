"""``einnorm``: the norms before and after a block, fused with its gate and the scaled residual stream.

For a residual stream ``x`` and a block's output ``y`` over named axes,

    p = norm(y) * post_weight + post_bias     (``post=True``; otherwise p = y)
    h = scale * x + gate * p                  the new stream
    n = norm(h) * weight + bias               the next block's input

in one pass over x and y (``csrc/norm.cu``), and one for the gradients of all of
them.  ``kind`` is "layer" (mean and variance) or "rms".  The gate has its own
axes: a vector of the normalised axis, a row for every batch entry, one for
every token, a scalar; its gradient is summed over the axes it lacks.  (A gate
without the normalised axis, or with axes of the stream between its own, is
written out to rows in 32 bits, and so is its gradient before it is summed.)
The statistics, h before its norm and all sums are 32-bit; h and n are rounded
once, and n is the norm of h before that rounding.

Every axis but the normalised one may be sharded (the operation is local to a
rank; gradients of replicated parameters are reduced as those of any other
local operation are, by the registered hooks).  CUDA tensors of 16 and 32 bits
run natively, everything else on torch.  An extension of this framework.
"""

import math
from dataclasses import dataclass
from functools import lru_cache

import torch

from ..notation.families import cached_expand_axis_families
from ..notation.parser import parse_sharding
from ..notation.spec import AxisGroup, EllipsisAxis
from . import _native

__all__ = ["einnorm"]

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_FLOATS = (*_TYPES, torch.float64)


def _axes(formula, label):
    spec = parse_sharding(f"{formula} -> {formula}")[0]
    if getattr(spec, "partials", ()):
        raise ValueError(f"einnorm does not take partial sums in {label}")
    names = set()
    for axis in spec.axes:
        if isinstance(axis, AxisGroup):
            raise NotImplementedError(f"einnorm does not support factored axes in {label}")
        if axis.name in names:
            raise ValueError(f"Axis {axis.name!r} appears more than once in {label}")
        names.add(axis.name)
    return list(spec.axes)


def _written_out(axes, width):
    """Axis keys with the ellipsis replaced by one key for each of the ``width`` dimensions it covers."""
    out = []
    for a in axes:
        if isinstance(a, EllipsisAxis):
            out.extend(("...", i) for i in range(width))
        else:
            out.append(a)
    return out


@dataclass(frozen=True)
class _Plan:
    """What the formula and the shapes alone decide."""

    place: int       # the normalised dimension
    d: int
    lead: tuple      # lengths of the others, in order
    # the gate as [count, d], its row for a stream row r at (r // inner) % count: spread over d first
    # (it lacks the axis), permuted, viewed and expanded to the run of axes it covers (None where not needed)
    spread: bool = False
    order: tuple = None
    view: tuple = None
    run: tuple = None
    inner: int = 1
    count: int = 1


@lru_cache(maxsize=1024)
def _plan(shard, axis, gate_axes, shape, gate_shape):
    axes = _axes(shard, "the stream")
    width = max(len(shape) - sum(1 for a in axes if not isinstance(a, EllipsisAxis)), 0)
    keys = _written_out(axes, width)
    if len(keys) != len(shape):
        raise ValueError(f"The stream has {len(shape)} dimensions, {shard!r} names {len(axes)} axes")
    found = [k for k in keys if not isinstance(k, tuple) and k.name == axis]
    if not found:
        raise ValueError(f"Axis {axis!r} is not among the stream's axes")
    norm_key = found[0]
    if not norm_key.local():
        raise NotImplementedError(f"einnorm needs the normalised axis {axis!r} whole on every rank")
    place = keys.index(norm_key)
    d = shape[place]
    if d == 0:
        raise ValueError(f"The normalised axis {axis!r} is empty")
    lead_keys, lead = keys[:place] + keys[place + 1:], shape[:place] + shape[place + 1:]
    if gate_shape is None:
        if gate_axes is not None:
            raise ValueError("gate_axes without a gate")
        return _Plan(place, d, lead)
    if gate_axes is None:
        raise ValueError("gate needs gate_axes")
    gate_keys = _written_out(_axes(gate_axes, "the gate"), width) if gate_axes.strip() else []  # "": a scalar
    if len(gate_keys) != len(gate_shape):
        raise ValueError(f"The gate has {len(gate_shape)} dimensions, {gate_axes!r} names {len(gate_keys)} axes")
    for k, size in zip(gate_keys, gate_shape):
        if k not in keys:
            raise ValueError(f"The gate's axis {k} is not one of the stream's")
        if size != shape[keys.index(k)]:
            raise ValueError(f"The gate's axis {k} has length {size}, the stream's {shape[keys.index(k)]}")
    spread = norm_key not in gate_keys
    if spread:
        gate_keys = gate_keys + [norm_key]
    order = tuple(gate_keys.index(k) for k in [k for k in lead_keys if k in gate_keys] + [norm_key])
    # axes of length one change nothing; the others must cover a run of the stream's axes
    places = [i for i, k in enumerate(lead_keys) if k in gate_keys and lead[i] != 1]
    low, high = (places[0], places[-1] + 1) if places else (0, 0)
    run = lead[low:high]
    view = tuple(s if low + i in places else 1 for i, s in enumerate(run))
    inner = math.prod(lead[high:]) if places else math.prod(lead)
    return _Plan(place, d, lead, spread, None if order == tuple(range(len(order))) else order, view,
                 None if view == run else run, inner, math.prod(run))


def _check_like(t, x, name):
    if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} must have the stream's shape, dtype and device: {tuple(t.shape)}, {t.dtype} on "
                         f"{t.device} for {tuple(x.shape)}, {x.dtype} on {x.device}")


def _check_vector(t, x, d, name):
    if t is None:
        return
    if t.shape != (d,):
        raise ValueError(f"{name} must have the normalised axis alone ({d}), not {tuple(t.shape)}")
    _check_param(t, x, name)


def _check_param(t, x, name):
    if t.device != x.device or t.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{name} must be {x.dtype} or float32 on {x.device}, not {t.dtype} on {t.device}")


def _gate_rows(gate, plan):
    if plan.spread or plan.run is not None:
        # written out below: autograd sums the written-out rows' gradients, 32-bit ones, and rounds the sum once
        gate = gate.to(torch.promote_types(gate.dtype, torch.float32))
    if plan.spread:
        gate = gate.unsqueeze(-1).expand(*gate.shape, plan.d)
    if plan.order is not None:
        gate = gate.permute(plan.order)
    if plan.run is not None:
        # rows between the gate's own axes: written out (its gradient sums over them again, by autograd)
        gate = gate.reshape(*plan.view, plan.d).expand(*plan.run, plan.d)
    return gate.reshape(plan.count, plan.d)


def _last(t, plan):
    """t with the normalised axis last."""
    return t if t is None or plan.place == len(plan.lead) else t.movedim(plan.place, -1)


def _torch_norm(x, y, w, b, pw, pb, gate, conf):
    inner, count, post, center, scale, eps = conf
    dtype, shape = x.dtype, x.shape
    x = x.reshape(-1 if x.numel() else 0, shape[-1])
    y = None if y is None else y.reshape(x.shape)
    wide = torch.promote_types(dtype, torch.float32)

    def normed(t, weight, bias):
        if center:
            t = t - t.mean(-1, keepdim=True)
        t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps)
        t = t if weight is None else t * weight.to(wide)
        return t if bias is None else t + bias.to(wide)

    h = x.to(wide)
    if y is not None:
        p = y.to(wide)
        if post:
            p = normed(p, pw, pb)
        if gate is not None:
            rows = torch.arange(x.shape[0], device=x.device) // inner % count
            p = p * gate.to(wide)[rows]
        h = scale * h + p
    n = normed(h, w, b).to(dtype).view(shape)
    return (n,) if y is None else (h.to(dtype).view(shape), n)


def _on_kernels(x):
    if not x.is_cuda or x.dtype not in _TYPES:
        return False
    if _native.available():
        return True
    if _native.allow_fallback():
        return False
    _native.require()  # raises: native extension missing on a CUDA machine
    return False


def einnorm(shard, x, y=None, *, axis, weight=None, bias=None, kind="layer", eps=1e-5, post=False, post_weight=None,
            post_bias=None, gate=None, gate_axes=None, scale=1.0, families=None):
    """Residual stream and next input ``(h, n)`` after a block (see the module docstring).

    ``shard`` names the axes of ``x`` and ``y`` ("b s d"), ``axis`` the one that
    is normalised, ``gate_axes`` those of ``gate`` ("d", "b d", "b s d", "b", ...).
    Without ``y`` there is no block yet: ``h`` is ``x`` and ``n`` its norm.
    Parameters and gate are of the stream's type or fp32."""
    if families is not None:
        shard, _ = cached_expand_axis_families(shard, families=families)
        if gate_axes is not None:
            gate_axes, _ = cached_expand_axis_families(gate_axes, families=families)
    if x.dtype not in _FLOATS:
        raise TypeError(f"einnorm takes floating-point tensors, not {x.dtype}")
    plan = _plan(shard, axis, gate_axes, tuple(x.shape), None if gate is None else tuple(gate.shape))
    if kind not in ("layer", "rms"):
        raise ValueError(f"kind must be 'layer' or 'rms', not {kind!r}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps must be finite and not negative, not {eps}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, not {scale}")
    if y is None and (post or gate is not None or scale != 1.0):
        raise ValueError("post, gate and scale belong to a block's output y")
    if not post and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need post=True")
    if y is not None:
        _check_like(y, x, "y")
    _check_vector(weight, x, plan.d, "weight")
    _check_vector(bias, x, plan.d, "bias")
    _check_vector(post_weight, x, plan.d, "post_weight")
    _check_vector(post_bias, x, plan.d, "post_bias")
    inner, count = plan.inner, plan.count
    if gate is not None:
        _check_param(gate, x, "gate")
        if x.numel():
            gate = _gate_rows(gate, plan)
        else:
            gate, inner, count = gate.sum().expand(1, plan.d), 1, 1  # no row to weigh: a gradient of zero

    conf = (inner, count, bool(post), kind == "layer", float(scale), float(eps))
    args = [_last(x, plan), _last(y, plan)]
    args += [None if t is None else t.contiguous() for t in (weight, bias, post_weight, post_bias, gate)]
    if not _on_kernels(x):
        out = _torch_norm(*args, conf)
    else:
        out = _native.require().norm(*args, *conf)
    if plan.place != len(plan.lead):
        out = [t.movedim(-1, plan.place) for t in out]
    return (x, out[0]) if y is None else (out[0], out[1])
