"""Activations kept for backward in 8 bits: ``checkpoint8`` and the contractions that read it.

``checkpoint8(x)`` quantises ``x`` once and returns a :class:`Saved8` operand.
Given to :func:`einshard` as the first operand of a contraction, its value takes
part in the forward product as usual, and the codes (a quarter to a half of the
bytes) are what autograd keeps: the weight gradient is formed from what they
stand for,

    z = x w        dx = dz w^T        dw = x^^T dz

Several contractions of one operand (the q, k and v projections of a normed
stream) share its codes.  With ``activation="silu"`` the pre-activation is
kept in 8 bits too, quantised from the 32-bit product, and the result is
again a ``Saved8``: its value is the activation in the operand's type, and the
next contraction rebuilds the activation from the same codes instead of keeping
one of its own,

    a = silu(h)    dh = da silu'(h^)   dw2 = silu(h^)^T dz

Format: blocks of 32 consecutive channels of the last axis (a row's last block
may be shorter) share an exponent e = floor(log2 max|x|) - 6, one more if the
largest code would round to 128; codes are rint(x 2^-e) in int8, so a value is
at most half a step 2^(e-1) off.  Scaling by a power of two is exact, so codes
do not depend on the machine.  A block that holds an infinity or a NaN reads
back as NaN.

CUDA tensors of 16 and 32 bits run on ``csrc/quant8.cu``, everything else on
torch with the same results.  An extension of this framework: the reference
keeps activations whole or recomputes them.
"""

import math
import string
from dataclasses import dataclass
from functools import cached_property, lru_cache

import torch
from torch.autograd.function import once_differentiable

from . import _native, gemm
from .contraction import canonical_gemm, contract

__all__ = ["Saved8", "checkpoint8", "contract_saved", "silu_saved"]

_BLOCK = 32
_NAN = 255
_VALUE, _SILU, _SILU_GRAD = 0, 1, 2
_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _on_kernels(t, dtype) -> bool:
    if not t.is_cuda or dtype not in _CODE:
        return False
    if _native.available():
        return True
    if _native.allow_fallback():
        return False
    _native.require()  # raises: native extension missing on a CUDA machine
    return False


def _quantise(x):
    """(codes, exponent bytes) of a [rows, d] tensor."""
    if _on_kernels(x, x.dtype):
        return tuple(_native.require().quant8(x.contiguous()))
    x = x if x.dtype == torch.float64 else x.float()
    rows, d = x.shape
    blocks = torch.nn.functional.pad(x, (0, -d % _BLOCK)).reshape(rows, -(-d // _BLOCK), _BLOCK)
    amax = blocks.abs().amax(-1) if x.numel() else x.new_zeros(blocks.shape[:2])
    bad = ~torch.isfinite(amax)
    amax = torch.where(bad, 0, amax)
    e = (torch.frexp(amax).exponent - 7).clamp(min=-126)
    e = e + (torch.round(torch.ldexp(amax, -e)) > 127)
    bad |= e > 126  # outside fp32's range (fp64 values)
    q = torch.round(torch.ldexp(torch.where(bad[..., None], 0, blocks), -e[..., None]))
    codes = q.to(torch.int8).flatten(1)[:, :d].contiguous()
    return codes, torch.where(bad, _NAN, e + 127).to(torch.uint8)


def _restored(codes, exps, dtype, mode, grad=None):
    """[rows, d] values of the codes through ``mode`` (value, silu, grad * silu')."""
    if _on_kernels(codes, dtype):
        return _native.require().restore8(codes.contiguous(), exps, grad, _CODE[dtype], mode)
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    e = exps.to(torch.int32).repeat_interleave(_BLOCK, dim=1)[:, :codes.shape[1]]
    x = torch.ldexp(codes.to(wide), e - 127)
    limit = torch.finfo(dtype if mode == _VALUE else wide).max
    x = torch.where(e == _NAN, float("nan"), x.clamp(-limit, limit))
    if mode == _VALUE:
        return x.to(dtype)
    s = torch.sigmoid(x)
    if mode == _SILU:
        return (x * s).to(dtype)
    return (grad.to(wide) * s * (1 + x * (1 - s))).to(dtype)


def _rows(t):
    return t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(t.shape[:-1].numel(), t.shape[-1])


class Saved8:
    """A contraction operand that backward keeps in 8 bits.

    ``value`` is the tensor the forward pass uses (on the autograd graph);
    ``codes`` [rows, d] int8 and ``exps`` [rows, ceil(d / 32)] uint8 are what is
    kept.  ``restore()`` gives the values that backward sees.
    """

    __slots__ = ("value", "codes", "exps", "_act", "_base", "_order", "_pre", "_readers", "_box", "_version", "_ready")

    def __init__(self, value, codes, exps, act=False, base=None, order=None, pre=None):
        self.value, self.codes, self.exps = value, codes, exps
        self._act = act  # the codes are a pre-activation: the operand is its silu
        self._base = tuple(value.shape) if base is None else base  # shape of the tensor that was quantised
        self._order = order  # permutation from there to the value's axes
        self._pre = pre  # the pre-activation's place in the graph (a tensor without values of its own)
        self._readers = None  # the place where the gradients of its native contractions meet
        self._box = None  # and of the others, with what they leave there
        self._ready = None  # the operand's matrix where contractions read it from a copy with padded rows
        self._version = None if value.is_inference() else value._version  # what the codes were formed from

    @property
    def shape(self):
        return self.value.shape

    @property
    def dtype(self):
        return self.value.dtype

    @property
    def device(self):
        return self.value.device

    @property
    def nbytes(self):
        """Bytes that backward keeps."""
        rows, d = self.codes.shape
        return rows * (self.codes.stride(0) if d else 0) + self.exps.numel()  # up to 15 codes lie between two rows

    def restore(self):
        """The operand as backward reads it, in the value's type (no gradient)."""
        return _restore_operand(self.codes, self.exps, self._meta())

    def with_value(self, value):
        """The same codes for a value that differs by its place in the graph alone."""
        self.check_unchanged()
        if value is self.value:
            return self
        return Saved8(value, self.codes, self.exps, self._act, self._base, self._order)

    def check_unchanged(self):
        """Raise where the value has been modified in place since its codes were formed."""
        if self._version is not None and self.value._version != self._version:
            raise RuntimeError("a Saved8 operand's value has been modified in place since its codes were formed")

    def _meta(self):
        return self._act, self._base, self._order, self.value.dtype

    def __repr__(self):
        return f"Saved8({'silu, ' if self._act else ''}shape={tuple(self.shape)}, dtype={self.dtype}, {self.nbytes} bytes kept)"


def _restore_operand(codes, exps, meta):
    act, base, order, dtype = meta
    x = _restored(codes, exps, dtype, _SILU if act else _VALUE).view(base)
    return x if order is None else x.permute(order)


def checkpoint8(x):
    """Quantise ``x`` along its last axis and return it as a :class:`Saved8` operand."""
    if isinstance(x, Saved8):
        raise TypeError("checkpoint8 takes a tensor, not a Saved8")
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"checkpoint8 takes a tensor, not {type(x).__name__}")
    if x.dim() == 0:
        raise ValueError("checkpoint8 needs at least one axis")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32, torch.float64):
        raise TypeError(f"checkpoint8 takes a floating-point tensor, not {x.dtype}")
    x = x.resolve_neg()  # the kernels read raw memory
    codes, exps = _quantise(_rows(x.detach()))
    return Saved8(x, codes, exps)


# ------------------------------------------------------------------ contractions

def _explicit(equation, x_rank):
    """The equation with an ellipsis of the first operand written out, or None."""
    if "..." not in equation:
        return equation
    (ex, ey), ez = equation.split("->")[0].split(","), equation.split("->")[1]
    width = x_rank - len(ex.replace("...", ""))
    if "..." in ey or "..." not in ez or width < 0:
        return None
    free = [c for c in string.ascii_letters if c not in equation][:width]
    fill = "".join(free)
    return f"{ex.replace('...', fill)},{ey}->{ez.replace('...', fill)}"


def _inverse(order):
    back = [0] * len(order)
    for i, o in enumerate(order):
        back[o] = i
    return tuple(back)


def _moved(t, order):
    return t if order is None else t.permute(order)


def _order(names, wanted):
    """Permutation that brings axes ``names`` into the order ``wanted`` (None: they are in it)."""
    order = tuple(names.index(c) for c in wanted)
    return None if order == tuple(range(len(order))) else order


@dataclass(frozen=True)
class _Product:
    """A two-operand contraction as [batch, rows, red] x [batch, red, cols]."""

    equation: str
    gemm: tuple       # batch, rows, cols, red extents
    x_order: tuple    # x's axes to batch + rows + red, y's to batch + red + cols, the product's to the result's
    y_order: tuple
    z_order: tuple
    x_shape: tuple    # lengths in those orders
    y_shape: tuple
    z_shape: tuple    # (of the product)

    @cached_property
    def on_kernels(self):
        """The plan of csrc/bindings_saved8.cpp."""
        orders = [() if o is None else o for o in (self.x_order, self.y_order, self.z_order)]
        return _native.require().ContractPlan(self.gemm, *orders, self.x_shape, self.y_shape, self.z_shape)


@lru_cache(maxsize=1024)
def _product(equation, x_shape, y_shape):
    explicit = _explicit(equation, len(x_shape))
    plan = None if explicit is None else canonical_gemm(explicit, x_shape, y_shape)
    if plan is None or plan["x_only"] or plan["y_only"]:
        raise NotImplementedError("a Saved8 operand takes part in plain two-operand contractions only: no repeated, "
                                  "broadcast or summed-out axes")
    size = plan["size"]
    batch, rows, cols, red = (plan[k] for k in ("batch", "rows", "cols", "red"))

    def lengths(letters):
        return tuple(size[c] for c in letters)

    extents = tuple(math.prod(lengths(k)) for k in (batch, rows, cols, red))
    return _Product(explicit, extents, _order(list(plan["ex"]), batch + rows + red),
                    _order(list(plan["ey"]), batch + red + cols), _order(batch + rows + cols, list(plan["ez"])),
                    lengths(batch + rows + red), lengths(batch + red + cols), lengths(batch + rows + cols))


def _silu_forward(h, dtype):
    """(silu(h) in dtype, codes, exps) of an fp32 (fp64) [rows, d] pre-activation."""
    if h.dtype == torch.float32 and _on_kernels(h, dtype):
        return tuple(_native.require().quant8_silu(h.contiguous(), _CODE[dtype]))
    codes, exps = _quantise(h)
    return (h * torch.sigmoid(h)).to(dtype), codes, exps


def _silu_grad(grad, codes, exps, order):
    """grad * silu'(h^), in grad's axes; ``order`` leads from the quantised tensor's axes to them."""
    g = _moved(grad.resolve_neg(), None if order is None else _inverse(order))
    d = _restored(codes, exps, grad.dtype, _SILU_GRAD, g.reshape(codes.shape).contiguous()).view(g.shape)
    return _moved(d, order)


def _place_of(a):
    """A tensor that stands for a's pre-activation in the graph: its shape, without values."""
    return a.new_empty(()).expand(a.shape)


class _Final(torch.autograd.Function):
    """A gradient without a derivative of its own: under create_graph, using it further raises."""

    @staticmethod
    def forward(ctx, t, source):
        return t.view_as(t)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("trying to differentiate twice a function that was marked with once_differentiable")

    @classmethod
    def of(cls, grads, sources):
        """``grads`` as results of ``sources``, where a graph of the backward pass is wanted."""
        if torch.is_grad_enabled():
            for source in sources:
                if source is not None and source.requires_grad:
                    grads = tuple(None if g is None else cls.apply(g, source) for g in grads)
        return grads


class _Readers(torch.autograd.Function):
    """The place in the graph where the gradients of an operand's contractions meet.

    sum_i dz_i y_i^T is formed at once, in 32 bits, and rounded once; autograd
    would add the contractions' rounded gradients one by one.  A contraction's
    backward leaves its factors in the box, under the number of the backward
    pass, and hands on no gradient."""

    @staticmethod
    def forward(ctx, x, box):
        ctx.set_materialize_grads(False)
        ctx.box = box
        return _place_of(x)

    @staticmethod
    def backward(ctx, _):
        parts = ctx.box.pop(torch._C._current_graph_task_id(), [])
        if not parts:
            return None, None
        total = None
        with torch.no_grad():
            for equation, dz, y in parts:
                wide = torch.promote_types(dz.dtype, torch.float32) if len(parts) > 1 else dz.dtype
                dx = _operand_grad(equation, dz.to(wide), y.to(wide))
                total = dx if total is None else total + dx
            total = total.to(parts[0][1].dtype)
        return _Final.of((total, None), [t for _, dz, y in parts for t in (dz, y)])


def _operand_grad(equation, dz, y):
    (ex, ey), ez = equation.split("->")[0].split(","), equation.split("->")[1]
    return contract(f"{ez},{ey}->{ex}", dz, y)


class _Contraction8(torch.autograd.Function):
    """x y with x kept in 8 bits, on torch's own products (the native ones' nodes are in csrc/bindings_saved8.cpp).

    ``x`` carries the values.  Its gradient goes to ``place`` (``x`` is detached
    then): its pre-activation's place in the graph where x is a silu, and with a
    ``box`` the place where its contractions' gradients meet.  Without a place it
    has none.  With ``silu`` the result is silu(x y), its pre-activation in
    8 bits and that one's place."""

    @staticmethod
    def forward(ctx, x, place, box, y, equation, codes, exps, meta, silu):
        ctx.set_materialize_grads(False)
        ctx.equation, ctx.meta, ctx.silu, ctx.box = equation, meta, silu, box
        if not silu:
            ctx.save_for_backward(y, codes, exps)
            return contract(equation, x, y)
        wide = torch.promote_types(x.dtype, torch.float32)
        h = contract(equation, x.to(wide), y.to(wide))
        a, h_codes, h_exps = _silu_forward(_rows(h) if h.dim() else h.view(1, 1), x.dtype)
        a = a.view(h.shape)
        ctx.save_for_backward(y, codes, exps, h_codes, h_exps)
        ctx.mark_non_differentiable(h_codes, h_exps)
        return a, _place_of(a), h_codes, h_exps

    @staticmethod
    def backward(ctx, *grads):
        with torch.no_grad():
            saved = ctx.saved_tensors  # once: a recomputed block's are given out once
            found = _Contraction8.gradients(ctx, saved, *grads)
        return _Final.of(found, (*grads, saved[0]))

    @staticmethod
    def gradients(ctx, saved, grad, grad_pre=None, *_):
        y, codes, exps = saved[:3]
        if grad is not None and ctx.silu:
            grad = _silu_grad(grad, *saved[3:], None)
        if grad_pre is not None:
            grad = grad_pre if grad is None else grad + grad_pre
        if grad is None:
            return (None,) * 9
        want_place, _, want_y = ctx.needs_input_grad[1:4]
        dplace = dy = None
        if ctx.box is not None:
            if torch._C._will_engine_execute_node(ctx.next_functions[1][0]):  # the operand's gradient is asked for
                ctx.box.setdefault(torch._C._current_graph_task_id(), []).append((ctx.equation, grad, y))
        elif want_place:
            dplace = _silu_grad(_operand_grad(ctx.equation, grad, y), codes, exps, ctx.meta[2])
        if want_y:
            (ex, ey), ez = ctx.equation.split("->")[0].split(","), ctx.equation.split("->")[1]
            dy = contract(f"{ez},{ex}->{ey}", grad, _restore_operand(codes, exps, ctx.meta))
        return None, dplace, None, dy, None, None, None, None, None


def _reading(plan, x):
    """What has to be alike for a contraction to read an earlier one's copy: the matrix, the stream, the capture (a
    graph makes the copies that it reads)."""
    return (plan.x_order, plan.gemm[:2], torch.cuda.current_stream(x.device),
            _native.require().capture_of(x.device.index))


def contract_saved(equation, saved, y, activation=None):
    """:func:`contract` with a :class:`Saved8` first operand."""
    x = saved.value
    if activation not in (None, "silu"):
        raise ValueError(f"unsupported activation {activation!r} (supported: 'silu')")
    if y.dtype != x.dtype or y.device != x.device:
        raise ValueError(f"a Saved8 operand of {x.dtype} on {x.device} needs the other one alike, "
                         f"not {y.dtype} on {y.device}")
    saved.check_unchanged()
    y = y.resolve_neg()
    plan = _product(equation, tuple(x.shape), tuple(y.shape))
    silu = activation is not None
    if all(plan.gemm) and gemm.eligible(x, y):
        _native.refuse_tangents("a Saved8 contraction", x, y)
        mod, err = _native.require(), _native.error_word(x.device)
        place = saved._pre
        if place is None and x.requires_grad and torch.is_grad_enabled():
            place = saved._readers
            if place is None:
                place = saved._readers = mod.readers8(x, err)
        order = () if saved._order is None else saved._order
        ready = None
        if saved._ready is not None and saved._ready[0] == _reading(plan, x):
            ready = saved._ready[1]
        out = mod.contract8(x, place, y, plan.on_kernels, saved.codes, saved.exps, saved._act, saved._base, order,
                            silu, err, ready)
        if len(out) > (4 if silu else 1) and saved._version is not None:  # a copy that a change would be told from
            saved._ready = _reading(plan, x), out[-1]
        if not silu:
            return out[0]
        a, pre, codes, exps = out[:4]
        return Saved8(a, codes, exps, True, plan.z_shape, plan.z_order, pre)
    place, box = saved._pre, None
    if place is None and x.requires_grad and torch.is_grad_enabled():
        if saved._box is None:
            box = {}
            saved._box = _Readers.apply(x, box), box
        place, box = saved._box
    out = _Contraction8.apply(x if place is None else x.detach(), place, box, y, plan.equation, saved.codes,
                              saved.exps, saved._meta(), silu)
    if not silu:
        return out
    a, pre, codes, exps = out
    return Saved8(a, codes, exps, True, None, None, pre)


class _SiluSaved(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h):
        wide = torch.promote_types(h.dtype, torch.float32)
        ctx.set_materialize_grads(False)
        h = h.resolve_neg()
        a, codes, exps = _silu_forward((_rows(h) if h.dim() else h.view(1, 1)).to(wide), h.dtype)
        ctx.save_for_backward(codes, exps)
        ctx.mark_non_differentiable(codes, exps)
        return a.view(h.shape), codes, exps

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, *_):
        return None if grad is None else _silu_grad(grad, *ctx.saved_tensors, None)


def silu_saved(h):
    """silu of a tensor whose own value is kept in 8 bits, as a :class:`Saved8`."""
    return Saved8(*_SiluSaved.apply(h), True)
