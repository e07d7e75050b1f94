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

import string

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
        return _native.require().restore8(codes, exps, grad, _CODE[dtype], mode)
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

    __slots__ = ("value", "codes", "exps", "_act", "_base", "_order")

    def __init__(self, value, codes, exps, act=False, base=None, order=None):
        self.value, self.codes, self.exps = value, codes, exps
        self._act = act  # the codes are a pre-activation: the operand is its silu
        self._base = tuple(value.shape) if base is None else base  # shape of the tensor that was quantised
        self._order = order  # permutation from there to the value's axes

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
        return self.codes.numel() + self.exps.numel()

    def restore(self):
        """The operand as backward reads it, in the value's type (no gradient)."""
        return _restore_operand(self.codes, self.exps, self._meta())

    def with_value(self, value):
        """The same codes for a value that differs by its place in the graph alone."""
        return Saved8(value, self.codes, self.exps, self._act, self._base, self._order)

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
    codes, exps = _quantise(_rows(x.detach()))
    return Saved8(x, codes, exps)


# ------------------------------------------------------------------ contractions

def _explicit(equation, x_rank, y_rank):
    """The equation with an ellipsis of the first operand written out."""
    if "..." not in equation:
        return equation
    (ex, ey), ez = equation.split("->")[0].split(","), equation.split("->")[1]
    width = x_rank - len(ex.replace("...", ""))
    if "..." in ey or "..." not in ez or width < 0:
        return None
    free = [c for c in string.ascii_letters if c not in equation][:width]
    fill = "".join(free)
    return f"{ex.replace('...', fill)},{ey}->{ez.replace('...', fill)}"


def _silu_forward(h, dtype):
    """(silu(h) in dtype, codes, exps) of an fp32 (fp64) [rows, d] pre-activation."""
    if h.dtype == torch.float32 and _on_kernels(h, dtype):
        return tuple(_native.require().quant8_silu(h.contiguous(), _CODE[dtype]))
    codes, exps = _quantise(h)
    return (h * torch.sigmoid(h)).to(dtype), codes, exps


def _inverse(order):
    back = [0] * len(order)
    for i, o in enumerate(order):
        back[o] = i
    return back


def _extents(plan):
    return [_product(plan["size"][c] for c in plan[k]) for k in ("batch", "rows", "cols", "red")]


def _product(sizes):
    out = 1
    for s in sizes:
        out *= s
    return out


def _act_layout(plan, x, y):
    """How the pre-activation is kept: (on the native GEMM, shape of the quantised tensor, permutation from its
    axes to the result's).  The native product is quantised as it comes, [batch, rows, cols]."""
    size, ez = plan["size"], plan["ez"]
    if all(_extents(plan)) and gemm.eligible(x, y):
        letters = plan["batch"] + plan["rows"] + plan["cols"]
        return True, tuple(size[c] for c in letters), [letters.index(c) for c in ez]
    return False, tuple(size[c] for c in ez), None


def _product_silu(plan, equation, layout, x, y):
    """(silu of the contraction, codes, exps of its pre-activation)."""
    native, base, order = layout
    if native:
        batch, rows, cols, red = (plan[k] for k in ("batch", "rows", "cols", "red"))
        B, M, N, K = _extents(plan)
        xv = x.permute([plan["ex"].index(c) for c in batch + rows + red]).reshape(B, M, K)
        yv = y.permute([plan["ey"].index(c) for c in batch + red + cols]).reshape(B, K, N)
        h = gemm.native_bmm(xv, yv, out_dtype=torch.float32)
        a, codes, exps = _silu_forward(h.view(B * M, N), x.dtype)
        return a.view(base).permute(order), codes, exps
    wide = torch.promote_types(x.dtype, torch.float32)
    h = contract(equation, x.to(wide), y.to(wide))
    a, codes, exps = _silu_forward(_rows(h) if h.dim() else h.view(1, 1), x.dtype)
    return a.view(base), codes, exps


class _SavedContraction(torch.autograd.Function):
    """x y with x kept in 8 bits; with a ``layout``, silu of it and its pre-activation in 8 bits."""

    @staticmethod
    def forward(ctx, x, y, equation, plan, codes, exps, meta, layout):
        ctx.set_materialize_grads(False)
        ctx.equation, ctx.meta, ctx.layout = equation, meta, layout
        if layout is None:
            ctx.save_for_backward(y, codes, exps)
            return contract(equation, x, y)
        a, h_codes, h_exps = _product_silu(plan, equation, layout, x, y)
        ctx.save_for_backward(y, codes, exps, h_codes, h_exps)
        ctx.mark_non_differentiable(h_codes, h_exps)
        return a, h_codes, h_exps

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, *_):
        if grad is None:
            return (None,) * 8
        y, codes, exps = ctx.saved_tensors[:3]
        if ctx.layout is not None:
            grad = _silu_grad(grad, *ctx.saved_tensors[3:], ctx.layout)
        (ex, ey), ez = ctx.equation.split("->")[0].split(","), ctx.equation.split("->")[1]
        dx = dy = None
        if ctx.needs_input_grad[0]:
            dx = contract(f"{ez},{ey}->{ex}", grad, y)
        if ctx.needs_input_grad[1]:
            x = _restore_operand(codes, exps, ctx.meta)
            own = next((c for c in ey if c not in ex or c not in ez), "")
            # the product's rows are the letters that come first in y: its gradient comes out in y's order
            if own and own in ez:
                dy = contract(f"{ez},{ex}->{ey}", grad, x)
            else:
                dy = contract(f"{ex},{ez}->{ey}", x, grad)
        return dx, dy, None, None, None, None, None, None


def _silu_grad(grad, codes, exps, layout):
    """grad * silu'(h^), in grad's axes."""
    _, _, order = layout
    g = grad if order is None else grad.permute(_inverse(order))
    d = _restored(codes, exps, grad.dtype, _SILU_GRAD, g.reshape(codes.shape).contiguous()).view(g.shape)
    return d if order is None else d.permute(order)


def contract_saved(equation, saved, y, activation=None):
    """:func:`contract` with a :class:`Saved8` first operand."""
    x = saved.value
    if activation not in (None, "silu"):
        raise ValueError(f"unsupported activation {activation!r} (supported: 'silu')")
    if y.dtype != x.dtype or y.device != x.device:
        raise ValueError(f"a Saved8 operand of {x.dtype} on {x.device} needs the other one alike, "
                         f"not {y.dtype} on {y.device}")
    explicit = _explicit(equation, x.dim(), y.dim())
    plan = None if explicit is None else canonical_gemm(explicit, tuple(x.shape), tuple(y.shape))
    if plan is None or plan["x_only"] or plan["y_only"]:
        raise NotImplementedError("a Saved8 operand takes part in plain two-operand contractions only: no repeated, "
                                  "broadcast or summed-out axes")
    layout = None if activation is None else _act_layout(plan, x, y)
    out = _SavedContraction.apply(x, y, explicit, plan, saved.codes, saved.exps, saved._meta(), layout)
    if layout is None:
        return out
    return Saved8(*out, True, *layout[1:])


class _SiluSaved(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h):
        wide = torch.promote_types(h.dtype, torch.float32)
        ctx.set_materialize_grads(False)
        a, codes, exps = _silu_forward((_rows(h) if h.dim() else h.view(1, 1)).to(wide), h.dtype)
        ctx.save_for_backward(codes, exps)
        ctx.mark_non_differentiable(codes, exps)
        return a.view(h.shape), codes, exps

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, *_):
        return None if grad is None else _silu_grad(grad, *ctx.saved_tensors, (False, None, None))


def silu_saved(h):
    """silu of a tensor whose own value is kept in 8 bits, as a :class:`Saved8`."""
    return Saved8(*_SiluSaved.apply(h), True)
