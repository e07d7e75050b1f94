"""Activations kept for backward in 8 bits (checkpoint8, Saved8 operands of einshard).

The oracle quantises in 64 bits.  Codes must be equal, not close: every scaling
is by a power of two.  Products are compared within the roundings of their
output (half a step of the type), of the 16-bit intermediates (half a step of
each factor, carried through the product of absolute values) and of the 32-bit
accumulation (2^-23 a term at most, which the same product bounds).
"""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
import torch.distributed as dist
import torch.utils.checkpoint
from dist_harness import run_ranks

import torch_einshard_b200 as es
from torch_einshard_b200.models.tp_mlp import TPMLP
from torch_einshard_b200.models.transformer import TPTransformer, TransformerConfig
from torch_einshard_b200.ops.saved8 import silu_saved

cuda = pytest.param("cuda", marks=pytest.mark.gpu)
DEVICES = ["cpu", cuda]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def oracle(x):
    """(restored values in fp64, half steps) of x by the definition, block by block."""
    x = x.detach().double().cpu()
    flat = x.reshape(x.shape[:-1].numel(), x.shape[-1])
    out, half = torch.zeros_like(flat), torch.zeros_like(flat)
    for start in range(0, flat.shape[1], 32):
        block = flat[:, start:start + 32]
        amax = block.abs().amax(1)
        bad = ~torch.isfinite(amax)
        amax = torch.where(bad, 1.0, amax)
        e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -1000))) - 6  # exact in 64 bits away from powers of two
        e = torch.where(torch.exp2(e + 7) <= amax, e + 1, e)
        e = torch.where(torch.exp2(e + 6) > amax, e - 1, e).clamp(min=-126)
        e = torch.where(torch.round(amax / torch.exp2(e)) > 127, e + 1, e)
        step = torch.exp2(e)[:, None]
        q = torch.round(block / step) * step
        out[:, start:start + 32] = torch.where(bad[:, None], float("nan"), q)
        half[:, start:start + 32] = step / 2
    return out.reshape(x.shape), half.reshape(x.shape)


def check_restore(x):
    got = es.checkpoint8(x).restore()
    assert got.dtype == x.dtype and got.shape == x.shape and not got.requires_grad
    limit = torch.finfo(x.dtype).max
    want = oracle(x)[0]
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.cpu().double()), torch.nan_to_num(want.clamp(-limit, limit)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (32,), (33,), (1, 1), (3, 31), (2, 3, 64), (5, 40), (4, 1000), (2, 1001),
                                   (1, 8200), (300, 96), (0, 64), (5, 0)])
def test_restore_is_the_definition(device, dtype, shape):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(shape, generator=gen) * torch.exp(3 * torch.randn(shape, generator=gen))
    check_restore(x.to(dtype).to(device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [32, 50, 96])
def test_special_values(device, dtype, width):
    info = torch.finfo(dtype)
    x = torch.zeros(12, width, dtype=dtype)
    x[1, 3] = info.max
    x[2] = info.max
    x[3, :] = -info.max
    x[4, 0] = float("inf")
    x[5, width - 1] = float("nan")
    x[6, 1] = -float("inf")
    x[7] = info.smallest_normal
    x[8, 2] = info.smallest_normal * info.eps  # the smallest subnormal
    x[9, :2] = torch.tensor([1.0, 0.5])  # a tie: 63.5 steps would round either way under a scale of max / 127
    x[10] = 127.5 / 64
    x[11, 0] = -0.0
    check_restore(x.to(device))


@pytest.mark.parametrize("device", DEVICES)
def test_error_is_half_a_step(device):
    x = torch.randn(64, 257, generator=torch.Generator().manual_seed(1)).to(device)
    s = es.checkpoint8(x)
    _, half = oracle(x)
    assert ((s.restore() - x).abs().cpu().double() <= half).all()
    assert s.nbytes == 64 * 257 + 64 * 9


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [3, 7, 9, 15, 31, 33, 39, 65, 511, 513, 2047, 2048, 2049, 4001, 8127, 8191, 8195])
def test_rows_without_alignment(dtype, width):
    """Every start of a row inside a 16-byte word, in the values, the codes and the result."""
    gen = torch.Generator().manual_seed(width)
    base = (torch.randn(21 * width + 16, generator=gen) * 3).to(dtype).cuda()
    for off in (0, 1, 2, 3, 5, 7):
        check_restore(base[off:off + 19 * width].view(19, width))
    x = base[1:1 + 9 * width].view(9, width).clone()
    x[3, width // 2] = float("nan")
    x[5, 0] = float("inf")
    x[8, width - 1] = -float("inf")
    check_restore(x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(5003, 9), (3001, 33), (1999, 65), (701, 301), (67, 8191), (3, 40001)])
def test_blocks_across_tiles(dtype, rows, width):
    """Rows of odd widths over many blocks of the grid, and the gradient of a SiLU kept with them."""
    gen = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, width, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen))).to(dtype)
    check_restore(x.cuda())


@pytest.mark.parametrize("device", DEVICES)
def test_views_and_alignments(device):
    base = torch.randn(6, 130, 70, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(device)
    check_restore(base.transpose(1, 2))
    check_restore(base[:, 1:, 3:67])
    check_restore(base.flatten()[1:1 + 64 * 64].view(64, 64))
    check_restore(base[:, :, :1].expand(6, 130, 40))


def _case(device, dtype, b, s, c, h, seed=0):
    gen = torch.Generator().manual_seed(seed)
    def make(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen) * scale).to(dtype).to(device)
    return make(b, s, c), make(h, c, scale=c ** -0.5), make(c, h, scale=h ** -0.5), make(b, s, c), make(b, s, h)


def close(got, want, slack, dtype, terms):
    """|got - want| within the output's rounding, `terms` half steps of 16-bit factors and the accumulation."""
    bound = half_step(dtype) * want.abs() + (terms * half_step(dtype) + 2.0 ** -20) * 1.01 * slack
    bound = bound + torch.finfo(dtype).smallest_normal
    err = (got.detach().double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


SHAPES = [(1, 1, 32, 8), (2, 5, 40, 48), (3, 33, 100, 72), (1, 7, 33, 31), (2, 130, 256, 520)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("transposed", [False, True])
def test_linear(device, dtype, shape, transposed):
    x, w, _, _, dz = _case(device, dtype, *shape)
    if transposed:
        w = w.t().contiguous()
    x.requires_grad_(True)
    w.requires_grad_(True)
    s = es.checkpoint8(x)
    z = es.einshard("b s c, c h -> b s h" if transposed else "b s c, h c -> b s h", s, w)
    dx, dw = torch.autograd.grad(z, (x, w), dz)
    xd, zd = x.detach().double().cpu(), dz.double().cpu()
    wd = (w.t() if transposed else w).detach().double().cpu()
    kept = s.restore().double().cpu()
    close(z, xd @ wd.t(), xd.abs() @ wd.abs().t(), dtype, 0)
    close(dx, zd @ wd, zd.abs() @ wd.abs(), dtype, 0)
    want = torch.einsum("bsh,bsc->hc", zd, kept)
    slack = torch.einsum("bsh,bsc->hc", zd.abs(), kept.abs())
    close(dw.t() if transposed else dw, want, slack, dtype, 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("transposed", [False, True])
def test_mlp(device, dtype, shape, transposed):
    check_mlp(device, dtype, shape, transposed)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("shape", [(2, 2500, 128, 2048), (1, 5003, 200, 1040), (3, 1111, 72, 4112), (1, 4736, 64, 256),
                                   (1, 2400, 96, 1000), (1, 2400, 96, 1032)])
def test_mlp_in_the_product(dtype, transposed, shape):
    """Shapes whose pre-activation is quantised, and whose gradient takes silu', in the products' epilogues (16-byte
    rows of codes; the last two are not), with ragged edges."""
    check_mlp("cuda", dtype, shape, transposed)


def check_mlp(device, dtype, shape, transposed):
    x, w1, w2, dy, _ = _case(device, dtype, *shape, seed=5)
    if transposed:
        w1, w2 = w1.t().contiguous(), w2.t().contiguous()
    for t in (x, w1, w2):
        t.requires_grad_(True)
    s = es.checkpoint8(x)
    a = es.einshard("b s c, c h -> b s h" if transposed else "b s c, h c -> b s h", s, w1, activation="silu")
    assert isinstance(a, es.Saved8) and a.value.dtype == dtype
    y = es.einshard("b s h, h c -> b s c" if transposed else "b s h, c h -> b s c", a, w2)
    dx, dw1, dw2 = torch.autograd.grad(y, (x, w1, w2), dy)
    if transposed:
        w1, w2, dw1, dw2 = w1.t(), w2.t(), dw1.t(), dw2.t()

    xd, w1d, w2d, dyd = (t.detach().double().cpu() for t in (x, w1, w2, dy))
    pre = xd @ w1d.t()
    codes = a.codes.cpu().double().view(*pre.shape)
    step = torch.exp2(a.exps.cpu().double().repeat_interleave(32, 1)[:, :pre.shape[-1]] - 127).view(*pre.shape)
    kept = codes * step
    # the pre-activation is kept from the 32-bit product: half a step off, and the accumulation
    assert ((kept - pre).abs() <= step / 2 + 2.0 ** -20 * (xd.abs() @ w1d.abs().t())).all()
    act = pre * torch.sigmoid(pre)
    # the sigmoid's own error is below 2^-20 of the value; |d silu| <= 1.1 |d pre|
    close(a.value, act, act.abs() + xd.abs() @ w1d.abs().t(), dtype, 0)
    close(y, a.value.detach().double().cpu() @ w2d.t(), act.abs() @ w2d.abs().t() * 1.1 + 1e-6, dtype, 0)
    sig = torch.sigmoid(kept)
    akept = kept * sig
    assert torch.allclose(a.restore().double().cpu(), akept, rtol=half_step(dtype) + 2.0 ** -20, atol=1e-7)
    close(dw2, torch.einsum("bsc,bsh->ch", dyd, akept), torch.einsum("bsc,bsh->ch", dyd.abs(), akept.abs()), dtype, 1)
    da, da_abs = dyd @ w2d, dyd.abs() @ w2d.abs()
    slope = sig * (1 + kept * (1 - sig))
    dh = da * slope
    # da is rounded to the type, its product with silu' once more; the accumulation's part goes by da_abs
    dh_err = dh.abs() * 2.01 + da_abs * slope.abs() * 2.0 ** -20 / half_step(dtype) + 1e-9
    close(dx, dh @ w1d, (dh_err + dh.abs() * 2.0 ** -6) @ w1d.abs(), dtype, 1)
    xk = s.restore().double().cpu()
    close(dw1, torch.einsum("bsh,bsc->hc", dh, xk), torch.einsum("bsh,bsc->hc", dh_err + dh.abs() * 2.0 ** -6, xk.abs()),
          dtype, 1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("odd", [0, 5])
def test_slope_of_large_pre_activations(device, dtype, odd):
    """silu' far from 0 is 1 or 0: 1 - sigmoid has no error of its own there that x could multiply.  Blocks with large
    values at their ends beside blocks of small ones; the gradient is one product with 1 (and zeros), rounded to the
    type once or, behind the second product, twice."""
    gen = torch.Generator().manual_seed(17)
    sizes = [3.0, 12.0, 40.0, 300.0, 5e3, 2.0 ** 15] + ([1e6, 1e12, 1e30] if dtype != torch.float16 else [])
    values = torch.tensor([s * sign for s in sizes for sign in (1, -1)], dtype=torch.float64)
    width = 64 * len(values) + odd
    x = torch.randn(8, width, generator=gen).double()
    for i, v in enumerate(values):
        x[:, 64 * i:64 * i + 32] *= 0.004 * v.abs()
        x[:, 64 * i] = x[:, 64 * i + 31] = v
    x = x.to(dtype).to(device).requires_grad_(True)
    w = torch.eye(width, dtype=dtype, device=device)
    a = es.einshard("b c, h c -> b h", es.checkpoint8(x), w, activation="silu")
    y = es.einshard("b h, c h -> b c", a, w)
    kept = a.codes.double().cpu() * torch.exp2(a.exps.cpu().double().repeat_interleave(32, 1)[:, :width] - 127)
    s, rest = torch.sigmoid(kept), torch.sigmoid(-kept)
    want = s * (1 + kept * rest)
    for out in (a.value, y):
        (dx,) = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
        # the sigmoid and what is left of 1 are each off by 2^-20 of themselves; 16-bit results take what is below -43
        # as -43, where |silu'| < 42 e^-43 < 1e-17
        bound = 2.01 * half_step(dtype) * want.abs() + 2.0 ** -20 * s * (1 + kept.abs() * rest) + 1e-17
        assert ((dx.double().cpu() - want).abs() <= bound + torch.finfo(dtype).smallest_normal).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [40, 64])
def test_pre_activations_of_the_largest_value(device, width):
    """bf16's largest value is kept as 64 steps of 2^122, which is past 32 bits: it reads back as the largest 32-bit value,
    where silu' is 1 (and 0 on the other side)."""
    top = torch.finfo(torch.bfloat16).max
    x = torch.zeros(2, 3, width, dtype=torch.bfloat16, device=device)
    x[0, 0, 1], x[0, 1, 2], x[1, 2, 5] = top, -top, top / 2
    x.requires_grad_(True)
    w = torch.eye(width, dtype=torch.bfloat16, device=device)
    a = es.einshard("b s c, h c -> b s h", es.checkpoint8(x), w, activation="silu")
    y = es.einshard("b s h, c h -> b s c", a, w)
    for out in (a.value, y):  # through both forms of the gradient
        (dx,) = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
        want = torch.full(x.shape, 0.5, device=device)
        want[0, 0, 1], want[0, 1, 2], want[1, 2, 5] = 1, 0, 1
        assert ((dx.float() - want).abs() <= half_step(x.dtype)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_against_differences(device):
    """Where x is on the grid of its blocks, x^ = x and gradients are those of the product: central differences of
    a bilinear form have no error but rounding (64 bits on the CPU, whole numbers on the GPU)."""
    dtype = torch.float64 if device == "cpu" else torch.float32
    gen = torch.Generator().manual_seed(4)
    x = torch.randint(-60, 61, (2, 3, 8), generator=gen).to(dtype).to(device).requires_grad_(True)
    w = torch.randint(-4, 5, (5, 8), generator=gen).to(dtype).to(device).requires_grad_(True)
    g = torch.randint(-4, 5, (2, 3, 5), generator=gen).to(dtype).to(device)

    def f(xv, wv):
        return (es.einshard("b s c, h c -> b s h", es.checkpoint8(xv), wv) * g).sum()

    dx, dw = torch.autograd.grad(f(x, w), (x, w))
    for t, grad, which in ((x, dx, 0), (w, dw, 1)):
        flat = t.detach().flatten()
        for i in range(0, flat.numel(), 3):
            hi, lo = flat.clone(), flat.clone()
            hi[i] += 1
            lo[i] -= 1
            args = [[x.detach(), w.detach()] for _ in range(2)]
            args[0][which], args[1][which] = hi.view(t.shape), lo.view(t.shape)
            assert float(grad.flatten()[i]) == float((f(*args[0]) - f(*args[1])) / 2)


def negated(t):
    """-t as a view that only says so (what the imaginary part of a conjugate is)."""
    return torch._neg_view(t.detach())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [40, 37])
def test_negated_views(device, dtype, width):
    """Operands and gradients whose sign is kept beside their memory."""
    x, w1, w2, dy, da = _case(device, dtype, 2, 6, width, 48, seed=16)
    results = []
    for sign in (torch.neg, negated):
        u = [sign(-t).detach().requires_grad_(True) for t in (x, w1, w2)]
        kept = es.checkpoint8(u[0])
        a = es.einshard("b s c, h c -> b s h", kept, u[1], activation="silu")
        y = es.einshard("b s h, c h -> b s c", a, u[2])
        z = es.einshard("b s c, h c -> b s h", kept, u[1])
        s = silu_saved(z)
        grads = torch.autograd.grad((y, z, a.value, s.value), u, tuple(sign(t) for t in (dy, da, da, da)))
        results.append([kept.restore(), y.detach(), z.detach(), s.value.detach(), s.restore(), *grads,
                        silu_saved(sign(da)).value])
    for got, want in zip(*results):
        assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_axis_orders_and_ellipsis(device):
    x, w, _, _, _ = _case(device, torch.float32, 2, 6, 40, 48, seed=7)
    x.requires_grad_(True)
    w.requires_grad_(True)
    s = es.checkpoint8(x)
    kept = s.restore().double().cpu()
    wd = w.detach().double().cpu()
    for formula, fn, batched in [
        ("b s c, h c -> h b s", lambda a, b: torch.einsum("bsc,hc->hbs", a, b), False),
        ("b s c, h c -> s h b", lambda a, b: torch.einsum("bsc,hc->shb", a, b), False),
        ("... c, h c -> ... h", lambda a, b: torch.einsum("bsc,hc->bsh", a, b), False),
    ]:
        z = es.einshard(formula, s, w)
        dz = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).to(device)
        (dw,) = torch.autograd.grad(z, w, dz)
        wr = wd.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(fn(kept, wr), wr, dz.double().cpu())
        assert torch.allclose(dw.double().cpu(), want, rtol=1e-5, atol=1e-5)
        a = es.einshard(formula, s, w, activation="silu")
        assert a.restore().shape == a.value.shape
        assert torch.allclose(a.restore(), a.value, atol=0.05)
        (dw,) = torch.autograd.grad(a.value, w, dz)
        pre = fn(x.detach().double().cpu(), wr)
        (want,) = torch.autograd.grad(torch.nn.functional.silu(pre), wr, dz.double().cpu())
        assert (dw.double().cpu() - want).norm() <= 0.02 * want.norm()  # 8-bit x and pre-activation: steps of 1/64


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["b s h", "h b s", "s h b"])
def test_activation_layouts_16_bit(order):
    x, w, _, _, _ = _case("cuda", torch.bfloat16, 2, 6, 40, 48, seed=8)
    w.requires_grad_(True)
    a = es.einshard(f"b s c, h c -> {order}", es.checkpoint8(x), w, activation="silu")
    pre = torch.einsum(f"bsc,hc->{order.replace(' ', '')}", x.double(), w.detach().double())
    want = pre * torch.sigmoid(pre)
    assert ((a.value.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()
    dz = torch.randn_like(a.value)
    (dw,) = torch.autograd.grad(a.value, w, dz)
    sig = torch.sigmoid(pre)
    dh = dz.double() * sig * (1 + pre * (1 - sig))
    want = torch.einsum(f"{order.replace(' ', '')},bsc->hc", dh, x.double())
    assert (dw.double() - want).norm() <= 0.02 * want.norm()


def same_value(got, want):
    """Two values of silu in one type: each within half a step of the exact one, and 2^-20 of it from the sigmoid."""
    far = (torch.finfo(got.dtype).eps + 2.0 ** -19) * want.double().abs() + torch.finfo(got.dtype).smallest_normal
    return bool(((got.double() - want.double()).abs() <= far).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 40, 37])
def test_nan_columns_stay_in_their_column(device, dtype, width):
    """A NaN row of the weight is a NaN column of the activation: its neighbours keep their values, whatever they are."""
    x, w, _, _, _ = _case(device, dtype, 2, 9, 48, width, seed=12)
    w[1] = 0
    w[4] *= 100
    clean = es.einshard("b s c, h c -> b s h", es.checkpoint8(x), w, activation="silu").value
    bad = [0, 5, 6, 33]
    w[bad[:2]] = float("nan")
    w[bad[2:], 3] = float("nan")
    got = es.einshard("b s c, h c -> b s h", es.checkpoint8(x), w, activation="silu").value
    fine = [i for i in range(width) if i not in bad]
    assert torch.isnan(got[..., bad]).all() and same_value(got[..., fine], clean[..., fine])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 40, 37, 5])
def test_nan_values_stay_in_their_place(device, dtype, width):
    """The same for the activation of a pre-activation in memory (where a plan's last step is not the product)."""
    h = (3 * torch.randn(4, 6, width, generator=torch.Generator().manual_seed(13))).to(dtype).to(device)
    clean = silu_saved(h).value
    bad = torch.zeros(h.shape, dtype=torch.bool, device=device)
    bad.flatten()[1::7] = True
    got = silu_saved(torch.where(bad, float("nan"), h)).value
    assert torch.isnan(got[bad]).all() and same_value(got[~bad], clean[~bad])
    up = torch.where(bad, float("inf"), h)
    assert same_value(silu_saved(up).value[~bad], clean[~bad]) and torch.isinf(silu_saved(up).value[bad]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.randn(2, 3, 8, device=device)
    w = torch.randn(5, 8, device=device)
    s = es.checkpoint8(x)
    with pytest.raises(TypeError):
        es.checkpoint8(s)
    with pytest.raises(TypeError):
        es.checkpoint8([1.0])
    with pytest.raises(TypeError):
        es.checkpoint8(torch.ones(4, dtype=torch.int64, device=device))
    with pytest.raises(TypeError):
        es.checkpoint8(torch.ones(4, dtype=torch.complex64, device=device))
    with pytest.raises(ValueError):
        es.checkpoint8(torch.tensor(1.0, device=device))
    with pytest.raises(TypeError, match="goes first"):
        es.einshard("h c, b s c -> b s h", w, s)
    with pytest.raises(TypeError, match="second operand"):
        es.einshard("b s c -> b c s", s)
    with pytest.raises(ValueError, match="alike"):
        es.einshard("b s c, h c -> b s h", s, w.double())
    with pytest.raises(ValueError, match="activation"):
        es.einshard("b s c, h c -> b s h", s, w, activation="gelu")
    with pytest.raises(NotImplementedError):
        es.einshard("b s c, h -> b h", s, w[:, 0])  # s and c summed out
    with pytest.raises(NotImplementedError):
        es.einshard("b s (c k), h c k -> b s h", s, torch.randn(5, 4, 2, device=device), sizes={"k": 2})
    with pytest.raises(RuntimeError):  # no second derivative through rounded codes
        xg = x.clone().requires_grad_(True)
        z = es.einshard("b s c, h c -> b s h", es.checkpoint8(xg), w).square().sum()
        (dx,) = torch.autograd.grad(z, xg, create_graph=True)
        torch.autograd.grad(dx.sum(), xg)


@pytest.mark.parametrize("device", DEVICES)
def test_activation_used_twice(device):
    """The activation's value, and two products that read it, send their gradients to one pre-activation."""
    x, w1, w2, dy, da = _case(device, torch.float32, 2, 6, 40, 48, seed=11)
    w1.requires_grad_(True)
    a = es.einshard("b s c, h c -> b s h", es.checkpoint8(x), w1, activation="silu")
    y1 = es.einshard("b s h, c h -> b s c", a, w2)
    y2 = es.einshard("b s h, c h -> s b c", a, 2 * w2)
    parts = [torch.autograd.grad(y1, w1, dy, retain_graph=True)[0],
             torch.autograd.grad(y2, w1, dy.transpose(0, 1), retain_graph=True)[0],
             torch.autograd.grad(a.value, w1, da, retain_graph=True)[0]]
    (both,) = torch.autograd.grad((y1, y2, a.value), w1, (dy, dy.transpose(0, 1), da))
    assert torch.allclose(both, sum(parts), rtol=1e-4, atol=1e-4)
    assert torch.allclose(parts[1], 2 * parts[0], rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
def test_capture_and_replay():
    x, w1, w2, dy, _ = _case("cuda", torch.bfloat16, 2, 64, 64, 96, seed=9)

    def step():
        s = es.checkpoint8(x)
        a = es.einshard("b s c, h c -> b s h", s, w1, activation="silu")
        return es.einshard("b s h, c h -> b s c", a, w2), a.restore()

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, kept = step()
    x.copy_(torch.randn_like(x))
    graph.replay()
    want_y, want_kept = step()
    assert torch.equal(y, want_y) and torch.equal(kept, want_kept)


@pytest.fixture
def one_rank_mesh(request):
    from torch.distributed.device_mesh import init_device_mesh
    device = request.param
    if not dist.is_initialized():
        dist.init_process_group("gloo" if device == "cpu" else "nccl", init_method="tcp://127.0.0.1:0", rank=0,
                                world_size=1)
    yield device, init_device_mesh(device, (1,), mesh_dim_names=("tp",))
    dist.destroy_process_group()


@pytest.mark.parametrize("one_rank_mesh", DEVICES, indirect=True)
def test_models_keep_their_outputs_and_gradients(one_rank_mesh):
    """The forward pass does not change; gradients are those of activations within half a step."""
    device, mesh = one_rank_mesh
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    models = [TPMLP(64, 256, mesh, dtype=dtype, device=device, std=0.1, checkpoint=c) for c in (None, "int8")]
    x = torch.randn(2, 32, 64, generator=torch.Generator().manual_seed(0)).to(device, dtype)
    outs = [m(x) for m in models]
    assert (outs[0] - outs[1]).abs().max() <= 4 * half_step(dtype) * outs[0].abs().max()
    for m, y in zip(models, outs):
        y.float().square().sum().backward()
    for p, q in zip(models[0].parameters(), models[1].parameters()):
        assert (p.grad.float() - q.grad.float()).norm() <= 0.03 * p.grad.float().norm()

    cfg = TransformerConfig(layers=2, d=64, heads=4, mlp=128, vocab=97, seq=16, dtype=dtype)
    tokens = torch.randint(0, 97, (2, 16), generator=torch.Generator().manual_seed(1)).to(device)
    losses, grads = [], []
    for mode in (False, "int8"):
        model = TPTransformer(cfg, mesh, device=device, checkpoint=mode)
        loss = model(tokens, tokens.roll(-1, 1))
        loss.backward()
        losses.append(float(loss))
        grads.append([p.grad.float() for p in model.parameters()])
    assert abs(losses[0] - losses[1]) <= (1e-5 if device == "cpu" else 0.02) * abs(losses[0])
    for p, q in zip(*grads):
        assert (p - q).norm() <= 0.05 * p.norm() + 1e-6
    with pytest.raises(ValueError):
        TPMLP(64, 256, mesh, dtype=dtype, device=device, checkpoint="int4")


# ------------------------------------------------------------------ one operand, several contractions

def shared_case(dtype, device, shape, outs, gen):
    """x [b, s, c], weights and gradients of ``outs`` projections of different widths, and dx in 64 bits."""
    b, s, c = shape
    widths = [max(8, c // (i + 1)) for i in range(outs)]
    x = torch.randn(shape, generator=gen).to(dtype).to(device).requires_grad_(True)
    w = [(torch.randn(n, c, generator=gen) / c ** 0.5).to(dtype).to(device).requires_grad_(True) for n in widths]
    dy = [torch.randn(b, s, n, generator=gen).to(dtype).to(device) for n in widths]
    with torch.no_grad():
        want = sum(d.double() @ v.double() for d, v in zip(dy, w))
        size = sum(d.double().abs() @ v.double().abs() for d, v in zip(dy, w))
    return x, w, dy, want, size


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,outs", [((2, 5, 24), 2), ((1, 300, 136), 3), ((3, 64, 129), 4), ((2, 33, 256), 6),
                                        ((1, 1, 64), 3), ((1, 1024, 512), 3), ((1, 700, 615), 3), ((2, 3, 7), 2)])
def test_shared_operand_is_rounded_once(device, dtype, shape, outs):
    """dx = sum_i dz_i w_i: half a step of the result, and for the 32-bit sums 2^-22 of the sum of absolute values.

    An fp32 product is a library's: K products and additions one after the other, each off by at most 2^-24 of a
    partial sum, which the sum of absolute values bounds, so (K + 1) 2^-24 of it."""
    x, w, dy, want, size = shared_case(dtype, device, shape, outs, torch.Generator().manual_seed(outs))
    kept = es.checkpoint8(x)
    ys = [es.einshard("b s c, n c -> b s n", kept, v) for v in w]
    assert all(y.is_contiguous() for y in ys)
    for y, v in zip(ys, w):
        exact = x.detach().double() @ v.detach().double().t()
        sums = (x.shape[-1] + 1) * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -22
        bound = half_step(dtype) * exact.abs() + sums * (x.detach().double().abs() @ v.detach().double().abs().t())
        assert ((y.detach().double() - exact).abs() <= bound + torch.finfo(dtype).tiny).all()
    dx = torch.autograd.grad(ys, x, dy, retain_graph=True)[0]
    terms = sum(v.shape[0] for v in w)
    sums = (terms + 1) * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -22
    allowed = half_step(dtype) * want.abs() + size * sums + torch.finfo(dtype).tiny
    assert ((dx.double() - want).abs() <= allowed).all()
    # again, a part of them, and the weights alone: nothing is left over from one pass to the next
    assert torch.equal(dx, torch.autograd.grad(ys, x, dy, retain_graph=True)[0])
    dw = torch.autograd.grad(ys, w, dy, retain_graph=True)
    one = torch.autograd.grad(ys[1], x, dy[1], retain_graph=True)[0]
    want1 = dy[1].double() @ w[1].double()
    size1 = dy[1].double().abs() @ w[1].double().abs()
    assert ((one.double() - want1).abs() <= half_step(dtype) * want1.abs() + size1 * sums + torch.finfo(dtype).tiny).all()
    both = torch.autograd.grad(ys, [x, *w], dy)
    assert torch.equal(both[0], dx) and all(torch.equal(a, b) for a, b in zip(both[1:], dw))


@pytest.mark.parametrize("device", DEVICES)
def test_shared_operand_in_different_equations(device):
    """Gradients meet in the operand's axes, whatever the contractions' layouts."""
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(2, 16, 4, 32, generator=gen).to(torch.bfloat16).to(device).requires_grad_(True)
    w = torch.randn(4, 32, 24, generator=gen).to(torch.bfloat16).to(device)
    v = torch.randn(32, 8, generator=gen).to(torch.bfloat16).to(device)
    kept = es.checkpoint8(x)
    a = es.einshard("b s h d, h d n -> b s n", kept, w)
    b = es.einshard("b s h d, d n -> b h s n", kept, v)
    c = es.einshard("b s h d, h d n -> n b s", kept, w)
    ga, gb, gc = (torch.randn(t.shape, generator=gen).to(torch.bfloat16).to(device) for t in (a, b, c))
    dx = torch.autograd.grad([a, b, c], x, [ga, gb, gc])[0]
    d = [t.double() for t in (ga, gb, gc, w, v)]
    want = [torch.einsum("bsn,hdn->bshd", d[0], d[3]), torch.einsum("bhsn,dn->bshd", d[1], d[4]),
            torch.einsum("nbs,hdn->bshd", d[2], d[3])]
    size = sum(torch.einsum(e, p.abs(), q.abs()) for e, p, q in (
        ("bsn,hdn->bshd", d[0], d[3]), ("bhsn,dn->bshd", d[1], d[4]), ("nbs,hdn->bshd", d[2], d[3])))
    # at most two groups are rounded by themselves before they are added
    allowed = half_step(x.dtype) * (2 * (want[0] + want[2]).abs() + 2 * want[1].abs() + sum(want).abs()) + size * 2.0 ** -22
    assert ((dx.double() - sum(want)).abs() <= allowed).all()


@pytest.mark.gpu
def test_shared_operand_on_two_streams():
    """The same bits as on one stream."""
    x, w, dy, _, _ = shared_case(torch.bfloat16, "cuda", (4, 512, 512), 3, torch.Generator().manual_seed(4))

    def contractions(stream):
        kept = es.checkpoint8(x)
        ys = [es.einshard("b s c, n c -> b s n", kept, w[0])]
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ys.append(es.einshard("b s c, n c -> b s n", kept, w[1], activation="silu").value)
            ys.append(es.einshard("b s c, n c -> b s n", kept, w[2]))
        torch.cuda.current_stream().wait_stream(stream)
        return ys

    ys, alone = contractions(torch.cuda.Stream()), contractions(torch.cuda.current_stream())
    want = torch.autograd.grad(alone, x, dy)[0]
    for _ in range(4):
        assert torch.equal(torch.autograd.grad(ys, x, dy, retain_graph=True)[0], want)


@pytest.mark.gpu
def test_shared_operand_captured():
    x, w, dy, want, size = shared_case(torch.bfloat16, "cuda", (2, 128, 256), 3, torch.Generator().manual_seed(5))

    def step():
        kept = es.checkpoint8(x)
        ys = [es.einshard("b s c, n c -> b s n", kept, v) for v in w]
        return torch.autograd.grad(ys, [x, *w], dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.mul_(0.5)
        dy[0].mul_(2)
    graph.replay()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_copies_stay_on_their_stream():
    """An odd width is read from a copy: a contraction on another stream does not take one that is still being made."""
    gen = torch.Generator().manual_seed(8)
    x, w, dy, _, _ = shared_case(torch.bfloat16, "cuda", (8, 1024, 1021), 2, gen)
    want = [es.einshard("b s c, n c -> b s n", es.checkpoint8(x), v) for v in w]
    side = torch.cuda.Stream()
    for _ in range(4):
        kept = es.checkpoint8(x)
        torch.cuda.synchronize()
        first = es.einshard("b s c, n c -> b s n", kept, w[0])
        with torch.cuda.stream(side):
            second = es.einshard("b s c, n c -> b s n", kept, w[1])
        torch.cuda.synchronize()
        assert torch.equal(first, want[0]) and torch.equal(second, want[1])


@pytest.mark.gpu
def test_kept_operand_in_two_graphs():
    """An odd width is read from a copy: each graph makes its own, so they may be replayed in any order."""
    gen = torch.Generator().manual_seed(14)
    x, w, _, _, _ = shared_case(torch.bfloat16, "cuda", (2, 64, 127), 3, gen)
    other = torch.randn(x.shape, generator=gen).to(x)
    side = torch.cuda.Stream()
    with torch.no_grad():
        kept = es.checkpoint8(x)
        for v in w:
            es.einshard("b s c, n c -> b s n", es.checkpoint8(x), v)
        torch.cuda.synchronize()
        graphs, outs = [], []
        for v in w:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                outs.append(es.einshard("b s c, n c -> b s n", kept, v))
        want = [es.einshard("b s c, n c -> b s n", es.checkpoint8(other), v) for v in w]
        x.copy_(other)
        for i in (2, 1, 0):
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [64, 37])
def test_inside_a_recomputed_block(device, width):
    x, w, dy, _, _ = shared_case(torch.bfloat16, device, (2, 16, width), 2, torch.Generator().manual_seed(10))

    def block(x, *w):
        kept = es.checkpoint8(x)
        a = es.einshard("b s c, n c -> b s n", kept, w[0], activation="silu")
        return es.einshard("b s n, n c -> b s c", a, w[0]), es.einshard("b s c, n c -> b s n", kept, w[1])

    dz = [torch.randn(2, 16, width, generator=torch.Generator().manual_seed(11)).to(x), dy[1]]
    plain = torch.autograd.grad(block(x, *w), [x, *w], dz)
    again = torch.utils.checkpoint.checkpoint(block, x, *w, use_reentrant=False)
    for g, h in zip(plain, torch.autograd.grad(again, [x, *w], dz)):
        assert torch.equal(g, h)


@pytest.mark.parametrize("device", DEVICES)
def test_second_derivatives_are_refused(device):
    x, w, dy, _, _ = shared_case(torch.bfloat16, device, (2, 16, 32), 2, torch.Generator().manual_seed(6))
    for activation in (None, "silu"):
        kept = es.checkpoint8(x)
        ys = [es.einshard("b s c, n c -> b s n", kept, v, activation=activation) for v in w]
        ys = [y.value if activation else y for y in ys]
        dx, dw = torch.autograd.grad(ys, [x, w[0]], dy, create_graph=True)
        for g in (dx, dw):
            with pytest.raises(RuntimeError):
                torch.autograd.grad((g + 0 * w[0].sum()).sum(), w[0], retain_graph=True)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["x", "w"])
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(device, which, activation, grad):
    x, w, _, _, _ = _case(device, torch.bfloat16, 2, 5, 40, 48)
    x.requires_grad_(grad)
    with forward_ad.dual_level():
        if which == "x":
            x = forward_ad.make_dual(x, torch.ones_like(x))
        else:
            w = forward_ad.make_dual(w, torch.ones_like(w))
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|forward mode|forward AD"):
            es.einshard("b s c, h c -> b s h", es.checkpoint8(x), w, activation=activation)


@pytest.mark.parametrize("device", DEVICES)
def test_operands_changed_in_place(device):
    x, w, dy, _, _ = shared_case(torch.bfloat16, device, (2, 16, 32), 1, torch.Generator().manual_seed(7))
    h = x * 1
    kept = es.checkpoint8(h)
    y = es.einshard("b s c, n c -> b s n", kept, w[0])
    h.add_(1)  # the product is done, the codes are their own
    torch.autograd.grad(y, x, dy[0], retain_graph=True)
    with pytest.raises(RuntimeError):
        es.einshard("b s c, n c -> b s n", kept, w[0])  # its value is no longer what the codes stand for
    with torch.no_grad():
        w[0].mul_(2)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, dy[0])
    with torch.inference_mode():
        es.einshard("b s c, n c -> b s n", es.checkpoint8(torch.ones(2, 3, 32, dtype=torch.bfloat16, device=device)),
                    torch.ones(8, 32, dtype=torch.bfloat16, device=device))


@pytest.mark.parametrize("device", DEVICES)
def test_inference_tensors_are_read_as_they_are(device):
    """They carry no version that would show a change: every product reads the operand itself, not an earlier copy."""
    with torch.inference_mode():
        x = torch.randn(2, 8, 37, generator=torch.Generator().manual_seed(15)).to(torch.bfloat16).to(device)
        w = torch.eye(37, device=device).to(torch.bfloat16)
        kept = es.checkpoint8(x)
        assert torch.equal(es.einshard("b s c, n c -> b s n", kept, w), x)
        x.mul_(2)
        assert torch.equal(es.einshard("b s c, n c -> b s n", kept, w), x)


# ------------------------------------------------------------------ two ranks

def _sharded_models(ctx):
    """Values are those of whole operands; gradients those of operands within half a step (1/128 of a block's largest)."""
    mesh = ctx.mesh((2,), ("tp",))
    gen = torch.Generator().manual_seed(0)
    models = [TPMLP(64, 256, mesh, dtype=torch.float32, device="cpu", std=0.1, checkpoint=c) for c in (None, "int8")]
    x = [torch.randn(2, 24, 64, generator=gen).requires_grad_(True)]
    x.append(x[0].detach().clone().requires_grad_(True))
    ys = [m(v) for m, v in zip(models, x)]
    assert (ys[0] - ys[1]).abs().max() <= 2.0 ** -20 * ys[0].abs().max()
    for y in ys:
        y.square().sum().backward()
    assert (x[0].grad - x[1].grad).norm() <= 0.03 * x[0].grad.norm()
    for p, q in zip(models[0].parameters(), models[1].parameters()):
        assert (p.grad - q.grad).norm() <= 0.03 * p.grad.norm()

    cfg = TransformerConfig(layers=2, d=64, heads=4, mlp=128, vocab=97, seq=16, dtype=torch.float32, norm="sandwich")
    tokens = torch.randint(0, 97, (2, 16), generator=gen)
    losses, grads = [], []
    for mode in (False, "int8"):
        model = TPTransformer(cfg, mesh, device="cpu", checkpoint=mode)
        loss = model(tokens, tokens.roll(-1, 1))
        loss.backward()
        losses.append(loss.item())
        grads.append([p.grad for p in model.parameters()])
    assert abs(losses[0] - losses[1]) <= 1e-5 * abs(losses[0])
    for p, q in zip(*grads):
        assert (p - q).norm() <= 0.05 * p.norm() + 1e-6


def _sharded_equations(ctx):
    """Column parallel contractions of one operand are local, like those of a plain one: dx is the rank's share."""
    mesh = ctx.mesh((2,), ("tp",))
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 6, 32, generator=gen).requires_grad_(True)
    w = [torch.randn(n, 32, generator=gen) for n in (16, 24)]
    local = [v.chunk(2, 0)[ctx.rank].clone().requires_grad_(True) for v in w]
    kept = es.checkpoint8(x)
    ys = [es.einshard("b s c, n/tp c -> b s n/tp", kept, v, mesh=mesh) for v in local]
    dy = [torch.randn(2, 6, v.shape[0], generator=gen) for v in w]
    mine = [d.chunk(2, -1)[ctx.rank].contiguous() for d in dy]
    dx, *dw = torch.autograd.grad(ys, [x, *local], mine)
    with torch.no_grad():
        want = sum(d.double() @ v.double() for d, v in zip(mine, local))
        size = sum(d.double().abs() @ v.double().abs() for d, v in zip(mine, local))
    assert ((dx.double() - want).abs() <= size * 21 * 2.0 ** -24).all()  # 20 products and their sum
    restored = kept.restore().double()
    for g, d in zip(dw, mine):
        full = torch.einsum("bsn,bsc->nc", d.double(), restored)
        bound = torch.einsum("bsn,bsc->nc", d.double().abs(), restored.abs())
        assert ((g.double() - full).abs() <= bound * 13 * 2.0 ** -24).all()

    # a plan with communication: the same values and operand gradient as for the plain operand
    for formula in ("b s c, n/tp c -> b s n", "b s c, n c -> b s n/tp"):
        got = []
        for operand in (x, es.checkpoint8(x)):
            v = (local[0] if "n/tp c" in formula else w[0]).detach().clone().requires_grad_(True)
            y = es.einshard(formula, operand, v, mesh=mesh)
            d = dy[0] if formula.endswith("s n") else mine[0]
            got.append((y.detach(), *torch.autograd.grad(y, [x, v], d)))
        assert torch.equal(got[0][0], got[1][0])
        assert (got[0][1] - got[1][1]).norm() <= 2.0 ** -20 * got[0][1].norm()
        assert (got[0][2] - got[1][2]).norm() <= 0.03 * got[0][2].norm()


@pytest.mark.parametrize("body", [_sharded_models, _sharded_equations])
def test_two_ranks(body):
    run_ranks(body, world_size=2)


def _changed_operand(ctx):
    """Where a plan hands the operand on unchanged, a change since its codes were formed is noticed there too."""
    mesh = ctx.mesh((2,), ("tp",))
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(2, 6, 32, generator=gen).requires_grad_(True)
    w = torch.randn(16, 32, generator=gen)
    for formula, v in (("b s c, n c -> b s n/tp", w), ("b s c, n/tp c -> b s n", w[:8])):
        h = x * 1
        kept = es.checkpoint8(h)
        es.einshard(formula, kept, v, mesh=mesh)
        with torch.no_grad():
            h.add_(1)
        with pytest.raises(RuntimeError, match="modified in place"):
            es.einshard(formula, kept, v, mesh=mesh)


def test_changed_operand_on_two_ranks():
    run_ranks(_changed_operand, world_size=2)
