"""einnorm: norms around a block with gate and residual scale, and their gradients.

The oracle evaluates the formulas in 64 bits, gradients by autograd.  Tolerances:
an output's own rounding is half a step of its type; the 32-bit arithmetic
before it is bounded by the same formulas evaluated on absolute values (every
subtraction an addition), times 2^-24 for each of at most 64 operations on the
way of a term, and one more for each row of a sum over rows.
"""

import pytest
import torch
import torch.distributed as dist

import torch_einshard_b200 as es
from torch_einshard_b200.models.transformer import TPTransformer, TransformerConfig

cuda = pytest.param("cuda", marks=pytest.mark.gpu)
DEVICES = ["cpu", cuda]
TYPES = [torch.bfloat16, torch.float16, torch.float32]
GATES = {"none": None, "channel": "d", "batch": "b d", "token": "b s d", "seq": "s d", "scalar": "", "row": "b s"}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(device, dtype, shape, gate="channel", kind="layer", post=True, seed=0, param_dtype=None, affine=True):
    b, s, d = shape
    gen = torch.Generator().manual_seed(seed)
    pd = param_dtype or dtype

    def r(*sh, scale=1.0, shift=0.0, t=dtype):
        return (torch.randn(sh, generator=gen) * scale + shift).to(t).to(device).requires_grad_(True)

    t = dict(x=r(b, s, d, shift=0.2), y=r(b, s, d, shift=-0.1))
    if affine:
        t["weight"] = r(d, scale=0.2, shift=1.0, t=pd)
        if kind == "layer":
            t["bias"] = r(d, scale=0.2, t=pd)
        if post:
            t["post_weight"] = r(d, scale=0.2, shift=1.0, t=pd)
            if kind == "layer":
                t["post_bias"] = r(d, scale=0.2, t=pd)
    axes = GATES[gate]
    if axes is not None:
        t["gate"] = r(*[dict(b=b, s=s, d=d)[a] for a in axes.split()], scale=0.3, shift=0.5, t=pd)
    conf = dict(kind=kind, post=post, gate_axes=axes, scale=0.75)
    dh, dn = (torch.randn(b, s, d, generator=gen).to(dtype).to(device) for _ in range(2))
    return t, conf, dh, dn


def run(t, conf, formula="b s d", axis="d"):
    return es.einnorm(formula, axis=axis, **t, **conf)


def wide_gate(gate, axes, shape):
    if gate is None:
        return torch.ones((), dtype=torch.float64)
    view = [n if a in axes.split() else 1 for a, n in zip("bsd", shape)]
    return gate.reshape(view)


def reference(t, conf, dh, dn, eps=1e-5):
    """{output or gradient: (value, slack)}; slack: the formulas on absolute values."""
    v = {k: u.detach().double().cpu().requires_grad_(True) for k, u in t.items()}
    layer, shape = conf["kind"] == "layer", t["x"].shape
    mean = lambda u: u.mean(-1, keepdim=True)  # noqa: E731

    def norm(u):
        c = u - mean(u) if layer else u
        r = 1 / torch.sqrt(mean(c * c) + eps)
        return c * r, r

    one = torch.ones((), dtype=torch.float64)
    gate = wide_gate(v.get("gate"), conf["gate_axes"] or "", shape)
    pw, pb, w, b = (v.get(k) for k in ("post_weight", "post_bias", "weight", "bias"))
    yh, ry = norm(v["y"]) if conf["post"] else (v["y"], one)
    p = yh * (one if pw is None else pw) + (0 if pb is None else pb)
    h = conf["scale"] * v["x"] + gate * p
    hh, rh = norm(h)
    n = hh * (one if w is None else w) + (0 if b is None else b)
    grads = torch.autograd.grad((h, n), list(v.values()), (dh.double().cpu(), dn.double().cpu()))
    # the same on absolute values
    with torch.no_grad():
        a = {k: u.abs() for k, u in v.items()}
        dha, dna, ga = dh.double().cpu().abs(), dn.double().cpu().abs(), gate.abs()
        one_or = lambda u: one if u is None else u.abs()  # noqa: E731
        zero_or = lambda u: torch.zeros(()) if u is None else u.abs()  # noqa: E731
        yh_s = (a["y"] + mean(a["y"])) * ry if conf["post"] else a["y"]
        p_s = yh_s * one_or(pw) + zero_or(pb)
        h_s = abs(conf["scale"]) * a["x"] + ga * p_s
        hh_s = (h_s + mean(h_s)) * rh
        n_s = hh_s * one_or(w) + zero_or(b)
        gn = dna * one_or(w)
        D = dha + rh * (gn + mean(gn) + hh_s * mean(gn * hh_s))
        tD = ga * one_or(pw) * D
        s = dict(x=abs(conf["scale"]) * D, gate=D * p_s, weight=dna * hh_s, bias=dna, post_weight=ga * D * yh_s,
                 post_bias=ga * D, y=ry * (tD + mean(tD) + yh_s * mean(tD * yh_s)) if conf["post"] else ga * D)

        def fold(slack, like):
            for i, k in enumerate("bsd"):
                if i < 3 and k not in (conf["gate_axes"] or "").split():
                    slack = slack.sum(i, keepdim=True)
            return slack.reshape(like.shape)

        out = dict(h=(h.detach(), h_s), n=(n.detach(), n_s))
        for k, g in zip(v, grads):
            sl = s[k]
            if k == "gate":
                sl = fold(sl.expand(shape), v[k])
            elif k not in ("x", "y"):
                sl = sl.expand(shape).sum((0, 1))
            out["d" + k] = (g, sl)
    return out


def close(got, want, slack, rows):
    bound = half_step(got.dtype) * want.abs() + (64 + rows) * 2.0 ** -24 * slack * (1 + half_step(got.dtype))
    bound = bound + torch.finfo(got.dtype).smallest_normal
    err = (got.detach().double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), float((err / bound).max())


def check(t, conf, dh, dn):
    h, n = run(t, conf)
    grads = torch.autograd.grad((h, n), list(t.values()), (dh, dn))
    ref = reference(t, conf, dh, dn)
    rows = h.shape[0] * h.shape[1]
    for name, got in [("h", h), ("n", n)] + [("d" + k, g) for k, g in zip(t, grads)]:
        want, slack = ref[name]
        assert got.shape == want.shape
        # the sum over a broadcast gate's rows may go through a product rounded to 32 bits
        close(got, want, slack, rows + 8)


SHAPES = [(1, 1, 1), (1, 1, 64), (2, 3, 33), (3, 17, 256), (2, 40, 1000), (1, 5, 2047), (2, 9, 4096)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(device, dtype, kind, shape):
    if shape[2] == 1 and kind == "layer":
        pytest.skip("one channel minus its mean is zero: the norm is the bias")
    check(*make(device, dtype, shape, kind=kind))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("d", [4104, 8192, 8191, 8200, 10001, 16384, 32776, 65536, 65544])
@pytest.mark.parametrize("gate", ["channel", "token"])
def test_wide_rows(dtype, kind, d, gate):
    check(*make("cuda", dtype, (2, 21, d), kind=kind, gate=gate))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("shape", [(3, 20, 96), (2, 16, 41), (5, 1, 64), (1, 24, 64)])
def test_gates(device, kind, post, gate, shape):
    check(*make(device, torch.float32, shape, gate=gate, kind=kind, post=post))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("shape", [(3, 20, 96), (2, 16, 41), (5, 1, 64), (1, 24, 64)])
def test_gates_of_16_bits(device, dtype, post, gate, shape):
    """A gate's gradient is summed in 32 bits, over the normalised axis too, and rounded once."""
    check(*make(device, dtype, shape, gate=gate, post=post))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES[:2])
def test_gate_of_16_bits_over_separated_axes(device, dtype):
    gen = torch.Generator().manual_seed(0)
    x, y, g = (torch.randn(*s, generator=gen).to(dtype).to(device).requires_grad_(True)
               for s in ((2, 33, 4, 16), (2, 33, 4, 16), (4, 2, 16)))
    h, _ = es.einnorm("b s h d", x, y, axis="d", gate=g, gate_axes="h b d")
    dh = torch.randn(h.shape, generator=gen).to(dtype).to(device)
    (got,) = torch.autograd.grad(h, g, dh)
    terms = (dh.double() * y.detach().double()).cpu()
    # 33 products and additions in 32 bits, one rounding
    close(got, terms.sum(1).permute(1, 0, 2), terms.abs().sum(1).permute(1, 0, 2), 33)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [(1, 5000), (7, 700), (300, 3), (40, 16)])
@pytest.mark.parametrize("gate", ["channel", "batch", "token", "seq"])
def test_many_rows(rows, gate):
    check(*make("cuda", torch.bfloat16, (*rows, 128), gate=gate))
    check(*make("cuda", torch.bfloat16, (*rows, 100), gate=gate, kind="rms"))


@pytest.mark.parametrize("device", DEVICES)
def test_no_affine_and_fp32_parameters(device):
    check(*make(device, torch.bfloat16, (2, 7, 64), affine=False))
    check(*make(device, torch.bfloat16, (2, 7, 64), affine=False, gate="none", kind="rms"))
    check(*make(device, torch.bfloat16, (2, 7, 72), param_dtype=torch.float32))
    check(*make(device, torch.float16, (2, 7, 33), param_dtype=torch.float32, kind="rms", gate="token"))


@pytest.mark.parametrize("device", DEVICES)
def test_rms_with_biases(device):
    t, conf, dh, dn = make(device, torch.float32, (2, 7, 64), kind="layer")
    check(t, dict(conf, kind="rms"), dh, dn)


def without(made, *keys):
    t, *rest = made
    return ({k: v for k, v in t.items() if k not in keys}, *rest)


ABSENT = [(), ("weight", "bias"), ("bias", "post_bias"), ("post_weight",), ("post_weight", "post_bias"),
          ("weight", "bias", "post_weight", "post_bias")]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("absent", ABSENT)
def test_absent_vectors(device, dtype, kind, post, gate, absent):
    """Columns that a row does not have add nothing, whichever vectors are there: rows that fill a block and rows that
    do not, aligned and not."""
    for d in (33, 64, 256, 1000):
        check(*without(make(device, dtype, (2, 9, d), gate=gate, kind=kind, post=post), *absent))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [512, 2047, 4104, 8191, 8200, 10001, 32776, 65544])
@pytest.mark.parametrize("absent", [("post_weight",), ("weight", "bias", "post_weight", "post_bias")])
def test_absent_vectors_of_wide_rows(dtype, d, absent):
    check(*without(make("cuda", dtype, (2, 21, d), gate="none"), *absent))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("d", [64, 37])
def test_without_a_block(device, kind, d):
    gen = torch.Generator().manual_seed(0)
    x, w, dn, dh = (torch.randn(*s, generator=gen).to(device) for s in ((3, 5, d), (d,), (3, 5, d), (3, 5, d)))
    x.requires_grad_(True)
    w.requires_grad_(True)
    h, n = es.einnorm("b s d", x, axis="d", kind=kind, weight=w)
    assert h is x
    xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    c = xd - xd.mean(-1, keepdim=True) if kind == "layer" else xd
    want = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * wd
    assert torch.allclose(n.double(), want, atol=1e-5)
    got = torch.autograd.grad((h, n), (x, w), (dh, dn))
    ref = torch.autograd.grad((xd, want), (xd, wd), (dh.double(), dn.double()))
    for a, b in zip(got, ref):
        assert torch.allclose(a.double(), b, rtol=1e-5, atol=2e-5)


def test_against_differences():
    t, conf, dh, dn = make("cpu", torch.float64, (2, 3, 6), gate="batch")
    names = list(t)

    def f(*vals):
        return run(dict(zip(names, vals)), conf)

    assert torch.autograd.gradcheck(f, list(t.values()))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_against_differences_on_the_kernels(kind):
    """Directional derivatives: central differences of the kernel's own 32-bit outputs (step 1e-2, third-order
    error; rounding 2^-24 / step of the outputs' size each)."""
    t, conf, dh, dn = make("cuda", torch.float32, (2, 3, 40), gate="batch", kind=kind)
    h, n = run(t, conf)
    grads = torch.autograd.grad((h, n), list(t.values()), (dh, dn))
    gen = torch.Generator().manual_seed(5)
    for (k, u), g in zip(t.items(), grads):
        v = torch.randn(u.shape, generator=gen).cuda()
        v /= v.norm()
        outs = []
        for sign in (1, -1):
            moved = {**{a: b.detach() for a, b in t.items()}, k: u.detach() + sign * 1e-2 * v}
            hs, ns = run(moved, conf)
            outs.append((hs.double() * dh).sum() + (ns.double() * dn).sum())
        diff = float((outs[0] - outs[1]) / 2e-2)
        assert abs(diff - float((g * v).sum())) <= 2e-3 * (1 + float(g.norm()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["h", "n"])
def test_one_output_used(device, which):
    t, conf, dh, dn = make(device, torch.float32, (2, 5, 40))
    out = dict(zip("hn", run(t, conf)))
    zero = torch.zeros_like(dh)
    ref = reference(t, conf, dh if which == "h" else zero, dn if which == "n" else zero)
    grads = torch.autograd.grad(out[which], list(t.values()), dh if which == "h" else dn, allow_unused=True)
    for (k, u), g in zip(t.items(), grads):
        want, slack = ref["d" + k]
        close(torch.zeros_like(u) if g is None else g, want, slack, 18)


@pytest.mark.parametrize("device", DEVICES)
def test_subsets_of_gradients(device):
    t, conf, dh, dn = make(device, torch.float32, (2, 20, 40), gate="channel")
    full = dict(zip(t, torch.autograd.grad(run(t, conf), list(t.values()), (dh, dn))))
    for wanted in (["x"], ["y"], ["gate"], ["weight", "post_bias"], ["x", "post_weight"]):
        u = {k: v.detach().requires_grad_(k in wanted) for k, v in t.items()}
        grads = torch.autograd.grad(run(u, conf), [u[k] for k in wanted], (dh, dn))
        for k, g in zip(wanted, grads):
            assert torch.equal(g, full[k])


@pytest.mark.parametrize("device", DEVICES)
def test_axes_strides_and_offsets(device):
    t, conf, dh, dn = make(device, torch.float32, (4, 6, 48), gate="batch")
    h, n = run(t, conf)
    # the normalised axis in the middle
    m = {k: v.detach().movedim(-1, 1) if v.dim() == 3 else v.detach() for k, v in t.items()}
    h2, n2 = run(m, conf, "b d s")
    assert torch.allclose(h2.movedim(1, -1), h, atol=1e-6) and torch.allclose(n2.movedim(1, -1), n, atol=1e-5)
    # slices of wider rows, an offset base, a transposed stream, an ellipsis
    wide = torch.zeros(4, 6, 60, device=device)
    for off in (0, 1, 4):
        xs = wide.clone()
        xs[..., off:off + 48] = t["x"].detach()
        h2, n2 = run({**t, "x": xs[..., off:off + 48]}, conf)
        assert torch.allclose(h2, h, atol=1e-6) and torch.allclose(n2, n, atol=1e-5)
    xt = t["x"].detach().transpose(0, 1).contiguous().transpose(0, 1)
    h2, n2 = run({**t, "x": xt}, conf)
    assert torch.allclose(h2, h, atol=1e-6) and torch.allclose(n2, n, atol=1e-5)
    conf2 = dict(conf, gate_axes="b d")
    h2, n2 = es.einnorm("b ... d", axis="d", **t, **conf2)
    assert torch.equal(h2, h) and torch.equal(n2, n)
    expanded = {**t, "x": t["x"].detach()[:, :1].expand(4, 6, 48)}
    h3, _ = run(expanded, conf)
    h4, _ = run({**t, "x": expanded["x"].contiguous()}, conf)
    assert torch.allclose(h3, h4, atol=1e-6)
    # gradients through a transposed upstream
    g = torch.autograd.grad((h, n), list(t.values()), (dh, dn))
    g2 = torch.autograd.grad(run(t, conf), list(t.values()),
                             (dh.transpose(0, 1).contiguous().transpose(0, 1), dn.expand_as(dn)))
    for a, b in zip(g, g2):
        assert torch.allclose(a, b, atol=1e-6)


def negated(t):
    """-t as a view that only says so (what the imaginary part of a conjugate is)."""
    return torch._neg_view(t.detach())


@pytest.mark.parametrize("device", DEVICES)
def test_negated_views(device):
    """Inputs and gradients whose sign is kept beside their memory."""
    t, conf, dh, dn = make(device, torch.float32, (2, 9, 40), gate="batch")
    minus = {k: (-v.detach()).requires_grad_(True) for k, v in t.items()}
    views = {k: negated(v).requires_grad_(True) for k, v in t.items()}
    want = run(minus, conf)
    want = (*want, *torch.autograd.grad(want, list(minus.values()), (-dh, -dn)))
    got = run(views, conf)
    got = (*got, *torch.autograd.grad(got, list(views.values()), (negated(dh), negated(dn))))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_gate_over_separated_axes(device):
    """A gate that skips an axis between its own (b h of b s h d)."""
    gen = torch.Generator().manual_seed(0)
    x, y, g = (torch.randn(*s, generator=gen).to(device).requires_grad_(True)
               for s in ((2, 3, 4, 16), (2, 3, 4, 16), (4, 2, 16)))
    h, _ = es.einnorm("b s h d", x, y, axis="d", gate=g, gate_axes="h b d")
    want = x + g.permute(1, 0, 2)[:, None] * y
    assert torch.allclose(h, want, atol=1e-6)
    dh = torch.randn(h.shape, generator=gen).to(device)
    for a, b in zip(torch.autograd.grad(h, (x, y, g), dh), torch.autograd.grad(want, (x, y, g), dh)):
        assert torch.allclose(a, b, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
def test_empty_and_constant_rows(device):
    t, conf, dh, dn = make(device, torch.float32, (2, 0, 16), gate="batch")
    h, n = run(t, conf)
    assert h.shape == n.shape == (2, 0, 16)
    for k, g in zip(t, torch.autograd.grad((h, n), list(t.values()), (dh, dn))):
        assert g.shape == t[k].shape and not g.any()
    t, conf, dh, dn = make(device, torch.float32, (1, 4, 32))
    t["y"] = torch.full((1, 4, 32), 3.0, device=device, requires_grad=True)
    check(t, conf, dh, dn)


@pytest.mark.parametrize("device", DEVICES)
def test_non_finite_rows_stay_in_their_row(device):
    t, conf, dh, dn = make(device, torch.float32, (1, 6, 40), gate="token")
    clean = run(t, conf)
    t["y"] = t["y"].detach().clone()
    t["y"][0, 2, 5] = float("nan")
    t["y"][0, 4, 1] = float("inf")
    for got, want in zip(run(t, conf), clean):
        keep = torch.tensor([0, 1, 3, 5], device=device)
        assert torch.equal(got[0, keep], want[0, keep])
        assert torch.isnan(got[0, 2]).any() and not torch.isfinite(got[0, 4]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.randn(2, 3, 8, device=device)
    w = torch.ones(8, device=device)
    ok = dict(axis="d")
    for error, args, kw in [
        (ValueError, ("b s d", x), dict(axis="e")),
        (ValueError, ("b s", x), dict(axis="s")),
        (ValueError, ("b d d", x), ok),
        (ValueError, ("b s d // tp", x), ok),
        (NotImplementedError, ("b s d/tp", x), ok),
        (NotImplementedError, ("b (s d)", x.view(2, 24)), ok),
        (TypeError, ("b s d", x.long()), ok),
        (ValueError, ("b s d", x[..., :0]), ok),
        (ValueError, ("b s d", x), dict(axis="d", kind="batch")),
        (ValueError, ("b s d", x), dict(axis="d", eps=-1.0)),
        (ValueError, ("b s d", x, x), dict(axis="d", scale=float("nan"))),
        (ValueError, ("b s d", x), dict(axis="d", post=True)),
        (ValueError, ("b s d", x), dict(axis="d", scale=0.5)),
        (ValueError, ("b s d", x), dict(axis="d", gate=w, gate_axes="d")),
        (ValueError, ("b s d", x, x[:, :2]), ok),
        (ValueError, ("b s d", x, x.double()), ok),
        (ValueError, ("b s d", x, x), dict(axis="d", post_weight=w)),
        (ValueError, ("b s d", x, x), dict(axis="d", weight=w[:4])),
        (ValueError, ("b s d", x, x), dict(axis="d", weight=w.double())),
        (ValueError, ("b s d", x, x), dict(axis="d", weight=w.half())),
        (ValueError, ("b s d", x, x), dict(axis="d", gate=w)),
        (ValueError, ("b s d", x, x), dict(axis="d", gate_axes="d")),
        (ValueError, ("b s d", x, x), dict(axis="d", gate=w, gate_axes="e")),
        (ValueError, ("b s d", x, x), dict(axis="d", gate=w, gate_axes="s")),
        (ValueError, ("b s d", x, x), dict(axis="d", gate=w, gate_axes="b d")),
        (ValueError, ("b/dp s d", x, x), dict(axis="d", gate=x[:, 0], gate_axes="b d")),
    ]:
        with pytest.raises(error):
            es.einnorm(*args, **kw)


@pytest.mark.gpu
def test_no_second_derivative():
    t, conf, dh, dn = make("cuda", torch.float32, (2, 5, 40))
    h, n = run(t, conf)
    (dx,) = torch.autograd.grad((h, n), t["x"], (dh, dn), create_graph=True)
    assert torch.equal(dx.detach(), torch.autograd.grad(run(t, conf), t["x"], (dh, dn))[0])
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(dx.sum(), t["x"], allow_unused=True)


@pytest.mark.parametrize("device", DEVICES)
def test_results_may_be_changed_in_place(device):
    t, conf, dh, dn = make(device, torch.float32, (2, 5, 40))
    want = torch.autograd.grad(run(t, conf), t["x"], (dh, 2 * dn))
    h, n = run(t, conf)
    n *= 2
    assert torch.allclose(torch.autograd.grad((h, n), t["x"], (dh, dn))[0], want[0], atol=1e-6)
    # and an input changed between the passes is noticed
    x = t["x"].detach().clone().requires_grad_(True)
    moved = x * 1
    h, n = run({**t, "x": moved}, conf)
    moved.add_(1)
    if device == "cuda":
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad((h, n), x, (dh, dn))


@pytest.mark.gpu
def test_other_stream_and_capture():
    t, conf, dh, dn = make("cuda", torch.bfloat16, (2, 64, 256), gate="batch")
    want = run(t, conf)
    want_g = torch.autograd.grad(want, list(t.values()), (dh, dn))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = run(t, conf)
        grads = torch.autograd.grad(out, list(t.values()), (dh, dn))
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip((*out, *grads), (*want, *want_g)):
        assert torch.equal(a, b)
    # two graphs of the same leaves, replayed in turn: neither keeps state of the other
    del out, grads, a, b
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in t.items()}
    want = [u.detach().clone() for u in want]
    want_g = [u.clone() for u in want_g]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = run(leaves, conf)
            g = torch.autograd.grad(o, list(leaves.values()), (dh, dn))
        graphs.append((graph, [u.detach() for u in o], g))
        del o, g
    for graph, _, _ in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, o, g in graphs:
        for a, b in zip((*o, *g), (*want, *want_g)):
            assert torch.equal(a, b)


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
def test_sandwich_transformer(one_rank_mesh):
    """norm="sandwich" blocks against the same formulas on torch."""
    device, mesh = one_rank_mesh
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    cfg = TransformerConfig(layers=3, d=64, heads=4, mlp=128, vocab=97, seq=16, dtype=dtype, norm="sandwich")
    model = TPTransformer(cfg, mesh, device=device)
    tokens = torch.randint(0, 97, (2, 16), generator=torch.Generator().manual_seed(1)).to(device)
    logits = model(tokens)

    def ln(u, norm):
        return torch.nn.functional.layer_norm(u, (64,), norm.weight.float(), norm.bias.float())

    with torch.no_grad():
        x = torch.nn.functional.embedding(tokens, model.embed).float()
        for block in model.blocks:
            x = x + block.gate1.float() * ln(block.attention(ln(x, block.ln1).to(dtype), mesh).float(), block.post1)
            x = x + block.gate2.float() * ln(block.mlp(ln(x, block.ln2).to(dtype), mesh).float(), block.post2)
        want = ln(x, model.ln_f) @ model.embed.float().t()
    # 16-bit streams and contractions: a few roundings of 2^-8 through three blocks
    assert (logits.float() - want).norm() <= (1e-5 if dtype == torch.float32 else 0.02) * want.norm()
    loss = model(tokens, tokens.roll(-1, 1))
    loss.backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), name
    # the 8-bit operands and recomputed blocks give the same loss
    for mode in (True, "int8"):
        other = TPTransformer(cfg, mesh, device=device, checkpoint=mode)
        assert abs(float(other(tokens, tokens.roll(-1, 1)).detach()) - float(loss.detach())) <= 0.02 * float(loss.detach())
    with pytest.raises(ValueError):
        TransformerConfig(norm="post")
