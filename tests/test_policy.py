"""einpolicy: clipped policy loss with a KL term from logits, and its gradient.

The oracle works in 64 bits with torch's own log_softmax and autograd.
Tolerances: the log-probability is a difference of 32-bit numbers, off by a few
roundings of its largest parts (|z| / T and the log of the sum) and by the
exponentials' 2^-21 relative error in the sum; the rest follows by the
derivatives of the formula, and a gradient is rounded once to the logits' type.
"""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
import torch.distributed as dist

import torch_einshard_b200 as es
from torch_einshard_b200.models.transformer import TPTransformer, TransformerConfig

cuda = pytest.param("cuda", marks=pytest.mark.gpu)
DEVICES = ["cpu", cuda]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(device, dtype, b, s, v, seed=0, advantage="token", spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    z = (torch.randn(b, s, v, generator=gen) * spread).to(dtype)
    ids = torch.randint(0, v, (b, s), generator=gen)
    lp = torch.log_softmax(z.double(), -1).gather(-1, ids[..., None])[..., 0]
    old = (lp + 0.3 * torch.randn(b, s, generator=gen)).float()
    ref = (lp + 0.3 * torch.randn(b, s, generator=gen)).float()
    adv = torch.randn((b, s) if advantage == "token" else (b,), generator=gen)
    mask = torch.rand(b, s, generator=gen) < 0.7
    t = dict(logits=z, ids=ids, old_logp=old, ref_logp=ref, advantages=adv, mask=mask)
    return {k: u.to(device) for k, u in t.items()}


def off_border(t, lo, hi, temp=1.0):
    """old_logp moved where the ratio is within 1e-4 of a clip border (its side would hang on a rounding)."""
    z = t["logits"].double() / temp
    lp = torch.log_softmax(z, -1).gather(-1, t["ids"].clamp(0, z.shape[-1] - 1)[..., None])[..., 0]
    ratio = torch.exp(lp - t["old_logp"].double())
    near = ((ratio - 1 + lo).abs() < 1e-4) | ((ratio - 1 - hi).abs() < 1e-4)
    t["old_logp"] = torch.where(near, t["old_logp"] - 0.01, t["old_logp"])
    return t


def oracle(t, lo, hi, kl, temp, reduction, weight=1.0):
    """(loss, logp, kl, clipped, dlogits, d loss_t / d lp of each token) in 64 bits on the CPU."""
    u = {k: v.detach().cpu() for k, v in t.items() if v is not None}
    z = u["logits"].double().requires_grad_(True)
    mask = u.get("mask", torch.ones(u["ids"].shape, dtype=torch.bool))
    clean = torch.where(mask[..., None], z, 0)
    ids = torch.where(mask, u["ids"].long(), 0)
    lp = torch.log_softmax(clean / temp, -1).gather(-1, ids[..., None])[..., 0]
    adv = u["advantages"].double()
    adv = adv if adv.dim() == lp.dim() else adv[..., None].expand(lp.shape)
    adv = torch.where(mask, adv, 0)
    old = torch.where(mask, u["old_logp"].double(), 0) if "old_logp" in u else lp.detach()
    old = torch.where(mask, old, lp.detach())
    r = torch.exp(lp - old)
    s1, s2 = r * adv, r.clamp(1 - lo, 1 + hi) * adv
    loss = -torch.minimum(s1, s2)
    k3 = torch.zeros_like(lp)
    if "ref_logp" in u:
        d = torch.where(mask, u["ref_logp"].double(), lp.detach()) - lp
        k3 = torch.exp(d) - d - 1
    count = mask.sum(-1)
    if reduction == "sum":
        w = mask.double()
    elif reduction == "mean":
        w = mask.double() / max(int(count.sum()), 1)
    else:
        w = mask.double() / count.clamp(min=1)[..., None] / max(int((count > 0).sum()), 1)
    terms = loss + kl * k3
    total = weight * (w * terms).sum()
    (grad,) = torch.autograd.grad(total, z)
    slope = torch.where((s1 <= s2), -r * adv, 0) + (kl * (1 - torch.exp(torch.where(mask, u["ref_logp"].double(), lp) - lp)) if "ref_logp" in u else 0)
    values = [x.detach() for x in (total, torch.where(mask, lp, 0), (w * k3).sum(), (w * (s1 > s2)).sum(), grad)]
    return (*values, (w * slope).detach() * weight, (w * terms.abs()).detach().sum())


def check(t, lo=0.2, hi=0.2, kl=0.05, temp=1.0, reduction="mean", weight=1.0, upstream=1.0):
    logits = t["logits"].detach().requires_grad_(True)
    extra = {} if weight == 1.0 else dict(weight=weight)
    r = es.einpolicy("b s v", logits, t["ids"], axis="v", advantages=t["advantages"], old_logp=t["old_logp"],
                     ref_logp=t["ref_logp"], mask=t["mask"], clip=(lo, hi), kl=kl, temperature=temp,
                     reduction=reduction, **extra)
    (got,) = torch.autograd.grad(r.loss, logits, torch.tensor(upstream, device=logits.device))
    loss, lp, kl_ref, clipped, grad, slope, size = oracle(t, lo, hi, kl, temp, reduction, weight)
    assert r.loss.dtype == torch.float32 and r.loss.dim() == 0 and not r.logp.requires_grad
    live = t["mask"].cpu() if t["mask"] is not None else torch.ones(t["ids"].shape, dtype=torch.bool)
    top = torch.where(live, t["logits"].detach().double().cpu().abs().amax(-1), 0) / temp
    lp_err = 2.0 ** -21 + 8 * 2.0 ** -24 * (top + torch.log(torch.tensor(float(logits.shape[-1]))) + 1)
    assert ((r.logp.double().cpu() - lp).abs() <= lp_err).all()
    lp_err = float(lp_err.max())
    tol = abs(weight) * (float(size) + float(kl_ref)) * (1e-5 + 8 * lp_err) + float(slope.abs().sum()) * lp_err + 1e-7
    assert abs(float(r.loss) - float(loss)) <= tol
    assert abs(float(r.kl) - float(kl_ref)) <= 1e-5 * float(kl_ref) + 4 * lp_err * (1 + float(clipped) + float(kl_ref)) * (live.sum() if reduction == "sum" else 1) + 1e-7
    assert abs(float(r.clipped) - float(clipped)) <= 1e-6 * (1 + float(clipped))
    # k (1[j = a] - p): the slope and p are each off by a few lp_err relative to 1 (and the KL part's 1 - e^d by kl)
    k = (slope.abs() + kl * 1e-0 * abs(weight) * (slope != 0)) * abs(upstream) / temp
    hit = torch.zeros_like(grad)
    ids = torch.where(live, t["ids"].cpu().long(), 0)
    hit.scatter_(-1, ids[..., None], 1.0)
    p = torch.softmax(torch.where(live[..., None], t["logits"].detach().double().cpu(), 0) / temp, -1)
    bound = half_step(logits.dtype) * (grad * upstream).abs() + 16 * lp_err * k[..., None] * (hit + p) + \
        torch.finfo(logits.dtype).smallest_normal * (1 + half_step(logits.dtype))
    err = (got.double().cpu() - grad * upstream).abs()
    assert got.dtype == logits.dtype and (err <= bound).all(), float((err / bound).max())
    assert not got.cpu()[~live].any()


SHAPES = [(1, 1, 1), (1, 1, 7), (2, 3, 33), (1, 5, 1000), (3, 9, 4097), (2, 33, 511)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum"])
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradient(device, dtype, reduction, shape):
    check(off_border(make(device, dtype, *shape), 0.2, 0.2), reduction=reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [32000, 32003, 50257, 131071])
def test_large_vocabularies(dtype, vocab):
    check(off_border(make("cuda", dtype, 2, 7, vocab, advantage="sequence"), 0.1, 0.3), lo=0.1, hi=0.3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("temp", [0.5, 1.0, 1.7])
@pytest.mark.parametrize("clip", [(0.0, 0.0), (0.2, 0.28), (1.0, float("inf"))])
@pytest.mark.parametrize("kl", [0.0, 0.1])
def test_settings(device, temp, clip, kl):
    t = off_border(make(device, torch.float32, 3, 7, 65, advantage="sequence"), *clip, temp)
    if clip[0] == 0.0:  # a ratio of exactly 1 is on both borders: nothing else is
        t["old_logp"] = t["old_logp"] + 0.01
        t = off_border(t, *clip, temp)
    check(t, *clip, kl, temp)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("upstream", [0.0, -2.0, 0.3, 1024.0])
def test_upstream_gradient(device, upstream):
    check(off_border(make(device, torch.bfloat16, 2, 9, 300), 0.2, 0.2), upstream=upstream)


@pytest.mark.parametrize("device", DEVICES)
def test_fp16_gradients_below_its_range_come_back_scaled(device):
    """Loss scaling: the gradient is rounded after the upstream factor, so small ones are not lost before it."""
    t = off_border(make(device, torch.float16, 4, 64, 3001), 0.2, 0.2)
    check(t, upstream=65536.0)


@pytest.mark.parametrize("device", DEVICES)
def test_on_policy(device):
    """Without old_logp the ratio is 1: the gradient is that of -A lp."""
    t = make(device, torch.float32, 2, 9, 50)
    t["old_logp"] = t["ref_logp"] = None
    z = t["logits"].requires_grad_(True)
    r = es.einpolicy("b s v", z, t["ids"], axis="v", advantages=t["advantages"], mask=t["mask"], reduction="sum")
    (got,) = torch.autograd.grad(r.loss, z)
    zd = z.detach().double().requires_grad_(True)
    lp = torch.log_softmax(zd, -1).gather(-1, t["ids"][..., None])[..., 0]
    want = -(torch.where(t["mask"], t["advantages"].double() * lp, 0)).sum()
    (ref,) = torch.autograd.grad(want, zd)
    assert torch.allclose(got.double(), ref, atol=2e-6)
    assert torch.allclose(r.loss.double(), -torch.where(t["mask"], t["advantages"], 0).double().sum(), atol=1e-5)
    assert float(r.kl) == 0 and float(r.clipped) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_no_mask(device):
    t = off_border(make(device, torch.float32, 2, 9, 50), 0.2, 0.2)
    t["mask"] = None
    check(t)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum"])
def test_masked_tokens_may_hold_anything(device, dtype, reduction):
    t = off_border(make(device, dtype, 4, 6, 37), 0.2, 0.2)
    t["mask"][1] = False  # a sequence with no token at all
    t["mask"][2] = True
    gone = ~t["mask"]
    t["logits"][gone] = float("nan")
    t["logits"][1, 0] = float("inf")
    t["logits"][1, 1] = -float("inf")
    t["ids"] = torch.where(gone, torch.tensor([-100, 10 ** 12, 37], device=device)[torch.arange(6, device=device) % 3], t["ids"])
    for k in ("old_logp", "ref_logp", "advantages"):
        t[k] = torch.where(gone, torch.tensor([float("nan"), float("inf"), -float("inf")], device=device)[torch.arange(6, device=device) % 3], t[k])
    check(t, reduction=reduction)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum"])
def test_nothing_kept(device, reduction):
    t = make(device, torch.float32, 2, 3, 10)
    t["mask"][:] = False
    z = t["logits"].requires_grad_(True)
    r = es.einpolicy("b s v", z, t["ids"], axis="v", advantages=t["advantages"], old_logp=t["old_logp"],
                     mask=t["mask"], reduction=reduction)
    (g,) = torch.autograd.grad(r.loss, z)
    assert float(r.loss) == 0 and not g.any() and not r.logp.any()
    r = es.einpolicy("b s v", z[:, :0], t["ids"][:, :0], axis="v", advantages=t["advantages"][:, 0], reduction=reduction)
    (g,) = torch.autograd.grad(r.loss, z)
    assert float(r.loss) == 0 and r.logp.shape == (2, 0) and not g.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_banned_and_extreme_logits(device, dtype):
    t = make(device, dtype, 3, 6, 130)
    low = torch.finfo(dtype).min
    hit = t["ids"]
    other = (hit + 1) % 130
    z = t["logits"]
    z[0, 0] = -float("inf")          # everything but the sampled token is banned
    z[0, 0, hit[0, 0]] = 1.0
    z[0, 1, 64:] = -float("inf")
    z[0, 1, hit[0, 1]] = 0.5
    z[0, 2] = low                    # the type's lowest value everywhere: uniform
    z[0, 3, :] = low
    z[0, 3, hit[0, 3]] = 2.0
    z[0, 3, other[0, 3]] = 2.0
    z[1, 0, other[1, 0]] = 40.0      # the sampled token is very unlikely
    z[1, 1, hit[1, 1]] = 40.0        # and nearly certain
    z[1, 2] = torch.finfo(dtype).max / 4
    t["mask"][:] = True
    lp = torch.log_softmax(z.double(), -1).gather(-1, hit[..., None])[..., 0]
    assert torch.isfinite(lp).all()
    t["old_logp"] = (lp + 0.1).float()
    t["ref_logp"] = (lp - 0.2).float()
    zr = z.clone().requires_grad_(True)
    r = es.einpolicy("b s v", zr, hit, axis="v", advantages=t["advantages"], old_logp=t["old_logp"],
                     ref_logp=t["ref_logp"], mask=t["mask"], kl=0.1)
    (g,) = torch.autograd.grad(r.loss, zr)
    assert torch.allclose(r.logp.double(), lp, rtol=1e-6, atol=1e-5)
    assert torch.isfinite(g).all()
    want = oracle(t, 0.2, 0.2, 0.1, 1.0, "mean")[4]
    keep = torch.isfinite(z.double().cpu())
    assert torch.allclose(g.double().cpu()[keep], want[keep], rtol=half_step(dtype) * 1.01, atol=2e-5)
    assert not g.cpu()[~keep].any()


@pytest.mark.parametrize("device", DEVICES)
def test_bad_ids_and_logits_are_not_hidden(device):
    t = make(device, torch.float32, 2, 4, 12)
    t["mask"][:] = True
    for bad in (-1, 12, -100):
        ids = t["ids"].clone()
        ids[1, 2] = bad
        z = t["logits"].clone().requires_grad_(True)
        r = es.einpolicy("b s v", z, ids, axis="v", advantages=t["advantages"], old_logp=t["old_logp"], mask=t["mask"])
        assert torch.isnan(r.loss) and torch.isnan(r.logp[1, 2]) and torch.isfinite(r.logp[0]).all()
        (g,) = torch.autograd.grad(r.loss, z)
        assert torch.isfinite(g[0]).all()
    z = t["logits"].clone()
    z[0, 1, 3] = float("nan")
    r = es.einpolicy("b s v", z, t["ids"], axis="v", advantages=t["advantages"], old_logp=t["old_logp"])
    assert torch.isnan(r.loss) and torch.isnan(r.logp[0, 1])


@pytest.mark.parametrize("device", DEVICES)
def test_bad_tokens_without_advantage(device):
    """An advantage of 0 weighs nothing, but an id outside the vocabulary or a NaN logit still shows."""
    t = make(device, torch.float32, 2, 4, 12)
    t["mask"][:] = True
    t["advantages"][1] = 0
    for fault in ("id", "logit"):
        ids, z = t["ids"].clone(), t["logits"].clone()
        if fault == "id":
            ids[1, 2] = 12
        else:
            z[1, 2, 3] = float("nan")
        z.requires_grad_(True)
        for old in (t["old_logp"], None):
            r = es.einpolicy("b s v", z, ids, axis="v", advantages=t["advantages"], old_logp=old, mask=t["mask"])
            assert torch.isnan(r.loss) and torch.isnan(r.logp[1, 2]) and torch.isfinite(r.logp[0]).all()
    # a ratio past 32 bits times 0 is 0
    r = es.einpolicy("b s v", t["logits"], t["ids"], axis="v", advantages=0 * t["advantages"],
                     old_logp=t["old_logp"] - 200, mask=t["mask"])
    assert float(r.loss) == 0


def negated(t):
    """-t as a view that only says so (what the imaginary part of a conjugate is)."""
    return torch._neg_view(t.detach())


@pytest.mark.parametrize("device", DEVICES)
def test_negated_views(device):
    """Inputs and gradients whose sign is kept beside their memory."""
    t = off_border(make(device, torch.float32, 2, 9, 40), 0.2, 0.2)
    results = []
    for sign in (torch.neg, negated):
        u = {k: sign(-v) if v.is_floating_point() else v for k, v in t.items()}
        z = u.pop("logits").detach().requires_grad_(True)
        for upstream in (torch.ones((), device=device), sign(torch.ones((), device=device))):
            r = es.einpolicy("b s v", z, axis="v", kl=0.1, **u)
            results.append([r.loss.detach(), r.logp, torch.autograd.grad(r.loss, z, upstream)[0]])
        with torch.no_grad():
            results[-1].append(es.einpolicy("b s v", z, axis="v", kl=0.1, **u).loss)
    for got, want in zip(results[2:], results[:2]):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_axes_and_strides(device):
    t = off_border(make(device, torch.float32, 3, 5, 41), 0.2, 0.2)
    args = dict(advantages=t["advantages"], old_logp=t["old_logp"], ref_logp=t["ref_logp"], mask=t["mask"], kl=0.1)

    def both(formula, z, ids, **kw):
        z = z.detach().requires_grad_(True)
        r = es.einpolicy(formula, z, ids, axis="v", **kw)
        return r, torch.autograd.grad(r.loss, z)[0]

    r, g = both("b s v", t["logits"], t["ids"], **args)
    r2, g2 = both("b v s", t["logits"].transpose(1, 2).contiguous(), t["ids"], **args)
    assert torch.allclose(r.loss, r2.loss) and torch.allclose(g, g2.transpose(1, 2), atol=1e-7)
    wide = torch.zeros(3, 5, 60, device=device)
    for off in (0, 1, 4, 7):
        wide[..., off:off + 41] = t["logits"]
        r2, g2 = both("b s v", wide[..., off:off + 41], t["ids"].int(), **args)
        assert torch.allclose(r.loss, r2.loss) and torch.allclose(g, g2, atol=1e-7)
    swapped = {k: (v.transpose(0, 1).contiguous().transpose(0, 1) if torch.is_tensor(v) else v) for k, v in args.items()}
    r2, g2 = both("b s v", t["logits"].transpose(0, 1).contiguous().transpose(0, 1), t["ids"], **swapped)
    assert torch.allclose(r.loss, r2.loss) and torch.allclose(g, g2, atol=1e-7)
    one = {k: (v[0] if torch.is_tensor(v) else v) for k, v in args.items()}
    r1, _ = both("s v", t["logits"][0], t["ids"][0], **one)
    scalar = {k: (v[0, 0] if torch.is_tensor(v) else v) for k, v in args.items()}
    scalar["mask"] = None
    r0, _ = both("v", t["logits"][0, 0], t["ids"][0, 0], **scalar)
    assert r1.logp.shape == (5,) and r0.logp.shape == ()
    # three leading axes: sequences are all but the last one
    four = {k: (v.view(3, 1, 5) if torch.is_tensor(v) else v) for k, v in args.items()}
    r4, _ = both("a b s v", t["logits"].view(3, 1, 5, 41), t["ids"].view(3, 1, 5), **four, reduction="sequence")
    r5, _ = both("b s v", t["logits"], t["ids"], **args, reduction="sequence")
    assert torch.allclose(r4.loss, r5.loss)


def test_against_differences():
    t = off_border(make("cpu", torch.float64, 2, 3, 5), 0.2, 0.3)
    z = t.pop("logits").requires_grad_(True)
    for k in ("old_logp", "ref_logp", "advantages"):
        t[k] = t[k].double()
    for reduction in ("mean", "sequence", "sum"):
        assert torch.autograd.gradcheck(
            lambda z: es.einpolicy("b s v", z, axis="v", clip=(0.2, 0.3), kl=0.1, temperature=0.8,
                                   reduction=reduction, **t).loss, (z,))


@pytest.mark.gpu
def test_against_differences_on_the_kernels():
    """Central differences of the kernel's 32-bit loss along random directions: third-order error at a step of
    1e-2, and roundings of 2^-23 over it."""
    t = off_border(make("cuda", torch.float32, 2, 9, 64), 0.2, 0.2)
    z = t.pop("logits").requires_grad_(True)

    def f(z):
        return es.einpolicy("b s v", z, axis="v", kl=0.1, reduction="sum", **t).loss

    (g,) = torch.autograd.grad(f(z), z)
    gen = torch.Generator().manual_seed(3)
    for _ in range(8):
        v = torch.randn(z.shape, generator=gen).cuda()
        v /= v.norm()
        diff = (f(z.detach() + 1e-2 * v).double() - f(z.detach() - 1e-2 * v).double()) / 2e-2
        assert abs(float(diff - (g * v).sum())) <= 2e-3 * float(g.norm()) + 2e-3


@pytest.mark.parametrize("device", DEVICES)
def test_backward_twice_and_beside_another_loss(device):
    t = off_border(make(device, torch.bfloat16, 2, 9, 130), 0.2, 0.2)
    z = t.pop("logits").requires_grad_(True)
    loss = es.einpolicy("b s v", z, axis="v", kl=0.1, **t).loss
    (g1,) = torch.autograd.grad(loss, z, retain_graph=True)
    held = g1.clone()
    (g2,) = torch.autograd.grad(2 * loss, z, retain_graph=True)
    (g3,) = torch.autograd.grad(loss, z)
    assert torch.equal(g1, held) and torch.equal(g3, held) and torch.equal(g2, 2 * held)
    loss = es.einpolicy("b s v", z, axis="v", kl=0.1, **t).loss
    (g4,) = torch.autograd.grad(loss + z.float().sum(), z)
    assert torch.allclose(g4.float(), held.float() + 1, atol=2.0 ** -8)
    if device == "cuda":  # the kernels read the logits again: changed between the passes, they are refused
        y = z.detach().clone().requires_grad_(True)
        w = y * 1
        loss = es.einpolicy("b s v", w, axis="v", **t).loss
        w.add_(1)
        with pytest.raises(RuntimeError):
            loss.backward()
    with torch.no_grad():
        assert not es.einpolicy("b s v", z, axis="v", **t).loss.requires_grad


@pytest.mark.gpu
def test_no_second_derivative():
    t = off_border(make("cuda", torch.float32, 2, 5, 40), 0.2, 0.2)
    z = t.pop("logits").requires_grad_(True)
    (g,) = torch.autograd.grad(es.einpolicy("b s v", z, axis="v", **t).loss, z, create_graph=True)
    assert torch.equal(g.detach(), torch.autograd.grad(es.einpolicy("b s v", z, axis="v", **t).loss, z)[0])
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(g.sum(), z, allow_unused=True)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["logits", "old_logp", "ref_logp", "advantages"])
def test_forward_mode(device, which):
    """Torch's path carries tangents; the kernels have none and say so."""
    t = off_border(make(device, torch.float32, 2, 5, 40), 0.2, 0.2)
    gen = torch.Generator().manual_seed(2)
    v = torch.randn(t[which].shape, generator=gen).to(t[which])
    with forward_ad.dual_level():
        u = {**t, which: forward_ad.make_dual(t[which], v)}
        z = u.pop("logits")
        if device == "cuda":
            with pytest.raises(NotImplementedError, match="forward-mode"):
                es.einpolicy("b s v", z, axis="v", kl=0.1, **u)
            return
        tangent = forward_ad.unpack_dual(es.einpolicy("b s v", z, axis="v", kl=0.1, **u).loss).tangent
        assert tangent is not None
    if which == "logits":
        z = t.pop("logits").requires_grad_(True)
        (g,) = torch.autograd.grad(es.einpolicy("b s v", z, axis="v", kl=0.1, **t).loss, z)
        assert torch.allclose(tangent, (g * v).sum(), rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    t = make(device, torch.float32, 2, 3, 8)
    z, ids, adv = t["logits"], t["ids"], t["advantages"]
    ok = dict(axis="v", advantages=adv)
    for error, formula, logits, i, kw in [
        (ValueError, "b s", z, ids, ok),
        (ValueError, "b s v", z, ids, dict(ok, axis="w")),
        (ValueError, "b b v", z, ids, ok),
        (ValueError, "b s v // tp", z, ids, ok),
        (NotImplementedError, "b s v/tp", z, ids, ok),
        (NotImplementedError, "b/dp s v", z, ids, ok),
        (NotImplementedError, "... v", z, ids, ok),
        (NotImplementedError, "b (s v)", z.view(2, 24), ids, ok),
        (TypeError, "b s v", z.long(), ids, ok),
        (ValueError, "b s v", z[..., :0], ids, ok),
        (ValueError, "b s v", z, ids.float(), ok),
        (ValueError, "b s v", z, ids[:, :2], ok),
        (ValueError, "b s v", z, ids, dict(ok, mask=t["mask"].float())),
        (ValueError, "b s v", z, ids, dict(ok, mask=t["mask"][:1])),
        (ValueError, "b s v", z, ids, dict(ok, advantages=adv[:, :1])),
        (ValueError, "b s v", z, ids, dict(ok, advantages=ids)),
        (ValueError, "b s v", z, ids, dict(ok, advantages=adv.clone().requires_grad_(True))),
        (ValueError, "b s v", z, ids, dict(ok, old_logp=t["old_logp"][0])),
        (ValueError, "b s v", z, ids, dict(ok, old_logp=t["old_logp"].clone().requires_grad_(True))),
        (ValueError, "b s v", z, ids, dict(ok, kl=0.1)),
        (ValueError, "b s v", z, ids, dict(ok, kl=-0.1, ref_logp=t["ref_logp"])),
        (ValueError, "b s v", z, ids, dict(ok, clip=1.5)),
        (ValueError, "b s v", z, ids, dict(ok, clip=(0.2, -0.1))),
        (ValueError, "b s v", z, ids, dict(ok, temperature=0.0)),
        (ValueError, "b s v", z, ids, dict(ok, reduction="none")),
        (ValueError, "b s v", z, ids, dict(ok, weight=float("nan"))),
    ]:
        with pytest.raises(error):
            es.einpolicy(formula, logits, i, **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_weight(device):
    t = off_border(make(device, torch.bfloat16, 2, 9, 130), 0.2, 0.2)
    check(t, weight=0.25)
    check(t, weight=-3.0, upstream=0.5, reduction="sequence")


@pytest.mark.gpu
def test_other_stream_and_capture():
    t = off_border(make("cuda", torch.bfloat16, 2, 33, 1001), 0.2, 0.2)
    z = t.pop("logits")

    def step(z, factor=None):
        r = es.einpolicy("b s v", z, axis="v", kl=0.1, **t)
        return r.loss.detach(), r.logp, torch.autograd.grad(r.loss, z, factor)[0]

    want = step(z.clone().requires_grad_(True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(z.clone().requires_grad_(True))
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # graphs of the whole step, replayed in turn with other logits and other upstream gradients
    leaves = [z.clone().requires_grad_(True) for _ in range(2)]
    factor = torch.ones((), device="cuda")
    graphs = []
    for leaf in leaves:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(leaf, factor)
        graphs.append((graph, out))
    other = torch.randn(z.shape, generator=torch.Generator().manual_seed(9)).to(z)
    for value, scale in ((z, 1.0), (other, 0.5), (z, 2.0), (other, 1.0)):
        factor.fill_(scale)
        for leaf, (graph, _) in zip(leaves, graphs):
            with torch.no_grad():
                leaf.copy_(value)
            graph.replay()
        want = step(value.clone().requires_grad_(True), factor)
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_backward_captured_apart_from_forward(dtype):
    """An eager forward pass, its backward pass captured and replayed with other upstream gradients; and a captured
    forward pass with an eager backward pass, whose result a later replay leaves alone."""
    t = off_border(make("cuda", dtype, 2, 9, 130), 0.2, 0.2)
    z = t.pop("logits").requires_grad_(True)
    factor = torch.ones((), device="cuda")

    def gradient(scale):
        loss = es.einpolicy("b s v", z, axis="v", kl=0.1, **t).loss
        return torch.autograd.grad(loss, z, torch.tensor(scale, device="cuda"))[0]

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        loss = es.einpolicy("b s v", z, axis="v", kl=0.1, **t).loss
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (g,) = torch.autograd.grad(loss, z, factor)
    for scale in (0.5, 1.0, 1.0, 2.0, 0.0, 1.0):
        factor.fill_(scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, gradient(scale))
    del loss
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = es.einpolicy("b s v", z, axis="v", kl=0.1, **t).loss
    graph.replay()
    torch.cuda.synchronize()
    (g,) = torch.autograd.grad(loss, z, retain_graph=True)
    want = gradient(1.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(g, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_forward_and_backward_in_graphs_of_their_own(dtype):
    """The backward graph's result is its own: a replay of the forward graph leaves it alone, and so does a caller who
    changes it in place."""
    t = off_border(make("cuda", dtype, 2, 9, 130), 0.2, 0.2)
    values = [t.pop("logits")]
    values.append(torch.randn(values[0].shape, generator=torch.Generator().manual_seed(9)).to(values[0]))
    z = values[0].clone().requires_grad_(True)

    def gradient(value):
        leaf = value.clone().requires_grad_(True)
        return torch.autograd.grad(es.einpolicy("b s v", leaf, axis="v", kl=0.1, **t).loss, leaf)[0]

    want = [gradient(v) for v in values]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=side):
        loss = es.einpolicy("b s v", z, axis="v", kl=0.1, **t).loss
    with torch.cuda.graph(backward, stream=side):
        (g,) = torch.autograd.grad(loss, z)

    def replay(i):
        with torch.no_grad():
            z.copy_(values[i])
        forward.replay()
        backward.replay()
        torch.cuda.synchronize()

    replay(0)
    assert torch.equal(g, want[0])
    with torch.no_grad():
        z.copy_(values[1])
    forward.replay()
    torch.cuda.synchronize()
    assert torch.equal(g, want[0])
    backward.replay()
    torch.cuda.synchronize()
    assert torch.equal(g, want[1])
    g.mul_(3)
    backward.replay()
    torch.cuda.synchronize()
    assert torch.equal(g, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [(1, 16385), (4100, 5), (3, 7001)])
@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum"])
def test_many_tokens(tokens, reduction):
    check(off_border(make("cuda", torch.float32, *tokens, 40, advantage="sequence"), 0.2, 0.2), reduction=reduction)


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
def test_transformer_policy_step(one_rank_mesh):
    """The three operators together: sandwich norms, 8-bit operands and the policy loss in one training step."""
    device, mesh = one_rank_mesh
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    gen = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 97, (3, 16), generator=gen).to(device)
    mask = (torch.arange(15)[None] >= torch.tensor([[3], [5], [20]])).to(device)  # the last answer is empty
    adv = torch.randn(3, generator=gen).to(device)
    grads = []
    for checkpoint in (False, "int8"):
        cfg = TransformerConfig(layers=2, d=64, heads=4, mlp=128, vocab=97, seq=16, dtype=dtype, norm="sandwich")
        model = TPTransformer(cfg, mesh, device=device, checkpoint=checkpoint)
        with torch.no_grad():
            first = model.policy_loss(tokens, advantages=adv, mask=mask)
            logits = model(tokens[:, :-1]).float()
        lp = torch.log_softmax(logits, -1).gather(-1, tokens[:, 1:, None])[..., 0]
        assert torch.allclose(first.logp, torch.where(mask, lp, 0), atol=1e-4)
        r = model.policy_loss(tokens, advantages=adv, mask=mask, old_logp=first.logp + 0.1, ref_logp=first.logp - 0.1,
                              kl=0.05, reduction="sequence")
        r.loss.backward()
        grads.append([p.grad.float() for p in model.parameters()])
        assert all(torch.isfinite(g).all() for g in grads[-1])
    for a, b in zip(*grads):
        assert (a - b).norm() <= 0.06 * a.norm() + 1e-6


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("base", [-1e10, 1e10, -1e9, -3.0e7, 5.0e6, -5.0e6, 2.9e6, -2.9e6, 2907269.0, -2907270.0, 1e4])
def test_rows_far_from_zero(device, dtype, base):
    """A row is known by its differences: mask values and offsets of any size leave them alone.

    The differences of these logits are exact in 32 bits; each is scaled with one rounding, and the exponentials are
    2^-21 off."""
    gen = torch.Generator().manual_seed(3)
    z = torch.full((1, 6, 301), base, dtype=torch.float64)
    z[0, 1] += torch.randn(301, generator=gen).double()
    z[0, 2] += 4 * torch.randn(301, generator=gen).double()
    z[0, 3, :150] = 0.0
    z[0, 4] = torch.randn(301, generator=gen).double()
    z[0, 4, 7] = base
    z[0, 5, 9:] = -1e30
    z = z.to(dtype)
    t = make(device, dtype, 1, 6, 301)
    t["logits"] = z.to(device)
    t["ids"] = torch.tensor([[3, 5, 7, 11, 13, 2]], device=device)
    want = torch.log_softmax(z.double(), -1).gather(-1, t["ids"].cpu()[..., None])[..., 0]
    kept = want.abs() < 200  # further down 32 bits hold no ratio: old_logp's own rounding is more than 1e-5
    t["mask"] = kept.to(device)
    want = torch.where(kept, want, 0)
    t["old_logp"] = (want + 0.1).float().to(device)
    t["ref_logp"] = (want - 0.1).float().to(device)
    logits = t["logits"].requires_grad_(True)
    r = es.einpolicy("b s v", logits, t["ids"], axis="v", advantages=t["advantages"], old_logp=t["old_logp"],
                     mask=t["mask"], ref_logp=t["ref_logp"], kl=0.1)
    far = torch.where(kept, z.double().amax(-1) - z.double().gather(-1, t["ids"].cpu()[..., None])[..., 0], 0)
    assert ((r.logp.double().cpu() - want).abs() <= 2.0 ** -19 + 2.0 ** -22 * (far + want.abs())).all()
    (grad,) = torch.autograd.grad(r.loss, logits)
    ratio = torch.exp(want - t["old_logp"].double().cpu())
    adv = t["advantages"].double().cpu()
    slope = torch.where(ratio * adv <= ratio.clamp(0.8, 1.2) * adv, -ratio * adv, 0)
    slope = (slope + 0.1 * (1 - torch.exp(t["ref_logp"].double().cpu() - want))) / kept.sum() * kept
    hit = torch.zeros(1, 6, 301, dtype=torch.float64).scatter_(-1, t["ids"].cpu()[..., None], 1.0)
    p = torch.softmax(z.double(), -1)
    exact = slope[..., None] * (hit - p)
    # ratio (at most 1.2) and p follow the log-probability's error
    err = 2.0 ** -18 + 2.0 ** -21 * (far + want.abs())[..., None]
    bound = half_step(dtype) * exact.abs() + err * (hit + p) * (1.2 * adv.abs() + 0.2)[..., None] + 1e-30
    assert ((grad.double().cpu() - exact).abs() <= bound).all()
