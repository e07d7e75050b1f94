"""Workloads of the training step's operators around the contractions.

* ``norm``   - ``einnorm``: the norm after a block, its gate, the scaled residual stream and the norm before
               the next block (forward, and forward + backward).
* ``save``, ``linear``, ``mlp`` - ``checkpoint8``: activations kept for backward in 8 bits, and the products
               whose weight gradients read them back.
* ``policy`` - ``einpolicy``: the clipped policy loss with a KL term from logits (forward, and forward + backward).

With ``own`` false every operator is computed in its plain form, elementary torch operations in 32 bits; with
``own`` true the same inputs go through ``torch_einshard_b200``.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 32  # channels that share one exponent


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one new token of four sequences through a block's residual and norms, no gradients: launch latency
        dict(name="norm_step", op="norm", b=4, s=1, d=2048, dtype="bf16", kind="rms", post=True, gate="channel",
             scale=1.0, train=False),
        # the training transformer's width and length: both norms, a gate per channel
        dict(name="norm_train", op="norm", b=1, s=8192, d=2048, dtype="bf16", kind="layer", post=True,
             gate="channel", scale=1.0, train=True),
        # a wide stream, a gate per sequence and channel (conditioning), ragged row count; the largest of its kind
        dict(name="norm_wide", op="norm", b=7, s=2341, d=8192, dtype="bf16", kind="rms", post=True, gate="batch",
             scale=0.75, train=True),
        # fp32, odd width, a gate for every token, no norm after the block
        dict(name="norm_odd", op="norm", b=3, s=1777, d=1001, dtype="fp32", kind="layer", post=False, gate="token",
             scale=1.0, train=True),
        # a short batch kept in 8 bits and read back: launch latency
        dict(name="save_small", op="save", b=2, s=96, d=2048, dtype="bf16"),
        # a long batch of an odd width: the last block of a row is short and rows are not aligned
        dict(name="save_odd", op="save", b=4, s=6001, d=8191, dtype="fp16"),
        # one normed stream kept once in 8 bits for the three projections that read it, with gradients
        dict(name="linear_qkv", op="linear", b=1, s=8192, c=2048, n=2048, outs=3, dtype="bf16"),
        # the training transformer's MLP: input and pre-activation kept in 8 bits, with gradients; the largest case
        dict(name="mlp_train", op="mlp", b=4, s=8192, c=2048, h=8192, dtype="bf16"),
        # one short sequence: a step of on-policy training on 33 tokens, prompt masked
        dict(name="policy_small", op="policy", b=1, s=33, v=32000, dtype="bf16", lo=0.2, hi=0.2, kl=0.05, temp=1.0,
             reduction="mean", advantage="sequence", train=True),
        # the training transformer's vocabulary: a batch of ragged answers behind their prompts
        dict(name="policy_train", op="policy", b=8, s=1024, v=32000, dtype="bf16", lo=0.2, hi=0.28, kl=0.02,
             temp=1.0, reduction="sequence", advantage="sequence", train=True),
        # no gradients (a monitor of the same loss), fp32 logits, a vocabulary of odd size
        dict(name="policy_eval", op="policy", b=4, s=1021, v=50257, dtype="fp32", lo=0.2, hi=0.2, kl=0.1, temp=0.7,
             reduction="mean", advantage="token", train=False),
        # a large vocabulary of odd size: rows of logits are not aligned
        dict(name="policy_wide", op="policy", b=6, s=2048, v=128257, dtype="bf16", lo=0.1, hi=0.3, kl=0.0, temp=1.0,
             reduction="sum", advantage="token", train=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width between low and high: half of them multiples of 8, the rest whatever comes."""
    w = _log_int(rng, low, high)
    return max(8, w // 8 * 8) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(["norm", "norm", "save", "linear", "mlp", "policy", "policy"])
    if op == "norm":
        d = _width(rng, 64, 8192)
        b = rng.randint(1, 7)
        s = _log_int(rng, 1, max(1, min(16384, 7 * 2341 * 8192 // (b * d))))
        return dict(op=op, b=b, s=s, d=d, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    kind=rng.choice(["layer", "rms"]), post=rng.random() < 0.7,
                    gate=rng.choice(["none", "channel", "batch", "token"]), scale=rng.choice([1.0, 1.0, 0.5, 1.25]),
                    train=rng.random() < 0.7)
    if op == "save":
        d = _width(rng, 64, 8192)
        b = rng.randint(1, 4)
        s = _log_int(rng, 1, max(1, min(16384, 4 * 6001 * 8191 // (b * d))))
        return dict(op=op, b=b, s=s, d=d, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "linear":
        return dict(op=op, b=rng.randint(1, 3), s=_log_int(rng, 64, 4096), c=_width(rng, 256, 2048),
                    n=_width(rng, 256, 2048), outs=rng.randint(1, 3), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "mlp":
        return dict(op=op, b=rng.randint(1, 4), s=_log_int(rng, 64, 4096), c=_width(rng, 256, 2048),
                    h=_width(rng, 512, 8192), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    v = _width(rng, 1000, 131000)
    b = rng.randint(1, 8)
    s = _log_int(rng, 4, max(4, min(4096, 6 * 2048 * 128257 // (2 * b * v))))
    return dict(op=op, b=b, s=s, v=v, dtype=rng.choice(["bf16", "bf16", "fp32"]), lo=rng.choice([0.1, 0.2]),
                hi=rng.choice([0.2, 0.28, 0.3]), kl=rng.choice([0.0, 0.02, 0.1]), temp=rng.choice([1.0, 1.0, 0.7]),
                reduction=rng.choice(["mean", "sequence", "sum"]), advantage=rng.choice(["sequence", "token"]),
                train=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs

class _Rand:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device="cuda")

    def integer(self, low, high, *shape):
        return torch.randint(low, high, shape, generator=self.gen, device="cuda")


def _stream(rand, b, s, d, dtype):
    """Hidden states: a spread over channels (a few loud ones) and over tokens."""
    channels = torch.exp(0.5 * rand.normal(d))
    return (rand.normal(b, s, d) * channels + 0.1).to(dtype)


def _prepare_norm(case, rand):
    b, s, d, dtype = case["b"], case["s"], case["d"], _DTYPES[case["dtype"]]
    state = dict(x=_stream(rand, b, s, d, dtype), y=_stream(rand, b, s, d, dtype),
                 w=(1 + 0.1 * rand.normal(d)).to(dtype))
    if case["kind"] == "layer":
        state["bias"] = (0.1 * rand.normal(d)).to(dtype)
    if case["post"]:
        state["pw"] = (1 + 0.1 * rand.normal(d)).to(dtype)
        if case["kind"] == "layer":
            state["pb"] = (0.1 * rand.normal(d)).to(dtype)
    shape = {"none": None, "channel": (d,), "batch": (b, d), "token": (b, s, d)}[case["gate"]]
    if shape is not None:
        state["gate"] = (0.5 + 0.3 * rand.normal(*shape)).to(dtype)
    if case["train"]:
        state["leaves"] = [k for k in ("x", "y", "gate", "w", "bias", "pw", "pb") if k in state]
        for k in state["leaves"]:
            state[k].requires_grad_(True)
        state["dh"] = rand.normal(b, s, d).to(dtype)
        state["dn"] = rand.normal(b, s, d).to(dtype)
    return state


def _prepare_linear(case, rand):
    b, s, c, n, dtype = case["b"], case["s"], case["c"], case["n"], _DTYPES[case["dtype"]]
    return dict(x=_stream(rand, b, s, c, dtype).requires_grad_(True),
                w=[(rand.normal(n, c) / math.sqrt(c)).to(dtype).requires_grad_(True) for _ in range(case["outs"])],
                dy=[rand.normal(b, s, n).to(dtype) for _ in range(case["outs"])])


def _prepare_mlp(case, rand):
    b, s, c, h, dtype = case["b"], case["s"], case["c"], case["h"], _DTYPES[case["dtype"]]
    return dict(x=_stream(rand, b, s, c, dtype).requires_grad_(True),
                w1=(rand.normal(h, c) / math.sqrt(c)).to(dtype).requires_grad_(True),
                w2=(rand.normal(c, h) / math.sqrt(h)).to(dtype).requires_grad_(True),
                dy=rand.normal(b, s, c).to(dtype))


def _prepare_policy(case, rand):
    b, s, v = case["b"], case["s"], case["v"]
    logits = torch.empty(b, s, v, dtype=_DTYPES[case["dtype"]], device="cuda")
    ids = rand.integer(0, v, b, s)
    # sampled tokens are likely ones: lift each token's logit above the rest
    lift = 8 + 2 * rand.normal(b, s)
    logp = torch.empty(b, s, device="cuda")
    for i in range(b):
        z = 1.5 * rand.normal(s, v)
        z.scatter_add_(1, ids[i][:, None], lift[i][:, None])
        logits[i] = z.to(logits.dtype)
        z = logits[i].double() if s * v <= 1 << 28 else logits[i].float()
        z = z / case["temp"]
        logp[i] = (z.gather(1, ids[i][:, None])[:, 0] - torch.logsumexp(z, 1)).float()
    old = logp + 0.15 * rand.normal(b, s)
    # a ratio on the border of the clip range has no side that rounding could not change: keep clear of it
    for border in (1 - case["lo"], 1 + case["hi"]):
        near = (torch.exp(logp - old) - border).abs() < 1e-3
        old = torch.where(near, old - 0.01, old)
    # answers start behind a prompt and end before the row's end; a group of padding tokens has id -100
    start = rand.integer(0, max(1, s // 3), b, 1)
    stop = rand.integer(max(1, s // 2), s + 1, b, 1)
    pos = torch.arange(s, device="cuda")[None]
    mask = (pos >= start) & (pos < stop)
    shape = (b,) if case["advantage"] == "sequence" else (b, s)
    return dict(logits=logits.requires_grad_(case["train"]), ids=torch.where(mask, ids, -100), old=old,
                ref=logp + 0.3 * rand.normal(b, s), adv=rand.normal(*shape), mask=mask)


def prepare(case, seed):
    rand = _Rand(seed)
    op = case["op"]
    if op == "norm":
        state = _prepare_norm(case, rand)
    elif op == "save":
        state = dict(x=_stream(rand, case["b"], case["s"], case["d"], _DTYPES[case["dtype"]]).requires_grad_(True))
    elif op == "linear":
        state = _prepare_linear(case, rand)
    elif op == "mlp":
        state = _prepare_mlp(case, rand)
    else:
        state = _prepare_policy(case, rand)
    state["case"] = case
    return state


# ------------------------------------------------------------------------------------------------ plain forms

def _norm_plain(x, kind, w, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w
    return y if bias is None else y + bias


def _wide_gate(gate):
    """The gate in the stream's rank: [b, d] is one row for a whole sequence."""
    return gate[:, None] if gate.dim() == 2 else gate


def _plain_norm(state):
    case = state["case"]
    keys = [k for k in ("x", "y", "gate", "w", "bias", "pw", "pb") if k in state]
    with torch.enable_grad():
        t = {k: state[k].detach().float().requires_grad_(case["train"]) for k in keys}
        p = _norm_plain(t["y"], case["kind"], t["pw"], t.get("pb")) if case["post"] else t["y"]
        if "gate" in t:
            p = _wide_gate(t["gate"]) * p
        h = case["scale"] * t["x"] + p
        n = _norm_plain(h, case["kind"], t["w"], t.get("bias"))
        dtype = state["x"].dtype
        out = dict(h=h.detach().to(dtype), n=n.detach().to(dtype))
        if case["train"]:
            grads = torch.autograd.grad((h, n), [t[k] for k in keys], (state["dh"].float(), state["dn"].float()))
            out.update({"d" + k: g.to(state[k].dtype) for k, g in zip(keys, grads)})
    return out


def _round8(x):
    """x (fp32) as what its 8-bit form stands for: blocks of 32 channels share a power of two 2^e, the smallest
    for which every rounded multiple of it fits in -127 .. 127."""
    d = x.shape[-1]
    blocks = torch.nn.functional.pad(x, (0, -d % _BLOCK)).unflatten(-1, (-1, _BLOCK))
    amax = blocks.abs().amax(-1, keepdim=True)
    e = ((amax.contiguous().view(torch.int32) >> 23) - 127 - 6).clamp(min=-126)  # floor(log2 amax) - 6
    e = e + (torch.round(torch.ldexp(amax, -e)) > 127)
    q = torch.round(torch.ldexp(torch.ldexp(blocks, -(e // 2)), -(e - e // 2)))
    return torch.ldexp(torch.ldexp(q, e // 2), e - e // 2).flatten(-2)[..., :d]


def _plain_save(state):
    x = state["x"].detach()
    limit = torch.finfo(x.dtype).max
    return _round8(x.float()).clamp(-limit, limit).to(x.dtype)


def _plain_linear(state):
    x = state["x"].detach()
    xf = x.float().flatten(0, 1)
    kept = _round8(xf)
    dx = 0
    out = {}
    for i, (w, dy) in enumerate(zip(state["w"], state["dy"])):
        wf, dyf = w.detach().float(), dy.float().flatten(0, 1)
        out[f"y{i}"] = (xf @ wf.t()).view(dy.shape).to(x.dtype)
        out[f"dw{i}"] = (dyf.t() @ kept).to(x.dtype)
        dx = dx + dyf @ wf
    out["dx"] = dx.view(x.shape).to(x.dtype)
    return out


def _plain_mlp(state):
    x = state["x"].detach()
    xf, w1, w2 = x.float().flatten(0, 1), state["w1"].detach().float(), state["w2"].detach().float()
    dy = state["dy"].float().flatten(0, 1)
    pre = xf @ w1.t()
    y = (pre / (1 + torch.exp(-pre))) @ w2.t()
    pre = _round8(pre)
    sig = 1 / (1 + torch.exp(-pre))
    dw2 = dy.t() @ (pre * sig)
    dpre = (dy @ w2) * (sig * (1 + pre * (1 - sig)))
    return dict(y=y.view(x.shape).to(x.dtype), dx=(dpre @ w1).view(x.shape).to(x.dtype),
                dw1=(dpre.t() @ _round8(xf)).to(x.dtype), dw2=dw2.to(x.dtype))


def _policy_terms(lp, old, ref, adv, mask, case):
    """Loss, KL term and clipped share (each reduced as the case says) from the tokens' log-probabilities."""
    ratio = torch.exp(lp - old)
    fixed = torch.clamp(ratio, 1 - case["lo"], 1 + case["hi"])
    gain = torch.minimum(ratio * adv, fixed * adv)
    far = ref - lp
    kl = torch.exp(far) - far - 1
    clipped = (ratio * adv > fixed * adv).to(lp.dtype)

    def reduced(t):
        t = torch.where(mask, t, 0)
        count = mask.sum(-1)
        if case["reduction"] == "sum":
            return t.sum()
        if case["reduction"] == "mean":
            return t.sum() / count.sum().clamp(min=1)
        return (t.sum(-1) / count.clamp(min=1)).sum() / (count > 0).sum().clamp(min=1)

    return reduced(-gain + case["kl"] * kl), reduced(kl), reduced(clipped)


def _plain_policy(state):
    case, mask = state["case"], state["mask"]
    adv = state["adv"][:, None] if state["adv"].dim() == 1 else state["adv"]
    with torch.enable_grad():
        z32 = state["logits"].detach().float().requires_grad_(case["train"])
        z = z32 / case["temp"]
        top = z.detach().amax(-1, keepdim=True)
        lse = torch.log(torch.exp(z - top).sum(-1)) + top[..., 0]
        lp = z.gather(-1, state["ids"].clamp(min=0)[..., None])[..., 0] - lse
        lp = torch.where(mask, lp, 0)
        loss, kl, clipped = _policy_terms(lp, state["old"], state["ref"], adv, mask, case)
        out = dict(loss=loss.detach(), logp=lp.detach(), kl=kl.detach(), clipped=clipped.detach())
        if case["train"]:
            out["dlogits"] = torch.autograd.grad(loss, z32)[0].to(state["logits"].dtype)
    return out


# ------------------------------------------------------------------------------------------------ the framework

def _own_norm(state):
    import torch_einshard_b200 as es
    case = state["case"]
    axes = {"none": None, "channel": "d", "batch": "b d", "token": "b s d"}[case["gate"]]
    with torch.set_grad_enabled(case["train"]):
        h, n = es.einnorm("b s d", state["x"], state["y"], axis="d", kind=case["kind"], weight=state["w"],
                          bias=state.get("bias"), post=case["post"], post_weight=state.get("pw"),
                          post_bias=state.get("pb"), gate=state.get("gate"), gate_axes=axes, scale=case["scale"])
        out = dict(h=h.detach(), n=n.detach())
        if case["train"]:
            keys = state["leaves"]
            grads = torch.autograd.grad((h, n), [state[k] for k in keys], (state["dh"], state["dn"]))
            out.update({"d" + k: g for k, g in zip(keys, grads)})
    return {k: out[k] for k in _norm_keys(state)}


def _norm_keys(state):
    return ["h", "n"] + ["d" + k for k in state.get("leaves", ())]


def _own_save(state):
    import torch_einshard_b200 as es
    return es.checkpoint8(state["x"]).restore()


def _own_linear(state):
    import torch_einshard_b200 as es
    x = es.checkpoint8(state["x"])
    ys = [es.einshard("b s c, n c -> b s n", x, w) for w in state["w"]]
    grads = torch.autograd.grad(ys, [state["x"], *state["w"]], state["dy"])
    out = {}
    for i, y in enumerate(ys):
        out[f"y{i}"] = y.detach()
        out[f"dw{i}"] = grads[1 + i]
    out["dx"] = grads[0]
    return out


def _own_mlp(state):
    import torch_einshard_b200 as es
    x = es.checkpoint8(state["x"])
    a = es.einshard("b s c, h c -> b s h", x, state["w1"], activation="silu")
    y = es.einshard("b s h, c h -> b s c", a, state["w2"])
    dx, dw1, dw2 = torch.autograd.grad(y, [state["x"], state["w1"], state["w2"]], state["dy"])
    return dict(y=y.detach(), dx=dx, dw1=dw1, dw2=dw2)


def _own_policy(state):
    import torch_einshard_b200 as es
    case = state["case"]
    with torch.set_grad_enabled(case["train"]):
        r = es.einpolicy("b s v", state["logits"], state["ids"], axis="v", old_logp=state["old"],
                         advantages=state["adv"], ref_logp=state["ref"], mask=state["mask"],
                         clip=(case["lo"], case["hi"]), kl=case["kl"], temperature=case["temp"],
                         reduction=case["reduction"])
        out = dict(loss=r.loss.detach(), logp=r.logp, kl=r.kl, clipped=r.clipped)
        if case["train"]:
            out["dlogits"] = torch.autograd.grad(r.loss, state["logits"])[0]
    return out


_PLAIN = dict(norm=_plain_norm, save=_plain_save, linear=_plain_linear, mlp=_plain_mlp, policy=_plain_policy)
_OWN = dict(norm=_own_norm, save=_own_save, linear=_own_linear, mlp=_own_mlp, policy=_own_policy)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ work

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "norm":
        n = case["b"] * case["s"] * case["d"]
        gate = {"none": 0, "channel": case["d"], "batch": case["b"] * case["d"], "token": n}[case["gate"]]
        params = case["d"] * (1 + (case["kind"] == "layer")) * (1 + case["post"]) + gate
        streams = 8 if case["train"] else 4  # x, y -> h, n; with dh, dn -> dx, dy
        return dict(bytes=size * (streams * n + params * (2 if case["train"] else 1)),
                    flops=n * (60 if case["train"] else 20))
    if op == "save":
        n = case["b"] * case["s"] * case["d"]
        blocks = case["b"] * case["s"] * -(-case["d"] // _BLOCK)
        return dict(bytes=2 * size * n + 2 * (n + blocks), flops=4 * n)
    m = case["b"] * case["s"]
    if op == "linear":
        c, n = case["c"], case["n"] * case["outs"]
        return dict(bytes=size * (2 * m * c + 2 * m * n + 2 * n * c), flops=6 * m * n * c)
    if op == "mlp":
        c, h = case["c"], case["h"]
        return dict(bytes=size * (4 * m * c + 4 * h * c), flops=12 * m * h * c)
    n = m * case["v"]
    return dict(bytes=size * n * (2 if case["train"] else 1) + 17 * m, flops=n * (8 if case["train"] else 4))


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_unit(t, kind):
    """Rows of t with mean zero (layer) and unit mean square, and the factor that made them so."""
    c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
    f = (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    return c * f, f


def _exact_unit_grad(g, unit, factor, kind):
    mean = g.mean(-1, keepdim=True) if kind == "layer" else 0
    return factor * (g - mean - unit * (g * unit).mean(-1, keepdim=True))


def _exact_norm(case, state):
    kind, train = case["kind"], case["train"]
    t = {k: v.detach().double() for k, v in state.items() if torch.is_tensor(v)}
    y, fy = _exact_unit(t["y"], kind) if case["post"] else (t["y"], None)
    p = y * t["pw"] + t.get("pb", 0) if case["post"] else y
    gate = _wide_gate(t["gate"]) if "gate" in t else torch.ones((), dtype=torch.float64, device="cuda")
    h = t["x"] * case["scale"] + gate * p
    u, fh = _exact_unit(h, kind)
    out = dict(h=h, n=u * t["w"] + t.get("bias", 0))
    if train:
        full = t["dh"] + _exact_unit_grad(t["dn"] * t["w"], u, fh, kind)
        dp = full * gate
        out["dx"] = case["scale"] * full
        out["dy"] = _exact_unit_grad(dp * t["pw"], y, fy, kind) if case["post"] else dp
        if case["gate"] != "none":
            over = {"channel": (0, 1), "batch": (1,), "token": ()}[case["gate"]]
            out["dgate"] = (full * p).sum(over) if over else full * p
        out["dw"] = (t["dn"] * u).sum((0, 1))
        out["dbias"] = t["dn"].sum((0, 1))
        if case["post"]:
            out["dpw"] = (dp * y).sum((0, 1))
            out["dpb"] = dp.sum((0, 1))
    return {k: out[k] for k in _norm_keys(state)}


def _exact_round8(x):
    d = x.shape[-1]
    blocks = torch.nn.functional.pad(x, (0, -d % _BLOCK)).unflatten(-1, (-1, _BLOCK))
    amax = blocks.abs().amax(-1, keepdim=True)
    _, k = torch.frexp(amax)  # amax = m 2^k, 1/2 <= m < 1
    step = torch.ldexp(torch.ones_like(amax), (k - 7).clamp(min=-126))
    step = torch.where(torch.round(amax / step) > 127, 2 * step, step)
    return (torch.round(blocks / step) * step).flatten(-2)[..., :d]


def _exact_save(case, state):
    x = state["x"].detach()
    limit = torch.finfo(x.dtype).max
    return _exact_round8(x.double()).clamp(-limit, limit)


def _exact_linear(case, state):
    x = state["x"].detach().double()
    kept = _exact_round8(x)
    out, dx = {}, torch.zeros_like(x)
    for i, (w, dy) in enumerate(zip(state["w"], state["dy"])):
        w, dy = w.detach().double(), dy.double()
        out[f"y{i}"] = torch.einsum("bsc,nc->bsn", x, w)
        out[f"dw{i}"] = torch.einsum("bsn,bsc->nc", dy, kept)
        dx += torch.einsum("bsn,nc->bsc", dy, w)
    out["dx"] = dx
    return out


def _exact_mlp(case, state):
    x, w1, w2, dy = (state[k].detach().double() for k in ("x", "w1", "w2", "dy"))
    pre = torch.einsum("bsc,hc->bsh", x, w1)
    y = torch.einsum("bsh,ch->bsc", pre * torch.sigmoid(pre), w2)
    pre = _exact_round8(pre)
    sig = torch.sigmoid(pre)
    dw2 = torch.einsum("bsc,bsh->ch", dy, pre * sig)
    dpre = torch.einsum("bsc,ch->bsh", dy, w2) * (sig + pre * sig * (1 - sig))
    return dict(y=y, dx=torch.einsum("bsh,hc->bsc", dpre, w1),
                dw1=torch.einsum("bsh,bsc->hc", dpre, _exact_round8(x)), dw2=dw2)


def _exact_policy(case, state):
    b, s = case["b"], case["s"]
    mask, ids = state["mask"], state["ids"].clamp(min=0)
    adv = state["adv"].double()
    adv = adv[:, None].expand(b, s) if adv.dim() == 1 else adv
    lp = torch.zeros(b, s, dtype=torch.float64, device="cuda")
    for i in range(b):
        z = state["logits"][i].detach().double() / case["temp"]
        lp[i] = z.gather(1, ids[i][:, None])[:, 0] - torch.logsumexp(z, 1)
        del z
    lp = torch.where(mask, lp, 0)
    count = mask.sum(1, keepdim=True).double()
    if case["reduction"] == "sum":
        weight = mask.double()
    elif case["reduction"] == "mean":
        weight = mask.double() / count.sum().clamp(min=1)
    else:
        weight = mask.double() / count.clamp(min=1) / (count > 0).sum().clamp(min=1)
    ratio = torch.exp(lp - state["old"].double())
    high = (adv > 0) & (ratio > 1 + case["hi"])
    low = (adv < 0) & (ratio < 1 - case["lo"])
    border = torch.where(high, 1 + case["hi"], 1 - case["lo"])
    away = state["ref"].double() - lp
    kl = torch.expm1(away) - away
    loss = torch.where(high | low, -border * adv, -ratio * adv) + case["kl"] * kl
    out = dict(loss=(weight * torch.where(mask, loss, 0)).sum(), logp=lp,
               kl=(weight * torch.where(mask, kl, 0)).sum(), clipped=(weight * (high | low)).sum())
    if case["train"]:
        slope = torch.where(high | low, 0, -ratio * adv) - case["kl"] * torch.expm1(away)
        slope = torch.where(mask, weight * slope / case["temp"], 0)
        grad = torch.empty(b, s, case["v"], dtype=torch.float64, device="cuda")
        for i in range(b):
            grad[i] = torch.softmax(state["logits"][i].detach().double() / case["temp"], 1)
            grad[i] *= -slope[i][:, None]
            grad[i].scatter_add_(1, ids[i][:, None], slope[i][:, None])
        out["dlogits"] = grad
    return out


_EXACT = dict(norm=_exact_norm, save=_exact_save, linear=_exact_linear, mlp=_exact_mlp, policy=_exact_policy)


def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))
