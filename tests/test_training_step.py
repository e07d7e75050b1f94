"""The training-step operators as they are used together: norm, kept operand, contractions, policy loss."""

import threading

import pytest
import torch
import torch.utils.checkpoint

import torch_einshard_b200 as es

cuda = pytest.param("cuda", marks=pytest.mark.gpu)
DEVICES = ["cpu", cuda]


class Step:
    """One block and the loss of its logits: leaves, and a step that gives the loss and their gradients."""

    def __init__(self, device, dtype, b=2, s=24, d=96, n=160, v=203, seed=0):
        gen = torch.Generator().manual_seed(seed)

        def draw(*shape, scale=1.0):
            return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(device).requires_grad_(True)

        self.leaves = dict(x=draw(b, s, d), y=draw(b, s, d), gate=draw(b, d), w=draw(d), up=draw(n, d, scale=d ** -0.5),
                           down=draw(d, n, scale=n ** -0.5), head=draw(v, d, scale=d ** -0.5))
        self.ids = torch.randint(0, v, (b, s), generator=gen).to(device)
        self.adv = torch.randn(b, generator=gen).to(device)
        self.mask = (torch.rand(b, s, generator=gen) < 0.7).to(device)

    def loss(self, x, y, gate, w, up, down, head):
        h, n = es.einnorm("b s d", x, y, axis="d", kind="rms", weight=w, post=True, gate=gate, gate_axes="b d")
        a = es.einshard("b s d, n d -> b s n", es.checkpoint8(n), up, activation="silu")
        _, n = es.einnorm("b s d", h, es.einshard("b s n, d n -> b s d", a, down), axis="d", kind="rms")
        logits = es.einshard("b s d, v d -> b s v", es.checkpoint8(n), head)
        return es.einpolicy("b s v", logits, self.ids, axis="v", advantages=self.adv, mask=self.mask).loss

    def __call__(self):
        loss = self.loss(*self.leaves.values())
        return loss.detach(), *torch.autograd.grad(loss, list(self.leaves.values()))

    def exact(self):
        """The same in 64 bits with whole operands."""
        t = [p.detach().double().cpu().requires_grad_(True) for p in self.leaves.values()]
        x, y, gate, w, up, down, head = t

        def normed(z):
            return z / torch.sqrt(z.square().mean(-1, keepdim=True) + 1e-5)

        h = x + gate[:, None] * normed(y)
        h = h + torch.nn.functional.silu((normed(h) * w) @ up.t()) @ down.t()
        lp = torch.log_softmax(normed(h) @ head.t(), -1).gather(-1, self.ids.cpu()[..., None])[..., 0]
        mask, adv = self.mask.cpu(), self.adv.double().cpu()[:, None]
        loss = -(torch.exp(lp - lp.detach()) * adv * mask).sum() / mask.sum()
        return loss.detach(), *torch.autograd.grad(loss, t)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_against_64_bits(device, dtype):
    """Gradients of weights see operands within half a step of 1/64 (relative to a block's largest value): their error
    is that noise, averaged over the tokens.  bf16 adds a dozen roundings of half a step each."""
    step = Step(device, dtype)
    noise = 12 * torch.finfo(dtype).eps / 2
    got, want = step(), step.exact()
    assert abs(got[0].double().cpu() - want[0]) <= 1e-5 + noise * (1 + want[0].abs())
    for name, g, e in zip(step.leaves, got[1:], want[1:]):
        assert g.dtype == dtype and (g.double().cpu() - e).norm() <= (1 / 64 + noise) * e.norm(), name


@pytest.mark.parametrize("device", DEVICES)
def test_recomputed(device):
    step = Step(device, torch.bfloat16)
    leaves = list(step.leaves.values())
    loss = torch.utils.checkpoint.checkpoint(step.loss, *leaves, use_reentrant=False)
    for g, h in zip(step()[1:], torch.autograd.grad(loss, leaves)):
        assert torch.equal(g, h)


@pytest.mark.gpu
def test_two_captured_steps():
    """Graphs replayed in any order, with leaves that change between replays."""
    step = Step("cuda", torch.bfloat16, s=64, d=256, n=320, v=500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for order in ((0, 1), (1, 0), (1, 1, 0)):
        for i in order:
            graphs[i].replay()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        with torch.no_grad():
            for p in step.leaves.values():
                p.mul_(0.9)


@pytest.mark.parametrize("device", DEVICES)
def test_backward_passes_of_several_threads(device):
    step = Step(device, torch.bfloat16)
    x, up = step.leaves["x"], step.leaves["up"]
    kept = es.checkpoint8(x)
    ys = [es.einshard("b s d, n d -> b s n", kept, up) for _ in range(3)]
    dy = [torch.full_like(y, 0.5 + i) for i, y in enumerate(ys)]
    want = torch.autograd.grad(ys, [x, up], dy, retain_graph=True)
    got = [None] * 4

    def run(i):
        got[i] = torch.autograd.grad(ys, [x, up], dy, retain_graph=True)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
