"""The channel norms, the convolutions, AdamW and the gradient norm together: StepRunner with cfg.train.optimizer.type "AdamW" (eager, captured, parameters
that a step does not reach), and a residual block trained with them."""
import copy

import pytest
import torch

from codeps_amd import functional as F
from codeps_amd.optim import AdamW

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _setup(**options):
    import bench
    from codeps_amd import synthetic
    net, cfg = bench.build(torch.device(DEV), 18, 64, 128, "adapt")
    cfg.train.optimizer.update(options)
    return net, cfg, synthetic


def _runner(net, cfg):
    from codeps_amd.step import StepRunner
    return StepRunner(net, cfg, "adapt", 1)


def test_runner_follows_torch_adamw_and_leaves_unreached_parameters_alone():
    """Four steps against torch.optim.AdamW fed with the same gradients.  Both round a parameter (below 4 here) once per step: 2 * 4 * 2^-25 * 4; the steps of
    1e-4 themselves agree to a few 2^-24."""
    net, cfg, synthetic = _setup(type="AdamW", weight_decay=0.05, max_grad_norm=1.0)
    runner = _runner(net, cfg)
    assert all(g.m is None and g.v is None for g in runner.groups)
    ref = [[torch.nn.Parameter(g.flat[a:b].clone()) for a, b in zip(g.offsets[:-1], g.offsets[1:])] for g in runner.groups]
    dims = [[p.dim() for p in g.params] for g in runner.groups]
    part = lambda wide: [q for ps, ds in zip(ref, dims) for q, d in zip(ps, ds) if (d > 1) == wide]                 # noqa: E731
    opt = torch.optim.AdamW([{"params": part(True), "weight_decay": 0.05}, {"params": part(False), "weight_decay": 0.0}], lr=runner.lr)
    ema = [None if g.ema is None else g.ema.clone() for g in runner.groups]
    full, _ = synthetic.adapt_batch(64, 128, torch.device(DEV), 5, 1, 1, 1, 2)
    depth_only, _ = synthetic.adapt_batch(64, 128, torch.device(DEV), 6, 1, 1, 0, 0)
    for data in (depth_only, full, depth_only, full):
        runner.forward_backward(data)
        touched = runner._touched
        opt.zero_grad(set_to_none=True)
        for gi, g in enumerate(runner.groups):
            for pi, (q, a, b) in enumerate(zip(ref[gi], g.offsets[:-1], g.offsets[1:])):
                if touched is None or touched[gi] is None or touched[gi][pi]:
                    q.grad = g.grad[a:b].clone()
        have = [q.grad for ps in ref for q in ps if q.grad is not None]
        norm = float(torch.stack([g.double().square().sum() for g in have]).sum().sqrt())
        for q in have:
            q.mul_(min(1.0, 1.0 / norm))
        opt.step()
        for gi, g in enumerate(runner.groups):
            if ema[gi] is not None:
                ema[gi].mul_(runner.ema_alpha).add_(torch.cat([q.detach() for q in ref[gi]]), alpha=1 - runner.ema_alpha)
        runner.optimizer_step()
        assert abs(float(runner.adamw.grad_norm) - norm) <= 4 * U * norm
        for gi, g in enumerate(runner.groups):
            want = torch.cat([q.detach() for q in ref[gi]])
            assert torch.allclose(g.flat, want, rtol=0, atol=1e-6), (gi, float((g.flat - want).abs().max()))
            if ema[gi] is not None:
                assert torch.allclose(g.ema, ema[gi], rtol=0, atol=1e-6), gi
    assert set(runner.adamw.steps.tolist()) == {2, 4}                # the semantic head is out of reach of the depth losses


@pytest.mark.parametrize("bits", [32, 8])
def test_replayed_steps_equal_eager_steps(bits):
    net_a, cfg, synthetic = _setup(type="AdamW", state_bits=bits, max_grad_norm=5.0, seed=3)
    net_b = copy.deepcopy(net_a)
    data, _ = synthetic.adapt_batch(64, 128, torch.device(DEV), 5, 1, 1, 1, 2)
    ra, rb = _runner(net_a, cfg), _runner(net_b, cfg)
    for _ in range(3):
        ra.step(data)
    rb.capture(data)
    for _ in range(3):
        rb.replay()
    torch.cuda.synchronize()
    for ga, gb in zip(ra.groups, rb.groups):
        assert torch.equal(ga.flat, gb.flat) and (ga.ema is None or torch.equal(ga.ema, gb.ema))
    sa, sb = ra.adamw.state_dict(), rb.adamw.state_dict()
    assert all(torch.equal(sa[k], sb[k]) for k in sa if k != "param_groups")
    if bits == 8:                                                    # most of the parameters, in a quarter of the bytes
        n8 = sum(k for k, b in zip(ra.adamw._numels, ra.adamw._bits) if b == 8)
        assert n8 > 0.9 * sum(ra.adamw._numels) and ra.adamw.exp_avg_codes.numel() >= n8


def test_default_optimizer_is_unchanged():
    net, cfg, _ = _setup()
    runner = _runner(net, cfg)
    assert runner.adamw is None and all(g.m is not None for g in runner.groups)


# ------------------------------------------------------------------------------------------------------------------ a block, trained
class Block:
    """norm -> 1x1 convolution -> SiLU gate of a second one -> block end with residual, layer scale and the next norm -> 1x1 convolution, on [B, H, W, C]."""

    def __init__(self, c, seed):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s, m=0.0, k=1.0: torch.nn.Parameter((m + k * torch.randn(*s, generator=g)).to(DEV))          # noqa: E731
        self.p = {"w0": rand(c, m=1.0, k=0.1), "b0": rand(c, k=0.1), "conv0": rand(c, c, 1, 1, k=c ** -0.5), "gate": rand(c, c, 1, 1, k=c ** -0.5),
                  "w1": rand(c, m=1.0, k=0.1), "w2": rand(c, m=1.0, k=0.1), "b2": rand(c, k=0.1), "conv1": rand(c, c, 1, 1, k=c ** -0.5)}

    def loss(self, x, target):
        p = self.p
        h = F.channel_norm(x, p["w0"], p["b0"])
        y, n = F.channel_norm_residual(F.conv2d(h, p["conv0"]), x, p["w1"], kind="rms", gate=F.conv2d(h, p["gate"]), gate_act="silu", scale=0.5,
                                       next_kind="layer", next_weight=p["w2"], next_bias=p["b2"])
        out = F.conv2d(n, p["conv1"]) + y
        return ((out - target) ** 2).mean()


def _plain_loss(p, x, target):
    def norm(v, kind):
        v = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        return v * (v.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
    mix = lambda v, w: v @ w[:, :, 0, 0].t().contiguous()                                         # noqa: E731
    h = norm(x, "layer") * p["w0"] + p["b0"]
    g = mix(h, p["gate"])
    y = x + 0.5 * g * torch.sigmoid(g) * norm(mix(h, p["conv0"]), "rms") * p["w1"]
    n = norm(y, "layer") * p["w2"] + p["b2"]
    return ((mix(n, p["conv1"]) + y - target) ** 2).mean()


@pytest.mark.parametrize("c,hw", [(32, (5, 7)), (64, (9, 12))])
def test_block_gradients_against_64_bits(c, hw):
    """A product of c <= 64 terms is off by at most 2 c steps of its largest term; four of them and three norms lie in a row: 1024 * 2^-24 of a tensor's largest
    gradient."""
    block = Block(c, 1)
    g = torch.Generator().manual_seed(2)
    x, target = (torch.randn(2, *hw, c, generator=g).to(DEV) for _ in range(2))
    x.requires_grad_(True)
    names = list(block.p)
    got = torch.autograd.grad(block.loss(x, target), [x] + [block.p[k] for k in names])
    wide = {k: v.detach().double().cpu().requires_grad_(True) for k, v in block.p.items()}
    xd = x.detach().double().cpu().requires_grad_(True)
    want = torch.autograd.grad(_plain_loss(wide, xd, target.double().cpu()), [xd] + [wide[k] for k in names])
    for k, a, b in zip(["x"] + names, got, want):
        assert float((a.double().cpu() - b).abs().max()) <= 1024 * U * float(b.abs().max()), k


@pytest.mark.parametrize("bits", [32, 8])
def test_block_trains_eagerly_and_captured(bits):
    """Three whole steps (forward, backward, norm, update) from one captured graph equal three eager ones bit for bit."""
    def make():
        block = Block(64, 3)
        g = torch.Generator().manual_seed(4)
        x, target = (torch.randn(2, 8, 8, 64, generator=g).to(DEV) for _ in range(2))
        mats = [p for p in block.p.values() if p.dim() > 1]
        vecs = [p for p in block.p.values() if p.dim() == 1]
        opt = AdamW([{"params": mats, "weight_decay": 0.1}, {"params": vecs, "weight_decay": 0.0}], lr=1e-2, state_bits=bits, small_numel=1024, max_norm=0.5, seed=1)
        return block, x, target, opt

    def step(block, x, target, opt):
        loss = block.loss(x, target)
        grads = torch.autograd.grad(loss, opt.params)
        norm = F.grad_norm(grads)
        opt.step(grads)
        return loss.detach(), norm
    eager = make()
    seen = [tuple(float(v) for v in step(*eager)) for _ in range(4)]
    assert all(abs(n - float(eager[3].grad_norm)) <= 2 * U * n for _, n in seen[-1:])
    other = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = tuple(float(v) for v in step(*other))                # warm-up: the first step, eagerly
    torch.cuda.current_stream().wait_stream(side)
    assert first == seen[0]
    F.invalidate_weight_cache()                                      # the captured step re-packs the convolutions' weights
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*other)
    for k in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        assert tuple(float(v) for v in out) == seen[k], k
    assert all(torch.equal(a, b) for a, b in zip(eager[3].params, other[3].params))
