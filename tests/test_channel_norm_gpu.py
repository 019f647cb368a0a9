"""Channel norms (F.channel_norm, F.channel_norm_residual) against a plain implementation in 64 bits, forward and backward.

Tolerances (fixed before the first run).  An output of type T is off by at most half a step of T, eps(T) / 2 relative, plus what fp32 arithmetic adds:
sums of C <= 8192 terms are <= 16 terms per lane, a tree over 64 lanes and one over <= 8 waves, so a mean is off by at most ~32 steps of 2^-24 relative to
the row's largest value, and a deviation x - mean by the same absolute amount: relative to the normalised value that is 32 * 2^-24 * (1 + |x|max / sigma).
With a second norm behind the first the two factors multiply.  64 * 2^-24 * (size of the terms) * (amplification) covers both and the few products.
Column sums add at most 8 + 32 + 128 terms in sequence (rows of a block, row groups, blocks): 256 * 2^-24 * sum of the terms' sizes."""
import math

import pytest
import torch

from codeps_amd import functional as F
from codeps_amd._lib import CodepsHipError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24
VECTORS = ("weight", "bias", "next_weight", "next_bias")


def half_step(t):
    return torch.finfo(t).eps / 2


def act_of(g, act):
    sig = 1 / (1 + torch.exp(-g))
    return {None: (g, torch.ones_like(g)), "sigmoid": (sig, sig * (1 - sig)), "silu": (g * sig, sig + g * sig * (1 - sig))}[act]


def normed(v, kind, eps):
    mu = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    rho = ((v - mu).pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    return (v - mu) * rho, rho


def normed_back(t, u, rho, kind):
    s = t - u * (t * u).mean(-1, keepdim=True)
    return rho * (s - t.mean(-1, keepdim=True) if kind == "layer" else s)


def reference(c, d):
    """Values and tolerances of every output; c: the call's options, d: its tensors in 64 bits on the CPU (rows x channels, gate broadcast)."""
    one, zero = torch.ones(1, dtype=torch.float64), torch.zeros(1, dtype=torch.float64)
    w, b = d.get("weight", one), d.get("bias", zero)
    x, out = d["x"], {}
    size = lambda v: v.abs().amax(-1, keepdim=True)                                              # noqa: E731
    if c["kind"]:
        u, rho = normed(x, c["kind"], c["eps"])
        amp = 1 + size(x) * rho
    else:
        u, rho, amp = x, one, one
    a = u * w + b
    a_size = size(u) * amp * w.abs() + b.abs()
    rowsum = lambda v: v.sum(0)                                                                  # noqa: E731
    if not c["full"]:
        out["h"] = (a, 64 * U * a_size)
        da, da_size, ampd = d.get("dh"), None if "dh" not in d else d["dh"].abs(), one
    else:
        gate, slope = act_of(d["gate"], c["act"]) if "gate" in d else (one, None)
        s = c["scale"] * gate
        y = d.get("residual", zero) + s * a
        y_size = d.get("residual", zero).abs() + s.abs() * a_size
        out["y"] = (y, 64 * U * y_size)
        da = d.get("dy", torch.zeros_like(y)).clone() if ("dy" in d or "dh" in d) else None
        ampd = one
        if c["next"]:
            un, rhon = normed(y, c["next"], c["next_eps"])
            ampn = amp * (1 + size(y_size) * rhon)
            nw, nb = d.get("next_weight", one), d.get("next_bias", zero)
            out["h"] = (un * nw + nb, 64 * U * (size(un) * ampn * nw.abs() + nb.abs()))
            if "dh" in d:
                out["dnext_weight"] = (rowsum(d["dh"] * un), rowsum(d["dh"].abs() * (256 * U * un.abs() + 64 * U * ampn * (1 + size(un)))))
                out["dnext_bias"] = (rowsum(d["dh"]), 256 * U * rowsum(d["dh"].abs()))
                da = da + normed_back(d["dh"] * nw, un, rhon, c["next"])
                ampd = ampn * (1 + size(un)) ** 2
        if da is not None:
            da_size = d.get("dy", zero).abs() + (rhon * size(d["dh"] * nw) * ampd if (c["next"] and "dh" in d) else 0)
            out["dresidual"] = (da, 64 * U * da_size)
            if slope is not None:
                dg, dg_size = c["scale"] * a * da * slope, abs(c["scale"]) * a_size * da_size * (slope.abs() + 2 * U)
                k = c["gate"]
                if k == "element":
                    out["dgate"] = (dg, 64 * U * dg_size)
                elif k == "channel":
                    out["dgate"] = (rowsum(dg), 320 * U * rowsum(dg_size))
                else:
                    n = c["items"]
                    out["dgate"] = tuple(f * v.view(n, -1, v.shape[-1]).sum(1) for f, v in ((1, dg), (320 * U, dg_size)))
            da, da_size = da * s, da_size * s.abs()
    if da is not None:
        amp2 = amp * (1 + size(u))
        out["dweight"] = (rowsum(da * u), rowsum(320 * U * da_size * (u.abs() + amp2)))
        out["dbias"] = (rowsum(da), rowsum(320 * U * da_size))
        if c["kind"]:
            out["dx"] = (normed_back(da * w, u, rho, c["kind"]), 64 * U * rho * size(da_size * w.abs()) * amp2 * (1 + size(u)))
        else:
            out["dx"] = (da * w, 64 * U * da_size * w.abs())
    return out


def make(c, seed=0):
    """The call's tensors on the GPU.  c: shape, channels, dtype, res (dtype or None), kind, gate, act, next, vectors' dtype, slack, offset."""
    gen = torch.Generator().manual_seed(seed)
    lead, C, T = c["shape"], c["C"], c["dtype"]
    rand = lambda *s: torch.randn(*s, generator=gen)                                             # noqa: E731
    t = {}
    wide = (rand(*lead, C + c["slack"]) * torch.exp(0.5 * rand(*lead, 1)) + c["offset"]).to(T).to(DEV)
    first = 1 if c["slack"] > 1 else 0                                 # (rows that start at an odd element)
    t["x"] = wide[..., first:first + C]
    vt = c["vectors"]
    if c["affine"]:
        t["weight"], t["bias"] = (1 + 0.3 * rand(C)).to(vt).to(DEV), (0.3 * rand(C)).to(vt).to(DEV)
    R = T
    if c["full"]:
        if c["res"] is not None:
            R = c["res"]
            t["residual"] = (2 * rand(*lead, C)).to(R).to(DEV)
        if c["gate"]:
            shape = {"channel": (C,), "item": lead[:1] + (1,) * (len(lead) - 1) + (C,), "element": (*lead, C)}[c["gate"]]
            t["gate"] = (0.5 + rand(*shape)).to(T if c["gate"] != "channel" else vt).to(DEV)
        if c["next"] and c["affine"]:
            t["next_weight"], t["next_bias"] = (1 + 0.3 * rand(C)).to(vt).to(DEV), (0.3 * rand(C)).to(vt).to(DEV)
        if "y" in c["douts"]:
            t["dy"] = rand(*lead, C).to(R).to(DEV)
    if "h" in c["douts"] and (c["next"] or not c["full"]):
        t["dh"] = rand(*lead, C).to(T).to(DEV)
    return t


def call(c, t):
    if not c["full"]:
        return {"h": F.channel_norm(t["x"], t.get("weight"), t.get("bias"), kind=c["kind"], eps=c["eps"])}
    out = F.channel_norm_residual(t["x"], t.get("residual"), t.get("weight"), t.get("bias"), kind=c["kind"], eps=c["eps"], gate=t.get("gate"), gate_act=c["act"],
                                  scale=c["scale"], next_kind=c["next"], next_weight=t.get("next_weight"), next_bias=t.get("next_bias"), next_eps=c["next_eps"])
    return {"y": out[0], "h": out[1]} if c["next"] else {"y": out}


def run(c, t):
    """Outputs and gradients of one call."""
    names = [k for k in ("x", "residual", "gate") + VECTORS if k in t]
    leaves = {k: t[k].detach().requires_grad_(True) for k in names}
    out = call(c, {**t, **leaves})
    wanted = [k for k in out if "d" + k in t]
    if not wanted:
        return {k: v.detach() for k, v in out.items()}
    grads = torch.autograd.grad([out[k] for k in wanted], list(leaves.values()), [t["d" + k] for k in wanted], allow_unused=True)
    return {**{k: v.detach() for k, v in out.items()}, **{"d" + k: g for k, g in zip(names, grads) if g is not None}}


def compare(c, t, got):
    C = c["C"]
    d = {k: v.detach().double().cpu() for k, v in t.items()}
    rows = d["x"].numel() // C
    if c["gate"] == "item":
        d["gate"] = d["gate"].reshape(c["shape"][0], 1, C).expand(-1, rows // c["shape"][0], -1)
    c = dict(c, items=c["shape"][0] if c["shape"] else 1)
    ref = reference(c, {k: v if v.dim() == 1 and k in VECTORS + ("gate",) else v.reshape(-1, C) for k, v in d.items()})
    for k, g in got.items():
        want, tol = ref[k]
        g64 = g.double().cpu().reshape(want.shape)
        bar = half_step(g.dtype) * (want.abs() + tol) + tol + torch.finfo(g.dtype).tiny * (2.0 ** -10 if g.dtype == F16 else 1.0)
        bad = (g64 - want).abs() > bar
        assert not bad.any(), (k, int(bad.sum()), float(((g64 - want).abs() / bar).max()))
    return ref


def case(C, shape=(7,), dtype=F32, full=True, kind="layer", res=F32, gate=None, act=None, next="layer", affine=True, vectors=F32, slack=0, offset=0.0, scale=0.5,
         douts="yh", eps=1e-5, next_eps=1e-5):
    return dict(C=C, shape=shape, dtype=dtype, full=full, kind=kind, res=res, gate=gate, act=act, next=next, affine=affine, vectors=vectors, slack=slack,
                offset=offset, scale=scale, douts=douts, eps=eps, next_eps=next_eps)


def name_of(c):
    return "-".join(str(v).replace("torch.", "") for k, v in c.items() if k in ("C", "shape", "dtype", "kind", "gate", "next", "res", "slack"))


# every width where the layout of a row changes (lanes per row, pieces per lane, one wave or a block, registers or slab), and one beside it
WIDTHS = [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 64, 100, 255, 256, 257, 511, 512, 513, 1000, 1024, 1025, 2047, 4095, 4096, 4097, 5000, 8191, 8192]


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_norm_alone_every_width(C, dtype):
    for kind, rows in (("layer", (5,)), ("rms", (2, 67))):
        c = case(C, rows, dtype, full=False, kind=kind, next=None)
        t = make(c, C)
        compare(c, t, run(c, t))


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype,res", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)], ids=str)
def test_block_end_every_width(C, dtype, res):
    for c in (case(C, (3, 5), dtype, res=res, gate="channel", act="sigmoid"), case(C, (2, 33), dtype, res=res, kind="rms", next="rms", gate="item", act="silu", scale=-0.7),
              case(C, (9,), dtype, res=res, kind=None, affine=C % 2 == 0, gate="element", next="layer")):
        t = make(c, C)
        compare(c, t, run(c, t))


@pytest.mark.parametrize("c", [
    case(64, (2, 9, 11), gate="item", act=None),                              # NHWC, a gate per image
    case(48, (1, 1), gate="element"), case(48, (), gate="channel"),           # a single row, with and without leading dimensions
    case(40, (4, 3000), gate="channel", act="silu"),                          # many rows: several blocks, several rows per block
    case(40, (4, 3000), BF16, res=F32, gate="item", act="sigmoid", kind="rms", next="rms"),
    case(600, (2, 700), BF16, res=BF16, gate="item"),
    case(4100, (3, 40), BF16, res=F32, gate="item"), case(4100, (2, 150), F32, gate="channel"),
    case(24, (1500, 2), gate="item"), case(24, (1500, 1), gate="item", douts="h"),      # more items than blocks
    case(9, (130,), slack=7, offset=3.0), case(9, (130,), BF16, res=BF16, slack=7),      # a channel slice of a wider map
    case(1000, (33,), F16, res=F16, slack=3), case(513, (33,), BF16, res=F32, slack=5),
    case(512, (65,), offset=30.0), case(512, (65,), kind="rms", offset=30.0),            # a common offset far larger than the spread
    case(96, (31,), douts="y"), case(96, (31,), douts="h"),                              # one of the two outputs has no gradient
    case(96, (31,), next=None), case(96, (31,), next=None, res=None), case(96, (31,), res=None),
    case(96, (31,), BF16, res=BF16, vectors=BF16, gate="channel"), case(96, (31,), F16, res=F32, vectors=F16, gate="channel"),
    case(96, (31,), affine=False, gate="element", act="sigmoid"), case(96, (31,), eps=0.0, next_eps=0.1), case(96, (31,), scale=0.0),
], ids=name_of)
def test_block_end_forms(c):
    t = make(c, 3)
    compare(c, t, run(c, t))


def test_gradients_against_differences():
    """Directional differences of the 64-bit formula (central, step 1e-5: its own error is below 1e-8) against the kernel's gradients."""
    c = case(37, (2, 6), gate="item", act="silu", kind="layer", next="rms")
    t = make(c, 11)
    got = run(c, t)
    d = {k: v.double().cpu() for k, v in t.items()}

    def loss(v):
        u = normed(v["x"], "layer", 1e-5)[0] * v["weight"] + v["bias"]
        y = v["residual"] + 0.5 * v["gate"] * torch.sigmoid(v["gate"]) * u
        h = normed(y, "rms", 1e-5)[0] * v["next_weight"] + v["next_bias"]
        return float((y * d["dy"]).sum() + (h * d["dh"]).sum())
    gen = torch.Generator().manual_seed(5)
    for k in ("x", "residual", "gate") + VECTORS:
        v = torch.randn(d[k].shape, generator=gen, dtype=torch.float64)
        slope = (loss({**d, k: d[k] + 1e-5 * v}) - loss({**d, k: d[k] - 1e-5 * v})) / 2e-5
        mine = float((got["d" + k].double().cpu() * v).sum())
        size = float((got["d" + k].double().cpu() * v).abs().sum())
        assert abs(slope - mine) <= 1e-6 * max(1.0, abs(slope)) + 512 * U * size, (k, slope, mine)


def test_rows_with_infinities_and_nan_stay_alone():
    """A row with an infinity or a NaN leaves every other row's outputs and gradients bit for bit as they are."""
    for C in (24, 700, 4500):
        c = case(C, (13,), BF16, res=F32, gate="element")
        t = make(c, 2)
        clean = run(c, t)
        t2 = {k: v.clone() for k, v in t.items()}
        t2["x"][3, C // 2] = float("nan")
        t2["x"][7, 0] = float("inf")
        t2["residual"][9, 1] = float("-inf")
        got = run(c, t2)
        keep = [i for i in range(13) if i not in (3, 7, 9)]
        for k in ("y", "h", "dx", "dresidual", "dgate"):
            assert torch.equal(got[k][keep], clean[k][keep]), k
        assert torch.isnan(got["y"][3]).all() and torch.isnan(got["h"][9]).any() and not torch.isfinite(got["dweight"]).all()


def test_zero_rows_zero_deviation_and_lowest_values():
    c = case(33, (0,), gate="channel")
    t = make(c)
    got = run(c, t)
    assert got["y"].shape == (0, 33) and all(not got[k].any() for k in ("dweight", "dbias", "dgate", "dnext_weight", "dnext_bias"))
    for shape, gate in (((0, 4), "item"), ((4, 0), "item"), ((2, 0), "element")):
        c = case(33, shape, gate=gate)
        got = run(c, make(c))
        assert got["dgate"].numel() == 0 or not got["dgate"].any()
    c = case(64, (3,), eps=1e-5)                                     # a constant row: deviation 0, the output is the bias
    t = make(c)
    t["x"][1] = 5.0
    out = F.channel_norm(t["x"], t["weight"], t["bias"])
    assert torch.allclose(out[1], t["bias"], atol=64 * U * 5.0 / math.sqrt(1e-5) * 2, rtol=0)
    low = torch.full((2, 64), torch.finfo(BF16).min, dtype=BF16, device=DEV)      # the type's lowest value overflows the sum of squares, as the formula's does in fp32
    out = F.channel_norm(low, kind="rms")
    assert torch.isfinite(out).all() and float(out.abs().max()) == 0.0


def test_layouts_are_read_where_they_lie_or_copied():
    g = torch.Generator().manual_seed(1)
    base = torch.randn(6, 40, 5, generator=g).to(DEV)
    w = torch.randn(40, generator=g).to(DEV)
    x = base.transpose(1, 2)                                          # channels not dense
    assert torch.equal(F.channel_norm(x, w), F.channel_norm(x.contiguous(), w))
    x = torch.randn(4, 6, 40, generator=g).to(DEV)[:, ::2]            # rows at two distances
    assert torch.equal(F.channel_norm(x, w), F.channel_norm(x.contiguous(), w))
    x = torch.randn(1, 40, generator=g).to(DEV).expand(7, 40)         # one row read seven times
    leaf = x.detach().requires_grad_(True)
    out = F.channel_norm(leaf, w)
    assert torch.equal(out, F.channel_norm(x.contiguous(), w))
    (dx,) = torch.autograd.grad(out.sum(), [leaf])                    # (the gradient of a sum is an expanded scalar)
    like = x.contiguous().requires_grad_(True)
    assert torch.equal(dx, torch.autograd.grad(F.channel_norm(like, w), [like], [torch.ones(7, 40, device=DEV)])[0])
    mod = torch.randn(3, 80, generator=g).to(DEV)                     # a gate per image cut out of a modulation vector
    x = torch.randn(3, 5, 40, generator=g).to(DEV)
    assert torch.equal(F.channel_norm_residual(x, gate=mod[:, 40:]), F.channel_norm_residual(x, gate=mod[:, 40:].contiguous()))


def test_results_repeat_bit_for_bit_and_ignore_the_stream():
    c = case(72, (3, 900), BF16, res=F32, gate="channel", act="silu")
    t = make(c, 9)
    first = run(c, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(c, t)
    torch.cuda.current_stream().wait_stream(side)
    for k in first:
        assert torch.equal(first[k], second[k]), k


def test_two_captured_graphs_replay_side_by_side():
    """Forward and backward of two different calls, each captured into a graph of its own; replays with new inputs equal the eager results."""
    cs = [case(72, (2, 300), gate="channel"), case(700, (2, 60), BF16, res=F32, gate="item", act="sigmoid")]
    ts = [make(c, 4) for c in cs]
    for c, t in zip(cs, ts):
        run(c, t)
    graphs, outs = [], []
    for c, t in zip(cs, ts):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(c, t))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cs]
    for seed in (21, 22, 23):
        fresh = [make(c, seed) for c in cs]
        want = [run(c, f) for c, f in zip(cs, fresh)]
        for t, f in zip(ts, fresh):
            for k in t:
                t[k].copy_(f[k])
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for k in w:
                assert torch.equal(o[k], w[k]), (seed, k)


def test_capture_while_an_eager_graph_of_the_same_leaf_lives_is_refused():
    """Its gradient would be accumulated on the default stream in the middle of the capture.  Without that graph the capture works."""
    x, w, dh = torch.randn(9, 40, device=DEV), torch.nn.Parameter(torch.randn(40, device=DEV)), torch.randn(9, 40, device=DEV)
    live = F.channel_norm(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = x + 1.0
        for call in (lambda: F.channel_norm(x, w), lambda: F.channel_norm_residual(x, next_kind="rms", next_weight=w)):
            with pytest.raises(CodepsHipError, match="drop it before the capture"):
                call()
        with torch.no_grad():
            F.channel_norm(x, w)                                     # (nothing to accumulate)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, x + 1.0)
    del live
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.channel_norm(x, w).backward(dh)
    mine = w.grad
    for seed in (1, 2, 3):
        x.copy_(torch.randn(9, 40, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        fresh = w.detach().clone().requires_grad_(True)
        F.channel_norm(x, fresh).backward(dh)
        assert torch.equal(mine, fresh.grad), seed


def test_gradients_go_straight_into_registered_sinks():
    c = case(50, (40,))
    t = make(c, 6)
    want = run(c, t)
    flat = torch.arange(200, dtype=F32, device=DEV)
    params = [torch.nn.Parameter(t[k].clone()) for k in VECTORS]
    for i, p in enumerate(params):
        F.register_grad_sink(p, flat[50 * i:50 * i + 50])
    x = t["x"].detach().requires_grad_(True)
    y, h = F.channel_norm_residual(x, t["residual"], params[0], params[1], scale=0.5, next_kind="layer", next_weight=params[2], next_bias=params[3])
    torch.autograd.backward([y, h], [t["dy"], t["dh"]])
    assert all(p.grad is None for p in params) and torch.equal(x.grad, want["dx"])
    for i, k in enumerate(VECTORS):
        assert torch.equal(flat[50 * i:50 * i + 50], torch.arange(50 * i, 50 * i + 50, dtype=F32, device=DEV) + want["d" + k]), k


def test_one_parameter_as_both_norms_vectors():
    """Shared by the two norms of a block's end, with and without a sink: the gradients add up (two roundings of 2^-24 more: the sum, and the sink's)."""
    c = case(50, (400,))
    t = make(c, 6)
    t["next_weight"], t["next_bias"] = t["weight"], t["bias"]
    apart = run(c, t)
    x = t["x"].detach()
    for sink in (False, True):
        w, b = (torch.nn.Parameter(t[k].clone()) for k in ("weight", "bias"))
        flat = torch.zeros(100, device=DEV)
        if sink:
            F.register_grad_sink(w, flat[:50])
            F.register_grad_sink(b, flat[50:])
        for n in (1, 2):
            y, h = F.channel_norm_residual(x, t["residual"], w, b, scale=0.5, next_kind="layer", next_weight=w, next_bias=b)
            torch.autograd.backward([y, h], [t["dy"], t["dh"]])
            got = (flat[:50], flat[50:]) if sink else (w.grad, b.grad)
            for g, k in zip(got, ("weight", "bias")):
                parts = apart["d" + k].double(), apart["dnext_" + k].double()
                bar = 4 * n * U * (parts[0].abs() + parts[1].abs())
                assert ((g.double() - n * (parts[0] + parts[1])).abs() <= bar).all(), (sink, n, k)


def test_block_end_of_one_tensor_and_under_checkpointing():
    """x as its own residual: both gradients reach it.  Re-computation (torch.utils.checkpoint) gives the same bits."""
    from torch.utils.checkpoint import checkpoint
    c = case(48, (70,), gate="channel", act="silu")
    t = make(c, 3)
    leaves = [t[k].detach().clone().requires_grad_(True) for k in ("x", "gate") + VECTORS]

    def block(x, gate, w, b, nw, nb):
        return F.channel_norm_residual(x, x, w, b, scale=0.5, gate=gate, gate_act="silu", next_kind="layer", next_weight=nw, next_bias=nb)
    plain = torch.autograd.grad(block(*leaves), leaves, [t["dy"], t["dh"]])
    again = torch.autograd.grad(checkpoint(block, *leaves, use_reentrant=False), leaves, [t["dy"], t["dh"]])
    assert all(torch.equal(a, b) for a, b in zip(plain, again))
    x, other = (leaves[0].detach().clone().requires_grad_(True) for _ in range(2))
    y, h = F.channel_norm_residual(x, other, *leaves[2:4], scale=0.5, gate=leaves[1], gate_act="silu", next_kind="layer", next_weight=leaves[4], next_bias=leaves[5])
    parts = torch.autograd.grad([y, h], [x, other], [t["dy"], t["dh"]])
    assert torch.equal(plain[0], parts[0] + parts[1])


def test_rows_far_apart():
    """Rows further apart than 32-bit offsets allow are copied, not misread."""
    store = torch.zeros(2 * (1 << 24) + 40, dtype=BF16, device=DEV)
    x = store.as_strided((3, 40), ((1 << 24), 1))
    x.copy_(torch.randn(3, 40, device=DEV))
    near = store.as_strided((2, 40), ((1 << 24) - 1, 1), 1)
    near.copy_(torch.randn(2, 40, device=DEV))
    for v in (x, near):
        assert torch.equal(F.channel_norm(v), F.channel_norm(v.contiguous()))


def test_rows_beyond_32_bit_offsets():
    """2^31 + elements: the last rows of a large map come out as they do alone."""
    C, rows = 2048, (1 << 20) + 3
    x = torch.empty(rows, C, dtype=BF16, device=DEV)
    x[:] = torch.randn(1, C, device=DEV).to(BF16)
    tail = torch.randn(4, C, device=DEV).to(BF16)
    x[-4:] = tail
    w = torch.randn(C, device=DEV)
    out = F.channel_norm(x, w)
    assert torch.equal(out[-4:], F.channel_norm(tail, w)) and torch.equal(out[:1], F.channel_norm(x[:1].clone(), w))


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    for bad in (lambda: F.channel_norm(x.double()), lambda: F.channel_norm(torch.zeros(3, 0, device=DEV)), lambda: F.channel_norm(torch.zeros(2, 8193, device=DEV)),
                lambda: F.channel_norm(x, kind="batch"), lambda: F.channel_norm(x, kind=None), lambda: F.channel_norm(x, w[:7]), lambda: F.channel_norm(x, w.double()),
                lambda: F.channel_norm(x, w.cpu()), lambda: F.channel_norm(x, w, w.half()), lambda: F.channel_norm(x, eps=-1.0), lambda: F.channel_norm(x, eps=float("nan")),
                lambda: F.channel_norm_residual(x, x[:3]), lambda: F.channel_norm_residual(x, x.half()), lambda: F.channel_norm_residual(x.half(), x.to(BF16)),
                lambda: F.channel_norm_residual(x, x.cpu()), lambda: F.channel_norm_residual(x, gate_act="silu"), lambda: F.channel_norm_residual(x, gate=w, gate_act="gelu"),
                lambda: F.channel_norm_residual(x, gate=w[:4]), lambda: F.channel_norm_residual(x, gate=torch.zeros(2, 8, device=DEV)),
                lambda: F.channel_norm_residual(x.view(2, 2, 8), gate=torch.zeros(2, 2, 2, 8, device=DEV)), lambda: F.channel_norm_residual(x, next_weight=w),
                lambda: F.channel_norm_residual(x, next_kind="x"), lambda: F.channel_norm_residual(x, gate=w.double()),
                lambda: F.channel_norm_residual(x.half(), gate=x.float())):
        with pytest.raises(CodepsHipError):
            bad()
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):                                 # no second derivative
        (g,) = torch.autograd.grad(F.channel_norm(leaf).sum(), [leaf], create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("gate", ["channel", "item", "element"])
@pytest.mark.parametrize("dtype,res", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32)], ids=str)
def test_activated_gates_at_the_ends_of_their_type(dtype, res, gate):
    """Infinite gates and the largest finite ones are open or shut, and leave their neighbours alone: values and gradients of a sigmoid as everywhere (the 64-bit
    one is exact there: 1 or 0, slope 0), a SiLU's gate is g where g is large and 0 at the type's lowest value; at +inf it is infinite, its own element alone.

    1 / (1 + e^-g) is 0 once e^-g passes 2^126: the gate is off by at most |g| e^g < 2^7 2^-126 there (e^-g passes 2^150 at 104).  Behind it lie factors below
    2^7 and sums of at most 80 of them: `floor`.  A SiLU's slope s (1 + g (1 - s)) passes through 0: it is off by at most 16 roundings of 2^-24 (its factors and
    terms are below 1.3 where they matter, and take a dozen operations), whatever is left of it; the gate's gradient has that times |scale a da|, which `reference`
    gives with the slope as a factor (and 64 or, in sums, 320 roundings)."""
    C, floor = 72, 2.0 ** -126 * 2 ** 7 * 2 ** 7 * 80

    def near(c, t, got):
        d = {k: v.detach().double().cpu() for k, v in t.items()}
        if gate == "item":
            d["gate"] = d["gate"].reshape(rows[0], 1, C).expand(-1, math.prod(rows[1:]), -1)
        want = reference(dict(c, items=rows[0]), {k: v if v.dim() == 1 else v.reshape(-1, C) for k, v in d.items()})
        for k, g in got.items():
            v, tol = want[k]
            if k == "dgate":
                slope = act_of(t["gate"].detach().double().cpu(), c["act"])[1].reshape(v.shape).abs()
                tol = tol * (1 + 16 / (64 if gate == "element" else 320) / (slope + 2 * U))
            assert torch.isfinite(g).all(), k
            assert ((g.double().cpu().reshape(v.shape) - v).abs() <= half_step(g.dtype) * (v.abs() + tol) + tol + torch.finfo(g.dtype).tiny + floor).all(), k
    for rows in ((5,), (2, 40)):
        c = case(C, rows, dtype, res=res, gate=gate, act="sigmoid")
        t = make(c, 5)
        kept = t["gate"].dtype
        ends = torch.tensor([math.inf, -math.inf, torch.finfo(kept).max, torch.finfo(kept).min, torch.finfo(kept).max / 1.2, torch.finfo(kept).max / 2, 89.0, -89.0],
                            device=DEV).to(kept)
        t["gate"][..., 3:3 + 8 * len(ends):8] = ends
        near(c, t, run(c, t))
        c = case(C, rows, dtype, res=res, gate=gate, act="silu", scale=2.0 ** -6, next=None)
        t = make(c, 6)
        for k in ("weight", "bias"):
            t[k] *= 2.0 ** -6                                        # (so that the largest gates stay finite in y)
        large = min(torch.finfo(v).max for v in (kept, dtype, res)) / 256
        t["gate"][..., 3:51:8] = torch.tensor([torch.finfo(kept).min, large, 89.0, -89.0, 1000.0, -1000.0], device=DEV).to(kept)
        clean = run(c, t)
        near(c, t, clean)
        t["gate"][..., 60] = math.inf
        y = run(c, t)["y"]
        a = F.channel_norm(t["x"].float(), t["weight"].float(), t["bias"].float(), eps=c["eps"])[..., 60]
        keep = [i for i in range(C) if i != 60]
        assert torch.equal(y[..., keep], clean["y"][..., keep]) and torch.equal(y[..., 60].float(), torch.where(a > 0, math.inf, -math.inf))


def test_transformed_tensors_are_refused():
    """Dual tensors, and the wrappers of torch.func: an error, not an output without its derivative."""
    x = torch.randn(5, 8, device=DEV)
    for transform in (lambda f: torch.func.jvp(f, (x,), (x,)), lambda f: torch.func.grad(lambda v: f(v).sum())(x), lambda f: torch.vmap(f)(x)):
        for f in (F.channel_norm, lambda v: F.channel_norm_residual(v, x, next_kind="layer")[1], lambda v: F.channel_norm_residual(x, v), lambda v: F.grad_norm([v])):
            with pytest.raises(RuntimeError):
                transform(f)


def test_views_that_negate_are_read_with_their_sign():
    """The imaginary part of a conjugate holds the other sign in memory: rows (of one channel they need no copy for their strides), vectors, gates, gradients."""
    g = torch.Generator().manual_seed(4)
    for C in (1, 6):
        z = torch.randn(5, C, dtype=torch.complex64, generator=g).to(DEV).conj()
        v = torch.randn(C, dtype=torch.complex64, generator=g).to(DEV).conj()
        x, w = z.imag, v.imag
        assert x.is_neg() and w.is_neg()
        plain = lambda t: t.clone().contiguous()                                                   # noqa: E731
        for call in (lambda t, u: F.channel_norm(t, u, u, kind="rms"), lambda t, u: F.channel_norm_residual(t, t, u, kind=None, gate=u),
                     lambda t, u: F.channel_norm_residual(t, t, u, kind="rms", gate=t, next_kind="rms", next_weight=u)[1]):
            assert not plain(x).is_neg() and torch.equal(call(x, w), call(plain(x), plain(w)))
            grads = []
            for t, u, dy in ((x, w, x), (plain(x), plain(w), plain(x))):
                leaf, vec = t.detach().requires_grad_(True), u.detach().requires_grad_(True)
                grads.append(torch.autograd.grad(call(leaf, vec), [leaf, vec], [dy]))
            assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("rows", [1, 2])
def test_a_gate_per_item_has_a_type_of_its_own_where_an_item_is_one_row(rows):
    """[B, 1, C] beside x [B, N, C]: with N = 1 it has x's shape too, and is a gate per item all the same."""
    c = case(40, (3, rows), BF16, res=F32, gate="item", act="sigmoid")
    for kept in (F32, F16, BF16):
        t = make(c, 8)
        t["gate"] = t["gate"].to(kept)
        got = run(c, t)
        assert got["dgate"].dtype == kept and got["dgate"].shape == t["gate"].shape
        compare(c, t, got)
