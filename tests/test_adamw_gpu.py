"""codeps_amd.optim.AdamW and functional.grad_norm against a plain implementation in 64 bits on the CPU.

Tolerances (fixed before the first run).  32-bit states: a moment is two products and a sum, off by at most 3 roundings (3 * 2^-24 of the larger term) per
step, and errors of earlier steps only decay: 8 * 2^-24 * (|b1 m| + |(1 - b1) g'|) per step, twice that for v (g' is squared).  The parameter adds its own
rounding and lr * 32 * 2^-24 of the ratio, whose error is that of m, sqrt(v), a reciprocal and two scalars; m may cancel, so its error counts relative to
its terms.  8-bit states: codes and exponents are EQUAL to those of the 64-bit formula (the kernel decides in 64 bits where fp32 could be wrong)."""
import copy
import math

import numpy as np
import pytest
import torch

from codeps_amd import functional as F
from codeps_amd._lib import CodepsHipError
from codeps_amd.optim import AdamW

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24
MASK = (1 << 64) - 1


# ------------------------------------------------------------------------------------------------ the 8-bit format, element by element in 64 bits
def grid(mant):
    return [k * 2.0 ** (-14 - mant) for k in range(1 << mant)] + [(1 + k / (1 << mant)) * 2.0 ** e for e in range(-14, 1) for k in range(1 << mant)]


def random_bits(seed, tensor, step, n):
    z = (seed + step * 0x9E3779B97F4A7C15 + tensor * 0xD1B54A32D192ED03) & MASK
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & MASK
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & MASK
    z ^= z >> 31
    x = (np.arange(n, dtype=np.uint64) + np.uint64(z & 0xFFFFFFFF)) & np.uint64(0xFFFFFFFF)
    low = np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D)) & low
    x = x ^ (x >> np.uint64(15)) ^ np.uint64(z >> 32)
    x = (x * np.uint64(0x846CA68B)) & low
    x = x ^ (x >> np.uint64(16))
    return (x & np.uint64(0xFFFF)).astype(np.float64), (x >> np.uint64(16)).astype(np.float64)


def encode(x, rho, mant, signed):
    """x [n] float64 -> (codes padded to whole blocks, exponent bytes, values)."""
    g = np.array(grid(mant) + [2.0])
    n, k = len(x), -(-len(x) // 256)
    codes, exps, vals = np.zeros(k * 256, np.uint8), np.zeros(k, np.uint8), np.zeros(n)
    for b in range(k):
        v = x[256 * b:256 * (b + 1)]
        if not np.isfinite(v).all():
            exps[b] = 255
            vals[256 * b:256 * b + len(v)] = np.nan
            continue
        top = np.abs(v).max()
        e = -126
        while e < 128 and top > g[-2] * 2.0 ** e:
            e += 1
        if top < 2.0 ** -126:
            continue
        t = np.abs(v) / 2.0 ** e
        lo = np.searchsorted(g, t, side="right") - 1
        up = (t - g[lo]) / (g[lo + 1] - g[lo]) + rho[256 * b:256 * b + len(v)] / 65536.0 >= 1.0
        c = lo + up
        codes[256 * b:256 * b + len(v)] = c + (128 * (v < 0) if signed else 0)
        exps[b] = e + 127
        vals[256 * b:256 * b + len(v)] = np.where(v < 0, -1, 1) * g[c] * 2.0 ** e
    return codes, exps, vals


class Plain:
    """The same optimizer in 64 bits on the CPU, with a bound of the fp32 kernel's error beside every value."""

    def __init__(self, params, decays, bits, lr, betas, eps, max_norm=None, ema=None, ema_alpha=0.99, seed=0):
        self.p = [p.detach().double().cpu().numpy().reshape(-1).copy() for p in params]
        self.m, self.v = [np.zeros_like(p) for p in self.p], [np.zeros_like(p) for p in self.p]
        self.pe, self.me, self.ve = ([np.zeros_like(p) for p in self.p] for _ in range(3))
        self.steps = [0] * len(self.p)
        self.decays, self.bits, self.lr, self.betas, self.eps, self.max_norm, self.seed = decays, bits, lr, betas, eps, max_norm, seed
        self.ema = None if ema is None else [None if e is None else e.detach().double().cpu().numpy().reshape(-1).copy() for e in ema]
        self.ema_alpha, self.stored = ema_alpha, {}

    def step(self, grads, grad_scale=1.0, lr=None, apply_ema=True):
        lr = self.lr if lr is None else lr
        b1, b2 = self.betas
        gs = [None if g is None else g.double().cpu().numpy().reshape(-1) for g in grads]
        self.norm = abs(grad_scale) * math.sqrt(sum(float((g ** 2).sum()) for g in gs if g is not None))
        c = grad_scale * (self.max_norm / self.norm if self.max_norm and self.norm > self.max_norm else 1.0)
        for i, g in enumerate(gs):
            if g is not None:
                g = g * c
                self.steps[i] += 1
                t = self.steps[i]
                ms, vs = np.abs(b1 * self.m[i]) + np.abs((1 - b1) * g), b2 * self.v[i] + (1 - b2) * g * g
                self.me[i] = b1 * self.me[i] + 8 * U * ms
                self.ve[i] = b2 * self.ve[i] + 16 * U * vs
                self.m[i] = b1 * self.m[i] + (1 - b1) * g
                self.v[i] = vs
                den = np.sqrt(self.v[i] / (1 - b2 ** t)) + self.eps
                rate = lr / (1 - b1 ** t)
                with np.errstate(invalid="ignore"):
                    rel_v = np.where(self.v[i] > 0, self.ve[i] / np.maximum(self.v[i], 1e-300), 0.0)
                    self.pe[i] += 2 * U * np.abs(self.p[i]) + np.abs(rate) * (self.me[i] + ms * (rel_v + 32 * U)) / den
                    self.p[i] = self.p[i] * (1 - lr * self.decays[i]) - rate * self.m[i] / den
                if self.bits[i] == 8:
                    rm, rr = random_bits(self.seed, i, t, len(g))
                    cm, em, self.m[i] = encode(self.m[i], rm, 3, True)
                    cr, er, root = encode(np.sqrt(self.v[i]), rr, 4, False)
                    self.v[i] = root ** 2
                    self.me[i][:] = self.ve[i][:] = 0
                    self.stored[i] = (cm, em, cr, er)
            if self.ema is not None and apply_ema and self.ema[i] is not None:
                self.ema[i] = self.ema_alpha * self.ema[i] + (1 - self.ema_alpha) * self.p[i]


def check(opt, plain, copies=None):
    flat = lambda t: t.detach().double().cpu().numpy().reshape(-1)                                # noqa: E731
    assert opt.steps.tolist() == plain.steps
    for i, p in enumerate(opt.params):
        off, n = opt._offsets[i], p.numel()
        err = np.abs(flat(p) - plain.p[i])
        assert (err <= plain.pe[i] + 2 * U * np.abs(plain.p[i])).all(), ("p", i, float((err / (plain.pe[i] + 1e-300)).max()))
        if plain.bits[i] == 32:
            for have, want, bar in ((opt.exp_avg, plain.m[i], plain.me[i]), (opt.exp_avg_sq, plain.v[i], plain.ve[i])):
                assert (np.abs(flat(have[off:off + n]) - want) <= bar + 1e-44).all(), ("moments", i)
        elif i in plain.stored:
            k = -(-n // 256)
            cm, em, cr, er = plain.stored[i]
            assert np.array_equal(opt.exp_avg_exponents[off // 256:off // 256 + k].cpu().numpy(), em), ("exponents of m", i)
            assert np.array_equal(opt.root_exponents[off // 256:off // 256 + k].cpu().numpy(), er), ("exponents of the root", i)
            # (codes 0 and 128 both stand for zero: 0 and -0, and the sign of a sum that cancels to 1e-19 is that of its rounding)
            have = opt.exp_avg_codes[off:off + 256 * k].cpu().numpy()
            assert np.array_equal(np.where(have == 128, 0, have), np.where(cm == 128, 0, cm)), ("codes of m", i)
            assert np.array_equal(opt.root_codes[off:off + 256 * k].cpu().numpy(), cr), ("codes of the root", i)
        if plain.ema is not None and plain.ema[i] is not None:
            err = np.abs(flat(opt._ema[i]) - plain.ema[i])
            assert (err <= 8 * (plain.pe[i] + U * np.abs(plain.ema[i]) + U * np.abs(plain.p[i]))).all(), ("ema", i)
        if opt._copies[i] is not None and copies:
            assert torch.equal(opt._copies[i], p.detach().to(opt._copies[i].dtype)), ("copy", i)


def tensors(sizes, seed, spread=1e-2):
    g = torch.Generator().manual_seed(seed)
    return [(spread * torch.randn(*(s if isinstance(s, tuple) else (s,)), generator=g)).to(DEV) for s in sizes]


def gradients(params, seed, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return [(1e-3 * torch.randn(p.shape, generator=g) * torch.exp(2 * torch.randn(p.shape, generator=g))).to(dtype).to(DEV) for p in params]


SIZES = [1, 2, 3, 5, 255, 256, 257, (16, 16, 3, 3), 2047, 2048, 2049, (64, 100), 4099, 10001, (0,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_steps_against_64_bits(bits, dtype):
    """Every size around a chunk and a block; decay by group, EMA, copies, clipping, a scale, tensors without a gradient."""
    params = tensors(SIZES, 1, 0.05)
    ema = [p + 0.01 if i % 3 == 0 else None for i, p in enumerate(params)]
    copies = [torch.zeros_like(p, dtype=BF16 if i % 2 else F16) if i % 4 else None for i, p in enumerate(params)]
    mats = [i for i, p in enumerate(params) if i % 2 == 0]
    order = mats + [i for i in range(len(params)) if i % 2]
    params, ema, copies = ([v[i] for i in order] for v in (params, ema, copies))
    opt = AdamW([{"params": params[:len(mats)], "weight_decay": 0.1}, {"params": params[len(mats):], "weight_decay": 0.0, "lr": 3e-3}], lr=3e-3, betas=(0.9, 0.99),
                state_bits=bits, small_numel=256, ema=ema, ema_alpha=0.9, copies=copies, max_norm=0.05, seed=77)
    held = [bits if p.numel() >= 256 else 32 for p in params]
    plain = Plain(params, [0.1] * len(mats) + [0.0] * (len(params) - len(mats)), held, 3e-3, (0.9, 0.99), 1e-8, 0.05, ema, 0.9, 77)
    for k in range(4):
        grads = gradients(params, 100 + k, dtype)
        if k == 2:
            grads = [None if i % 3 == 1 else g for i, g in enumerate(grads)]
        opt.step(grads, grad_scale=0.5, apply_ema=k != 1)
        plain.step(grads, 0.5, apply_ema=k != 1)
        check(opt, plain, copies=k == 0)
        assert abs(float(opt.grad_norm) - plain.norm) <= 2 * U * plain.norm


def test_eight_bits_for_the_smallest_tensors():
    """Tensors shorter than a block, of one element, and empty ones, all in 8 bits."""
    params = tensors([1, 5, (0,), 300, 255, 2], 8, 0.1)
    opt = AdamW(params, lr=1e-2, state_bits=8, small_numel=0, max_norm=1e-3, seed=4)
    plain = Plain(params, [0.01] * 6, [8] * 6, 1e-2, (0.9, 0.999), 1e-8, 1e-3, seed=4)
    for k in range(3):
        grads = gradients(params, 30 + k, F16)
        opt.step(grads)
        plain.step(grads)
        check(opt, plain)
    assert opt.exp_avg is None and opt.moments_8bit()[0].numel() == 563


def test_default_gradients_mixed_types_and_zero_grad():
    params = [torch.nn.Parameter(p) for p in tensors([300, (7, 9), 4], 3)]
    opt = AdamW(params, lr=1e-2, weight_decay=0.0)
    plain = Plain(params, [0.0] * 3, [32] * 3, 1e-2, (0.9, 0.999), 1e-8)
    params[0].grad = gradients(params, 5)[0]
    params[2].grad = gradients(params, 6)[2]
    opt.step()
    plain.step([params[0].grad, None, params[2].grad])
    check(opt, plain)
    opt.zero_grad(set_to_none=False)
    assert not params[0].grad.any() and params[1].grad is None
    opt.zero_grad()
    before = [p.detach().clone() for p in params]
    opt.step()                                                       # nothing has a gradient: nothing moves
    assert all(torch.equal(a, b) for a, b in zip(before, params)) and opt.steps.tolist() == [1, 0, 1]
    grads = [g.to(t) for g, t in zip(gradients(params, 8), (F16, F32, BF16))]
    opt.step(grads)
    plain.step(grads)
    check(opt, plain)


def test_more_tensors_than_one_launch_takes_and_unaligned_views():
    """331 + 331 tensors as views of flat buffers (starts at any multiple of an element), 32 and 8 bits mixed by size."""
    g = torch.Generator().manual_seed(2)
    sizes = torch.randint(1, 700, (662,), generator=g).tolist()
    flat = 0.1 * torch.randn(sum(sizes) + 1, generator=g)
    flat, grad = flat.to(DEV), (1e-2 * torch.randn(sum(sizes) + 1, generator=g)).to(BF16).to(DEV)
    cut = lambda t: list(t[1:].split(sizes))                                                      # noqa: E731
    params, grads = cut(flat), cut(grad)
    opt = AdamW(params, lr=1e-3, state_bits=8, small_numel=300, max_norm=1.0, seed=5)
    plain = Plain(params, [0.01] * 662, [8 if n >= 300 else 32 for n in sizes], 1e-3, (0.9, 0.999), 1e-8, 1.0, seed=5)
    for _ in range(2):
        opt.step(grads)
        plain.step(grads)
        check(opt, plain)
    first = float(flat[0])
    assert first == float(flat[0])                                   # (the element in front of the views)
    m, r = opt.moments_8bit()
    big = [i for i, n in enumerate(sizes) if n >= 300]
    assert np.array_equal(m.double().cpu().numpy(), np.concatenate([plain.m[i] for i in big]))
    assert np.array_equal(r.double().cpu().numpy() ** 2, np.concatenate([plain.v[i] for i in big]))


def test_layouts():
    p = torch.randn(8, 6, 5, 5, device=DEV).contiguous(memory_format=torch.channels_last)
    q = p.detach().clone().contiguous()
    g = torch.randn(8, 6, 5, 5, device=DEV)
    a, b = AdamW([p], lr=1e-2), AdamW([q], lr=1e-2)
    for _ in range(2):
        a.step([g])                                                  # gradient in another layout than its parameter
        b.step([g])
        b.step([g.contiguous(memory_format=torch.channels_last)])
        a.step([g.contiguous(memory_format=torch.channels_last)])
    assert torch.equal(p, q)
    q.data = q.data.clone()                                          # moved: the table follows
    p2 = p.detach().clone()
    a.step([g])
    b.step([g])
    assert torch.equal(p, q) and not torch.equal(p, p2)


def test_sums_that_fall_exactly_on_a_border():
    """Gradients of four bits and codes of four bits: (9 a + b) / 10 is a whole number of 2^-16 quanta for every fifth element, and for some of those the random
    bits make it exactly the border between two codes.  The last bit of 64 decides, as in the formula."""
    n = 1 << 21
    g = torch.Generator().manual_seed(1)
    params = [torch.zeros(n, device=DEV)]
    opt, plain = AdamW(params, lr=1e-3, state_bits=8, seed=6), Plain(params, [0.01], [8], 1e-3, (0.9, 0.999), 1e-8, seed=6)
    for _ in range(2):
        grads = [(torch.randint(-15, 16, (n,), generator=g) / 1024.0).to(BF16).to(DEV)]
        opt.step(grads)
        plain.step(grads)
        check(opt, plain)


def test_eight_bit_rounding_is_unbiased_and_averages_decay():
    """65536 elements of one value: the mean of what is stored is the value (4 standard errors); with zero gradients the stored moments fall with b^t, which
    rounding to the nearest code would keep from happening (0.1 % of a value is far below half a code)."""
    n, lr = 65536, 0.0
    p = torch.zeros(n, device=DEV)
    opt = AdamW([p], lr=lr, betas=(0.5, 0.999), state_bits=8, seed=3)
    g = torch.full((n,), 1.37e-3, device=DEV)
    g[::256] = 5e-3                                                  # (the block's largest value, so that the others are not at its top)
    opt.step([g])
    m, r = (t.double() for t in opt.moments_8bit())
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[::256] = False
    for have, want in ((m[rest].mean(), 0.5 * 1.37e-3), (r[rest].mean(), math.sqrt(0.001) * 1.37e-3)):
        assert abs(float(have) / want - 1) <= 4 * 0.125 / 2 / math.sqrt(n)
    zero = torch.zeros_like(g)
    for _ in range(700):
        opt.step([zero])
    m, r = (t.double() for t in opt.moments_8bit())
    # the root's mean falls with sqrt(b2)^700 = 0.704 (its square is updated: a step's rounding noise, at most (2^-5)^2 / 4 of the square, pulls the mean of
    # the root up by about that share of b2's decay: the bound allows 0.72 to 0.99 of the value before, nearest rounding would leave 1.0)
    left = float(r[rest].mean()) / (math.sqrt(0.001) * 1.37e-3)
    assert 0.5 < left < 0.99, left
    assert float(m.abs().max()) == 0.0                               # 0.5^700


def test_non_finite_gradients():
    params = tensors([1000, 5000], 1)
    grads = gradients(params, 2)
    grads[1][4321] = float("inf")
    opt = AdamW(params, state_bits=8, small_numel=2000, max_norm=1.0, skip_nonfinite=True, ema=[p.clone() for p in params])
    keep = [p.clone() for p in params] + [e.clone() for e in opt._ema]
    opt.step(grads)
    assert all(torch.equal(a, b) for a, b in zip(keep, params + opt._ema)) and opt.steps.tolist() == [0, 0] and math.isinf(float(opt.grad_norm))
    assert not opt.exp_avg.any() and not opt.exp_avg_codes.any()
    opt.skip_nonfinite, opt.max_norm = False, None
    grads[1][4321] = float("nan")
    opt.step(grads)
    m, r = opt.moments_8bit()
    bad = torch.arange(5000, device=DEV) // 256 == 4321 // 256       # the block of the NaN, and nothing beside it
    assert torch.isnan(m[bad]).all() and torch.isnan(r[bad]).all() and torch.isfinite(m[~bad]).all() and torch.isfinite(r[~bad]).all()
    assert torch.isnan(params[1]).sum() == 1 and torch.isfinite(params[0]).all()


def test_tiny_and_huge_moments():
    """Blocks near both ends of fp32: zeros below 2^-126, NaN where the block's unit would be 2^128; values in between keep their bits."""
    p = tensors([1024], 1)[0]
    g = torch.zeros(1024)
    g[0], g[256], g[512], g[768] = 1e-39, 1e-30, 1.0, 3.4e38
    opt = AdamW([p], lr=0.0, betas=(0.0, 0.0), state_bits=8, small_numel=1, weight_decay=0.0)
    opt.step([g.to(DEV)])
    assert opt.exp_avg_exponents.tolist() == [0, 127 - 100, 127, 255]
    m = opt.moments_8bit()[0].float().cpu()
    assert float(m[0]) == 0.0 and abs(float(m[256]) / 1e-30 - 1) <= 0.125 and float(m[512]) == 1.0 and torch.isnan(m[768:]).all() and not m[1:256].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_replays_as_the_next_step(bits):
    """Capture with a learning rate on the device; every replay equals the eager step bit for bit (step counts, random bits and clipping are on the device)."""
    lr = torch.tensor(1e-2, device=DEV)
    mine, theirs = tensors([5000, 300, 9000], 4), tensors([5000, 300, 9000], 4)
    grads = gradients(mine, 1)
    a = AdamW(mine, lr=lr, state_bits=bits, max_norm=0.1, seed=9, ema=[p.clone() for p in mine])
    b = AdamW(theirs, lr=1e-2, state_bits=bits, max_norm=0.1, seed=9, ema=[p.clone() for p in theirs])
    a.step(grads)
    b.step(grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(grads)
    for k in range(4):
        fresh = gradients(mine, 10 + k)
        for g, f in zip(grads, fresh):
            g.copy_(f)
        rate = float(np.float32(1e-2 / (k + 1)))
        lr.fill_(rate)
        b.param_groups[0]["lr"] = rate
        graph.replay()
        b.step(fresh)
        torch.cuda.synchronize()
        for x, y in zip(mine + a._ema, theirs + b._ema):
            assert torch.equal(x, y), k
        sa, sb = a.state_dict(), b.state_dict()
        assert all(torch.equal(sa[n], sb[n]) for n in sa if n != "param_groups") and float(a.grad_norm) == float(b.grad_norm)


def test_state_dict_continues_the_run():
    a_p = tensors([6000, 50], 2)
    a = AdamW(a_p, lr=1e-2, state_bits=8, seed=1)
    for k in range(3):
        a.step(gradients(a_p, k))
    b_p = [p.clone() for p in a_p]
    b = AdamW(b_p, lr=5.0, state_bits=8, seed=1)
    b.load_state_dict(a.state_dict())
    for k in range(3, 5):
        a.step(gradients(a_p, k))
        b.step(gradients(b_p, k))
    assert all(torch.equal(x, y) for x, y in zip(a_p, b_p)) and b.param_groups[0]["lr"] == 1e-2
    for other in (AdamW([p.clone() for p in a_p], state_bits=32), AdamW(tensors([6000], 2), state_bits=8)):
        with pytest.raises(CodepsHipError):
            other.load_state_dict(a.state_dict())


def test_updates_are_seen_by_autograd_and_by_the_weight_packs():
    w = torch.nn.Parameter(torch.randn(16, 16, 1, 1, device=DEV))
    x = torch.randn(1, 8, 8, 16, device=DEV)
    opt = AdamW([w], lr=0.5, weight_decay=0.0)
    (w * w).sum().backward()
    held = (w * w).sum()                                             # its backward would need the weight from before the step
    y0 = F.conv2d(x, w).detach()
    opt.step()
    with pytest.raises(RuntimeError):
        held.backward()
    y1 = F.conv2d(x, w).detach()
    want = torch.einsum("bhwc,oc->bhwo", x.double().cpu(), w.detach().double().cpu()[:, :, 0, 0])
    assert not torch.equal(y0, y1) and float((y1.double().cpu() - want).abs().max()) <= 1e-4


def test_elements_beyond_32_bit_offsets():
    """One tensor of 2^31 + 300 elements with 8-bit states: its last elements are updated, and stored, as the formula says."""
    n = (1 << 31) + 300
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, dtype=BF16, device=DEV)
    tail = gradients([torch.zeros(600)], 3, BF16)[0]
    g[-600:] = tail
    opt = AdamW([p], lr=1e-2, state_bits=8, seed=12, max_norm=1e-3)
    opt.step([g])
    norm = float(tail.double().norm())
    assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm and abs(float(F.grad_norm([g])) - norm) <= 2 * U * norm
    scaled = tail.double().cpu().numpy() * min(1.0, 1e-3 / norm)
    want = -1e-2 * scaled / (np.abs(scaled) + 1e-8)
    assert np.abs(p[-600:].double().cpu().numpy() - want).max() <= 1e-2 * 64 * U
    assert not p[:1 << 20].any() and not p[(1 << 31) - 1000:(1 << 31) - 300].any()
    z = 0.1 * scaled
    blocks = opt.exp_avg_codes[-512:].cpu().numpy()                   # the last whole block and the padded one: 300 = 256 + 44 elements behind 2^31
    i = np.arange(1 << 31, n, dtype=np.uint64)
    seed = (12 + 0x9E3779B97F4A7C15) & MASK
    seed = ((seed ^ (seed >> 30)) * 0xBF58476D1CE4E5B9) & MASK
    seed = ((seed ^ (seed >> 27)) * 0x94D049BB133111EB) & MASK
    seed ^= seed >> 31
    low = np.uint64(0xFFFFFFFF)
    x = (i + np.uint64(seed & 0xFFFFFFFF)) & low
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D)) & low
    x = ((x ^ (x >> np.uint64(15)) ^ np.uint64(seed >> 32)) * np.uint64(0x846CA68B)) & low
    x ^= x >> np.uint64(16)
    codes, _, _ = encode(z[-300:], (x & np.uint64(0xFFFF)).astype(np.float64), 3, True)
    assert np.array_equal(blocks, codes)


# ------------------------------------------------------------------------------------------------------------------------ gradient norm
def test_grad_norm():
    g = torch.Generator().manual_seed(7)
    sizes = [1, 3, 4095, 4096, 4097, 100000] + torch.randint(1, 3000, (400,), generator=g).tolist()
    ts = [(torch.randn(n, generator=g) * 10.0 ** (i % 4)).to((F32, BF16, F16)[i % 3]).to(DEV) for i, n in enumerate(sizes)]
    ts.insert(5, torch.zeros(0, device=DEV))
    ts.insert(0, torch.zeros(0, device=DEV))
    want = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
    got = F.grad_norm([None] + ts + [None], scale=-0.25)
    assert got.shape == () and got.dtype == F32 and abs(float(got) - 0.25 * want) <= 2 * U * want
    assert float(F.grad_norm(ts)) == float(F.grad_norm(ts))
    strided = torch.randn(50, 70, device=DEV)[:, ::2]
    assert abs(float(F.grad_norm([strided])) - float(strided.double().norm())) <= 2 * U * float(strided.double().norm())
    assert abs(float(F.grad_norm([torch.full((1000,), 1e30, device=DEV)])) / (1e30 * math.sqrt(1000)) - 1) <= 2 * U
    assert math.isinf(float(F.grad_norm([torch.tensor([1.0, float("-inf")], device=DEV)]))) and math.isnan(float(F.grad_norm([torch.tensor([float("nan")], device=DEV)])))
    assert float(F.grad_norm([torch.zeros(0, device=DEV)])) == 0.0


def test_grad_norm_in_a_graph():
    ts = gradients([torch.zeros(5000), torch.zeros(70)], 1)
    F.grad_norm(ts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.grad_norm(ts)
    for k in range(3):
        for t, f in zip(ts, gradients(ts, 50 + k)):
            t.copy_(f)
        want = float(F.grad_norm(ts))
        graph.replay()
        torch.cuda.synchronize()
        assert float(out) == want


def test_refusals():
    p = torch.zeros(10, device=DEV)
    for bad in (lambda: AdamW([]), lambda: AdamW([{"params": []}]), lambda: AdamW([p.half()]), lambda: AdamW([p, p]), lambda: AdamW([torch.zeros(4, 6, device=DEV)[:, ::2]]),
                lambda: AdamW([p], state_bits=16), lambda: AdamW([p], max_norm=0.0), lambda: AdamW([p], ema=[p.half()]), lambda: AdamW([p], ema=[]),
                lambda: AdamW([p], copies=[p.clone()]), lambda: AdamW([p], copies=[torch.zeros(9, dtype=BF16, device=DEV)]), lambda: AdamW([{"params": [p], "momentum": 1}]),
                lambda: AdamW([{"params": [torch.zeros(1, device=DEV)]} for _ in range(17)]), lambda: F.grad_norm([]), lambda: F.grad_norm([None]),
                lambda: F.grad_norm([p.double()]), lambda: F.grad_norm([p, p.cpu()])):
        with pytest.raises(CodepsHipError):
            bad()
    opt = AdamW([p, torch.zeros(3, 4, device=DEV)])
    for grads in ([p], [p, torch.zeros(4, 3, device=DEV)], [p.cpu(), None], [p.double(), None]):
        with pytest.raises(CodepsHipError):
            opt.step(grads)
    for key, value in (("betas", (1.0, 0.9)), ("betas", (0.9, -0.1)), ("eps", -1.0)):
        opt = AdamW([p], **{key: value})
        with pytest.raises(CodepsHipError):
            opt.step([p])
    with pytest.raises(CodepsHipError):
        AdamW([p], lr=torch.zeros(2, device=DEV)).step([p])
    with pytest.raises(CodepsHipError):
        AdamW([p]).moments_8bit()


def test_tensors_that_share_memory_are_refused():
    """Two work groups would update the same elements."""
    p = torch.zeros(100, device=DEV)
    half = torch.zeros(64, dtype=BF16, device=DEV)
    for bad in (lambda: AdamW([p, p[50:]]), lambda: AdamW([p[:10], p], ema=[torch.zeros(10, device=DEV), None]), lambda: AdamW([p], ema=[p]),
                lambda: AdamW([p[:50], p[50:]], ema=[torch.zeros(50, device=DEV), p[:50]]), lambda: AdamW([p[:32], p[32:64]], copies=[half[:32], half[16:48]]),
                lambda: AdamW([p], ema_alpha=-0.1), lambda: AdamW([p], ema_alpha=float("nan")), lambda: copy.deepcopy(AdamW([p]))):
        with pytest.raises(CodepsHipError):
            bad()
    AdamW([p[:50], p[50:]], copies=[half[:0].new_zeros(50), None])                        # neighbours do not


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_move_between_steps(bits):
    """.data = of parameters, EMA tensors and copies: the next step writes where they are, and nothing where they were."""
    p, e, c = tensors([5000], 1)[0], torch.zeros(5000, device=DEV), torch.zeros(5000, dtype=BF16, device=DEV)
    q, f = p.clone(), e.clone()
    a, b = AdamW([p], lr=1e-2, state_bits=bits, ema=[e], copies=[c]), AdamW([q], lr=1e-2, state_bits=bits, ema=[f])
    for k in range(6):
        if k in (1, 4):
            p.data = p.data.clone()
        old = {2: e, 3: c}.get(k)
        if old is not None:
            was, before = old.data, old.data.clone()
            old.data = old.data.clone()
        g = gradients([q], 30 + k)
        a.step(g)
        b.step(g)
        assert torch.equal(p, q) and torch.equal(e, f) and torch.equal(c, p.to(BF16)), k
        assert old is None or torch.equal(was, before), k
    e.data = e.data.half()
    with pytest.raises(CodepsHipError):
        a.step(g)
    with pytest.raises(CodepsHipError):
        a.step(iter(g + g))
    b.step(iter(g))                                                  # (any iterable serves)
    assert b.steps.tolist() == [7]


def test_gradient_norm_of_gradients_with_a_graph():
    """Refused while a graph is recorded, taken under no_grad; a step with such gradients is none of autograd's business either way."""
    w = torch.nn.Parameter(torch.arange(1.0, 5.0, device=DEV))
    (g,) = torch.autograd.grad((w ** 3).sum(), [w], create_graph=True)
    with pytest.raises(CodepsHipError, match="no derivative"):
        F.grad_norm([g])
    with torch.no_grad():
        norm = F.grad_norm([g, w])
    want = math.sqrt(sum((3.0 * k * k) ** 2 + k * k for k in range(1, 5)))
    assert not norm.requires_grad and abs(float(norm) - want) <= 2 * U * want
    AdamW([w], lr=0.5, weight_decay=0.0).step([g])
    assert torch.allclose(w.detach(), torch.arange(1.0, 5.0, device=DEV) - 0.5, rtol=0, atol=1e-5)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_averages_and_copies_are_seen_to_change(dtype):
    """A graph that saved a working copy, or an average, and runs backward behind the step ends in autograd's error, as it does for a parameter; frozen convolution
    weights that are averages or copies are packed anew; apply_ema False leaves averages, and what was saved of them, alone."""
    w = torch.nn.Parameter(torch.randn(16, 16, 1, 1, device=DEV))
    other = torch.nn.Parameter(torch.randn(5, device=DEV))
    ema, copy_ = w.detach().clone(), w.detach().to(dtype)
    opt = AdamW([other, w], lr=0.5, weight_decay=0.0, ema=[None, ema], ema_alpha=0.5, copies=[None, copy_])
    x, leaf = torch.randn(1, 8, 8, 16, device=DEV), torch.ones(16, 16, 1, 1, device=DEV, requires_grad=True)
    conv = lambda t: torch.einsum("bhwc,oc->bhwo", x.double().cpu(), t.detach().double().cpu()[:, :, 0, 0])            # noqa: E731
    grads = [None, torch.ones_like(w)]
    for apply_ema in (True, False):
        saved = {"parameter": (leaf * w).sum(), "average": (leaf * ema).sum(), "copy": (leaf.to(dtype) * copy_).sum()}
        before = [F.conv2d(x, t).clone() for t in (ema, copy_)]
        versions = ema._version, copy_._version
        opt.step(grads, apply_ema=apply_ema)
        assert (ema._version > versions[0]) == apply_ema and copy_._version > versions[1]
        for k, loss in saved.items():
            if k == "average" and not apply_ema:
                loss.backward()
            else:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    loss.backward()
        for t, y, moved in zip((ema, copy_), before, (apply_ema, True)):
            now = F.conv2d(x, t)
            assert float((now.double().cpu() - conv(t)).abs().max()) <= 1e-4 and torch.equal(now, y) != moved
    fresh = torch.zeros(4, device=DEV)
    with torch.inference_mode():
        frozen = torch.zeros(4, device=DEV)                          # (an inference tensor has no version)
    AdamW([fresh], ema=[frozen]).step([torch.ones(4, device=DEV)])
    assert frozen.any()


def test_a_replayed_step_is_seen_by_the_weight_packs():
    """Parameters (trainable, and plain tensors with gradients of their own), averages and copies as convolution weights, before and behind replays."""
    made = [torch.nn.Parameter(torch.randn(16, 16, 1, 1, device=DEV)), torch.randn(16, 16, 1, 1, device=DEV)]
    ema, copies = [p.detach().clone() for p in made], [p.detach().to(BF16) for p in made]
    opt = AdamW(made, lr=0.5, weight_decay=0.0, ema=ema, ema_alpha=0.5, copies=copies)
    grads, x = [torch.ones_like(p) for p in made], torch.randn(1, 8, 8, 16, device=DEV)
    opt.step(grads)
    weights = made + ema + copies
    seen = [F.conv2d(x, w).detach().clone() for w in weights]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grads)
    for _ in range(3):
        graph.replay()
        F.invalidate_weight_cache()
        for i, w in enumerate(weights):
            now = F.conv2d(x, w).detach().clone()
            want = torch.einsum("bhwc,oc->bhwo", x.double().cpu(), w.detach().double().cpu()[:, :, 0, 0])
            assert float((now.double().cpu() - want).abs().max()) <= 1e-4 and not torch.equal(now, seen[i]), i
            seen[i] = now


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("betas,eps", [((0.9, 0.999), 1e-8), ((0.0, 0.0), 1e-8), ((0.9, 0.999), 0.0), ((0.5, 0.9999999), 1e-30)])
def test_eight_bit_states_over_the_whole_range(betas, eps, dtype):
    """Blocks from 2^-126 to 2^126: the root's square leaves fp32 at 2^-63 and 2^64.  Blocks of one size, blocks whose elements spread over 2^24, and blocks of one
    large and 255 far smaller elements; codes, units, values and parameters as the 64-bit formula has them, over steps in which the sizes change places."""
    gen = torch.Generator().manual_seed(13)
    rows = []
    for k in range(-126, 127, 3):
        base = torch.sign(torch.randn(3, 256, generator=gen, dtype=torch.float64)) * (1 + torch.rand(3, 256, generator=gen, dtype=torch.float64)) / 2
        base[1] *= 2.0 ** -(24 * torch.rand(256, generator=gen, dtype=torch.float64))
        base[2] *= 2.0 ** -(3.0 * (k % 8))
        base[2, 5] = 0.75
        rows.append(torch.sign(base) * (base.abs() * 2.0 ** k).clamp(min=2.0 ** -130))            # (no zeros: with eps = 0 their update is 0 / 0)
    sizes = torch.cat(rows)
    params = tensors([sizes.numel(), 100], 4)
    opt = AdamW(params, lr=1e-2, betas=betas, eps=eps, state_bits=8, small_numel=1, seed=21)
    plain = Plain(params, [0.01, 0.01], [8, 8], 1e-2, betas, eps, seed=21)
    small = gradients(params, 3)[1]
    # A root that was rounded to 0 beside a moment of 2^100 sends a parameter beyond fp32's range, by the formula: infinite from then on.
    gone = np.zeros(sizes.numel(), bool)
    for order in (sizes, sizes, sizes.roll(3, 0), sizes.flip(0), sizes * 0 + 2.0 ** -30):
        grads = [order.reshape(-1).float().to(dtype).to(DEV), small]
        assert (grads[0] != 0).all() and torch.isfinite(grads[0]).all()
        opt.step(grads)
        plain.step(grads)
        gone |= np.abs(plain.p[0]) > torch.finfo(F32).max
        assert np.array_equal(~torch.isfinite(params[0]).cpu().numpy(), gone) and gone.mean() < 0.01
        plain.pe[0][gone] = np.inf
        check(opt, plain)
        # handed out in bf16: every code is exact there but the lowest of blocks whose unit is below 2^-115, whose quanta (2^-18 of it) are below bf16's, 2^-133
        for have, want in zip(opt.moments_8bit(), (np.concatenate(plain.m), np.sqrt(np.concatenate(plain.v)))):
            assert torch.equal(have.cpu(), torch.from_numpy(want).to(BF16))
            assert np.array_equal(have.double().cpu().numpy()[256 * 14 * 3:], want[256 * 14 * 3:]) or order is not sizes


def test_units_of_both_moments_at_the_ends_of_fp32():
    """As test_tiny_and_huge_moments, the root's half: zeros below 2^-126, its own unit down to there, NaN where the unit would be 2^128 -- and from there on only."""
    p = tensors([1280], 1)[0]
    g = torch.zeros(1280)
    g[0], g[256], g[512], g[768], g[1024] = 1e-39, 1e-30, 1.0, 3.4e38, 3.1e38
    opt = AdamW([p], lr=0.0, betas=(0.0, 0.0), state_bits=8, small_numel=1, weight_decay=0.0)
    opt.step([g.to(DEV)])
    assert opt.root_exponents.tolist() == [0, 127 - 100, 127, 255, 254] and opt.exp_avg_exponents.tolist() == [0, 127 - 100, 127, 255, 254]
    m, r = (t.float().cpu() for t in opt.moments_8bit())
    for v, step in ((m, 2.0 ** -3), (r, 2.0 ** -4)):
        assert float(v[0]) == 0.0 and float(v[512]) == 1.0 and torch.isnan(v[768:1024]).all() and not v[1:256].any()
        assert abs(float(v[256]) / 1e-30 - 1) <= step and abs(float(v[1024]) / 3.1e38 - 1) <= step


def test_one_huge_gradient_leaves_its_block_alone():
    """A gradient whose square overflows fp32, for one step: what it leaves is finite, and the block goes on as the formula does."""
    params = tensors([1024], 2)
    opt, plain = AdamW(params, lr=1e-3, state_bits=8, small_numel=1, seed=3), Plain(params, [0.01], [8], 1e-3, (0.9, 0.999), 1e-8, seed=3)
    for k in range(3):
        grads = gradients(params, 60 + k)
        if k == 0:
            grads[0][300], grads[0][600] = 1e21, -3e38
        opt.step(grads)
        plain.step(grads)
        check(opt, plain)
        assert torch.isfinite(params[0]).all() and 255 not in opt.root_exponents.tolist()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_units_next_to_their_borders(dtype):
    """Blocks whose largest moment, or root, falls within a few roundings of the border between two units, from states and gradients chosen for it: 64 bits decide.
    One of them, m = 0.9 * -0.125 + 0.1 * 10.5, is 0.93749999999999978 in 64 bits and 0.9375000596 in 32, on both sides of a border."""
    b1, b2, blocks = 0.9, 0.999, 1500
    rng = np.random.default_rng(17)
    gm, gr = np.array(grid(3)), np.array(grid(4))
    n = 2 * blocks * 256
    cm, cr, g = rng.integers(0, 60, n).astype(np.uint8), rng.integers(0, 100, n).astype(np.uint8), 1e-6 * rng.standard_normal(n)
    near = torch.float32 if dtype is F32 else BF16

    def rounded(v, steps):                                           # v in the gradient's type, `steps` of its last place further
        t = torch.tensor(v, dtype=torch.float64).to(near)
        return float(t) + steps * float(t.abs()) * torch.finfo(near).eps / 2
    for b in range(2 * blocks):
        at, border = 256 * b + int(rng.integers(256)), 2.0 ** int(rng.integers(-3, 4))
        step = int(rng.integers(-2, 3)) if dtype is F32 else 0
        if b < blocks:                                               # the first moment, often out of a cancellation
            cm[at] = rng.integers(60, 127)
            sign = -1.0 if rng.random() < 0.5 else 1.0
            cm[at] |= 128 if sign < 0 else 0
            g[at] = rounded(((2 - 2.0 ** -3) * border - b1 * sign * gm[cm[at] & 127]) / (1 - b1), step)
        else:
            cr[at] = rng.integers(100, 200)
            g[at] = rounded(math.sqrt(max(((2 - 2.0 ** -4) * border) ** 2 - b2 * gr[cr[at]] ** 2, 1.0) / (1 - b2)), step)
    cm[0], g[0] = 128 + (12 << 3), 10.5
    grads = [torch.from_numpy(g).to(dtype).to(DEV)]
    params = [torch.zeros(n, device=DEV)]
    opt, plain = AdamW(params, lr=1e-3, betas=(b1, b2), state_bits=8, seed=2), Plain(params, [0.01], [8], 1e-3, (b1, b2), 1e-8, seed=2)
    opt.exp_avg_codes.copy_(torch.from_numpy(cm))
    opt.root_codes.copy_(torch.from_numpy(cr))
    opt.exp_avg_exponents.fill_(127)
    opt.root_exponents.fill_(127)
    plain.m[0][:] = np.where(cm >= 128, -1, 1) * gm[cm & 127]
    plain.v[0][:] = gr[cr] ** 2
    opt.step(grads)
    plain.step(grads)
    check(opt, plain)


@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_beside_the_tensors_is_written(bits):
    """Parameters, averages and copies as views of flat buffers with an element in front of, between and behind them, which keep their values; so do the states of
    tensors without a gradient, between the others'."""
    sizes = [1, 3, 255, 257, 2047, 2049, 700, 5000]
    total, mark = sum(sizes) + len(sizes) + 1, 0.7109375                     # (exact in 16 bits)
    flats = [torch.full((total,), mark, device=DEV), torch.full((total,), mark, device=DEV), torch.full((total,), mark, dtype=BF16, device=DEV)]
    starts = [1 + sum(sizes[:i]) + i for i in range(len(sizes))]
    cut = lambda flat: [flat[a:a + n] for a, n in zip(starts, sizes)]                              # noqa: E731
    guard = torch.ones(total, dtype=torch.bool, device=DEV)
    for a, n in zip(starts, sizes):
        guard[a:a + n] = False
    assert int(guard.sum()) == len(sizes) + 1
    params, ema, copies = map(cut, flats)
    opt = AdamW(params, lr=1e-2, state_bits=bits, small_numel=1, ema=ema, copies=copies, max_norm=1.0, seed=5)
    for k in range(3):
        grads = [None if k and i % 3 == 1 else g for i, g in enumerate(gradients(params, 40 + k, BF16))]
        held = {n: t.clone() for n, t in zip(opt._STATES[1:], opt._states()) if t is not None}
        opt.step(grads)
        for flat in flats:
            assert (flat[guard] == mark).all() and (flat[~guard] != mark).any()
        for name, old in held.items():
            unit = 256 if name.endswith("exponents") else 1
            for off, n, g in zip(opt._offsets, sizes, grads):
                a, b = off // unit, (off + (n if bits == 32 else -(-n // 256) * 256)) // unit
                assert g is not None or torch.equal(old[a:b], getattr(opt, name)[a:b]), (name, n)
    if bits == 8:                                                    # (the padding of a tensor's last block holds zeros)
        for off, n in zip(opt._offsets, sizes):
            end = off + -(-n // 256) * 256
            assert not (opt.exp_avg_codes[off + n:end] & 127).any() and not opt.root_codes[off + n:end].any()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_clipping_by_a_factor_below_fp32s_normal_range(bits, dtype):
    """Gradients near fp32's largest, clipped to a small norm: the factor, 1e-41, has a few bits in fp32; the scaled gradients are ordinary numbers."""
    params = tensors([1000, 300], 5)
    opt = AdamW(params, lr=1e-2, state_bits=bits, small_numel=1, max_norm=1e-2, seed=7)
    plain = Plain(params, [0.01] * 2, [bits] * 2, 1e-2, (0.9, 0.999), 1e-8, 1e-2, seed=7)
    for k in range(2):
        grads = [(g.double() / g.double().abs().max() * 3e38).to(dtype) for g in gradients(params, 70 + k)]
        opt.step(grads)
        plain.step(grads)
        check(opt, plain)


def test_gradients_that_negate_on_reading():
    """The imaginary part of a conjugate: the sign in memory is not the value's (one element has no strides that would have it copied)."""
    for n in (1, 7):
        z = torch.arange(1.0, n + 1, device=DEV).to(torch.complex64)
        g = (1j * z).conj().imag
        p, q = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
        assert g.is_neg() and float(g[0]) == -1.0
        AdamW([p], lr=0.5, weight_decay=0.0).step([g])
        AdamW([q], lr=0.5, weight_decay=0.0).step([g.clone()])
        assert torch.equal(p, q) and (p > 0).all()
        for bad in (lambda: AdamW([g[:1]]), lambda: AdamW([p[:1]], ema=[g[:1]])):
            with pytest.raises(CodepsHipError):
                bad()


def test_rows_without_gradients_in_eight_bits():
    """Blocks whose states and gradients are zeros, between others: they decay with the weight decay and keep zeros; they take part again as soon as a gradient comes,
    and stay in it when it goes.  Without an eps the formula is 0 / 0 there."""
    params = tensors([4096, 300], 6)
    opt = AdamW(params, lr=1e-2, weight_decay=0.1, state_bits=8, small_numel=1, seed=8)
    plain = Plain(params, [0.1] * 2, [8] * 2, 1e-2, (0.9, 0.999), 1e-8, seed=8)
    for k in range(4):
        grads = gradients(params, 80 + k)
        rows = grads[0].view(16, 256)
        rows[0], rows[3], rows[9:12], rows[15, :255] = 0.0, -0.0, 0.0, 0.0
        if k in (0, 2):
            rows[5], grads[1][:256] = 0.0, 0.0
        opt.step(grads)
        plain.step(grads)
        check(opt, plain)
        assert opt.exp_avg_exponents[0] == 0 and not opt.exp_avg_codes[:256].any() and not opt.root_codes[:256].any()
    q = torch.ones(512, device=DEV)
    g = torch.zeros(512, device=DEV)
    g[256:] = 1.0
    AdamW([q], lr=1e-2, eps=0.0, state_bits=8, small_numel=1).step([g])
    assert torch.isnan(q[:256]).all() and torch.isfinite(q[256:]).all()
