"""What the training-step operators of codeps_amd are measured on: the channel norms of a residual block (before the block; behind it with
gate, residual scale and the next block's norm) and the update of its parameters (AdamW over many tensors with 32-bit or 8-bit states, the
gradients' global norm).

`run(state)` with `own` false computes an operator in its plain form (elementary torch operations), with `own` true through codeps_amd."""
import torch

own = False

DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 256                    # elements of one tensor that share an exponent in the 8-bit states
SMALL = 4096                   # tensors with fewer elements keep 32-bit states
MANT_M, MANT_R = 3, 4          # stored mantissa bits: first moment (sign, 4, 3), root of the second moment (4, 4)
LOW = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------------------------------------------ cases
def _norm(name, items, per_item, channels, dtype, kind="layer", bias=True, grad=True, slack=0, offset=0.0):
    """channel_norm: `items` x `per_item` rows of `channels` values, rows `slack` values further apart than they are long."""
    return dict(name=name, op="norm", items=items, per_item=per_item, channels=channels, dtype=dtype, kind=kind, bias=bias, grad=grad, slack=slack,
                offset=offset)


def _residual(name, items, per_item, channels, dtype, res="same", kind="layer", bias=True, gate="none", act="none", scale=1.0, next="none",
              grad=True, slack=0, offset=0.0):
    return dict(name=name, op="residual", items=items, per_item=per_item, channels=channels, dtype=dtype, res=res, kind=kind, bias=bias, gate=gate,
                act=act, scale=scale, next=next, grad=grad, slack=slack, offset=offset)


def _adamw(name, layout, a, b, bits, grads="float32", max_norm=0.0, ema=False, copy=False, step=100):
    return dict(name=name, op="adamw", layout=layout, a=a, b=b, bits=bits, grads=grads, max_norm=max_norm, ema=ema, copy=copy, step=step)


def listed():
    return [
        # one row behind a pooled encoder map: what a call costs when there is next to nothing to compute
        _norm("norm one row", 1, 1, 2048, "bfloat16", kind="rms", bias=False, grad=False),
        # the stride-4 map of a batch of 8 images at 512 x 1024 in 16 bits, trained: the largest map a block of the encoder normalises
        _norm("norm stride 4", 8, 32768, 256, "bfloat16"),
        # 9 real channels of a map that is padded to 16 (class scores), odd height and width, large common offset
        _norm("norm padded classes", 2, 65 * 257, 9, "float32", slack=7, offset=3.0),
        # the block's end at stride 8: layer scale, residual, and the next block's norm in the same pass, trained
        _residual("residual stride 8", 8, 8192, 512, "float32", gate="channel", scale=0.5, next="layer"),
        # residual stream in 32 bits around 16-bit blocks, a gate per image, odd rows
        _residual("residual 32-bit stream", 5, 4097, 768, "bfloat16", res="float32", kind="rms", bias=False, gate="item", act="sigmoid", next="rms"),
        # inference on a handful of rows with an element-wise gate and an odd width
        _residual("residual few rows", 1, 77, 1000, "float16", gate="element", act="silu", grad=False),
        # a freshly started head: a dozen small tensors, 32-bit states
        _adamw("adamw head", "ragged", 12, 20000, 32, step=0),
        # a whole bottleneck network (3-4-6-3 blocks) with clipping and the averaged teacher copy, 32-bit states
        _adamw("adamw network", "bottleneck", 64, 3463, 32, max_norm=1.0, ema=True, step=1000),
        # the same network, 8-bit states, 16-bit gradients and a 16-bit working copy
        _adamw("adamw network 8 bit", "bottleneck", 64, 3463, 8, grads="bfloat16", max_norm=1.0, copy=True, step=1000),
        # wide matrices, 8-bit states: where the states' bytes are what counts
        _adamw("adamw wide 8 bit", "matrices", 6, 1440, 8, step=10),
        # the gradients' norm of the bottleneck network, and of the head's ragged set in 16 bits
        dict(name="grad norm network", op="grad_norm", layout="bottleneck", a=64, b=3463, grads="float32"),
        dict(name="grad norm head", op="grad_norm", layout="ragged", a=12, b=20000, grads="float16"),
    ]


def _log(rng, low, high):
    """An integer between low and high, spread over its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["norm", "norm", "residual", "residual", "residual", "adamw", "adamw", "adamw", "grad_norm"])
    if op in ("norm", "residual"):
        channels = _log(rng, 3, 8192)
        if rng.random() < 0.5:
            channels = (channels + 15) // 16 * 16
        rows = _log(rng, 1, max(1, (32 << 20) // channels))
        items = rng.choice([1, 2, 3, 8]) if rows >= 64 else 1
        c = dict(items=items, per_item=max(1, rows // items), channels=channels, dtype=rng.choice(list(TYPES)), kind=rng.choice(["layer", "rms"]),
                 bias=rng.random() < 0.5, grad=rng.random() < 0.7, slack=rng.choice([0, 0, 0, 16, 5]), offset=rng.choice([0.0, 0.0, 2.0]))
        c = dict(op=op, **c)
        if op == "residual":
            c.update(res=rng.choice(["same", "float32"]), kind=rng.choice(["layer", "rms", "none"]), gate=rng.choice(["none", "channel", "item", "element"]),
                     act=rng.choice(["none", "sigmoid", "silu"]), scale=rng.choice([1.0, 0.5, 0.1]), next=rng.choice(["none", "layer", "rms"]))
            if c["kind"] == "none":
                c["bias"] = False
            if c["gate"] == "none":
                c["act"] = "none"
        return c
    layout = rng.choice(["ragged", "ragged", "matrices", "bottleneck"])
    if layout == "ragged":
        a, b = _log(rng, 1, 300), _log(rng, 100, 1 << 20)
        b = min(b, (40 << 20) // a)
    elif layout == "matrices":
        a, b = rng.randint(1, 6), _log(rng, 64, 1400)
    else:
        a, b = rng.choice([8, 16, 24, 32, 48]), rng.choice([2222, 3463, 3333])
    c = dict(op=op, layout=layout, a=a, b=b, grads=rng.choice(list(TYPES)))
    if op == "adamw":
        c.update(bits=rng.choice([8, 32]), max_norm=rng.choice([0.0, 0.5, 100.0]), ema=rng.random() < 0.4, copy=rng.random() < 0.4, step=_log(rng, 1, 100000))
    return c


def _shapes(case):
    """(matrices, vectors) of a set of parameters: the vectors (norm scales, biases) take no weight decay."""
    a, b = case["a"], case["b"]
    if case["layout"] == "matrices":           # a blocks of a wide and a narrowing matrix with their biases
        return [s for _ in range(a) for s in ((4 * b, b), (b, 4 * b))], [s for _ in range(a) for s in ((4 * b,), (b,), (b,))]
    if case["layout"] == "ragged":             # a tensors, the largest of about b elements, sizes over four decades
        sizes = [max(1, int(b * 10.0 ** (-4.0 * ((i * 0.618034) % 1.0))) + i % 3) for i in range(a)]
        return [(n // 3, 3) for n in sizes if n >= 6 and n % 2], [(n,) for n in sizes if n < 6 or n % 2 == 0]
    mats, vecs, cin = [(a, 3, 7, 7)], [(a,), (a,)], a           # bottleneck network: a = stem width, b = the stages' block counts as digits
    for stage, blocks in enumerate(int(d) for d in str(b)):
        mid = a << stage
        for k in range(blocks):
            mats += [(mid, cin, 1, 1), (mid, mid, 3, 3), (4 * mid, mid, 1, 1)] + ([(4 * mid, cin, 1, 1)] if k == 0 else [])
            vecs += [(mid,)] * 4 + [(4 * mid,)] * (4 if k == 0 else 2)
            cin = 4 * mid
    return mats, vecs


def _numel(shape):
    n = 1
    for d in shape:
        n *= d
    return n


# ---------------------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)
    if case["op"] in ("norm", "residual"):
        return _prepare_norm(case, rand)
    return _prepare_step(case, seed, rand)


def _prepare_norm(case, rand):
    n, t, c, ty = case["items"], case["per_item"], case["channels"], TYPES[case["dtype"]]
    grad, offset = case["grad"], case["offset"]

    def rows(ty, spread=1.0):
        # rows of unequal size, like the activations behind a convolution; a few channels stand out
        v = rand(n, t, c + case["slack"])
        v *= torch.exp(0.5 * rand(n, t, 1)) * spread
        v += offset * rand(n, 1, c + case["slack"])
        return v.to(ty)[..., :c].detach().requires_grad_(grad)

    def vector(mean, spread, shape=(c,), ty=torch.float32):
        return (mean + spread * rand(*shape)).to(ty).requires_grad_(grad)
    s = {"op": case["op"], "kind": case["kind"], "eps": 1e-5, "x": rows(ty), "grad": grad}
    s["weight"] = vector(1.0, 0.2) if case["kind"] != "none" else None
    s["bias"] = vector(0.0, 0.2) if case["bias"] else None
    if case["op"] == "norm":
        s["dh"] = rand(n, t, c).to(ty) if grad else None
        s["inputs"] = [k for k in ("x", "weight", "bias") if s[k] is not None]
        return s
    rty = ty if case["res"] == "same" else torch.float32
    s["residual"] = rows(rty, 2.0)
    shape = {"none": None, "channel": (c,), "item": (n, 1, c), "element": (n, t, c)}[case["gate"]]
    s["gate"] = None if shape is None else vector(0.3, 0.5, shape, torch.float32 if case["gate"] == "channel" else ty)
    s["act"], s["scale"], s["next"] = case["act"], case["scale"], case["next"]
    s["next_weight"] = vector(1.0, 0.2) if case["next"] != "none" else None
    s["next_bias"] = vector(0.0, 0.2) if case["next"] == "layer" else None
    s["dy"] = rand(n, t, c).to(rty) if grad else None
    s["dh"] = rand(n, t, c).to(ty) if grad and case["next"] != "none" else None
    s["inputs"] = [k for k in ("x", "residual", "gate", "weight", "bias", "next_weight", "next_bias") if s[k] is not None]
    return s


def _prepare_step(case, seed, rand):
    mats, vecs = _shapes(case)
    shapes = mats + vecs
    sizes = [_numel(x) for x in shapes]
    total = sum(sizes)
    starts = [0]
    for k in sizes:
        starts.append(starts[-1] + k)

    def views(flat):
        return [flat[a:a + k].view(shape) for a, k, shape in zip(starts, sizes, shapes)]
    # gradients: noise whose size differs from tensor to tensor, and from row to row inside one
    size = torch.exp(1.5 * rand(len(sizes))).repeat_interleave(torch.tensor(sizes, device=DEV), output_size=total)
    wave = torch.exp(1.2 * torch.sin(torch.arange(total, device=DEV) * 0.037))
    spread = 1e-3 * size * wave
    g = (spread * rand(total)).to(TYPES[case["grads"]])
    s = {"op": case["op"], "g": g, "grads": views(g)}
    if case["op"] == "grad_norm":
        return s
    p = 0.05 * rand(total)
    s.update(p=p, sizes=sizes, decayed=len(mats), max_norm=case["max_norm"], lr=1e-3, betas=(0.9, 0.999), eps=1e-8, decay=0.01, seed=seed, ema_alpha=0.99)
    s["ema"] = p + 0.01 * rand(total) if case["ema"] else None
    s["copy"] = torch.empty(total, dtype=torch.bfloat16, device=DEV) if case["copy"] else None
    # states in the middle of a run: both moments belong to gradients of the same size; some tensors have seen fewer steps
    steps = torch.full((len(sizes),), case["step"], dtype=torch.int64, device=DEV)
    if case["step"] > 2:
        steps[::5] -= 2
    s["steps"] = steps
    m, r = 0.2 * spread * rand(total), spread * (0.5 + 0.5 * rand(total).abs())
    if case["step"] == 0:
        m.zero_()
        r.zero_()
    held8 = [case["bits"] == 8 and k >= SMALL for k in sizes]
    s["held8"] = held8
    if any(held8):
        at = torch.cat([_block_places(a, k) for a, k, q in zip(starts, sizes, held8) if q])
        s["places"] = at                                          # element of p behind every slot of the 8-bit states, -1: padding
        fill = (at >= 0).to(p.dtype)
        s["m_code"], s["m_exp"] = _encode(m[at.clamp(min=0)].double() * fill, None, MANT_M, True)
        s["r_code"], s["r_exp"] = _encode(r[at.clamp(min=0)].double() * fill, None, MANT_R, False)
    if not all(held8):
        at = None if not any(held8) else torch.cat([torch.arange(a, a + k, device=DEV) for a, k, q in zip(starts, sizes, held8) if not q])
        s["places32"] = at
        s["m"] = m.clone() if at is None else m[at]
        s["v"] = r.square() if at is None else r[at].square()
    if own:
        from codeps_amd import optim
        params, ema = views(p), None if s["ema"] is None else views(s["ema"])
        copies = None if s["copy"] is None else views(s["copy"])
        opt = optim.AdamW([{"params": params[:len(mats)], "weight_decay": s["decay"]}, {"params": params[len(mats):], "weight_decay": 0.0}],
                          lr=s["lr"], betas=s["betas"], eps=s["eps"], state_bits=case["bits"], small_numel=SMALL, ema=ema, ema_alpha=s["ema_alpha"],
                          copies=copies, max_norm=case["max_norm"] or None, seed=seed)
        state = {"steps": steps}
        if any(held8):
            state.update(exp_avg_codes=s["m_code"], exp_avg_exponents=s["m_exp"], root_codes=s["r_code"], root_exponents=s["r_exp"])
        if not all(held8):
            state.update(exp_avg=s["m"], exp_avg_sq=s["v"])
        opt.load_state_dict(state)
        s["opt"] = opt
    return s


def _block_places(start, n):
    at = torch.arange(-(-n // BLOCK) * BLOCK, device=DEV)
    return torch.where(at < n, at + start, -1)


# ------------------------------------------------------------------------------------------------------------------ 8-bit states, plain
def _two(e):
    """2^e in 64 bits for whole e, by the bits of the number itself."""
    return ((e + 1023) << 52).view(torch.float64)


def _encode(x, chance, mant, signed):
    """x [k * 256] (64 bits) -> codes and biased exponents of its blocks.  chance: 16 random bits per element; None rounds to nearest."""
    a = x.abs().view(-1, BLOCK)
    top = a.amax(1)
    f, e = torch.frexp(top)
    e = (e - 1 + (2 * f > 2.0 - 2.0 ** -mant)).to(torch.int64)             # the smallest exponent under which the block fits below 2 - 2^-mant
    held = torch.where(top < 2.0 ** -126, 0, torch.where(e > 127, 255, (e + 127).clamp(1, 254)))
    t = torch.where((held > 0)[:, None], a * _two((127 - held)[:, None]), 0.0)
    low = torch.where(t > 0, torch.frexp(t)[1].to(torch.int64) - 1, -14).clamp(min=-14)
    up = 0.5 if chance is None else chance.view(-1, BLOCK).double() / 65536.0
    q = torch.floor(t * _two(mant - low) + up).to(torch.int64)
    code = (((low + 14) << mant) + q).clamp(max=(16 << mant) - 1)
    if signed:
        code = code + 128 * (x.view(-1, BLOCK) < 0)
    return code.view(-1).to(torch.uint8), held.to(torch.uint8)


def _decode(code, held, mant, signed):
    code = code.to(torch.int64).view(-1, BLOCK)
    size = code & 127 if signed else code
    field, frac = size >> mant, size & ((1 << mant) - 1)
    v = torch.where(field == 0, frac, frac + (1 << mant)).double()
    v = v * _two(field.clamp(min=1) - 15 - mant + held.to(torch.int64)[:, None] - 127)
    v = torch.where((held == 255)[:, None], float("nan"), torch.where((held == 0)[:, None], 0.0, v))
    return (torch.where(code >= 128, -v, v) if signed else v).view(-1)


def _shift(z, k):
    return (z >> k) & ((1 << (64 - k)) - 1)


def _signed(c):
    return c - (1 << 64) if c >> 63 else c


def _keys(seed, tensors, steps):
    """Two 32-bit keys per tensor and step from a 64-bit multiply-xorshift mix of (seed, tensor's place, step)."""
    z = steps * _signed(0x9E3779B97F4A7C15) + tensors * _signed(0xD1B54A32D192ED03) + seed
    z = (z ^ _shift(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shift(z, 27)) * _signed(0x94D049BB133111EB)
    z = z ^ _shift(z, 31)
    return z & LOW, _shift(z, 32)


def _bits(i, k0, k1):
    """32 random bits of element i of a tensor with keys k0, k1: the low half rounds the first moment, the high half the root."""
    x = (i + (i >> 32) * 0x9E3779B1 + k0) & LOW
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & LOW
    x = x ^ (x >> 15) ^ k1
    x = (x * 0x846CA68B) & LOW
    return x ^ (x >> 16)


# ------------------------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(v, kind, weight, bias, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    v = v if weight is None else v * weight
    return v if bias is None else v + bias


def _plain_rows(s):
    x = s["x"].float()
    if s["op"] == "norm":
        return {"h": _plain_norm(x, s["kind"], s["weight"], s["bias"], s["eps"]).to(s["x"].dtype)}
    a = x if s["kind"] == "none" else _plain_norm(x, s["kind"], s["weight"], s["bias"], s["eps"])
    if s["gate"] is not None:
        g = s["gate"].float()
        a = a * (g if s["act"] == "none" else 1 / (1 + torch.exp(-g)) if s["act"] == "sigmoid" else g / (1 + torch.exp(-g)))
    y = s["residual"].float() + s["scale"] * a
    out = {"y": y.to(s["residual"].dtype)}
    if s["next"] != "none":
        out["h"] = _plain_norm(y, s["next"], s["next_weight"], s["next_bias"], s["eps"]).to(s["x"].dtype)
    return out


def _own_rows(s):
    from codeps_amd import functional as F
    if s["op"] == "norm":
        return {"h": F.channel_norm(s["x"], s["weight"], s["bias"], kind=s["kind"], eps=s["eps"])}
    none = lambda v: None if v == "none" else v                              # noqa: E731
    out = F.channel_norm_residual(s["x"], s["residual"], s["weight"], s["bias"], kind=none(s["kind"]), eps=s["eps"], gate=s["gate"],
                                  gate_act=none(s["act"]), scale=s["scale"], next_kind=none(s["next"]), next_weight=s["next_weight"],
                                  next_bias=s["next_bias"], next_eps=s["eps"])
    return {"y": out} if s["next"] == "none" else {"y": out[0], "h": out[1]}


def _plain_step(s):
    b1, b2 = s["betas"]
    s["steps"] += 1
    t = s["steps"].double()
    clip = torch.ones((), dtype=torch.float64, device=DEV)
    if s["max_norm"]:
        norm = s["g"].double().square().sum().sqrt()
        clip = torch.where(norm > s["max_norm"], s["max_norm"] / norm, clip)
    n = len(s["sizes"])
    first = torch.arange(n, device=DEV) < s["decayed"]
    keep = 1 - s["lr"] * s["decay"] * first.double()
    rate = s["lr"] / (1 - b1 ** t)
    root = (1 - b2 ** t).rsqrt()
    sizes = torch.tensor(s["sizes"], device=DEV)
    held8 = torch.tensor(s["held8"], device=DEV)
    p, out = s["p"], {"p": s["p"]}
    if "m" in s:
        at, count = s["places32"], torch.where(held8, 0, sizes)

        def each(v):
            return v.float().repeat_interleave(count, output_size=s["m"].numel())
        g = (s["g"] if at is None else s["g"][at]).float() * clip.float()
        s["m"].mul_(b1).add_((1 - b1) * g)
        s["v"].mul_(b2).add_((1 - b2) * g * g)
        new = (p if at is None else p[at]) * each(keep) - each(rate) * s["m"] / (s["v"].sqrt() * each(root) + s["eps"])
        if at is None:
            p.copy_(new)
        else:
            p[at] = new
        out.update(m=s["m"], v=s["v"])
    if "m_code" in s:                        # in 64 bits: a value next to a border between two codes has to fall on its own side
        at = s["places"]
        real, at = at >= 0, at.clamp(min=0)
        count = torch.where(held8, (sizes + BLOCK - 1) // BLOCK * BLOCK, 0)

        def each(v):
            return v.repeat_interleave(count, output_size=at.numel())
        g = s["g"][at].double() * clip * real
        m = b1 * _decode(s["m_code"], s["m_exp"], MANT_M, True) + (1 - b1) * g
        v = b2 * _decode(s["r_code"], s["r_exp"], MANT_R, False).square() + (1 - b2) * g * g
        new = p[at].double() * each(keep) - each(rate) * m / (v.sqrt() * each(root) + s["eps"])
        p[at[real]] = new[real].float()
        k0, k1 = _keys(s["seed"], torch.arange(n, device=DEV), s["steps"])
        inside = torch.arange(at.numel(), device=DEV) - each(torch.cumsum(count, 0) - count)
        chance = _bits(inside, each(k0), each(k1))
        for code, held, v, c, mant, signed in (("m_code", "m_exp", m, chance & 65535, MANT_M, True), ("r_code", "r_exp", v.sqrt(), chance >> 16, MANT_R, False)):
            s[code], s[held] = _encode(v, c, mant, signed)
            out[code[0] + "8"] = _decode(s[code], s[held], mant, signed)[real].to(torch.bfloat16)
    if s["ema"] is not None:
        s["ema"].mul_(s["ema_alpha"]).add_((1 - s["ema_alpha"]) * p)
        out["ema"] = s["ema"]
    if s["copy"] is not None:
        s["copy"].copy_(p)
        out["copy"] = s["copy"]
    return out


def _own_step(s):
    opt = s["opt"]
    opt.step(s["grads"])
    out = {"p": s["p"]}
    if "m" in s:
        out.update(m=opt.exp_avg, v=opt.exp_avg_sq)
    if "m_code" in s:
        out["m8"], out["r8"] = opt.moments_8bit()
    if s["ema"] is not None:
        out["ema"] = s["ema"]
    if s["copy"] is not None:
        out["copy"] = s["copy"]
    return out


def run(s):
    if s["op"] == "adamw":
        return _own_step(s) if own else _plain_step(s)
    if s["op"] == "grad_norm":
        if own:
            from codeps_amd import functional as F
            return {"norm": F.grad_norm(s["grads"])}
        return {"norm": s["g"].double().square().sum().sqrt().float()}
    rows = _own_rows if own else _plain_rows
    if not s["grad"]:
        with torch.no_grad():
            return rows(s)
    out = rows(s)
    names = [k for k in ("y", "h") if k in out]
    grads = torch.autograd.grad([out[k] for k in names], [s[k] for k in s["inputs"]], [s["d" + k] for k in names])
    return {**{k: out[k].detach() for k in names}, **{"d" + k: g for k, g in zip(s["inputs"], grads)}}


# -------------------------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Bytes: every input once, every output once.  Operations: the formulas' multiplications and additions."""
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    if case["op"] in ("norm", "residual"):
        n = case["items"] * case["per_item"] * case["channels"]
        x, grad = size[case["dtype"]], case["grad"]
        if case["op"] == "norm":
            return {"bytes": n * (2 * x + (2 * x if grad else 0)), "flops": n * (8 + (14 if grad else 0))}
        r = x if case["res"] == "same" else 4
        gate = x if case["gate"] == "element" else 0
        h = x if case["next"] != "none" else 0
        # forward: x, residual, gate -> y, h; backward: dy, dh, (x, residual, gate, read once already) -> dx, dresidual, dgate
        return {"bytes": n * (x + r + gate + r + h + ((r + h + x + r + gate) if grad else 0)), "flops": n * (18 + (36 if grad else 0))}
    sizes = [_numel(x) for part in _shapes(case) for x in part]
    total, g = sum(sizes), size[case["grads"]]
    if case["op"] == "grad_norm":
        return {"bytes": total * g, "flops": 2 * total}
    held8 = sum(k for k in sizes if case["bits"] == 8 and k >= SMALL)
    # parameter in and out, gradient in, states in and out (8 bits: codes and exponents, and the values that are handed out), copies
    per = 8 + g + (8 if case["ema"] else 0) + (2 if case["copy"] else 0)
    return {"bytes": total * per + (total - held8) * 16 + held8 * (4 + 4.0 / BLOCK + 4), "flops": total * 16}


# ------------------------------------------------------------------------------------------------------------------ 64 bits, on its own
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        if case["op"] == "grad_norm":
            return {"norm": sum((g.double() ** 2).sum() for g in s["grads"]) ** 0.5}
        return _exact_rows(s) if case["op"] in ("norm", "residual") else _exact_step(s)


def _centred(v, kind, eps):
    """(normalised rows, 1 / deviation) of v."""
    mu = v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else 0.0
    d = v - mu
    rho = 1.0 / torch.sqrt((d ** 2).sum(-1, keepdim=True) / v.shape[-1] + eps)
    return d * rho, rho


def _centred_back(du, u, rho, kind):
    c = u.shape[-1]
    out = du - u * (du * u).sum(-1, keepdim=True) / c
    if kind == "layer":
        out = out - du.sum(-1, keepdim=True) / c
    return rho * out


def _exact_rows(s):
    wide = {k: None if s.get(k) is None else s[k].detach().double() for k in ("x", "residual", "gate", "weight", "bias", "next_weight", "next_bias", "dy", "dh")}
    one = torch.ones((), dtype=torch.float64, device=DEV)
    w = one if wide["weight"] is None else wide["weight"]
    b = 0.0 if wide["bias"] is None else wide["bias"]
    rowsum = lambda v: v.sum(tuple(range(v.dim() - 1)))                      # noqa: E731
    x = wide["x"]
    if s["kind"] == "none":
        u, rho = x, None
    else:
        u, rho = _centred(x, s["kind"], s["eps"])
    a = u * w + b
    out = {}
    if s["op"] == "norm":
        out["h"] = a
        da = wide["dh"]
    else:
        if wide["gate"] is None:
            act, slope = one, None
        else:
            g = wide["gate"]
            sig = torch.special.expit(g)
            act, slope = {"none": (g, torch.ones_like(g)), "sigmoid": (sig, sig * (1 - sig)), "silu": (g * sig, sig * (1 + g * (1 - sig)))}[s["act"]]
        y = wide["residual"] + s["scale"] * act * a
        out["y"] = y
        back = wide["dy"]
        if s["next"] != "none":
            un, rhon = _centred(y, s["next"], s["eps"])
            nw = wide["next_weight"]
            out["h"] = un * nw + (0.0 if wide["next_bias"] is None else wide["next_bias"])
            if s["grad"]:
                back = back + _centred_back(wide["dh"] * nw, un, rhon, s["next"])
                out["dnext_weight"] = rowsum(wide["dh"] * un)
                if wide["next_bias"] is not None:
                    out["dnext_bias"] = rowsum(wide["dh"])
        if s["grad"]:
            out["dresidual"] = back
            da = s["scale"] * act * back
            if slope is not None:
                dg = s["scale"] * a * back * slope
                out["dgate"] = rowsum(dg) if s["gate"].dim() == 1 else dg.sum(1, keepdim=True) if s["gate"].shape[1] == 1 and dg.shape[1] > 1 else dg
    if s["grad"]:
        if wide["weight"] is not None:
            out["dweight"] = rowsum(da * u)
        if wide["bias"] is not None:
            out["dbias"] = rowsum(da)
        out["dx"] = da if s["kind"] == "none" else _centred_back(da * w, u, rho, s["kind"])
    return out


def _exact_step(s):
    b1, b2 = s["betas"]
    clip = 1.0
    if s["max_norm"]:
        norm = float(sum((g.double() ** 2).sum() for g in s["grads"]) ** 0.5)
        clip = min(1.0, s["max_norm"] / norm)
    tables, powers = {}, torch.tensor([2.0 ** k for k in range(-127, 129)], dtype=torch.float64, device=DEV)
    for mant in (MANT_M, MANT_R):              # every magnitude that a code stands for, in order
        low = [k * 2.0 ** (-14 - mant) for k in range(1 << mant)]
        tables[mant] = torch.tensor(low + [(1 + k / (1 << mant)) * 2.0 ** e for e in range(-14, 1) for k in range(1 << mant)], dtype=torch.float64, device=DEV)

    def values(code, held, mant, signed):
        c = code.long()
        v = tables[mant][c % 128 if signed else c]
        v = v * torch.where(held == 0, 0.0, powers[held.long()]).repeat_interleave(BLOCK)
        return torch.where(c >= 128, -v, v) if signed else v

    def stored(x, chance, mant):
        """Each |x| goes to one of its two neighbours among the block's values, to the upper one with the odds of its place between them."""
        k = -(-x.numel() // BLOCK)
        a = torch.zeros(k * BLOCK, dtype=torch.float64, device=DEV)
        a[:x.numel()] = x.abs()
        top = a.view(k, BLOCK).max(1).values
        unit = powers[torch.searchsorted((2 - 2.0 ** -mant) * powers, top).clamp(1, 255)]       # the smallest that the block fits under
        unit = torch.where(top < 2.0 ** -126, 0.0, unit).repeat_interleave(BLOCK)[:x.numel()]
        t = torch.where(unit > 0, x.abs() / unit, 0.0)
        grid = torch.cat([tables[mant], torch.tensor([2.0], dtype=torch.float64, device=DEV)])
        lo = torch.searchsorted(grid, t, right=True) - 1
        below, above = grid[lo], grid[lo + 1]
        up = (t - below) / (above - below) + chance.double() / 65536.0 >= 1.0
        return torch.where(x < 0, -1.0, 1.0) * torch.where(up, above, below) * unit
    out = {k: [] for k in ("p", "m", "v", "m8", "r8")}
    start, slot, slot32, mask = 0, 0, 0, (1 << 64) - 1
    for i, (n, q, done) in enumerate(zip(s["sizes"], s["held8"], s["steps"].tolist())):
        t = done + 1
        g, p = s["g"][start:start + n].double() * clip, s["p"][start:start + n].double()
        if q:
            k = -(-n // BLOCK)
            part, head = slice(slot * BLOCK, slot * BLOCK + k * BLOCK), slice(slot, slot + k)
            m = values(s["m_code"][part], s["m_exp"][head], MANT_M, True)[:n]
            v = values(s["r_code"][part], s["r_exp"][head], MANT_R, False)[:n] ** 2
            slot += k
        else:
            m, v = s["m"][slot32:slot32 + n].double(), s["v"][slot32:slot32 + n].double()
            slot32 += n
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        p = p * (1 - s["lr"] * (s["decay"] if i < s["decayed"] else 0.0)) - s["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + s["eps"])
        out["p"].append(p)
        if q:
            z = (s["seed"] + t * 0x9E3779B97F4A7C15 + i * 0xD1B54A32D192ED03) & mask
            z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
            z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
            z = z ^ (z >> 31)
            at = torch.arange(n, device=DEV)
            x = (at + (at // 2 ** 32) * 0x9E3779B1 + z % 2 ** 32) % 2 ** 32
            x = ((x ^ (x // 65536)) * 0x7FEB352D) & LOW
            x = ((x ^ (x // 32768) ^ (z // 2 ** 32)) * 0x846CA68B) & LOW
            x = x ^ (x // 65536)
            out["m8"].append(stored(m, x % 65536, MANT_M))
            out["r8"].append(stored(torch.sqrt(v), x // 65536, MANT_R))
        else:
            out["m"].append(m)
            out["v"].append(v)
        start += n
    out = {k: torch.cat(v) for k, v in out.items() if v}
    if s["ema"] is not None:
        out["ema"] = s["ema_alpha"] * s["ema"].double() + (1 - s["ema_alpha"]) * out["p"]
    if s["copy"] is not None:
        out["copy"] = out["p"]
    return out
