"""AdamW over many tensors at once, with 32-bit or 8-bit states (C ABI: codeps_adamw_*).

    opt = AdamW([{"params": matrices, "weight_decay": 1e-2}, {"params": vectors, "weight_decay": 0.0}], lr=1e-4, state_bits=8, max_norm=1.0)
    loss.backward(); opt.step(); opt.zero_grad()

Next to functional.adam_ema_step (Adam on flat fp32 buffers): decoupled weight decay, parameters that lie anywhere, gradients of any of the three float
types, global-norm clipping inside the step, 8-bit states.  A step is two launches for up to 320 tensors,
with clipping three for up to 160.
Step counts, the clipping factor and the random bits of the 8-bit rounding live on the device: a captured step() replays as the next step.
"""
import ctypes

import torch

from . import functional as F
from ._lib import AdamWGroup, CodepsHipError, StepBlock, bind, check, lib, ptr, require_cuda, stream_ptr

BLOCK = 256                     # elements of one tensor that share an exponent byte
CHUNK = 2048                    # elements of one tensor that a work group updates
MAX_GROUPS = 16


def _at(t):
    return None if t is None else t.data_ptr()


def _dense(t):
    """Whether t's elements fill one stretch of memory, in any order of its dimensions (contiguous, channels-last, ...)."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _same_layout(a, b):
    return a.shape == b.shape and (a.stride() == b.stride() or (a.is_contiguous() and b.is_contiguous()))


class AdamW:
    """m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)

    Not a torch.optim.Optimizer: torch's learning-rate schedulers do not take it.  Set param_groups[i]["lr"] between steps, or give a device scalar.

    params: fp32 tensors on one device, or dicts {"params": [...]} with their own lr, betas, eps, weight_decay, state_bits (at most 16).
        Parameters in 16 bits would lose every update below half a step: keep them in fp32 and ask for `copies`.
    lr: a float, or an fp32 device scalar that the step reads when it runs (schedules inside a captured graph).
    state_bits: 32 (fp32 moments), or 8 for tensors of `small_numel` elements or more: m as sign / 4 / 3 bits and sqrt(v) as 4 / 4 bits of floating
        point, each block of 256 elements with its own power of two, rounded stochastically (seed): 2 bytes per element instead of 8.
    ema, ema_alpha: per parameter an fp32 tensor (or None) that follows it: ema = alpha ema + (1 - alpha) p, also where a parameter has no gradient.
    copies: per parameter a bf16 / fp16 tensor (or None) that receives the updated parameter.
    max_norm: gradients are scaled by min(1, max_norm / norm) with the norm over all of them; `grad_norm` holds it after a step.
    skip_nonfinite: a step whose norm is not finite changes nothing at all."""

    def __init__(self, params, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, small_numel=4096, ema=None, ema_alpha=0.99,
                 copies=None, max_norm=None, skip_nonfinite=False, seed=0):
        if torch.is_tensor(params):
            raise CodepsHipError("AdamW: a list of parameters, got one tensor (its rows would be the parameters, without its gradient)")
        params = list(params)
        if not params:
            raise CodepsHipError("AdamW: no parameters")
        groups = [dict(g) for g in params] if isinstance(params[0], dict) else [{"params": params}]
        if len(groups) > MAX_GROUPS:
            raise CodepsHipError(f"AdamW: {len(groups)} groups, at most {MAX_GROUPS}")
        self.param_groups, self.params, self._bits, group_of = [], [], [], []
        for i, g in enumerate(groups):
            ps = g["params"]
            ps = [ps] if torch.is_tensor(ps) else list(ps)
            unknown = set(g) - {"params", "lr", "betas", "eps", "weight_decay", "state_bits"}
            if unknown:
                raise CodepsHipError(f"AdamW: unknown group options {sorted(unknown)}")
            full = {"params": ps, "lr": g.get("lr", lr), "betas": tuple(g.get("betas", betas)), "eps": g.get("eps", eps),
                    "weight_decay": g.get("weight_decay", weight_decay), "state_bits": g.get("state_bits", state_bits)}
            if full["state_bits"] not in (8, 32):
                raise CodepsHipError(f"AdamW: states have 32 or 8 bits, not {full['state_bits']}")
            self.param_groups.append(full)
            self.params += ps
            self._bits += [8 if full["state_bits"] == 8 and p.numel() >= small_numel else 32 for p in ps]
            group_of += [i] * len(ps)
        if not self.params:
            raise CodepsHipError("AdamW: no parameters")
        dev = self.params[0].device
        seen = set()
        for p in self.params:
            require_cuda(p)
            if p.dtype != torch.float32 or p.device != dev:
                raise CodepsHipError(f"AdamW: fp32 parameters on one device, got {p.dtype} on {p.device} (16-bit weights: `copies` of fp32 ones)")
            if not _dense(p) or p.is_neg():
                raise CodepsHipError(f"AdamW: a parameter of shape {tuple(p.shape)} with strides {p.stride()} is not dense, or is a view that negates")
            if p.numel() and p.data_ptr() in seen:
                raise CodepsHipError("AdamW: a parameter is listed twice")
            seen.add(p.data_ptr())
        n = len(self.params)
        self.device, self._groups_of = dev, group_of
        self._ema = self._beside(ema, (torch.float32,), "ema")
        self._copies = self._beside(copies, (torch.bfloat16, torch.float16), "copies")
        self.ema_alpha, self.max_norm, self.skip_nonfinite, self.seed = float(ema_alpha), max_norm, bool(skip_nonfinite), int(seed)
        if max_norm is not None and not max_norm > 0:
            raise CodepsHipError(f"AdamW: max_norm = {max_norm}")
        if not 0.0 <= self.ema_alpha <= 1.0:
            raise CodepsHipError(f"AdamW: ema_alpha = {ema_alpha}")
        # ---- states: the 32-bit tensors packed, the 8-bit ones in whole blocks
        self._numels = [p.numel() for p in self.params]
        self._offsets, self._packed, chunk0, n32, n8, packed = [], [], [0], 0, 0, 0
        for k, bits in zip(self._numels, self._bits):
            self._offsets.append(n32 if bits == 32 else n8)
            self._packed.append(packed)
            if bits == 32:
                n32 += k
            else:
                n8 += -(-k // BLOCK) * BLOCK
                packed += k
            chunk0.append(chunk0[-1] + -(-k // CHUNK))
        zeros = lambda count, dtype: torch.zeros(count, dtype=dtype, device=dev) if count else None          # noqa: E731
        self.steps = zeros(n, torch.int64)
        self.exp_avg, self.exp_avg_sq = zeros(n32, torch.float32), zeros(n32, torch.float32)
        self.exp_avg_codes, self.root_codes = zeros(n8, torch.uint8), zeros(n8, torch.uint8)
        self.exp_avg_exponents, self.root_exponents = zeros(n8 // BLOCK, torch.uint8), zeros(n8 // BLOCK, torch.uint8)
        if n32 == 0 and n8 == 0:                                  # (empty tensors only: the C ABI wants a state)
            self.exp_avg, self.exp_avg_sq = (torch.zeros(1, device=dev) for _ in range(2))
        self._n8 = packed
        want_norm = max_norm is not None or self.skip_nonfinite
        self.grad_norm = torch.zeros((), dtype=torch.float32, device=dev) if want_norm else None
        # ---- launch tables (csrc/bind.cpp: the step's constant part is handed over as one structure)
        self._chunk0 = (ctypes.c_longlong * (n + 1))(*chunk0)
        self._n_chunks = chunk0[-1]
        counts = torch.tensor([b - a for a, b in zip(chunk0, chunk0[1:])])
        self._chunk_items = torch.repeat_interleave(torch.arange(n, dtype=torch.int32), counts).to(dev) if chunk0[-1] else torch.zeros(1, dtype=torch.int32, device=dev)
        self._c_numels = (ctypes.c_longlong * n)(*self._numels)
        self._c_groups = (AdamWGroup * len(self.param_groups))()
        self._shapes = [p.shape for p in self.params]
        self._items = torch.zeros(n * lib().codeps_adamw_item_bytes(), dtype=torch.uint8, device=dev)
        self._by = [t for t in self._ema + self._copies if t is not None]
        for t in self.params + self._by:                          # a replayed step rewrites them and no version tells: weight packs go by the epoch
            t._codeps_volatile = True
        self._c_addresses = (ctypes.c_ulonglong * (n + len(self._by)))()
        self._fill_items()
        self._ws = torch.empty(lib().codeps_adamw_workspace_bytes(n), dtype=torch.uint8, device=dev)
        self._c_step = StepBlock(self._items.data_ptr(), n, self._chunk_items.data_ptr(), ctypes.addressof(self._chunk0), ctypes.addressof(self._c_numels),
                                 ctypes.addressof(self._c_groups), len(self.param_groups), self.steps.data_ptr(), *map(_at, self._states()), _at(self.grad_norm),
                                 self._ws.data_ptr(), self._ws.numel(), self.seed, ctypes.addressof(self._c_addresses))

    def _beside(self, tensors, dtypes, what):
        """ema / copies: one tensor (or None) per parameter, with its shape and layout."""
        tensors = [None] * len(self.params) if tensors is None else list(tensors)
        if len(tensors) != len(self.params):
            raise CodepsHipError(f"AdamW: {what}: one entry per parameter ({len(self.params)}), got {len(tensors)}")
        for p, t in zip(self.params, tensors):
            if t is not None and (t.dtype not in dtypes or t.device != self.device or not _same_layout(t, p) or t.is_neg()):
                raise CodepsHipError(f"AdamW: {what}: {tuple(t.shape)} {t.dtype} on {t.device} does not go with a parameter of {tuple(p.shape)}")
        return tensors

    def _fill_items(self):
        """(Re)writes the device table in place: a captured step reads the same table."""
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in self.params + self._by if t.numel())
        if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
            raise CodepsHipError("AdamW: parameters, EMA tensors or copies share memory")
        size = lib().codeps_adamw_item_bytes()
        host = ctypes.create_string_buffer(size * len(self.params))
        base = ctypes.addressof(host)
        for i, (p, e, c) in enumerate(zip(self.params, self._ema, self._copies)):
            k = lib().codeps_adamw_item_fill(base + i * size, p.data_ptr() or None, ptr(e), ptr(c), 0 if c is None else F._TYPES[c.dtype], self._numels[i],
                                             self._bits[i], self._offsets[i], self._packed[i], self._groups_of[i], self._chunk0[i])
            if k < 0:
                raise CodepsHipError("codeps_adamw_item_fill: " + lib().codeps_last_error().decode())
        self._items.copy_(torch.frombuffer(bytearray(host.raw), dtype=torch.uint8))
        self._c_addresses[:] = [t.data_ptr() for t in self.params + self._by]

    def _states(self):
        return self.exp_avg, self.exp_avg_sq, self.exp_avg_codes, self.exp_avg_exponents, self.root_codes, self.root_exponents

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()

    def step(self, grads=None, *, grad_scale=1.0, apply_ema=True):
        """One update of every parameter that has a gradient.  grads: one tensor (or None) per parameter in the order of `params`; default: their .grad.
        The others keep value, states and step count.  Behind the replay of a captured step, functional.invalidate_weight_cache() before eager convolutions with
        these tensors.  grad_scale multiplies the gradients (1 / world size after a summing all-reduce); apply_ema False
        leaves the EMA tensors alone."""
        params = self.params
        grads = [p.grad for p in params] if grads is None else list(grads)
        for c, g in zip(self._c_groups, self.param_groups):
            lr = g["lr"]
            if torch.is_tensor(lr):
                if lr.numel() != 1 or lr.dtype != torch.float32 or lr.device != self.device:
                    raise CodepsHipError("AdamW.step: lr is a float or an fp32 scalar on the parameters' device")
                c.lr, c.lr_device = 0.0, lr.data_ptr()
            else:
                c.lr, c.lr_device = lr, None
            (c.beta1, c.beta2), c.eps, c.weight_decay = g["betas"], g["eps"], g["weight_decay"]
        rest = (ctypes.addressof(self._c_step), grad_scale, self.max_norm or 0.0, self.skip_nonfinite, self.ema_alpha if apply_ema else -1.0)
        state = bind().adamw_step(params, self._by, grads, *rest)
        if state & 1:
            if [p.shape for p in params] != self._shapes or any(p.dtype != torch.float32 or p.device != self.device or not _dense(p) for p in params):
                raise CodepsHipError("AdamW.step: a parameter has changed its shape, type, layout or device since it was listed")
            if torch.cuda.is_current_stream_capturing():
                raise CodepsHipError("AdamW.step: a parameter (or a tensor beside it) has moved since the last step: run one step before the capture")
            self._beside(self._ema, (torch.float32,), "ema")
            self._beside(self._copies, (torch.bfloat16, torch.float16), "copies")
            self._fill_items()
        if state & 2:
            if not all(map(_dense, params)):
                raise CodepsHipError("AdamW.step: a parameter has changed its layout since it was listed")
            with torch.no_grad():
                grads = [g if g is None or _same_layout(g, p) and not g.is_neg() else torch.empty_like(p, dtype=g.dtype).copy_(g) for g, p in zip(grads, params)]
        if state and bind().adamw_step(params, self._by, grads, *rest):
            raise CodepsHipError("AdamW.step: a parameter or gradient changes under the step")
        F.invalidate_weight_cache()

    def moments_8bit(self):
        """(m, sqrt(v)) that the 8-bit states stand for, exact in bf16 (down to its 2^-133): the 8-bit tensors one after another, without padding."""
        if not self._n8:
            raise CodepsHipError("AdamW.moments_8bit: no tensor has 8-bit states")
        m = torch.empty(self._n8, dtype=torch.bfloat16, device=self.device)
        r = torch.empty_like(m)
        with torch.cuda.device(self.device):
            check(lib().codeps_adamw_moments_8bit(ptr(self._items), len(self.params), ptr(self._chunk_items), self._n_chunks, *map(ptr, self._states()[2:]), ptr(m),
                                                  ptr(r), stream_ptr()), "codeps_adamw_moments_8bit")
        return m, r

    def __reduce__(self):
        raise CodepsHipError("AdamW holds device addresses: pass on its state_dict()")

    _STATES = ("steps", "exp_avg", "exp_avg_sq", "exp_avg_codes", "exp_avg_exponents", "root_codes", "root_exponents")

    def state_dict(self):
        state = {k: getattr(self, k).clone() for k in self._STATES if getattr(self, k) is not None}
        state["param_groups"] = [{k: (float(v) if torch.is_tensor(v) else v) for k, v in g.items() if k != "params"} for g in self.param_groups]
        return state

    def load_state_dict(self, state):
        """States (and, where given, the groups' options; an lr that lives on the device is written there) of an optimizer over the same shapes and bits."""
        for k in self._STATES:
            have, got = getattr(self, k), state.get(k)
            if (have is None) != (got is None) or (have is not None and (have.shape != got.shape or have.dtype != got.dtype)):
                raise CodepsHipError(f"AdamW.load_state_dict: {k} does not fit")
        groups = state.get("param_groups", [])
        if groups and (len(groups) != len(self.param_groups) or any(a.get("state_bits", b["state_bits"]) != b["state_bits"] for a, b in zip(groups, self.param_groups))):
            raise CodepsHipError("AdamW.load_state_dict: other groups or state bits")
        for k in self._STATES:
            if getattr(self, k) is not None:
                getattr(self, k).copy_(state[k])
        for g, new in zip(self.param_groups, groups):
            for k, v in new.items():
                if k == "lr" and torch.is_tensor(g["lr"]):
                    g["lr"].fill_(v)
                elif k != "params":
                    g[k] = tuple(v) if k == "betas" else v
