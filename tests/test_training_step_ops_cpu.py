"""Refusals of the channel norms, AdamW and the gradient norm that need no GPU: CPU tensors, and the C entries' own checks (made before any launch)."""
import ctypes

import pytest
import torch

from codeps_amd import _lib
from codeps_amd import functional as F
from codeps_amd._lib import CodepsHipError
from codeps_amd.optim import AdamW


def test_cpu_tensors_are_refused():
    x = torch.zeros(3, 4)
    for call in (lambda: F.channel_norm(x), lambda: F.channel_norm_residual(x, x), lambda: AdamW([x]), lambda: F.grad_norm([x])):
        with pytest.raises(CodepsHipError, match="GPU only"):
            call()


def test_wrong_kinds_of_arguments_are_refused():
    x = torch.zeros(3, 4)
    for call in (lambda: F.channel_norm(None), lambda: F.channel_norm([1.0]), lambda: F.channel_norm(x, 3), lambda: F.channel_norm(x, eps="small"),
                 lambda: F.channel_norm(x, kind="batch"), lambda: F.channel_norm_residual(x, next_kind="x"), lambda: F.channel_norm_residual(x, gate_act="gelu"),
                 lambda: F.channel_norm_residual(x, scale=None), lambda: F.grad_norm(None), lambda: F.grad_norm([1.0]), lambda: F.grad_norm([])):
        with pytest.raises(CodepsHipError):
            call()
    native = _lib.bind()
    for call in (lambda: native.channel_norm(x), lambda: native.grad_norm(), lambda: native.adamw_step([], []), lambda: native.init(1)):
        with pytest.raises(TypeError):
            call()
    numels, places = (ctypes.c_longlong * 1)(12), (ctypes.c_ulonglong * 1)(x.data_ptr())
    block = _lib.StepBlock(n_items=1, numels=ctypes.addressof(numels), addresses=ctypes.addressof(places))
    at = ctypes.addressof(block)
    for args in (([x], [], [x], 0), ([x], [], [x], None), ([x], [], [], at), ([x, x], [], [x, x], at), ([1], [], [x], at), ([x], [], [2], at), ([x], None, [x], at),
                 ([x], [], [x], at)):
        with pytest.raises(CodepsHipError):
            native.adamw_step(*args, 1.0, 0.0, False, 0.9)


def _desc(**over):
    d = _lib.ChannelNormDesc()
    values = dict(rows=4, x_pitch=8, res_pitch=8, gate_pitch=8, dy_pitch=8, dh_pitch=8, channels=8, rows_per_item=1, full=1, kind=1, next_kind=0, gate_mode=0,
                  gate_act=0, x_type=0, res_type=0, weight_type=0, gate_type=0, next_weight_type=0, scale=1.0, eps=1e-5, next_eps=1e-5)
    for k, v in {**values, **over}.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over", [dict(rows=-1), dict(rows=1 << 31), dict(channels=0), dict(channels=8193), dict(x_type=3), dict(res_type=1), dict(x_type=1, res_type=2),
                                  dict(kind=3), dict(next_kind=-1), dict(gate_mode=4), dict(gate_act=3), dict(gate_mode=2, rows_per_item=0),
                                  dict(gate_mode=2, rows_per_item=3), dict(x_pitch=7), dict(res_pitch=7), dict(gate_mode=3, gate_pitch=7), dict(full=0, kind=0),
                                  dict(full=0, next_kind=1), dict(gate_mode=3, gate_type=1), dict(x_pitch=1 << 24), dict(dy_pitch=1 << 24), dict(full=0, gate_mode=1), dict(weight_type=9), dict(gate_type=-1)])
def test_channel_norm_descriptor_is_checked(over):
    lib, d, none = _lib.lib(), _desc(**over), [None] * 12
    assert lib.codeps_channel_norm_fwd(ctypes.byref(d), *none[:11]) == -1 and lib.codeps_last_error()
    assert lib.codeps_channel_norm_bwd_workspace_bytes(ctypes.byref(d)) == 0
    assert lib.codeps_channel_norm_bwd(ctypes.byref(d), *[None] * 16, 0, None, 0, None) == -1


def test_channel_norm_null_pointers_and_workspaces_are_refused():
    lib, d = _lib.lib(), _desc()
    fake = ctypes.c_void_p(64)                                       # never read: every one of these calls ends in the host's checks
    assert lib.codeps_channel_norm_fwd(None, *[None] * 11) == -1
    assert lib.codeps_channel_norm_fwd(ctypes.byref(d), *[None] * 11) == -1
    assert lib.codeps_channel_norm_fwd(ctypes.byref(_desc(next_kind=1)), fake, fake, None, None, None, None, None, fake, None, None, None) == -1
    assert lib.codeps_channel_norm_fwd(ctypes.byref(_desc(x_type=1)), fake, None, None, None, None, None, None, fake, None, None, None) == -1     # y in fp32 without a residual
    assert lib.codeps_channel_norm_fwd(ctypes.byref(_desc(gate_mode=1)), fake, fake, None, None, None, None, None, fake, None, None, None) == -1
    need = lib.codeps_channel_norm_bwd_workspace_bytes(ctypes.byref(d))
    assert need > 0
    args = [fake] * 16
    assert lib.codeps_channel_norm_bwd(ctypes.byref(d), *args, 0, fake, need - 1, None) == -2
    assert lib.codeps_channel_norm_bwd(ctypes.byref(d), *args, 0, None, need, None) == -2
    assert lib.codeps_channel_norm_bwd(ctypes.byref(d), *args, 16, fake, need, None) == -1
    assert lib.codeps_channel_norm_bwd(ctypes.byref(_desc(weight_type=1)), *args, 1, fake, need, None) == -1
    assert lib.codeps_channel_norm_bwd(ctypes.byref(_desc(dy_pitch=7)), *args, 0, fake, need, None) == -1
    apart = [fake] * 9 + [64 * (i + 2) for i in range(7)]
    for i in range(10, 16):                                          # two gradients at one address
        assert lib.codeps_channel_norm_bwd(ctypes.byref(d), *apart[:i], apart[i - 1], *apart[i + 1:], 0, fake, need, None) == -1
    no_dy = list(apart)
    no_dy[7] = None                                                  # neither dy nor a next norm
    assert lib.codeps_channel_norm_bwd(ctypes.byref(d), *no_dy, 0, fake, need, None) == -1
    assert lib.codeps_channel_norm_fwd(ctypes.byref(_desc(rows=0)), *[None] * 11) == 0


def test_adamw_entries_check_their_arguments():
    lib = _lib.lib()
    size = lib.codeps_adamw_item_bytes()
    buf = ctypes.create_string_buffer(size)
    item, fake = ctypes.addressof(buf), 64
    good = [item, fake, None, None, 0, 5000, 8, 256, 0, 0, 0]
    assert lib.codeps_adamw_item_fill(*good) == 3                    # chunks of 2048 elements
    for at, value in ((0, None), (1, None), (5, -1), (6, 16), (7, 255), (7, -256), (8, -1), (9, 16), (9, -1), (10, -1), (1, 66)):
        bad = list(good)
        bad[at] = value
        assert lib.codeps_adamw_item_fill(*bad) < 0, (at, value)
    assert lib.codeps_adamw_item_fill(item, fake, None, fake, 0, 10, 32, 0, 0, 0, 0) < 0          # a copy in fp32
    assert lib.codeps_adamw_workspace_bytes(0) == 0 and lib.codeps_grad_norm_workspace_bytes(0) == 0
    need = lib.codeps_adamw_workspace_bytes(1)
    group = (_lib.AdamWGroup * 1)(_lib.AdamWGroup(1e-3, 0.9, 0.999, 1e-8, 0.0, None))
    chunk0, grads, types, numels = (ctypes.c_longlong * 2)(0, 3), (ctypes.c_void_p * 1)(fake), (ctypes.c_ubyte * 1)(0), (ctypes.c_longlong * 1)(5000)

    def step(**over):
        a = dict(items=fake, n=1, map=fake, chunk0=chunk0, grads=grads, types=types, numels=numels, groups=group, ng=1, steps=fake, m=fake, v=fake, mc=None, me=None,
                 rc=None, re=None, scale=1.0, max_norm=0.0, skip=0, norm=None, seed=0, alpha=0.9, ws=fake, bytes=need, stream=None)
        a.update(over)
        return lib.codeps_adamw_step(*a.values())
    bad_group = lambda **f: (_lib.AdamWGroup * 1)(_lib.AdamWGroup(*{**dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, lr_device=None), **f}.values()))  # noqa: E731
    for over in (dict(items=None), dict(map=None), dict(chunk0=None), dict(grads=None), dict(types=None), dict(numels=None), dict(groups=None), dict(steps=None), dict(n=0),
                 dict(ng=0), dict(ng=17), dict(v=None), dict(m=None, v=None), dict(mc=fake), dict(ws=None), dict(types=(ctypes.c_ubyte * 1)(3)),
                 dict(grads=(ctypes.c_void_p * 1)(66)), dict(numels=(ctypes.c_longlong * 1)(-1)), dict(numels=(ctypes.c_longlong * 1)(7000)),
                 dict(groups=bad_group(beta1=1.0)), dict(groups=bad_group(beta2=-0.1)), dict(groups=bad_group(eps=-1.0)), dict(groups=bad_group(beta1=float("nan")))):
        assert step(**over) == -1, over
    assert step(bytes=need - 1) == -2
    assert lib.codeps_adamw_moments_8bit(fake, 1, fake, 0, fake, fake, fake, fake, fake, fake, None) == -1
    assert lib.codeps_grad_norm(grads, types, numels, 1, 1.0, None, fake, 1 << 20, None) == -2
    assert lib.codeps_grad_norm(None, types, numels, 1, 1.0, fake, fake, 1 << 20, None) == -1


def test_struct_layouts():
    assert ctypes.sizeof(_lib.ChannelNormDesc) == 112 and _lib.ChannelNormDesc.channels.offset == 48 and _lib.ChannelNormDesc.scale.offset == 96
    assert ctypes.sizeof(_lib.StepBlock) == 19 * 8
    assert ctypes.sizeof(_lib.AdamWGroup) == 48 and _lib.AdamWGroup.lr_device.offset == 40


def test_forward_mode_derivatives_are_refused():
    """Every tensor of a call, on its own: a dual tensor's derivative is not dropped silently (refused before the device is looked at)."""
    import torch.autograd.forward_ad as forward
    x, v = torch.ones(3, 4), torch.ones(4)
    with forward.dual_level():
        dx, dv = forward.make_dual(x, x), forward.make_dual(v, v)
        for call in (lambda: F.channel_norm(dx), lambda: F.channel_norm(x, dv), lambda: F.channel_norm(x, v, dv), lambda: F.channel_norm_residual(dx),
                     lambda: F.channel_norm_residual(x, dx), lambda: F.channel_norm_residual(x, gate=dv), lambda: F.channel_norm_residual(x, next_kind="rms", next_weight=dv),
                     lambda: F.channel_norm_residual(x, next_kind="rms", next_weight=v, next_bias=dv), lambda: F.grad_norm([dx])):
            for mode in (torch.enable_grad(), torch.no_grad()):
                with mode, pytest.raises(CodepsHipError, match="forward-mode"):
                    call()


def test_gradient_norm_of_tensors_that_require_a_gradient_is_refused():
    """It would come back as a constant; under no_grad that is what is asked for (and the call goes on to the next check: the device)."""
    plain, leaf = torch.ones(3), torch.nn.Parameter(torch.ones(3))
    (graph,) = torch.autograd.grad((leaf ** 3).sum(), [leaf], create_graph=True)
    for t in (leaf, graph):
        with pytest.raises(CodepsHipError, match="no derivative"):
            F.grad_norm([t, plain])
        with torch.no_grad(), pytest.raises(CodepsHipError, match="GPU only"):
            F.grad_norm([t, plain])
        with pytest.raises(CodepsHipError, match="GPU only"):
            F.grad_norm([t.detach(), plain])


def test_a_trace_is_refused():
    """torch.jit.trace would keep the example's outputs as constants."""
    x = torch.ones(3, 4)
    for call in (F.channel_norm, lambda v: F.channel_norm_residual(v, v), lambda v: F.grad_norm([v])):
        with pytest.raises(CodepsHipError, match="trace"):
            torch.jit.trace(call, (x,))
    with pytest.raises(CodepsHipError, match="trace"):
        torch.jit.trace(lambda v: v + _lib.bind().adamw_step([v], [], [v], 0, 1.0, 0.0, False, 0.9), (x,))
    with pytest.raises(CodepsHipError, match="GPU only"):             # (and nothing of it stays behind)
        F.channel_norm(x)


def test_adamw_of_one_tensor_instead_of_a_list_is_refused():
    """list(tensor) are views of its rows, which never have a gradient: nothing would ever move."""
    for params in (torch.zeros(3), torch.nn.Parameter(torch.zeros(2, 3))):
        with pytest.raises(CodepsHipError, match="a list of parameters"):
            AdamW(params)
