"""The dense operators without a device: refusals, argument checks of the C entries, modules and their state."""
import ctypes

import pytest
import torch

import granulelayer_b200 as gl
from granulelayer_b200 import _native


def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 16), torch.randn(8, 16)
    for call in (lambda: gl.linear_act(x, w), lambda: gl.linear_act(x.requires_grad_(True), w),
                 lambda: gl.group_norm_act(x, 4), lambda: gl.encode_activation(x.detach())):
        with pytest.raises(_native.NativeLibraryError):
            call()


@pytest.mark.parametrize("call", [
    lambda x, w: gl.linear_act(x, w[:, :15]), lambda x, w: gl.linear_act(x, w, torch.randn(7)),
    lambda x, w: gl.linear_act(x, w, None, torch.randn(4, 7)), lambda x, w: gl.linear_act(x, w.bfloat16()),
    lambda x, w: gl.linear_act(x.double(), w.double()), lambda x, w: gl.linear_act(x, w, activation="tanh"),
    lambda x, w: gl.linear_act(x, w, checkpoint="fp8"), lambda x, w: gl.linear_act(x, torch.randn(0, 16)),
    lambda x, w: gl.group_norm_act(x, 3), lambda x, w: gl.group_norm_act(x, 0),
    lambda x, w: gl.group_norm_act(x, 4, torch.ones(15)), lambda x, w: gl.group_norm_act(x[0], 4),
    lambda x, w: gl.group_norm_act(x, 4, eps=0.0), lambda x, w: gl.group_norm_act(x, 4, activation="tanh"),
    lambda x, w: gl.group_norm_act(x, 4, torch.ones(16), torch.ones(16).bfloat16()),
    lambda x, w: gl.group_norm_act(x.half(), 4), lambda x, w: gl.encode_activation(x.half()),
    lambda x, w: gl.encode_activation(torch.randn(3, 0)), lambda x, w: gl.LinearAct(0, 4),
    lambda x, w: gl.LinearAct(4, 4, dtype=torch.float16), lambda x, w: gl.GroupNormAct(10, 3),
    lambda x, w: gl.GroupNormAct(8, 2, activation="elu")])
def test_arguments_that_do_not_fit(call):
    with pytest.raises(ValueError):
        call(torch.randn(4, 16), torch.randn(8, 16))


def test_modules_are_seeded_and_load_state():
    a, b = gl.LinearAct(24, 10, seed=5, dtype=torch.float32), gl.LinearAct(24, 10, seed=5, dtype=torch.float32)
    assert torch.equal(a.weight, b.weight) and a.weight.shape == (10, 24) and not a.bias.any()
    assert not torch.equal(a.weight, gl.LinearAct(24, 10, seed=6, dtype=torch.float32).weight)
    assert abs(float(a.weight.detach().std()) - 24 ** -0.5) < 0.05
    n = gl.GroupNormAct(12, 3, dtype=torch.float32)
    assert set(n.state_dict()) == {"weight", "bias"} and set(a.state_dict()) == {"weight", "bias"}
    b.load_state_dict(a.state_dict())
    assert gl.LinearAct(4, 4, bias=False).bias is None and gl.GroupNormAct(4, 2, affine=False).weight is None
    a.enable_main_grad()
    a.weight.main_grad.fill_(1)
    a.zero_main_grad()
    assert a.weight.main_grad.dtype == torch.float32 and not a.weight.main_grad.any()


def test_c_entries_check_before_the_device():
    lib = _native.load()
    for fn in (lib.gl_linear_fwd, lib.gl_linear_bwd, lib.gl_norm_fwd, lib.gl_norm_bwd, lib.gl_act8_encode,
               lib.gl_act8_decode):
        assert fn(None, None) == -1
    a = _native.GlLinearArgs()
    a.M, a.N, a.K, a.ldx, a.ldw, a.ldy = 4, 8, 16, 15, 16, 8             # a row stride below the row
    assert lib.gl_linear_fwd(ctypes.byref(a), None) == -2
    a.ldx = 16
    assert lib.gl_linear_fwd(ctypes.byref(a), None) == -1                # null pointers
    a.act = 7
    assert lib.gl_linear_fwd(ctypes.byref(a), None) == -4
    a.act, a.slope_kind = 2, 9
    assert lib.gl_linear_fwd(ctypes.byref(a), None) == -4
    a.slope_kind, a.M = 0, 0                                             # no rows: nothing to do
    assert lib.gl_linear_fwd(ctypes.byref(a), None) == 0
    a.N = 0
    assert lib.gl_linear_fwd(ctypes.byref(a), None) == -2
    b = _native.GlLinearBwdArgs()
    b.M, b.N, b.K, b.lddy = 4, 8, 16, 8                                  # no output wanted: nothing to do
    assert lib.gl_linear_bwd(ctypes.byref(b), None) == 0
    b.dw, b.ldx = 1 << 20, 8
    assert lib.gl_linear_bwd(ctypes.byref(b), None) == -2                # x's row stride
    b.ldx = 16
    assert lib.gl_linear_bwd(ctypes.byref(b), None) == -1                # no dy
    b.dy, b.codes, b.exps, b.ldc = 1 << 20, (1 << 20) + 4, 1 << 20, 32
    assert lib.gl_linear_bwd(ctypes.byref(b), None) == -3                # codes not 16-byte aligned
    b.ldc = 48
    assert lib.gl_linear_bwd(ctypes.byref(b), None) == -2                # not whole blocks of 32 channels
    n = _native.GlNormArgs()
    n.S, n.P, n.C, n.G, n.px, n.eps = 2, 3, 10, 4, 10, 1e-5              # 10 channels in 4 groups
    assert lib.gl_norm_fwd(ctypes.byref(n), None) == -2
    n.G, n.pdtype = 5, 3
    assert lib.gl_norm_fwd(ctypes.byref(n), None) == -4
    n.pdtype = 0
    assert lib.gl_norm_fwd(ctypes.byref(n), None) == -1
    n.S = 0
    assert lib.gl_norm_fwd(ctypes.byref(n), None) == 0
    c = _native.GlAct8Args()
    c.rows, c.C, c.ldx, c.ldc = 3, 33, 33, 32
    assert lib.gl_act8_encode(ctypes.byref(c), None) == -2
    c.ldc = 64
    assert lib.gl_act8_encode(ctypes.byref(c), None) == -1
    c.rows = 0
    assert lib.gl_act8_decode(ctypes.byref(c), None) == 0
    assert lib.gl_linear_work_bytes(-1, 1, 1, 0, 0) == -2
    assert lib.gl_norm_work_bytes(1, 1, 10, 4, 0, 0) == -2
    assert lib.gl_status_string(-9) != b"unknown status"
