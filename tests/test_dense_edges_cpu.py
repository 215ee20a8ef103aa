"""What the dense operators have to refuse or carry along before a kernel sees it; no device."""
import ctypes

import pytest
import torch

import granulelayer_b200 as gl
from granulelayer_b200 import _native, dense


# ---- main_grad ----

def test_a_main_grad_on_another_device_is_refused():
    """The kernels write main_grad by its address, so it has to lie where the parameter does."""
    p = torch.nn.Parameter(torch.empty(8, 4, device="meta"))
    b = torch.nn.Parameter(torch.empty(8, device="meta"))
    p.main_grad = torch.zeros(8, 4)
    with pytest.raises(ValueError, match="device"):
        dense._grad_buffers(p, True, b, True)
    with pytest.raises(ValueError, match="device"):
        dense._grad_buffers(p, True, None, False)
    dw, db, main = dense._grad_buffers(p, False, b, True)     # not wanted: not looked at
    assert dw is None and db.device.type == "meta" and not main
    p.main_grad = torch.zeros(8, 4, device="meta")
    dw, db, main = dense._grad_buffers(p, True, b, True)
    assert dw is p.main_grad and db.dtype == torch.float32 and main


@pytest.mark.parametrize("make", [lambda: gl.LinearAct(8, 4), lambda: gl.GroupNormAct(8, 2)])
def test_main_grad_moves_with_its_module(make):
    """main_grad follows its parameter to another device, and stays fp32 when the parameters change type."""
    lay = make()
    lay.enable_main_grad()
    for p in lay.parameters():
        p.main_grad.fill_(3)
    net = torch.nn.Sequential(lay)
    net.to(torch.float32)
    for p in lay.parameters():
        assert p.dtype == torch.float32 and p.main_grad.dtype == torch.float32 and bool((p.main_grad == 3).all())
    net.to("meta")
    for p in lay.parameters():
        assert p.main_grad.device.type == "meta" and p.main_grad.dtype == torch.float32
        assert p.main_grad.shape == p.shape
    net.to_empty(device="cpu")                                # nothing to carry from there: zeros
    for p in lay.parameters():
        assert p.main_grad.device.type == "cpu" and not p.main_grad.any()


# ---- C entries: alignment ----

A = 1 << 20                       # an address that no check refuses; nothing is read through it


def linear_args(dtype=0):
    a = _native.GlLinearArgs()
    a.x = a.w = a.bias = a.residual = a.y = a.slope = A
    a.M, a.N, a.K, a.ldx, a.ldw, a.ldr, a.ldy, a.lds = 64, 8, 16, 16, 16, 8, 8, 8
    a.dtype, a.act, a.slope_kind = dtype, 2, 1 if dtype == 0 else 2
    return a


def linear_bwd_args(dtype=0):
    a = _native.GlLinearBwdArgs()
    a.dy = a.slope = a.x = a.w = a.dx = a.dw = a.db = A
    a.M, a.N, a.K, a.lddy, a.lds, a.ldx, a.ldw, a.lddx = 64, 8, 16, 8, 8, 16, 16, 16
    a.dtype, a.slope_kind = dtype, 1 if dtype == 0 else 2
    return a


def norm_args(dtype=0):
    a = _native.GlNormArgs()
    a.x = a.w = a.b = a.y = a.mean = a.rstd = a.work = A
    a.S, a.P, a.C, a.G, a.sx, a.px, a.work_bytes = 2, 3, 8, 2, 24, 8, 1 << 20
    a.dtype, a.pdtype, a.eps = dtype, dtype, 1e-5
    return a


def norm_bwd_args(dtype=0):
    a = _native.GlNormBwdArgs()
    a.dy = a.x = a.w = a.b = a.mean = a.rstd = a.dx = a.dw = a.db = a.work = A
    a.S, a.P, a.C, a.G, a.sx, a.px, a.sdy, a.pdy, a.work_bytes = 2, 3, 8, 2, 24, 8, 24, 8, 1 << 20
    a.dtype, a.pdtype = dtype, dtype
    return a


def act8_args(dtype=0):
    a = _native.GlAct8Args()
    a.x = a.out = a.codes = a.exps = A
    a.rows, a.C, a.ldx, a.ldc, a.dtype = 3, 32, 32, 32, dtype
    return a


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("entry,make,fields", [
    ("gl_linear_fwd", linear_args, ("x", "w", "bias", "residual", "y", "slope")),
    ("gl_linear_bwd", linear_bwd_args, ("dy", "slope", "x", "w", "dx", "dw", "db")),
    ("gl_norm_fwd", norm_args, ("x", "w", "b", "y", "mean", "rstd", "work")),
    ("gl_norm_bwd", norm_bwd_args, ("dy", "x", "w", "b", "mean", "rstd", "dx", "dw", "db", "work")),
    ("gl_act8_encode", act8_args, ("x",)), ("gl_act8_decode", act8_args, ("out",))])
def test_c_entries_refuse_pointers_off_their_type(entry, make, fields, dtype):
    """A pointer that its element type (or, for a workspace, 16 bytes) does not divide would fault the kernel: the
    entry says GL_ERR_ALIGN (-3) before it looks for a device."""
    fn = getattr(_native.load(), entry)
    for f in fields:
        a = make(dtype)
        setattr(a, f, A + (8 if f == "work" else 1))
        assert fn(ctypes.byref(a), None) == -3, f


def test_accumulated_gradients_are_fp32_pointers():
    """With `accumulate` dw and db are fp32 whatever the storage type: two-byte alignment is not enough."""
    lib = _native.load()
    for fn, make in ((lib.gl_linear_bwd, linear_bwd_args), (lib.gl_norm_bwd, norm_bwd_args)):
        for f in ("dw", "db"):
            a = make(1)
            a.accumulate = 1
            setattr(a, f, A + 2)
            assert fn(ctypes.byref(a), None) == -3


# ---- products whose waits ran out ----

def test_a_wait_that_ran_out_is_raised_by_the_next_call(monkeypatch):
    """The kernels set a word in host memory; the next call reads it, resets it and raises."""
    t = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(_native, "_wait_word", (t, ctypes.c_int32.from_address(t.data_ptr()), t.data_ptr()))
    assert _native._wait_status() == t.data_ptr()
    t.fill_(1)
    with pytest.raises(_native.NativeLibraryError, match="ran out"):
        _native._wait_status()
    assert _native._wait_status() == t.data_ptr() and int(t) == 0


@pytest.mark.parametrize("entry,make", [("gl_linear_fwd", linear_args), ("gl_linear_bwd", linear_bwd_args)])
def test_the_status_word_is_an_aligned_int32(entry, make):
    a = make(1)
    a.status = A + 2
    assert getattr(_native.load(), entry)(ctypes.byref(a), None) == -3
