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
