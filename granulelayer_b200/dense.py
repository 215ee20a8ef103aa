"""Dense operators around sparse-pooling layers (no counterpart in the reference).

``linear_act``          y = act(x W^T + b) + residual, forward and backward;
``group_norm_act``      channels-last group norm with an affine map and an activation, forward and backward;
``encode_activation`` / ``decode_activation``   an activation in 8 bits and back;
``LinearAct`` / ``GroupNormAct``                the first two as modules, with the framework's ``main_grad``.

``checkpoint="int8"`` makes the first two keep what their backward pass reads in 8 bits: the input as int8 codes
with one power-of-two scale per 32 channels (1.03 bytes per element), and ``linear_act`` the activation's
derivative as one byte (multiples of 1/192, exact at 0 and 1).  The forward result does not change.  The gradients are
the usual formulas with the read-back input in the input's place, and with what the forward pass found: act'(z) of the
original z (in steps of 1/192) for ``linear_act``, mean and 1 / deviation of the original input for ``group_norm_act``.
They are close to those at the original input, and exactly those of no input.

Storage is float32 or bfloat16; sums and statistics are float32.  The kernels run in the in-tree sm_100a library on
the current CUDA stream; there is no CPU path (``NativeLibraryError``) and nothing falls back to PyTorch math.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch import nn

from . import _native

BLOCK = 32        # channels that share an exponent in an 8-bit checkpoint
CHECKPOINTS = ("none", "int8")
_DTYPES = (torch.float32, torch.bfloat16)


_ACT_IDS = _native.DENSE_ACT_IDS


def _act_id(activation: str) -> int:
    act = _ACT_IDS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {tuple(_ACT_IDS)}, not {activation!r}")
    return act


def _check_checkpoint(checkpoint: str):
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"checkpoint must be one of {CHECKPOINTS}, not {checkpoint!r}")


def _check_tensors(name: str, x: torch.Tensor, dtype, **tensors):
    """``x`` of a supported dtype on a GPU; every other given tensor on its device and, where one is named, of
    ``dtype``."""
    if x.dtype not in _DTYPES or dtype not in _DTYPES:
        raise ValueError(f"{name}: float32 or bfloat16 tensors, not {x.dtype if x.dtype not in _DTYPES else dtype}")
    for k, t in tensors.items():
        if t is not None and t.dtype != dtype:
            raise ValueError(f"{name}: {k} is {t.dtype}, expected {dtype}")
        if t is not None and t.device != x.device:
            raise ValueError(f"{name}: {k} is on {t.device}, the input on {x.device}")
    _native._require_cuda(x)


def _no_double_backward(name: str):
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name}: the backward pass is not differentiable (create_graph=True)")


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` [..., width] as [rows, width] with unit column stride and rows that do not overlap (a copy where the
    strides allow no such view)."""
    t2 = t if t.dim() == 2 else t.reshape(-1, width)
    if (width > 1 and t2.stride(1) != 1) or t2.stride(0) < width:
        t2 = t2.contiguous()
        if t2.stride(0) < width or (width > 1 and t2.stride(1) != 1):   # one row or column: any stride is "contiguous"
            t2 = t2.as_strided(t2.shape, (width, 1))
    return t2


# ---- 8-bit checkpoints ----

@dataclass(frozen=True)
class Activation8:
    """An activation [..., C] in 8 bits: ``codes`` [rows, C rounded up to 32] int8, ``exponents`` [rows,
    ceil(C / 32)] uint8, and the shape and dtype it had.  A value is code * 2^(exponent - 127); a block that held a
    NaN or an infinity has exponent 255 and reads back as NaN."""
    codes: torch.Tensor
    exponents: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype

    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()


def _encode(x2: torch.Tensor):
    rows, C = x2.shape
    nblk = -(-C // BLOCK)
    codes = x2.new_empty((rows, nblk * BLOCK), dtype=torch.int8)
    exps = x2.new_empty((rows, nblk), dtype=torch.uint8)
    if rows:
        _native.act8_encode(x2, codes, exps)
    return codes, exps


def encode_activation(x: torch.Tensor) -> Activation8:
    """``x`` [..., C] (float32 or bfloat16) in 8 bits."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"encode_activation: x needs at least one channel, got shape {tuple(x.shape)}")
    _check_tensors("encode_activation", x, x.dtype)
    codes, exps = _encode(_rows(x.detach(), x.shape[-1]))
    return Activation8(codes, exps, tuple(x.shape), x.dtype)


def decode_activation(a: Activation8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values of ``a`` in ``dtype`` (default: what it was); exact in both float32 and bfloat16."""
    dtype = dtype or a.dtype
    if dtype not in _DTYPES:
        raise ValueError(f"decode_activation: float32 or bfloat16, not {dtype}")
    out = torch.empty(a.shape, dtype=dtype, device=a.codes.device)
    if out.numel():
        _native.act8_decode(a.codes, a.exponents, out.view(-1, a.shape[-1]))
    else:
        _native._require_cuda(a.codes)
    return out


def _empty_as(t: torch.Tensor) -> torch.Tensor:
    """Contiguous uninitialised memory of ``t``'s shape and type (empty_like is the cheapest call for it)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


# ---- gradients of parameters ----

def _grad_buffers(weight, need_w: bool, bias, need_b: bool):
    """(weight's buffer, bias's buffer, accumulate): where their gradients go (None: not wanted).  With a ``main_grad``
    on either, both buffers are fp32 and added to (fresh zeros for one without), as SparsePoolingLayer's are."""
    need_w, need_b = need_w and weight is not None, need_b and bias is not None
    main = (need_w and hasattr(weight, "main_grad") and weight.main_grad is not None or
            need_b and hasattr(bias, "main_grad") and bias.main_grad is not None)
    if not main:
        return _empty_as(weight) if need_w else None, _empty_as(bias) if need_b else None, False
    out = []
    for p, want in ((weight, need_w), (bias, need_b)):
        g = getattr(p, "main_grad", None) if want else None
        if g is not None and (g.dtype != torch.float32 or not g.is_contiguous() or g.shape != p.shape):
            raise ValueError("main_grad must be a contiguous float32 tensor of the parameter's shape")
        if g is not None and g.device != p.device:      # the kernels take its address
            raise ValueError(f"main_grad is on device {g.device}, its parameter on {p.device}")
        out.append(g if g is not None or not want else torch.zeros(p.shape, dtype=torch.float32, device=p.device))
    return out[0], out[1], True


def _returned(p, buf, main: bool):
    """What autograd gets for a parameter: None for ``main_grad``, else the buffer in the parameter's dtype."""
    if buf is None or not main:
        return buf
    return None if getattr(p, "main_grad", None) is not None else buf.to(p.dtype)


# ---- linear ----

# act'(z) as the backward pass keeps it: as it is in fp32 layers, in steps of 2^-14 (bf16 would cost the gradient a
# second rounding to 8 bits) in bf16 ones, in steps of 1/192 in an 8-bit checkpoint
_SLOPE_DTYPES = {torch.float32: torch.float32, torch.bfloat16: torch.int16}


def _linear_forward(x2, weight, bias, r2, act, slope):
    y = x2.new_empty((x2.shape[0], weight.shape[0]))
    if x2.shape[0]:
        _native.linear_fwd(x2, weight, bias, r2, y, slope, act)
    return y


class LinearActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, checkpoint):
        N, K = weight.shape
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        x2, w2 = _rows(x, K), _rows(weight, K)
        slope = codes = exps = None
        if act != 0 and (need_x or need_w or need_b):
            slope = x2.new_empty((x2.shape[0], N), dtype=torch.uint8 if checkpoint == "int8" else _SLOPE_DTYPES[x.dtype])
        y = _linear_forward(x2, w2, bias, None if residual is None else _rows(residual, N), act, slope)
        if not need_w:                                   # only dW reads x
            x2 = None
        elif checkpoint == "int8":
            codes, exps = _encode(x2)
            x2 = None
        ctx.save_for_backward(x2, codes, exps, weight if need_x or need_w else None, bias if need_b else None, slope)
        ctx.xshape, ctx.K = x.shape, K
        return y if x.dim() == 2 else y.view(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        _no_double_backward("linear_act")
        x2, codes, exps, weight, bias, slope = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        N, K = dy.shape[-1], ctx.K
        dx = w2 = None
        if need_x:
            dx, w2 = dy.new_empty(ctx.xshape), _rows(weight, K)
        dw, db, main = _grad_buffers(weight, need_w, bias, need_b)
        if need_x or dw is not None or db is not None:
            _native.linear_bwd(_rows(dy, N), slope, x2, codes, exps, w2, dx, dw, db, K, main)
        return dx, _returned(weight, dw, main), _returned(bias, db, main), dy if need_r else None, None, None


def _check_linear(x, weight, bias, residual):
    """Raises for arguments that do not belong together."""
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"linear_act: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    N = weight.shape[0]
    if bias is not None and (bias.shape != (N,) or (N > 1 and bias.stride(0) != 1)):
        raise ValueError(f"linear_act: bias must be a contiguous [{N}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != x.shape[:-1] + (N,):
        raise ValueError(f"linear_act: residual {tuple(residual.shape)} must have the output's shape "
                         f"{tuple(x.shape[:-1]) + (N,)}")
    _check_tensors("linear_act", x, x.dtype, weight=weight, bias=bias, residual=residual)


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, activation: str = "identity",
               checkpoint: str = "none") -> torch.Tensor:
    """act(x W^T + bias) + residual for x [..., K], weight [N, K], bias [N], residual [..., N].

    ``activation``: "identity", "relu", "gelu" (erf form) or "silu".  ``checkpoint="int8"`` keeps the input and the
    activation's derivative in 8 bits for the backward pass.  All tensors share one dtype (float32 or bfloat16;
    float32 products run as exact three-term bf16 splits on the tensor cores, where an infinity in x, weight or an output
    gradient gives NaN, or in fp32 for up to 8 rows).  bfloat16 layers round the gradient of z to bfloat16 before its products.
    Parameters with a ``main_grad`` receive their gradients there."""
    act = _ACT_IDS.get(activation)
    xs, ws, dt, dev = x.shape, weight.shape, x.dtype, x.device
    # one expression for what is right; the exact complaint is _check_linear's
    if not (act is not None and checkpoint in CHECKPOINTS and dt in _DTYPES and x.is_cuda and len(ws) == 2 and
            len(xs) > 0 and xs[-1] == ws[1] and 0 not in ws and weight.dtype == dt and weight.device == dev and
            (bias is None or bias.shape == ws[:1] and bias.dtype == dt and bias.device == dev and bias.is_contiguous())
            and (residual is None or residual.shape == xs[:-1] + ws[:1] and residual.dtype == dt and
                 residual.device == dev)):
        _act_id(activation)
        _check_checkpoint(checkpoint)
        _check_linear(x, weight, bias, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    bias is not None and bias.requires_grad or
                                    residual is not None and residual.requires_grad):
        return LinearActFunction.apply(x, weight, bias, residual, act, checkpoint)
    N, K = weight.shape
    y = _linear_forward(_rows(x, K), _rows(weight, K), bias, None if residual is None else _rows(residual, N), act,
                        None)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


# ---- group norm ----

def _positions(t: torch.Tensor, S: int, P: int, C: int) -> torch.Tensor:
    """``t`` [S, ..., C] as [S, P, C] with unit channel stride and positions that do not overlap."""
    if t.is_contiguous() and C > 1:      # strides of dimensions of size one may still be anything
        return t.as_strided((S, P, C), (P * C, C, 1))
    t3 = t.reshape(S, P, C)
    if (C > 1 and t3.stride(2) != 1) or (P > 1 and t3.stride(1) < C) or (S > 1 and t3.stride(0) < C):
        t3 = t3.contiguous()
    if t3.stride(1) < C or t3.stride(0) < C or (C == 1 and t3.stride(2) != 1):
        t3 = t3.as_strided(t3.shape, (t3.stride(0) if S > 1 else P * C, t3.stride(1) if P > 1 else C, 1))
    return t3


def _norm_forward(x, num_groups, weight, bias, act, eps):
    S, C = x.shape[0], x.shape[-1]
    y = _empty_as(x)
    stats = x.new_empty((2, S, num_groups), dtype=torch.float32)   # mean, rstd
    x3 = None
    n = x.numel()
    if n:
        x3 = _positions(x, S, n // (S * C), C)
        _native.norm_fwd(x3, weight, bias, y, stats, num_groups, act, eps)
    return y, x3, stats


class GroupNormActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, act, eps, checkpoint):
        y, x3, stats = _norm_forward(x, num_groups, weight, bias, act, eps)
        codes = exps = None
        if checkpoint == "int8" and x3 is not None:
            codes, exps = _encode(_rows(x3, x.shape[-1]))
            x3 = None
        ctx.save_for_backward(x3, codes, exps, weight, bias, stats)
        ctx.act, ctx.groups = act, num_groups
        return y

    @staticmethod
    def backward(ctx, dy):
        _no_double_backward("group_norm_act")
        x3, codes, exps, weight, bias, stats = ctx.saved_tensors
        _, need_w, need_b = ctx.needs_input_grad[:3]
        dx = _empty_as(dy)
        dw, db, main = _grad_buffers(weight, need_w, bias, need_b)
        S, C = dy.shape[0], dy.shape[-1]
        if dx.numel():
            dy3 = _positions(dy, S, dx.numel() // (S * C), C)
            _native.norm_bwd(dy3, x3, codes, exps, weight, bias, stats, dx, dw, db, ctx.groups, ctx.act, main)
        elif not main:
            for g in (dw, db):
                if g is not None:
                    g.zero_()
        return dx, _returned(weight, dw, main), _returned(bias, db, main), None, None, None, None


def _check_norm(x, num_groups, weight, bias, eps):
    """Raises for arguments that do not belong together."""
    if x.dim() < 2 or x.shape[-1] < 1:
        raise ValueError(f"group_norm_act: x must be [samples, ..., channels], got {tuple(x.shape)}")
    C = x.shape[-1]
    if num_groups < 1 or C % num_groups:
        raise ValueError(f"group_norm_act: {C} channels do not split into {num_groups} groups")
    if not eps > 0:
        raise ValueError("group_norm_act: eps must be positive")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.shape != (C,) or (C > 1 and p.stride(0) != 1)):
            raise ValueError(f"group_norm_act: {name} must be a contiguous [{C}], got {tuple(p.shape)}")
    ptype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
    _check_tensors("group_norm_act", x, ptype, weight=weight, bias=bias)


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: str = "identity",
                   checkpoint: str = "none") -> torch.Tensor:
    """act(group_norm(x) * weight + bias) over channels-last x [S, ..., C].

    Statistics (mean, biased variance) run over a sample's positions and each of ``num_groups`` groups of
    consecutive channels; with x [S, C] that is per token.  ``weight`` and ``bias`` [C] are float32 or bfloat16 (one
    dtype for both), whatever x's.  ``activation`` and ``checkpoint`` as in ``linear_act``."""
    act = _ACT_IDS.get(activation)
    xs, dev = x.shape, x.device
    ptype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
    # one expression for what is right; the exact complaint is _check_norm's
    if not (act is not None and checkpoint in CHECKPOINTS and x.dtype in _DTYPES and ptype in _DTYPES and x.is_cuda and
            len(xs) > 1 and num_groups > 0 and xs[-1] > 0 and xs[-1] % num_groups == 0 and eps > 0 and
            (weight is None or weight.shape == xs[-1:] and weight.device == dev and weight.is_contiguous()) and
            (bias is None or bias.shape == xs[-1:] and bias.dtype == ptype and bias.device == dev and
             bias.is_contiguous())):
        _act_id(activation)
        _check_checkpoint(checkpoint)
        _check_norm(x, num_groups, weight, bias, eps)
    if torch.is_grad_enabled() and (x.requires_grad or weight is not None and weight.requires_grad or
                                    bias is not None and bias.requires_grad):
        return GroupNormActFunction.apply(x, weight, bias, num_groups, act, eps, checkpoint)
    return _norm_forward(x, num_groups, weight, bias, act, eps)[0]


# ---- modules ----

class _MainGradModule(nn.Module):
    def _apply(self, fn, recurse=True):
        """Moves ``main_grad`` to where its parameter goes (to(), cuda()); its type stays fp32."""
        kept = {n: getattr(p, "main_grad", None) for n, p in self._parameters.items()}
        super()._apply(fn, recurse)
        for n, p in self._parameters.items():
            g = kept[n]
            if g is not None:
                p.main_grad = (g if g.device == p.device else torch.zeros(g.shape, dtype=g.dtype, device=p.device)
                               if g.is_meta else g.to(p.device))
        return self

    def enable_main_grad(self):
        """Accumulate parameter gradients into persistent FP32 ``main_grad`` buffers (autograd then returns None
        for them), as SparsePoolingLayer.enable_main_grad."""
        for p in self.parameters(recurse=False):
            if getattr(p, "main_grad", None) is None:
                p.main_grad = torch.zeros(p.shape, device=p.device, dtype=torch.float32)

    def zero_main_grad(self):
        for p in self.parameters(recurse=False):
            if getattr(p, "main_grad", None) is not None:
                p.main_grad.zero_()


class LinearAct(_MainGradModule):
    """``linear_act`` with its parameters: weight [out, in] drawn from N(0, 1 / in), bias zero."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "identity",
                 checkpoint: str = "none", dtype: torch.dtype = torch.bfloat16, device=None, seed: int = 0):
        super().__init__()
        _act_id(activation)
        _check_checkpoint(checkpoint)
        if in_features < 1 or out_features < 1 or dtype not in _DTYPES:
            raise ValueError("LinearAct: positive sizes and float32 or bfloat16 parameters")
        self.in_features, self.out_features = in_features, out_features
        self.activation, self.checkpoint = activation, checkpoint
        gen = torch.Generator().manual_seed(seed)
        w = torch.randn(out_features, in_features, generator=gen) * in_features ** -0.5
        self.weight = nn.Parameter(w.to(device=device or "cpu", dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) if bias else None

    def forward(self, x, residual=None):
        return linear_act(x, self.weight, self.bias, residual, self.activation, self.checkpoint)

    def extra_repr(self):
        return (f"in={self.in_features}, out={self.out_features}, bias={self.bias is not None}, "
                f"activation={self.activation}, checkpoint={self.checkpoint}")


class GroupNormAct(_MainGradModule):
    """``group_norm_act`` with its parameters (ones and zeros)."""

    def __init__(self, channels: int, num_groups: int, eps: float = 1e-5, activation: str = "identity",
                 checkpoint: str = "none", affine: bool = True, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        _act_id(activation)
        _check_checkpoint(checkpoint)
        if num_groups < 1 or channels < 1 or channels % num_groups or dtype not in _DTYPES or not eps > 0:
            raise ValueError("GroupNormAct: channels in whole groups, positive eps, float32 or bfloat16 parameters")
        self.channels, self.num_groups, self.eps = channels, num_groups, eps
        self.activation, self.checkpoint = activation, checkpoint
        self.weight = nn.Parameter(torch.ones(channels, device=device, dtype=dtype)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels, device=device, dtype=dtype)) if affine else None

    def forward(self, x):
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.activation, self.checkpoint)

    def extra_repr(self):
        return (f"channels={self.channels}, groups={self.num_groups}, eps={self.eps}, "
                f"activation={self.activation}, checkpoint={self.checkpoint}")
