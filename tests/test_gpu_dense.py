"""The dense operators (linear_act, group_norm_act, 8-bit activation checkpoints) against plain float64
restatements of their definitions, at sizes that no tile or vector divides, with strided, empty and non-finite
inputs, and against differences of their own forward passes.

Tolerances, elementwise.  fp32 products: the sum of K products is built 16 at a time by up to six products of split
terms, each step rounding (at worst truncating) a partial sum that is at most sum |x w|, so the error is below
(16 + 6 K / 16) 2^-23 sum_k |x_k w_k| (also above the K 2^-24 of plain fp32 sums for K <= 64, and of sums in blocks).
bf16 adds the rounding of what is stored, 2^-8 |value| (half an ulp is 2^-9), of z before act' (2^-8 |z|, act'' <= 1.2)
and of dz before its products (2^-8 sum |dz w|)."""
import math

import pytest
import torch

import granulelayer_b200 as gl
from granulelayer_b200 import _native

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
ACTS = ("identity", "relu", "gelu", "silu")


def act64(z, act):
    if act == "identity":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def read_back64(x):
    """An 8-bit checkpoint's values: the smallest power of two s per 32 channels with max |x| <= 127 s."""
    C = x.shape[-1]
    v = torch.nn.functional.pad(x.double(), (0, -C % 32)).unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    s = torch.exp2(torch.where(m <= 127 / 128, e - 7, e - 6).clamp(min=-126).double())
    q = torch.round(v / s)
    out = torch.where(s == 2.0 ** 122, q.clamp(-63, 63), q) * s     # 64 * 2^122 would not be finite
    out = torch.where(torch.isfinite(top), out, torch.full_like(out, float("nan")))
    return out.flatten(-2)[..., :C]


def data(*shape, dtype=F32, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                                 f"{float(((got - want).abs() / tol).max()):.3g} x the tolerance")


# ---- 8-bit checkpoints ----

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 3, 257), (7, 1000), (64, 4096)])
def test_codec_is_the_definition(shape, dtype):
    x = data(*shape, dtype=dtype, seed=1) * torch.exp2(torch.randint(-20, 20, shape[:1] + (1,) * (len(shape) - 1),
                                                                     device="cuda")).to(dtype)
    a = gl.encode_activation(x)
    assert a.nbytes() == math.prod(shape[:-1]) * -(-shape[-1] // 32) * 33
    back = gl.decode_activation(a)
    assert back.dtype == dtype and back.shape == x.shape
    assert torch.equal(back.double(), read_back64(x))
    assert torch.equal(gl.decode_activation(a, F32).double(), gl.decode_activation(a, BF16).double())
    assert torch.equal(gl.decode_activation(gl.encode_activation(back)), back)      # reading back changes nothing more


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_codec_edges(dtype):
    big = torch.finfo(dtype).max
    x = torch.zeros(10, 64, device="cuda", dtype=dtype)
    x[1, 3], x[1, 4] = 127.0, -127.0            # the largest code, both signs
    x[2, 0], x[2, 1] = 127.5, 0.5               # past it: the next scale (127.5 is a bf16 number)
    x[3, 40] = float("nan")
    x[4, 0] = float("inf")
    x[5, 63] = -float("inf")
    x[6, 0], x[6, 1] = big, -big
    x[7, 0] = 2.0 ** -126
    x[8, 5] = 2.0 ** -133                       # below half the smallest scale: reads back as 0
    x[9, :32] = torch.arange(32, device="cuda", dtype=dtype) + 0.5     # ties between codes: to even
    x[9, 0] = 127
    back = gl.decode_activation(gl.encode_activation(x))
    want = read_back64(x)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert int(torch.isnan(back).sum()) == 3 * 32
    assert torch.equal(back.nan_to_num().double(), want.nan_to_num())


def test_codec_strides_and_empty():
    base = data(9, 200, dtype=BF16, seed=3)
    for x in (base[:, 3:70], base.t(), base[::2, 8:136], base[0], base[:, :1]):
        assert torch.equal(gl.decode_activation(gl.encode_activation(x)).double(), read_back64(x))
    e = gl.decode_activation(gl.encode_activation(base[:0]))
    assert e.shape == (0, 200)


# ---- linear ----

def linear_case(M, K, N, dtype, act, ckpt, bias=True, residual=True, seed=0):
    x, w = data(M, K, dtype=dtype, seed=seed), data(N, K, dtype=dtype, seed=seed + 1, scale=K ** -0.5)
    b = data(N, dtype=dtype, seed=seed + 2) if bias else None
    r = data(M, N, dtype=dtype, seed=seed + 3) if residual else None
    return x, w, b, r, data(M, N, dtype=dtype, seed=seed + 4)


def check_linear(x, w, b, r, dy, act, ckpt):
    """Forward and gradients of one call against float64."""
    dtype, K = x.dtype, x.shape[1]
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = gl.linear_act(*leaves, activation=act, checkpoint=ckpt)
    given = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip("xwbr", leaves) if t is not None], torch.autograd.grad(y, given, dy)))
    eps = 2.0 ** -8 if dtype == BF16 else 0.0
    M, N = dy.shape

    def step(k):
        return (16 + 6 * k / 16) * 2.0 ** -23

    X, W, DY = x.double(), w.double(), dy.double()
    z = X @ W.t() + (b.double() if b is not None else 0)
    mag = X.abs() @ W.abs().t() + (b.double().abs() if b is not None else 0)
    zt = step(K) * mag + 2.0 ** -22
    a, slope = act64(z, act)
    want = a + (r.double() if r is not None else 0)
    rmag = r.double().abs() if r is not None else 0
    within(y, want, 1.13 * zt + (2.0 ** -22 + eps) * (want.abs() + rmag) + 2.0 ** -21, "y")
    # act' at a z that is off by at most zt (and by its bf16 rounding): its second derivative is at most 1.2; a
    # ReLU within that of 0 may take either side
    dz_off = 1.2 * (zt + eps * z.abs()) + 2.0 ** -21
    if act == "identity":
        dz_off = torch.zeros_like(z)
    elif act == "relu":
        dz_off = (z.abs() <= zt).double()
    if ckpt == "int8":
        X = read_back64(x)
        if act != "identity":
            code = torch.round(slope * 192) / 192
            near = ((slope * 192 - torch.floor(slope * 192) - 0.5).abs() / 192 <= dz_off + 1e-6).double() / 192
            dz_off = near + (dz_off > 0.5) * dz_off
            slope = code
    dz = DY * slope
    doff = DY.abs() * dz_off + (2.0 ** -22 + eps) * dz.abs()
    within(grads["x"], dz @ W, doff @ W.abs() + step(N) * (dz.abs() @ W.abs()) + eps * (dz @ W).abs() + 2.0 ** -40,
           "dx")
    dw = dz.t() @ X
    within(grads["w"], dw, doff.t() @ X.abs() + step(M) * (dz.abs().t() @ X.abs()) + eps * dw.abs() + 2.0 ** -40, "dw")
    if b is not None:
        db = dz.sum(0)
        within(grads["b"], db, (DY.abs() * dz_off).sum(0) + (M + 16) * 2.0 ** -23 * dz.abs().sum(0) + eps * db.abs() +
               2.0 ** -40, "db")
    if r is not None:
        assert torch.equal(grads["r"], dy)


LINEAR_SIZES = [(1, 1, 1), (1, 64, 40), (2, 7, 3), (5, 129, 65), (3, 4096, 24), (17, 100, 1), (33, 72, 200),
                (64, 64, 64), (128, 256, 128), (129, 65, 257), (200, 520, 136), (300, 1001, 515), (513, 192, 384)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", LINEAR_SIZES)
def test_linear_sizes(M, K, N, dtype):
    check_linear(*linear_case(M, K, N, dtype, "gelu", "none", seed=M + K), "gelu", "none")


@pytest.mark.parametrize("ckpt", ["none", "int8"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_activations(dtype, act, ckpt):
    check_linear(*linear_case(70, 136, 200, dtype, act, ckpt, seed=5), act, ckpt)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_optional_inputs(dtype, bias, residual):
    check_linear(*linear_case(40, 96, 72, dtype, "silu", "none", bias, residual, seed=6), "silu", "none")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(1, 4096, 512), (2, 1001, 77), (4, 256, 1000), (7, 512, 96), (8, 333, 130),
                                   (9, 640, 64), (16, 2048, 200), (37, 1024, 520), (2000, 64, 16), (60, 8192, 42),
                                   (130, 8192, 72), (1, 8192, 33), (4, 2056, 264)])
def test_linear_without_gradients(M, K, N, dtype):
    """The serving calls (no saved tensors), one token to many."""
    x, w, b, r, _ = linear_case(M, K, N, dtype, "silu", "none", seed=9)
    with torch.no_grad():
        y = gl.linear_act(x, w, b, r, activation="silu")
        plain = gl.linear_act(x, w)
    z0, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    step, eps = (16 + 6 * K / 16) * 2.0 ** -23, 2.0 ** -8 if dtype == BF16 else 2.0 ** -22
    within(plain, z0, step * mag + eps * z0.abs() + 2.0 ** -40, "z")
    want = act64(z0 + b.double(), "silu")[0] + r.double()
    within(y, want, 1.13 * step * (mag + b.double().abs()) + eps * (want.abs() + r.double().abs()) + 2.0 ** -21, "y")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_strides(dtype):
    """Rows that are windows of larger tensors, transposed weights, expanded gradients, leading dimensions."""
    x, w = data(40, 300, dtype=dtype, seed=1)[:, 5:133], data(128, 90, dtype=dtype, seed=2).t()
    r = data(40, 201, dtype=dtype, seed=3)[:, 1:91]
    check_linear(x, w, data(90, dtype=dtype, seed=4), r, data(1, 90, dtype=dtype, seed=5).expand(40, 90), "gelu",
                 "none")
    xs, ws = data(2, 3, 5, 64, dtype=dtype, seed=6), data(16, 64, dtype=dtype, seed=7)
    with torch.no_grad():
        y = gl.linear_act(xs, ws)
        assert y.shape == (2, 3, 5, 16) and torch.equal(y.reshape(30, 16), gl.linear_act(xs.reshape(30, 64), ws))
        t = gl.linear_act(xs[0, 0, 0], ws)
        assert t.shape == (16,)
    within(t, (xs[0, 0, 0].double() @ ws.double().t()), 0.02 * ws.double().abs().sum(1) * 4, "vector")


def test_linear_empty_and_unneeded():
    w = data(8, 16, seed=1).requires_grad_(True)
    b = data(8, seed=2).requires_grad_(True)
    y = gl.linear_act(torch.empty(0, 16, device="cuda"), w, b, activation="gelu")
    gw, gb = torch.autograd.grad(y, (w, b), torch.empty(0, 8, device="cuda"))
    assert y.shape == (0, 8) and not gw.any() and not gb.any()
    x = data(4, 16, seed=3).requires_grad_(True)
    (dx,) = torch.autograd.grad(gl.linear_act(x, w.detach(), None, activation="silu").sum(), x)   # dx alone
    (dw,) = torch.autograd.grad(gl.linear_act(x.detach(), w, None).sum(), w)                        # dw alone
    within(dw, x.detach().double().sum(0).expand(8, 16), 2.0 ** -20 * x.detach().double().abs().sum(0), "dw")
    z = x.detach().double() @ w.detach().double().t()
    within(dx, act64(z, "silu")[1] @ w.detach().double(), 1e-5 * w.detach().double().abs().sum(0), "dx")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [3, 200])
def test_linear_non_finite_rows_stay_apart(M, dtype):
    """A NaN or an infinity in one row of x reaches that row of y only, and does not come out as a number."""
    x, w, b, r, _ = linear_case(M, 160, 96, dtype, "identity", "none", seed=12)
    with torch.no_grad():
        clean = gl.linear_act(x, w, b, r)
        x[1, 7], x[2, 3] = float("nan"), float("inf")
        y = gl.linear_act(x, w, b, r)
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[1:3] = False
    assert torch.equal(y[keep], clean[keep])
    assert bool(torch.isnan(y[1]).all()) and not bool(torch.isfinite(y[2]).any())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_main_grad(dtype):
    """Parameters with a main_grad get fp32 sums over calls there, and autograd gets nothing for them."""
    lay = gl.LinearAct(96, 80, activation="gelu", dtype=dtype, device="cuda", seed=3)
    x, dy = data(50, 96, dtype=dtype, seed=4), data(50, 80, dtype=dtype, seed=5)
    lay(x).backward(dy)
    gw, gb = lay.weight.grad.double(), lay.bias.grad.double()
    lay.weight.grad = lay.bias.grad = None
    lay.enable_main_grad()
    for _ in range(2):
        lay(x).backward(dy)
    assert lay.weight.grad is None and lay.weight.main_grad.dtype == F32
    tol = 2.0 ** -8 if dtype == BF16 else 2.0 ** -20
    within(lay.weight.main_grad / 2, gw, tol * (gw.abs() + gw.abs().mean()), "dw")
    within(lay.bias.main_grad / 2, gb, tol * (gb.abs() + gb.abs().mean()), "db")
    opt = gl.FusedAdamW(lay.parameters(), lr=1e-2, moments="fp32")
    before = lay.weight.detach().clone()
    opt.step()
    assert not torch.equal(before, lay.weight) and not lay.weight.main_grad.any()


@pytest.mark.parametrize("ckpt", ["none", "int8"])
def test_linear_repeats_bit_for_bit(ckpt):
    case = linear_case(300, 520, 264, BF16, "gelu", ckpt, seed=2)
    runs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_(True) for t in case[:4]]
        y = gl.linear_act(*leaves, activation="gelu", checkpoint=ckpt)
        runs.append([y, *torch.autograd.grad(y, leaves, case[4])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def directional(f, leaf, grad, h):
    """(difference of f along a random direction, the gradient's product with it), both float64."""
    v = torch.randn(leaf.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(99))
    v = v / v.norm()
    with torch.no_grad():
        up, down = f(leaf + h * v), f(leaf - h * v)
        span = (leaf + h * v).double() - (leaf - h * v).double()
    return float(up - down), float((grad.double() * span).sum())


@pytest.mark.parametrize("act", ["identity", "gelu", "silu"])
def test_linear_gradient_against_differences(act):
    """Central differences of the fp32 forward over 2 h: the third derivative term is below h^2 of the gradient's
    size, the forward's rounding below 1e-6 of sum |y dy| ~ 30."""
    x, w, b, r, dy = linear_case(24, 40, 36, F32, act, "none", seed=21)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(gl.linear_act(*leaves, activation=act), leaves, dy)
    for i, (leaf, g) in enumerate(zip(leaves, grads)):
        def f(t):
            args = [u.detach() for u in leaves]
            args[i] = t
            return (gl.linear_act(*args, activation=act).double() * dy.double()).sum()

        diff, dot = directional(f, leaf.detach(), g, 0.125)
        assert abs(diff - dot) <= 0.03 * float(g.double().norm()) * 0.25 + 1e-4


def test_linear_on_another_stream():
    case = linear_case(256, 256, 256, BF16, "gelu", "none", seed=8)
    with torch.no_grad():
        want = gl.linear_act(*case[:4], activation="gelu")
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = [gl.linear_act(*case[:4], activation="gelu") for _ in range(4)]
        s.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_in_a_cuda_graph():
    """Forward calls captured on a stream replay on new contents of the same tensors."""
    x, w, b, r, _ = linear_case(200, 320, 264, BF16, "gelu", "none", seed=4)
    gam = 1 + data(264, dtype=BF16, seed=5, scale=0.1)

    def call():
        return gl.group_norm_act(gl.linear_act(x, w, b, r, activation="gelu"), 8, gam, activation="silu")

    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call()
        x.copy_(data(200, 320, dtype=BF16, seed=77))
        want = call()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_second_derivatives_are_refused():
    x = data(8, 32, seed=1).requires_grad_(True)
    for y in (gl.linear_act(x, data(16, 32, seed=2), activation="gelu"), gl.group_norm_act(x, 4)):
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_linear_as_a_threads_first_cuda_call():
    """A thread that has not touched the device yet (autograd's, on its first backward) has no current context."""
    import threading

    x, w = data(64, 128, dtype=BF16, seed=1), data(64, 128, dtype=BF16, seed=2)
    with torch.no_grad():
        want = gl.linear_act(x, w)
    got = []

    def run():
        with torch.no_grad():
            got.append(gl.linear_act(x, w))

    t = threading.Thread(target=run)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_linear_refusals():
    x, w = data(4, 16), data(8, 16)
    for args, kw in (((x, data(8, 15)), {}), ((x, w, data(7)), {}), ((x, w, None, data(4, 7)), {}),
                     ((x, w.to(BF16)), {}), ((x.double(), w.double()), {}), ((x, w), dict(activation="tanh")),
                     ((x, w), dict(checkpoint="fp8")), ((x, w, data(8), data(1, 8)), {}), ((x, data(16)), {}),
                     ((x, w, data(16)[::2]), {}), ((x, w.cpu()), {})):
        with pytest.raises(ValueError):
            gl.linear_act(*args, **kw)
    with pytest.raises(_native.NativeLibraryError):
        gl.linear_act(x.cpu(), w.cpu())


# ---- group norm ----

def norm64(x, G, w, b, eps, act, dy=None, ckpt="none"):
    S, C = x.shape[0], x.shape[-1]
    X = x.double().reshape(S, -1, G, C // G)
    gam = (w.double() if w is not None else torch.ones(C, device="cuda", dtype=torch.float64)).reshape(G, -1)
    bet = (b.double() if b is not None else torch.zeros(C, device="cuda", dtype=torch.float64)).reshape(G, -1)
    mu = X.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((X - mu) ** 2).mean((1, 3), keepdim=True) + eps)
    out = dict(y=act64((X - mu) * rstd * gam + bet, act)[0].reshape(x.shape), rstd=rstd, mu=mu)
    if dy is not None:
        if ckpt == "int8":
            X = read_back64(x).reshape(X.shape)
        h = (X - mu) * rstd
        du = dy.double().reshape(X.shape) * act64(h * gam + bet, act)[1]
        q = du * gam
        m1, m2 = q.mean((1, 3), keepdim=True), (q * h).mean((1, 3), keepdim=True)
        out.update(dx=(rstd * (q - m1 - h * m2)).reshape(x.shape), dw=(du * h).sum((0, 1)).reshape(C),
                   db=du.sum((0, 1)).reshape(C), du=du, h=h, q=q)
    return out


def check_norm(x, G, w, b, dy, act="silu", ckpt="none", eps=1e-5):
    """fp32 statistics over m values in blocks: relative error of mean and variance far below 2^-16 of the values'
    size for these m; an h off by d h moves y by 1.13 |gamma| d h, act' by 1.2 |gamma| d h."""
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    given = [t for t in leaves if t is not None]
    y = gl.group_norm_act(leaves[0], G, leaves[1], leaves[2], eps=eps, activation=act, checkpoint=ckpt)
    grads = dict(zip([n for n, t in zip("xwb", leaves) if t is not None], torch.autograd.grad(y, given, dy)))
    ref = norm64(x, G, w, b, eps, act, dy, ckpt)
    e = 2.0 ** -8 if x.dtype == BF16 else 0.0
    ep = 2.0 ** -8 if any(p is not None and p.dtype == BF16 for p in (w, b)) else 0.0
    gmax = float(w.double().abs().max()) if w is not None else 1.0
    off = 2.0 ** -18 * (1 + float(ref["h"].abs().max()))          # of h
    if float((ref["mu"].abs() * ref["rstd"]).max()) > 1:           # x - mu loses the bits that mu shares with x
        off *= float((ref["mu"].abs() * ref["rstd"]).max())
    within(y, ref["y"], 1.13 * gmax * off + (e + 2.0 ** -20) * ref["y"].abs() + 2.0 ** -20, "y")
    dmax = float(dy.double().abs().max()) * 1.13
    doff = dmax * (1.2 * gmax * off + 2.0 ** -19)                  # of du
    hmax = 1 + float(ref["h"].abs().max())
    rs = float(ref["rstd"].max())
    within(grads["x"], ref["dx"], rs * gmax * (doff * (2 + hmax) + dmax * off * (2 + hmax)) + e * ref["dx"].abs(),
           "dx")
    n = ref["h"].shape[0] * ref["h"].shape[1]
    if w is not None:
        within(grads["w"], ref["dw"], (doff * hmax + dmax * off) * n + ep * ref["dw"].abs(), "dw")
    if b is not None:
        within(grads["b"], ref["db"], doff * n + ep * ref["db"].abs(), "db")
    return y


NORM_SIZES = [((1, 1), 1), ((1, 8), 8), ((3, 40), 4), ((1, 4096), 32), ((300, 512), 8), ((2, 5, 24), 3),
              ((2, 3, 7, 33), 11), ((4, 1000, 64), 8), ((3, 129, 1000), 8), ((2, 64, 64, 512), 32), ((1, 70000, 8), 2),
              ((5, 1, 1, 96), 96), ((2, 2000, 1001), 7), ((1, 3, 40000), 2), ((1, 1, 200001), 3)]


# token rows: groups of one vector, of as many as lanes, of several a lane, of no power of two; samples past a block's
# walk; and groups too wide for a block's sums
NORM_SIZES += [((7, 4096), 1), ((7, 2048), 1), ((130, 1024), 1), ((5, 800), 5), ((3, 96), 12), ((9, 160), 8),
               ((5000, 64), 4), ((2, 3, 65536), 1), ((1, 40, 131072), 2)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,G", NORM_SIZES)
def test_norm_sizes(shape, G, dtype):
    C = shape[-1]
    x = data(*shape, dtype=dtype, seed=1) + data(C, dtype=dtype, seed=2, scale=0.5)
    w, b = 1 + data(C, dtype=dtype, seed=3, scale=0.1), data(C, dtype=dtype, seed=4, scale=0.1)
    check_norm(x, G, w, b, data(*shape, dtype=dtype, seed=5))


@pytest.mark.parametrize("ckpt", ["none", "int8"])
@pytest.mark.parametrize("act", ["identity", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_activations(dtype, act, ckpt):
    x, dy = data(6, 50, 72, dtype=dtype, seed=1), data(6, 50, 72, dtype=dtype, seed=2)
    w, b = 1 + data(72, dtype=dtype, seed=3, scale=0.1), data(72, dtype=dtype, seed=4, scale=0.1)
    check_norm(x, 9, w, b, dy, act, ckpt)


@pytest.mark.parametrize("shape,G", [((12, 77, 1000), 8), ((3, 4000, 33), 3), ((1, 70000, 40), 2), ((9, 130), 13)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_checkpoint_sizes(shape, G, dtype):
    x, dy = data(*shape, dtype=dtype, seed=1), data(*shape, dtype=dtype, seed=2)
    w = 1 + data(shape[-1], dtype=dtype, seed=3, scale=0.1)
    check_norm(x, G, w, None, dy, "gelu", "int8")


@pytest.mark.parametrize("xd,pd", [(BF16, F32), (F32, BF16)])
def test_norm_parameter_types_and_options(xd, pd):
    x, dy = data(4, 33, 48, dtype=xd, seed=1), data(4, 33, 48, dtype=xd, seed=2)
    w, b = 1 + data(48, dtype=pd, seed=3, scale=0.1), data(48, dtype=pd, seed=4)
    check_norm(x, 6, w, b, dy)
    check_norm(x, 6, None, b, dy)
    check_norm(x, 6, w, None, dy)
    check_norm(x, 6, None, None, dy)


def test_norm_relu_forward_and_gradient():
    x, dy = data(8, 20, 64, seed=1), data(8, 20, 64, seed=2)
    x.requires_grad_(True)
    y = gl.group_norm_act(x, 4, activation="relu")
    ref = norm64(x.detach(), 4, None, None, 1e-5, "relu", dy)
    within(y, ref["y"], 1e-4 + 0 * ref["y"], "y")
    (dx,) = torch.autograd.grad(y, x, dy)
    assert int((ref["h"].abs() < 1e-5).sum()) == 0       # no element so near 0 that fp32 could take the other side
    within(dx, ref["dx"], 1e-4 + 0 * ref["dx"], "dx")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_large_mean_and_constant_groups(dtype):
    """A mean of 200 standard deviations, and groups without any variance (rstd = 1 / sqrt(eps))."""
    x = data(3, 400, 32, dtype=F32, seed=1) + 200
    x[1, :, :8] = 5.0
    x = x.to(dtype)
    check_norm(x, 4, None, None, data(3, 400, 32, dtype=dtype, seed=2), "identity")


def test_norm_strides_and_streams():
    base = data(4, 9, 11, 80, dtype=BF16, seed=1)
    w = data(48, dtype=BF16, seed=2)
    for x in (base[..., 5:53], base[:, :, ::2, 8:56], base.permute(0, 2, 1, 3)[..., :48],
              base[..., :48].transpose(0, 1)):
        check_norm(x, 6, w, None, data(*x.shape, dtype=BF16, seed=3))
    x = base[..., :48]
    dy = data(4, 1, 1, 48, dtype=BF16, seed=4).expand(x.shape)
    check_norm(x, 6, w, None, dy)
    want = gl.group_norm_act(x, 6, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = gl.group_norm_act(x, 6, w)
    s.synchronize()
    assert torch.equal(got, want)


def test_norm_empty_and_non_finite():
    w = data(16, seed=1).requires_grad_(True)
    for shape in ((0, 16), (0, 5, 16), (3, 0, 16)):
        y = gl.group_norm_act(torch.empty(*shape, device="cuda"), 4, w)
        assert y.shape == shape
        assert not torch.autograd.grad(y, w, torch.empty(*shape, device="cuda"))[0].any()
    x = data(5, 30, 16, seed=2)
    clean = gl.group_norm_act(x, 4)
    x[1, 3, 2], x[3, 29, 15] = float("nan"), float("inf")
    y = gl.group_norm_act(x, 4)
    hit = torch.zeros(5, 30, 16, dtype=torch.bool, device="cuda")
    hit[1, :, 0:4] = hit[3, :, 12:16] = True           # only the groups that hold them
    assert torch.equal(y[~hit], clean[~hit]) and bool(torch.isnan(y[1, :, 0:4]).all())
    assert bool(torch.isnan(y[3, :, 12:16]).all())


@pytest.mark.parametrize("ckpt", ["none", "int8"])
@pytest.mark.parametrize("shape", [(5, 60, 64), (1, 70000, 16)])
def test_norm_repeats_bit_for_bit(shape, ckpt):
    x, dy, w = data(*shape, dtype=BF16, seed=1), data(*shape, dtype=BF16, seed=2), data(shape[-1], dtype=BF16, seed=3)
    x.requires_grad_(True)
    w.requires_grad_(True)
    runs = []
    for _ in range(2):
        y = gl.group_norm_act(x, 4, w, activation="gelu", checkpoint=ckpt)
        runs.append([y, *torch.autograd.grad(y, (x, w), dy)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_norm_gradient_against_differences():
    """As test_linear_gradient_against_differences."""
    x, dy = data(4, 6, 40, seed=1), data(4, 6, 40, seed=2)
    leaves = [x.requires_grad_(True), (1 + data(40, seed=3, scale=0.1)).requires_grad_(True),
              data(40, seed=4).requires_grad_(True)]

    def call(x, w, b):
        return gl.group_norm_act(x, 5, w, b, activation="gelu")

    grads = torch.autograd.grad(call(*leaves), leaves, dy)
    for i, (leaf, g) in enumerate(zip(leaves, grads)):
        def f(t):
            args = [u.detach() for u in leaves]
            args[i] = t
            return (call(*args).double() * dy.double()).sum()

        diff, dot = directional(f, leaf.detach(), g, 0.125)
        assert abs(diff - dot) <= 0.03 * float(g.double().norm()) * 0.25 + 1e-4


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_main_grad(dtype):
    mod = gl.GroupNormAct(48, 6, activation="gelu", dtype=dtype, device="cuda")
    x, dy = data(7, 21, 48, dtype=dtype, seed=1), data(7, 21, 48, dtype=dtype, seed=2)
    mod(x).backward(dy)
    gw, gb = mod.weight.grad.double(), mod.bias.grad.double()
    mod.weight.grad = mod.bias.grad = None
    mod.enable_main_grad()
    mod(x).backward(dy)
    mod(x).backward(dy)
    assert mod.weight.grad is None
    tol = 2.0 ** -8 if dtype == BF16 else 2.0 ** -20
    within(mod.weight.main_grad / 2, gw, tol * (gw.abs() + gw.abs().mean()), "dw")
    within(mod.bias.main_grad / 2, gb, tol * (gb.abs() + gb.abs().mean()), "db")


def test_norm_refusals():
    x, w = data(4, 5, 16), data(16)
    for args, kw in (((x, 3), {}), ((x, 0), {}), ((x, 4, data(15)), {}), ((x, 4, w, w.to(BF16)), {}),
                     ((x.double(), 4), {}), ((x[0, 0], 4), {}), ((x, 4), dict(eps=0.0)),
                     ((x, 4), dict(activation="tanh")), ((x, 4), dict(checkpoint="int4")), ((x, 4, w.cpu()), {}),
                     ((x, 4, data(32)[::2]), {})):
        with pytest.raises(ValueError):
            gl.group_norm_act(*args, **kw)
    with pytest.raises(_native.NativeLibraryError):
        gl.group_norm_act(x.cpu(), 4)


# ---- together ----

@pytest.mark.parametrize("dtype", [F32, BF16])
def test_block_trains_with_and_without_checkpoints(dtype):
    """norm -> linear -> sparse pooling -> linear + residual: with either form of saved activations steps of the
    optimizer descend, and the first loss, before any gradient, is the same."""
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("dense_block", Path(__file__).resolve().parent.parent / "examples" /
                                                  "dense_block.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    plain = mod.train("none", dtype, steps=12)
    kept = mod.train("int8", dtype, steps=12)
    assert plain[-1] < plain[0] and kept[-1] < kept[0]
    assert kept[0] == plain[0]                                  # the forward pass does not change
