"""Inputs at which the dense operators could come out wrong though ordinary draws do not show it: outliers where a
chunk of the norm's statistics begins, non-finite values in the backward passes, fp32 values past bf16's range."""
import pytest
import torch

import granulelayer_b200 as gl
from granulelayer_b200 import _native, dense

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def data(*shape, dtype=F32, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


# ---- group norm: statistics ----

@pytest.mark.parametrize("rest", ["normal", "constant"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,G", [((64, 4096, 512), 32), ((600, 4096, 64), 8), ((16, 4096, 512), 32),
                                     ((300, 5000, 24), 3)])
def test_norm_statistics_with_an_outlier_at_the_first_position(shape, G, dtype, rest):
    """One channel of every group is 1000 at position 0, the other positions are N(0, 1) or all alike.  A thread sums
    squared deviations, all positive, over at most 256 positions of its column, two roundings for four positions; some 60 more
    follow where threads, channels and chunks meet: (2 * 64 + 64) 2^-24 = 1.1e-5 < 2^-16."""
    S, P, C = shape
    x = data(*shape, seed=1) if rest == "normal" else torch.full(shape, 0.5, device="cuda")
    x[:, 0, :: C // G] = 1000.0
    x = x.to(dtype)
    _, _, stats = dense._norm_forward(x, G, None, None, 0, 1e-5)
    var, mean = torch.var_mean(x.double().reshape(S, P, G, C // G), dim=(1, 3), correction=0)
    got_var = stats[1].double() ** -2 - 1e-5
    assert float(((got_var - var).abs() / (var + 1e-5)).max()) < 2.0 ** -16
    assert float(((stats[0].double() - mean).abs() / (mean.abs() + var.sqrt())).max()) < 2.0 ** -16


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_non_finite_values_in_long_samples(dtype):
    """A NaN and an infinity, at a chunk's first position and inside, reach their groups only."""
    x = data(2, 70000, 16, dtype=dtype, seed=2)
    clean = gl.group_norm_act(x, 4)
    x[0, 0, 1], x[1, 0, 6], x[1, 33333, 15] = float("nan"), float("inf"), -float("inf")
    y = gl.group_norm_act(x, 4)
    hit = torch.zeros(2, 1, 16, dtype=torch.bool, device="cuda")
    hit[0, :, 0:4] = hit[1, :, 4:8] = hit[1, :, 12:16] = True
    hit = hit.expand(x.shape)
    assert torch.equal(y[~hit], clean[~hit]) and bool(torch.isnan(y[hit]).all())


# ---- linear: non-finite values ----

@pytest.mark.parametrize("ckpt", ["none", "int8"])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [3, 70])
def test_linear_gradients_keep_a_nan(M, dtype, act, ckpt):
    """A NaN in the bias makes act'(z) of its column NaN, one in a row of x that of its row: with a finite dy the
    gradients that contain it are NaN, the others are what they were."""
    x, w, b = data(M, 96, dtype=dtype, seed=1), data(40, 96, dtype=dtype, seed=2, scale=0.1), data(40, dtype=dtype, seed=3)
    dy = data(M, 40, dtype=dtype, seed=4)

    def grads(x, b):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
        return torch.autograd.grad(gl.linear_act(*leaves, activation=act, checkpoint=ckpt), leaves, dy)

    dx0, dw0, db0 = grads(x, b)
    bad = b.clone()
    bad[7] = float("nan")
    dx, dw, db = grads(x, bad)
    keep = torch.arange(40, device="cuda") != 7
    assert bool(torch.isnan(dx).all()) and bool(torch.isnan(dw[7]).all()) and bool(torch.isnan(db[7]))
    assert torch.equal(dw[keep], dw0[keep]) and torch.equal(db[keep], db0[keep])
    bad = x.clone()
    bad[1, 5] = float("nan")
    dx, dw, db = grads(bad, b)
    keep = torch.arange(M, device="cuda") != 1
    assert bool(torch.isnan(dx[1]).all()) and torch.equal(dx[keep], dx0[keep])
    assert bool(torch.isnan(db).all()) and bool(torch.isnan(dw).all())


@pytest.mark.parametrize("M", [8, 9, 200])
def test_linear_fp32_values_past_the_range_of_bf16(M):
    """Finite fp32 values above bf16's largest, 3.39e38: their products with small weights and gradients are numbers,
    by the row kernels (8 rows) and by the tensor cores alike.  Six products of split terms per 16 k in any order:
    (16 + 6 K / 16) 2^-23 of the sum of magnitudes."""
    K, N = 64, 48
    x = data(M, K, seed=1)
    x[0, 3], x[1, 40], x[M - 1, 0] = torch.finfo(F32).max, -3.4e38, 3.395e38
    w = data(N, K, seed=2, scale=1e-3).requires_grad_(True)
    x.requires_grad_(True)
    dy = data(M, N, seed=3, scale=1e-3)
    y = gl.linear_act(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    X, W, DY = x.detach().double(), w.detach().double(), dy.double()

    def close(got, a, b, k):
        err = (got.double() - a @ b).abs()
        assert bool((err <= (16 + 6 * k / 16) * 2.0 ** -23 * (a.abs() @ b.abs())).all())

    close(y, X, W.t(), K)
    close(dw, DY.t(), X, M)
    close(dx, DY, W, N)
    big = torch.full((M, N), 3.4e38, device="cuda")                   # and as an output gradient
    (dx,) = torch.autograd.grad(gl.linear_act(x, w), x, big * torch.eye(M, N, device="cuda"))
    close(dx, (big * torch.eye(M, N, device="cuda")).double(), W, N)


# ---- what is kept between the passes ----

def kept_by(call):
    """(output, what autograd keeps for it as (shape, dtype)) of a call."""
    kept = []

    def pack(t):
        kept.append((tuple(t.shape), t.dtype))
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = call()
    return out, kept


@pytest.mark.parametrize("ckpt", ["none", "int8"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wants", ["x", "w", "b", "r", "xb", "wr"])
def test_linear_keeps_what_its_gradients_need(wants, dtype, ckpt):
    """x (or its codes, whose encoding is a launch) only for the weight's gradient, act'(z) only for those of x, weight
    and bias; the gradients are those of a call that wants them all."""
    M, K, N = 72, 160, 48
    given = dict(x=data(M, K, dtype=dtype, seed=1), w=data(N, K, dtype=dtype, seed=2, scale=0.1),
                 b=data(N, dtype=dtype, seed=3), r=data(M, N, dtype=dtype, seed=4))
    dy = data(M, N, dtype=dtype, seed=5)

    def run(names):
        """The gradients that are asked for, of a call whose `names` can have one."""
        leaves = {n: t.clone().requires_grad_(n in names) for n, t in given.items()}
        n0 = _native.launch_count()
        y, kept = kept_by(lambda: gl.linear_act(*leaves.values(), activation="gelu", checkpoint=ckpt))
        launches = _native.launch_count() - n0
        return dict(zip(wants, torch.autograd.grad(y, [leaves[n] for n in wants], dy))), kept, launches, y

    every, _, most, y0 = run("xwbr")
    got, kept, launches, y = run(wants)
    assert torch.equal(y, y0)
    for n in wants:
        assert torch.equal(got[n], every[n]), n
    shapes = [s for s, _ in kept]
    assert ((M, K) in shapes) == ("w" in wants)                     # x, or its codes (K is whole blocks)
    assert ((M, N) in shapes) == any(n in wants for n in "xwb")     # act'(z)
    assert launches == most - (ckpt == "int8" and "w" not in wants)


@pytest.mark.parametrize("ckpt,per_x,per_z", [("none", 2, 2), ("int8", 33 / 32, 1)])
def test_checkpoints_lower_the_memory_between_the_passes(ckpt, per_x, per_z):
    """Bytes held from a forward pass to its backward pass, beside output and parameters: x and act'(z) in two bytes
    each (bf16), or in 33/32 and one.  The allocator rounds each of at most four tensors up to 512 bytes."""
    M, K, N, G = 512, 1024, 768, 32
    base = data(M, K, dtype=BF16, seed=1).requires_grad_(True)
    w = data(N, K, dtype=BF16, seed=2, scale=0.03).requires_grad_(True)
    gam = data(K, dtype=BF16, seed=3).requires_grad_(True)
    for call, held in ((lambda x: gl.linear_act(x, w, activation="gelu", checkpoint=ckpt), M * K * per_x + M * N * per_z),
                       (lambda x: gl.group_norm_act(x, G, gam, checkpoint=ckpt), M * K * per_x + 2 * M * G * 4)):
        call(base * 1)                                              # anything that first calls allocate
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = call(base * 1)
        now = torch.cuda.memory_allocated() - before - y.numel() * 2
        assert held <= now <= held + 5 * 512, (now, held)
        del y


# ---- products whose waits ran out ----

def test_products_report_through_the_status_word():
    """Products leave the word at 0; one that a product had set is raised by the next call, forward or backward, and
    the call after that works."""
    x, w = data(64, 128, dtype=BF16, seed=1).requires_grad_(True), data(64, 128, dtype=BF16, seed=2)
    y = gl.linear_act(x, w)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    torch.cuda.synchronize()
    tensor, word, address = _native._wait_word
    assert tensor.is_pinned() and address == tensor.data_ptr() and word.value == 0
    word.value = 1
    with pytest.raises(_native.NativeLibraryError, match="ran out"):
        gl.linear_act(x, w)
    assert torch.equal(gl.linear_act(x, w), y)
    word.value = 1
    with pytest.raises(_native.NativeLibraryError, match="ran out"):
        torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0], dx)


# rows (token groups of a power of two and not, several samples), resident samples, long samples in chunks (aligned and
# not), groups wider than a block
@pytest.mark.parametrize("shape,G", [((9, 4096), 32), ((5, 96 * 8), 8), ((3, 130), 13), ((4, 37, 72), 9), ((2, 300, 64), 4),
                                     ((1, 70000, 16), 4), ((40, 5000, 48), 6), ((2, 3000, 33), 3), ((2, 3, 65536), 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_of_constant_groups(shape, G, dtype):
    """Groups whose values are all alike, each a small whole number: every sum of up to 2^24 of its last bits is exact, the
    mean is the value, the deviations are 0 and y is beta, however small eps is."""
    S, C = shape[0], shape[-1]
    c = torch.randint(1, 60, (S, G), generator=torch.Generator().manual_seed(3)).to("cuda")
    x = c.repeat_interleave(C // G, 1).reshape(S, *[1] * (len(shape) - 2), C).expand(shape).to(dtype).contiguous()
    gam, bet = 1 + data(C, dtype=dtype, seed=4, scale=0.1), data(C, dtype=dtype, seed=5)
    y = gl.group_norm_act(x, G, gam, bet, eps=1e-9)
    assert torch.equal(y, bet.expand(shape))
    _, _, stats = dense._norm_forward(x, G, None, None, 0, 1e-9)
    assert torch.equal(stats[0], c.float())


# ---- activations ----

@pytest.mark.parametrize("M", [1, 3, 2000])
def test_bf16_gelu_in_its_tail(M):
    """GELU of bf16 layers down to z = -12.5, where it is z times a tail probability of 1e-36: off by its rounding to bf16
    (half a step, at most 2^-8) and the tail's 1.4e-4 < 2^-12, relative."""
    z = torch.linspace(-12.5, -0.01, max(M, 60), device="cuda").to(BF16)
    one = torch.ones(1, 1, device="cuda", dtype=BF16)
    with torch.no_grad():
        y = torch.cat([gl.linear_act(part.reshape(-1, 1), one, activation="gelu") for part in z.split(M)]).flatten()
    want = z.double() * torch.special.erfc(-z.double() / 2 ** 0.5) / 2
    assert bool(((y.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -12) * want.abs()).all())
