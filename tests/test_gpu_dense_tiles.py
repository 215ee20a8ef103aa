"""The linear operator at sizes that the tile planner (for 148 SMs) sends to each form of its product kernel: CTA pairs of
256 x 256 and 256 x 128 tiles, single CTAs of 128 x 128, 64 and 32; whole and split sums over k; more work items than CTAs
(an accumulator and the ring taken again); and, for fp32, more than three chunks of 512 k in an item (an accumulator given
back inside it).  `forward` and `backward` name what the planner chooses: CTAs of a tile, its columns, and m(ore items than
CTAs), s(plit), c(hunks).  Checks and tolerances are those of test_gpu_dense."""
import pytest
import torch

import granulelayer_b200 as gl
from test_gpu_dense import BF16, F32, check_linear, data, linear_case, within

pytestmark = pytest.mark.gpu

TILES = [
    # M, K, N, dtype           # forward     backward
    (4669, 941, 539, BF16),    # 2x256       2x128 ms
    (671, 4023, 1742, BF16),   # 2x256 s     2x128 m
    (1563, 4053, 357, BF16),   # 2x128 s     2x256 m
    (1398, 975, 4092, BF16),   # 2x128 m     2x256 ms
    (707, 737, 3734, BF16),    # 2x128 m     2x128 ms
    (147, 2904, 1836, BF16),   # 2x128 s     2x128 m
    (2853, 73, 2105, BF16),    # 1x128 m     2x128 s
    (811, 3779, 45, BF16),     # 1x32 s      1x128 m
    (290, 873, 3883, BF16),    # 2x128       1x128 ms
    (155, 49, 2550, BF16),     # 1x32 m      1x64 s
    (1024, 4096, 4096, BF16),  # 2x256       2x256 m
    (490, 1790, 1583, F32),    # 2x128 s     2x128 mc
    (3721, 889, 601, F32),     # 2x128 m     2x128 msc
    (2120, 2262, 1808, F32),   # 2x128 mc    1x128 mc
    (2342, 3247, 298, F32),    # 1x128 ms    1x128 mc
    (1587, 417, 2332, F32),    # 2x128 m     1x128 msc
    (2853, 73, 2105, F32),     # 1x128 m     2x128 s
    (267, 2947, 3088, F32),    # 1x64 c      1x128 mc
    (1562, 2740, 47, F32),     # 1x64 s      1x64 mc
]


@pytest.mark.parametrize("M,K,N,dtype", TILES)
def test_linear_in_every_form_of_the_product_kernel(M, K, N, dtype):
    check_linear(*linear_case(M, K, N, dtype, "gelu", "none", seed=M), "gelu", "none")


@pytest.mark.parametrize("M,K,N,dtype", [(671, 4023, 1742, BF16), (1563, 4053, 357, BF16), (147, 2904, 1836, BF16),
                                         (490, 1790, 1583, F32), (2342, 3247, 298, F32), (1562, 2740, 47, F32)])
def test_checkpointed_products_in_pairs_and_chunks(M, K, N, dtype):
    """One plane of x by three of dz in fp32 layers."""
    check_linear(*linear_case(M, K, N, dtype, "identity", "int8", seed=M), "identity", "int8")


@pytest.mark.parametrize("M,K,N,dtype", [(1563, 4053, 357, BF16), (1024, 4096, 4096, BF16), (490, 1790, 1583, F32),
                                         (2342, 3247, 298, F32)])
def test_large_products_repeat_bit_for_bit(M, K, N, dtype):
    case = linear_case(M, K, N, dtype, "silu", "none", seed=3)
    runs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_(True) for t in case[:4]]
        y = gl.linear_act(*leaves, activation="silu")
        runs.append([y, *torch.autograd.grad(y, leaves, case[4])])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


@pytest.mark.parametrize("M,K,N,dtype", [(1563, 4053, 357, BF16), (1024, 4096, 2048, BF16), (671, 4024, 1744, BF16),
                                         (490, 1790, 1583, F32), (2342, 3247, 298, F32)])
def test_products_without_an_epilogue_one_at_a_time(M, K, N, dtype):
    """y without bias or activation, and each gradient by itself."""
    x, w = data(M, K, dtype=dtype, seed=1), data(N, K, dtype=dtype, seed=2, scale=K ** -0.5)
    dy = data(M, N, dtype=dtype, seed=3)
    eps = 2.0 ** -8 if dtype == BF16 else 0.0

    def check(got, a, b, k, what):
        want, mag = a.double() @ b.double(), a.double().abs() @ b.double().abs()
        within(got, want, (16 + 6 * k / 16) * 2.0 ** -23 * mag + eps * want.abs() + 2.0 ** -40, what)

    with torch.no_grad():
        check(gl.linear_act(x, w), x, w.t(), K, "y")
    leaf = x.detach().requires_grad_(True)
    check(torch.autograd.grad(gl.linear_act(leaf, w), leaf, dy)[0], dy, w, N, "dx")
    leaf = w.detach().requires_grad_(True)
    check(torch.autograd.grad(gl.linear_act(x, leaf), leaf, dy)[0], dy.t(), x, M, "dw")


def test_many_pair_launches_in_a_row():
    """Launches back to back on one stream, each as the first: a CTA that left too early would leave its partner, or the
    next launch, with something unfinished."""
    x, w = data(512, 1024, dtype=BF16, seed=1), data(4096, 1024, dtype=BF16, seed=2, scale=0.03)
    with torch.no_grad():
        want = gl.linear_act(x, w)
        got = [gl.linear_act(x, w) for _ in range(200)]
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("M,K,N", [(65536, 2048, 1800), (40000, 4096, 1024), (262144, 512, 512), (70001, 136, 200)])
def test_long_sums_into_fp32_gradients(M, K, N):
    """dW of many rows of one sign, added to an fp32 main_grad.  The tensor core truncates after each 16 k to 2^-23 of a
    partial sum that grows evenly: over a chunk of 32 x 64 k by at most half of 128 2^-23 of the chunk's sum; chunks, splits
    and the main_grad that is there are added in fp32, rounding to nearest: 2^-24 each."""
    lay = gl.LinearAct(K, N, bias=False, dtype=BF16, device="cuda")
    lay.enable_main_grad()
    x, dy = data(M, K, dtype=BF16, seed=1).abs(), data(M, N, dtype=BF16, seed=2).abs()
    want = torch.zeros(N, K, dtype=torch.float64, device="cuda")
    for i in range(0, M, 8192):
        want += dy[i:i + 8192].double().t() @ x[i:i + 8192].double()
    for calls in (1, 2):
        lay(x).backward(dy)
        err = (lay.weight.main_grad.double() - calls * want).abs()
        assert float((err / (calls * want)).max()) <= (128 / 2) * 2.0 ** -23 + (M / 2048 + 32 + calls) * 2.0 ** -24


def test_bf16_gradients_of_very_many_rows():
    """A bf16 dW sums at most 2048 blocks of 64 rows in one accumulator, that is 8192 truncations to 2^-23: what sums of one
    sign lose on average.  (Rounding to bf16 averages out over columns of unlike size.)"""
    M, K, N = 262144, 2048, 2304
    x = data(M, K, dtype=BF16, seed=1).abs_()
    dy = (data(M, N, seed=2).abs_() * torch.linspace(1, 2, N, device="cuda")).to(BF16)
    w = data(N, K, dtype=BF16, seed=3).requires_grad_(True)
    (dw,) = torch.autograd.grad(gl.linear_act(x, w), w, dy)
    want = torch.zeros(N, K, dtype=torch.float64, device="cuda")
    for i in range(0, M, 8192):
        want += dy[i:i + 8192].double().t() @ x[i:i + 8192].double()
    assert abs(float(((dw.double() - want) / want).mean())) <= 8192 * 2.0 ** -23
