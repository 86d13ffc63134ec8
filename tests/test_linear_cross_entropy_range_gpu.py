"""linear_cross_entropy against its statement in 64 bits with the error that its arithmetic is expected to have, not the most it could have; where
counted rows begin and end; sizes at which the rows are cut."""
import pytest
import torch

from supergrok15_b200 import _build
from supergrok15_b200.ops import gemm, nn_ops

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
LOSS_SCALE = {torch.float32: 1.0, torch.bfloat16: 0.3, torch.float16: 8192.0}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(N, V, D, dtype, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(5 + N + V + D)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    w = torch.randn(V, D, generator=g, device="cuda") * (std / D ** 0.5)
    x = torch.randn(N, D, generator=g, device="cuda") + w[t]
    return x.to(dtype), w.to(dtype), t


def tolerance(x, w):
    """(loss, gradients).  A logit is summed over D products in fp32: an addition is off by half a step of the partial sum, which is about as large as
    the norm of the products and as the logit itself, and the errors of D additions add up like their square root (four times that, for the largest
    of all logits and for accumulators that cut instead of rounding).  A probability is off by the logit's error and the row's sum's; sums of V and N
    terms like their square roots.  16 bits: u, d (or the scaled row of x) and the result are rounded, half a step each."""
    (N, D), V = x.shape, w.shape[0]
    xd, wd = x.double(), w.double()
    z = 4 * HALF_STEP[torch.float32] * D ** 0.5 * float(((xd ** 2) @ (wd ** 2).t()).sqrt().max() + (xd @ wd.t()).abs().max())
    return 2 * z + 1e-7, 2 * z + 4 * HALF_STEP[torch.float32] * max(V, N) ** 0.5 + (0 if x.dtype == torch.float32 else 3 * HALF_STEP[x.dtype])


def check(x, w, t, gout=1.0):
    tol_l, tol_g = tolerance(x, w)
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    go = torch.tensor(gout, device="cuda")
    loss = nn_ops.linear_cross_entropy(x, w, t)
    got = torch.autograd.grad(loss, (x, w), go)
    with torch.no_grad():
        alone = nn_ops.linear_cross_entropy(x, w, t)
    gemm.check(x.device)
    r = [a.detach().double().requires_grad_(True) for a in (x, w)]
    want = nn_ops.linear_cross_entropy_reference(*r, t)
    for l in (loss, alone):
        assert abs(float(l) - float(want)) <= tol_l * max(1.0, float(want)), (float(l), float(want), tol_l)
    for n, a, b in zip(("dx", "dw"), got, torch.autograd.grad(want, r, go.double())):
        d, size = float((a.double() - b).norm()), float(b.norm())
        # half the least number for each element of the result
        least = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}[a.dtype] * a.numel() ** 0.5
        assert d <= tol_g * size + least, (n, d / size if size else d, tol_g)
    return tol_g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,D", [(129, 513, 1000), (256, 256, 2048), (300, 4099, 256), (700, 300, 64), (1, 32000, 256), (13, 32000, 512), (65, 257, 72), (70, 130, 33)])
def test_expected_error(N, V, D, dtype):
    tol = check(*inputs(N, V, D, dtype), gout=LOSS_SCALE[dtype])
    if dtype == torch.float32:
        assert tol < 0.0005                                               # operands rounded to 16 bits would not pass (0.0017 in bf16, 0.0002 and more in fp16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("std", [0.0, 10.0, 30.0, 200.0])
def test_expected_error_of_confident_rows(std, dtype):
    check(*inputs(150, 700, 128, dtype, std), gout=LOSS_SCALE[dtype])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [4097, 16385, 30000])
def test_runs_of_counted_rows(N, dtype):
    """Counted rows are moved together by work items of 16 rows and, above 16,384 rows, behind counts of 4,096: runs that begin and end at either side of
    both, and one counted row alone in the last item."""
    x, w, t = inputs(N, 300, 16, dtype)
    ends = (15, 16, 17, 31, 33, 4095, 4096, 4097)
    for lo, hi in [(a, b) for a in (0, *ends[:3], 4080) for b in ends if b > a] + [(N - 1, N), (N - N % 16 - 1, N), (N - 17, N - 16)]:
        s = torch.full_like(t, -100)
        s[lo:hi] = t[lo:hi]
        s[(lo + hi) // 2] = -100 if hi - lo > 2 else s[(lo + hi) // 2]
        check(x, w, s)


def test_a_large_vocabulary_is_evaluated_in_pieces():
    """Without gradients the statistics are what is bounded: the mean over all rows is that of calls of a few rows each."""
    N, V, D = 1200, (1 << 22) - 7, 8
    assert _build.require().lce_piece_rows(N, V, 2, False) < N
    x, w, t = inputs(N, V, D, torch.bfloat16)
    t[1024 + 20:1024 + 90] = -100
    counts = [int((c >= 0).sum()) for c in t.split(300)]
    parts = [float(nn_ops.linear_cross_entropy(a, w, c)) * n for a, c, n in zip(x.split(300), t.split(300), counts)]
    want = sum(parts) / sum(counts)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = float(nn_ops.linear_cross_entropy(x, w, t))
    assert abs(got - want) <= 1e-6 * want                                 # a few fp32 roundings of the mean
    assert torch.cuda.max_memory_allocated() - before < 300 << 20
    gemm.check(x.device)


def test_millions_of_rows_over_a_tiny_vocabulary():
    """More tile rows than the second dimension of a grid has: 8,400,000 rows are more than one piece although they take little memory."""
    x, w, t = inputs(8_400_000, 5, 4, torch.float32)
    check(x, w, t)
