"""linear_cross_entropy on the GPU against its statement in 64 bits."""
import pytest
import torch

from supergrok15_b200 import _build
from supergrok15_b200.ops import gemm, nn_ops

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def inputs(N, V, D, dtype, ignored=0, seed=0, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed + N + V + D)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    w = torch.randn(V, D, generator=g, device="cuda") * (std / D ** 0.5)
    x = torch.randn(N, D, generator=g, device="cuda") + w[t]
    t[torch.randperm(N, generator=g, device="cuda")[:ignored]] = -100
    return x.to(dtype), w.to(dtype), t


def far(a, b):
    b = b.double()
    d, n = float((a.double() - b).norm()), float(b.norm())
    return d / n if n else d


def check(x, w, t, gout=1.0, repeat=True):
    dtype, (N, D), V = x.dtype, x.shape, w.shape[0]
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = nn_ops.linear_cross_entropy(x, w, t)
    go = torch.tensor(gout, device="cuda")
    gx, gw = torch.autograd.grad(loss, (x, w), go, retain_graph=True)
    again = torch.autograd.grad(loss, (x, w), go)
    with torch.no_grad():
        alone = nn_ops.linear_cross_entropy(x, w, t)
    gemm.check(x.device)
    assert torch.equal(gx, again[0]) and torch.equal(gw, again[1]) and gx.dtype == gw.dtype == dtype and loss.dtype == torch.float32
    if repeat:
        l2 = nn_ops.linear_cross_entropy(x, w, t)
        assert torch.equal(l2, loss) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(l2, (x, w), go), (gx, gw)))
    xr, wr = (a.detach().double().requires_grad_(True) for a in (x, w))
    want = nn_ops.linear_cross_entropy_reference(xr, wr, t)
    wx, ww = torch.autograd.grad(want, (xr, wr), go.double())
    # a logit is a sum of D products in fp32, each addition off by half a step of at most sum |x||w|; the sum of the exponentials has V terms
    amp = float((x.detach().abs().double() @ w.detach().abs().double().t()).max()) if N else 0.0
    z_off = HALF_STEP[torch.float32] * (D * amp + V)
    assert abs(float(loss) - float(want)) <= z_off * 2 + 1e-7 and abs(float(alone) - float(want)) <= z_off * 2 + 1e-7
    # fp32: the logits' error and sums of V (dx) or N (dw) terms; 16 bits: u, d and the result are rounded, half a step each
    tol = z_off * 2 + HALF_STEP[torch.float32] * max(V, N) + (0 if dtype == torch.float32 else 3 * HALF_STEP[dtype])
    assert far(gx, wx) <= tol, ("dx", far(gx, wx), tol)
    assert far(gw, ww) <= tol, ("dw", far(gw, ww), tol)
    assert not gx[(t < 0) | (t >= V)].any()
    return loss, gx, gw


def check_quick(x, w, t):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = nn_ops.linear_cross_entropy(x, w, t)
    return [loss, *torch.autograd.grad(loss, (x, w))]


DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LOSS_SCALE = {torch.float32: 1.0, torch.bfloat16: 0.3, torch.float16: 8192.0}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,D", [(1, 1, 8), (1, 9, 8), (3, 255, 64), (64, 64, 16), (65, 257, 72), (127, 1000, 128), (129, 513, 1000), (300, 4099, 256),
                                   (700, 300, 64), (1, 32000, 256), (256, 256, 2048), (2, 70, 8)])
def test_sizes(N, V, D, dtype):
    check(*inputs(N, V, D, dtype, ignored=N // 3), gout=LOSS_SCALE[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,D", [(40, 77, 1), (5, 50, 7), (70, 130, 33)])
def test_odd_widths(N, V, D, dtype):
    check(*inputs(N, V, D, dtype), gout=LOSS_SCALE[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces(dtype):
    """More rows than one piece takes: the weight's gradient is added over the pieces."""
    N, V, D = 1100, 200000, 32
    x, w, t = inputs(N, V, D, dtype, ignored=50)
    piece = _build.require().lce_piece_rows(N, V, x.element_size(), True)
    assert N > 2 * piece or dtype != torch.float32
    assert N > piece
    check(x, w, t, gout=LOSS_SCALE[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [33, 4096, 16384, 16385, 30000])
def test_many_rows_few_counted(N, dtype):
    """The counted rows are found across work items of 32 rows and, above 16,384 rows, blocks of 4,096; whole pieces may be empty."""
    x, w, t = inputs(N, 300, 16, dtype)
    for lo, hi in ((0, 40), (N // 2, N // 2 + 70), (N - 5, N)):
        s = torch.full_like(t, -100)
        s[lo:hi] = t[lo:hi]
        check(x, w, s, gout=LOSS_SCALE[dtype])
    check(x, w, torch.where(torch.arange(N, device="cuda") % 3 == 0, t, 300), gout=LOSS_SCALE[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_without_counted_rows(dtype):
    N, V, D = 1100, 200000, 16
    x, w, t = inputs(N, V, D, dtype)
    t[300:] = -100
    check(x, w, t, gout=LOSS_SCALE[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
def test_confident_and_hopeless_rows(dtype):
    """Targets with a probability of nearly one (p - 1 must not be the rounding of p) and logits hundreds apart."""
    for std, at in ((30.0, 1.0), (200.0, 1.0), (0.0, 1.0)):
        x, w, t = inputs(150, 700, 128, dtype, std=std)
        check((x * at).to(dtype), w, t, gout=LOSS_SCALE[dtype])
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.nn.functional.normalize(torch.randn(400, 128, generator=g, device="cuda"), dim=1)
    t = torch.randint(0, 400, (90,), generator=g, device="cuda")
    for gain in (12.0, 20.0):                                             # 1 - p around 1e-3 and 1e-6
        check((w[t] * gain).to(dtype), w.to(dtype), t, gout=LOSS_SCALE[dtype] * (1.0 if dtype != torch.float16 else 100.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_counted(dtype):
    x, w, t = inputs(130, 500, 64, dtype)
    t[::2] = -100
    t[1::8] = 500
    t[3::8] = -7
    want = check(x, w, t)
    keep = (t >= 0) & (t < 500)
    loss, gx, gw = check(x[keep], w, t[keep])
    assert far(want[0], loss) < 1e-6 and far(want[1][keep], gx) <= 2 * HALF_STEP[dtype] and far(want[2], gw) <= 2 * HALF_STEP[dtype] + 1e-6
    bad = x.clone()
    bad[~keep] = float("nan")
    assert all(torch.equal(a, b) for a, b in zip(check_quick(bad, w, t), want))        # what stands there reaches nothing
    none = torch.full_like(t, -100)
    loss, gx, gw = check(x, w, none)
    assert float(loss) == 0.0 and not gx.any() and not gw.any()
    loss, gx, gw = check(x[:0], w, t[:0])
    assert float(loss) == 0.0 and gx.shape == (0, 64) and not gw.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_one_sided_gradients(dtype):
    x, w, t = inputs(100, 333, 96, dtype)
    _, gx, gw = check(x, w, t)
    N, D = x.shape
    x3 = torch.empty(N, D + 8, dtype=dtype, device="cuda")[:, 8:].copy_(x)
    odd = torch.empty(N, D + 3, dtype=dtype, device="cuda")[:, 1:D + 1].copy_(x)
    wt = w.t().contiguous().t()
    for a, b in ((x3, w), (odd, w), (x, wt), (x[::2], w[3:])):
        check(a, b, t[: a.shape[0]].clamp(max=b.shape[0] - 1))
    xa, wa = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(nn_ops.linear_cross_entropy(xa, w, t), xa)[0], gx)
    assert torch.equal(torch.autograd.grad(nn_ops.linear_cross_entropy(x, wa, t), wa)[0], gw)
    assert not nn_ops.linear_cross_entropy(x, w, t).requires_grad
    l3 = nn_ops.linear_cross_entropy(xa.view(4, 25, D), w, t.view(4, 25))
    g3, = torch.autograd.grad(l3, xa)
    assert torch.equal(g3, gx)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_step_and_streams(dtype):
    x, w, t = inputs(140, 900, 128, dtype)
    x.requires_grad_(True), w.requires_grad_(True)

    def step():
        loss = nn_ops.linear_cross_entropy(x, w, t)
        return [loss.detach(), *torch.autograd.grad(loss, (x, w))]         # no autograd graph of the leaves lives on into a capture
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    t.copy_((t + 17) % 900)
    with torch.no_grad():
        x.mul_(1.1)
    for g, _ in graphs:
        g.replay()
    for a, b, c in zip(step(), graphs[0][1], graphs[1][1]):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("rows,dtype", [(140, torch.bfloat16), (140, torch.float32), (13, torch.float16)])
def test_captured_backward_behind_a_copy_and_a_joined_stream(rows, dtype):
    """The backward pass's first kernel has something else than one kernel ahead of it."""
    x, w, t = inputs(rows, 900, 128, dtype)
    x.requires_grad_(True), w.requires_grad_(True)
    seed, side = torch.full((), 3.0, device="cuda"), torch.cuda.Stream()

    def step(join):
        loss = nn_ops.linear_cross_entropy(x, w, t)
        go = torch.zeros((), device="cuda")
        go.copy_(seed)
        if join:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = seed * 2
            torch.cuda.current_stream().wait_stream(side)
        res = [loss.detach(), *torch.autograd.grad(loss, (x, w), go)]
        return res + [other] if join else res
    for join in (False, True):
        step(join)                                                        # what a first call sets up
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step(join)
        for value in (1.0, 5.0):
            seed.fill_(value)
            g.replay()
            for a, b in zip(step(join), got):
                assert torch.equal(a, b)
    gemm.check(x.device)


def test_refusals():
    x, w, t = inputs(10, 30, 16, torch.float32)
    with pytest.raises(ValueError, match="one device"):
        nn_ops.linear_cross_entropy(x, w, t.cpu())
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        nn_ops.linear_cross_entropy(x.double(), w.double(), t)
    for args in ((x, w[0], t), (x, w[:, :8], t), (x, w, t[:9]), (x, w[:0], t), (x, w.double(), t), (x, w, t.int()), (x[None], w, t), (x[0, 0], w, t), (x, w[:, :0], t)):
        with pytest.raises(ValueError, match="linear_cross_entropy"):
            nn_ops.linear_cross_entropy(*args)
    loss = nn_ops.linear_cross_entropy(x.requires_grad_(True), w, t)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(loss, x, create_graph=True)
