"""attention_packed in 16 bits over the range of its operands: what a tensor core multiplies is a 16-bit number, and in fp16 one below 2^-14 has
fewer bits and one above 65,504 is infinite, although the gradients that it is summed to are ordinary numbers."""
import pytest
import torch

from supergrok15_b200.ops import gemm, nn_ops

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}          # half the distance of the smallest numbers
DTYPES = [torch.bfloat16, torch.float16]


def tensors(lens, H, Hk, hd, dtype, qs=1.0, ks=1.0, ds=1.0, vs=1.0):
    g = torch.Generator(device="cuda").manual_seed(11 + sum(lens) + hd)
    T = sum(lens)
    q, do = (torch.randn(T, H, hd, generator=g, device="cuda") * s for s in (qs, ds))
    k, v = (torch.randn(T, Hk, hd, generator=g, device="cuda") * s for s in (ks, vs))
    return [t.to(dtype) for t in (q, k, v, do)] + [torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)]


def both(q, k, v, do, cu, causal, scale=None):
    """[out, dq, dk, dv] of the kernels, and of the statement in 64 bits on the same numbers."""
    a = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = nn_ops.attention_packed(*a, cu, causal, scale)
    got = [out.detach(), *torch.autograd.grad(out, a, do)]
    gemm.check(q.device)
    r = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    want = nn_ops.attention_packed_reference(*r, cu, causal, scale)
    return got, [want.detach(), *torch.autograd.grad(want, r, do.double())]


def compare(got, want, roundings=4):
    """Half a step per rounding (probability, dS, the output inside delta, the result), and half the least number for each element of the result."""
    for n, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        d, size = float((a.double() - b).norm()), float(b.norm())
        assert d <= roundings * HALF_STEP[a.dtype] * size + LEAST[a.dtype] * a.numel() ** 0.5, (n, d / size if size else d)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,hd,ds", [([4096], 128, 1e-3), ([8192], 64, 2.0 ** -8), ([8192], 64, 2.0 ** -12), ([300, 5000, 70], 80, 2.0 ** -10)])
def test_small_gradients_of_long_sequences(lens, hd, ds, dtype):
    """dS = P (dP - delta) of thousands of keys.  Large keys (queries) with small queries (keys) keep dq (dk) itself a normal number."""
    for qs, ks in ((2.0 ** -4, 2.0 ** 4), (2.0 ** 4, 2.0 ** -4)):
        for causal in (True, False):
            compare(*both(*tensors(lens, 2, 1, hd, dtype, qs, ks, ds), causal))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_gradients(dtype):
    """dS beyond 65,504 whose sums over small keys and queries are not."""
    for causal in (True, False):
        got, want = both(*tensors([5, 200, 70], 4, 2, 128, dtype, 0.25, 0.05, 1.0e4, 4.0), causal)
        compare(got[:3], want[:3])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_loud_and_quiet_rows(hd, dtype):
    """Gradients 2^24 apart in neighbouring sequences, and a few loud rows at the begin of a causal one: the rows that do not meet them are as
    exact as without them."""
    lens = [333, 2048, 61]
    q, k, v, do, cu = tensors(lens, 4, 2, hd, dtype, 1.0, 8.0, 1.0)
    do[:333] *= 2.0 ** 12
    do[333:] *= 2.0 ** -12
    got, want = both(q, k, v, do, cu, False, 0.02)
    for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]):
        compare([t[a:b] for t in got], [t[a:b] for t in want])
    do = do.clone()
    do[333:340] = 2.0 ** 10
    got, want = both(q, k, v, do, cu, True, 0.02)
    compare([t[333 + 128:333 + 2048] for t in got], [t[333 + 128:333 + 2048] for t in want])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_one_row_length_everywhere(dtype):
    """Sequences around the 32 rows whose norms are looked up together, with the loudest row first, last, and at either side of a border."""
    lens = [1, 31, 32, 33, 63, 64, 65, 95, 97, 160]
    q, k, v, do, cu = tensors(lens, 4, 1, 64, dtype, 0.5, 0.5, 1.0)
    rows = cu.tolist()
    for at in (0, -1, 31, 32):
        d, vv = do.clone(), v.clone()
        for a, b in zip(rows[:-1], rows[1:]):
            if at < b - a:
                d[b - 1 if at < 0 else a + at] *= 2.0 ** 13
                vv[b - 1 if at < 0 else a + at] *= 2.0 ** 6
        for causal in (True, False):
            got, want = both(q, k, vv, d, cu, causal)
            assert all(bool(t.isfinite().all()) == bool(w.abs().max() < 65504) or t.dtype != torch.float16 for t, w in zip(got, want))
            got, want = both(q * 2.0 ** -5, k * 2.0 ** -5, vv * 2.0 ** -5, d, cu, causal)
            # a sequence of one row has ds = 0 but for rounding
            compare([t[1:] for t in got], [t[1:] for t in want])


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_gradient_at_all(dtype):
    q, k, v, do, cu = tensors([100, 300], 4, 2, 64, dtype)
    got, _ = both(q, k, v, do * 0, cu, True)
    assert not any(t.any() for t in got[1:])
    got, _ = both(q, k, v * 0, do, cu, True)
    assert not any(t.any() for t in got[:3]) and got[3].any()


def one_key_above_the_others(T, hd, gap, dtype, alike=False):
    """Every query gives the first key a score `gap` powers of two above the others'."""
    q, k, v, do, cu = tensors([T], 1, 1, hd, dtype, 0.0, 0.0)
    q[:, 0, 0] = 4.0
    k[0, 0, 0] = gap * 0.6931471805599453 / 4.0
    if alike:
        do[:] = 1.0
        v[:] = 1.0
        v[0] = 0.0
    return q, k, v, do, cu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [16.7, 20.3, 24.6])
def test_unlikely_keys_have_their_gradient(gap, dtype):
    """dv_j = sum_i p_ij do_i of thousands of queries that all find a key equally unlikely: the rounding of the probability is the same in all of them."""
    got, want = both(*one_key_above_the_others(4096, 64, gap, dtype, True), False, 1.0)
    compare([t[1:] for t in got[3:]] * 4, [t[1:] for t in want[3:]] * 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [19.4, 20.6])
def test_unlikely_keys_have_their_share(gap, dtype):
    """One key above thousands of equally unlikely ones that alone have something to say, before and behind them."""
    q, k, v, do, cu = one_key_above_the_others(4096, 64, gap, dtype, True)
    for at in (0, 2000, 4095):
        k2, v2 = k.roll(at, 0), v.roll(at, 0)
        got, want = both(q, k2, v2, do, cu, False, 1.0)
        compare(got[:1], want[:1])


def test_many_backward_passes_agree_in_fp16():
    """Warps drift apart, and the units of an item are looked for while its predecessor ends: no wait may miss its phase, no value may be overwritten."""
    for lens, H, Hk, hd in (([42, 120, 77, 464, 33, 56, 409, 783, 2309, 36, 1897, 272, 1676, 18], 16, 2, 128), ([26] * 90 + [0, 3, 160], 8, 2, 64)):
        q, k, v, do, cu = tensors(lens, H, Hk, hd, torch.float16)
        a = [t.requires_grad_(True) for t in (q, k, v)]
        out = nn_ops.attention_packed(*a, cu)
        first = torch.autograd.grad(out, a, do, retain_graph=True)
        for _ in range(400):
            again = torch.autograd.grad(out, a, do, retain_graph=True)
        gemm.check(q.device)
        assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_captured_fp16_step_follows_new_offsets_and_values():
    q, k, v, do, cu = tensors([100, 156, 44, 12], 4, 2, 64, torch.float16)
    a = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        out = nn_ops.attention_packed(*a, cu)
        return [out.detach(), *torch.autograd.grad(out, a, do)]
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for offs, gain in (([0, 100, 256, 300, 312], 1.0), ([0, 1, 1, 312, 312], 2.0 ** -9), ([0, 7, 200, 310, 311], 2.0 ** 11)):
        cu.copy_(torch.tensor(offs, dtype=torch.int32))
        do.mul_(gain)
        for g, _ in graphs:
            g.replay()
        for want, x, y in zip(step(), graphs[0][1], graphs[1][1]):
            assert torch.equal(want, x) and torch.equal(want, y)
