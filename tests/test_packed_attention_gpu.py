"""attention_packed on the GPU against its statement in 64 bits, at the lengths, head layouts and strides where it can go wrong."""
import pytest
import torch

from supergrok15_b200.ops import gemm, nn_ops

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def tolerance(dtype, longest, hd, roundings):
    """Distance over norm.  16-bit: the roundings on the way (probabilities and result; backward: also ds, and the output inside delta), half a
    step each.  fp32: sums of up to hd, then `longest` terms, each at most that many half steps off."""
    return HALF_STEP[dtype] * (roundings if dtype != torch.float32 else hd + longest)


def far(a, b, scale=0.0):
    b = b.double()
    d, n = float((a.double() - b).norm()), max(float(b.norm()), scale)
    return d / n if n else d


def inputs(lens, pad, H, Hk, hd, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(lens) + 7 * hd + H)
    T = sum(lens) + pad
    q, do = (torch.randn(T, H, hd, generator=g, device="cuda").to(dtype) for _ in range(2))
    k, v = (torch.randn(T, Hk, hd, generator=g, device="cuda").to(dtype) for _ in range(2))
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    return q, k, v, do, cu


def check(q, k, v, do, cu, causal, scale=None):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = nn_ops.attention_packed(q, k, v, cu, causal, scale)
    grads = torch.autograd.grad(out, (q, k, v), do)
    again = torch.autograd.grad(nn_ops.attention_packed(q, k, v, cu, causal, scale), (q, k, v), do)
    gemm.check(q.device)
    ref = [t.detach().double().requires_grad_(True) for t in (q, k, v)]
    want = nn_ops.attention_packed_reference(*ref, cu, causal, scale)
    wgrads = torch.autograd.grad(want, ref, do.double())
    longest = int((cu[1:] - cu[:-1]).max()) if cu.numel() > 1 else 0
    assert out.dtype == q.dtype and out.is_contiguous()
    assert far(out, want.detach()) <= tolerance(q.dtype, longest, q.shape[2], 2), ("out", far(out, want.detach()))
    for n, a, b, c in zip(("dq", "dk", "dv"), grads, wgrads, again):
        assert torch.equal(a, c), n                                       # no atomics: fixed order
        # a sequence of one row has p = 1, ds = do.v - do.o = 0: what is left is the rounding of the two products, so they are the scale
        size = float(do.norm() * v.detach().norm() * (k if n == "dq" else q).detach().norm()) if longest <= 1 and n != "dv" else 0.0
        assert far(a, b, size) <= tolerance(q.dtype, longest, q.shape[2], 4), (n, far(a, b, size))
    return out, grads


LENGTHS = [([1], 0), ([0], 5), ([0, 5, 0, 0, 3], 0), ([63, 64, 65], 1), ([127, 1, 128, 129], 0), ([255, 0, 257, 384], 200), ([700, 3], 0), ([2] * 70, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,pad", LENGTHS)
def test_lengths(lens, pad, dtype):
    for causal in (True, False):
        check(*inputs(lens, pad, 4, 2, 64, dtype), causal)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hk,hd", [(1, 1, 128), (3, 3, 128), (8, 1, 64), (7, 1, 128), (6, 2, 32), (16, 8, 80), (4, 4, 96), (2, 2, 40), (2, 1, 8), (2, 1, 7), (3, 1, 1)])
def test_heads(H, Hk, hd, dtype):
    check(*inputs([40, 300, 131], 3, H, Hk, hd, dtype), True, scale=0.2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequence(dtype):
    for causal in (True, False):
        check(*inputs([2600, 1500], 20, 2, 1, 128, dtype), causal)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_sequences(dtype):
    """More sequences than two levels of the 32-ary search tell apart, many of them empty."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 4, (1500,), generator=g).tolist()
    lens[700] = 333
    check(*inputs(lens, 9, 2, 1, 32, dtype), True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mostly_padding(dtype):
    """Long runs of work items without a sequence, before, between and behind items with one."""
    q, k, v, do, cu = inputs([300], 30000, 4, 4, 64, dtype)
    for start in (0, 15000, 30000):
        check(q, k, v, do, cu + start, True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """Views of one fused projection, heads before rows, a row pitch TMA cannot take, a base that is not 16-byte aligned, a broadcast head."""
    q, k, v, do, cu = inputs([70, 200], 2, 4, 4, 64, dtype)
    want, wg = check(q, k, v, do, cu, True)
    T = q.shape[0]
    fused = torch.cat([q, k, v], 1)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    odd = [torch.empty(T, 4, 67, dtype=dtype, device="cuda")[:, :, :64].copy_(t) for t in (q, k, v)]
    off = [torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    across = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    for views in ([fused[:, :4], fused[:, 4:8], fused[:, 8:]], heads_first, odd, off, across):
        out, grads = check(*views, do, cu, True)
        assert far(out, want) <= tolerance(dtype, 200, 64, 4)
        assert all(far(a, b) <= tolerance(dtype, 200, 64, 8) for a, b in zip(grads, wg))
    one = [t[:, :1].expand(-1, 4, -1) for t in (k, v)]
    check(q, *one, do.transpose(0, 1).contiguous().transpose(0, 1), cu, True)
    check(q, *one, do[:1].expand(T, -1, -1), cu, True)


def test_broadcast_inputs_gather_their_gradient():
    q, k, v, do, cu = inputs([50, 90], 0, 4, 4, 64, torch.float32)
    k1 = k[:, :1].detach().requires_grad_(True)
    g1, = torch.autograd.grad(nn_ops.attention_packed(q, k1.expand(-1, 4, -1), v, cu), k1, do)
    g2, = torch.autograd.grad(nn_ops.attention_packed(q, k1, v[:, :1], cu), k1, do)
    vv = v[:, :1].expand(-1, 4, -1)
    g3, = torch.autograd.grad(nn_ops.attention_packed(q, k1.expand(-1, 4, -1), vv, cu), k1, do)
    assert far(g3, g2) < 1e-5 and g1.shape == k1.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_values_outside_a_sequence_never_reach_it(dtype):
    """NaN, infinities and the type's largest values behind the last sequence and in the neighbouring ones."""
    q, k, v, do, cu = inputs([90, 130, 61], 40, 4, 2, 64, dtype)
    out, grads = check(q, k, v, do, cu, True)
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).max):
        z = [t.detach().clone() for t in (q, k, v, do)]
        for t in z:
            t[:90] = bad
            t[220:] = bad
        a = [t.requires_grad_(True) for t in z[:3]]
        o = nn_ops.attention_packed(*a, cu)
        g = torch.autograd.grad(o, a, z[3])
        assert torch.equal(o[90:220], out[90:220])
        assert all(torch.equal(x[90:220], y[90:220]) for x, y in zip(g, grads))
        assert not any(x[281:].any() for x in (o, *g))


def test_scores_far_apart():
    """Scores of several hundred: the running maximum moves by more than any exponential can hold."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        q, k, v, do, cu = inputs([300, 140], 0, 2, 2, 64, dtype)
        ramp = torch.linspace(-3, 3, q.shape[0], device="cuda")[:, None, None]
        check((q * 4 + 8).to(dtype), (k + ramp * 2).to(dtype), v, do, cu, True)


def test_long_offsets_int64_and_streams():
    q, k, v, do, cu = inputs([33, 250], 5, 4, 2, 64, torch.bfloat16)
    want = nn_ops.attention_packed(q, k, v, cu)
    assert torch.equal(nn_ops.attention_packed(q, k, v, cu.long()), want)
    assert torch.equal(nn_ops.attention_packed(q, k, v, torch.stack([cu, cu], 1)[:, 0]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = nn_ops.attention_packed(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_step_follows_new_offsets(dtype):
    q, k, v, do, cu = inputs([100, 156, 44], 12, 4, 2, 64, dtype)
    a = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        out = nn_ops.attention_packed(*a, cu)
        return [out.detach(), *torch.autograd.grad(out, a, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                                    # two graphs over the same inputs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for offs in ([0, 100, 256, 300], [0, 1, 1, 312], [0, 7, 200, 310]):
        cu.copy_(torch.tensor(offs, dtype=torch.int32))
        for g, _ in graphs:
            g.replay()
        for want, x, y in zip(step(), graphs[0][1], graphs[1][1]):
            assert torch.equal(want, x) and torch.equal(want, y)


def test_offsets_out_of_order_stay_in_range():
    """Offsets that do not ascend or point past the rows give undefined rows, not an access out of range (every offset is clamped, every store
    checked against its segment): the call returns and the next one is right."""
    q, k, v, do, cu = inputs([100, 156, 44], 12, 4, 2, 64, torch.float32)
    want = nn_ops.attention_packed(q, k, v, cu)
    for bad in ([0, 400, 50, 312], [-5, 9999, 2 ** 31 - 1, 17]):
        nn_ops.attention_packed(q, k, v, torch.tensor(bad, dtype=torch.int32, device="cuda"))
    assert torch.equal(nn_ops.attention_packed(q, k, v, cu), want)


def test_refusals():
    q, k, v, _, cu = inputs([5], 0, 4, 2, 64, torch.float32)
    with pytest.raises(ValueError, match="one device"):
        nn_ops.attention_packed(q, k, v, cu.cpu())
    with pytest.raises(ValueError, match="head sizes up to 128"):
        nn_ops.attention_packed(q.repeat(1, 1, 3), k.repeat(1, 1, 3), v.repeat(1, 1, 3), cu)
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        nn_ops.attention_packed(q.double(), k.double(), v.double(), cu)
    for args in ((q[0], k, k, cu), (q, k, k[:, :1], cu), (q, k[:3], k[:3], cu), (q, k[..., :32], k[..., :32], cu), (q, k.repeat(1, 3, 1)[:, :3], k.repeat(1, 3, 1)[:, :3], cu),
                 (q, k[:, :0], k[:, :0], cu), (q, k, k, cu[None]), (q, k, k, cu[:0]), (q, k, k, cu.float()), (q, k, k.half(), cu), (q[..., :0], k[..., :0], k[..., :0], cu)):
        with pytest.raises(ValueError, match="attention_packed"):
            nn_ops.attention_packed(*args)
    out = nn_ops.attention_packed(q.requires_grad_(True), k, v, cu)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        torch.autograd.grad(out.sum(), q, create_graph=True)
    assert nn_ops.attention_packed(q[:0], k[:0], v[:0], cu[:1] * 0).shape == (0, 4, 64)


def test_many_backward_passes_agree():
    """Warps of one CTA drift apart by more than a tile now and then (once in some hundred passes of this size): no wait may miss its phase."""
    q, k, v, do, cu = inputs([42, 120, 77, 464, 33, 56, 409, 783, 2309, 36, 1897, 272, 1676, 18], 0, 16, 2, 128, torch.bfloat16)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = nn_ops.attention_packed(q, k, v, cu)
    first = torch.autograd.grad(out, (q, k, v), do, retain_graph=True)
    for _ in range(600):
        again = torch.autograd.grad(out, (q, k, v), do, retain_graph=True)
    gemm.check(q.device)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_no_query_heads():
    k, v = (torch.randn(10, 2, 32, device="cuda", dtype=torch.bfloat16).requires_grad_(True) for _ in range(2))
    q = torch.empty(10, 0, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = nn_ops.attention_packed(q, k, v, torch.tensor([0, 10], device="cuda"))
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.empty_like(out))
    assert out.shape == dq.shape == q.shape and not dk.any() and not dv.any()
