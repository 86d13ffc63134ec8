"""attention_packed and linear_cross_entropy through their Python autograd functions (inside a gradient sink, while tracing) beside the C++ nodes."""
import pytest
import torch

from supergrok15_b200.ops import gemm, nn_ops

pytestmark = pytest.mark.gpu


def attention(dtype, H=4, Hk=2, hd=64):
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(300, H, hd, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(300, Hk, hd, generator=g, device="cuda").to(dtype) for _ in range(2))
    cu = torch.tensor([0, 120, 121, 290], device="cuda", dtype=torch.int32)
    return [q, k, v], lambda q, k, v: nn_ops.attention_packed(q, k, v, cu, True, 0.1)


def loss(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = torch.randn(140, 64, generator=g, device="cuda").to(dtype), torch.randn(300, 64, generator=g, device="cuda").to(dtype)
    t = torch.randint(-20, 300, (140,), generator=g, device="cuda")
    return [x, w], lambda x, w: nn_ops.linear_cross_entropy(x, w, t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("make", [attention, loss])
def test_both_nodes_agree(make, dtype):
    """Bit for bit, for every choice of the inputs that want a gradient; views that the kernels cannot load from among them."""
    inputs, fn = make(dtype)
    odd = [torch.empty(*t.shape[:-1], t.shape[-1] + 3, dtype=dtype, device="cuda")[..., :t.shape[-1]].copy_(t) for t in inputs]
    for args in (inputs, odd):
        for mask in range(1, 2 ** len(args)):
            res = []
            for sink in (False, True):
                a = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(args)]
                with nn_ops.grad_sink(sink):
                    out = fn(*a)
                    res.append([out.detach(), *torch.autograd.grad(out, [t for t in a if t.requires_grad], torch.ones_like(out))])
            for a, b in zip(*res):
                assert torch.equal(a, b)
    with nn_ops.grad_sink(True):
        plain = fn(*inputs)
        assert not plain.requires_grad
    assert torch.equal(plain, fn(*inputs))
    gemm.check(plain.device)


def peak_of(call):
    call()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = call()
    assert not out.requires_grad
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("wanted", [False, True])
def test_nothing_is_kept_without_a_gradient(wanted, sink):
    """A call that no gradient is asked of (no input wants one, or gradients are off) writes its output alone: no statistics, no rest of the
    rounding, no exponentials."""
    q, k, v = (torch.randn(4096, 8, 128, device="cuda", dtype=torch.bfloat16, requires_grad=wanted) for _ in range(3))
    cu = torch.tensor([0, 4096], device="cuda", dtype=torch.int32)
    x, w = (torch.randn(n, 64, device="cuda", dtype=torch.bfloat16, requires_grad=wanted) for n in (2048, 16000))
    t = torch.randint(0, 16000, (2048,), device="cuda")
    with nn_ops.grad_sink(sink), torch.set_grad_enabled(not wanted):
        assert q.numel() * 2 <= peak_of(lambda: nn_ops.attention_packed(q, k, v, cu)) < 1.2 * q.numel() * 2
        assert peak_of(lambda: nn_ops.linear_cross_entropy(x, w, t)) < 2048 * 16000 * 2 // 8
