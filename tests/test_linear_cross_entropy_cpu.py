"""linear_cross_entropy on the CPU: the reference against F.cross_entropy, its gradients against differences, its refusals."""
import pytest
import torch
import torch.nn.functional as F

from supergrok15_b200.ops import nn_ops


def test_reference_is_the_cross_entropy():
    g = torch.Generator().manual_seed(0)
    x, w = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((2, 7, 5), (11, 5)))
    t = torch.randint(0, 11, (2, 7), generator=g)
    t[0, 3] = t[1, 0] = -100
    loss = nn_ops.linear_cross_entropy(x, w, t)
    want = F.cross_entropy((x @ w.t()).reshape(-1, 11), t.reshape(-1))
    torch.testing.assert_close(loss, want, rtol=1e-13, atol=0)
    for a, b in zip(torch.autograd.grad(loss, (x, w)), torch.autograd.grad(want, (x, w))):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-14)
    assert torch.autograd.gradcheck(lambda a, b: nn_ops.linear_cross_entropy(a, b, t), (x, w))


def test_positions_that_are_not_counted():
    x, w = torch.randn(4, 3, requires_grad=True), torch.randn(6, 3)
    assert float(nn_ops.linear_cross_entropy(x, w, torch.full((4,), -100))) == 0.0
    got = nn_ops.linear_cross_entropy(x, w, torch.tensor([2, 6, -1, 5]))              # outside the vocabulary: like ignore_index
    torch.testing.assert_close(got, nn_ops.linear_cross_entropy(x[[0, 3]], w, torch.tensor([2, 5])))
    assert not torch.autograd.grad(got, x)[0][1:3].any()
    assert float(nn_ops.linear_cross_entropy(x[:0], w, torch.zeros(0, dtype=torch.int64))) == 0.0


def test_refusals():
    x, w, t = torch.zeros(4, 8), torch.zeros(6, 8), torch.zeros(4, dtype=torch.int64)
    for args in ((x, w[0], t), (x, w[:, :4], t), (x, w, t[:3]), (x, w[:0], t), (x, w.double(), t), (x, w, t.int()), (x[None], w, t)):
        with pytest.raises(ValueError, match="linear_cross_entropy"):
            nn_ops.linear_cross_entropy(*args)
