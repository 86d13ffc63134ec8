"""attention_packed on the CPU: the reference against a dense masked softmax, its gradients against differences, its refusals."""
import pytest
import torch

from supergrok15_b200.ops import nn_ops


def dense(q, k, v, cu, causal, scale):
    """All pairs of rows in one score matrix, masked."""
    T, H, hd = q.shape
    k, v = (t.repeat_interleave(H // t.shape[1], 1) for t in (k, v))
    seq = torch.searchsorted(cu.long(), torch.arange(T), right=True)
    live = (seq > 0) & (seq < cu.numel())
    mask = (seq[:, None] == seq[None]) & live[:, None]
    if causal:
        mask &= torch.arange(T)[None] <= torch.arange(T)[:, None]
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    p = torch.where(mask, s.masked_fill(~mask, float("-inf")).softmax(-1), torch.zeros((), dtype=q.dtype))
    return torch.einsum("hij,jhd->ihd", p, v)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("cu,T", [([0, 5, 5, 12], 15), ([0, 1], 1), ([0, 0], 4), ([3, 7, 11], 11), ([0], 3)])
def test_reference_is_the_masked_softmax(cu, T, causal):
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(T, h, 6, generator=g, dtype=torch.float64, requires_grad=True) for h in (4, 2, 2))
    cu = torch.tensor(cu, dtype=torch.int32)
    out = nn_ops.attention_packed(q, k, v, cu, causal, scale=0.3)
    want = dense(q, k, v, cu, causal, 0.3)
    torch.testing.assert_close(out, want, rtol=1e-12, atol=1e-12)
    do = torch.randn(out.shape, generator=g, dtype=torch.float64)
    for a, b in zip(torch.autograd.grad(out, (q, k, v), do), torch.autograd.grad(want, (q, k, v), do)):
        torch.testing.assert_close(a, b.nan_to_num(), rtol=1e-12, atol=1e-12)


def test_gradients_are_differences():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(9, h, 3, generator=g, dtype=torch.float64, requires_grad=True) for h in (6, 2, 2))
    cu = torch.tensor([0, 4, 8], dtype=torch.int64)
    assert torch.autograd.gradcheck(lambda *a: nn_ops.attention_packed(*a, cu), (q, k, v))


def test_rows_of_no_sequence_are_not_read():
    q, k, v = (torch.randn(6, 2, 4) for _ in range(3))
    cu = torch.tensor([0, 4], dtype=torch.int32)
    want = nn_ops.attention_packed(q, k, v, cu)
    for t in (q, k, v):
        t[4:] = float("nan")
    assert torch.equal(nn_ops.attention_packed(q, k, v, cu), want) and not want[4:].any()


def test_refusals():
    q, k, cu = torch.zeros(4, 4, 8), torch.zeros(4, 2, 8), torch.tensor([0, 4], dtype=torch.int32)
    bad = [(q[0], k, k, cu), (q, k, k[:, :1], cu), (q, k[:3], k[:3], cu), (q, k[..., :4], k[..., :4], cu), (q, torch.zeros(4, 3, 8), torch.zeros(4, 3, 8), cu),
           (q, k[:, :0], k[:, :0], cu), (q, k, k, cu[None]), (q, k, k, cu[:0]), (q, k, k, cu.float()), (q, k.double(), k.double(), cu),
           (q, k, k.to(torch.bfloat16), cu)]
    for args in bad:
        with pytest.raises(ValueError, match="attention_packed"):
            nn_ops.attention_packed(*args)
