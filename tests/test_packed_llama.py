"""The decoder over packed documents: attention, positions and loss together, against the documents one by one."""
import pytest
import torch
import torch.nn.functional as F

from supergrok15_b200.models.llama import LLAMA_TINY, Llama, LlamaConfig
from supergrok15_b200.ops import nn_ops

DOCS = [5, 1, 0, 19, 7]


def model(kv, device="cpu", dtype=torch.float64):
    torch.manual_seed(0)
    m = Llama(LlamaConfig(n_layers=2, d_model=64, n_heads=4, d_ff=96, vocab=61, max_seq=32, n_kv_heads=kv)).to(device, dtype)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "norm" in n:
                p.add_(0.1 * torch.randn_like(p))
    return m


def batch(device="cpu", pad=3):
    g = torch.Generator().manual_seed(1)
    T = sum(DOCS) + pad
    ids, y = torch.randint(0, 61, (T,), generator=g).to(device), torch.randint(0, 61, (T,), generator=g).to(device)
    y[::4] = -100
    y[T - pad:] = -100
    return ids, y, torch.tensor([0] + DOCS).cumsum(0).to(device)


def one_by_one(m, ids, y, cu):
    """The mean loss with stored logits, every document in a batch of its own."""
    logits, ys = [], []
    for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]):
        if b > a:
            logits.append(m(ids[None, a:b])[0])
            ys.append(y[a:b])
    return F.cross_entropy(torch.cat(logits), torch.cat(ys), ignore_index=-100)


@pytest.mark.parametrize("kv", [None, 2, 1])
def test_packed_documents_are_documents(kv):
    m = model(kv)
    ids, y, cu = batch()
    want = one_by_one(m, ids, y, cu)
    for got in (m.loss(ids, y, cu), m.loss(ids[None], y[None], cu.to(torch.int32))):
        torch.testing.assert_close(got, want, rtol=1e-10, atol=0)
    ps = list(m.parameters())
    for a, b in zip(torch.autograd.grad(m.loss(ids, y, cu), ps), torch.autograd.grad(want, ps)):
        torch.testing.assert_close(a, b, rtol=1e-8, atol=1e-12)
    assert m(ids, cu).shape == (len(ids), 61)
    with pytest.raises(ValueError, match="one row of tokens"):
        m(ids[:30].view(2, 15), cu)
    with pytest.raises(ValueError, match="not a multiple"):
        model(3)


def test_grouped_heads_of_rows_of_one_length():
    m = model(2)
    ids = torch.randint(0, 61, (3, 9))
    torch.testing.assert_close(m(ids), torch.cat([m(r[None]) for r in ids]), rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(m.loss(ids, ids), F.cross_entropy(m(ids).reshape(-1, 61), ids.reshape(-1)), rtol=1e-10, atol=0)


def test_positions():
    cu = torch.tensor([2, 5, 5, 9], dtype=torch.int32)
    assert nn_ops.packed_positions(cu, 11).tolist() == [0, 1, 0, 1, 2, 0, 1, 2, 3, 0, 1]


def test_default_configuration_is_unchanged():
    torch.manual_seed(3)
    a = Llama(LLAMA_TINY)
    assert [tuple(p.shape) for p in a.layers[0].parameters()] == [(128,), (128,), (128, 128), (128, 128), (128, 128), (128, 128), (352, 128), (352, 128), (128, 352)]


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [None, 2])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_step_on_the_gpu(kv, dtype):
    """One training step's loss and gradients of the whole model against the same documents one by one in 64 bits."""
    from supergrok15_b200.ops import gemm
    m, ref = model(kv, "cuda", dtype), model(kv, "cpu", torch.float64)
    ref.load_state_dict({k: v.double().cpu() for k, v in m.state_dict().items()})
    ids, y, cu = batch("cuda")
    loss = m.loss(ids, y, cu)
    got = torch.autograd.grad(loss, list(m.parameters()))
    gemm.check(ids.device)
    want = one_by_one(ref, ids.cpu(), y.cpu(), cu.cpu())
    wgrads = torch.autograd.grad(want, list(ref.parameters()))
    # each of two layers rounds about twenty times on the way to and back from the loss (projections, rotary, attention, norms, MLP): half a
    # step each, 64 x 2^-8 in bf16; in fp32 sums of up to 96 terms besides
    tol = 64 * 2.0 ** -8 if dtype == torch.bfloat16 else 64 * 96 * 2.0 ** -24
    assert abs(float(loss) - float(want)) <= tol * float(want)
    for (n, _), a, b in zip(m.named_parameters(), got, wgrads):
        assert float((a.double().cpu() - b).norm()) <= tol * float(b.norm()), (n, float((a.double().cpu() - b).norm() / b.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_engine_with_the_models_loss(graph):
    """ZeroEngine(model_loss=True): the loss without stored logits, eager and as a captured step, beside the default path."""
    from supergrok15_b200.parallel import ZeroEngine
    first = []
    for own in (False, True):
        torch.manual_seed(0)
        m = Llama(LLAMA_TINY).cuda()
        ids = torch.randint(0, LLAMA_TINY.vocab, (8, 33), device="cuda")
        eng = ZeroEngine(m, "adamw", dict(lr=1e-3), param_dtype=torch.bfloat16, graph=graph, graph_warmup=1, model_loss=own)
        first.append([float(eng.train_step(ids[:, :-1].contiguous(), ids[:, 1:].contiguous(), micro_batches=2)) for _ in range(4)])
        eng.check()
    # the stored logits are rounded to bf16, half a step of values up to about 4
    assert all(abs(a - b) < 4 * 2.0 ** -8 for a, b in zip(*first)), first
    with pytest.raises(ValueError, match="model_loss"):
        ZeroEngine(Llama(LLAMA_TINY).cuda(), "adamw", dict(lr=1e-3), gather="gemm", model_loss=True)
