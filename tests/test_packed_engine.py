"""The training engine around the operators of packed training."""
import pytest
import torch

from supergrok15_b200.models.llama import LLAMA_TINY, Llama, LlamaConfig
from supergrok15_b200.ops import gemm
from supergrok15_b200.parallel import ZeroEngine


@pytest.mark.gpu
@pytest.mark.parametrize("graph,overlap", [(False, False), (True, False), (False, True)])
def test_a_wait_that_ran_out_inside_a_kernel_is_reported(graph, overlap):
    """The word in which a kernel records such a wait, written here by hand: check() raises for it, and so does the step behind the one that left it."""
    m = Llama(LLAMA_TINY).cuda()
    ids = torch.randint(0, LLAMA_TINY.vocab, (2, 17), device="cuda")
    eng = ZeroEngine(m, "adamw", dict(lr=1e-3), param_dtype=torch.bfloat16, graph=graph, graph_warmup=1, overlap=overlap, model_loss=True)

    def step():
        return eng.train_step(ids[:, :-1].contiguous(), ids[:, 1:].contiguous())
    for _ in range(3):
        step()
    eng.check()
    word = gemm._err_flag(eng.device)
    word.fill_(85)
    with pytest.raises(RuntimeError, match="site 85"):
        eng.check()
    eng.check()                                                           # cleared
    torch.cuda.synchronize()
    step()
    torch.cuda.synchronize()
    word.fill_(93)
    step()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="site 93"):
        step()
    torch.cuda.synchronize()
    assert bool(step().isfinite())
    eng.check()


DOCS = [5, 1, 0, 19, 7]


def packed(device="cpu", shift=0):
    g = torch.Generator().manual_seed(1 + shift)
    T = sum(DOCS) + 3
    ids, y = torch.randint(0, 61, (T,), generator=g).to(device), torch.randint(0, 61, (T,), generator=g).to(device)
    y[::4] = -100
    y[T - 3:] = -100
    docs = DOCS[shift:] + DOCS[:shift]
    return ids, y, torch.tensor([0] + docs).cumsum(0).to(device)


def small(kv, device="cpu"):
    torch.manual_seed(0)
    return Llama(LlamaConfig(n_layers=2, d_model=64, n_heads=4, d_ff=96, vocab=61, max_seq=64, n_kv_heads=kv)).to(device)


@pytest.mark.parametrize("model_loss", [True, False])
def test_engine_trains_on_packed_documents(model_loss):
    """A step on a packed row is the step on its documents: same loss, same parameters afterwards (single process on the CPU)."""
    def train(step):
        m = small(2)
        eng = ZeroEngine(m, "adamw", dict(lr=1e-2), comm="nccl", param_dtype=torch.float32, model_loss=model_loss)
        losses = [float(step(eng, *packed(shift=s))) for s in range(3)]
        return losses, [p.detach().clone() for p in m.parameters()]

    def documents(eng, ids, y, cu):                                       # the rows of a packed batch, one document at a time, through the plain model
        eng.zero_grad()
        keep = [(a, b) for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]) if b > a]
        logits = torch.cat([eng.model(ids[None, a:b])[0] for a, b in keep])
        loss = torch.nn.functional.cross_entropy(logits, torch.cat([y[a:b] for a, b in keep]), ignore_index=-100)
        loss.backward()
        eng.step()
        return loss.detach()
    want = train(documents)
    for got in (train(lambda e, ids, y, cu: e.train_step(ids, y, cu_seqlens=cu)), train(lambda e, ids, y, cu: e.train_step(ids[None], y[None], cu_seqlens=cu.int()))):
        assert all(abs(a - b) <= 1e-5 * b for a, b in zip(got[0], want[0])), (got[0], want[0])
        for a, b in zip(got[1], want[1]):
            torch.testing.assert_close(a, b, rtol=0, atol=2e-4)            # three AdamW steps of 1e-2: a sign that flips on a zero gradient would show


def test_packed_batches_that_are_refused():
    eng = ZeroEngine(small(2), "adamw", dict(lr=1e-2), comm="nccl", param_dtype=torch.float32, model_loss=True)
    ids, y, cu = packed()
    with pytest.raises(ValueError, match="micro_batches"):
        eng.train_step(ids, y, micro_batches=2, cu_seqlens=cu)
    with pytest.raises(ValueError, match="one row of tokens"):
        eng.train_step(ids[:30].view(2, 15), y[:30].view(2, 15), cu_seqlens=cu)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [None, 2])
@pytest.mark.parametrize("model_loss", [True, False])
def test_packed_gradients_through_the_engine(kv, model_loss):
    """Inside the engine (gradient sink, Python autograd functions), against the documents one by one in 64 bits."""
    from test_packed_llama import one_by_one
    m = small(kv, "cuda")
    eng = ZeroEngine(m, "adamw", dict(lr=1e-3), param_dtype=torch.bfloat16, model_loss=model_loss)
    ref = small(kv).double()
    ref.load_state_dict({k: v.double().cpu() for k, v in m.state_dict().items()})
    ids, y, cu = packed()
    loss = eng._fwd_bwd(ids.cuda(), y.cuda(), 1, cu.cuda())
    eng.check()
    want = one_by_one(ref, ids, y, cu)
    want.backward()
    tol = 64 * 2.0 ** -8                                                  # two layers round about twenty times there and back, half a step each
    assert abs(float(loss) - float(want)) <= tol * float(want)
    for (n, p), r in zip(m.named_parameters(), ref.parameters()):
        assert float((p.grad.double().cpu() - r.grad).norm()) <= tol * float(r.grad.norm()), n


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["adamw", "muon"])
def test_captured_packed_steps_follow_the_offsets(optimizer):
    """Batches of one shape with other offsets, from pinned host memory: captured steps beside eager ones."""
    runs = []
    for graph in (False, True):
        m = small(2, "cuda")
        eng = ZeroEngine(m, optimizer, dict(lr=1e-3), param_dtype=torch.bfloat16, graph=graph, graph_warmup=1, model_loss=True)
        runs.append([float(eng.train_step(*(t.pin_memory() for t in packed(shift=s)[:2]), cu_seqlens=packed(shift=s)[2].pin_memory())) for s in (0, 1, 2, 3, 4, 1)])
        eng.check()
        assert not graph or len(eng._graphs) == 1
    assert all(abs(a - b) <= 2.0 ** -8 * abs(b) for a, b in zip(*runs)), runs
