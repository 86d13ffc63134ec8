"""The training engine around the operators of packed training."""
import pytest
import torch

from supergrok15_b200.models.llama import LLAMA_TINY, Llama
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
