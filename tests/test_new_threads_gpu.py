"""Products and what is built on them called from a thread whose first CUDA call they are."""
import threading

import pytest
import torch

from llm_in_practise_b200.ops.gemm import gemm
from llm_in_practise_b200.ops.logprobs import linear_token_logprobs


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["gemm", "logprobs", "backward"])
def test_first_cuda_call_of_a_thread(what):
    """All memory comes from torch's cache, so that nothing before the product's tensor maps makes the runtime give the thread its context."""
    x, w = torch.randn(64, 128, device="cuda").bfloat16(), torch.randn(1000, 128, device="cuda").bfloat16().requires_grad_(True)
    t = torch.randint(0, 1000, (64,), device="cuda")

    def run():
        if what == "gemm":
            return gemm(x, w.detach())
        r = linear_token_logprobs(x, w, t).logprob
        return torch.autograd.grad(r.sum(), w)[0] if what == "backward" else r.detach()
    want = run()
    run()
    got = []
    th = threading.Thread(target=lambda: got.append(run()))
    th.start()
    th.join()
    assert len(got) == 1 and torch.equal(got[0], want)
