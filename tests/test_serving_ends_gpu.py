"""Speculative sampling where sequences of a batch end rounds apart."""
import pytest
import torch

from conftest import pkg
from test_serving_gpu import V, test_speculative_sampling as sampling
from test_serving_steps_gpu import laid_out

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafts", [3, 5])
def test_sequences_that_end_early_stay_inside_their_caches(drafts):
    """One sequence accepts every draft, another hardly any: the first is decoded along for many rounds, and nothing is reported. Its
    tokens are those it gets alone."""
    sv, ops = pkg("serving"), pkg("operators")
    model, other = laid_out(3, torch.float32), laid_out(4, torch.float32)
    P, new = 8, 3 * (drafts + 1) + 1
    prompt = torch.randint(1, V, (2, P), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()
    lens = torch.tensor([P, 3], device="cuda", dtype=torch.int32)
    u = torch.rand((new, 2, 2 * drafts + 1), generator=torch.Generator().manual_seed(6)).cuda()
    u[:, 0, drafts:2 * drafts] = 0.0  # every draft of the first sequence stands
    u[:, 1, drafts:2 * drafts] = 1 - 2.0**-20
    ops.last_kernel_fault()
    tokens, rounds = sv.speculate(model, other, prompt, new, u, drafts=drafts, prompt_lens=lens, page_size=1)
    assert ops.last_kernel_fault() == 0 and rounds > 4
    alone, few = sv.speculate(model, other, prompt[:1], new, u[:, :1].contiguous(), drafts=drafts, page_size=1)
    assert few == 4 and torch.equal(tokens[:1], alone) and ops.last_kernel_fault() == 0


@pytest.mark.parametrize("budget,recent", [(None, 0), (14, 5)])
def test_prompts_in_small_steps(budget, recent, monkeypatch):
    """The same tokens as the float64 models' where prompts take several steps."""
    monkeypatch.setattr(pkg("serving"), "PROMPT_TOKENS", 6)
    sampling(budget, recent)
