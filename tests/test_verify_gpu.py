"""Verification of drafted tokens: accepted counts and drawn tokens equal those of float64 on the CPU."""
import pytest
import torch

import serving_ref as ref
from conftest import pkg

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def inputs(B, K, V, dtype=F32, dists=True, seed=0, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = sharp * torch.randn((B, K + 1, V), generator=g)
    target = torch.softmax(logits, dim=-1).to(dtype)
    draft = torch.softmax(logits[:, :K] + torch.randn((B, K, V), generator=g), dim=-1).to(dtype) if dists else None
    if dists and K:
        tokens = torch.multinomial(draft.float().reshape(B * K, V), 1, generator=g).view(B, K).to(torch.int32)
    else:
        tokens = torch.where(torch.rand((B, K), generator=g) < 0.7, logits[:, :K].argmax(-1),
                             torch.randint(0, V, (B, K), generator=g)).to(torch.int32)
    return target, tokens, torch.rand((B, K + 1), generator=g), draft


def check(target, tokens, uniforms, draft=None, counts=None):
    dev = lambda t: None if t is None else t.cuda()
    out, n = pkg("operators").verify_drafts(dev(target), dev(tokens), dev(uniforms), draft_probs=dev(draft), counts=dev(counts))
    out_want, n_want = ref.verify(target, tokens, uniforms, draft, counts)
    assert torch.equal(n.cpu(), n_want)
    assert torch.equal(out.cpu(), out_want)
    return n_want


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dists", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 4, 50257), (7, 5, 1000), (40, 1, 257), (3, 8, 35374), (5, 3, 1), (200, 2, 33), (2, 0, 5000),
                                   (300, 3, 4099)])
def test_verification(B, K, V, dists, dtype):
    for seed in (0, 1):
        check(*inputs(B, K, V, dtype, dists, seed))


def test_every_outcome_and_counts():
    """Rejections at each place and none, sequences with fewer drafts than columns."""
    target, tokens, uniforms, draft = inputs(64, 4, 500)
    uniforms[:16, :4] = 0.0                        # everything is accepted
    for b in range(16, 32):
        uniforms[b, :4] = 0.0
        tokens[b, b % 4] = int(target[b, b % 4].argmin())
        draft[b, b % 4, tokens[b, b % 4]] = 1.0
        uniforms[b, b % 4] = 0.999                 # a rejection at place b % 4
    counts = torch.arange(64, dtype=torch.int32) % 5
    assert set(check(target, tokens, uniforms, draft).tolist()) == {0, 1, 2, 3, 4}
    check(target, tokens, uniforms, draft, counts)
    check(target, tokens, uniforms, None, counts)


def test_borders():
    """Equality is a rejection; the running sum has to pass its mark; steps of exact powers of two."""
    V = 1024
    target = torch.full((6, 2, V), 1.0 / V)
    tokens = torch.tensor([[5]] * 6, dtype=torch.int32)
    draft = torch.full((6, 1, V), 1.0 / V)
    uniforms = torch.tensor([[0.0, 0.0], [0.5, 0.5], [0.999, 0.25], [0.25, 1023.0 / 1024], [0.1, 1 - 2.0**-24], [0.0, 2.0**-30]])
    check(target, tokens, uniforms, draft)
    draft[:, 0, 5] = 0.5                           # accepted below 2 / V only
    draft[:, 0, 6:] = 0.0
    uniforms[:, 0] = torch.tensor([2.0 / V, 1.9 / V, 2.1 / V, 0.9, 0.8, 0.7])
    n = check(target, tokens, uniforms, draft)
    assert n.tolist() == [0, 1, 0, 0, 0, 0]


def test_nothing_left_to_draw_from():
    """A draft rejected although both models agree: the likeliest token, the first among equals. NaN counts as nothing."""
    target = torch.zeros((3, 2, 300))
    target[:, 0, 17] = target[:, 0, 200] = 0.5
    target[:, 1, 3] = 1.0
    draft = target[:, :1].clone()
    tokens = torch.tensor([[9], [17], [-1]], dtype=torch.int32)
    uniforms = torch.tensor([[0.5, 0.5], [1.0, 0.5], [0.0, 0.3]])
    check(target, tokens, uniforms, draft)
    target[:, 0, :10] = float("nan")
    draft[:, 0, 280:] = float("nan")
    check(target, tokens, uniforms, draft)
    target[:] = float("nan")
    target[:, :, 41] = 0.25
    check(target, torch.full((3, 1), 41, dtype=torch.int32), uniforms, None)


def test_tokens_outside_the_vocabulary_are_rejected():
    target, tokens, uniforms, draft = inputs(4, 3, 100)
    tokens[0, 0], tokens[1, 1], tokens[2, 2], tokens[3, 0] = -1, 100, 2**31 - 1, -2**31
    uniforms[:, :3] = 0.0
    assert check(target, tokens, uniforms, draft).tolist() == [0, 1, 2, 0]
    assert check(target, tokens, uniforms, None).tolist() == [0, 1, 2, 0]


def test_views_and_replay():
    """Rows of padded logits (first vocab columns) and a recorded call replayed with other numbers."""
    ops = pkg("operators")
    target, tokens, uniforms, draft = inputs(5, 3, 1001)
    wide_t, wide_d = torch.full((5, 4, 1024), 9.0), torch.full((5, 3, 1100), 9.0)
    wide_t[:, :, :1001], wide_d[:, :, 3:1004] = target, draft
    wide_t, wide_d = wide_t.cuda()[:, :, :1001], wide_d.cuda()[:, :, 3:1004]
    du, dt = uniforms.cuda(), tokens.cuda()
    out, n = ops.verify_drafts(wide_t, dt, du, draft_probs=wide_d)
    want = ref.verify(target, tokens, uniforms, draft)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(n.cpu(), want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, n = ops.verify_drafts(wide_t, dt, du, draft_probs=wide_d)
    uniforms = 1.0 - 2.0**-24 - uniforms
    du.copy_(uniforms)
    graph.replay()
    torch.cuda.synchronize()
    want = ref.verify(target, tokens, uniforms, draft)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(n.cpu(), want[1])


def test_tokens_are_distributed_as_the_target():
    """20000 sequences of one draft: frequencies of the first token against the target's probabilities. The number of hits of a
    token is binomial; all of 12 counts lie within 5 standard deviations but for a chance of 1e-5."""
    V, N = 12, 20000
    g = torch.Generator().manual_seed(0)
    p, q = (torch.softmax(torch.randn(V, generator=g), 0) for _ in range(2))
    target, draft = p.expand(N, 2, V).contiguous(), q.expand(N, 1, V).contiguous()
    tokens = torch.multinomial(q, N, replacement=True, generator=g).view(N, 1).to(torch.int32)
    out, _ = pkg("operators").verify_drafts(target.cuda(), tokens.cuda(), torch.rand((N, 2), generator=g).cuda(), draft_probs=draft.cuda())
    hits = torch.bincount(out[:, 0].cpu().long(), minlength=V).double()
    assert bool(((hits - N * p.double()).abs() <= 5 * (N * p.double() * (1 - p.double())).sqrt()).all())
