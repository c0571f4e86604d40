"""Decoding with a paged cache as it is used: prompt, steps, drafted tokens, eviction, against a float64 model on the CPU."""
import math

import pytest
import torch

import serving_ref as ref
from conftest import pkg, rel_err
from oracle import gpt2_oracle as orc

pytestmark = pytest.mark.gpu
V, D, L, H, F, S = 97, 64, 2, 4, 128, 96


class Model:
    """GPT-2 with kept keys and values, float64, one sequence: lists of rows per layer and head, eviction by weight."""

    def __init__(self, params, p):
        self.w = [[t.double() for t in g] for g in params]
        self.p, self.pos = p, 0
        self.k, self.v, self.a = ([[[] for _ in range(H)] for _ in range(L)] for _ in range(3))

    def token(self, t):
        keep, dh = 1.0 - self.p, D // H
        (emb, b_head), (w_pos,) = self.w[0], self.w[1]
        x = (emb[t] * math.sqrt(D) + w_pos[self.pos]) * keep
        for l in range(L):
            g1, b1, w_qkv, w_o, g2, b2, w1, b1f, w2, b2f = self.w[2 + l]
            n = orc.layernorm(g1, b1, x)
            heads = []
            for h in range(H):
                q, k, v = (w_qkv[h, i] @ n for i in range(3))
                self.k[l][h].append(k)
                self.v[l][h].append(v)
                self.a[l][h].append(torch.zeros((), dtype=torch.float64))
                a = torch.softmax(torch.stack(self.k[l][h]) @ q / math.sqrt(dh), dim=0)
                self.a[l][h] = [x + y for x, y in zip(self.a[l][h], a)]
                heads.append(a @ torch.stack(self.v[l][h]) * keep)
            x = x + (w_o @ torch.cat(heads)) * keep
            y = orc.gelu(w1 @ orc.layernorm(g2, b2, x) + b1f)
            x = x + (w2 @ y + b2f) * keep
        self.pos += 1
        g, b = self.w[-1]
        return emb @ orc.layernorm(g, b, x) + b_head

    def rewind(self, n):
        self.pos -= n
        for lists in (self.k, self.v, self.a):
            for l in range(L):
                for h in range(H):
                    del lists[l][h][len(lists[l][h]) - n:]

    def evict(self, budget, recent):
        for l in range(L):
            for h in range(H):
                w = torch.stack(self.a[l][h]).float().view(1, 1, -1)
                kept = [int(i) for i in ref.evict(w, [w.shape[2]], budget, recent)[0, 0] if i >= 0]
                for lists in (self.k, self.v, self.a):
                    lists[l][h] = [lists[l][h][i] for i in kept]


def models(seed, dtype, layers_scale=1.0):
    params = orc.init_params(V, D, L, H, F, S, seed=seed)
    return [[(t * (3.0 if t.dim() > 1 else 1.0)).to(dtype).float() for t in g] for g in params]  # (peaked enough to tell tokens apart)


def on_gpu(params, dtype):
    return [[(t.to(dtype) if t.dim() > 1 else t).cuda() for t in g] for g in params]


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
def test_steps_equal_the_whole_sequence(dtype, bound):
    """A ragged prompt, single tokens and several at once give the logits of the full forward pass (the bounds of the model
    tests: 1e-4 for float32, 2e-2 for bf16, relative to the largest logit)."""
    sv, ev, ops = pkg("serving"), pkg("evaluate"), pkg("operators")
    params = on_gpu(models(0, dtype), dtype)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(1, V, (3, S), generator=g, dtype=torch.int32).cuda()
    full = ev.t_gpt2_forward(params, ids, train=False)
    cache = sv.PagedCache(ev.config_from_params(params, ops.DROPOUT_RATE), 3, page_size=16, dtype=dtype)
    lens = [40, 1, 33]
    counts = torch.tensor(lens, dtype=torch.int32).cuda()
    got = sv.decode_step(params, ids[:, :40], cache, counts)
    for b, n in enumerate(lens):
        assert rel_err(got[b, :n], full[b, :n]) < bound
    at = counts.long()
    for T in (1, 1, 4, 1, 7):
        step = torch.stack([ids[b, at[b]:at[b] + T] for b in range(3)])
        got = sv.decode_step(params, step, cache)
        for b in range(3):
            assert rel_err(got[b], full[b, at[b]:at[b] + T]) < bound
        at = at + T
    # taken back and decoded again, with other tokens in between
    sv.decode_step(params, torch.ones((3, 5), device="cuda", dtype=torch.int32), cache)
    cache.rewind(torch.full((3,), 5, device="cuda", dtype=torch.int32))
    step = torch.stack([ids[b, at[b]:at[b] + 2] for b in range(3)])
    got = sv.decode_step(params, step, cache)
    for b in range(3):
        assert rel_err(got[b], full[b, at[b]:at[b] + 2]) < bound
    assert ops.last_kernel_fault() == 0


def test_evicted_cache():
    """Logits after the caches were cut down, twice, equal those of the float64 model that forgets the same keys."""
    sv, ops = pkg("serving"), pkg("operators")
    prm = models(1, torch.float32)
    params = on_gpu(prm, torch.float32)
    ids = torch.randint(1, V, (2, 60), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    cache = sv.PagedCache(pkg("evaluate").config_from_params(params, ops.DROPOUT_RATE), 2, page_size=8, dtype=torch.float32, track_weights=True)
    plain = [Model(prm, ops.DROPOUT_RATE) for _ in range(2)]
    at = 0
    for n, budget, recent in ((30, 12, 4), (20, 10, 3), (10, 64, 8)):
        for i in range(n):
            got = sv.decode_step(params, ids[:, at:at + 1].cuda(), cache)
            want = torch.stack([m.token(int(ids[b, at])) for b, m in enumerate(plain)])
            assert rel_err(got[:, 0], want) < 1e-4
            at += 1
        cache.evict(budget, recent)
        for m in plain:
            m.evict(budget, recent)
        assert cache.lengths.tolist() == [len(m.k[0][0]) for m in plain]
    assert cache.positions.tolist() == [60, 60] and ops.last_kernel_fault() == 0


@pytest.mark.parametrize("budget,recent", [(None, 0), (14, 5)])
def test_speculative_sampling(budget, recent):
    """Tokens drawn with a draft model equal those of the same procedure on the float64 models with the same random numbers."""
    sv, ops = pkg("serving"), pkg("operators")
    K, new, P = 3, 24, 9
    prm = models(3, torch.float32)
    noise = models(4, torch.float32)
    draft = [[t + 0.2 * n if t.dim() > 1 else t for t, n in zip(a, b)] for a, b in zip(prm, noise)]
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(1, V, (2, P), generator=g, dtype=torch.int32)
    lens = [9, 4]
    u = torch.rand((40, 2, 2 * K + 2), generator=g)
    tokens, rounds = sv.speculate(on_gpu(prm, torch.float32), on_gpu(draft, torch.float32), prompt.cuda(), new, u.cuda(), drafts=K,
                                  temperature=0.8, prompt_lens=torch.tensor(lens, dtype=torch.int32).cuda(), page_size=8, budget=budget,
                                  recent=recent)
    assert ops.last_kernel_fault() == 0
    room = P + new + K + 1 if budget is None else min(P + new + K + 1, max(P, 2 * budget) + K + 1)
    prob = lambda logits: torch.softmax(logits / 0.8, dim=-1)
    accepted_all = 0
    for b in range(2):
        t, d = Model(prm, ops.DROPOUT_RATE), Model(draft, ops.DROPOUT_RATE)
        for x in prompt[b, :lens[b] - 1]:
            t.token(int(x)), d.token(int(x))
        last, out, most = int(prompt[b, lens[b] - 1]), [], P
        for r in range(rounds):
            if budget is not None and most + K + 1 > room:
                t.evict(budget, recent)
                most = budget
            if len(out) >= new:
                most += K + 1
                continue
            fed, guess, q = last, [], []
            for i in range(K + 1):
                logits = d.token(fed)
                if i == K:
                    break
                q.append(prob(logits))
                fed = int(ref.verify(q[-1].view(1, 1, V), torch.empty(1, 0), u[r, b, i].view(1, 1))[0])
                guess.append(fed)
            p = torch.stack([prob(t.token(x)) for x in [last] + guess])
            got, n = ref.verify(p[None], torch.tensor([guess]), u[r, b, K:2 * K + 1][None], torch.stack(q)[None])
            n = int(n)
            accepted_all += n
            t.rewind(K - n), d.rewind(K - n)
            out += got[0, :n + 1].tolist()
            last = out[-1]
            most += K + 1
        assert tokens[b].tolist() == out[:new]
    assert accepted_all > 4


def test_bf16_weights_run_together():
    """bf16: the same calls, tokens within the vocabulary, caches bounded, nothing reported."""
    sv, ops = pkg("serving"), pkg("operators")
    prm = models(6, torch.bfloat16)
    params = on_gpu(prm, torch.bfloat16)
    g = torch.Generator().manual_seed(7)
    prompt = torch.randint(1, V, (5, 20), generator=g, dtype=torch.int32).cuda()
    u = torch.rand((60, 5, 10), generator=g).cuda()
    tokens, rounds = sv.speculate(params, params, prompt, 40, u, drafts=4, budget=16, recent=8)
    assert tokens.shape == (5, 40) and bool(((tokens >= 0) & (tokens < V)).all()) and ops.last_kernel_fault() == 0
    assert rounds <= 40


def test_speculation_takes_a_configuration_and_weights():
    """(GPT2Config, Weights) in place of the pytree: the same tokens."""
    sv, gpt2, ops = pkg("serving"), pkg("gpt2"), pkg("operators")
    params = on_gpu(models(6, torch.bfloat16), torch.bfloat16)
    cfg = gpt2.config_from_params(params, ops.DROPOUT_RATE)
    laid_out = (cfg, gpt2.Weights.from_pytree(params, cfg, torch.bfloat16))
    g = torch.Generator().manual_seed(8)
    prompt = torch.randint(1, V, (2, 9), generator=g, dtype=torch.int32).cuda()
    u = torch.rand((20, 2, 6), generator=g).cuda()
    runs = [sv.speculate(x, x, prompt, 12, u, drafts=2) for x in (params, laid_out)]
    assert torch.equal(runs[0][0], runs[1][0]) and runs[0][1] == runs[1][1]
