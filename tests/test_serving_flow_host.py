"""What serving does on the host: sizes that are kept between calls, caches behind calls that fail, the order of speculative rounds."""
import pytest
import torch

from conftest import pkg
from test_serving_host import BF16, F32, I32, cache, ops, rows  # noqa: F401 (ops: a fixture)


@pytest.mark.parametrize("refused", [dict(out=torch.zeros(2, 1, 1, 64, dtype=BF16).expand(2, 4, 1, 64)), dict(k=rows())])
def test_a_refused_call_leaves_later_ones_alone(ops, refused):  # noqa: F811
    """A call that the library refuses, then a good one of the same sizes that needs a workspace: it gets past the workspace's check."""
    if torch.cuda.is_available():
        pytest.skip("host addresses must not reach a GPU")
    ops._DECODE_BYTES.clear()
    w = torch.zeros(2, 2, 32)
    with pytest.raises(RuntimeError, match="bad shape"):
        ops.attn_decode(rows(4), **cache(), weights=w, **refused)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="sm_100"):
            ops.attn_decode(rows(4), **cache(), weights=w)


class Rounds:
    """speculate on the CPU with a model that knows no tokens: every step is checked against its cache's room, drafts stand as told."""

    def __init__(self, monkeypatch, stands, seq=64):
        sv, gpt2 = pkg("serving"), pkg("gpt2")
        self.sv, self.stands, self.steps = sv, torch.tensor(stands, dtype=I32), []
        cfg = gpt2.GPT2Config(vocab=10, dim=8, layers=1, heads=2, ffn=16, seq=seq)
        monkeypatch.setattr(sv, "_weights", lambda params, dtype, p=None: (cfg, params))
        monkeypatch.setattr(sv, "decode_step", self.decode_step)
        monkeypatch.setattr(sv, "probabilities", lambda logits, temperature=1.0: logits)
        monkeypatch.setattr(sv.ops, "verify_drafts", self.verify)

    def decode_step(self, model, ids, cache, counts=None):
        added = torch.full_like(cache.lengths, ids.shape[1]) if counts is None else counts
        assert bool(((added >= 0) & (added <= ids.shape[1])).all())
        cache.lengths += added
        cache.positions += added
        assert int(cache.lengths.max()) <= cache.capacity and int(cache.positions.max()) <= cache.cfg.seq
        self.steps.append((cache, ids, counts))
        return torch.zeros(*ids.shape, 10)

    def verify(self, target, tokens, uniforms, draft_probs=None):
        B, K = tokens.shape
        out = torch.arange(K + 1, dtype=I32).repeat(B, 1)
        n = torch.minimum(self.stands, torch.full((B,), K, dtype=I32))
        return torch.where(out <= n[:, None], out, 0), n

    def __call__(self, P, new, drafts, rounds, **kw):
        B = len(self.stands)
        return self.sv.speculate([[torch.zeros(1)]], [[torch.zeros(1)]], torch.ones(B, P, dtype=I32), new,
                                 torch.zeros(rounds, B, 2 * drafts + 1), drafts=drafts, **kw)


@pytest.mark.parametrize("drafts", [1, 2, 3, 5])
@pytest.mark.parametrize("new", [1, 6, 13])
def test_sequences_that_end_early_need_no_more_room(monkeypatch, drafts, new):
    """All drafts of one sequence stand, none of another's: no step goes beyond the caches, and the tokens are the rounds' own."""
    run = Rounds(monkeypatch, [drafts, 0, 1])
    tokens, rounds = run(8, new, drafts, new, page_size=1)
    assert rounds == new
    for b, n in enumerate((drafts, 0, min(1, drafts))):
        assert tokens[b].tolist() == [i % (n + 1) for i in range(new)]


def small_cache(**kw):
    sv, gpt2 = pkg("serving"), pkg("gpt2")
    cfg = gpt2.GPT2Config(vocab=10, dim=8, layers=3, heads=2, ffn=16, seq=32)
    c = sv.PagedCache(cfg, 2, capacity=20, page_size=4, device="cpu", **kw)
    c.lengths += 6
    c.positions += 7
    return sv, cfg, c


@pytest.mark.parametrize("counts", [None, torch.tensor([1, 0], dtype=I32), torch.tensor([1, 0])])
def test_a_step_that_fails_leaves_the_cache_as_it_was(counts):
    """(It fails here for want of a GPU.) What the cache counts is what it holds."""
    sv, cfg, c = small_cache()
    w = dict(w_emb=torch.zeros(10, 8), w_pos=torch.zeros(32, 8))
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        sv.decode_step((cfg, w), torch.zeros(2, 3, dtype=I32), c, counts)
    assert c.lengths.tolist() == [6, 6] and c.positions.tolist() == [7, 7]


def test_an_eviction_that_fails_half_way_is_not_decoded_on(monkeypatch):
    """The first layer is cut, the second one's call raises: lengths stand for neither, so the cache refuses to go on. A call that is
    refused before any layer is cut leaves it usable."""
    sv, cfg, c = small_cache(track_weights=True)
    done = []

    def evict(k, v, table, lengths, weights, budget, recent):
        if budget < 1:
            raise ValueError("budget")
        if len(done) == 1:
            raise RuntimeError("out of memory")
        done.append(1)
        return None, torch.clamp(lengths, max=budget)

    monkeypatch.setattr(sv.ops, "kv_evict", evict)
    with pytest.raises(ValueError, match="budget"):
        c.evict(0, 0)
    with pytest.raises(RuntimeError, match="out of memory"):
        c.evict(4, 2)
    for call in (lambda: c.evict(4, 2), lambda: sv.decode_step((cfg, None), torch.zeros(2, 1, dtype=I32), c)):
        with pytest.raises(RuntimeError, match="some of its layers"):
            call()


@pytest.mark.parametrize("back", [9, 40, 1 << 20])
def test_positions_before_the_first_are_no_index(back):
    """More tokens taken back than were seen: the position table is read inside its rows (beyond them an index ends a GPU's context)."""
    sv, cfg, c = small_cache()
    c.rewind(torch.full((2,), back, dtype=I32))
    w = dict(w_emb=torch.zeros(10, 8), w_pos=torch.zeros(32, 8))
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        sv.decode_step((cfg, w), torch.zeros(2, 3, dtype=I32), c)


@pytest.mark.parametrize("change", [dict(prompt=torch.ones(2, 0, dtype=I32)), dict(prompt_lens=torch.tensor([6, 2], dtype=I32)),
                                    dict(prompt_lens=torch.tensor([5, 0], dtype=I32)), dict(prompt_lens=torch.tensor([-1, 5], dtype=I32)),
                                    dict(prompt_lens=torch.tensor([5], dtype=I32)), dict(prompt_lens=torch.tensor([5, 5]))])
def test_prompts_have_a_token_and_lengths_within_them(monkeypatch, change):
    """The last token of each prompt is picked by its length: an index outside the prompt would end a GPU's context."""
    run = Rounds(monkeypatch, [1, 0])
    args = dict(prompt=torch.ones(2, 5, dtype=I32), new_tokens=3, uniforms=torch.zeros(9, 2, 5), drafts=2)
    run.sv.speculate([[torch.zeros(1)]], [[torch.zeros(1)]], **args, prompt_lens=torch.tensor([1, 5], dtype=I32))
    args.update(change)
    with pytest.raises(ValueError, match="prompt"):
        run.sv.speculate([[torch.zeros(1)]], [[torch.zeros(1)]], **args)


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan")])
def test_temperatures_that_leave_no_probabilities_are_refused(monkeypatch, temperature):
    """(Divided by 0, a row of logits has no softmax, and token 0 came of it.)"""
    real = pkg("serving").probabilities
    run = Rounds(monkeypatch, [1, 0])
    with pytest.raises(ValueError, match="temperature"):
        run(5, 3, 2, 9, temperature=temperature)
    assert not run.steps
    with pytest.raises(ValueError, match="temperature"):
        real(torch.zeros(1, 4), temperature)


def test_random_numbers_are_used_once(monkeypatch):
    """Two rounds' numbers for what takes three: tokens of numbers used again would not be independent."""
    run = Rounds(monkeypatch, [2, 0])
    tokens, rounds = run(5, 3, 2, 3)
    assert rounds == 3
    with pytest.raises(ValueError, match="uniforms"):
        run(5, 3, 2, 2)


def test_no_new_tokens_leave_the_weights_they_were_given(ops):  # noqa: F811
    """T == 0: weights_out holds what the call adds nothing to, below each length; slots behind are left as they were. Tensors that do
    not fit are refused as ever."""
    c = cache()
    c["lengths"].copy_(torch.tensor([5, 0], dtype=I32))
    w, out = torch.rand(2, 2, 33), torch.full((2, 2, 33), 7.0)
    assert ops.attn_decode(rows(T=0), **c, weights=w, weights_out=out).shape == (2, 2, 0, 64)
    want = torch.full((2, 2, 33), 7.0)
    want[0, :, :5] = w[0, :, :5]
    assert torch.equal(out, want)
    ops.attn_decode(rows(T=0), **c, weights_out=out)  # weights None: zeros
    want[0, :, :5] = 0.0
    assert torch.equal(out, want)
    before = w.clone()
    ops.attn_decode(rows(T=0), **c, weights=w)
    assert torch.equal(w, before)
    for bad in (dict(weights=torch.zeros(2, 2, 31)), dict(weights=torch.zeros(2, 2, 32, dtype=BF16)),
                dict(weights=torch.zeros(2, 2, 32), weights_out=torch.zeros(2, 2, 33))):
        with pytest.raises(ValueError):
            ops.attn_decode(rows(T=0), **c, **bad)


@pytest.mark.parametrize("P,lens", [(1, [1, 1, 1]), (2, [2, 1, 2]), (101, [101, 1, 60]), (5000, [5000, 4097, 33])])
def test_prompts_are_fed_in_bounded_steps(monkeypatch, P, lens):
    """Every token of a prompt but its last once and in order, into both caches, never more tokens at once than a step is allowed."""
    run = Rounds(monkeypatch, [1, 0, 2], seq=6000)
    most = run.sv.PROMPT_TOKENS
    monkeypatch.setattr(run.sv, "PROMPT_TOKENS", 96 if P < 1000 else most)
    prompt = torch.arange(3 * P, dtype=I32).view(3, P)
    run.sv.speculate([[torch.zeros(1)]], [[torch.zeros(1)]], prompt, 2, torch.zeros(2, 3, 5), drafts=2,
                     prompt_lens=torch.tensor(lens, dtype=I32))
    for c in {id(c): c for c, _, _ in run.steps}.values():
        fed = [[] for _ in lens]
        for _, ids, counts in (s for s in run.steps if s[0] is c and s[2] is not None):
            assert ids.numel() <= run.sv.PROMPT_TOKENS and ids.shape[1] <= 4096
            for b, n in enumerate(counts.tolist()):
                fed[b] += ids[b, :n].tolist()
        assert fed == [prompt[b, :n - 1].tolist() for b, n in enumerate(lens)]
