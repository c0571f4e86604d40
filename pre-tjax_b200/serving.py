"""Decoding with kept keys and values on the sm_100a kernels, ``train=False`` semantics, float32 or bf16 weights.

The reference's ``predict`` runs the whole sequence for every new token (loss_and_optimizer_triton.py:203-212). Here the keys and
values of earlier tokens stay in a paged cache (``operators.attn_decode``), so that a token costs one row of every product:

* ``PagedCache``   pages, page table and lengths of a batch of sequences, all layers
* ``decode_step``  logits of the newest tokens of each sequence: one, a prompt, or several drafted ones
* ``speculate``    sampling with a draft model: the draft proposes tokens, the target looks at all of them in one step and
                   ``operators.verify_drafts`` keeps those that leave the target's distribution unchanged

A cache may be bounded: ``PagedCache.evict`` keeps the last keys and those that received the most attention
(``operators.kv_evict``). Positions go on counting the tokens, not the keys that are left.
"""
from __future__ import annotations

import torch

from . import _lib, operators as ops
from .gpt2 import GPT2Config, Weights, config_from_params


class PagedCache:
    """Keys and values of `batch` sequences of a model, at most `capacity` keys each, in pages of `page_size`. One page table serves
    all layers; ``k[l]`` and ``v[l]`` are layer l's pools [pages, heads, page_size, d_head]. lengths int32 [batch]: keys kept;
    positions int64 [batch]: tokens seen. weights (track_weights): the attention that every key received, per layer. All of them
    change in place."""

    def __init__(self, cfg: GPT2Config, batch: int, capacity: int = None, page_size: int = 16, dtype=torch.bfloat16, device="cuda",
                 track_weights: bool = False):
        capacity = cfg.seq if capacity is None else capacity
        if batch < 1 or capacity < 1 or page_size < 1:
            raise ValueError("a cache needs at least one sequence, one key and one slot per page")
        width = -(-capacity // page_size)
        self.cfg, self.batch, self.capacity = cfg, batch, capacity
        shape = (cfg.layers, batch * width, cfg.heads, page_size, cfg.d_head)
        self.k, self.v = (torch.empty(shape, device=device, dtype=dtype) for _ in range(2))
        self.page_table = torch.arange(batch * width, device=device, dtype=torch.int32).view(batch, width)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        self.positions = torch.zeros(batch, device=device, dtype=torch.int64)
        self._cut = 0  # layers that an unfinished eviction has cut
        self.weights = None
        if track_weights:
            self.weights = torch.zeros((cfg.layers, batch, cfg.heads, width * page_size), device=device, dtype=torch.float32)

    def rewind(self, counts: torch.Tensor) -> None:
        """Takes the last counts[b] (int32) tokens of each sequence back: drafted tokens that were not accepted. (The attention
        they paid to earlier keys stays in the weights.)"""
        self.lengths -= counts
        self.positions -= counts

    def evict(self, budget: int, recent: int) -> None:
        """Cuts every sequence down to `budget` keys per head: the last `recent` and the heaviest of the others."""
        if self.weights is None:
            raise RuntimeError("eviction goes by attention weights: make the cache with track_weights=True")
        self.check_whole()
        for l in range(self.cfg.layers):
            _, lengths = ops.kv_evict(self.k[l], self.v[l], self.page_table, self.lengths, self.weights[l], budget, recent)
            self._cut = l + 1
        self.lengths.copy_(lengths)
        self._cut = 0

    def check_whole(self) -> None:
        """Raises where an eviction failed between two layers: no lengths fit all of them any more."""
        if self._cut:
            raise RuntimeError("an eviction from this cache failed behind some of its layers: its sequences have to be decoded anew")


def decode_step(params, ids: torch.Tensor, cache: PagedCache, counts: torch.Tensor = None, p: float = None) -> torch.Tensor:
    """Appends the tokens ids [B, T], T <= 4096, to the sequences of a cache and returns their logits [B, T, vocab] (train=False).
    counts int32 [B]: the first counts[b] of a sequence's T ids are tokens (default T); what comes back behind them means nothing.
    params: the reference's pytree (model_torch_func.py:36-43) or (GPT2Config, gpt2.Weights). A cache that tracks weights takes a
    workspace of B * heads * T * (slots of a sequence) floats: long prompts go in several steps. The caller sees to it that no
    sequence passes the cache's capacity or the model's positions: keys beyond are reported by operators.last_kernel_fault. A step
    with laid-out weights may be recorded in a CUDA graph: every replay advances the cache, which keeps its tensors, by one more step
    of the ids then in place."""
    cfg, w = _weights(params, cache.k.dtype, p)
    if (cfg.layers, cfg.heads, cfg.d_head) != (cache.cfg.layers, cache.cfg.heads, cache.cfg.d_head):
        raise ValueError("the cache was made for another model")
    cache.check_whole()
    B, T = ids.shape
    if B != cache.batch:
        raise ValueError(f"{B} sequences for a cache of {cache.batch}")
    D, H, dh, rows, p = cfg.dim, cfg.heads, cfg.d_head, B * T, cfg.dropout
    added = T if counts is None else counts.clamp(0, T)  # (what the kernels bring out of range to its nearer bound)
    lengths = cache.lengths + added
    at = (cache.positions[:, None] + torch.arange(T, device=ids.device)).clamp_(0, cfg.seq - 1)
    x = ops.embed_fwd(ids.reshape(1, rows), w["w_emb"], w["w_pos"][at.reshape(-1)], False, 0, out_dtype=cache.k.dtype, p=p).view(rows, D)
    for l in range(cfg.layers):
        g = lambda n: w[f"l{l}.{n}"]
        qkv = ops.gemm(ops.t_layernorm_fwd_t((g("g1"), g("b1")), x), g("w_qkv").view(3 * D, D))  # columns (head, q/k/v, d_head)
        q, k, v = qkv.view(B, T, H, 3, dh).permute(3, 0, 2, 1, 4).unbind(0)
        attn = x.new_empty((rows, D))
        ops.attn_decode(q, cache.k[l], cache.v[l], cache.page_table, lengths, k=k, v=v, counts=counts,
                        weights=None if cache.weights is None else cache.weights[l], out=attn.view(B, T, H, dh).transpose(1, 2), p=p)
        x = ops.gemm(attn, g("w_o"), epilogue=_lib.EPI_DROPOUT_RESID, aux=x, dropout_args=(p, False, 0, 0))
        h = ops.gemm(ops.t_layernorm_fwd_t((g("g2"), g("b2")), x), g("w1"), bias=g("b1f"), epilogue=_lib.EPI_GELU)
        x = ops.gemm(h, g("w2"), bias=g("b2f"), epilogue=_lib.EPI_DROPOUT_RESID, aux=x, dropout_args=(p, False, 0, 0))
    x = ops.t_layernorm_fwd_t((w["g_f"], w["b_f"]), x)
    logits = x.new_empty((rows, (cfg.vocab + 127) // 128 * 128))
    ops.gemm(x, w["w_emb"], bias=w["b_head"], out=logits, N=cfg.vocab, ldc=logits.stride(0))
    # Behind all calls: one that raises leaves no tokens counted that the cache does not hold. In place: a recorded step goes on where
    # the last replay ended.
    cache.lengths.copy_(lengths)
    cache.positions += added
    return logits.view(B, T, -1)[:, :, :cfg.vocab]


def _weights(params, dtype, p=None):
    if isinstance(params[0], GPT2Config):
        return params
    cfg = config_from_params(params, ops.DROPOUT_RATE if p is None else p)
    return cfg, Weights.from_pytree(params, cfg, dtype)


# Tokens of a batch that speculate feeds at once of its prompts. A step's logits take tokens * vocabulary elements, and with a budget its
# scores heads * tokens * capacity floats: with GPT-2 medium 0.8 and 0.5 GB, where 64 whole prompts of 1023 tokens took 6.6 and 4.3.
PROMPT_TOKENS = 8192


def _check_temperature(temperature):
    if not temperature > 0.0:
        raise ValueError(f"temperature must be positive, not {temperature} (for the likeliest token take the logits' maximum)")


def probabilities(logits: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """softmax(logits / temperature) in float32 (bf16 log-probabilities would be off by percents); temperature > 0."""
    _check_temperature(temperature)
    x = logits.float()
    return ops.t_log_softmax_fwd_t(x if temperature == 1.0 else x / temperature).exp_()


def speculate(params, draft_params, prompt: torch.Tensor, new_tokens: int, uniforms: torch.Tensor, drafts: int = 4,
              temperature: float = 1.0, prompt_lens: torch.Tensor = None, page_size: int = 16, budget: int = None, recent: int = 0):
    """Samples new_tokens tokens behind each prompt: (tokens int32 [B, new_tokens], rounds). params, draft_params: as for decode_step.

    prompt int [B, P], padded on the right; prompt_lens int32 [B], 1 to P (default P; read by the host). Every round the draft model
    (same vocabulary and positions) proposes `drafts` tokens and the target accepts a part of them and adds one of its own, so that
    tokens are distributed as if the target had drawn each. uniforms float32 [rounds, B, >= 2 * drafts + 1] in [0, 1): of round r, the
    first `drafts` draw the draft's tokens, the next drafts + 1 go to verify_drafts. new_tokens rounds are always enough, fewer where
    drafts stand; a call that runs out of them raises ValueError. The target's cache is cut down to `budget` keys per head, the last
    `recent` among them, whenever it may hold that many more (None: it grows). One host synchronisation per round (the fewest tokens of
    a sequence so far)."""
    B, P = prompt.shape
    dtype = (params[1]["w_emb"] if isinstance(params[0], GPT2Config) else params[0][0]).dtype
    target, draft = (_weights(x, dtype) for x in (params, draft_params))
    if target[0].vocab != draft[0].vocab:
        raise ValueError("target and draft model must share a vocabulary")
    if drafts < 1 or uniforms.dim() != 3 or uniforms.shape[1] != B or uniforms.shape[2] < 2 * drafts + 1:
        raise ValueError(f"uniforms must be [rounds, {B}, >= {2 * drafts + 1}] and drafts >= 1")
    if P < 1:
        raise ValueError("a prompt has at least one token")
    if prompt_lens is not None and (prompt_lens.dtype != torch.int32 or prompt_lens.shape != (B,) or
                                    bool(((prompt_lens < 1) | (prompt_lens > P)).any())):
        raise ValueError(f"prompt_lens must be an int32 tensor of shape [{B}] with values from 1 to {P}")
    longest = P + new_tokens + drafts + 1
    if longest > min(target[0].seq, draft[0].seq):
        raise ValueError(f"{longest} positions (prompt, new tokens and drafts ahead) exceed the models'")
    if budget is not None and not (0 <= recent <= budget and budget >= 1):
        raise ValueError("speculate needs 0 <= recent <= budget and budget >= 1")
    _check_temperature(temperature)
    room = longest if budget is None else min(longest, max(P, 2 * budget) + drafts + 1)
    device = prompt.device
    cache = PagedCache(target[0], B, room, page_size, dtype, device, track_weights=budget is not None)
    ahead = PagedCache(draft[0], B, longest, page_size, dtype, device)
    lens = torch.full((B,), P, device=device, dtype=torch.int32) if prompt_lens is None else prompt_lens
    rows = torch.arange(B, device=device)
    # the prompts but their last tokens, which the first round starts from
    ids = prompt.to(torch.int32)
    step = min(4096, max(1, PROMPT_TOKENS // B))
    for at in range(0, P - 1, step):
        part = ids[:, at:min(at + step, P - 1)]
        for model, c in ((target, cache), (draft, ahead)):
            decode_step(model, part, c, (lens - 1 - at).clamp_(0, part.shape[1]))
    last = ids[rows, lens.long() - 1][:, None]
    out = torch.zeros((B, new_tokens + drafts + 1), device=device, dtype=torch.int32)
    done = torch.zeros(B, device=device, dtype=torch.int64)
    least, most, rounds = 0, P, 0  # of the tokens so far; of a sequence's keys
    none = torch.empty((B, 0), device=device, dtype=torch.int32)
    columns = torch.arange(drafts + 1, device=device)
    while least < new_tokens:
        if rounds == uniforms.shape[0]:
            raise ValueError(f"uniforms has numbers for {rounds} rounds, and {least} of {new_tokens} tokens are there (each round gives at "
                             "least one)")
        u = uniforms[rounds]
        if budget is not None and most + drafts + 1 > room:
            cache.evict(budget, recent)
            most = budget
        # the draft's tokens; its last one is fed too, so that both caches end alike
        fed, guesses, dists = last, [], []
        for i in range(drafts + 1):
            logits = decode_step(draft, fed, ahead)
            if i == drafts:
                break
            dists.append(probabilities(logits, temperature))
            fed, _ = ops.verify_drafts(dists[-1], none, u[:, i:i + 1].contiguous())
            guesses.append(fed)
        guess = torch.cat(guesses, dim=1)
        probs = probabilities(decode_step(target, torch.cat([last, guess], dim=1), cache), temperature)
        tokens, accepted = ops.verify_drafts(probs, guess, u[:, drafts:2 * drafts + 1].contiguous(), draft_probs=torch.cat(dists, dim=1))
        # accepted tokens and the one behind them to their places; zeros behind those are overwritten by the next round
        place = done[:, None] + columns
        out.scatter_(1, place, torch.where((done < new_tokens)[:, None], tokens, out.gather(1, place)))
        last = tokens.gather(1, accepted[:, None].long())
        # A sequence that has its tokens stays where it is and is decoded along, one round over and over. Its last round's tokens beyond
        # those are taken back with the drafts that did not stand: the caches have room for one round behind the last token.
        more = torch.minimum(accepted + 1, new_tokens - done)
        back = drafts + 1 - more
        cache.rewind(back)
        ahead.rewind(back)
        done += more
        rounds += 1
        most += drafts + 1
        least = int(done.min())
    return out[:, :new_tokens], rounds
