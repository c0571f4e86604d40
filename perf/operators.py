"""Timed operators of serving a trained model: attention over a paged key-value cache, eviction from it, drafted tokens.

Each case is a dict of plain values with a ``kind``:

* ``attend``  one layer's share of a decoding step: the keys and values of ``tokens`` new tokens per sequence are written into the
              pages and the new tokens attend to the sequence (``operators.attn_decode``); with ``weights`` the attention that
              every cached key received is added up for a later eviction
* ``evict``   the caches of a layer are cut down to ``budget`` keys by accumulated attention weight (``operators.kv_evict``)
* ``verify``  drafted tokens are accepted or replaced by the target's probabilities (``operators.verify_drafts``)

With ``own`` false the operators run in their plain form, elementary torch operations in 32 bits (64 for sums next to a border).
Lengths are spread between ``least`` and ``most`` the same way for every seed; contents come from the seed alone.
"""
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
DEVICE = "cuda"


def listed():
    return [
        # the toy model's decoding step: four rows of a few keys, launches and latency are all there is
        dict(name="attend tiny f32", kind="attend", dtype="f32", batch=4, heads=4, kv_heads=4, d_head=32, tokens=1, page=16,
             least=1, most=128, weights=False),
        # samples drawn during training: eight sequences of GPT-2 small, caches of every length up to the model's
        dict(name="attend small", kind="attend", dtype="bf16", batch=8, heads=12, kv_heads=12, d_head=64, tokens=1, page=16,
             least=30, most=1024, weights=False),
        # the same on the float32 master weights, rows of the reference's own length
        dict(name="attend small f32", kind="attend", dtype="f32", batch=16, heads=12, kv_heads=12, d_head=64, tokens=1, page=32,
             least=400, most=512, weights=False),
        # a full server batch of GPT-2 medium that adds up attention weights
        dict(name="attend medium 64", kind="attend", dtype="bf16", batch=64, heads=16, kv_heads=16, d_head=64, tokens=1, page=16,
             least=700, most=1024, weights=True),
        # drafted tokens: five new tokens per sequence against long caches with shared key heads, pages that are no power of two
        dict(name="attend drafts", kind="attend", dtype="bf16", batch=16, heads=16, kv_heads=4, d_head=128, tokens=5, page=48,
             least=1000, most=8000, weights=False),
        # one very long sequence: the only parallelism is over its length
        dict(name="attend long", kind="attend", dtype="bf16", batch=1, heads=32, kv_heads=8, d_head=128, tokens=1, page=64,
             least=131072, most=131072, weights=True),
        # full caches of GPT-2 small are halved
        dict(name="evict small", kind="evict", dtype="bf16", batch=8, kv_heads=12, d_head=64, page=16, least=1000, most=1024,
             budget=512, recent=128),
        # ragged float32 caches, some below the budget
        dict(name="evict ragged f32", kind="evict", dtype="f32", batch=5, kv_heads=12, d_head=64, page=24, least=100, most=512,
             budget=301, recent=33),
        # two long contexts cut to a quarter
        dict(name="evict long", kind="evict", dtype="bf16", batch=2, kv_heads=8, d_head=128, page=64, least=60000, most=65536,
             budget=16384, recent=1024),
        # one user, four drafted tokens, GPT-2's vocabulary
        dict(name="verify one", kind="verify", dtype="f32", batch=1, drafts=4, vocab=50257, dists=True),
        # a server batch with the draft model's distributions
        dict(name="verify batch", kind="verify", dtype="f32", batch=64, drafts=5, vocab=50257, dists=True),
        # drafts looked up in the text itself (no distribution), many sequences, the reference's vocabulary
        dict(name="verify lookup", kind="verify", dtype="f32", batch=256, drafts=8, vocab=35374, dists=False),
    ]


# ---- drawn cases ------------------------------------------------------------------------------------------------------
MOST_CACHE = 500e6   # bytes of keys and values of a drawn attend or evict case, and bytes that it has to move
MOST_PROBS = 320e6   # bytes of probabilities of a drawn verify case


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "evict", "verify"])
    while True:
        if kind == "verify":
            c = dict(kind=kind, dtype=rng.choice(["f32", "f32", "bf16"]), batch=_log_int(rng, 1, 256), drafts=_log_int(rng, 1, 8),
                     vocab=_log_int(rng, 1000, 50257), dists=rng.random() < 0.7)
            if _probs_bytes(c) <= MOST_PROBS:
                return c
            continue
        kv_heads = _log_int(rng, 1, 16)
        dtype = rng.choice(["bf16", "bf16", "f32"])
        most = _log_int(rng, 1, 131072 if kind == "attend" else 65536)
        c = dict(kind=kind, dtype=dtype, batch=_log_int(rng, 1, 64), kv_heads=kv_heads,
                 d_head=rng.choice([32, 64, 64, 80, 96, 128, 128]), page=rng.choice([16, 16, 32, 64, 128, 24, 7]),
                 least=_log_int(rng, 1, most), most=most)
        if kind == "attend":
            group = rng.choice([1, 1, 1, 2, 4, 8]) if dtype == "bf16" else rng.choice([1, 1, 2])
            c.update(heads=kv_heads * group, tokens=rng.choice([1, 1, 1, 2, 4, 5, 8]), weights=rng.random() < 0.4)
        else:
            c.update(budget=_log_int(rng, 1, most))
            c.update(recent=int(c["budget"] * rng.choice([0.0, 0.1, 0.25, 0.5])))
        if _cache_bytes(c) <= MOST_CACHE and work(c)["bytes"] <= MOST_CACHE:
            return c


# ---- sizes ------------------------------------------------------------------------------------------------------------
def _size(c):
    return 2 if c["dtype"] == "bf16" else 4


def _lengths(c):
    """A length for every sequence, spread over [least, most], the longest first."""
    span = c["most"] - c["least"]
    return [c["most"] - int(span * ((0.6180339887 * b) % 1.0)) for b in range(c["batch"])]


def _pages_per_sequence(c):
    return -(-c["most"] // c["page"])


def _cache_bytes(c):
    return 2 * c["batch"] * _pages_per_sequence(c) * c["page"] * c["kv_heads"] * c["d_head"] * _size(c)


def _probs_bytes(c):
    return c["batch"] * (c["drafts"] + 1 + (c["drafts"] if c["dists"] else 0)) * c["vocab"] * 4


def work(case):
    c, size = case, _size(case)
    if c["kind"] == "attend":
        keys = sum(_lengths(c))
        rows = c["batch"] * c["tokens"] * c["d_head"]
        # the visible keys and values (the new ones come from the call's own tensors), those new ones written, q and the output
        nbytes = (2 * keys * c["kv_heads"] * c["d_head"] + 2 * rows * c["kv_heads"] + 2 * rows * c["heads"]) * size
        if c["weights"]:
            nbytes += 2 * keys * c["kv_heads"] * 4
        nbytes += c["batch"] * 4 + sum(-(-n // c["page"]) for n in _lengths(c)) * 4
        return dict(bytes=nbytes, flops=4 * keys * c["heads"] * c["tokens"] * c["d_head"])
    if c["kind"] == "evict":
        lens = _lengths(c)
        kept = sum(min(n, c["budget"]) for n in lens)
        # kept keys and values read and written; weights read, the kept ones written with their positions
        nbytes = c["kv_heads"] * (4 * kept * c["d_head"] * size + 4 * sum(lens) + 8 * kept)
        return dict(bytes=nbytes, flops=sum(lens) * c["kv_heads"])
    # the row that the last token is drawn from: the target's, and the draft's where one was rejected (nearly every sequence)
    nbytes = c["batch"] * c["vocab"] * size * (2 if c["dists"] else 1) + c["batch"] * (c["drafts"] + 1) * 8
    return dict(bytes=nbytes, flops=2 * c["batch"] * c["vocab"])


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)
    st = dict(case=dict(case))
    if case["kind"] == "verify":
        return _prepare_verify(st, case, dtype, g, randn)
    B, Hk, D, page = case["batch"], case["kv_heads"], case["d_head"], case["page"]
    per = _pages_per_sequence(case)
    st["lengths"] = torch.tensor(_lengths(case), device=DEVICE, dtype=torch.int32)
    if case["kind"] == "attend":
        pages = B * per
        order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
        st["table"] = order.view(B, per)
        st["k_pages"], st["v_pages"] = (_pool(pages, Hk, page, D, dtype, g) for _ in range(2))
        H, T = case["heads"], case["tokens"]
        # one projection's output, heads ordered as the framework's: strided views of it, as a layer has them
        new = randn(B, T, H + 2 * Hk, D).to(dtype)
        st["q"] = new[:, :, :H].transpose(1, 2)
        st["k"] = new[:, :, H:H + Hk].transpose(1, 2)
        st["v"] = new[:, :, H + Hk:].transpose(1, 2)
        if case["weights"]:
            # what the keys received so far: a few heavy ones, most of them light
            st["weights"] = torch.exp(2.0 * randn(B, Hk, per * page)) * 0.01
            st["weights_out"] = torch.zeros_like(st["weights"])
        st["counts"] = torch.clamp(st["lengths"], max=T)
        return st
    # eviction copies what stays into fresh pages of the same pool
    kept_per = -(-min(case["budget"], case["most"]) // page)
    pages = B * (per + kept_per)
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    st["table"] = order[:B * per].view(B, per)
    st["dst_table"] = order[B * per:].view(B, kept_per)
    st["k_pages"], st["v_pages"] = (_pool(pages, Hk, page, D, dtype, g) for _ in range(2))
    st["weights"] = torch.exp(2.0 * randn(B, Hk, per * page)) * 0.01
    st["weights_out"] = torch.zeros((B, Hk, case["budget"]), device=DEVICE, dtype=torch.float32)
    return st


def _pool(pages, heads, page, d, dtype, g):
    pool = torch.empty((pages, heads, page, d), device=DEVICE, dtype=dtype)
    return pool.normal_(generator=g)


def _prepare_verify(st, c, dtype, g, randn):
    B, K, V = c["batch"], c["drafts"], c["vocab"]
    # a language model's next-token distributions: one token with about half of the probability, a long tail of others; the
    # draft model agrees roughly
    logits = 3.0 * randn(B, K + 1, V)
    favourite = torch.randint(0, V, (B, K + 1, 1), generator=g, device=DEVICE)
    logits.scatter_(2, favourite, torch.logsumexp(logits, dim=2, keepdim=True) + 1.5 * randn(B, K + 1, 1))
    st["target"] = torch.softmax(logits, dim=-1).to(dtype)
    if c["dists"]:
        draft = torch.softmax(logits[:, :K] + randn(B, K, V), dim=-1).to(dtype)
        st["draft"] = draft
        st["tokens"] = torch.multinomial(draft.float().view(B * K, V), 1, generator=g).view(B, K).to(torch.int32)
    else:
        st["draft"] = None
        # looked-up tokens: the likeliest one mostly, any other sometimes
        likely = logits[:, :K].argmax(dim=-1)
        other = torch.randint(0, V, (B, K), generator=g, device=DEVICE)
        hit = torch.rand((B, K), generator=g, device=DEVICE) < 0.7
        st["tokens"] = torch.where(hit, likely, other).to(torch.int32)
    st["uniforms"] = torch.rand((B, K + 1), generator=g, device=DEVICE)
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------
P_DROP = 0.1  # the models' dropout rate: evaluation multiplies the attention's output by 1 - p


def run(st):
    kind = st["case"]["kind"]
    if not own:
        return {"attend": _attend_plain, "evict": _evict_plain, "verify": _verify_plain}[kind](st)
    ops = importlib.import_module("pre-tjax_b200").operators
    if kind == "attend":
        out = ops.attn_decode(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], k=st["k"], v=st["v"],
                              counts=st["counts"], weights=st.get("weights"), weights_out=st.get("weights_out"), p=P_DROP)
        return _attend_outputs(st, out)
    if kind == "evict":
        kept, lengths = ops.kv_evict(st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["weights"],
                                     st["case"]["budget"], st["case"]["recent"], dst_table=st["dst_table"],
                                     weights_out=st["weights_out"])
        return dict(kept=kept, lengths=lengths, weights=st["weights_out"], k_pages=st["k_pages"], v_pages=st["v_pages"])
    tokens, accepted = ops.verify_drafts(st["target"], st["tokens"], st["uniforms"], draft_probs=st["draft"])
    return dict(tokens=tokens, accepted=accepted)


def _attend_outputs(st, out):
    res = dict(out=out, k_pages=st["k_pages"], v_pages=st["v_pages"])
    if "weights" in st:
        res["weights"] = st["weights_out"]
    return res


def _append(st, k_pages, v_pages):
    """The new rows into their pages; rows t >= counts belong to nobody."""
    c = st["case"]
    T, page = c["tokens"], c["page"]
    t = torch.arange(T, device=DEVICE)
    pos = (st["lengths"] - st["counts"]).long()[:, None] + t  # [B, T]
    valid = t < st["counts"][:, None]
    pos = torch.where(valid, pos, 0)
    pg = torch.gather(st["table"].long(), 1, pos // page)
    b, tt = valid.nonzero(as_tuple=True)
    for pool, new in ((k_pages, st["k"]), (v_pages, st["v"])):
        pool[pg[b, tt], :, pos[b, tt] % page] = new[b, :, tt]
    return pos, valid


def _attend_plain(st):
    c = st["case"]
    B, H, Hk, D, T, page = (c[n] for n in ("batch", "heads", "kv_heads", "d_head", "tokens", "page"))
    pos, valid = _append(st, st["k_pages"], st["v_pages"])
    table = st["table"].long()
    n = table.shape[1] * page
    k, v = (pool[table].transpose(2, 3).reshape(B, n, Hk, D).permute(0, 2, 1, 3).float()
            for pool in (st["k_pages"], st["v_pages"]))  # [B, Hk, n, D]
    q = st["q"].float().reshape(B, Hk, (H // Hk) * T, D)
    s = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(D)
    j = torch.arange(n, device=DEVICE)
    seen = (j <= pos[:, :, None]) & valid[:, :, None]  # [B, T, n]
    seen = seen[:, None, None].expand(B, Hk, H // Hk, T, n).reshape(B, Hk, -1, n)
    s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(m == float("-inf"), 0.0, m))
    total = e.sum(dim=-1, keepdim=True)
    a = e / torch.where(total == 0, 1.0, total)
    v = v.masked_fill((j >= st["lengths"][:, None])[:, None, :, None], 0.0)
    out = (torch.matmul(a, v) * (1.0 - P_DROP)).reshape(B, H, T, D).to(st["q"].dtype)
    if "weights" in st:
        old = torch.where((j < (st["lengths"] - st["counts"])[:, None])[:, None], st["weights"], 0.0)
        mine = (j < st["lengths"][:, None])[:, None]
        st["weights_out"].copy_(torch.where(mine, old + a.sum(dim=2), st["weights_out"]))
    return _attend_outputs(st, out)


def _evict_plain(st):
    c = st["case"]
    B, Hk, page, budget, recent = (c[n] for n in ("batch", "kv_heads", "page", "budget", "recent"))
    n = st["weights"].shape[2]
    lengths = st["lengths"].long()
    j = torch.arange(n, device=DEVICE)
    w = torch.where((j < lengths[:, None])[:, None], st["weights"], float("-inf"))
    w = torch.where(((j >= (lengths - recent)[:, None]) & (j < lengths[:, None]))[:, None], float("inf"), w)
    order = torch.sort(w, dim=2, descending=True, stable=True).indices[:, :, :min(budget, n)]
    new = torch.clamp(lengths, max=budget)
    order = torch.where((torch.arange(order.shape[2], device=DEVICE) < new[:, None])[:, None], order, n)
    order = torch.sort(order, dim=2).values
    kept = torch.full((B, Hk, budget), -1, device=DEVICE, dtype=torch.int32)
    kept[:, :, :order.shape[2]] = torch.where(order < n, order, -1).to(torch.int32)
    i = torch.arange(budget, device=DEVICE)
    b, i = (i < new[:, None]).nonzero(as_tuple=True)
    src = kept[b, :, i].long()  # [rows, Hk]
    table, dst = st["table"].long(), st["dst_table"].long()
    h = torch.arange(Hk, device=DEVICE)
    for pool in (st["k_pages"], st["v_pages"]):
        rows = pool[table[b[:, None], src // page], h, src % page]
        pool[dst[b, i // page][:, None], h, (i % page)[:, None]] = rows
    st["weights_out"][b[:, None], h, i[:, None]] = st["weights"][b[:, None], h, src]
    return dict(kept=kept, lengths=new.to(torch.int32), weights=st["weights_out"], k_pages=st["k_pages"],
                v_pages=st["v_pages"])


def _verify_plain(st):
    c = st["case"]
    B, K, V = c["batch"], c["drafts"], c["vocab"]
    x = st["tokens"].long()
    px = torch.gather(st["target"][:, :K], 2, x[:, :, None])[:, :, 0].double()
    qx = torch.ones_like(px) if st["draft"] is None else torch.gather(st["draft"], 2, x[:, :, None])[:, :, 0].double()
    ok = st["uniforms"][:, :K].double() * qx < px
    n = torch.cumprod(ok.long(), dim=1).sum(dim=1)  # drafts accepted
    b = torch.arange(B, device=DEVICE)
    w = st["target"][b, n].double()
    last = torch.clamp(n, max=K - 1)
    if st["draft"] is None:
        taken = torch.zeros_like(w).scatter_(1, x[b, last][:, None], float("inf"))
    else:
        taken = st["draft"][b, last].double()
    w = torch.where((n < K)[:, None], torch.clamp(w - taken, min=0.0), w)
    cum = torch.cumsum(w, dim=1)
    drawn = (cum > st["uniforms"][:, K:].double() * cum[:, -1:]).to(torch.uint8).argmax(dim=1)
    i = torch.arange(K + 1, device=DEVICE)
    tokens = torch.zeros((B, K + 1), device=DEVICE, dtype=torch.int32)
    tokens[:, :K] = st["tokens"]
    tokens = torch.where(i == n[:, None], drawn[:, None].to(torch.int32), torch.where(i < n[:, None], tokens, 0))
    return dict(tokens=tokens, accepted=n.to(torch.int32))


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    """Outputs that are computed numbers, sequence by sequence in float64; None for those that are moved or chosen."""
    if case["kind"] != "attend":
        return None
    st = prepare(case, seed)
    H, Hk, D, T, page = (case[n] for n in ("heads", "kv_heads", "d_head", "tokens", "page"))
    outs = []
    weights = st["weights_out"].double() if case["weights"] else None
    for b, n in enumerate(_lengths(case)):
        new = min(n, T)
        old = n - new
        ids = st["table"][b, :-(-n // page)].long()
        kv = []
        for pool, fresh in ((st["k_pages"], st["k"]), (st["v_pages"], st["v"])):
            rows = torch.cat([pool[ids, h].reshape(-1, D)[None] for h in range(Hk)])[:, :old]  # [Hk, old, D]
            kv.append(torch.cat([rows, fresh[b, :, :new]], dim=1).double())
        q = st["q"][b].double().view(Hk, H // Hk, T, D)
        out = torch.zeros((Hk, H // Hk, T, D), device=DEVICE, dtype=torch.float64)
        if weights is not None:
            weights[b, :, :old] = st["weights"][b, :, :old].double()
        for t in range(new):
            m = old + t + 1
            score = torch.einsum("hgd,hnd->hgn", q[:, :, t], kv[0][:, :m]) * D ** -0.5
            prob = torch.softmax(score, dim=-1)
            out[:, :, t] = torch.einsum("hgn,hnd->hgd", prob, kv[1][:, :m]) * (1.0 - P_DROP)
            if weights is not None:
                weights[b, :, :m] += prob.sum(dim=1)
        outs.append(out.view(H, T, D))
    res = dict(out=torch.stack(outs), k_pages=None, v_pages=None)
    if weights is not None:
        res["weights"] = weights
    return res
