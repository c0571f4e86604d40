"""Plain float64 forms of the serving operators, one sequence at a time on the CPU, and paged caches to try them on."""
import math

import torch


def gather(pool, table_row, n, h):
    """Rows 0 .. n-1 of key head h of a sequence, [n, D] float64."""
    page = pool.shape[2]
    j = torch.arange(n)
    return pool[table_row.long()[j // page], h, j % page].double()


def attend(q, k_pages, v_pages, table, lengths, counts, weights=None, p=0.0):
    """(out [B, H, T, D], weights_out or None, scale of a row's error [B, H, T, 1]) in float64, everything on the CPU."""
    B, H, T, D = q.shape
    Hk = k_pages.shape[1]
    G = H // Hk
    out = torch.zeros((B, H, T, D), dtype=torch.float64)
    spread = torch.zeros((B, H, T, 1), dtype=torch.float64)
    w = None if weights is None else weights.double().clone()
    for b in range(B):
        n, c = int(lengths[b]), int(counts[b])
        for h in range(Hk):
            k, v = (gather(x, table[b], n, h) for x in (k_pages, v_pages))
            if w is not None:
                w[b, h, max(n - c, 0):n] = 0.0
            for t in range(c):
                m = n - c + t + 1
                if m <= 0:
                    continue
                for g in range(G):
                    qq = q[b, h * G + g, t].double()
                    s = k[:m] @ qq / math.sqrt(D)
                    a = torch.softmax(s, dim=0)
                    out[b, h * G + g, t] = (1.0 - p) * (a @ v[:m])
                    if w is not None:
                        w[b, h, :m] += a
                    size = (k[:m].abs() @ qq.abs()).max() / math.sqrt(D)
                    spread[b, h * G + g, t] = attention_error(float(size), m, D) * float(v[:m].abs().max())
    return out, w, spread


def attention_error(size, n, D):
    """Bound of the relative error of a probability that float32 sums leave. size: largest sum of |q_d k_d| / sqrt(D).

    A score is a sum of D products, off by (D + 2) 2^-24 of that sum (scaling by log2 e and 1 / sqrt(D) adds two roundings); an
    exponential turns an absolute error of its argument into a relative one, once for the term and once for the sum, and is
    itself off by 2^-22; the sum of n terms and the weighted sum of n values by n 2^-24 each, at worst. Probabilities that are
    multiplied in two bf16 parts keep 16 bits: each part is off by half a step, 2^-9 of the value, then 2^-9 of that."""
    return 2 * (D + 2) * 2.0**-24 * size + 2 * 2.0**-22 * (1 + size) + 2 * n * 2.0**-24 + 2.0**-16


def paged(lengths, Hk, D, page, dtype, seed=0, extra_pages=3, width=None, fill=float("nan"), heads_first=True):
    """(k_pages, v_pages, table, lengths): random rows where a sequence has keys, `fill` everywhere else, pages in random order,
    table entries behind a sequence's last page out of range."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    width = max(need + [1]) if width is None else width
    pages = sum(need) + extra_pages
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lengths), width), -7, dtype=torch.int32)
    pools = []
    for _ in range(2):
        shape = (pages, Hk, page, D) if heads_first else (pages, page, Hk, D)
        x = torch.full(shape, fill, dtype=dtype)
        pools.append(x if heads_first else x.transpose(1, 2))
    at = 0
    for b, n in enumerate(lengths):
        ids = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = ids.to(torch.int32)
        j = torch.arange(n)
        for x in pools:
            x[ids[j // page], :, j % page] = torch.randn((n, Hk, D), generator=g).to(dtype)
    return pools[0], pools[1], table, torch.tensor(lengths, dtype=torch.int32)


def evict(weights, lengths, budget, recent):
    """kept positions per sequence and key head, by sorting."""
    B, Hk, _ = weights.shape
    kept = torch.full((B, Hk, budget), -1, dtype=torch.int32)
    for b in range(B):
        n = int(lengths[b])
        for h in range(Hk):
            if n <= budget:
                ids = list(range(n))
            else:
                w = weights[b, h, :n - recent].tolist()
                rank = lambda j: (1, 0.0, j) if math.isnan(w[j]) else (0, -w[j], j)
                ids = sorted(sorted(range(n - recent), key=rank)[:budget - recent]) + list(range(n - recent, n))
            kept[b, h, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return kept


def verify(target, tokens, uniforms, draft=None, counts=None):
    """(tokens [B, K + 1], accepted [B]) with float64 sums from left to right."""
    B, K1, V = target.shape
    out = torch.zeros((B, K1), dtype=torch.int32)
    accepted = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        c = K1 - 1 if counts is None else int(counts[b])
        n = 0
        while n < c:
            x = int(tokens[b, n])
            if not 0 <= x < V:
                break
            q = 1.0 if draft is None else float(draft[b, n, x])
            if not float(uniforms[b, n]) * q < float(target[b, n, x]):
                break
            n += 1
        w = target[b, n].double().clone()
        if n < c:
            if draft is not None:
                w -= draft[b, n].double()
            elif 0 <= int(tokens[b, n]) < V:
                w[int(tokens[b, n])] = 0.0
        w = torch.where(w > 0, w, 0.0)
        total = float(w.sum())
        if total > 0:
            cum = torch.cumsum(w, dim=0)
            j = int((cum > float(uniforms[b, K1 - 1]) * float(cum[-1])).to(torch.uint8).argmax())
        else:
            row = target[b, n].float()
            j = int(torch.where(row.isnan(), float("-inf"), row).argmax())
        out[b, :n] = tokens[b, :n]
        out[b, n] = j
        accepted[b] = n
    return out, accepted
