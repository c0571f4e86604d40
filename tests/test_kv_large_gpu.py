"""The largest forms of attention over a paged cache and of eviction: whole prompts, as many query rows as are taken, long caches in place."""
import pytest
import torch

import serving_ref as ref
from conftest import pkg
from test_kv_cache_gpu import BF16, F32, check_out, run
from test_kv_evict_gpu import check as check_evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,H,Hk,D,T,page,lengths,room", [
    (BF16, 3, 3, 64, 1023, 16, [1023, 300, 1], 0),       # prompts of a model of 1024 positions
    (BF16, 2, 2, 64, 1023, 16, [1023, 700], 1 << 18),
    (BF16, 4, 1, 128, 1024, 32, [1024, 1500], 0),        # 4096 query rows per key head
    (BF16, 4, 1, 128, 1024, 32, [1024, 1500], 1 << 18),
    (BF16, 1, 1, 72, 513, 24, [600, 513], 0),
    (BF16, 1, 1, 256, 500, 16, [500, 40], 0),
    (F32, 3, 3, 64, 1023, 16, [1023, 77], 0),
    (F32, 4, 1, 64, 1024, 48, [1100], 0),
    (F32, 1, 1, 256, 300, 7, [300, 301], 0),
])
@pytest.mark.parametrize("with_weights", [False, True])
def test_whole_prompts(dtype, H, Hk, D, T, page, lengths, room, with_weights):
    """Prompts of different lengths, padded on the right with NaN, are written and attended to in one call."""
    kp, vp, table, lens = ref.paged(lengths, Hk, D, page, dtype)
    counts = torch.clamp(lens, max=T)
    g = torch.Generator().manual_seed(80)
    B = len(lengths)
    q, k, v = (torch.randn((B, h, T, D), generator=g).to(dtype) for h in (H, Hk, Hk))
    for b, n in enumerate(counts.tolist()):
        for x in (q, k, v):
            x[b, :, n:] = float("nan")
    k_want, v_want = kp.clone(), vp.clone()
    for b, n in enumerate(lengths):
        c = int(counts[b])
        j = torch.arange(n - c, n)
        for pool, x in ((k_want, k), (v_want, v)):
            pool[table[b].long()[j // page], :, j % page] = x[b, :, :c].transpose(0, 1)
    w = torch.rand((B, Hk, table.shape[1] * page), generator=g) if with_weights else None
    want, w_want, spread = ref.attend(q, k_want, v_want, table, lens, counts, w, p=0.1)
    out, k_got, v_got, got = run(q, kp, vp, table, lens, counts, w, wide_table=0 if with_weights else room, k=k.cuda(), v=v.cuda())
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))
    assert same(k_got, k_want) and same(v_got, v_want)
    check_out(out, want, spread, dtype)
    if with_weights:
        got = got.double().cpu()
        for b, n in enumerate(lengths):
            rel = ref.attention_error(6.0 * D**0.5, n, D) + (H // Hk * T + 2) * 2.0**-23
            assert bool(((got[b, :, :n] - w_want[b, :, :n]).abs() <= rel * w_want[b, :, :n] + 1e-30).all())


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lengths,Hk,D,page,dtype,budget,recent", [
    ([20000, 9000, 40], 2, 128, 64, BF16, 5000, 100),
    ([12000, 4097], 2, 256, 16, F32, 4000, 0),
    ([9000], 3, 80, 24, BF16, 8999, 8000),
    ([6000, 5000], 1, 7, 7, BF16, 2500, 1000),  # rows off 16-byte boundaries
    ([6000], 1, 33, 16, F32, 513, 1),
])
def test_long_caches_are_cut(lengths, Hk, D, page, dtype, budget, recent, in_place):
    check_evict(lengths, Hk, D, page, dtype, budget, recent, in_place=in_place, seed=90)
