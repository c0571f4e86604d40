"""Eviction from a paged cache: which keys stay, in which order, and what is moved."""
import pytest
import torch

import serving_ref as ref
from conftest import pkg

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def check(lengths, Hk, D, page, dtype, budget, recent, weights=None, in_place=True, heads_first=True, seed=0):
    ops = pkg("operators")
    ops.last_kernel_fault()
    kp, vp, table, lens = ref.paged(lengths, Hk, D, page, dtype, heads_first=heads_first, seed=seed,
                                    extra_pages=3 + len(lengths) * -(-budget // page))
    B, cap = len(lengths), table.shape[1] * page
    if weights is None:
        weights = torch.rand((B, Hk, cap), generator=torch.Generator().manual_seed(seed + 1))
        for b, n in enumerate(lengths):
            weights[b, :, n:] = float("nan")
    kept_want = ref.evict(weights, lens, budget, recent)
    if in_place:
        dst = table
    else:
        used = set(table[table >= 0].tolist())
        free = [i for i in range(kp.shape[0]) if i not in used]
        w = -(-min(budget, cap) // page)
        dst = torch.tensor(free[:B * w], dtype=torch.int32).view(B, w)
    dev = lambda t: t.cuda() if t.is_contiguous() else t.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    dk, dv, dw, dt = dev(kp), dev(vp), weights.cuda(), table.cuda()
    kept, new = ops.kv_evict(dk, dv, dt, lens.cuda(), dw, budget, recent, dst_table=None if in_place else dst.cuda())
    assert ops.last_kernel_fault() == 0
    assert torch.equal(kept.cpu(), kept_want)
    assert new.tolist() == [min(n, budget) for n in lengths]
    want = [kp.clone(), vp.clone()]
    w_want = weights.clone()
    for b, n in enumerate(lengths):
        m = min(n, budget)
        i = torch.arange(m)
        for h in range(Hk):
            src = kept_want[b, h, :m].long()
            for x, y in ((kp, want[0]), (vp, want[1])):
                y[dst[b].long()[i // page], h, i % page] = x[table[b].long()[src // page], h, src % page]
            w_want[b, h, :m] = weights[b, h, src]
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))
    assert same(dk, want[0]) and same(dv, want[1])  # slots behind the kept ones, other pages: as they were
    assert same(dw, w_want)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64), (BF16, 256), (BF16, 12), (F32, 5), (BF16, 7)])
def test_eviction(dtype, D, in_place):
    check([300, 1, 0, 100, 101, 99, 777], 3, D, 16, dtype, 100, 25, in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("page", [1, 7, 48, 64])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (50, 0), (50, 50), (200, 13), (10000, 3)])
def test_budgets_and_pages(page, budget, recent, in_place):
    check([260, 51, 50, 2], 2, 64, page, BF16, budget, recent, in_place=in_place, heads_first=page != 48)


@pytest.mark.parametrize("n,budget,recent", [(5000, 1024, 128), (40000, 10007, 1000), (9001, 9000, 0), (70001, 4, 1)])
def test_long_sequences(n, budget, recent):
    check([n, 17, n // 3], 2, 64, 64, BF16, budget, recent)


@pytest.mark.parametrize("n,budget,recent", [(5000, 1024, 128), (40000, 10007, 1000), (4096, 4000, 1), (2000, 700, 700)])
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F32, 64)])
def test_long_sequences_into_other_pages(n, budget, recent, dtype, D):
    check([n, 17, n // 3], 2, D, 48, dtype, budget, recent, in_place=False)


def test_equal_weights_and_special_values():
    """Ties go to the lowest position; both zeros are equal, infinities rank at the ends, a NaN below all."""
    w = torch.zeros((1, 5, 400))
    w[0, 0, :] = 1.0
    w[0, 1, ::2] = -0.0
    w[0, 2, ::3] = float("nan")
    w[0, 2, 1::3] = float("-inf")
    w[0, 3, :] = float("nan")
    w[0, 3, 7] = float("-inf")
    w[0, 3, 300] = float("inf")
    w[0, 4] = torch.randint(-2, 3, (400,), generator=torch.Generator().manual_seed(0)) * 1e-40  # denormal
    for budget, recent in ((100, 30), (200, 0), (390, 5)):
        check([400], 5, 64, 16, BF16, budget, recent, weights=w.clone())


def test_many_heads_and_skew():
    """More caches than SMs, weights that share their leading bits."""
    g = torch.Generator().manual_seed(3)
    w = 1.0 + torch.rand((20, 12, 320), generator=g) * 2.0**-12
    check([320 - i for i in range(20)], 12, 64, 16, BF16, 128, 16, weights=w)


def test_separate_weights_out_and_replay():
    ops = pkg("operators")
    kp, vp, table, lens = ref.paged([500, 90], 2, 64, 16, BF16, extra_pages=30, fill=0.0)
    free = [i for i in range(kp.shape[0]) if i not in set(table[table >= 0].tolist())][:20]
    dst = torch.tensor(free, dtype=torch.int32).view(2, 10).cuda()
    w = torch.rand((2, 2, table.shape[1] * 16), generator=torch.Generator().manual_seed(0))
    out = torch.full((2, 2, 128), -1.0, device="cuda")
    args = (kp.cuda(), vp.cuda(), table.cuda(), lens.cuda(), w.cuda(), 128, 32)
    ops.kv_evict(*args, dst_table=dst, weights_out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, new = ops.kv_evict(*args, dst_table=dst, weights_out=out)
    args[4].copy_(1.0 - w.cuda())
    graph.replay()
    torch.cuda.synchronize()
    want = ref.evict(1.0 - w, lens, 128, 32)
    assert torch.equal(kept.cpu(), want) and new.tolist() == [128, 90]
    for b, m in ((0, 128), (1, 90)):
        for h in range(2):
            assert torch.equal(out[b, h, :m].cpu(), (1.0 - w)[b, h, want[b, h, :m].long()])
            assert bool((out[b, h, m:] == -1.0).all())


def test_missing_page_is_reported():
    ops = pkg("operators")
    kp, vp, table, lens = ref.paged([100, 100], 2, 64, 16, BF16)
    w = torch.rand((2, 2, 112), generator=torch.Generator().manual_seed(0)).cuda()
    broken = table.clone()
    broken[0, 5] = kp.shape[0]
    dk = kp.cuda()
    ops.kv_evict(dk, vp.cuda(), broken.cuda(), lens.cuda(), w.clone(), 50, 50)
    assert ops.last_kernel_fault() == 0x3201
    good = kp.cuda()
    ops.kv_evict(good, vp.cuda(), table.cuda(), lens.cuda(), w.clone(), 50, 50)
    mine = table[1].long()
    assert torch.equal(dk[mine].nan_to_num(7.0), good[mine].nan_to_num(7.0))
