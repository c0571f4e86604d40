"""Attention over a paged key-value cache and writing to it, against float64 on the CPU."""
import pytest
import torch

import serving_ref as ref
from conftest import pkg

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_faults():
    ops = pkg("operators")
    ops.last_kernel_fault()
    yield
    assert ops.last_kernel_fault() == 0


def check_out(out, want, spread, dtype):
    """Half a step of the stored type, and what float32 sums are off by in proportion to the largest value."""
    err = (out.double().cpu() - want).abs()
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 1.01 * spread
    assert not out.isnan().any() and bool((err <= bound).all()), float((err / bound.clamp(min=1e-30)).max())


def run(q, kp, vp, table, lengths, counts=None, weights=None, p=0.1, wide_table=0, **kw):
    """wide_table: keys that a row of the table has room for, at least; the choice of a kernel goes by the room."""
    ops = pkg("operators")
    page = kp.shape[2]
    if wide_table > table.shape[1] * page:
        table = torch.cat([table, torch.full((table.shape[0], -(-wide_table // page) - table.shape[1]), -9, dtype=torch.int32)], dim=1)
        if weights is not None:
            weights = torch.cat([weights, weights.new_zeros((*weights.shape[:2], table.shape[1] * page - weights.shape[2]))], dim=2)
    dev = lambda t: None if t is None else (t.cuda() if t.is_contiguous() else t.transpose(1, 2).contiguous().cuda().transpose(1, 2))
    kp, vp, w = dev(kp), dev(vp), dev(weights)
    out = ops.attn_decode(q.cuda(), kp, vp, table.cuda(), lengths.cuda(), counts=dev(counts), weights=w, p=p, **kw)
    return out, kp, vp, w


CASES = [
    # dtype, H, Hk, D, T, page, lengths
    (BF16, 4, 4, 64, 1, 16, [0, 1, 15, 16, 17, 63, 64, 65, 500]),
    (BF16, 2, 2, 64, 1, 7, [1, 6, 7, 8, 129, 300]),
    (BF16, 12, 12, 64, 1, 16, [1024, 3, 700]),
    (BF16, 8, 2, 128, 1, 48, [1, 100, 0, 777]),
    (BF16, 8, 1, 96, 1, 32, [257, 31]),
    (BF16, 16, 1, 64, 1, 16, [257, 31]),
    (BF16, 3, 3, 80, 2, 24, [2, 1, 200]),
    (BF16, 8, 2, 64, 5, 16, [5, 7, 3, 0, 333]),
    (BF16, 16, 2, 128, 4, 64, [4, 1000]),
    (BF16, 2, 1, 64, 40, 16, [40, 333]),
    (BF16, 8, 1, 128, 4, 16, [4, 127, 128, 129, 3, 0, 700]),   # 32 query rows per key head
    (BF16, 10, 2, 64, 7, 7, [7, 300]),
    (BF16, 6, 2, 96, 13, 48, [13, 1, 500]),
    (BF16, 8, 1, 72, 9, 24, [9, 260]),
    (BF16, 2, 2, 8, 1, 1, [1, 5, 40]),
    (BF16, 2, 2, 16, 3, 5, [3, 41]),
    (BF16, 2, 2, 256, 1, 16, [1, 99]),
    (BF16, 4, 2, 160, 3, 16, [3, 130]),
    (BF16, 2, 2, 5, 2, 16, [2, 50]),
    (BF16, 2, 1, 33, 1, 3, [70]),
    (F32, 4, 4, 64, 1, 16, [0, 1, 15, 16, 17, 65, 500]),
    (F32, 4, 2, 32, 1, 8, [9, 100, 0]),
    (F32, 8, 2, 128, 4, 48, [4, 1, 555]),
    (F32, 12, 12, 64, 1, 32, [512, 400]),
    (F32, 16, 1, 48, 2, 16, [2, 200]),
    (F32, 2, 2, 256, 2, 16, [2, 99]),
    (F32, 2, 2, 7, 1, 4, [1, 66]),
    (F32, 2, 2, 4, 1, 16, [30]),
    (F32, 3, 1, 129, 2, 16, [77]),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{'bf16' if c[0] == BF16 else 'f32'}-{c[1]}x{c[2]}x{c[3]}-T{c[4]}-page{c[5]}-{max(c[6])}")
@pytest.mark.parametrize("with_weights", [False, True])
def test_attention(case, with_weights):
    dtype, H, Hk, D, T, page, lengths = case
    kp, vp, table, lens = ref.paged(lengths, Hk, D, page, dtype)
    counts = torch.clamp(lens, max=T)
    g = torch.Generator().manual_seed(1)
    B = len(lengths)
    q = torch.randn((B, H, T, D), generator=g).to(dtype)
    cap = table.shape[1] * page
    weights = torch.rand((B, Hk, cap + 3), generator=g) if with_weights else None
    before = None if weights is None else weights.clone()
    if weights is not None:  # what new keys and slots behind the last key hold does not matter
        for b in range(B):
            weights[b, :, max(lengths[b] - int(counts[b]), 0):] = float("nan")
    many = dtype == BF16 and H // Hk * T > 16  # (room for long sequences: the tcgen05 kernel)
    want, w_want, spread = ref.attend(q, kp, vp, table, lens, counts, before, p=0.1)
    if many:
        out, _, _, _ = run(q, kp, vp, table, lens, counts, before, wide_table=1 << 20)
        check_out(out, want, spread, dtype)
    out, _, _, w = run(q, kp, vp, table, lens, counts, weights)
    check_out(out, want, spread, dtype)
    if with_weights:
        w = w.double().cpu()
        for b in range(B):
            n = lengths[b]
            size = 6.0 * D**0.5
            rel = ref.attention_error(size, n, D) + (H // Hk * T + 2) * 2.0**-23
            assert bool(((w[b, :, :n] - w_want[b, :, :n]).abs() <= rel * w_want[b, :, :n] + 1e-30).all())
            assert w[b, :, n:].isnan().all()  # left as they were


def test_long_sequence_splits_and_joins():
    """One sequence far longer than a block's share, next to short ones; bit-equal on a second run."""
    lengths = [30001, 1, 0, 4000]
    kp, vp, table, lens = ref.paged(lengths, 2, 64, 16, BF16)
    q = torch.randn((4, 4, 2, 64), generator=torch.Generator().manual_seed(2)).to(BF16) * 2
    counts = torch.clamp(lens, max=2)
    w = torch.zeros((4, 2, table.shape[1] * 16))
    out, _, _, w1 = run(q, kp, vp, table, lens, counts, w)
    want, w_want, spread = ref.attend(q, kp, vp, table, lens, counts, w, p=0.1)
    check_out(out, want, spread, BF16)
    size = 12.0 * 64**0.5
    assert bool(((w1.double().cpu() - w_want).abs() <= ref.attention_error(size, 30001, 64) * w_want + 1e-30).all())
    again, _, _, w2 = run(q, kp, vp, table, lens, counts, w)
    assert torch.equal(out, again) and torch.equal(w1, w2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_peaked_scores_and_order_of_magnitude(dtype):
    """A score that outgrows the earlier ones by far, late in the sequence, and values of very different size."""
    kp, vp, table, lens = ref.paged([900], 1, 64, 16, dtype)
    q = torch.randn((1, 1, 1, 64), generator=torch.Generator().manual_seed(3)).to(dtype)
    for at, size in ((3, 10.0), (450, 25.0), (899, 40.0)):
        page, slot = int(table[0, at // 16]), at % 16
        kp[page, 0, slot] = (q[0, 0, 0].double() / q.double().norm() * size * 8 / q.double().norm()).to(dtype)
        vp[page, 0, slot] *= 100.0
    out, _, _, _ = run(q, kp, vp, table, lens)
    want, _, spread = ref.attend(q, kp, vp, table, lens, torch.ones(1, dtype=torch.int32), p=0.1)
    check_out(out, want, spread, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), float("-inf")])
def test_rows_read_only_what_they_attend(dtype, bad):
    """Keys and values of a later drafted token, infinite or NaN, reach no earlier token's row."""
    T = 4
    kp, vp, table, lens = ref.paged([70, 9], 2, 64, 16, dtype)
    q = torch.randn((2, 4, T, 64), generator=torch.Generator().manual_seed(4)).to(dtype)
    counts = torch.full((2,), T, dtype=torch.int32)
    want, _, spread = ref.attend(q, kp, vp, table, lens, counts, p=0.0)
    for b, n in enumerate((70, 9)):
        for pool, at in ((vp, n - 1), (kp, n - 1), (vp, n - 2)):
            pool[int(table[b, at // 16]), :, at % 16, 5:9] = bad
    out, _, _, w = run(q, kp, vp, table, lens, counts, torch.zeros(2, 2, table.shape[1] * 16), p=0.0)
    check_out(out[:, :, :2], want[:, :, :2], spread[:, :, :2], dtype)
    assert not out[:, :, 2, 5:9].isfinite().any() and out[:, :, 2, 9:].isfinite().all()
    assert not out[:, :, 3].isfinite().all()


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (BF16, 128), (F32, 64), (BF16, 20), (F32, 6)])
@pytest.mark.parametrize("T", [1, 3])
def test_append_and_attend(dtype, D, T):
    """New rows of a fused projection are written and attended to; other slots keep what they hold."""
    ops = pkg("operators")
    lengths, Hk, H, page = [1, 0, 33, 64, 200], 2, 4, 16
    kp, vp, table, lens = ref.paged(lengths, Hk, D, page, dtype, heads_first=False)
    counts = torch.tensor([1, 0, T, max(T - 1, 1), T], dtype=torch.int32)
    new = torch.randn((5, T, H + 2 * Hk, D), generator=torch.Generator().manual_seed(5)).to(dtype)
    q, k, v = (x.transpose(1, 2) for x in (new[:, :, :H], new[:, :, H:H + Hk], new[:, :, H + Hk:]))
    k_want, v_want = kp.clone(), vp.clone()
    for b, n in enumerate(lengths):
        for t in range(int(counts[b])):
            at = n - int(counts[b]) + t
            for pool, x in ((k_want, k), (v_want, v)):
                pool[int(table[b, at // page]), :, at % page] = x[b, :, t]
    dnew = new.cuda()
    dq, dk, dv = (x.transpose(1, 2) for x in (dnew[:, :, :H], dnew[:, :, H:H + Hk], dnew[:, :, H + Hk:]))
    out, k_got, v_got, _ = run(dq, kp, vp, table, lens, counts, k=dk, v=dv)
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))
    assert same(k_got, k_want) and same(v_got, v_want)
    want, _, spread = ref.attend(q, k_want, v_want, table, lens, counts, p=0.1)
    check_out(out, want, spread, dtype)
    # the same rows through kv_append, and the attention alone
    kp2, vp2 = (x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (kp, vp))
    ops.kv_append(dk, dv, kp2, vp2, table.cuda(), lens.cuda(), counts.cuda())
    assert same(kp2, k_want) and same(vp2, v_want)
    again = ops.attn_decode(dq, kp2, vp2, table.cuda(), lens.cuda(), counts=counts.cuda(), p=0.1)
    assert torch.equal(out, again)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_many_rows_read_only_what_they_attend(D, bad):
    """32 query rows per key head: later tokens' keys and values that are not finite, across the border of two tiles of 128."""
    T = 16
    kp, vp, table, lens = ref.paged([262, 16, 300], 1, D, 16, BF16)
    q = torch.randn((3, 2, T, D), generator=torch.Generator().manual_seed(20)).to(BF16)
    counts = torch.full((3,), T, dtype=torch.int32)
    want, _, spread = ref.attend(q, kp, vp, table, lens, counts, p=0.0)
    for b, n in enumerate((262, 16)):
        for pool, at in ((vp, n - 1), (kp, n - 2), (vp, n - 3)):
            pool[int(table[b, at // 16]), :, at % 16, 5:9] = bad
    out, _, _, _ = run(q, kp, vp, table, lens, counts, p=0.0, wide_table=1 << 20)
    check_out(out[:2, :, :T - 3], want[:2, :, :T - 3], spread[:2, :, :T - 3], BF16)
    check_out(out[2], want[2], spread[2], BF16)
    assert not out[:2, :, T - 3, 5:9].isfinite().any() and out[:2, :, T - 3, 9:].isfinite().all()
    assert not out[:2, :, T - 1].isfinite().all()


def test_many_rows_append_split_and_replay():
    """28 rows, long and short sequences: new rows are written, the pieces of a sequence joined, twice the same bits."""
    ops = pkg("operators")
    lengths, Hk, H, T, D, page = [20000, 6, 0, 1500], 2, 8, 7, 128, 32
    kp, vp, table, lens = ref.paged(lengths, Hk, D, page, BF16)
    counts = torch.clamp(lens, max=T)
    new = torch.randn((4, T, H + 2 * Hk, D), generator=torch.Generator().manual_seed(21)).to(BF16)
    q, k, v = (x.transpose(1, 2) for x in (new[:, :, :H], new[:, :, H:H + Hk], new[:, :, H + Hk:]))
    k_want, v_want = kp.clone(), vp.clone()
    for b, n in enumerate(lengths):
        for t in range(int(counts[b])):
            at = n - int(counts[b]) + t
            for pool, x in ((k_want, k), (v_want, v)):
                pool[int(table[b, at // page]), :, at % page] = x[b, :, t]
    dnew = new.cuda()
    dq, dk, dv = (x.transpose(1, 2) for x in (dnew[:, :, :H], dnew[:, :, H:H + Hk], dnew[:, :, H + Hk:]))
    w = torch.zeros((4, Hk, table.shape[1] * page))
    out, k_got, v_got, got = run(dq, kp, vp, table, lens, counts, w, wide_table=1 << 19, k=dk, v=dv)
    got = got[:, :, :w.shape[2]]
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))
    assert same(k_got, k_want) and same(v_got, v_want)
    want, w_want, spread = ref.attend(q, k_want, v_want, table, lens, counts, w, p=0.1)
    check_out(out, want, spread, BF16)
    rel = ref.attention_error(6.0 * D**0.5, 20000, D) + (H // Hk * T + 2) * 2.0**-23
    assert bool(((got.double().cpu() - w_want).abs() <= rel * w_want + 1e-30).all())
    room = torch.cat([table, torch.full((4, (1 << 19) // page - table.shape[1]), -9, dtype=torch.int32)], dim=1).cuda()
    again = ops.attn_decode(dq, k_got, v_got, room, lens.cuda(), counts=counts.cuda(), p=0.1)
    assert torch.equal(out, again)


@pytest.mark.parametrize("wide_table", [0, 1 << 20])
@pytest.mark.parametrize("T", [1, 2, 3])
def test_new_rows_at_the_borders_of_tiles(T, wide_table):
    """New rows that start, end or cross where a step or a tile of 128 keys does, all of them written."""
    lengths, Hk, H, D, page = [128, 129, 130, 255, 256, 257, 16, 17, 144, 1], 1, 20, 128, 16
    kp, vp, table, lens = ref.paged(lengths, Hk, D, page, BF16)
    counts = torch.clamp(lens, max=T)
    q, k, v = (torch.randn((len(lengths), h, T, D), generator=torch.Generator().manual_seed(30 + h)).to(BF16) for h in (H, Hk, Hk))
    v = v + 1
    k_want, v_want = kp.clone(), vp.clone()
    for b, n in enumerate(lengths):
        for t in range(int(counts[b])):
            at = n - int(counts[b]) + t
            for pool, x in ((k_want, k), (v_want, v)):
                pool[int(table[b, at // page]), :, at % page] = x[b, :, t]
    out, k_got, v_got, _ = run(q, kp, vp, table, lens, counts, wide_table=wide_table, k=k.cuda(), v=v.cuda())
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))
    assert same(k_got, k_want) and same(v_got, v_want)
    want, _, spread = ref.attend(q, k_want, v_want, table, lens, counts, p=0.1)
    check_out(out, want, spread, BF16)


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("D", [64, 120, 128])
@pytest.mark.parametrize("H,T", [(12, 1), (4, 5), (8, 4), (5, 7)])
def test_many_rows_of_a_long_sequence(H, T, D, aligned):
    """Few caches, one of them long: the work is shared out over its length, on and off 16-byte boundaries."""
    lengths = [9000, 5, 0, 300]
    kp, vp, table, lens = ref.paged(lengths, 1, D, 16, BF16)
    counts = torch.clamp(lens, max=T)
    q = torch.randn((4, H, T, D), generator=torch.Generator().manual_seed(22)).to(BF16)
    w = torch.rand((4, 1, table.shape[1] * 16), generator=torch.Generator().manual_seed(23))
    want, w_want, spread = ref.attend(q, kp, vp, table, lens, counts, w, p=0.1)
    off = lambda t: t.cuda() if aligned else torch.cat([t.new_zeros(1), t.reshape(-1)]).cuda()[1:].view(t.shape)
    got = w.cuda()
    out = pkg("operators").attn_decode(off(q), off(kp), off(vp), table.cuda(), lens.cuda(), counts=counts.cuda(), p=0.1, weights=got)
    check_out(out, want, spread, BF16)
    got, rel = got.double().cpu(), (H * T + 2) * 2.0**-23
    for b, n in enumerate(lengths):
        bound = rel + ref.attention_error(6.0 * D**0.5, n, D)
        assert bool(((got[b, :, :n] - w_want[b, :, :n]).abs() <= bound * w_want[b, :, :n] + 1e-30).all())
    assert torch.equal(out, pkg("operators").attn_decode(off(q), off(kp), off(vp), table.cuda(), lens.cuda(), counts=counts.cuda(),
                                                         p=0.1, weights_out=torch.empty_like(w, device="cuda")))


def test_append_of_a_prompt():
    """Whole prompts of different lengths, padded on the right, go into empty caches."""
    ops = pkg("operators")
    lengths, Hk, D, page = [130, 1, 77, 0], 3, 64, 16
    kp, vp, table, lens = ref.paged(lengths, Hk, D, page, BF16, fill=0.0)
    k_want, v_want = kp.clone(), vp.clone()
    k, v = torch.full((2, 4, Hk, 130, D), float("nan"), dtype=BF16)
    for b, n in enumerate(lengths):
        for h in range(Hk):
            k[b, h, :n], v[b, h, :n] = (ref.gather(x, table[b], n, h).to(BF16) for x in (kp, vp))
    kp, vp = torch.zeros_like(kp).cuda(), torch.zeros_like(vp).cuda()
    ops.kv_append(k.cuda(), v.cuda(), kp, vp, table.cuda(), lens.cuda(), lens.cuda())
    assert torch.equal(kp.cpu(), k_want) and torch.equal(vp.cpu(), v_want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_unaligned_pools_and_queries(dtype):
    """Pools, queries and outputs that start one element behind a 16-byte boundary."""
    kp, vp, table, lens = ref.paged([50, 3], 2, 64, 16, dtype)
    q = torch.randn((2, 2, 1, 64), generator=torch.Generator().manual_seed(6)).to(dtype)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)]).cuda()[1:].view(t.shape)
    out = torch.empty(2 * 2 * 64 + 1, dtype=dtype, device="cuda")[1:].view(2, 2, 1, 64)
    pkg("operators").attn_decode(off(q), off(kp), off(vp), table.cuda(), lens.cuda(), p=0.1, out=out)
    want, _, spread = ref.attend(q, kp, vp, table, lens, torch.ones(2, dtype=torch.int32), p=0.1)
    check_out(out, want, spread, dtype)
    only_q = pkg("operators").attn_decode(off(q), kp.cuda(), vp.cuda(), table.cuda(), lens.cuda(), p=0.1)
    check_out(only_q, want, spread, dtype)


def test_sequences_share_a_prefix():
    kp, vp, table, lens = ref.paged([64, 40], 2, 64, 16, BF16)
    table[1, :2] = table[0, :2]
    q = torch.randn((2, 2, 1, 64), generator=torch.Generator().manual_seed(7)).to(BF16)
    out, _, _, _ = run(q, kp, vp, table, lens)
    want, _, spread = ref.attend(q, kp, vp, table, lens, torch.ones(2, dtype=torch.int32), p=0.1)
    check_out(out, want, spread, BF16)


def test_strided_table_and_default_rate():
    """A table that is a slice of a wider one; p defaults to the module's rate; out and T == 1 without counts."""
    ops = pkg("operators")
    kp, vp, table, lens = ref.paged([64, 40], 2, 64, 16, BF16)
    wide = torch.full((2, 9), 1 << 30, dtype=torch.int32)
    wide[:, 2:2 + table.shape[1]] = table
    q = torch.randn((2, 2, 1, 64), generator=torch.Generator().manual_seed(7)).to(BF16)
    out = ops.attn_decode(q.cuda(), kp.cuda(), vp.cuda(), wide.cuda()[:, 2:2 + table.shape[1]], lens.cuda())
    want, _, spread = ref.attend(q, kp, vp, table, lens, torch.ones(2, dtype=torch.int32), p=ops.DROPOUT_RATE)
    check_out(out, want, spread, BF16)


def test_offsets_beyond_32_bits():
    """Pages that lie more than 2^32 bytes and 2^31 elements into their pool."""
    ops = pkg("operators")
    small_k, small_v, table, lens = ref.paged([100, 37], 4, 128, 64, BF16, fill=0.0, extra_pages=0)
    n = small_k.shape[0]
    pages = (1 << 31) // (4 * 128 * 64) + n + 1
    kp, vp = (torch.empty((pages, 4, 64, 128), device="cuda", dtype=BF16) for _ in range(2))
    kp[-n:], vp[-n:] = small_k.cuda(), small_v.cuda()
    q, k, v = (torch.randn((2, 4, 1, 128), generator=torch.Generator().manual_seed(s)).to(BF16) for s in (8, 9, 10))
    out = ops.attn_decode(q.cuda(), kp, vp, (table + (pages - n)).cuda(), lens.cuda(), k=k.cuda(), v=v.cuda(), p=0.1)
    for b, at in enumerate((99, 36)):
        small_k[int(table[b, at // 64]), :, at % 64], small_v[int(table[b, at // 64]), :, at % 64] = k[b, :, 0], v[b, :, 0]
    assert torch.equal(kp[-n:].cpu(), small_k) and torch.equal(vp[-n:].cpu(), small_v)
    want, _, spread = ref.attend(q, small_k, small_v, table, lens, torch.ones(2, dtype=torch.int32), p=0.1)
    check_out(out, want, spread, BF16)


def test_many_sequences():
    """More sequences than a block has threads, most of them empty or of one key."""
    lengths = [(i * 7919) % 3 for i in range(1500)] + [300]
    kp, vp, table, lens = ref.paged(lengths, 1, 32, 16, BF16)
    q = torch.randn((1501, 1, 1, 32), generator=torch.Generator().manual_seed(11)).to(BF16)
    counts = torch.clamp(lens, max=1)
    out, _, _, _ = run(q, kp, vp, table, lens, counts)
    want, _, spread = ref.attend(q, kp, vp, table, lens, counts, p=0.1)
    check_out(out, want, spread, BF16)


def test_captured_and_replayed_on_two_streams():
    """Two recorded calls of one shape replayed side by side, with lengths that changed after the recording."""
    ops = pkg("operators")
    jobs = []
    for seed in (0, 1):
        kp, vp, table, lens = ref.paged([3000, 17], 2, 64, 16, BF16, seed=seed, width=200)
        q = torch.randn((2, 2, 1, 64), generator=torch.Generator().manual_seed(seed)).to(BF16)
        dev = [x.cuda() for x in (q, kp, vp, torch.where(table < 0, 0, table), torch.tensor([5, 2], dtype=torch.int32))]
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            ops.attn_decode(*dev, p=0.1)
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = ops.attn_decode(*dev, p=0.1)
        dev[4].copy_(lens)
        jobs.append((graph, st, out, dev, ref.attend(q, kp, vp, table, lens, torch.ones(2, dtype=torch.int32), p=0.1)))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, st, _, _, _ in jobs:
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, _, (want, _, spread) in jobs:
        check_out(out, want, spread, BF16)


def test_pages_and_lengths_out_of_range_are_reported():
    """The kernels skip what the tables name outside the pool, and say so; other sequences are not touched by it."""
    ops = pkg("operators")
    for dtype in (BF16, F32):
        kp, vp, table, lens = ref.paged([40, 40], 2, 64, 16, dtype)
        q, k, v = (torch.randn((2, 2, 1, 64), generator=torch.Generator().manual_seed(s)).to(dtype) for s in (12, 13, 14))
        want, _, spread = ref.attend(q, kp, vp, table, lens, torch.ones(2, dtype=torch.int32), p=0.1)
        for page in (-1, kp.shape[0], -(1 << 31), (1 << 31) - 1):
            broken = table.clone()
            broken[0, 1] = page
            out, _, _, _ = run(q, kp, vp, broken, lens)
            assert ops.last_kernel_fault() == 0x3201
            check_out(out[1:], want[1:], spread[1:], dtype)
            # the keys of the missing page count as absent
            keep = torch.cat([torch.arange(16), torch.arange(32, 40)])
            for h in range(2):
                kk, vv = (ref.gather(x, table[0], 40, h)[keep] for x in (kp, vp))
                a = torch.softmax(kk @ q[0, h, 0].double() / 8.0, dim=0)
                bound = torch.finfo(dtype).eps / 2 * (a @ vv).abs() + 1.01 * spread[0, h, 0]
                assert bool(((out[0, h, 0].double().cpu() - 0.9 * (a @ vv)).abs() <= bound).all())
        broken = table.clone()
        broken[0, 2] = -1  # the page of the new row: nothing is written
        dk, dv = kp.cuda(), vp.cuda()
        ops.kv_append(k.cuda(), v.cuda(), dk, dv, broken.cuda(), lens.cuda())
        assert ops.last_kernel_fault() == 0x3201
        at = int(table[1, 2])
        kp[at, :, 7], vp[at, :, 7] = k[1, :, 0], v[1, :, 0]
        assert torch.equal(dk.cpu().nan_to_num(7.0), kp.nan_to_num(7.0))
        for n in (-1, 49, 1 << 30):
            run(q, kp, vp, table, torch.tensor([n, 40], dtype=torch.int32))
            assert ops.last_kernel_fault() in (0x3202, 0x3201)
        run(q, kp, vp, table, lens, torch.tensor([2, 1], dtype=torch.int32))
        assert ops.last_kernel_fault() == 0x3202


@pytest.mark.parametrize("wide_table", [0, 1 << 20])
@pytest.mark.parametrize("D", [64, 128])
def test_missing_pages_and_many_rows(D, wide_table):
    """20 query rows per key head: pages and lengths out of range are skipped and reported, nothing is written for them."""
    ops = pkg("operators")
    kp, vp, table, lens = ref.paged([300, 40], 1, D, 16, BF16)
    q, k, v = (torch.randn((2, h, 1, D), generator=torch.Generator().manual_seed(40 + i)).to(BF16) for i, h in enumerate((20, 1, 1)))
    one = torch.ones(2, dtype=torch.int32)
    want, _, spread = ref.attend(q, kp, vp, table, lens, one, p=0.1)
    ops.last_kernel_fault()
    for page in (-1, kp.shape[0], -(1 << 31), (1 << 31) - 1):
        broken = table.clone()
        broken[0, 9] = page
        out, _, _, _ = run(q, kp, vp, broken, lens, wide_table=wide_table)
        assert ops.last_kernel_fault() == 0x3201
        check_out(out[1:], want[1:], spread[1:], BF16)
        keep = torch.cat([torch.arange(144), torch.arange(160, 300)])  # the keys of the missing page count as absent
        kk, vv = (ref.gather(x, table[0], 300, 0)[keep] for x in (kp, vp))
        a = torch.softmax(q[0, :, 0].double() @ kk.T / D**0.5, dim=1) @ vv
        bound = torch.finfo(BF16).eps / 2 * a.abs() + 1.01 * spread[0, :, 0]
        assert bool(((out[0, :, 0].double().cpu() - 0.9 * a).abs() <= bound).all())
    broken = table.clone()
    broken[0, 18] = -1  # the page of the new row
    _, k_got, v_got, _ = run(q, kp, vp, broken, lens, wide_table=wide_table, k=k.cuda(), v=v.cuda())
    assert ops.last_kernel_fault() == 0x3201
    at = int(table[1, 2])
    kp[at, :, 7], vp[at, :, 7] = k[1, :, 0], v[1, :, 0]
    same = lambda x, y: torch.equal(x.cpu().nan_to_num(7.0), y.nan_to_num(7.0))
    assert same(k_got, kp) and same(v_got, vp)
    run(q, kp, vp, table, torch.tensor([-1, 40], dtype=torch.int32), wide_table=wide_table)
    assert ops.last_kernel_fault() == 0x3202
    run(q, kp, vp, table, lens, torch.tensor([2, 1], dtype=torch.int32), wide_table=wide_table)
    assert ops.last_kernel_fault() == 0x3202
