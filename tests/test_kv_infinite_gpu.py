"""Attention over a paged cache where attended values are infinite or NaN: the same elements as in float64 have the same values."""
import pytest
import torch

import serving_ref as ref
from conftest import pkg
from test_kv_cache_gpu import BF16, F32, check_out, run

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")

# dtype, H, Hk, D, T, room of the table: every number of rows that a kernel takes at a time, one cluster per cache or a list of stretches
FORMS = [
    (BF16, 1, 1, 64, 1, 0), (BF16, 4, 1, 128, 1, 0), (BF16, 7, 1, 64, 1, 0), (BF16, 8, 1, 128, 1, 0), (BF16, 3, 1, 80, 4, 0),
    (BF16, 12, 1, 64, 1, 0), (BF16, 16, 1, 128, 1, 0), (BF16, 30, 1, 64, 1, 0), (BF16, 24, 1, 128, 1, 0), (BF16, 10, 1, 128, 5, 0),
    (BF16, 2, 2, 64, 1, 1 << 20), (BF16, 4, 2, 128, 3, 1 << 20), (BF16, 8, 2, 64, 4, 1 << 20),
    (BF16, 20, 1, 128, 1, 1 << 20), (BF16, 8, 2, 128, 6, 1 << 20), (BF16, 20, 1, 64, 2, 1 << 20), (BF16, 9, 1, 72, 5, 1 << 20),
    (BF16, 2, 1, 256, 2, 0), (F32, 4, 2, 64, 2, 0), (F32, 2, 1, 128, 1, 1 << 20),
]


def same_values(out, want, spread, dtype):
    """Infinities and NaN where the definition has them, everything else within the bound of finite values."""
    got = out.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], want[inf])
    fine = want.isfinite()
    zero = torch.zeros((), dtype=torch.float64)
    check_out(torch.where(fine, got, zero).to(dtype), torch.where(fine, want, zero), spread, dtype)


@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{'bf16' if f[0] == BF16 else 'f32'}-{f[1]}x{f[2]}x{f[3]}-T{f[4]}-room{f[5]}")
@pytest.mark.parametrize("at", ["first", "middle", "last"])
def test_attended_infinities(form, at):
    """One key alone, keys early, in the middle and at the end of a sequence, with +inf, -inf, both and NaN in single elements: a sum
    with one of them is that, a sum with both infinities or a NaN is NaN, and the other elements do not notice."""
    dtype, H, Hk, D, T, room = form
    lengths = [T, 333, 4000]
    kp, vp, table, lens = ref.paged(lengths, Hk, D, 16, dtype)
    q = torch.randn((3, H, T, D), generator=torch.Generator().manual_seed(50)).to(dtype)
    counts = torch.full((3,), T, dtype=torch.int32)
    finite = vp.clone()
    for b, n in enumerate(lengths):
        j = {"first": 0, "middle": n // 2, "last": n - 1}[at]
        other = max(j - 1, 0) if at == "last" else min(j + 1, n - 1)
        for key, d, bad in ((j, 0, INF), (j, 3, -INF), (j, 5, INF), (other, 5, -INF), (j, 6, NAN), (other, 7, INF), (j, 7, INF)):
            if key == other == j and d == 5 and bad < 0:
                continue
            vp[int(table[b, key // 16]), :, key % 16, d] = bad
            finite[int(table[b, key // 16]), :, key % 16, d] = 0.0
    want, _, _ = ref.attend(q, kp, vp, table, lens, counts, p=0.1)
    _, _, spread = ref.attend(q, kp, finite, table, lens, counts, p=0.1)
    out, _, _, _ = run(q, kp, vp, table, lens, counts, wide_table=room)
    same_values(out, want, spread, dtype)
    again, _, _, _ = run(q, kp, vp, table, lens, counts, wide_table=room)
    assert torch.equal(out.nan_to_num(7.0), again.nan_to_num(7.0))


@pytest.mark.parametrize("H,D,room", [(4, 64, 0), (8, 128, 0), (2, 64, 1 << 20), (20, 128, 1 << 20), (20, 64, 1 << 20)])
def test_infinities_of_new_rows_and_weights(H, D, room):
    """New rows with infinite values are written, attended and do not change the weights; unaligned pools too."""
    lengths, T = [2, 700], 2
    kp, vp, table, lens = ref.paged(lengths, 1, D, 16, BF16)
    q, k, v = (torch.randn((2, h, T, D), generator=torch.Generator().manual_seed(60 + h)).to(BF16) for h in (H, 1, 1))
    v[:, :, 0, 2], v[:, :, 1, 4] = INF, -INF
    counts = torch.full((2,), T, dtype=torch.int32)
    k_want, v_want = kp.clone(), vp.clone()
    for b, n in enumerate(lengths):
        for t in range(T):
            for pool, x in ((k_want, k), (v_want, v)):
                pool[int(table[b, (n - T + t) // 16]), :, (n - T + t) % 16] = x[b, :, t]
    w = torch.zeros((2, 1, table.shape[1] * 16))
    want, w_want, _ = ref.attend(q, k_want, v_want, table, lens, counts, w, p=0.1)
    _, _, spread = ref.attend(q, k_want, v_want.nan_to_num(0.0, 0.0, 0.0), table, lens, counts, p=0.1)
    out, k_got, v_got, got = run(q, kp, vp, table, lens, counts, w, wide_table=room, k=k.cuda(), v=v.cuda())
    same_values(out, want, spread, BF16)
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))
    assert same(k_got, k_want) and same(v_got, v_want)
    got = got.double().cpu()
    for b, n in enumerate(lengths):
        rel = ref.attention_error(6.0 * D**0.5, n, D) + (H * T + 2) * 2.0**-23
        assert bool(((got[b, :, :n] - w_want[b, :, :n]).abs() <= rel * w_want[b, :, :n] + 1e-30).all())
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)]).cuda()[1:].view(t.shape)
    plain = pkg("operators").attn_decode(q.cuda(), off(k_want), off(v_want), table.cuda(), lens.cuda(), counts=counts.cuda(), p=0.1)
    same_values(plain, want, spread, BF16)
