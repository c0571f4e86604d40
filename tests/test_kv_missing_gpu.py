"""Attention over a paged cache of which a sequence's every page is out of range: nothing is there to attend."""
import pytest
import torch

import serving_ref as ref
from conftest import pkg
from test_kv_cache_gpu import BF16, F32, check_out, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,H,D,room,n", [
    (BF16, 1, 64, 0, 9), (BF16, 8, 128, 0, 40), (BF16, 12, 64, 0, 300), (BF16, 2, 64, 1 << 18, 40), (BF16, 4, 128, 1 << 18, 5000),
    (BF16, 20, 128, 1 << 18, 40), (BF16, 20, 64, 1 << 18, 3000), (BF16, 2, 256, 0, 40), (F32, 2, 64, 0, 40), (F32, 4, 128, 1 << 18, 3000)])
def test_a_sequence_without_pages_attends_nothing(dtype, H, D, room, n):
    """Zero rows, weights as they were, the report, and other sequences as ever; a row whose scores are all -inf is another thing: its
    softmax is not a number."""
    ops = pkg("operators")
    lengths = [n, 50, n]
    kp, vp, table, lens = ref.paged(lengths, 1, D, 16, dtype)
    q = torch.rand((3, H, 1, D), generator=torch.Generator().manual_seed(70)).to(dtype) + 1
    w = torch.rand((3, 1, table.shape[1] * 16), generator=torch.Generator().manual_seed(71))
    one = torch.ones(3, dtype=torch.int32)
    want, w_want, spread = ref.attend(q, kp, vp, table, lens, one, w, p=0.1)
    for j in range(n):  # the last sequence's scores
        kp[int(table[2, j // 16]), 0, j % 16, 0] = float("-inf")
    broken = table.clone()
    broken[0] = torch.where(torch.arange(table.shape[1]) % 2 == 0, -1, kp.shape[0])
    ops.last_kernel_fault()
    out, _, _, got = run(q, kp, vp, broken, lens, None, w, wide_table=room)
    assert ops.last_kernel_fault() == 0x3201
    assert bool((out[0] == 0).all())
    check_out(out[1:2], want[1:2], spread[1:2], dtype)
    assert out[2].isnan().all()
    got = got.cpu()
    assert torch.equal(got[0, 0, :n - 1], w[0, 0, :n - 1]) and float(got[0, 0, n - 1]) == 0.0  # (the new key's start at zero)
    rel = ref.attention_error(6.0 * D**0.5 * 2, 50, D) + (H + 2) * 2.0**-23
    assert bool(((got[1, 0, :50].double() - w_want[1, 0, :50]).abs() <= rel * w_want[1, 0, :50] + 1e-30).all())
    plain, _, _, _ = run(q, kp, vp, broken, lens, wide_table=room)
    assert ops.last_kernel_fault() == 0x3201
    assert bool((plain[0] == 0).all()) and plain[2].isnan().all()
    check_out(plain[1:2], want[1:2], spread[1:2], dtype)
