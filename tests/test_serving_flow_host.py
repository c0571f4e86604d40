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
