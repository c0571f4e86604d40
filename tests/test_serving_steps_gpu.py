"""Decoding steps recorded in a CUDA graph."""
import pytest
import torch

from conftest import pkg
from test_serving_gpu import V, models, on_gpu

pytestmark = pytest.mark.gpu


def laid_out(seed, dtype):
    gpt2, ops = pkg("gpt2"), pkg("operators")
    params = on_gpu(models(seed, dtype), dtype)
    cfg = gpt2.config_from_params(params, ops.DROPOUT_RATE)
    return cfg, gpt2.Weights.from_pytree(params, cfg, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("track", [False, True])
def test_replays_of_a_recorded_step_equal_steps(dtype, track):
    """Three replays of one recorded step, other tokens each, give the logits, lengths, positions and weights of three calls."""
    sv, ops = pkg("serving"), pkg("operators")
    model = laid_out(0, dtype)
    ids = torch.randint(1, V, (2, 20), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    caches = [sv.PagedCache(model[0], 2, capacity=40, page_size=8, dtype=dtype, track_weights=track) for _ in range(2)]
    for c in caches:
        sv.decode_step(model, ids[:, :14], c, torch.tensor([14, 9], device="cuda", dtype=torch.int32))
        sv.decode_step(model, ids[:, 14:16], c)
    plain, recorded = caches
    fed = ids[:, 16:17].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        logits = sv.decode_step(model, fed, recorded)
    assert torch.equal(recorded.lengths, plain.lengths)  # recording runs nothing
    for i in range(16, 19):
        fed.copy_(ids[:, i:i + 1])
        graph.replay()
        want = sv.decode_step(model, ids[:, i:i + 1], plain)
        assert torch.equal(logits, want)
        assert torch.equal(recorded.lengths, plain.lengths) and torch.equal(recorded.positions, plain.positions)
    assert plain.lengths.tolist() == [19, 14] and plain.positions.tolist() == [19, 14]
    if track:
        assert torch.equal(recorded.weights, plain.weights)
        for c in caches:  # the buffers that were recorded stay the cache's own
            c.evict(7, 2)
        fed.copy_(ids[:, 19:20])
        graph.replay()
        assert torch.equal(logits, sv.decode_step(model, ids[:, 19:20], plain))
        assert recorded.lengths.tolist() == plain.lengths.tolist() == [8, 8]
    assert ops.last_kernel_fault() == 0


@pytest.mark.parametrize("counts,held", [([9, 2], [3, 2]), ([-4, 3], [0, 3])])
def test_counts_out_of_range_are_reported_and_counted_as_written(counts, held):
    """The kernels take the nearer bound and report it; the cache counts the rows that were written, so that the next step is right."""
    sv, ops = pkg("serving"), pkg("operators")
    model = laid_out(0, torch.float32)
    ids = torch.randint(1, V, (2, 20), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    c, good = (sv.PagedCache(model[0], 2, capacity=40, page_size=8, dtype=torch.float32) for _ in range(2))
    ops.last_kernel_fault()
    sv.decode_step(model, ids[:, :3], c, torch.tensor(counts, device="cuda", dtype=torch.int32))
    assert ops.last_kernel_fault() == 0x3202
    sv.decode_step(model, ids[:, :3], good, torch.tensor(held, device="cuda", dtype=torch.int32))
    assert c.lengths.tolist() == c.positions.tolist() == held
    assert torch.equal(sv.decode_step(model, ids[:, 3:4], c), sv.decode_step(model, ids[:, 3:4], good)) and ops.last_kernel_fault() == 0
