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
