"""Calls captured into CUDA graphs: a graph's scratch is its own, whatever is called, captured or freed around it."""
import pytest
import torch

import tritonformer_b200._lib as L
from test_generate import _model
from test_kvcache import Cache, _gen
from tritonformer_b200 import _host, kvcache
from tritonformer_b200.generate import Generator

pytestmark = pytest.mark.gpu


def _attention(c, q):
    return kvcache.paged_attention(q, c.k, c.v, c.tables, c.len)


def _captured(call, **how):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, **how):
        out = call()
    return graph, out


def _shared_rows(seed):
    """A row of scores that many blocks share, so that counters in the workspace are needed."""
    c = Cache([9000], 1, 64, 64, torch.float16, seed=seed)
    return c, torch.randn((1, 2, 64), device="cuda", generator=_gen(seed)).half()


def test_graphs_of_one_stream_in_any_order():
    """Both captures are on torch's capture stream, on which nothing has run; the memory they get holds ones."""
    pool = torch.cuda.graph_pool_handle()
    dirty, ones = _captured(lambda: torch.full((1 << 26,), 255, dtype=torch.uint8, device="cuda"), pool=pool)
    dirty.replay()
    torch.cuda.synchronize()
    assert (ones == 255).all()
    del ones
    c, q = _shared_rows(1)
    d, r = _shared_rows(2)
    want = _attention(c, q), _attention(d, r)
    first, x = _captured(lambda: _attention(c, q), pool=pool)
    second, y = _captured(lambda: _attention(d, r), pool=pool)
    for graph, out, expected in ((second, y, want[1]), (first, x, want[0]), (second, y, want[1])):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expected)
    assert L.device_status() == 0


def test_graphs_replayed_at_once():
    sets = [_shared_rows(s) for s in (3, 4)]
    want = [_attention(*s) for s in sets]
    graphs = [_captured(lambda s=s: _attention(*s)) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(50):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, w) for (_, out), w in zip(graphs, want)) and L.device_status() == 0


def test_a_workspace_per_capture_and_stream():
    device, side = torch.cuda.current_device(), torch.cuda.Stream()
    eager = _host.gemm_workspace(device, side.cuda_stream)
    seen = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            seen.append(_host.gemm_workspace(device, side.cuda_stream))
            assert _host.gemm_workspace(device, side.cuda_stream).data_ptr() == seen[-1].data_ptr()
            other = torch.cuda.Stream()
            other.wait_stream(side)
            seen.append(_host.gemm_workspace(device, other.cuda_stream))
            side.wait_stream(other)
        graph.replay()
        torch.cuda.synchronize()
        assert all((w[:8192] == 0).all() for w in seen[-2:])
    assert len({w.data_ptr() for w in seen + [eager]}) == 5
    assert _host.gemm_workspace(device, side.cuda_stream).data_ptr() == eager.data_ptr()


def test_many_generators_with_graphs():
    """More than the library keeps workspaces of streams; the first one's step still runs on its own."""
    model = _model(layers=1, alibi=True)
    ids = torch.randint(0, 1000, (2, 70), device="cuda", generator=_gen(5))
    want = Generator(model, 2, 128).generate(ids, None, 12)
    generators = [Generator(model, 2, 128, graph=True) for _ in range(12)]
    for g in generators:
        assert torch.equal(want, g.generate(ids, None, 12))
    ones = [torch.full((20 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(16)]  # what has been freed is in use again
    for g in generators:
        assert torch.equal(want, g.generate(ids, None, 12))
    assert all((x == 255).all() for x in ones)
    L.check_status()
