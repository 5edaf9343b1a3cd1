"""GPU checks of attention over the INT8 cache in captured graphs: each graph keeps to itself, in whatever order and at
whatever time it is replayed."""
import pytest
import torch

from tests import helpers as H
from tests.test_gpu_kv_int8 import filled

pytestmark = pytest.mark.gpu


@pytest.fixture
def inputs(monkeypatch):
    """A cache, and queries of rows whose cache several blocks share; no stream has a workspace yet."""
    from reax_engine_runtime_v3_b200 import _native
    monkeypatch.setattr(_native, "_workspaces", {})
    lens = [9000, 40, 3000]
    cache, tables = filled(4, lens, 2, 128, 64)
    queries = [torch.randn(3, 8, 128, generator=H.gen(i)).bfloat16().cuda() for i in range(2)]
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    return cache, tables.cuda(), ln, queries, [cache.attend(q, tables.cuda(), ln) for q in queries]


def capture(stream, body, pool=None):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, pool=pool):
        body()
    return graph


def test_second_graph_replayed_first_over_used_memory(inputs):
    """Two graphs captured on one stream that no call had run on; the memory that they share holds something else."""
    cache, tables, ln, queries, want = inputs
    outs = [torch.empty_like(q) for q in queries]
    stream, pool = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
    torch.cuda.synchronize()

    def scribble():
        for _ in range(2):
            torch.full((64 << 20,), 0x55, dtype=torch.uint8, device="cuda")
    first = capture(stream, scribble, pool)
    graphs = [capture(stream, lambda: cache.attend(queries[i], tables, ln, out=outs[i]), pool) for i in range(2)]
    for order in ((1, 0), (0, 1)):
        for i in order:
            first.replay()
            outs[i].zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i]), f"graph {i} of order {order}"


def test_graphs_of_one_capturing_stream_replayed_at_the_same_time(inputs):
    cache, tables, ln, queries, want = inputs
    outs = [[torch.empty_like(queries[0]) for _ in range(40)] for _ in queries]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()

    def body(i):
        for out in outs[i]:
            cache.attend(queries[i], tables, ln, out=out)
    graphs = [capture(streams[2], lambda: body(i)) for i in range(2)]
    for _ in range(20):
        for out in outs[0] + outs[1]:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, w) for some, w in zip(outs, want) for out in some)


def test_a_call_beside_a_replay(inputs):
    """A plain call on a stream that graphs were captured on, while one of them is replayed elsewhere."""
    cache, tables, ln, queries, want = inputs
    out = torch.empty_like(queries[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graph = capture(streams[0], lambda: [cache.attend(queries[0], tables, ln, out=out) for _ in range(40)])
    for _ in range(20):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[1]):
            graph.replay()
        with torch.cuda.stream(streams[0]):
            got = [cache.attend(queries[1], tables, ln) for _ in range(10)]
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and all(torch.equal(x, want[1]) for x in got)
