"""Split decodes on a pool's own workspace, captured into graphs."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


@pytest.fixture(params=["f32", "bf16", "4 bits"])
def batch(request, torch):
    import inferlab_b200 as il

    gen = torch.Generator(device="cuda:0").manual_seed(7)
    bits = 4 if request.param == "4 bits" else None
    pool = il.CudaKvPool(0, 0 if request.param == "f32" else 2, 256, 16, 4, 128, kv_bits=bits)
    tables = torch.randint(0, 256, (24, 32), device="cuda:0", dtype=torch.int32, generator=gen)
    rows = torch.randn((256 * 16, 8, 128), device="cuda:0", generator=gen)
    every = torch.arange(256 * 16, device="cuda:0", dtype=torch.int32)
    pool.append_rotary(None, rows[:, :4], rows[:, 4:], None, every // 4096, every, torch.arange(256, device="cuda:0", dtype=torch.int32)[None])
    pool.set_decode_split(4)
    lens = torch.randint(200, 513, (24,), device="cuda:0", dtype=torch.int32, generator=gen)
    queries = torch.randn((24, 16, 128), device="cuda:0", generator=gen)
    yield pool, lambda n, **more: pool.decode(queries[:n], tables[:n], lens[:n], 512, **more)
    pool.synchronize()
    pool.close()


def test_a_graph_that_is_replayed_before_an_earlier_one(torch, batch):
    """Each graph brings its own zeroed counters: neither waits for another one's first run, nor shares its partials."""
    pool, decode = batch
    first = decode(24, workspace=pool.make_workspace(24, 16, 512))
    outs, graphs = [torch.zeros_like(first) for _ in range(2)], []
    torch.cuda.synchronize()
    for out in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            decode(24, out=out)
        graphs.append(graph)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[1], first)
    for _ in range(10):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            decode(24)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    del graphs


def test_a_graph_outlives_an_outgrown_workspace(torch, batch):
    """A larger batch after the capture replaces the stream's workspace; the graph does not write where that one was."""
    pool, decode = batch
    alone = decode(3, workspace=pool.make_workspace(3, 16, 512))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(alone)
    with torch.cuda.stream(side):
        assert torch.equal(decode(3), alone)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            decode(3, out=out)
        decode(24)
        victims = [torch.full((1 << 16,), 77, dtype=torch.uint8, device="cuda:0") for _ in range(64)]
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alone)
    assert all(bool((v == 77).all()) for v in victims)
    del graph


def test_partials_captured(torch):
    import inferlab_b200 as il

    pool = il.CudaKvPool(0, 2, 64, 16, 2, 64)
    pool.key_arena.normal_()
    pool.value_arena.normal_()
    pool.set_decode_split(2)
    q = torch.randn((3, 4, 64), device="cuda:0")
    tables = torch.randint(0, 64, (3, 16), device="cuda:0", dtype=torch.int32)
    lens = torch.tensor([256, 100, 7], device="cuda:0", dtype=torch.int32)
    want = pool.decode_partials(q, tables, lens, 256)
    packed = [torch.zeros(12 * 66, device="cuda:0") for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for to in packed:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pool.decode_partials(q, tables, lens, 256, packed=to)
        graphs.append(graph)
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    for to in packed:
        assert torch.equal(to, torch.cat([x.flatten() for x in want]))
    pool.synchronize()
    del graphs
    pool.close()
