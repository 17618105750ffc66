"""Calls that are given a stream: what they allocate is ordered on it."""
from __future__ import annotations

import types

import pytest

pytestmark = pytest.mark.gpu


def stream_of(torch, tensor):
    """The handle of the stream that the tensor's memory was allocated on."""
    at = tensor.data_ptr()
    for segment in torch.cuda.memory_snapshot():
        if segment["address"] <= at < segment["address"] + segment["total_size"]:
            return segment["stream"]
    raise AssertionError("not the caching allocator's memory")


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("handle_only", [False, True])
def test_outputs_belong_to_the_stream_given(bits, handle_only):
    """Memory of the current stream may be reused from work that it has not finished, which another stream does not wait for. A
    stream may also be any object with a cuda_stream."""
    import torch

    import inferlab_b200 as il
    from inferlab_b200.paged import lse_combine, lse_combine_packed

    assert torch.cuda.is_available(), "these tests need a CUDA device"
    pool = il.CudaKvPool(0, 2, 64, 16, 2, 64, kv_bits=bits)
    side = torch.cuda.Stream()
    given = types.SimpleNamespace(cuda_stream=side.cuda_stream) if handle_only else side
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda:0")  # noqa: E731
    qkv = torch.randn((3, 8, 64), device="cuda:0")
    table, seqs, pos = i32([1, 2], [3, 4]), i32(0, 0, 1), i32(0, 1, 0)
    tables1, lens = table, i32(2, 1)
    hidden = torch.randn((3, 64), device="cuda:0", dtype=torch.bfloat16)
    weights = torch.randn((8 * 64, 64), device="cuda:0", dtype=torch.bfloat16)
    q = torch.randn((2, 4, 64), device="cuda:0")
    side.wait_stream(torch.cuda.current_stream())
    made = [pool.append_rotary(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], None, seqs, pos, table, stream=given),
            *pool.gather(table[0], 32, stream=given), *pool.gather_rows(seqs, pos, table, stream=given),
            pool.decode(q, tables1, lens, 2, stream=given),
            pool.prefill(q, tables1, i32(1, 0), i32(1, 1), i32(0, 1), 1, stream=given),
            pool.output_project(hidden, weights, stream=given), pool.make_workspace(2, 4, 32, stream=given)]
    if bits is None:
        partials = pool.decode_partials(q, tables1, lens, 2, stream=given)
        made += [*partials, pool.project_append(hidden, weights, 4, seqs, pos, table, stream=given),
                 lse_combine(*(x[None] for x in partials), stream=given),
                 lse_combine_packed(torch.cat([x.flatten() for x in partials]), 1, 8, 64, stream=given)]
    torch.cuda.synchronize()
    assert [stream_of(torch, t) for t in made] == [side.cuda_stream] * len(made)
    # and without one they belong to the current stream
    assert stream_of(torch, pool.decode(q, tables1, lens, 2)) == torch.cuda.current_stream().cuda_stream
    with torch.cuda.stream(side):
        again = pool.decode(q, tables1, lens, 2)
    torch.cuda.synchronize()
    assert stream_of(torch, again) == side.cuda_stream
    pool.synchronize()
    pool.close()


def test_calls_leave_the_current_stream_and_device_alone():
    """Also where an allocation on the stream given fails."""
    import torch

    import inferlab_b200 as il
    from inferlab_b200.paged import _made

    pool = il.CudaKvPool(0, 2, 64, 16, 2, 64)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    q = torch.randn((1, 2, 64), device="cuda:0")
    table = torch.zeros((1, 4), dtype=torch.int32, device="cuda:0")
    lens = torch.ones(1, dtype=torch.int32, device="cuda:0")
    torch.cuda.synchronize()
    for here in (torch.cuda.default_stream(), other):
        with torch.cuda.stream(here):
            handles = [types.SimpleNamespace(cuda_stream=n) for n in (0, 1, 2, side.cuda_stream)]
            for stream in (None, side, here, torch.cuda.default_stream(), *handles):
                pool.decode(q, table, lens, 1, stream=stream)
                assert torch.cuda.current_stream() == here and torch.cuda.current_device() == 0
            with pytest.raises(RuntimeError):
                _made((-1,), torch.float32, 0, side)
            assert torch.cuda.current_stream() == here
    torch.cuda.synchronize()
    pool.synchronize()
    pool.close()


def test_a_stream_under_capture_is_known():
    import torch

    from inferlab_b200 import _lib

    lib = _lib.lib()
    side = torch.cuda.Stream()
    x = torch.zeros(4, device="cuda:0")
    assert lib.inferlab_cuda_stream_is_capturing(None) == 0
    assert lib.inferlab_cuda_stream_is_capturing(side.cuda_stream) == 0
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        assert lib.inferlab_cuda_stream_is_capturing(here.cuda_stream) == 1
        assert lib.inferlab_cuda_stream_is_capturing(side.cuda_stream) == 0
        side.wait_stream(here)
        assert lib.inferlab_cuda_stream_is_capturing(side.cuda_stream) == 1
        here.wait_stream(side)
        x += 1
    assert lib.inferlab_cuda_stream_is_capturing(side.cuda_stream) == 0
    graph.replay()
    torch.cuda.synchronize()
    assert bool((x == 1).all())
    del graph


@pytest.mark.parametrize("bits", [None, 4])
def test_a_captured_call_on_a_forked_stream(bits):
    """Inside a capture, with the stream given and without, each call has a workspace of its own."""
    import torch

    import inferlab_b200 as il

    gen = torch.Generator(device="cuda:0").manual_seed(1)
    pool = il.CudaKvPool(0, 2, 64, 16, 2, 64, kv_bits=bits)
    rows = torch.randn((1024, 4, 64), device="cuda:0", generator=gen)
    at = torch.arange(1024, device="cuda:0", dtype=torch.int32)
    pool.append_rotary(None, rows[:, :2], rows[:, 2:], None, at // 1024, at, torch.arange(64, device="cuda:0", dtype=torch.int32)[None])
    pool.set_decode_split(2)
    q = torch.randn((8, 4, 64), device="cuda:0", generator=gen)
    table = torch.randint(0, 64, (8, 16), device="cuda:0", dtype=torch.int32, generator=gen)
    lens = torch.randint(100, 257, (8,), device="cuda:0", dtype=torch.int32, generator=gen)
    want = pool.decode(q, table, lens, 256)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        assert torch.equal(pool.decode(q, table, lens, 256), want)
    torch.cuda.synchronize()
    outs = [torch.zeros_like(q) for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        pool.decode(q, table, lens, 256, out=outs[0], stream=side)
        pool.decode(q, table, lens, 256, out=outs[1])
        made = pool.decode(q, table, lens, 256, stream=side)
        here.wait_stream(side)
        outs[2].copy_(made)
    for _ in range(5):
        graph.replay()
        pool.decode(q, table, lens, 256, stream=side)
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)
    pool.synchronize()
    del graph
    pool.close()
