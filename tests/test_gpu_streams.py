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
