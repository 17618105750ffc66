"""A pool's own decode workspace over batches of very many rows."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


@pytest.mark.parametrize("dtype", [0, 1])
def test_drifting_batch_sizes_keep_one_workspace(torch, dtype):
    """Around 16384 (sequence, kv-head) pairs, where the split counters outgrow 64 KB: every batch as on a workspace of its own,
    and the pool keeps no more than its largest batch needs."""
    import inferlab_b200 as il

    gen = torch.Generator(device="cuda:0").manual_seed(6)
    heads, dim = 64, 64
    pool = il.CudaKvPool(0, dtype, 64, 16, heads, dim)
    pool.key_arena.normal_(generator=gen)
    pool.value_arena.normal_(generator=gen)
    pool.set_decode_split(1)
    sizes = [250, 256, 257, 1, 300, 310, 255, 320, 330, 2, 256, 330]
    tables = torch.randint(0, 64, (330, 3), device="cuda:0", dtype=torch.int32, generator=gen)
    lens = torch.randint(1, 49, (330,), device="cuda:0", dtype=torch.int32, generator=gen)
    queries = torch.randn((330, heads, dim), device="cuda:0", generator=gen)
    own = [pool.decode(queries[:n], tables[:n], lens[:n], 48, workspace=pool.make_workspace(n, heads, 48)) for n in sizes]
    out = torch.empty_like(queries)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(0)
    for n, alone in zip(sizes, own):
        assert torch.equal(pool.decode(queries[:n], tables[:n], lens[:n], 48, out=out[:n]), alone)
    pool.synchronize()
    # the counters' front is a power of two and at least 64 KB
    assert torch.cuda.memory_allocated(0) - before <= pool.workspace_size(330, heads, 48) + (1 << 17)
    pool.close()


def test_a_workspace_that_two_shapes_outgrow_in_turn_settles(torch):
    """Many sequences of short contexts and few of long ones: both fit after each was seen once."""
    import inferlab_b200 as il

    pool = il.CudaKvPool(0, 2, 64, 16, 32, 64)
    pool.set_decode_split(1)
    many = torch.randn((600, 32, 64), device="cuda:0")
    zeros = torch.zeros((600, 64), device="cuda:0", dtype=torch.int32)
    lens = torch.full((600,), 1024, device="cuda:0", dtype=torch.int32)
    held = []
    for _ in range(3):
        pool.decode(many, zeros, lens, 1024)
        held.append(torch.cuda.memory_allocated(0))
        pool.decode(many[:3], zeros[:3], lens[:3], 1024)
        held.append(torch.cuda.memory_allocated(0))
    pool.synchronize()
    assert len(set(held)) == 1
    pool.close()


@pytest.mark.parametrize("heads,largest", [(8, 130), (64, 330)])
@pytest.mark.parametrize("dtype", [0, 2])
def test_one_workspace_of_the_caller_serves_batches_of_all_sizes(torch, dtype, heads, largest):
    """In any order, also around 16384 (sequence, kv-head) pairs: the bits are those of a workspace made for the batch."""
    import inferlab_b200 as il

    gen = torch.Generator(device="cuda:0").manual_seed(8)
    pool = il.CudaKvPool(0, dtype, 64, 16, heads, 64)
    pool.key_arena.normal_(generator=gen)
    pool.value_arena.normal_(generator=gen)
    pool.set_decode_split(1)
    sizes = [1, 2, 5, 40, 3, largest, 1, largest * 3 // 4, largest - 1, 17, largest * 4 // 5, largest, 2, largest // 2]
    tables = torch.randint(0, 64, (largest, 6), device="cuda:0", dtype=torch.int32, generator=gen)
    lens = torch.randint(1, 97, (largest,), device="cuda:0", dtype=torch.int32, generator=gen)
    queries = torch.randn((largest, heads, 64), device="cuda:0", generator=gen)
    shared = pool.make_workspace(largest, heads, 96)
    for n in sizes:
        args = queries[:n], tables[:n], lens[:n], 96
        alone = pool.decode(*args, workspace=pool.make_workspace(n, heads, 96))
        assert torch.equal(pool.decode(*args, workspace=shared), alone)
        assert torch.equal(pool.decode(*args), alone)
        # both kinds of output leave the counters as they found them
        m, l, o = pool.decode_partials(*args, workspace=shared)
        assert torch.allclose(o / l[..., None], alone, rtol=1e-5, atol=1e-6)
    pool.synchronize()
    pool.close()
