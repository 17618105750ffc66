"""Split decodes of different batch sizes on a pool's own workspace."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch


@pytest.mark.parametrize("dtype", [0, 2])
def test_batches_of_all_sizes_in_turn(torch, dtype):
    """A batch after a smaller one gives the bits that it gives on a workspace of its own."""
    import inferlab_b200 as il

    gen = torch.Generator(device="cuda:0").manual_seed(5)
    pool = il.CudaKvPool(0, dtype, 512, 16, 8, 64)
    pool.key_arena.normal_(generator=gen)
    pool.value_arena.normal_(generator=gen)
    pool.set_decode_split(4)
    sizes = [96, 1, 9, 33, 96, 2, 64, 96, 1, 130, 17, 130]
    tables = torch.randint(0, 512, (130, 32), device="cuda:0", dtype=torch.int32, generator=gen)
    queries = torch.randn((130, 8, 64), device="cuda:0", generator=gen)
    lens = torch.randint(300, 512, (130,), device="cuda:0", dtype=torch.int32, generator=gen)
    for n in sizes:
        args = queries[:n], tables[:n], lens[:n], 512
        alone = pool.decode(*args, workspace=pool.make_workspace(n, 8, 512))
        assert torch.equal(pool.decode(*args), alone)
    pool.synchronize()
    pool.close()
