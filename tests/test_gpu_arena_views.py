"""The arenas' torch views."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("change", ["unsqueeze", "transpose", "swap", "flat", "set", "grad"])
def test_a_view_changed_in_place_is_not_handed_out(dtype, change):
    """Whatever a holder makes of its view, the next access is the whole arena as it lies."""
    import torch

    import inferlab_b200 as il

    assert torch.cuda.is_available(), "these tests need a CUDA device"
    pool = il.CudaKvPool(0, dtype, 4, 16, 16, 16)
    for name in ("key_arena", "value_arena"):
        held = getattr(pool, name)
        held.copy_(torch.arange(held.numel(), device="cuda:0").view(held.shape) % 256)
        whole = held.clone()
        if change == "unsqueeze":
            held.unsqueeze_(0)
        elif change == "transpose":
            held.transpose_(0, 1)
        elif change == "swap":  # the shape stays
            held.transpose_(1, 2)
        elif change == "flat":
            held.resize_(held.numel())
        elif change == "set":
            held.set_(torch.zeros_like(held))
        else:
            held.requires_grad_()
        now = getattr(pool, name)
        assert now.shape == (4, 16, 16, 16) and now.is_contiguous() and not now.requires_grad
        assert torch.equal(now, whole)
        now.fill_(1.0)
        assert bool((getattr(pool, name) == 1).all())
    pool.close()
