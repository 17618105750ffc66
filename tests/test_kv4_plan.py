"""CPU checks of what attention over a 4-bit pool launches: which kernel, how the keys are split, how much workspace."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FP32, F16, BF16 = 0, 1, 2


def plan_of(kv_heads, head_dim, seqs, q_heads, dtype, count, context, split=0):
    from inferlab_b200 import _lib

    plan, err = _lib.InferlabCudaKv4Plan(), ctypes.create_string_buffer(256)
    if _lib.lib().inferlab_cuda_kv4_plan(kv_heads, head_dim, seqs, q_heads, dtype, count, context, split, ctypes.byref(plan),
                                         err, 256):
        raise ValueError(err.value.decode())
    return plan


def test_structure_matches_the_header(tmp_path):
    from inferlab_b200 import _lib

    src = tmp_path / "sizes.c"
    names = [name for name, _ in _lib.InferlabCudaKv4Plan._fields_]
    prints = "".join(f'printf("%zu\\n", offsetof(InferlabCudaKv4Plan, {n}));' for n in names)
    src.write_text('#include "inferlab_attention.h"\n#include <stdio.h>\nint main(void) {' + prints +
                   'printf("%zu\\n", sizeof(InferlabCudaKv4Plan)); return 0; }')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(_lib.InferlabCudaKv4Plan, n).offset for n in names] + [ctypes.sizeof(_lib.InferlabCudaKv4Plan)]


@pytest.mark.parametrize("context", [16, 1000, 4096, 32768, 131072, 1 << 20, 0x7FFFFF00])
@pytest.mark.parametrize("group,count", [(1, 1), (4, 1), (8, 1), (16, 1), (4, 5), (4, 15), (1, 31)])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_many_sequences_with_a_large_bound_stay_within_bounds(context, group, count, dtype):
    """The bound of one long context must not multiply the CTAs and the partials of a batch of short ones."""
    heads, dim = 8, 128
    for seqs in (1, 2, 31, 33, 64, 300, 512, 1024, 2047, 2048, 2049, 4096, 20000):
        p = plan_of(heads, dim, seqs, heads * group, dtype, count, context)
        assert p.kernel == 0
        units = seqs * heads * -(-group * count // p.tile_rows)
        assert p.ctas == units * p.max_splits <= max(32768, units)
        assert p.max_splits * p.tokens_per_split >= context
        assert p.workspace_bytes == (65536 + p.ctas * p.tile_rows * (dim + 4) * 4 if p.max_splits > 1 else 0)
        assert p.workspace_bytes <= 140 << 20
        if p.max_splits > 1:  # every unit has a counter in the region that all batches share
            assert units <= 16384


def test_the_number_of_splits_falls_step_by_step():
    """More sequences: fewer splits of one context, down to one."""
    splits = [plan_of(8, 128, n, 32, BF16, 1, 131072).max_splits for n in (128, 256, 512, 1024, 2048, 2049)]
    assert splits == [32, 16, 8, 4, 2, 1]


@pytest.mark.parametrize("dtype", [FP32, F16])
def test_row_tiles_stay_within_bounds(dtype):
    for seqs in (64, 1000, 20000):
        for context in (4096, 1 << 20):
            p = plan_of(8, 128, seqs, 32, dtype, 64, context)
            units = seqs * 8 * (4 if dtype == FP32 else 2)
            assert p.kernel == (1 if dtype == FP32 else 2) and p.ctas <= max(2048, units)


def test_which_kernel_takes_how_many_rows():
    """16-bit queries: the tensor cores from 64 rows a kv-head on; fp32 ones: row tiles from 128 rows and 148 tiles on."""
    for group, count, dtype, seqs, kernel in [(4, 15, BF16, 4, 0), (4, 16, BF16, 4, 2), (64, 1, BF16, 4, 0), (1, 64, F16, 1, 2),
                                              (4, 31, FP32, 400, 0), (4, 32, FP32, 9, 0), (4, 32, FP32, 10, 1)]:
        p = plan_of(8, 64, seqs, 8 * group, dtype, count, 500)
        assert p.kernel == kernel, (group, count, dtype, seqs)
        assert p.tile_rows == ((4 if group * count <= 4 else 8) if kernel == 0 else 64 if kernel == 1 else 128)


def test_refusals():
    for args, message in [((0, 64, 1, 8, 0, 1, 16), "multiple of kv_heads"), ((8, 64, 1, 12, 0, 1, 16), "multiple of kv_heads"),
                          ((8, 80, 1, 8, 0, 1, 16), "head_dim must be 64 or 128"), ((8, 64, 0, 8, 0, 1, 16), "bounds must be positive"),
                          ((8, 64, 1, 8, 0, 0, 16), "bounds must be positive"), ((8, 64, 1, 8, 0, 1, 0), "bounds must be positive"),
                          ((8, 64, 1, 8, 0, 1, 0x7FFFFF01), "bounds must be positive"), ((8, 64, 1, 8, 3, 1, 16), "query dtype"),
                          ((8, 64, 1, 8, 0, 1, 16, 1025), "at most 1024 blocks"),
                          ((1 << 20, 64, 1 << 20, 1 << 20, 0, 1, 16), "batch is too large"),
                          ((1, 64, 1, 1 << 16, 0, 1 << 16, 16), "batch is too large")]:
        with pytest.raises(ValueError, match=message):
            plan_of(*args)
    from inferlab_b200 import _lib

    err = ctypes.create_string_buffer(256)
    assert _lib.lib().inferlab_cuda_kv4_plan(8, 64, 1, 8, 0, 1, 16, 0, None, err, 256) == -1
    assert err.value == b"4-bit attention plan output pointer is null"
