"""CPU checks of the 4-bit pool: the format's plain statement, and the refusals that need no device."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from oracle import kv4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("dim", [64, 128])
def test_every_byte_of_a_tile_has_one_use(dim):
    used = np.zeros(kv4.tile_bytes(dim) * 8, np.int64)
    for which in (0, 1):
        at, shift, pairs = kv4.places(dim, which)
        for bit in range(4):
            np.add.at(used, at * 8 + shift + bit, 1)
        for bit in range(32):
            np.add.at(used, pairs * 8 + bit, 1)
    assert (used == 1).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_quantised_rows_are_within_half_a_step(dim, kind):
    rng = np.random.default_rng(dim)
    x = kv4.round_to(rng.standard_normal((40, 3, dim)) * np.exp2(rng.integers(-8, 9, (40, 3, 1))), kind)
    x[0] = 0
    x[1] = 1.25  # exactly an f16 number: a constant group comes back as it was
    codes, scale, zero = kv4.quantise(x)
    got = kv4.values_of(codes, scale, zero)
    # Half a step, plus what rounding scale (15 steps of it, half an ulp 2^-11 each) and zero to f16 may clip at the
    # ends, plus f16's subnormal spacing 2^-24 for both.
    s, z = scale.astype(np.float64), zero.astype(np.float64)
    bound = 0.5 * s + 15 * 2.0 ** -11 * s + 2.0 ** -11 * np.abs(z) + 16 * 2.0 ** -24
    assert (np.abs(got - x).reshape(*scale.shape, 64) <= bound[..., None] * (1 + 1e-6)).all()
    assert (got[:2] == x[:2]).all()


def test_rows_written_are_the_rows_read():
    rng = np.random.default_rng(2)
    arena = rng.integers(0, 255, (5, 2, 2, kv4.tile_bytes(128)), dtype=np.uint8)
    before = arena.copy()
    keys, values = rng.standard_normal((2, 3, 2, 128)).astype(np.float32)
    blocks, slots = [4, 4, 1], [0, 31, 17]
    kv4.write_rows(arena, blocks, slots, keys, values)
    for r in range(3):
        for which, x in enumerate((keys, values)):
            got = kv4.read_rows(arena, [blocks[r]], 32, 128)[which][:, slots[r]]
            assert np.array_equal(got, kv4.values_of(*kv4.quantise(x[r])))
    assert (arena != before).any(-1).sum() == 3 * 2  # tiles that changed: one per row and head


def _refusal(entry, *args):
    from inferlab_b200 import _lib

    err = ctypes.create_string_buffer(256)
    assert getattr(_lib.lib(), entry)(*args, err, 256) == -1
    return err.value.decode()


def test_create_refuses_geometries_it_cannot_hold():
    handle = ctypes.c_void_p()
    ref = ctypes.byref(handle)
    name = "inferlab_cuda_pool_create_kv4"
    assert _refusal(name, 0, 0, 16, 16, 8, 64, ref) == "4-bit paged KV row dtype must be 1 (FP16) or 2 (BF16)"
    assert _refusal(name, 0, 5, 16, 16, 8, 64, ref) == "4-bit paged KV row dtype must be 1 (FP16) or 2 (BF16)"
    assert _refusal(name, 0, 2, 0, 16, 8, 64, ref) == "paged KV cache dimensions must be positive"
    assert _refusal(name, 0, 2, 1 << 31, 16, 8, 64, ref) == "paged KV num_blocks must fit a 32-bit block id"
    assert _refusal(name, 0, 2, 16, 8, 8, 64, ref) == "4-bit paged KV block_tokens must be a multiple of 16"
    assert _refusal(name, 0, 2, 16, 24, 8, 64, ref) == "4-bit paged KV block_tokens must be a multiple of 16"
    assert _refusal(name, 0, 2, 16, 16, 8, 80, ref) == "4-bit paged KV head_dim must be 64 or 128"
    assert _refusal(name, 0, 2, 16, 16, 8, 64, None) == "paged KV pool output pointer is null"
    assert handle.value is None


def test_entries_refuse_a_null_pool():
    from inferlab_b200 import _lib

    message = "paged KV pool pointer is null"
    call = _lib.InferlabCudaRotaryAppend()
    assert _refusal("inferlab_cuda_kv_append_rotary", None, ctypes.byref(call), None) == message
    assert _refusal("inferlab_cuda_kv_gather_rows", None, None, None, 1, None, 1, 1, None, None, None) == message
    assert _refusal("inferlab_cuda_kv4_decode", None, None, 0, None, 1, None, 1, 1, 1, None, None, 0, None) == message
    assert _refusal("inferlab_cuda_kv4_prefill", None, None, 0, None, 1, None, None, None, 1, 1, 1, 1, 1, None, None, 0,
                    None) == message
    assert _lib.lib().inferlab_cuda_kv4_workspace_size(None, 1, 1, 1, 1) == 0


def test_python_call_structure_matches_the_header(tmp_path):
    from inferlab_b200 import _lib

    src = tmp_path / "sizes.c"
    names = [name for name, _ in _lib.InferlabCudaRotaryAppend._fields_]
    prints = "".join(f'printf("%zu\\n", offsetof(InferlabCudaRotaryAppend, {n}));' for n in names)
    src.write_text('#include "inferlab_attention.h"\n#include <stdio.h>\nint main(void) {' + prints +
                   'printf("%zu\\n", sizeof(InferlabCudaRotaryAppend)); return 0; }')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(_lib.InferlabCudaRotaryAppend, n).offset for n in names] + \
        [ctypes.sizeof(_lib.InferlabCudaRotaryAppend)]


def test_pool_refuses_other_bit_widths():
    import inferlab_b200 as il

    with pytest.raises(il.AttentionError, match="^paged KV kv_bits must be None or 4$"):
        il.CudaKvPool(0, 2, 16, 16, 8, 64, kv_bits=8)
