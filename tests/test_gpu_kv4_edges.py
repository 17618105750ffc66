"""GPU tests of the 4-bit pool at the ends of its ranges: very large scores, values of very different size, many rows with bad
segments, and calls that share or outgrow workspaces. Statements in float64 are oracle/kv4.py's; tolerances count roundings as
tests/test_gpu_kv4.py does (half a unit in the last place, relative: 2^-24, 2^-11, 2^-8).
"""
import numpy as np
import pytest

from test_gpu_kv4 import KINDS, deal, filled_pool, host, i32, il, kind_of, kv4, rounding, torch, within  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- scores of any size ---------------------------------------------------------------------------------------------------
def stepped_keys(length, heads, dim, size):
    """Keys that every type and the 4-bit format hold exactly: (a_j + p_d) 2^c, a_j in eighths, p_d in sixteenths 0..15."""
    a = (np.arange(length) * 5 % 16) / 8.0
    pattern = (np.arange(dim) * 7 % 16) / 16.0
    return np.repeat(((a[:, None] + pattern) * size)[:, None], heads, 1).astype(np.float32)


@pytest.mark.parametrize("kind,q_kind,q_log2,key_log2", [
    ("bf16", "bf16", 8, 0), ("bf16", "bf16", 20, 0), ("bf16", "bf16", 23, 0), ("bf16", "bf16", 24, 0), ("bf16", "bf16", 25, 0),
    ("bf16", "bf16", 26, 0), ("bf16", "bf16", 40, -8), ("bf16", "bf16", 100, 0), ("f16", "f16", 14, 8), ("f16", "f16", 14, 10),
    ("f16", "f16", 14, 11), ("bf16", "f32", 23, 0), ("bf16", "f32", 24, 0), ("bf16", "f32", 25, 0), ("bf16", "f32", 60, 0),
    ("f16", "f32", 14, 11)])
@pytest.mark.parametrize("form,group,count,seqs,heads", [("decode", 1, 1, 2, 2), ("decode", 8, 1, 2, 1), ("prefill", 4, 5, 2, 2),
                                                         ("prefill", 4, 80, 8, 4)])
@pytest.mark.parametrize("dim,split", [(64, 0), (128, 2)])
def test_scores_of_any_size_pick_their_keys(torch, kv4, il, kind, q_kind, q_log2, key_log2, form, group, count, seqs, heads, dim, split):  # noqa: F811
    """One key's score (or that of some equal ones) leads by far more than scores are off by, so the output is that key's value (or
    their mean): however large the scores and small the values, weights must neither overflow nor vanish.

    A lead is 2^(q + c) dim / 8 / sqrt(dim) at least, the largest sum |q k| 2^(q + c) dim 3 / sqrt(dim): its fp32 error (dim + 64) 2^-24
    is below 2^-9 of the lead, and exp of what is left of it below 2^-200. So only the weights' own rounding counts, as in
    tests/test_gpu_kv4.py: f16 (2^-11) or two parts of it (2^-17), keys and values of the many-row kernel of 16-bit queries another
    2^-11, twice for a quotient of two sums."""
    rng = np.random.default_rng(q_log2 + dim)
    length = 100
    tables, blocks = deal(rng, [length], 16)
    for v_log2 in (-20, -12, 0, 11):
        values = rng.standard_normal((length, heads, dim)).astype(np.float32)
        values = kv4.round_to(np.clip(values, -4, 4) * np.float32(2.0 ** v_log2), kind)
        values[::9] = np.float32(1.5 * 2.0 ** v_log2)  # groups without a range
        keys = stepped_keys(length, heads, dim, 2.0 ** key_log2)
        arena = np.zeros((blocks, heads, 1, kv4.tile_bytes(dim)), np.uint8)
        kv4.write_rows(arena, tables[0, np.arange(length) // 16], np.arange(length) % 16, keys, values)
        pool = filled_pool(torch, il, arena, kind, 16, dim)
        pool.set_decode_split(split)
        raw = np.full((count, heads * group, dim), 2.0 ** q_log2, np.float32)
        raw[:, 1::2] *= -1  # the smallest key wins
        q = torch.from_numpy(np.concatenate([raw] * seqs)).to("cuda:0", kind_of(torch, q_kind))
        table = i32(torch, np.repeat(tables, seqs, 0))
        first = length - count
        if form == "decode":
            got = pool.decode(q, table, i32(torch, [length] * seqs), length)
        else:
            got = pool.prefill(q, table, i32(torch, [first] * seqs), i32(torch, [count] * seqs),
                               i32(torch, np.arange(seqs) * count), count, max_context_len=length)
        pool.synchronize()
        got = host(got).reshape(seqs, count, heads * group, dim)
        k, v = kv4.read_rows(arena, tables[0], length, dim)
        assert np.array_equal(k, keys.transpose(1, 0, 2))
        out, _, size = kv4.attend(raw.astype(np.float64), k, v, first)
        share = (2.0 ** -17 if q_kind == "f32" else 2.0 ** -11) + 2.0 ** -21
        if q_kind != "f32" and group * count >= 64:
            share += 2.0 ** -11
        extra = (2 * share * size)[..., None]
        for i in range(seqs):
            within(got[i], out, rounding(q_kind, np.abs(out) + extra) + extra)
        pool.close()
