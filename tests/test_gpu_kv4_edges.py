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


# ---- many rows: which kernel, and what it cannot read -----------------------------------------------------------------------
def kernel_of(torch, pool, q_kind, seqs, q_heads, count, context, split=0):  # noqa: F811
    from test_kv4_plan import plan_of

    return plan_of(pool.kv_heads, pool.head_dim, seqs, q_heads, KINDS[q_kind], count, context, split)


@pytest.mark.parametrize("split", [0, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_kind,heads,kernel", [("bf16", 2, 2), ("f32", 19, 1)])
def test_row_kernels_report_what_they_cannot_read(torch, kv4, il, q_kind, heads, kernel, dim, split):  # noqa: F811
    """Two segments of 240 rows; the second is bad in every way, the first as without it."""
    rng = np.random.default_rng(17)
    group = 8
    tables, blocks = deal(rng, [90, 90], 16)
    arena = rng.integers(0, 256, (blocks, heads, 1, kv4.tile_bytes(dim)), dtype=np.uint8)
    for which in (0, 1):  # any codes; pairs (1/8, 0)
        _, _, pair_at = kv4.places(dim, which)
        pair = np.array([0.125, 0.0], np.float16).view(np.uint8)
        arena[..., (pair_at[..., None] + np.arange(4)).ravel()] = np.tile(pair, pair_at.size)
    pool = filled_pool(torch, il, arena, "bf16", 16, dim)
    pool.set_decode_split(split)
    plan = kernel_of(torch, pool, q_kind, 2, heads * group, 30, 90, split)
    assert plan.kernel == kernel and plan.max_splits == (2 if split else 1)
    raw = kv4.bf16(rng.standard_normal((60, heads * group, dim)))
    q = torch.from_numpy(raw).to("cuda:0", kind_of(torch, q_kind))

    def run(queries=q, starts=(60, 60), counts=(30, 30), offsets=(0, 30), at=tables):
        out = torch.full(q.shape, 7.0, device="cuda:0", dtype=q.dtype)
        pool.prefill(queries, i32(torch, at), i32(torch, starts), i32(torch, counts), i32(torch, offsets), 30, max_context_len=90, out=out)
        return out

    good = run()
    pool.synchronize()
    assert bool(torch.isfinite(good).all()) and not bool((good == 7.0).any())
    for change, rows in ((dict(starts=(60, 61)), 0.0), (dict(starts=(60, -1)), 0.0), (dict(starts=(60, (1 << 31) - 1)), 0.0),
                         (dict(counts=(30, 31)), 7.0), (dict(offsets=(0, 31)), 7.0), (dict(offsets=(0, -1)), 7.0),
                         (dict(offsets=(0, (1 << 31) - 1)), 7.0), (dict(counts=(30, -1)), 7.0)):
        out = run(**change)
        with pytest.raises(il.AttentionError, match="^paged prefill segment is invalid$"):
            pool.synchronize()
        assert torch.equal(out[:30], good[:30]) and bool((out[30:] == rows).all())
    for at, bad in ((4, -1), (4, blocks), (0, 1 << 30), (5, -(1 << 31))):
        broken = tables.copy()
        broken[1, at] = bad
        out = run(at=broken)
        with pytest.raises(il.AttentionError, match="^paged KV block table contains an invalid page$"):
            pool.synchronize()
        assert torch.equal(out[:30], good[:30])
    for row, head, value in ((40, 1, float("nan")), (59, heads * group - 1, float("inf")), (30, 0, float("-inf"))):
        wrong = q.clone()
        wrong[row, head, 5] = value
        out = run(wrong)
        with pytest.raises(il.AttentionError, match="^attention input must be finite$"):
            pool.synchronize()
        rest = torch.ones((60, heads * group), dtype=torch.bool, device="cuda:0")
        rest[row, head] = False
        assert torch.equal(out[rest], good[rest])
    # rows behind and between the segments stay as they are; a segment of none has no rows
    out = run(counts=(20, 25))
    assert bool((out[20:30] == 7.0).all()) and bool((out[55:] == 7.0).all())
    assert torch.equal(run(counts=(30, 0))[:30], good[:30]) and bool((run(counts=(30, 0))[30:] == 7.0).all())
    pool.synchronize()
    assert torch.equal(run(), good)
    pool.close()


def uneven_rows(kv4, rng, length, heads, dim, spread, kind):  # noqa: F811
    """Normal keys; values whose size differs token by token and between the groups of a row, some without a range."""
    keys = rng.standard_normal((length, heads, dim)).astype(np.float32)
    values = rng.standard_normal((length, heads, dim)) * spread ** rng.uniform(-1, 1, (length, heads, 1))
    groups = spread ** rng.uniform(-1, 1, (length, heads, dim // 64, 1))
    values = (values.reshape(length, heads, dim // 64, 64) * groups).reshape(length, heads, dim).astype(np.float32)
    values[::7] = np.float32(0.25)
    values[3::11, :, :64] = 0.0
    return kv4.round_to(keys, kind), kv4.round_to(values, kind)


def attention_bound(kind, out, reach, size, dim, f16_cache=False):
    from test_gpu_kv4 import attention_bound as bound

    return bound(kind, out, reach, size, dim, f16_cache=f16_cache)


@pytest.mark.parametrize("split", [0, 8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind,q_kind,heads,kernel", [("bf16", "bf16", 2, 2), ("f16", "f16", 2, 2), ("bf16", "f32", 25, 1), ("f16", "f32", 25, 1)])
def test_row_kernels_on_values_of_different_size(torch, kv4, il, kind, q_kind, heads, kernel, dim, split):  # noqa: F811
    """Two segments of 160 rows a kv-head on 333 tokens: keys whose scores differ a lot, values of very different size."""
    rng = np.random.default_rng(dim + split)
    length, count, group = 333, 40, 4
    tables, blocks = deal(rng, [length], 16)
    checked = [0, heads // 2, heads - 1][:min(3, heads)]
    for q_size, spread in ((0.0, 1.0), (1.0, 30.0), (12.0, 1.0), (1e-4, 10.0), (5.0, 100.0)):
        keys, values = uneven_rows(kv4, rng, length, heads, dim, spread, kind)
        arena = np.zeros((blocks, heads, 1, kv4.tile_bytes(dim)), np.uint8)
        kv4.write_rows(arena, tables[0, np.arange(length) // 16], np.arange(length) % 16, keys, values)
        pool = filled_pool(torch, il, arena, kind, 16, dim)
        pool.set_decode_split(split)
        plan = kernel_of(torch, pool, q_kind, 2, heads * group, count, length, split)
        assert plan.kernel == kernel and plan.max_splits == (3 if split else 1)
        raw = kv4.round_to(rng.standard_normal((count, heads * group, dim)) * q_size, kind)
        q = torch.from_numpy(np.concatenate([raw, raw])).to("cuda:0", kind_of(torch, q_kind))
        got = pool.prefill(q, i32(torch, np.concatenate([tables, tables])), i32(torch, [length - count] * 2), i32(torch, [count] * 2),
                           i32(torch, [0, count]), count, max_context_len=length)
        pool.synchronize()
        assert torch.equal(got[:count], got[count:])
        got = host(got[:count])
        k, v = kv4.read_rows(arena, tables[0], length, dim)
        for h in checked:
            at = slice(h * group, h * group + group)
            out, reach, size = kv4.attend(raw[:, at].astype(np.float64), k[h:h + 1], v[h:h + 1], length - count)
            within(got[:, at], out, attention_bound(q_kind, out, reach, size, dim, f16_cache=kernel == 2))
        pool.close()


@pytest.mark.parametrize("split", [0, 3])
@pytest.mark.parametrize("kind,q_kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("dim,group,count", [(64, 1, 1), (128, 1, 1), (128, 4, 1), (64, 8, 1), (128, 8, 1), (128, 4, 5), (64, 3, 5), (128, 5, 7)])
def test_column_kernel_on_values_of_different_size(torch, kv4, il, kind, q_kind, dim, group, count, split):  # noqa: F811
    """One token and a few per sequence, 16-bit queries above all: their weights are one f16 number."""
    rng = np.random.default_rng(dim + group)
    length, heads = 333, 2
    tables, blocks = deal(rng, [length, 50], 16)
    for q_size, spread in ((0.0, 1.0), (1.0, 30.0), (12.0, 1.0), (1e-4, 10.0), (5.0, 100.0)):
        keys, values = uneven_rows(kv4, rng, length, heads, dim, spread, kind)
        arena = np.zeros((blocks, heads, 1, kv4.tile_bytes(dim)), np.uint8)
        lengths = np.array([length, 50])
        for i, n in enumerate(lengths):
            kv4.write_rows(arena, tables[i, np.arange(n) // 16], np.arange(n) % 16, keys[:n], values[-n:])
        pool = filled_pool(torch, il, arena, kind, 16, dim)
        pool.set_decode_split(split)
        assert kernel_of(torch, pool, q_kind, 2, heads * group, count, length, split).kernel == 0
        raw = kv4.round_to(rng.standard_normal((2 * count, heads * group, dim)) * q_size, kind)
        q = torch.from_numpy(raw).to("cuda:0", kind_of(torch, q_kind))
        if count == 1:
            got = pool.decode(q, i32(torch, tables), i32(torch, lengths), length)
        else:
            got = pool.prefill(q, i32(torch, tables), i32(torch, lengths - count), i32(torch, [count] * 2), i32(torch, [0, count]), count,
                               max_context_len=length)
        pool.synchronize()
        got = host(got)
        for i, n in enumerate(lengths):
            k, v = kv4.read_rows(arena, tables[i], int(n), dim)
            at = slice(i * count, i * count + count)
            out, reach, size = kv4.attend(raw[at].astype(np.float64), k, v, int(n) - count)
            within(got[at], out, attention_bound(q_kind, out, reach, size, dim))
        pool.close()


# ---- rows read back where no 16-byte store reaches ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits,kind", [(4, "f16"), (4, "bf16"), (None, "f32"), (None, "f16"), (None, "bf16")])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_gathered_to_any_address(torch, kv4, il, bits, kind, dim):  # noqa: F811
    """A C caller's outputs need no alignment beyond their type's; the rows are those of aligned outputs, bit for bit."""
    import ctypes

    pool = il.CudaKvPool(0, KINDS[kind], 4, 16, 3, dim, kv_bits=bits)
    gen = torch.Generator(device="cuda:0").manual_seed(3)
    rows = torch.randn((40, 6, dim), device="cuda:0", generator=gen) * torch.tensor([1.0, 1e3, 1e-3, 2e4], device="cuda:0").repeat(10)[:, None, None]
    rows[7] = 65504.0 if kind == "f16" else 5e4  # a constant group at the end of the range
    rows[8, :, ::2] = -60000.0  # two values only: the ends of the codes
    rows[8, :, 1::2] = 60000.0
    table, zero = i32(torch, [[2, 0, 3]]), i32(torch, [0] * 40)
    at = i32(torch, range(40))
    pool.append_rotary(None, rows[:, :3], rows[:, 3:], None, zero, at, table)
    if kind == "f16":  # normal numbers times 2e4 pass 65504 in some rows: those are refused, the others land
        assert bool((rows.abs() >= 65520).any())
        with pytest.raises(il.AttentionError, match="^attention input must be finite$"):
            pool.synchronize()
    pool.synchronize()
    seqs = i32(torch, [0, -1, 0, 0, 0, 0])
    where = i32(torch, [39, 0, 0, 7, 8, 16])
    keys, values = pool.gather_rows(seqs, where, table)
    width, size = 3 * dim, keys.element_size()
    flat = torch.full((2, 6 * width + 8), 5.0, device="cuda:0", dtype=keys.dtype)
    err = ctypes.create_string_buffer(256)
    for shift in (1, 3):
        flat.fill_(5.0)
        assert pool._lib.inferlab_cuda_kv_gather_rows(
            pool._handle, seqs.data_ptr(), where.data_ptr(), 6, table.data_ptr(), 1, 3, flat[0].data_ptr() + shift * size,
            flat[1].data_ptr() + shift * size, None, err, 256) == 0, err.value
        torch.cuda.synchronize()
        pool.synchronize()
        for got, want in zip(flat, (keys, values)):
            inner = got[shift:shift + 6 * width].view(6, 3, dim)
            for r in (0, 2, 3, 4, 5):
                assert torch.equal(inner[r], want[r]) and bool(torch.isfinite(want[r]).all())
            assert bool((inner[1] == 5).all()) and bool((got[:shift] == 5).all()) and bool((got[shift + 6 * width:] == 5).all())
    pool.close()


@pytest.mark.parametrize("shift", [0, 1])
def test_gathered_rows_saturate(torch, kv4, il, shift):  # noqa: F811
    """From -65504 to 65504 the scale is f16(8733.87) = 8736 and the zero f16(-65504 + 69888) = 4384: code 15 stands for
    4384 + 7 x 8736 = 65536, which f16 gives as its largest finite number; code 0 for 4384 - 8 x 8736 = -65504."""
    import ctypes

    pool = il.CudaKvPool(0, 1, 2, 16, 1, 64, kv_bits=4)
    rows = torch.zeros((1, 2, 64), device="cuda:0", dtype=torch.float16)
    rows[..., 0], rows[..., 1] = 65504.0, -65504.0
    table, zero = i32(torch, [[1]]), i32(torch, [0])
    pool.append_rotary(None, rows[:, :1], rows[:, 1:], None, zero, zero, table)
    flat = torch.zeros((2, 64 + 8), device="cuda:0", dtype=torch.float16)
    err = ctypes.create_string_buffer(256)
    assert pool._lib.inferlab_cuda_kv_gather_rows(pool._handle, zero.data_ptr(), zero.data_ptr(), 1, table.data_ptr(), 1, 1,
                                                  flat[0].data_ptr() + 2 * shift, flat[1].data_ptr() + 2 * shift, None, err, 256) == 0
    torch.cuda.synchronize()
    pool.synchronize()
    got = flat[:, shift:shift + 64].cpu().numpy()
    # the others: (0 - 4384) / 8736 rounds to -1, code 7
    assert (got[:, 0] == 65504.0).all() and (got[:, 1] == -65504.0).all() and (got[:, 2:] == np.float16(4384 - 8736)).all()
    pool.close()


@pytest.mark.parametrize("split", [0, 1, 3])
@pytest.mark.parametrize("kind,q_kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("dim,heads,group,counts", [(64, 2, 1, (1, 3, 4, 2, 0, 4)), (128, 2, 1, (4, 4, 1, 2, 3, 0)), (128, 3, 2, (2, 0, 1, 2, 2, 1)),
                                                    (64, 1, 2, (1, 2, 2, 0, 1, 2)), (128, 1, 3, (1,) * 6), (64, 2, 3, (1,) * 6), (128, 2, 4, (1,) * 6)])
def test_segments_of_at_most_four_rows(torch, kv4, il, dim, heads, group, counts, kind, q_kind, split):  # noqa: F811
    """Up to four rows a kv-head take a form of their own, whose columns stand twice; here rows that see different numbers of keys."""
    from test_gpu_kv4 import check_attention

    starts = np.array([0, 15, 13, 300, 40, 62])
    counts = np.array(counts)
    assert group * counts.max() <= 4
    check_attention(torch, kv4, il, kind, q_kind, heads, heads * group, dim, 16, starts, counts, seed=split, split=split)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_ties_follow_the_rounded_reciprocal(torch, kv4, il, kind, shift):  # noqa: F811
    """Rows of steps and half steps: the codes are those of the product with the fp32 reciprocal, as the header says, also where a
    quotient would round a tie to the other side. `shift` 1: rows that no 16-byte load reaches."""
    n = np.arange(1, 101, dtype=np.float32)
    x = kv4.round_to((np.arange(64) % 31 / 2 - 7.5).astype(np.float32) * (n * np.float32(2.0 ** -6))[:, None], kind)
    codes, scale, zero = kv4.quantise(x)
    quotient = np.clip(np.rint((x - zero.astype(np.float32)) / scale.astype(np.float32)) + 8, 0, 15)
    assert (quotient != codes).sum() > 20
    arena = np.zeros((7, 1, 1, kv4.tile_bytes(64)), np.uint8)
    pool = filled_pool(torch, il, arena, kind, 16, 64)
    flat = torch.zeros((100, 64 + shift), device="cuda:0", dtype=kind_of(torch, kind))
    rows = flat[:, shift:].unsqueeze(1)
    rows.copy_(torch.from_numpy(x)[:, None])
    pool.append_rotary(None, rows, rows, None, i32(torch, [0] * 100), i32(torch, range(100)), i32(torch, [list(range(7))]))
    pool.synchronize()
    kv4.write_rows(arena, np.arange(100) // 16, np.arange(100) % 16, x[:, None], x[:, None])
    assert np.array_equal(pool.arena.cpu().numpy(), arena)
    pool.close()
