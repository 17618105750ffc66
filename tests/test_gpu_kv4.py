"""GPU tests of the rotary append, of 4-bit pools and of attention over them, against the float64 statements in
oracle/kv4.py.

Tolerances count roundings. eps below is half a unit in the last place of the type, relative (2^-24, 2^-11, 2^-8; f16 also
2^-25 absolute below its normal range).
- rotation: two products and a sum in fp32, each 2^-24 relative to at most |a| + |b|: 2^-23 (|a| + |b|), then the type's
  rounding.
- attention: the result's rounding, and on the weights p what scores, exponentials and splits of p cost: at most dim + 64
  fp32 roundings of the sum |q k| (2^-24 each), 2^-21 for its exponential, and p's own rounding: one f16 number for 16-bit
  queries (2^-11), two f16 parts for fp32 queries (2^-17 with room for the second part's subnormals). A weight off by a
  share w moves the output by at most 2 w max|v|.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

KINDS = {"f32": 0, "f16": 1, "bf16": 2}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    import torch

    assert torch.cuda.is_available(), "these tests need a CUDA device"
    return torch


@pytest.fixture(scope="module")
def kv4():
    from oracle import kv4

    return kv4


@pytest.fixture(scope="module")
def il():
    import inferlab_b200

    return inferlab_b200


def kind_of(torch, kind):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


def i32(torch, a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda:0")


def host(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def within(got, ref, bound):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert np.isfinite(got).all()
    over = np.abs(got - ref) - bound
    assert (over <= 0).all(), f"{(over > 0).sum()} of {over.size} over the bound, by up to {over.max():.3e}"


def rounding(kind, ref):
    return EPS[kind] * np.abs(ref) + (2.0 ** -25 if kind == "f16" else 0.0)


def attention_bound(kind, out, reach, size, dim, f16_cache=False):
    """Share of the largest value by which weights may be off (relative errors of scores, weights, sums), twice for a
    quotient of two sums. `f16_cache`: keys and values are widened to f16 of an exact power of two, which is off by 2^-11
    of each: a score sum q k by 2^-11 of sum |q k| (and with it exp of it), a value by 2^-11 of it (below 2^-14 of the
    row's largest by 2^-40 of that, covered by the last term)."""
    share = (dim + 64) * 2.0 ** -24 * reach + (2.0 ** -17 if kind == "f32" else 2.0 ** -11) + 2.0 ** -21
    if f16_cache:
        share = share + 2.0 ** -11 * reach + 2.0 ** -11
    extra = (2 * share * size)[..., None]
    return rounding(kind, np.abs(out) + extra) + extra


def angles_of(positions, rotary):
    turn = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(rotary // 2) * 2 / max(1, rotary))
    return np.concatenate([np.cos(turn), np.sin(turn)], 1).astype(np.float32)


def random_arena(kv4, rng, blocks, heads, block, dim, kind="bf16"):
    """A packed arena whose every slot holds quantised normal rows."""
    tiles = blocks * heads * block // 16
    arena = np.zeros((tiles, kv4.tile_bytes(dim)), np.uint8)
    for which in (0, 1):
        at, _, pair_at = kv4.places(dim, which)
        x = kv4.round_to(rng.standard_normal((tiles, 16, dim)).astype(np.float32), kind)
        codes, scale, zero = kv4.quantise(x)
        arena[:, at[:, 0::2]] = codes[..., 0::2] | (codes[..., 1::2] << 4)
        pairs = np.stack([scale, zero], -1).view(np.uint8).reshape(tiles, 16, dim // 64, 4)
        arena[:, pair_at[..., None] + np.arange(4)] = pairs
    return arena.reshape(blocks, heads, block // 16, -1)


def filled_pool(torch, il, arena, kind, block, dim):
    pool = il.CudaKvPool(0, KINDS[kind], arena.shape[0], block, arena.shape[1], dim, kv_bits=4)
    pool.arena.copy_(torch.from_numpy(arena))
    return pool


def deal(rng, lengths, block, spare=3):
    """Tables over a shuffled pool; entries behind a sequence's last block are no block at all."""
    need = [(int(n) + block - 1) // block for n in lengths]
    blocks = sum(need) + spare
    order = rng.permutation(blocks)
    tables = np.full((len(need), max(1, max(need)) + 1), -7, np.int64)
    first = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[first:first + n]
        first += n
    return tables, blocks


# ---- append -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,rows_kind,out_kind", [("f32", "f32", "f32"), ("f16", "f16", "f16"), ("f16", "f32", "f16"),
                                                     ("bf16", "bf16", "f32"), ("bf16", "f32", "f32")])
@pytest.mark.parametrize("heads,q_heads,dim,rotary,interleaved,block", [
    (8, 32, 128, 128, False, 16), (2, 2, 64, 32, True, 16), (3, 9, 80, 80, False, 5), (1, 4, 6, 2, False, 16),
    (2, 4, 128, 64, False, 32), (4, 4, 64, 64, True, 1), (1, 0, 33, 32, True, 16), (2, 2, 128, 0, False, 16),
    (2, 6, 96, 48, False, 16)])
def test_append_rotary_wide_pools(torch, il, kv4, kind, rows_kind, out_kind, heads, q_heads, dim, rotary, interleaved, block):
    rng = np.random.default_rng(dim + rotary + heads)
    rows = 37
    lengths = [20, 1, 33]
    tables, blocks = deal(rng, lengths, block)
    seqs = np.concatenate([np.repeat(np.arange(3), [12, 1, 20]), [-1] * 4])
    positions = np.concatenate([np.arange(8, 20), [0], np.arange(13, 33), [0, 5, 999, -3]])
    mixed = kv4.round_to(rng.standard_normal((rows, q_heads + 2 * heads, dim)), rows_kind)
    qkv = torch.from_numpy(mixed).to("cuda:0", kind_of(torch, rows_kind))
    pool = il.CudaKvPool(0, KINDS[kind], blocks, block, heads, dim)
    pool.key_arena.fill_(3.0)
    pool.value_arena.fill_(-2.0)
    angles = angles_of(40, rotary)
    q_out = torch.full((rows, q_heads, dim), 7.0, device="cuda:0", dtype=kind_of(torch, out_kind)) if q_heads else None
    got = pool.append_rotary(qkv[:, :q_heads] if q_heads else None, qkv[:, q_heads:q_heads + heads], qkv[:, q_heads + heads:],
                             torch.from_numpy(angles).to("cuda:0") if rotary else None, i32(torch, seqs), i32(torch, positions),
                             i32(torch, tables), interleaved=interleaved, q_out=q_out)
    pool.synchronize()
    live = slice(0, 33)
    turn = angles[positions[live]]
    x = mixed[live].astype(np.float64)
    ref = kv4.rotate(x[:, :q_heads + heads], turn, interleaved, np.float64)
    size = np.abs(x[:, :q_heads + heads]).max(-1, keepdims=True) * 2
    if q_heads:
        assert got is q_out
        within(host(got)[live], ref[:, :q_heads], 2.0 ** -23 * size[:, :q_heads] + rounding(out_kind, ref[:, :q_heads]) * 1.001)
        assert (host(got)[33:] == 7).all()
    keys, values = host(pool.key_arena), host(pool.value_arena)
    seen = np.zeros(keys.shape, bool)
    for r in range(33):
        b, s = tables[seqs[r], positions[r] // block], positions[r] % block
        want = ref[r, q_heads:]
        within(keys[b, :, s], want, 2.0 ** -23 * size[r, q_heads:] + rounding(kind, want) * 1.001)
        within(values[b, :, s], x[r, q_heads + heads:], rounding(kind, x[r, q_heads + heads:]))
        seen[b, :, s] = True
    assert (keys[~seen] == 3).all() and (values[~seen] == -2).all()
    # rows read back are the pool's own, bit for bit
    back_k, back_v = pool.gather_rows(i32(torch, seqs[live]), i32(torch, positions[live]), i32(torch, tables))
    pool.synchronize()
    for r in (0, 11, 12, 32):
        b, s = tables[seqs[r], positions[r] // block], positions[r] % block
        assert torch.equal(back_k[r], pool.key_arena[b, :, s]) and torch.equal(back_v[r], pool.value_arena[b, :, s])
    pool.close()


@pytest.mark.parametrize("rows_kind", ["same", "f32"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,q_heads,dim,rotary,interleaved,block,rows", [
    (8, 32, 128, 128, False, 16, 61), (1, 1, 64, 64, True, 32, 5), (3, 6, 128, 32, False, 48, 40), (2, 0, 64, 16, False, 16, 1),
    (2, 2, 128, 0, False, 64, 20), (40, 40, 128, 64, True, 16, 3), (5, 5, 64, 6, False, 16, 9)])
def test_append_rotary_four_bits(torch, il, kv4, rows_kind, kind, heads, q_heads, dim, rotary, interleaved, block, rows):
    rows_kind = kind if rows_kind == "same" else rows_kind
    rng = np.random.default_rng(rows + dim)
    before = rng.integers(0, 40, 3)
    new = np.array([rows - 2 * (rows // 3), rows // 3, rows // 3])
    tables, blocks = deal(rng, before + new, block)
    arena = random_arena(kv4, rng, blocks, heads, block, dim, kind)
    pool = filled_pool(torch, il, arena, kind, block, dim)
    seqs = np.repeat(np.arange(3), new)
    positions = np.concatenate([b + np.arange(n) for b, n in zip(before, new)])
    order = rng.permutation(rows)  # the rows of a call come in any order
    seqs, positions = seqs[order], positions[order]
    x = rng.standard_normal((rows, q_heads + 2 * heads, dim)) * np.exp2(rng.integers(-6, 7, (rows, 1, 1)))
    x[0, -1] = 0.0
    x[rows // 2, q_heads] = 0.5
    mixed = kv4.round_to(x, rows_kind)
    qkv = torch.from_numpy(mixed).to("cuda:0", kind_of(torch, rows_kind))
    angles = angles_of(128, rotary)
    pool.append_rotary(qkv[:, :q_heads] if q_heads else None, qkv[:, q_heads:q_heads + heads], qkv[:, q_heads + heads:],
                       torch.from_numpy(angles).to("cuda:0") if rotary else None, i32(torch, seqs), i32(torch, positions),
                       i32(torch, tables), interleaved=interleaved)
    pool.synchronize()
    # the float32 statement takes the kernel's steps one by one, so the bytes are the same
    keys = kv4.round_to(kv4.rotate(mixed[:, q_heads:q_heads + heads], angles[positions], interleaved), kind)
    values = kv4.round_to(mixed[:, q_heads + heads:], kind)
    place = tables[seqs, positions // block]
    kv4.write_rows(arena, place, positions % block, keys, values)
    assert np.array_equal(pool.arena.cpu().numpy(), arena)
    back_k, back_v = pool.gather_rows(i32(torch, seqs), i32(torch, positions), i32(torch, tables))
    pool.synchronize()
    for back, rows_in in ((back_k, keys), (back_v, values)):
        want = kv4.values_of(*kv4.quantise(rows_in))
        # product and sum in fp32 before the type's rounding
        within(host(back), want, rounding(kind, want) * 1.001 + 2.0 ** -23 * (np.abs(want) + np.abs(rows_in).max()))
    # one sequence's rows, and append without rotation
    n = int((before + new)[0])
    got_k, got_v = pool.gather(i32(torch, tables[0, :(n + block - 1) // block]), n)
    whole_k, whole_v = kv4.read_rows(arena, tables[0], n, dim)
    for got, want in ((got_k, whole_k), (got_v, whole_v)):
        within(host(got), want.transpose(1, 0, 2), rounding(kind, want.transpose(1, 0, 2)) * 1.001 + 2.0 ** -22 * np.abs(want).max())
    pool.append(torch.from_numpy(keys).to("cuda:0").contiguous(), torch.from_numpy(values).to("cuda:0").contiguous(),
                i32(torch, seqs), i32(torch, positions), i32(torch, tables))
    pool.synchronize()
    assert np.array_equal(pool.arena.cpu().numpy(), arena)
    pool.close()


def test_append_rotary_far_positions_and_bad_rows(torch, il, kv4):
    """Each bad row is reported and skipped whole, the others land."""
    rng = np.random.default_rng(5)
    for bits in (None, 4):
        pool = il.CudaKvPool(0, 2, 40, 16, 2, 64, kv_bits=bits)
        arena = (lambda p=pool: p.arena.clone()) if bits else (lambda p=pool: torch.stack([p.key_arena, p.value_arena]).clone())
        tables = i32(torch, [[5, 99, 6], [7, 8, -2]])
        angles = torch.from_numpy(angles_of(40, 64)).to("cuda:0")
        cases = [(0, 20, "paged KV block table contains an invalid page"), (1, 40, "paged KV append position is outside the block table"),
                 (1, 33, "paged KV block table contains an invalid page"), (2, 3, "paged KV append position is outside the block table"),
                 (-2, 3, "paged KV append position is outside the block table"), (0, -1, "paged KV append position is outside the block table"),
                 (0, 48, "paged KV append position is outside the block table")]
        rows = torch.from_numpy(rng.standard_normal((2, 6, 64)).astype(np.float32)).to("cuda:0")
        for seq, pos, message in cases:
            was = arena()
            q_out = torch.full((2, 2, 64), 9.0, device="cuda:0")
            pool.append_rotary(rows[:, :2], rows[:, 2:4], rows[:, 4:], angles, i32(torch, [seq, 1]), i32(torch, [pos, 4]), tables,
                               q_out=q_out)
            with pytest.raises(il.AttentionError, match=f"^{message}$"):
                pool.synchronize()
            now = arena()
            assert (q_out[0] == 9).all() and not (q_out[1] == 9).any()
            changed = (now != was).flatten(2 if bits is None else 1).any(-1)
            only = changed if bits else changed.any(0)
            assert only.nonzero().flatten().tolist() in ([8 - 1], [])  # row 1 went to block 7 (the same bytes the second time)
        # non-finite rows: not written, whichever of K and V holds the value
        for at in (2, 5):
            bad = rows.clone()
            bad[0, at, 17] = float("nan") if at == 2 else float("inf")
            was = arena()
            pool.append_rotary(bad[:, :2], bad[:, 2:4], bad[:, 4:], angles, i32(torch, [0, 1]), i32(torch, [3, 4]), tables)
            with pytest.raises(il.AttentionError, match="^attention input must be finite$"):
                pool.synchronize()
            assert torch.equal(arena()[..., 5, :, :, :] if bits is None else arena()[5], was[..., 5, :, :, :] if bits is None else was[5])
            # so in rows that no 16-byte load reaches; Q leaves either way
            odd = torch.zeros((2, 6 * 64 + 1), device="cuda:0")
            odd[:, 1:] = bad.flatten(1)
            odd = odd[:, 1:].unflatten(1, (6, 64))
            outs = [torch.full((2, 2, 64), 9.0, device="cuda:0") for _ in range(2)]
            for source, out in zip((bad, odd), outs):
                pool.append_rotary(source[:, :2], source[:, 2:4], source[:, 4:], angles, i32(torch, [0, 1]), i32(torch, [3, 4]), tables,
                                   q_out=out)
                with pytest.raises(il.AttentionError, match="^attention input must be finite$"):
                    pool.synchronize()
            assert torch.equal(arena()[..., 5, :, :, :] if bits is None else arena()[5], was[..., 5, :, :, :] if bits is None else was[5])
            assert torch.equal(outs[0], outs[1]) and not (outs[0] == 9).any()
        # a 4-bit group whose scale f16 cannot hold
        if bits:
            wide = rows.clone()
            wide[0, 3, 0], wide[0, 3, 1] = 3e6, -3e6
            was = arena()
            pool.append_rotary(None, wide[:, 2:4], wide[:, 4:], None, i32(torch, [0, -1]), i32(torch, [3, 4]), tables)
            with pytest.raises(il.AttentionError, match="^attention input must be finite$"):
                pool.synchronize()
            assert torch.equal(arena(), was)
        pool.close()


@pytest.mark.parametrize("shift", [0, 1])
def test_append_rotary_rejects_what_the_row_type_cannot_hold(torch, il, shift):
    """fp32 rows over 16-bit pools: 65520 is the first number that f16 rounds to infinity, and a rotation can reach it. `shift` 1:
    rows that no 16-byte load reaches."""
    turn = torch.tensor([[0.6] * 32 + [0.8] * 32] * 8, device="cuda:0")
    for kind, bits, value, angles, ok in ((1, None, 65519.0, None, True), (1, None, 65520.0, None, False), (1, 4, 70000.0, None, False),
                                          (2, None, 70000.0, None, True), (2, None, 3.4e38, None, False), (1, None, 60000.0, turn, False),
                                          (1, None, 40000.0, turn, True), (2, 4, 4e5, None, True), (2, 4, 6e5, None, False)):
        for which in (0, 1):
            if angles is not None and which == 1:
                continue  # values are not rotated
            pool = il.CudaKvPool(0, kind, 4, 16, 2, 64, kv_bits=bits)
            flat = torch.zeros((1, 4 * 64 + shift), device="cuda:0")
            rows = flat[:, shift:].unflatten(1, (4, 64))
            rows[0, 2 * which + 1, 3] = value
            rows[0, 2 * which + 1, 35] = -value
            pool.append_rotary(None, rows[:, :2], rows[:, 2:], angles, i32(torch, [0]), i32(torch, [5]), i32(torch, [[2]]))
            if ok:
                pool.synchronize()
            else:
                with pytest.raises(il.AttentionError, match="^attention input must be finite$"):
                    pool.synchronize()
                assert not (pool.arena if bits else torch.stack([pool.key_arena, pool.value_arena])).any()
            pool.close()


@pytest.mark.parametrize("bits", [None, 4])
def test_no_rows_and_rows_behind_the_last(torch, il, bits):
    """Calls of no rows write nothing; so do padded rows among others, in the pool and in q_out."""
    pool = il.CudaKvPool(0, 2, 6, 16, 2, 64, kv_bits=bits)
    tables = i32(torch, [[1, 2], [3, 4]])
    none = torch.zeros((0, 2, 64), device="cuda:0")
    assert pool.append_rotary(none, none, none, None, i32(torch, []), i32(torch, []), tables).shape == none.shape
    keys, values = pool.gather_rows(i32(torch, []), i32(torch, []), tables)
    assert keys.shape == values.shape == none.shape
    rows = torch.randn((5, 6, 64), device="cuda:0")
    angles = torch.from_numpy(angles_of(32, 64)).to("cuda:0")
    out = torch.full((5, 2, 64), 9.0, device="cuda:0")
    pool.append_rotary(rows[:, :2], rows[:, 2:4], rows[:, 4:], angles, i32(torch, [0, -1, 1, -1, -1]), i32(torch, [17, 5, 31, -7, 1 << 30]), tables,
                       q_out=out)
    pool.synchronize()
    assert [(out[r] == 9).all().item() for r in range(5)] == [False, True, False, True, True]
    written = (pool.arena if bits else torch.stack([pool.key_arena, pool.value_arena], 1)).flatten(1).any(1)
    assert written.nonzero().flatten().tolist() == [2, 4]
    pool.close()


def test_append_rotary_refusals(torch, il):
    pool = il.CudaKvPool(0, 2, 8, 16, 2, 64, kv_bits=4)
    rows = torch.randn((4, 8, 64), device="cuda:0")
    seqs, pos, tables = i32(torch, [0] * 4), i32(torch, range(4)), i32(torch, [[1, 2]])
    angles = torch.ones((8, 64), device="cuda:0")
    good = dict(queries=rows[:, :4], key_rows=rows[:, 4:6], value_rows=rows[:, 6:], cos_sin=angles, row_sequences=seqs, positions=pos,
                block_tables=tables)
    for change, message in [
            (dict(key_rows=rows[:, 4:6].half()), "paged KV row dtype must be FP32 or the pool dtype"),
            (dict(value_rows=rows[:, 6:].bfloat16()), "value_rows must have dtype"),
            (dict(key_rows=rows[:, 4:7]), "shapes do not match"),
            (dict(key_rows=rows[:, 4:6, :32]), "shapes do not match"),
            (dict(value_rows=rows[:3, 6:]), "shapes do not match"),
            (dict(queries=rows[:3, :4]), "shapes do not match"),
            (dict(key_rows=rows[:, 4:8:2]), "key_rows must have contiguous heads"),
            (dict(key_rows=rows[:, 4:6].cpu()), "key_rows must live on"),
            (dict(cos_sin=angles[:, :33].contiguous()), "rotary_dim must be even"),
            (dict(cos_sin=torch.ones((8, 66), device="cuda:0")), "rotary_dim must be even"),
            (dict(cos_sin=angles.half()), "cos_sin must have dtype"),
            (dict(positions=pos.long()), "positions must have dtype"),
            (dict(row_sequences=seqs[:2]), "shapes do not match"),
            (dict(q_out=torch.empty((4, 4, 64), device="cuda:0", dtype=torch.float16)), "q_out must be shaped like the queries"),
            (dict(q_out=torch.empty((4, 3, 64), device="cuda:0")), "q_out must be shaped like the queries"),
            (dict(queries=None, q_out=torch.empty((4, 4, 64), device="cuda:0")), "q_out needs queries"),
            (dict(block_tables=tables[0]), "shapes do not match")]:
        with pytest.raises(il.AttentionError, match=message):
            pool.append_rotary(**{**good, **change})
    q = rows[:, :4].contiguous()
    with pytest.raises(il.AttentionError, match="query output overlaps its input rows"):
        pool.append_rotary(**{**good, "queries": q, "q_out": q})
    # entries that read whole elements name the refusal
    table, lens = i32(torch, [[1, 2]]), i32(torch, [5])
    query = torch.randn((1, 4, 64), device="cuda:0")
    with pytest.raises(il.AttentionError, match="partials do not read a 4-bit pool"):
        pool.decode_partials(query, table, lens, 5)
    with pytest.raises(il.AttentionError, match="decode step does not read a 4-bit pool"):
        pool.decode_step_host(query.cpu().numpy(), table.cpu().numpy(), lens.cpu().numpy())
    with pytest.raises(il.AttentionError, match="projection does not append to a 4-bit pool"):
        pool.project_append(torch.zeros((4, 64), device="cuda:0", dtype=torch.bfloat16),
                            torch.zeros((8 * 64, 64), device="cuda:0", dtype=torch.bfloat16), 4, seqs, pos, tables)
    with pytest.raises(il.AttentionError, match="one packed arena"):
        pool.key_arena
    for entry, message in (("inferlab_cuda_paged_decode", "inferlab_cuda_kv4_decode reads a 4-bit pool"),
                           ("inferlab_cuda_paged_decode_noalloc", "without a workspace does not read a 4-bit pool")):
        err = ctypes.create_string_buffer(256)
        args = [pool._handle, query.data_ptr(), table.data_ptr(), 2, lens.data_ptr(), 1, 4, 5, query.data_ptr()]
        args += [None, 0, None] if entry.endswith("decode") else [None]
        assert getattr(pool._lib, entry)(*args, err, 256) == -1 and message in err.value.decode()
    wide = il.CudaKvPool(0, 2, 8, 16, 2, 64)
    err = ctypes.create_string_buffer(256)
    assert wide._lib.inferlab_cuda_kv4_decode(wide._handle, query.data_ptr(), 0, table.data_ptr(), 2, lens.data_ptr(), 1, 4, 5,
                                              query.data_ptr(), None, 0, None, err, 256) == -1
    assert err.value == b"4-bit attention needs a 4-bit pool"
    with pytest.raises(il.AttentionError, match="only a 4-bit pool has a packed arena"):
        wide.arena
    wide.close()
    pool.close()


# ---- attention ------------------------------------------------------------------------------------------------------------
def check_attention(torch, kv4, il, kind, q_kind, heads, q_heads, dim, block, starts, counts, seed=0, decode=False, split=0, poison=True):
    rng = np.random.default_rng(seed + dim + q_heads)
    starts, counts = np.asarray(starts), np.asarray(counts)
    totals = starts + counts
    tables, blocks = deal(rng, totals, block)
    arena = random_arena(kv4, rng, blocks, heads, block, dim, kind)
    if poison:  # what no sequence owns may hold anything: here f16 NaN pairs
        live = np.zeros((blocks, block), bool)
        for i, n in enumerate(totals):
            for t in range(int(n)):
                live[tables[i, t // block], t % block] = True
        for which in (0, 1):
            at, _, pair_at = kv4.places(dim, which)
            for b, t in zip(*np.nonzero(~live)):
                arena[b, :, t // 16][:, at[t % 16]] = 0xFF
                arena[b, :, t // 16][:, (pair_at[t % 16][:, None] + np.arange(4)).ravel()] = 0xFF
    pool = filled_pool(torch, il, arena, kind, block, dim)
    if split:
        pool.set_decode_split(split)
    total = int(counts.sum())
    raw = kv4.round_to(rng.standard_normal((total, q_heads, dim)) * 1.5, q_kind)
    q = torch.from_numpy(raw).to("cuda:0", kind_of(torch, q_kind))
    if decode:
        got = pool.decode(q, i32(torch, tables), i32(torch, totals), max(1, int(totals.max())))
    else:
        offsets = np.concatenate([[0], np.cumsum(counts)[:-1]])
        got = pool.prefill(q, i32(torch, tables), i32(torch, starts), i32(torch, counts), i32(torch, offsets), int(counts.max()),
                           max_context_len=int(totals.max()))
    pool.synchronize()
    assert got.dtype == q.dtype
    got, at = host(got), 0
    rounded = kv4.round_to(raw, kind).astype(np.float64)
    for i, (first, n) in enumerate(zip(starts, counts)):
        if n == 0:
            continue
        keys, values = kv4.read_rows(arena, tables[i], int(totals[i]), dim)
        out, reach, size = kv4.attend(rounded[at:at + n], keys, values, int(first))
        many = not decode and q_kind != "f32" and q_heads // heads * int(counts.max()) >= 64
        within(got[at:at + n], out, attention_bound(q_kind, out, reach, size, dim, f16_cache=many))
        at += n
    pool.close()


GEOMETRIES = [(8, 8, 64, 16), (2, 8, 128, 16), (8, 8, 128, 32), (1, 5, 64, 48), (2, 14, 128, 16), (1, 16, 128, 64), (3, 3, 128, 16),
              (1, 24, 64, 16), (2, 4, 64, 16)]


@pytest.mark.parametrize("heads,q_heads,dim,block", GEOMETRIES)
@pytest.mark.parametrize("kind,q_kind", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
def test_decode(torch, kv4, il, kind, q_kind, heads, q_heads, dim, block):
    lengths = np.array([1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 129, 300, 0])
    starts = lengths - 1
    check_attention(torch, kv4, il, kind, q_kind, heads, q_heads, dim, block, starts, np.ones_like(lengths), decode=True)


@pytest.mark.parametrize("split", [1, 3, 7, 0])
@pytest.mark.parametrize("heads,q_heads,dim,block", [(2, 8, 128, 16), (1, 7, 64, 32)])
def test_decode_splits(torch, kv4, il, split, heads, q_heads, dim, block):
    lengths = np.array([1, 16, 17, 100, 0, 937])
    for q_kind in ("bf16", "f32"):
        check_attention(torch, kv4, il, "bf16", q_kind, heads, q_heads, dim, block, lengths - 1, np.ones_like(lengths), decode=True,
                        split=split)


@pytest.mark.parametrize("heads,q_heads,dim,block", GEOMETRIES)
@pytest.mark.parametrize("kind,q_kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
def test_prefill(torch, kv4, il, kind, q_kind, heads, q_heads, dim, block):
    starts = [0, 0, 5, 16, 100, 31, 0, 300, 7]
    counts = [1, 17, 5, 16, 1, 33, 0, 2, 70]
    check_attention(torch, kv4, il, kind, q_kind, heads, q_heads, dim, block, starts, counts)


@pytest.mark.parametrize("split", [1, 5])
def test_prefill_splits(torch, kv4, il, split):
    check_attention(torch, kv4, il, "bf16", "bf16", 2, 8, 128, 16, [0, 200, 3, 90], [40, 5, 1, 6], split=split)


@pytest.mark.parametrize("heads,q_heads,dim,block,start,count", [(1, 4, 128, 16, 0, 600), (2, 2, 64, 32, 1000, 300), (1, 8, 128, 16, 2500, 130)])
def test_prefill_long_chunks(torch, kv4, il, heads, q_heads, dim, block, start, count):
    check_attention(torch, kv4, il, "bf16", "bf16", heads, q_heads, dim, block, [start, 0], [count, 37], poison=False)


@pytest.mark.parametrize("heads,q_heads,dim,block", [(2, 8, 128, 16), (1, 7, 64, 32), (3, 3, 128, 64), (1, 16, 64, 16)])
@pytest.mark.parametrize("kind,q_kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
def test_prefill_around_row_tiles(torch, kv4, il, kind, q_kind, heads, q_heads, dim, block):
    """Rows one below, at and above 64 and 128, keys around 64, with and without splits of the keys."""
    group = q_heads // heads
    counts = [max(1, n // group + extra) for n in (63, 64, 127, 128, 256) for extra in (0, 1)] + [0, 1]
    starts = [0, 1, 63, 64, 65, 127, 0, 300, 15, 0, 20, 0]
    for split in (0, 4, 12):
        check_attention(torch, kv4, il, kind, q_kind, heads, q_heads, dim, block, starts, counts, seed=split, split=split)


@pytest.mark.parametrize("q_kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_many_rows_large_and_tiny_scales(torch, kv4, il, dim, q_kind):
    """40 query tokens: keys whose scores differ a lot, values of very different size token by token."""
    rng = np.random.default_rng(dim)
    length, count = 333, 40
    tables, blocks = deal(rng, [length], 16)
    for q_size, spread in ((0.0, 1.0), (1.0, 1e3), (12.0, 1.0), (1e-20, 1e-2), (3e2, 10.0)):
        arena = np.zeros((blocks, 2, 1, kv4.tile_bytes(dim)), np.uint8)
        keys = rng.standard_normal((length, 2, dim)).astype(np.float32)
        values = (rng.standard_normal((length, 2, dim)) * spread ** rng.uniform(-1, 1, (length, 2, 1))).astype(np.float32)
        values[::7] = np.float32(0.25)  # groups without a range: scale 0
        kv4.write_rows(arena, tables[0, np.arange(length) // 16], np.arange(length) % 16, kv4.bf16(keys), kv4.bf16(values))
        pool = filled_pool(torch, il, arena, "bf16", 16, dim)
        raw = kv4.bf16(rng.standard_normal((count, 8, dim)) * q_size)
        q = torch.from_numpy(raw).to("cuda:0", kind_of(torch, q_kind))
        got = host(pool.prefill(q, i32(torch, tables), i32(torch, [length - count]), i32(torch, [count]), i32(torch, [0]), count,
                                max_context_len=length))
        pool.synchronize()
        k, v = kv4.read_rows(arena, tables[0], length, dim)
        out, reach, size = kv4.attend(raw.astype(np.float64), k, v, length - count)
        within(got, out, attention_bound(q_kind, out, reach, size, dim, f16_cache=q_kind != "f32"))
        pool.close()


@pytest.mark.parametrize("q_kind", ["bf16", "f32"])
def test_prefill_of_many_rows_reports_what_it_cannot_read(torch, kv4, il, q_kind):
    rng = np.random.default_rng(13)
    tables, blocks = deal(rng, [90, 90], 16)
    arena = random_arena(kv4, rng, blocks, 1, 16, 64)
    pool = filled_pool(torch, il, arena, "bf16", 16, 64)
    raw = kv4.bf16(rng.standard_normal((60, 2, 64)))
    q = torch.from_numpy(raw).to("cuda:0", kind_of(torch, q_kind))

    def run(queries=q, starts=(60, 60), counts=(30, 30), offsets=(0, 30), at=tables):
        out = torch.full((60, 2, 64), 7.0, device="cuda:0", dtype=q.dtype)
        pool.prefill(queries, i32(torch, at), i32(torch, starts), i32(torch, counts), i32(torch, offsets), 30, max_context_len=90, out=out)
        return host(out)

    good = run()
    pool.synchronize()
    for change, rows in ((dict(starts=(60, 61)), "zero"), (dict(starts=(60, -1)), "zero"), (dict(counts=(30, 31)), "kept"),
                         (dict(offsets=(0, 31)), "kept"), (dict(offsets=(0, -1)), "kept"), (dict(counts=(30, -1)), "kept")):
        out = run(**change)
        with pytest.raises(il.AttentionError, match="^paged prefill segment is invalid$"):
            pool.synchronize()
        assert np.array_equal(out[:30], good[:30]) and (out[30:] == (0.0 if rows == "zero" else 7.0)).all()
    for bad in (-1, blocks, 1 << 30):
        broken = tables.copy()
        broken[1, 4] = bad
        out = run(at=broken)
        with pytest.raises(il.AttentionError, match="^paged KV block table contains an invalid page$"):
            pool.synchronize()
        assert np.array_equal(out[:30], good[:30])
    for value in (float("nan"), float("inf")):
        wrong = q.clone()
        wrong[40, 1, 5] = value
        out = run(wrong)
        with pytest.raises(il.AttentionError, match="^attention input must be finite$"):
            pool.synchronize()
        assert np.array_equal(out[:30], good[:30])
    # rows behind and between the segments stay as they are
    out = run(counts=(20, 25))
    pool.synchronize()
    assert (out[20:30] == 7.0).all() and (out[55:] == 7.0).all()
    pool.close()


@pytest.mark.parametrize("seqs", [2, 31, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("split", [0, 2])
def test_batches_in_any_order_of_lengths(torch, kv4, il, seqs, split):
    """Ascending, equal and mixed lengths, empty sequences among them; more CTAs than run at once, whole and split."""
    rng = np.random.default_rng(seqs)
    for lengths in (np.arange(seqs) + 6, np.full(seqs, 20), rng.integers(0, 90, seqs)):
        counts = np.minimum(lengths, 5)
        check_attention(torch, kv4, il, "bf16", "bf16", 4, 32, 64, 16, lengths - counts, counts, split=split, poison=False)
        check_attention(torch, kv4, il, "bf16", "f32", 4, 32, 64, 16, lengths - 1, np.ones_like(lengths), decode=True, split=split, poison=False)
    # a bad length among them: its rows are zero, the others' as before
    tables, blocks = deal(rng, np.full(seqs, 40), 16)
    pool = filled_pool(torch, il, random_arena(kv4, rng, blocks, 4, 16, 64), "bf16", 16, 64)
    pool.set_decode_split(split)
    q = torch.randn((seqs, 32, 64), device="cuda:0")
    good = host(pool.decode(q, i32(torch, tables), i32(torch, np.full(seqs, 40)), 40))
    pool.synchronize()
    for bad in (-1, -2, -(1 << 31), 41, (1 << 31) - 1):
        lens = np.full(seqs, 40)
        lens[seqs // 2] = bad
        out = host(pool.decode(q, i32(torch, tables), i32(torch, lens), 40))
        with pytest.raises(il.AttentionError, match="^paged KV context length is invalid$"):
            pool.synchronize()
        assert not out[seqs // 2].any()
        rest = np.arange(seqs) != seqs // 2
        assert np.array_equal(out[rest], good[rest])
    pool.close()


def test_decode_long_flat_and_sharp(torch, kv4, il):
    """20,000 keys: queries of zero weigh all alike, large ones pick a few."""
    rng = np.random.default_rng(8)
    dim, length = 128, 20000
    tables, blocks = deal(rng, [length, length], 16)
    arena = random_arena(kv4, rng, blocks, 2, 16, dim)
    pool = filled_pool(torch, il, arena, "bf16", 16, dim)
    raw = rng.standard_normal((2, 8, dim)) * np.array([0.0, 1e-3, 0.1, 1.0, 1.0, 5.0, 20.0, 0.3])[None, :, None]
    raw = kv4.round_to(raw, "bf16")
    for q_kind in ("bf16", "f32"):
        q = torch.from_numpy(raw).to("cuda:0", kind_of(torch, q_kind))
        got = host(pool.decode(q, i32(torch, tables), i32(torch, [length, length]), length))
        pool.synchronize()
        for i in range(2):
            keys, values = kv4.read_rows(arena, tables[i], length, dim)
            out, reach, size = kv4.attend(raw[i:i + 1].astype(np.float64), keys, values, length - 1)
            within(got[i:i + 1], out, attention_bound(q_kind, out, reach, size, dim))
    pool.close()


def test_decode_large_and_tiny_scales(torch, kv4, il):
    """Queries and caches of very large and very small numbers, within bf16's range."""
    rng = np.random.default_rng(9)
    dim, length = 64, 200
    tables, blocks = deal(rng, [length], 16)
    for q_size, v_size in ((1e-20, 1e4), (1e20, 1e-3), (3e4, 2.0), (1e-30, 1e-2)):
        arena = np.zeros((blocks, 1, 1, kv4.tile_bytes(dim)), np.uint8)
        keys = rng.standard_normal((length, 1, dim)).astype(np.float32) * np.float32(min(1.0, 1 / q_size) if q_size < 1e10 else 1e-4)
        values = rng.standard_normal((length, 1, dim)).astype(np.float32) * np.float32(v_size)
        kv4.write_rows(arena, tables[0, np.arange(length) // 16], np.arange(length) % 16, kv4.bf16(keys), kv4.bf16(values))
        pool = filled_pool(torch, il, arena, "bf16", 16, dim)
        raw = kv4.bf16(rng.standard_normal((1, 2, dim)) * q_size)
        q = torch.from_numpy(raw).to("cuda:0")
        got = host(pool.decode(q, i32(torch, tables), i32(torch, [length]), length))
        pool.synchronize()
        k, v = kv4.read_rows(arena, tables[0], length, dim)
        out, reach, size = kv4.attend(raw.astype(np.float64), k, v, length - 1)
        if reach.max() < 1e4:  # beyond, fp32 scores themselves decide which key wins
            within(got, out, attention_bound("f32", out, reach, size, dim))
        pool.close()


def test_attention_reports_what_it_cannot_read(torch, kv4, il):
    rng = np.random.default_rng(3)
    tables, blocks = deal(rng, [40, 40], 16)
    arena = random_arena(kv4, rng, blocks, 1, 16, 64)
    pool = filled_pool(torch, il, arena, "bf16", 16, 64)
    q = torch.randn((2, 2, 64), device="cuda:0")
    good = host(pool.decode(q, i32(torch, tables), i32(torch, [40, 40]), 40))
    pool.synchronize()
    for lens in ([40, 41], [40, -1], [40, 70]):
        out = host(pool.decode(q, i32(torch, tables), i32(torch, lens), 40))
        with pytest.raises(il.AttentionError, match="^paged KV context length is invalid$"):
            pool.synchronize()
        assert np.array_equal(out[0], good[0]) and not out[1].any()
    for bad in (-1, blocks, 1 << 30):
        broken = tables.copy()
        broken[1, 1] = bad
        out = host(pool.decode(q, i32(torch, broken), i32(torch, [40, 40]), 40))
        with pytest.raises(il.AttentionError, match="^paged KV block table contains an invalid page$"):
            pool.synchronize()
        assert np.array_equal(out[0], good[0])
    nan = q.clone()
    nan[1, 0, 3] = float("nan")
    out = host(pool.decode(nan, i32(torch, tables), i32(torch, [40, 40]), 40))
    with pytest.raises(il.AttentionError, match="^attention input must be finite$"):
        pool.synchronize()
    assert np.array_equal(out[0], good[0])
    zero, one = i32(torch, [0, 1]), i32(torch, [1, 1])
    for starts, counts in (([39, 40], [1, 1]), ([39, -1], [1, 1])):
        out = host(pool.prefill(q, i32(torch, tables), i32(torch, starts), i32(torch, counts), zero, 1, max_context_len=40))
        with pytest.raises(il.AttentionError, match="^paged prefill segment is invalid$"):
            pool.synchronize()
        assert np.array_equal(out[0], good[0]) and not out[1].any()
    del one
    for change, message in [(dict(queries=q.half()), "query dtype"), (dict(queries=q[:, :, :32].contiguous()), "shapes do not match"),
                            (dict(context_lens=i32(torch, [4])), "shapes do not match"), (dict(out=q.bfloat16()), "out must have dtype"),
                            (dict(queries=q[:1]), "shapes do not match"),
                            (dict(out=torch.empty((2, 1, 64), device="cuda:0")), "shaped like the queries")]:
        args = dict(queries=q, block_tables=i32(torch, tables), context_lens=i32(torch, [40, 40]), max_context_len=40)
        with pytest.raises(il.AttentionError, match=message):
            pool.decode(**{**args, **change})
    pool.close()


def test_cache_beyond_32_bit_offsets(torch, kv4, il):
    """A sequence in the last blocks of a cache of more than 2^32 bytes."""
    rng = np.random.default_rng(4)
    heads, dim, length = 8, 128, 300
    blocks = (9 << 29) // (heads * kv4.tile_bytes(dim))
    assert blocks * heads * kv4.tile_bytes(dim) > 1 << 32
    small = random_arena(kv4, rng, 19, heads, 16, dim)
    pool = il.CudaKvPool(0, 2, blocks, 16, heads, dim, kv_bits=4)
    pool.arena[blocks - 19:].copy_(torch.from_numpy(small))
    table = np.arange(19)[None]
    raw = kv4.bf16(rng.standard_normal((1, 32, dim)))
    rows = kv4.bf16(rng.standard_normal((1, 2 * heads, dim)))
    qkv = torch.from_numpy(rows).to("cuda:0")
    far = i32(torch, table + blocks - 19)
    pool.append_rotary(None, qkv[:, :heads], qkv[:, heads:], None, i32(torch, [0]), i32(torch, [length - 1]), far)
    kv4.write_rows(small, [18], [(length - 1) % 16], rows[:, :heads], rows[:, heads:])
    got = host(pool.decode(torch.from_numpy(raw).to("cuda:0"), far, i32(torch, [length]), length))
    pool.synchronize()
    assert np.array_equal(pool.arena[blocks - 19:].cpu().numpy(), small)
    keys, values = kv4.read_rows(small, table[0], length, dim)
    out, reach, size = kv4.attend(raw.astype(np.float64), keys, values, length - 1)
    within(got, out, attention_bound("f32", out, reach, size, dim))
    pool.close()


def test_views_keep_their_pool(torch, il):
    """An arena outlives the name of its pool: its memory goes with the last view."""
    import gc
    import weakref

    for bits in (None, 4):
        pool = il.CudaKvPool(0, 2, 4, 16, 2, 64, kv_bits=bits)
        alive = weakref.ref(pool)
        view = pool.arena if bits else pool.key_arena
        if bits is None:
            assert pool.key_arena is view
        view.fill_(3)
        del pool
        gc.collect()
        assert alive() is not None and bool((view == 3).all())
        del view
        gc.collect()
        assert alive() is None


def test_pages_copied_and_shared(torch, il, kv4):
    """The page manager's copy on write moves a 4-bit block, and counts its bytes."""
    from inferlab_b200.pages import PageManager, copy_blocks

    rng = np.random.default_rng(6)
    pool = filled_pool(torch, il, random_arena(kv4, rng, 6, 2, 32, 128), "bf16", 32, 128)
    manager = PageManager.for_pool(pool)
    assert manager.stats()["page_bytes"] == pool.block_bytes == 2 * 2 * kv4.tile_bytes(128)
    was = pool.arena.clone()
    copy_blocks(pool, [(1, 4), (2, 0)])
    pool.synchronize()
    assert torch.equal(pool.arena[4], was[1]) and torch.equal(pool.arena[0], was[2]) and torch.equal(pool.arena[3], was[3])
    pool.close()


def test_repeated_and_captured_calls_agree(torch, il, kv4):
    """The same bits eagerly, from two graphs replayed side by side, and on another stream."""
    rng = np.random.default_rng(11)
    lengths = np.array([900, 1, 333, 64])
    tables, blocks = deal(rng, lengths, 16)
    pool = filled_pool(torch, il, random_arena(kv4, rng, blocks, 2, 16, 128), "bf16", 16, 128)
    pool.set_decode_split(4)
    q = torch.randn((4, 8, 128), device="cuda:0").bfloat16()
    lens, table = i32(torch, lengths), i32(torch, tables)
    first = pool.decode(q, table, lens, 900)
    for _ in range(3):
        assert torch.equal(pool.decode(q, table, lens, 900), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs, graphs = [torch.zeros_like(q), torch.zeros_like(q)], []
    torch.cuda.synchronize()
    for out in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pool.decode(q, table, lens, 900, out=out)
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    with torch.cuda.stream(side):
        elsewhere = pool.decode(q, table, lens, 900)
        back = pool.decode(q, table, lens, 900, stream=torch.cuda.default_stream())
    torch.cuda.synchronize()
    assert torch.equal(elsewhere, first) and torch.equal(back, first)
    pool.synchronize()
    pool.close()


def test_batches_of_all_shapes_share_a_workspace(torch, il, kv4):
    """Split decodes and prefills of few and many rows in turn on one workspace: each as on a workspace of its own."""
    rng = np.random.default_rng(21)
    lengths = np.array([1500, 700, 1, 64, 333, 80, 1200, 16] * 6)
    tables, blocks = deal(rng, lengths, 16)
    pool = filled_pool(torch, il, random_arena(kv4, rng, blocks, 2, 16, 128), "bf16", 16, 128)
    pool.set_decode_split(4)
    table, lens = i32(torch, tables), i32(torch, lengths)
    calls = []
    for kind in (torch.bfloat16, torch.float32):
        for seqs in (1, 3, 48):
            q = torch.randn((seqs, 8, 128), device="cuda:0").to(kind)
            calls.append((seqs, 1, lambda ws, q=q, n=seqs: pool.decode(q, table[:n], lens[:n], 1500, workspace=ws)))
            for count in (5, 40):
                q = torch.randn((seqs * count, 8, 128), device="cuda:0").to(kind)
                counts = torch.minimum(lens[:seqs], lens.new_tensor(count))
                at = (torch.arange(seqs, device="cuda:0", dtype=torch.int32) * count).contiguous()
                out = torch.zeros_like(q)
                calls.append((seqs, count, lambda ws, q=q, n=seqs, c=count, k=counts, at=at: pool.prefill(
                    q, table[:n], (lens[:n] - k).contiguous(), k, at, c, out=torch.zeros_like(q), max_context_len=1500, workspace=ws)))
    alone = []
    for seqs, count, call in calls:
        alone.append(call(pool.make_workspace(seqs, 8, 1500, max_query_count=count)))
    shared = pool.make_workspace(48, 8, 1500, max_query_count=40)
    for _ in range(2):
        for i in list(range(len(calls))) + list(rng.permutation(len(calls))):
            assert torch.equal(calls[i][2](shared), alone[i])
            assert torch.equal(calls[i][2](None), alone[i])
    pool.synchronize()
    # too small a workspace, or one that no 16-byte load can read, is refused
    need = pool.workspace_size(48, 8, 1500, 40)
    with pytest.raises(il.AttentionError, match="workspace is too small"):
        calls[5][2](torch.zeros(256, dtype=torch.uint8, device="cuda:0"))
    with pytest.raises(il.AttentionError, match="workspace must be 16-byte aligned"):
        calls[5][2](torch.zeros(need + 64, dtype=torch.uint8, device="cuda:0")[8:])
    flat = torch.zeros(8 * 128 + 1, device="cuda:0", dtype=torch.bfloat16)
    with pytest.raises(il.AttentionError, match="must be 16-byte aligned"):
        pool.decode(flat[1:].view(1, 8, 128), table[:1], lens[:1], 1500)
    none = torch.zeros((0, 8, 128), device="cuda:0", dtype=torch.bfloat16)
    assert pool.decode(none, table[:0], lens[:0], 1500).shape == none.shape
    assert pool.prefill(none, table[:1], lens[:1], lens[:1] * 0, lens[:1] * 0, 40, max_context_len=1500).shape == none.shape
    pool.synchronize()
    pool.close()


@pytest.mark.parametrize("q_kind", ["bf16", "f32"])
def test_prefill_of_many_rows_captured_and_side_by_side(torch, il, kv4, q_kind):
    """The same bits eagerly, from two graphs replayed side by side, and on another stream."""
    rng = np.random.default_rng(31)
    lengths = np.array([900, 130, 333, 640])
    tables, blocks = deal(rng, lengths, 16)
    pool = filled_pool(torch, il, random_arena(kv4, rng, blocks, 16, 16, 64), "bf16", 16, 64)
    pool.set_decode_split(8)
    counts = np.array([130, 130, 1, 77])
    args = (i32(torch, tables), i32(torch, lengths - counts), i32(torch, counts), i32(torch, [0, 130, 260, 261]), 130)
    q = torch.randn((338, 32, 64), device="cuda:0").to(kind_of(torch, q_kind))

    def call(out=None, stream=None):
        return pool.prefill(q, *args, out=out, stream=stream, max_context_len=900)

    first = call()
    for _ in range(3):
        assert torch.equal(call(), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs, graphs = [torch.zeros_like(q), torch.zeros_like(q)], []
    torch.cuda.synchronize()
    for out in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out)
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(10):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            elsewhere = call()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first) and torch.equal(elsewhere, first)
    back = call(stream=side)
    torch.cuda.synchronize()
    assert torch.equal(back, first)
    pool.synchronize()
    pool.close()


def test_serving_run_over_a_four_bit_pool(torch, il, kv4):
    """Projection, rotary append, prompt attention, two decode steps and the output projection, as a layer runs them."""
    rng = np.random.default_rng(12)
    heads, q_heads, dim, model, block = 2, 8, 128, 256, 16
    prompts = np.array([37, 20])
    tables, blocks = deal(rng, prompts + 2, block)
    arena = np.zeros((blocks, heads, 1, kv4.tile_bytes(dim)), np.uint8)
    pool = filled_pool(torch, il, arena, "bf16", block, dim)
    weights = torch.from_numpy(kv4.bf16(rng.standard_normal(((q_heads + 2 * heads) * dim, model)) / 16)).to("cuda:0").bfloat16()
    w_out = torch.from_numpy(kv4.bf16(rng.standard_normal((model, q_heads * dim)) / 32)).to("cuda:0").bfloat16()
    angles = angles_of(64, dim)
    on_device, table = torch.from_numpy(angles).to("cuda:0"), i32(torch, tables)

    def layer(seqs, positions, attention):
        hidden = torch.from_numpy(kv4.bf16(rng.standard_normal((len(seqs), model)))).to("cuda:0").bfloat16()
        qkv = pool.output_project(hidden, weights).view(len(seqs), q_heads + 2 * heads, dim)
        q = pool.append_rotary(qkv[:, :q_heads], qkv[:, q_heads:q_heads + heads], qkv[:, q_heads + heads:], on_device,
                               i32(torch, seqs), i32(torch, positions), table)
        out = attention(q)
        projected = pool.output_project(out.view(len(seqs), -1), w_out)
        pool.synchronize()
        rows = qkv.cpu().numpy()
        turned = kv4.rotate(rows[:, :q_heads + heads], angles[positions], False)
        kv4.write_rows(arena, tables[seqs, positions // block], positions % block, kv4.bf16(turned[:, q_heads:]),
                       kv4.bf16(rows[:, q_heads + heads:]))
        assert np.array_equal(pool.arena.cpu().numpy(), arena)
        assert np.array_equal(q.cpu().numpy(), turned[:, :q_heads])
        for i in range(len(prompts)):
            at = np.nonzero(seqs == i)[0]
            k, v = kv4.read_rows(arena, tables[i], int(positions[at].max()) + 1, dim)
            ref, reach, size = kv4.attend(kv4.bf16(turned[at, :q_heads]).astype(np.float64), k, v, int(positions[at].min()))
            within(host(out)[at], ref, attention_bound("f32", ref, reach, size, dim))
        want = kv4.bf16(host(out).reshape(len(seqs), -1)).astype(np.float64) @ host(w_out).T
        assert np.abs(host(projected) - want).max() <= 1e-4 * np.abs(want).max()

    seqs = np.repeat([0, 1], prompts)
    positions = np.concatenate([np.arange(n) for n in prompts])
    layer(seqs, positions, lambda q: pool.prefill(q, table, i32(torch, [0, 0]), i32(torch, prompts), i32(torch, [0, prompts[0]]), 37))
    for step in range(2):
        layer(np.array([0, 1]), prompts + step, lambda q: pool.decode(q, table, i32(torch, prompts + step + 1)))
    pool.close()
