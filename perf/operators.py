"""Cases of the operators around a paged cache held in 4 bits: the rotary append, one decode step, and several query
tokens per sequence.

A 4-bit cache is one byte tensor [num_blocks][kv_heads][block_tokens / 16][tile]; a tile holds 16 tokens of one kv-head:
key codes, key parameters, value codes, value parameters. Every 64 dims of a token's row share a float16 pair
(scale, zero); a code c in 0..15 stands for zero + (c - 8) * scale. Rows are quantised from values already rounded to the
cache's row type:

    scale = f16((max - min) / 15)    zero = f16(min + 8 * scale)    c = clamp(rint((x - zero) * (1 / scale)) + 8, 0, 15)

with c = 8 where scale is 0. The rotation of a pair (a, b) by the table's (cos, sin) is (a cos - b sin, b cos + a sin).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KV_TYPES = {"f32": 0, "f16": 1, "bf16": 2}
GROUP = 64


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    gqa = {"q_heads": 32, "kv_heads": 8, "dim": 128, "block": 16}
    return [
        # One user's next token into a 4-bit cache: what a single-stream server waits for, layer by layer.
        dict(gqa, name="append 1 token, 4-bit", kind="append", bits=4, type="bf16", rows_type="bf16", rows=1, seqs=1, rotary=128,
             interleaved=False, low=700, high=700, pad=0, lens_seed=1),
        # The next tokens of a padded decode batch into a 16-bit cache.
        dict(gqa, name="append 256 tokens, 16-bit", kind="append", bits=16, type="bf16", rows_type="bf16", rows=256, seqs=256, rotary=128,
             interleaved=False, low=1, high=512, pad=11, lens_seed=2),
        # Packed prompts of a prefill step into a 4-bit cache.
        dict(gqa, name="append 8192 tokens, 4-bit", kind="append", bits=4, type="bf16", rows_type="bf16", rows=8192, seqs=9, rotary=128,
             interleaved=False, low=0, high=300, pad=0, lens_seed=3),
        # Eight prompts of 1024 from float32 projections, half of each head rotated pair by pair, 16-bit cache.
        dict(name="append 8192 tokens, f32 rows", kind="append", bits=16, type="f16", rows_type="f32", rows=8192, seqs=8, q_heads=16,
             kv_heads=16, dim=128, block=16, rotary=64, interleaved=True, low=0, high=0, pad=0, lens_seed=4),
        # One short conversation, every head its own keys: the smallest decode, where latency counts.
        dict(name="decode 1 x 700, 8x64", kind="decode", type="f16", q_heads=8, kv_heads=8, dim=64, block=16, seqs=1, low=700, high=700,
             zipf=False, lens_seed=5),
        # The small decode batch, uniform context lengths.
        dict(name="decode 64 x 64..2048, 8x64", kind="decode", type="f16", q_heads=8, kv_heads=8, dim=64, block=16, seqs=64, low=64,
             high=2048, zipf=False, lens_seed=6),
        # The decode part of a mixed step: most contexts short, a few long.
        dict(gqa, name="decode 32 x zipf 8192", kind="decode", type="bf16", seqs=32, low=32, high=8192, zipf=True, lens_seed=7),
        # One very long document.
        dict(gqa, name="decode 1 x 131072", kind="decode", type="bf16", seqs=1, low=131072, high=131072, zipf=False, lens_seed=8),
        # The long-context batch.
        dict(gqa, name="decode 64 x 4096..32768", kind="decode", type="bf16", seqs=64, low=4096, high=32768, zipf=False, lens_seed=9),
        # Five drafted tokens per sequence checked in one pass.
        dict(gqa, name="prefill 64 x 5 drafts", kind="prefill", type="bf16", seqs=64, count=5, ragged=False, low=64, high=2048, zipf=False,
             lens_seed=10),
        # The chunked-prefill part of a mixed step.
        dict(gqa, name="prefill 4 x 512 on zipf 8192", kind="prefill", type="bf16", seqs=4, count=512, ragged=False, low=32, high=8192,
             zipf=True, lens_seed=11),
        # Whole prompts of uneven length, 32-token blocks, every head its own keys.
        dict(name="prefill 8 x 1..1024", kind="prefill", type="bf16", q_heads=16, kv_heads=16, dim=128, block=32, seqs=8, count=1024,
             ragged=True, low=0, high=0, zipf=False, lens_seed=12),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 4, 5, 7, 8, 16]) if kv_heads <= 4 else rng.choice([1, 2, 3, 4])
    c = {"kind": kind, "kv_heads": kv_heads, "q_heads": kv_heads * group, "dim": rng.choice([64, 128, 128]), "block": rng.choice([16, 16, 32, 64]),
         "type": rng.choice(["f16", "bf16"]), "lens_seed": rng.randrange(1 << 30)}
    if kind == "append":
        rows = _log(rng, 1, 8192)
        c.update(rows=rows, seqs=min(rows, _log(rng, 1, 300)), bits=rng.choice([4, 4, 16, 32]), rotary=rng.choice([c["dim"], c["dim"] // 2]),
                 interleaved=rng.random() < 0.3, low=0, high=_log(rng, 1, 1000), pad=rng.choice([0, 0, 1]) * (rows // 7))
        c["rows_type"] = "f32" if c["bits"] == 32 else rng.choice([c["type"], "f32"])
        while c["rows"] * c["q_heads"] * c["dim"] > 8192 * 16 * 128:
            c["rows"] = c["rows"] // 2 + 1
        c["seqs"], c["pad"] = min(c["seqs"], c["rows"]), min(c["pad"], c["rows"] - 1)
        return c
    c["zipf"] = rng.random() < 0.3
    if kind == "decode":
        c["seqs"], c["high"] = _log(rng, 1, 300), _log(rng, 1, 131072)
        while c["seqs"] * c["high"] * kv_heads * c["dim"] > 1 << 28:
            c["high"] = c["high"] * 2 // 3 + 1
        c["low"] = rng.choice([0, 1, c["high"], (c["high"] + 1) // 2])
    else:
        c["type"] = "bf16"
        c["seqs"], c["count"], c["high"] = _log(rng, 1, 64), _log(rng, 1, 600), _log(rng, 1, 8192)
        while c["seqs"] * c["count"] * c["q_heads"] * (c["high"] + c["count"]) > 1 << 29 or c["seqs"] * c["high"] * kv_heads * c["dim"] > 1 << 28:
            c["count"], c["high"] = c["count"] * 2 // 3 + 1, c["high"] * 2 // 3 + 1
            c["seqs"] = c["seqs"] * 3 // 4 + 1 if c["seqs"] > 1 else 1
        c["ragged"], c["low"] = rng.random() < 0.6, rng.choice([0, 0, c["high"]])
    return c


def _lengths(c):
    """Host arrays that follow from the case alone: per sequence what it holds before the call, and its new tokens."""
    r = np.random.RandomState(c["lens_seed"] % (1 << 31))
    n = c["seqs"]
    if c.get("zipf"):
        before = np.clip(r.zipf(1.1, size=n), max(1, c["low"]), max(1, c["high"])).astype(np.int64)
    else:
        before = r.randint(c["low"], c["high"] + 1, size=n).astype(np.int64)
    if c["kind"] == "decode":
        if n > 2 and c["low"] == 0:
            before[n // 2] = 0  # a slot of the batch that holds no sequence
        return before, np.ones(n, np.int64)
    if c["kind"] == "prefill":
        new = r.randint(1, c["count"] + 1, size=n).astype(np.int64) if c["ragged"] else np.full(n, c["count"], np.int64)
        return before, new
    new = r.multinomial(c["rows"] - n, r.dirichlet(np.ones(n))) + 1 if c["rows"] > n else np.ones(n, np.int64)
    return before, new.astype(np.int64)


def _tile_bytes(dim):
    return 2 * 16 * (dim // 2 + dim // GROUP * 4)


def work(c):
    before, new = _lengths(c)
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    token4 = _tile_bytes(d) // 16 * hk  # bytes of one token, keys and values, all kv-heads
    if c["kind"] == "append":
        rows, size = c["rows"] - c["pad"], 4 if c["rows_type"] == "f32" else 2
        token = token4 if c["bits"] == 4 else 2 * hk * d * c["bits"] // 8
        # rows in, rotated queries and cache rows out, one table row per row, its place; a 4-bit cache's rows are read back
        total = rows * ((hq + 2 * hk) * d * size + hq * d * size + token + c["rotary"] * 4 + 12)
        if c["bits"] == 4:
            total += rows * (token4 + 2 * hk * d * 2 + 12)
        return {"bytes": total, "flops": rows * (hq + hk) * c["rotary"] * 3}
    if c["kind"] == "decode":
        ctx, queries, pairs = before, int((before >= 0).sum()), int(before.sum())
    else:
        ctx, queries, pairs = before + new, int(new.sum()), int((before * new + new * (new + 1) // 2).sum())
    tables = int(((ctx + c["block"] - 1) // c["block"]).sum()) * 4
    return {"bytes": int(ctx.sum()) * token4 + 2 * queries * hq * d * 2 + tables + 12 * len(ctx), "flops": 4 * d * hq * pairs}


# ----------------------------------------------------------------------------------------------- the packed cache's layout
def _places(dim):
    """Byte of (token, dim) among a tile's codes, and its shift, for keys [0] and values [1]; both [16][dim] / [dim]."""
    t, d = np.arange(16)[:, None], np.arange(dim)[None, :]
    nibble = (d & 7) >> 1
    key = t * (dim // 2) + ((d >> 3) & 3) * (dim // 8) + (d >> 5) * 4 + nibble
    chunk = (d >> 3) & 7
    if dim == 128:
        chunk = chunk ^ (((t >> 1) & 1) * 4)
    value = t * (dim // 2) + chunk * (dim // 16) + (d >> 6) * 4 + nibble
    value = value + 16 * (dim // 2 + dim // GROUP * 4)
    return key, value, (np.arange(dim) & 1) * 4


def _parameters(dim):
    """Byte of the (scale, zero) pairs of a token, [16][groups], for keys and for values."""
    at = (np.arange(16)[:, None] * (dim // GROUP) + np.arange(dim // GROUP)[None, :]) * 4
    return 16 * (dim // 2) + at, _tile_bytes(dim) // 2 + 16 * (dim // 2) + at


def _layout(dim):
    key, value, shift = _places(dim)
    kp, vp = _parameters(dim)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    return {"codes": (dev(key), dev(value)), "shift": dev(shift.astype(np.uint8)), "params": (dev(kp), dev(vp))}


def _quantise(x):
    """float32 rows [..., dim] of the row type's values -> codes (uint8), scale and zero (float16, [..., groups])."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    scale = ((high - low) / 15).to(torch.float16)
    s = scale.float()
    zero = (low + 8 * s).to(torch.float16)
    inverse = torch.where(s > 0, 1 / s, torch.zeros_like(s))
    codes = ((g - zero.float()[..., None]) * inverse[..., None]).round().add(8).clamp(0, 15).to(torch.uint8)
    return codes.flatten(-2), scale, zero


def _pair_bytes(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _param_bytes(scale, zero):
    return torch.stack([scale, zero], -1).flatten(-2).contiguous().view(torch.uint8)


def _write_rows(cache, lay, block, sub, slot, keys, values):
    """Puts quantised rows [n][kv_heads][dim] (float32) at (block, 16-token tile, slot) of a packed cache."""
    heads = torch.arange(cache.shape[1], device=DEV)[None, :, None]
    b, s = block[:, None, None], sub[:, None, None]
    for which, x in enumerate((keys, values)):
        codes, scale, zero = _quantise(x)
        at = lay["codes"][which][slot][:, None, 0::2]
        cache[b, heads, s, at] = _pair_bytes(codes)
        at = (lay["params"][which][slot][:, :, None] + torch.arange(4, device=DEV)).flatten(1)[:, None, :]
        cache[b, heads, s, at] = _param_bytes(scale, zero)


def _read_tiles(tiles, lay, which):
    """Tiles [..., tile] -> the values they stand for, float32 [..., 16, dim]."""
    codes = (tiles[..., lay["codes"][which]] >> lay["shift"]) & 15
    at = lay["params"][which]
    pairs = tiles[..., at[..., None] + torch.arange(4, device=DEV)].contiguous().view(torch.float16).float()  # [..., 16, groups, 2]
    x = codes.float().sub_(8).unflatten(-1, (-1, GROUP))
    return x.mul_(pairs[..., 0:1]).add_(pairs[..., 1:2]).flatten(-2)


# --------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _tables(c, totals, seed):
    """Block tables dealt from a permutation of the pool; entries behind a sequence's last block name some other block."""
    need = (totals + c["block"] - 1) // c["block"]
    blocks, wide = max(1, int(need.sum())), max(1, int(need.max()))
    r = np.random.RandomState(seed % (1 << 31))
    perm = r.permutation(blocks).astype(np.int32)
    tables = r.randint(0, blocks, size=(len(need), wide)).astype(np.int32)
    first = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[first:first + n]
        first += n
    return torch.from_numpy(tables).to(DEV), blocks


def _filled_cache(c, blocks, seed):
    lay, d = _layout(c["dim"]), c["dim"]
    cache = torch.empty((blocks, c["kv_heads"], c["block"] // 16, _tile_bytes(d)), dtype=torch.uint8, device=DEV)
    flat, g = cache.view(-1, _tile_bytes(d)), _gen(seed, 7)
    step = max(1, (1 << 27) // (16 * d))
    for first in range(0, flat.shape[0], step):
        part = flat[first:first + step]
        for which in (0, 1):
            # keys lean to some dims, as rotated keys do; values carry a small offset per token
            x = torch.randn((part.shape[0], 16, d), generator=g, device=DEV)
            x = x * (1 + 2 * (torch.arange(d, device=DEV) % 16 == 3)) if which == 0 else x + 0.1 * torch.randn((part.shape[0], 16, 1), generator=g, device=DEV)
            codes, scale, zero = _quantise(x.to(TYPES[c["type"]]).float())
            part[:, lay["codes"][which][:, 0::2].flatten()] = _pair_bytes(codes).flatten(1)
            at = (lay["params"][which][..., None] + torch.arange(4, device=DEV)).flatten()
            part[:, at] = _param_bytes(scale, zero).flatten(1)
    return cache


def _pool(c, bits, blocks):
    from inferlab_b200 import CudaKvPool

    dtype = KV_TYPES["f32" if bits == 32 else c["type"]]
    more = {"kv_bits": 4} if bits == 4 else {}
    return CudaKvPool(0, dtype, blocks, c["block"], c["kv_heads"], c["dim"], **more)


def prepare(case, seed):
    c = dict(case)
    before, new = _lengths(c)
    s = {"case": c}
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)  # noqa: E731
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    g = _gen(seed, 3)
    if c["kind"] == "append":
        totals = before + new
        s["tables"], blocks = _tables(c, totals, seed)
        rows_of = np.repeat(np.arange(c["seqs"]), new)
        positions = np.concatenate([b + np.arange(n) for b, n in zip(before, new)])
        if c["pad"]:  # the last rows of the batch hold no token
            rows_of[c["rows"] - c["pad"]:], positions[c["rows"] - c["pad"]:] = -1, 0
        s["seqs"], s["positions"] = i32(rows_of), i32(positions)
        # one projection's output holds the queries, keys and values of a token side by side
        qkv = torch.randn((c["rows"], hq + 2 * hk, d), generator=g, device=DEV).to(TYPES[c["rows_type"]])
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        angle = torch.arange(int(totals.max()), device=DEV, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(c["rotary"] // 2, device=DEV, dtype=torch.float64) * 2 / c["rotary"])
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["q_out"] = torch.zeros((c["rows"], hq, d), dtype=TYPES[c["rows_type"]], device=DEV)
        if c["bits"] == 4:
            s["cache"], s["layout"] = _filled_cache(c, blocks, seed), _layout(d)
        else:
            kind = TYPES["f32" if c["bits"] == 32 else c["type"]]
            s["keys"], s["values"] = (torch.randn((blocks, hk, c["block"], d), generator=g, device=DEV).to(kind) for _ in range(2))
        if own:
            s["pool"] = _pool(c, c["bits"], blocks)
            if c["bits"] == 4:
                s["pool"].arena.copy_(s["cache"])
            else:
                s["pool"].key_arena.copy_(s["keys"])
                s["pool"].value_arena.copy_(s["values"])
        return s
    totals = before if c["kind"] == "decode" else before + new
    s["tables"], blocks = _tables(c, totals, seed)
    s["cache"], s["layout"], s["longest"] = _filled_cache(c, blocks, seed), _layout(d), max(1, int(totals.max()))
    if c["kind"] == "decode":
        s["lens"] = i32(before)
        queries = c["seqs"]
    else:
        s["starts"], s["counts"], s["most"] = i32(before), i32(new), int(new.max())
        s["offsets"] = i32(np.concatenate([[0], np.cumsum(new)[:-1]]))
        queries = int(new.sum())
    s["q"] = torch.randn((queries, hq, d), generator=g, device=DEV).to(TYPES[c["type"]])
    if own:
        s["pool"] = _pool(c, 4, blocks)
        s["pool"].arena.copy_(s["cache"])
    return s


# ----------------------------------------------------------------------------------------------------------- one pass
def _rotate(x, cos, sin, interleaved):
    """float32 [rows][heads][dim]; cos and sin [rows][rotary / 2]."""
    half = cos.shape[-1]
    cos, sin, turned, rest = cos[:, None], sin[:, None], x[..., :2 * half], x[..., 2 * half:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([c, d], -1).flatten(-2) if interleaved else torch.cat([c, d], -1)
    return torch.cat([turned, rest], -1)


def _plain_append(s):
    c = s["case"]
    live = torch.nonzero(s["seqs"] >= 0).flatten()
    seq, pos = s["seqs"][live].long(), s["positions"][live].long()
    row_type = TYPES["f32" if c["bits"] == 32 else c["type"]]
    cos, sin = s["cos_sin"][pos].chunk(2, -1)
    s["q_out"][live] = _rotate(s["q"][live].float(), cos, sin, c["interleaved"]).to(s["q_out"].dtype)
    keys = _rotate(s["k"][live].float(), cos, sin, c["interleaved"]).to(row_type)
    values = s["v"][live].to(row_type)
    block, slot = s["tables"][seq, pos // c["block"]].long(), pos % c["block"]
    if c["bits"] != 4:
        s["keys"][block, :, slot], s["values"][block, :, slot] = keys, values
        return s["q_out"], s["keys"], s["values"]
    _write_rows(s["cache"], s["layout"], block, slot // 16, slot % 16, keys.float(), values.float())
    tiles = s["cache"][block, :, slot // 16]
    at = torch.arange(len(live), device=DEV)
    back = [_read_tiles(tiles, s["layout"], which)[at, :, slot % 16].to(row_type) for which in (0, 1)]
    return s["q_out"], back[0], back[1]


def _plain_attention(s, q, first):
    """q [seqs][most][q_heads][dim] float32; query i of sequence n sees keys 0 .. first[n] + i (none where that is below 0)."""
    c, longest = s["case"], s["longest"]
    n, most, hq, d = q.shape
    hk, blocks = c["kv_heads"], (longest + c["block"] - 1) // c["block"]
    tiles = s["cache"][s["tables"][:, :blocks].long()].transpose(1, 2)  # [seqs][kv_heads][blocks][block / 16][tile]
    keys = _read_tiles(tiles, s["layout"], 0).flatten(2, 4)[:, :, :longest]
    q = q.view(n, most, hk, hq // hk, d).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [seqs][kv_heads][most * group][dim]
    scores = q @ keys.transpose(-1, -2) * (1 / math.sqrt(d))
    del keys
    last = (first[:, None] + torch.arange(most, device=DEV)).repeat_interleave(hq // hk, 1)
    seen = torch.arange(longest, device=DEV) <= last[:, None, :, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = (scores - torch.where(top > -math.inf, top, 0)).exp()
    values = _read_tiles(tiles, s["layout"], 1).flatten(2, 4)[:, :, :longest]
    out = weights @ values / weights.sum(-1, keepdim=True).clamp_min(1e-30)
    return out.view(n, hk, most, hq // hk, d).transpose(1, 2).reshape(n, most, hq, d)


def _plain_decode(s):
    return _plain_attention(s, s["q"].float()[:, None], s["lens"].long() - 1)[:, 0].to(s["q"].dtype)


def _plain_prefill(s):
    rows = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(s["offsets"].long(), rows, right=True) - 1
    at = rows - s["offsets"].long()[seq]
    q = torch.zeros((s["case"]["seqs"], s["most"], *s["q"].shape[1:]), device=DEV)
    q[seq, at] = s["q"].float()
    return _plain_attention(s, q, s["starts"].long())[seq, at].to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[c["kind"]](s)
    pool = s["pool"]
    if c["kind"] == "append":
        q = pool.append_rotary(s["q"], s["k"], s["v"], s["cos_sin"], s["seqs"], s["positions"], s["tables"], interleaved=c["interleaved"],
                               q_out=s["q_out"])
        if c["bits"] != 4:
            return q, pool.key_arena, pool.value_arena
        live = c["rows"] - c["pad"]
        return (q, *pool.gather_rows(s["seqs"][:live], s["positions"][:live], s["tables"]))
    if c["kind"] == "decode":
        return pool.decode(s["q"], s["tables"], s["lens"], s["longest"])
    return pool.prefill(s["q"], s["tables"], s["starts"], s["counts"], s["offsets"], s["most"], max_context_len=s["longest"])


# ------------------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_rows(cache, table, length, dim):
    """Values a packed cache stands for: one sequence's keys and values, float64 [kv_heads][length][dim]."""
    per = cache.shape[2] * 16
    blocks = cache[table[:(length + per - 1) // per].long()].permute(1, 0, 2, 3).flatten(1, 2)  # [kv_heads][tiles][tile]
    heads, tiles, half, groups = blocks.shape[0], blocks.shape[1], dim // 2, dim // GROUP
    got = []
    for which in (0, 1):
        part = blocks[..., which * blocks.shape[-1] // 2:(which + 1) * blocks.shape[-1] // 2]
        raw = part[..., :16 * half].reshape(heads, tiles, 16, half)
        params = part[..., 16 * half:].contiguous().view(torch.float16).double().view(heads, tiles, 16, groups, 2)
        x = torch.empty((heads, tiles, 16, dim), dtype=torch.float64, device=cache.device)
        for d0 in range(0, dim, 8):  # eight dims share one 32-bit word
            for odd in (0, 1):  # tokens 2, 3 of four keep a 128-dim value row's halves swapped
                word = ((d0 // 8) % 4 * (dim // 32) + d0 // 32) if which == 0 else ((d0 // 8) % 8 ^ (4 * odd if dim == 128 else 0)) * groups + d0 // 64
                rows = [t for t in range(16) if (t // 2) % 2 == odd]
                bytes4 = raw[:, :, rows][..., 4 * word:4 * word + 4].long()
                for k in range(8):
                    code = bytes4[..., k // 2] // (16 if k % 2 else 1) % 16
                    pair = params[:, :, rows, (d0 + k) // GROUP]
                    x[:, :, rows, d0 + k] = pair[..., 1] + (code.double() - 8) * pair[..., 0]
        got.append(x.flatten(1, 2)[:, :length])
    return got


def _exact_attention(q, keys, values, first):
    """q [count][q_heads][dim], keys and values [kv_heads][length][dim], all float64; query i sees keys 0 .. first + i."""
    count, hq, d = q.shape
    hk, length, _ = keys.shape
    out = torch.zeros_like(q)
    for h in range(hq if length else 0):
        score = q[:, h] @ keys[h // (hq // hk)].T / d ** 0.5
        score.masked_fill_(torch.arange(length, device=q.device) > first + torch.arange(count, device=q.device)[:, None], -math.inf)
        out[:, h] = torch.softmax(score, 1) @ values[h // (hq // hk)]
    return out


def _exact_turn(x, angle_row, interleaved):
    half = angle_row.shape[-1] // 2
    out, cos, sin = x.clone(), angle_row[:, None, :half], angle_row[:, None, half:]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., second] * cos + x[..., first] * sin
    return out


def _exact_held(x, row_type):
    """What a 4-bit cache holds of rows x (float64): the values, float64."""
    x = x.to(row_type).double().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / 15).half().double()
    zero = (low + 8 * scale).half().double()
    code = torch.where(scale > 0, torch.round((x - zero) / scale.clamp_min(1e-9)), 0).clamp(-8, 7)
    return (zero + code * scale).flatten(-2)


def exact(case, seed):
    global own
    kept, own = own, False
    s = prepare(case, seed)
    own = kept
    c = s["case"]
    before, new = _lengths(c)
    if c["kind"] == "append":
        live = c["rows"] - c["pad"]
        seq, pos = s["seqs"][:live].long(), s["positions"][:live].long()
        turn = s["cos_sin"].double()[pos]
        q = torch.zeros_like(s["q_out"], dtype=torch.float64)
        q[:live] = _exact_turn(s["q"][:live].double(), turn, c["interleaved"])
        keys, values = _exact_turn(s["k"][:live].double(), turn, c["interleaved"]), s["v"][:live].double()
        if c["bits"] == 4:
            return q, _exact_held(keys, TYPES[c["type"]]), _exact_held(values, TYPES[c["type"]])
        whole_k, whole_v = s["keys"].double(), s["values"].double()
        block = s["tables"].long()[seq, torch.div(pos, c["block"], rounding_mode="floor")]
        whole_k[block, :, pos % c["block"]], whole_v[block, :, pos % c["block"]] = keys, values
        return q, whole_k, whole_v
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), 0
    for i in range(c["seqs"]):
        length, count = int(before[i] + (new[i] if c["kind"] == "prefill" else 0)), int(new[i])
        keys, values = _exact_rows(s["cache"], s["tables"][i], length, c["dim"])
        out[at:at + count] = _exact_attention(s["q"][at:at + count].double(), keys, values, int(before[i]) - (c["kind"] == "decode"))
        at += count
    return out
