"""Plain numpy statements of the 4-bit pool's format, the rotary append and attention over it.

Quantisation and rotation come in the working type given (float32 follows the kernels operation by operation, so bytes
can be compared; float64 is the definition), attention in float64 only.
"""
import numpy as np

GROUP = 64
TILE = 16


def bf16(x):
    """float32 values rounded to bfloat16 (nearest even), as float32."""
    bits = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    bits = (bits + 0x7FFF + ((bits >> 16) & 1)) & 0xFFFF0000
    return bits.astype(np.uint32).view(np.float32)


def round_to(x, kind):
    """Rounds to "f16", "bf16" or "f32"; float32 result."""
    x = np.asarray(x, np.float32)
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    return bf16(x) if kind == "bf16" else x


def rotate(x, angles, interleaved, work=np.float32):
    """x [rows][heads][dim], angles [rows][rotary] (cosines, then sines)."""
    x, angles = np.asarray(x, work), np.asarray(angles, work)
    half = angles.shape[-1] // 2
    if half == 0:
        return x.copy()
    out, cos, sin = x.copy(), angles[:, None, :half], angles[:, None, half:]
    a = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., b] * cos + x[..., a] * sin
    return out


def quantise(x):
    """x [..., dim] float32 of row-type values -> codes uint8, scale and zero float16 [..., dim / 64]."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, GROUP)
    low, high = g.min(-1), g.max(-1)
    scale = ((high - low) / np.float32(15)).astype(np.float16)
    s = scale.astype(np.float32)
    zero = (low + np.float32(8) * s).astype(np.float16)
    with np.errstate(divide="ignore"):
        inverse = np.where(s > 0, np.float32(1) / s, np.float32(0))
    steps = np.rint((g - zero.astype(np.float32)[..., None]) * inverse[..., None])
    return np.clip(steps + 8, 0, 15).astype(np.uint8).reshape(x.shape), scale, zero


def values_of(codes, scale, zero):
    """float64 values the codes stand for."""
    g = codes.reshape(*scale.shape, GROUP).astype(np.float64) - 8
    return (zero.astype(np.float64)[..., None] + g * scale.astype(np.float64)[..., None]).reshape(codes.shape)


def tile_bytes(dim):
    return 2 * TILE * (dim // 2 + dim // GROUP * 4)


def places(dim, value):
    """Byte and shift of (slot, dim)'s code and byte of (slot, group)'s pair within a tile."""
    half = tile_bytes(dim) // 2
    codes, shifts = np.empty((TILE, dim), np.int64), np.empty((TILE, dim), np.int64)
    for t in range(TILE):
        for d in range(dim):
            u = d // 8
            if value:
                word = ((u % 8) ^ (4 if dim == 128 and (t // 2) % 2 else 0)) * (dim // 16) + (u // 8) * 4
            else:
                word = (u % 4) * (dim // 8) + (u // 4) * 4
            codes[t, d] = (half if value else 0) + t * (dim // 2) + word + (d % 8) // 2
            shifts[t, d] = 4 * (d % 2)
    pairs = (half if value else 0) + TILE * (dim // 2) + \
        (np.arange(TILE)[:, None] * (dim // GROUP) + np.arange(dim // GROUP)) * 4
    return codes, shifts, pairs


def write_rows(arena, blocks, slots, keys, values):
    """Quantises rows [n][heads][dim] into a packed arena [blocks][heads][tiles][tile] (in place)."""
    dim = keys.shape[-1]
    for which, x in enumerate((keys, values)):
        at, shift, pair_at = places(dim, which)
        codes, scale, zero = quantise(x)
        pairs = np.stack([scale, zero], -1).view(np.uint8).reshape(*scale.shape, 4)
        for r in range(len(blocks)):
            t, s = divmod(int(slots[r]), TILE)
            for h in range(arena.shape[1]):
                tile = arena[blocks[r], h, t]
                tile[at[s, 0::2]] = codes[r, h, 0::2] | (codes[r, h, 1::2] << 4)
                for g in range(dim // GROUP):
                    tile[pair_at[s, g]:pair_at[s, g] + 4] = pairs[r, h, g]


def read_rows(arena, table, length, dim):
    """float64 keys and values [heads][length][dim] of one sequence."""
    per_block = arena.shape[2] * TILE
    table = np.asarray(table[:(length + per_block - 1) // per_block])
    tiles = arena[table].transpose(1, 0, 2, 3).reshape(arena.shape[1], -1, arena.shape[3])
    got = []
    for which in (0, 1):
        at, shift, pair_at = places(dim, which)
        codes = (tiles[..., at] >> shift.astype(np.uint8)) & 15
        pairs = np.ascontiguousarray(tiles[..., pair_at[..., None] + np.arange(4)]).view(np.float16)
        got.append(values_of(codes, pairs[..., 0], pairs[..., 1]).reshape(arena.shape[1], -1, dim)[:, :length])
    return got


def attend(q, keys, values, first):
    """float64 attention: q [count][q_heads][dim], query i sees keys 0 .. first + i. Returns the output, and per
    (query, head) the largest sum |q k| / sqrt(dim) and the largest |value| it sees, for error bounds."""
    count, q_heads, dim = q.shape
    heads, length, _ = keys.shape
    out = np.zeros((count, q_heads, dim))
    reach, size = np.zeros((count, q_heads)), np.zeros((count, q_heads))
    for h in range(q_heads):
        k, v = keys[h // (q_heads // heads)], values[h // (q_heads // heads)]
        for i in range(count):
            n = min(length, first + i + 1)
            if n <= 0:
                continue
            s = k[:n] @ q[i, h] / np.sqrt(dim)
            p = np.exp(s - s.max())
            out[i, h] = p @ v[:n] / p.sum()
            reach[i, h] = (np.abs(k[:n]) @ np.abs(q[i, h])).max() / np.sqrt(dim)
            size[i, h] = np.abs(v[:n]).max()
    return out, reach, size
