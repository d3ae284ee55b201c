"""The 4-bit cache restated on the CPU from its definition, place by place, and attention over it in 64 bits.

A tile of 16 positions of one kv head is 10 * hd bytes.  Keys: the 4 bits of row r, channel c = 32 u + 8 t + i lie in word
r * 4 NG + t * NG + u (NG = hd / 32), at place i; the pair (scale, minimum) of (r, u) behind the codes.  Values: row r =
4 t + 2 p + e, channel c = 32 u + 4 g + j: word ((u * 8 + g) * 4 + t) * 2 + p, place 4 e + j; the scales of rows 4 t..4 t + 3
of group u, then their minima."""
import numpy as np
import torch


def places(hd, values):
    """Of every (row, channel) of a tile: its 4-bit place, and the byte offsets of its scale and its minimum."""
    r, c = np.meshgrid(np.arange(16), np.arange(hd), indexing="ij")
    ng, u = hd // 32, c // 32
    if not values:
        t, i = (c % 32) // 8, c % 8
        scale = 8 * hd + (r * ng + u) * 4
        return (r * 4 * ng + t * ng + u) * 8 + i, scale, scale + 2
    g, j, t, p, e = (c % 32) // 4, c % 4, r // 4, (r % 4) // 2, r % 2
    scale = 8 * hd + ((u * 4 + t) * 8 + r % 4) * 2
    return (((u * 8 + g) * 4 + t) * 2 + p) * 8 + 4 * e + j, scale, scale + 8


def bf16(x):
    """float32 values rounded to bfloat16, as float32."""
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).float().numpy()


def bits16(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)


def quantise(x):
    """(codes, scale, minimum) of rows [..., hd] float32, the last two [..., hd / 32] float32."""
    x = np.asarray(x, np.float32)
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        s, m = bf16((hi - lo) / np.float32(15)), bf16(lo)
        bad = ~(np.isfinite(g).all(-1) & np.isfinite(s) & np.isfinite(m))
        code = np.clip(np.rint((g - m[..., None]) / np.where(s > 0, s, 1)[..., None]), 0, 15)
        code = np.where(((s > 0) & ~bad)[..., None], code, 0).astype(np.uint8)
    s, m = np.where(bad, np.nan, s).astype(np.float32), np.where(bad, np.nan, m).astype(np.float32)
    return code.reshape(x.shape), s, m


def pack(x, values):
    """Tiles of bytes from rows [..., 16, hd] float32."""
    hd = x.shape[-1]
    code, s, m = quantise(x)
    out = np.zeros(x.shape[:-2] + (10 * hd,), np.uint8)
    nib, at_s, at_m = places(hd, values)
    flat = code.reshape(x.shape[:-2] + (-1,))
    order = nib.reshape(-1)
    inverse = np.empty_like(order)
    inverse[order] = np.arange(order.size)
    by_place = flat[..., inverse]
    out[..., :8 * hd] = by_place[..., 0::2] | by_place[..., 1::2] << 4
    for at, v in ((at_s, s), (at_m, m)):
        w, first = bits16(v).reshape(x.shape[:-2] + (-1,)), at[:, ::32].reshape(-1)
        w = np.where(np.isnan(v).reshape(w.shape), np.uint16(0x7fff), w)
        out[..., first], out[..., first + 1] = w & 255, w >> 8
    return out


def unpack(tiles, values):
    """float64 rows [..., 16, hd] of tiles [..., 10 hd]."""
    tiles = np.asarray(tiles)
    hd = tiles.shape[-1] // 10
    nib, at_s, at_m = places(hd, values)
    code = (tiles[..., nib // 2] >> (4 * (nib % 2))) & 15
    wide = lambda at: ((tiles[..., at + 1].astype(np.uint32) << 24) | (tiles[..., at].astype(np.uint32) << 16)).view(np.float32)  # noqa: E731
    with np.errstate(invalid="ignore"):
        return code * wide(at_s).astype(np.float64) + wide(at_m).astype(np.float64)


def cache_rows(cache, values):
    """float64 [pages, kv heads, page_size, hd] of a cache [pages, kv heads, tiles, 10 hd] (numpy)."""
    x = unpack(cache, values)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def attend(q, k, v, first_pos, scale, window=None):
    """In 64 bits: q [n, H, hd] at positions first_pos.., k and v [L, G, hd].  Returns (output [n, H, hd], the same with |v|,
    the largest sum of |q k| scale of a row [n, H])."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, H, hd = q.shape
    L, G = k.shape[:2]
    out, mass, most = np.zeros((n, H, hd)), np.zeros((n, H, hd)), np.zeros((n, H))
    for i in range(n):
        pos = first_pos + i
        lo, hi = (max(0, pos - window + 1) if window else 0), min(pos + 1, L)
        if hi <= lo:
            continue
        for h in range(H):
            g = h // (H // G)
            s = k[lo:hi, g] @ q[i, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h], mass[i, h] = w @ v[lo:hi, g], w @ np.abs(v[lo:hi, g])
            most[i, h] = (np.abs(k[lo:hi, g]) @ np.abs(q[i, h])).max() * abs(scale)
    return out, mass, most


def bound(out, mass, most, hd, keys, dtype, rounded_keys=False):
    """How far a kernel may be from ``attend``.  With A = sum of p |v| (``mass``): a probability and a value that enter a product in
    bfloat16 are each off by at most 2^-8 of themselves (A 2^-7 together), the output by 2^-8 of itself; a score summed in float32
    from hd products is off by at most (hd + 8) 2^-23 of sum |q k| (twice the products' roundings; sums that go through 1024 + code in
    the place of a code, about 7.5 from a group's middle: 136 times, the share by which that raises the terms), by 2^-8 of it more where the keys were rounded to bfloat16;
    errors up to d in the scores move a probability by a factor within exp(-2 d)..exp(2 d); exponentials and the sums over the keys are off by 2^-21 and
    keys 2^-23 of A."""
    d = most * (hd + 8) * 2.0 ** -23 * (1 if dtype == torch.float32 else 136)
    if rounded_keys:
        d = d + most * 2.0 ** -8
    A = mass
    err = A * (np.expm1(np.minimum(2 * d, 5))[..., None] + 2.0 ** -21 + (keys + 16) * 2.0 ** -23)
    if dtype == torch.bfloat16:
        err = err + A * 2.0 ** -7 + np.abs(out) * 2.0 ** -8
    return err + np.abs(out) * 2.0 ** -23 + 1e-30
