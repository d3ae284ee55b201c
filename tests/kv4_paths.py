"""Attention over the 4-bit cache by each of its ways, in 64 bits with the roundings that the way makes of keys and values, and how far a
kernel of that way may be from it.

* "direct": keys as codes, scales and minima (nothing rounded); values s c + m in float16 after a power of two that follows the largest
  magnitude, 2^14 at most, which is brought to 2^10 at least; probabilities in float16, 2^7 over the reference.
* "half": keys and values in float16 after a power of two that brings the largest magnitude that a (request, kv head) sees to 2^13..2^14;
  probabilities in float16, 2^7 over the reference.
* "bfloat16": keys, values and probabilities in bfloat16.
* "float32": float32 arithmetic throughout."""
import numpy as np
import torch

import kv4_cases as kc


class Rows:
    """A pool with the given rows (lists over requests of [n, kv heads, hd] float32; not-a-number: a group that holds nothing), pages in no
    order, and in every row that belongs to nobody pairs that are not numbers."""

    def __init__(self, k, v, page_size=16, device="cuda:0", seed=0, spare=2):
        rng = np.random.default_rng(seed)
        self.page_size, self.k, self.v, self.lens = page_size, k, v, [len(x) for x in k]
        self.nkv, self.hd = k[0].shape[1:]
        counts = [-(-n // page_size) for n in self.lens]
        total = sum(counts) + spare
        order = rng.permutation(total)
        self.table = np.full((len(k), max(counts + [1]) + 1), -1, np.int32)
        rows = np.full((2, total, self.nkv, page_size, self.hd), np.nan, np.float32)
        at = 0
        for b, n in enumerate(self.lens):
            for j in range(counts[b]):
                page = self.table[b, j] = int(order[at])
                at += 1
                lo, hi = j * page_size, min(n, (j + 1) * page_size)
                rows[0, page, :, :hi - lo], rows[1, page, :, :hi - lo] = k[b][lo:hi].transpose(1, 0, 2), v[b][lo:hi].transpose(1, 0, 2)
        packed = [kc.pack(r.reshape(total, self.nkv, page_size // 16, 16, self.hd), values) for r, values in zip(rows, (False, True))]
        self.k_cache, self.v_cache = (torch.from_numpy(p).to(device) for p in packed)


def random_rows(seed, lens, nkv, hd, k_spread=1.0, v_spread=1.0):
    rng = np.random.default_rng(seed)
    k = [rng.standard_normal((n, nkv, hd)).astype(np.float32) * np.float32(k_spread) for n in lens]
    v = [(rng.standard_normal((n, nkv, hd)) + 0.25 * rng.standard_normal((nkv, hd))).astype(np.float32) * np.float32(v_spread) for n in lens]
    return k, v


def stored(x):
    """(what rows [n, kv heads, hd] stand for in float64, the same with |minimum| and the group's largest magnitude in it)."""
    code, s, m = kc.quantise(x)
    c = code.reshape(s.shape + (32,)).astype(np.float64)
    s, m = s[..., None].astype(np.float64), m[..., None].astype(np.float64)
    most = np.maximum(np.abs(m), np.abs(m + 15 * s))
    return ((s * c + m).reshape(x.shape), (s * c + np.abs(m)).reshape(x.shape), np.broadcast_to(most, c.shape).reshape(x.shape))


def as_bfloat16(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).double().numpy()


def as_half(x, most):
    """x [n, kv heads, hd] in float16 times the power of two of each kv head's largest magnitude."""
    top = np.nanmax(most.transpose(1, 0, 2).reshape(x.shape[1], -1), axis=1, initial=0.0)
    by = 2.0 ** (13 - np.clip(np.floor(np.log2(np.maximum(top, 1e-300))), -113, 127))[:, None]
    return (x * by).astype(np.float32).astype(np.float16).astype(np.float64) / by


def way_of(rows, q_len, heads, dtype, scale, simple=False, direct_rows=128):
    if simple or dtype == torch.float32 or (q_len * (heads // rows.nkv) > direct_rows and not scale > 0):
        return "float32"
    if q_len * (heads // rows.nkv) <= direct_rows:
        return "direct"
    return "half" if rows.hd in (64, 128) and heads // rows.nkv <= 128 and (128 % rows.page_size == 0 or rows.page_size % 128 == 0) else "bfloat16"


def expected(rows, b, q, scale, window, way, dtype):
    """(output [n, heads, hd] of the last n positions of request b, its tolerance)."""
    n, heads, hd = q.shape
    L, G = rows.lens[b], rows.nkv
    lo_all = max(0, L - n - window + 1) if window else 0
    with np.errstate(invalid="ignore"):
        (k, k_terms, k_most), (v, _, v_most) = (stored(x[b][lo_all:]) for x in (rows.k, rows.v))
        kr = {"half": lambda: as_half(k, k_most), "bfloat16": lambda: as_bfloat16(k)}.get(way, lambda: k)()
        vr = {"half": lambda: as_half(v, v_most), "bfloat16": lambda: as_bfloat16(v)}.get(way, lambda: v)()
    out, tol = np.zeros((n, heads, hd)), np.zeros((n, heads, hd))
    # roundings of a score, in units of 2^-23 of the sum of its terms' magnitudes: a group's 32 products, the groups' and the sum of the minima's;
    # or hd products; and the factors' roundings beside
    steps = 64 + hd // 32 if way == "direct" else hd + 16
    # the rounding of a probability, and of a value where it is not in vr
    weight = {"direct": 2.0 ** -10, "half": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -23}[way]
    least = np.nanmax(v_most.transpose(1, 0, 2).reshape(G, -1), axis=1, initial=0.0) * 2.0 ** -34 if way == "direct" else np.zeros(G)      # a value's absolute rounding
    for i in range(n):
        pos = L - n + i
        lo, hi = (max(0, pos - window + 1) if window else 0) - lo_all, pos + 1 - lo_all
        if hi <= lo:
            continue
        for h in range(heads):
            g, qi = h // (heads // G), np.asarray(q[i, h], np.float64)
            z = kr[lo:hi, g] @ qi * scale
            terms = (np.abs(k_terms if way == "direct" else kr)[lo:hi, g] @ np.abs(qi)).max() * abs(scale)
            w = np.exp(z - z.max())
            w /= w.sum()
            vv = vr[lo:hi, g]
            out[i, h] = w @ vv
            A, d = w @ np.abs(vv), terms * steps * 2.0 ** -23
            # errors up to d in the scores move a probability by a factor within exp(-2 d)..exp(2 d); exponentials 2^-20; sums over the keys
            tol[i, h] = A * (np.expm1(min(2 * d, 5)) + weight + 2.0 ** -20 + (hi - lo + 16) * 2.0 ** -23)
            # A probability under the smallest normal float32 is none; in float16, 2^7 over the reference, steps are 2^-24 under 2^-14.
            tol[i, h] += (hi - lo) * (2.0 ** -32 if way in ("half", "direct") else 2.0 ** -126) * np.abs(vv).max(0) + least[g]
    return out, tol + np.abs(out) * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23) + (2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -140)


def attend(ops, rows, q, q_lens, heads, window=None, scale=None, simple=False, runs=True, device="cuda:0", out=None, **more):
    """The operator's call over the last q_lens positions of the requests; q [T, heads * hd] on the device."""
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=device)      # noqa: E731
    out = torch.full_like(q, 7.0) if out is None else out
    positions = np.concatenate([np.arange(n - m, n) for n, m in zip(rows.lens, q_lens)])
    kw = dict(cu_q=i32(np.concatenate([[0], np.cumsum(q_lens)])), kv_lens=i32(rows.lens), q_lens=list(q_lens), max_kv_len=max(rows.lens)) if runs else {}
    ops.attention_kv4_rows(q, out, rows.k_cache, rows.v_cache, i32(rows.table), i32(np.repeat(np.arange(len(q_lens)), q_lens)), i32(positions), heads,
                           rows.nkv, rows.hd, rows.page_size, window, rows.hd ** -0.5 if scale is None else scale, force_simple=simple, **{**kw, **more})
    return out


def check(rows, q, out, q_lens, heads, dtype, window=None, scale=None, simple=False, direct_rows=128):
    scale = rows.hd ** -0.5 if scale is None else scale
    got, qh = out.double().cpu().numpy(), q.double().cpu().numpy().reshape(-1, heads, rows.hd)
    at = 0
    for b, n in enumerate(q_lens):
        if n:
            way = way_of(rows, n, heads, dtype, scale, simple, direct_rows)
            want, tol = expected(rows, b, qh[at:at + n], scale, window, way, dtype)
            x = got[at:at + n].reshape(want.shape)
            assert np.isfinite(x).all(), f"request {b}, {way}: {int((~np.isfinite(x)).sum())} of {x.size} not finite"
            err = np.abs(x - want)
            assert (err <= tol).all(), f"request {b}, {way}: {float((err / tol).max()):.2f} of the bound"
        at += n
