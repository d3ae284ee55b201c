"""The 4-bit cache without a GPU: calls without the module that checks operands, and the bounds of its attention (what a way's own roundings
give lies inside, a way that loses more lies outside)."""
import numpy as np
import pytest
import torch

import kv4_paths as kp
from coheryn_ai_studio_b200 import ops


def rounded_output(rows, q, keys, values, probabilities, dtype=torch.bfloat16):
    """A way's answer from its parts: ``keys``, ``values`` and ``probabilities`` say how those are rounded; float64 elsewhere, one rounding at the end."""
    n, heads, hd = q.shape
    (k, _, k_most), (v, _, v_most) = (kp.stored(x[0]) for x in (rows.k, rows.v))
    half = lambda x: (x * 128).astype(np.float32).astype(np.float16).astype(np.float64) / 128      # noqa: E731
    k = {"exact": lambda: k, "half": lambda: kp.as_half(k, k_most), "bfloat16": lambda: kp.as_bfloat16(k)}[keys]()
    v = kp.as_half(v, v_most) if values == "half" else kp.as_bfloat16(v)
    out = np.zeros(q.shape)
    for i in range(n):
        for h in range(heads):
            z = k[:rows.lens[0] - n + i + 1, 0] @ q[i, h] * hd ** -0.5
            p = np.exp(z - z.max())
            used = {"half": half, "bfloat16": kp.as_bfloat16}[probabilities](p)
            out[i, h] = used @ v[:len(p), 0] / p.sum()
    return torch.from_numpy(out).to(dtype).double().numpy()


# Lost bits of a key show where scores are large, those of a probability where few keys meet (and their values may cancel).
@pytest.mark.parametrize("way,keys,values,probabilities,spread,context,inside", [
    ("direct", "exact", "half", "half", 6.0, 700, True), ("direct", "exact", "half", "half", 1.0, 12, True), ("direct", "bfloat16", "half", "half", 6.0, 700, False),
    ("direct", "exact", "bfloat16", "half", 1.0, 12, False),
    ("half", "half", "half", "half", 6.0, 700, True), ("half", "half", "half", "half", 1.0, 12, True), ("half", "bfloat16", "half", "half", 6.0, 700, False),
    ("half", "half", "bfloat16", "half", 1.0, 12, False), ("half", "half", "half", "bfloat16", 1.0, 12, False),
    ("bfloat16", "bfloat16", "bfloat16", "bfloat16", 1.0, 700, True)])
def test_a_bound_holds_for_its_way_alone(way, keys, values, probabilities, spread, context, inside):
    k, v = kp.random_rows(1, [context], 1, 64, k_spread=spread)
    rows = kp.Rows(k, v, device="cpu")
    q = kp.as_bfloat16(np.random.default_rng(2).standard_normal((12, 4, 64)) * (8.0 if spread > 1 else 1.5))
    want, tol = kp.expected(rows, 0, q, 64 ** -0.5, None, way, torch.bfloat16)
    err = np.abs(rounded_output(rows, q, keys, values, probabilities) - want)
    assert bool((err <= tol).all()) == inside, float((err / tol).max())


def test_rows_come_through_the_pool():
    """The pool's bytes stand for the rows that the bounds are formed from."""
    import kv4_cases as kc
    k, v = kp.random_rows(3, [40, 17], 2, 96)
    rows = kp.Rows(k, v, 32, device="cpu")
    for cache, values, x in ((rows.k_cache, False, k), (rows.v_cache, True, v)):
        held = kc.cache_rows(cache.numpy(), values)
        for b, n in enumerate(rows.lens):
            got = held[[p for p in rows.table[b] if p >= 0]].transpose(0, 2, 1, 3).reshape(-1, 2, 96)
            assert np.array_equal(got[:n], kp.stored(x[b])[0]) and np.isnan(got[n:]).all()


def test_without_the_module_of_checked_calls(monkeypatch):
    """A machine without the headers that it needs runs the calls from Python, and says so once."""
    import warnings
    from coheryn_ai_studio_b200.csrc import build

    def missing():
        raise build.BuildError("the module of checked calls did not compile:\nPython.h: No such file or directory")
    monkeypatch.setattr(build, "calls_module", missing)
    monkeypatch.setattr(ops, "_calls_module", None)
    with pytest.warns(RuntimeWarning, match="checked calls"):
        calls = ops._calls()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert all(getattr(ops._calls(), n)(1, 2, 3) is None for n in ("layout", "write", "pages", "attention"))
    assert ops._calls() is calls
