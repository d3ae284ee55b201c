"""The engine over a cache in 4 bits, against the plain implementation whose keys and values are quantised by the same
definition, and the step's arrays made on the device against those made on the host."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import kv4_cases as kc
import plain_qwen2 as plain
import tiny

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return tiny.make_folder(tmp_path_factory.mktemp("kv4"), "B", policy=tiny.POLICY_LOUD)


def held(x, kv_heads):
    """Rows [T, kv heads * hd] as a cache in 4 bits holds them."""
    rows = x.reshape(len(x), kv_heads, -1)
    c, s, m = kc.quantise(rows)
    return (c.reshape(c.shape[:-1] + (-1, 32)) * s[..., None].astype(np.float64) + m[..., None]).astype(np.float32).reshape(x.shape)


def plain_four_bits(cfg, w, ids, monkeypatch, rows=None):
    exact = plain.attention
    with monkeypatch.context() as m:
        m.setattr(plain, "attention", lambda q, k, v, heads, kv_heads, hd, window=None: exact(q, held(k, kv_heads), held(v, kv_heads), heads,
                                                                                              kv_heads, hd, window))
        return plain.forward(cfg, w, ids, rows=rows)


@pytest.mark.parametrize("graphs", [False, True])
def test_logits_follow_the_plain_model_with_quantised_rows(folder, graphs, monkeypatch):
    """float32, prompts cut into portions beside decoded tokens.  The engine's keys differ from the plain ones in the last bits, so a
    value next to a border between two codes may fall to either side, a step of that one value: the yardstick is what
    quantising all of them moves the logits by.  A wrong row or scale moves them by as much as that."""
    from coheryn_ai_studio_b200.engine import Engine, StepEntry
    cfg, w = plain.read_model(folder)
    eng = Engine.from_folder(folder, "float32", context=256, max_num_seqs=4, kv_bits=4, use_graphs=graphs)
    assert eng.cache.groups[0].tensor.dtype == torch.uint8 and eng.cache.bytes_per_token() == 3 * 1 * 2 * 32 * 5 // 8
    seqs = {"a": tiny.prompt(1, 150, 1000), "b": tiny.prompt(2, 60, 1000)}
    cuts = {"a": [0, 70, 71, 118] + list(range(119, 151)), "b": [0, 1, 2, 30] + list(range(31, 61))}
    for rid in seqs:
        eng.cache.admit(rid)
    got = {"a": {}, "b": {}}
    for i in range(max(len(c) for c in cuts.values()) - 1):
        entries = [StepEntry(r, seqs[r][c[i]:c[i + 1]], [c[i + 1] - c[i] - 1]) for r, c in cuts.items() if i + 1 < len(c)]
        logits = eng.runner.step(entries).cpu().numpy()
        for e, row in zip(entries, logits):
            got[e.request_id][cuts[e.request_id][i + 1] - 1] = row
    eng.runner.check_status()
    for r, ids in seqs.items():
        rows = sorted(got[r])
        want, full = plain_four_bits(cfg, w, ids, monkeypatch, rows), plain.forward(cfg, w, ids, rows=rows)
        yard = float(np.abs(want - full).max())
        d = np.array([np.abs(got[r][p] - want[i]).max() for i, p in enumerate(rows)])
        assert yard > 0.05 and np.median(d) < 2e-3 * yard and d.max() < 0.1 * yard, (yard, np.median(d), d.max())


def test_generation_in_both_types_and_lookahead(folder, monkeypatch):
    """Greedy tokens: float32 the plain model's with quantised rows (or a near-tie), and the same with and without graphs and steps
    launched ahead; bfloat16 runs whole prompts and decoding, its tokens near the plain choice."""
    from coheryn_ai_studio_b200.engine import Engine
    cfg, w = plain.read_model(folder)
    prompts = [tiny.prompt(5 + i, n, 1000) for i, n in enumerate((3, 90, 17))]
    outs = []
    for dtype, kw in (("float32", {}), ("float32", dict(lookahead=False, use_graphs=False)), ("bfloat16", {}), ("bfloat16", dict(max_num_batched_tokens=24))):
        eng = Engine.from_folder(folder, dtype, context=128, max_num_seqs=3, kv_bits=4, **kw)
        outs.append([r.token_ids for r in eng.generate(prompts, max_tokens=6)])
        assert eng.cache.available_pages() == [eng.cache.num_pages]
    assert outs[0] == outs[1]
    for dtype, tokens in zip(("float32", "float32", "bfloat16", "bfloat16"), outs):
        for p, toks in zip(prompts, tokens):
            ids = list(p)
            for t in toks:
                ref = plain_four_bits(cfg, w, ids, monkeypatch, rows=[len(ids) - 1])[0]
                full = plain.forward(cfg, w, ids, rows=[len(ids) - 1])[0]
                gap, yard = float(ref.max() - ref[t]), float(np.abs(ref - full).max())
                assert gap <= (0.2 if dtype == "float32" else 1.0) * yard + (0.0 if dtype == "float32" else 0.1 * float(np.std(ref))), (dtype, gap, yard)
                ids.append(t)


def test_prefix_reuse_over_pages_in_four_bits(folder):
    from coheryn_ai_studio_b200.engine import Engine
    eng = Engine.from_folder(folder, "float32", context=128, max_num_seqs=2, kv_bits=4)
    p = tiny.prompt(9, 70, 1000)
    first = eng.generate([p], max_tokens=4)[0]
    again = eng.generate([p], max_tokens=4)[0]
    assert again.reused_prompt_tokens == 64 and again.token_ids == first.token_ids


def test_models_and_sizes_that_do_not_read_four_bits_are_refused(folder, tmp_path):
    from coheryn_ai_studio_b200.engine import Engine
    with pytest.raises(ValueError, match="multiple of 16"):
        Engine.from_folder(folder, "bfloat16", context=64, page_size=8, kv_bits=4)
    with pytest.raises(ValueError, match="not in 8"):
        Engine.from_folder(folder, "bfloat16", context=64, kv_bits=8)
    with pytest.raises(ValueError, match="does not read a cache in 4 bits"):      # head size 16
        Engine.from_folder(tiny.make_folder(tmp_path, "A"), "bfloat16", context=64, kv_bits=4)


def test_command_line(folder):
    cmd = [sys.executable, os.path.join(ROOT, "bin", "coheryn"), "--json", "run", folder, "--tokens", "5,17,3", "--max-tokens", "4", "--context", "64",
           "--dtype", "float32", "--kv-bits", "4"]
    p = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr
    from coheryn_ai_studio_b200.engine import Engine
    eng = Engine.from_folder(folder, "float32", context=64, max_num_seqs=1, kv_bits=4)
    assert json.loads(p.stdout)["token_ids"] == eng.generate([[5, 17, 3]], max_tokens=4)[0].token_ids


# ------------------------------------------------------------------------------------ the step's arrays
@pytest.mark.parametrize("want", ["few", "all", "none"])
def test_step_arrays_from_the_device_are_those_of_the_host(want, monkeypatch):
    """Two groups (one with a window that gives pages back), portions beside single tokens, wanted rows of their own."""
    from coheryn_ai_studio_b200.cache import CacheManager
    from coheryn_ai_studio_b200.engine.step import StepEntry, StepRunner
    from coheryn_ai_studio_b200.parts.base import PagedKV

    class Model:                       # as much of a model as a runner asks for
        class runtime: device = torch.device("cuda:0")
        class spec: max_positions, vocab_size = 4096, 100
        capturable, status = False, torch.zeros(1, dtype=torch.int32, device="cuda:0")
    cache = CacheManager([PagedKV(1, 4, None), PagedKV(1, 4, 9)], [None, None], torch.float32, Model.runtime.device, page_size=4, num_pages=200,
                         max_requests=8)
    runner = StepRunner(Model, cache)
    rng = np.random.default_rng(3)
    for rid in "abcd":
        cache.admit(rid)
    for step in range(6):
        entries = []
        for rid in "abcd":
            n = int(rng.choice([1, 1, 5, 23]))
            places = {"few": [n - 1] if n > 1 else [], "all": list(range(n)), "none": []}[want]
            entries.append(StepEntry(rid, rng.integers(0, 100, n).tolist(), places))
        runner._check(entries)
        runner._reserve(entries)
        lay = runner._layout(entries)
        ctx, rows = runner._context(lay)
        with monkeypatch.context() as m:
            m.setattr(StepRunner, "_device_context", StepRunner._host_context)
            host, host_rows = runner._context(lay)
        assert torch.equal(rows, host_rows) and (ctx.tail is None) == (host.tail is None)
        for a, b in ((ctx, host),) + (((ctx.tail, host.tail),) if ctx.tail is not None else ()):
            for name in ("token_ids", "positions", "token_req", "cu_q", "kv_lens", "state_slots"):
                x, y = getattr(a, name), getattr(b, name)
                assert x.dtype == torch.int32 and x.is_contiguous() and torch.equal(x, y), name
            for x, y in zip(a.block_tables + a.slots, b.block_tables + b.slots):
                assert torch.equal(x, y)
            for name in ("num_tokens", "num_requests", "q_lens", "kv_lens_host", "max_q_len", "max_kv_len", "prior_positions_settled"):
                assert getattr(a, name) == getattr(b, name), name
        for e in entries:
            cache.commit(e.request_id)
