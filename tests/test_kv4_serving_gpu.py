"""The engine over a cache in 4 bits beyond plain decoding: padded batches, windows that give pages back, entries that read another's cache,
page lists that do not hold a step's positions."""
import numpy as np
import pytest
import torch

import plain_qwen2 as plain
from test_kv4_engine_gpu import held

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


# ------------------------------------------------------------------------------------ pages that do not hold a step's positions
class Model:                       # as much of a model as a runner asks for
    class runtime: device = DEV
    class spec: max_positions, vocab_size = 4096, 100
    capturable, status = False, None


@pytest.fixture
def runner():
    from coheryn_ai_studio_b200.cache import CacheManager
    from coheryn_ai_studio_b200.engine.step import StepRunner
    from coheryn_ai_studio_b200.parts.base import PagedKV
    Model.status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache = CacheManager([PagedKV(1, 4, None), PagedKV(1, 4, 9)], [None, None], torch.float32, DEV, page_size=16, num_pages=40, max_requests=4)
    return StepRunner(Model, cache)


def test_a_page_list_that_is_too_short_is_reported(runner):
    """Its rows would be dropped by the write; the step's status says so."""
    starts, q_lens = np.array([14, 3], np.int32), [4, 1]
    whole, short = [np.array([7, 8], np.int32), np.array([1], np.int32)], [np.array([7], np.int32), np.array([1], np.int32)]
    fields, _ = runner._step_arrays(starts, q_lens, [whole, whole], [])
    assert fields["slots"][0].tolist() == [126, 127, 128, 129, 19]
    runner.check_status()
    for tables in ([whole, short], [short, whole]):
        runner._step_arrays(starts, q_lens, tables, [])      # (-1 in the place of the slots behind the list)
        with pytest.raises(RuntimeError, match="pages do not hold"):
            runner.check_status()
    runner._step_arrays(np.array([-1, 3], np.int32), q_lens, [whole, whole], [])
    with pytest.raises(RuntimeError, match="lengths are negative"):
        runner.check_status()
    runner.check_status()              # reported once


def test_pages_that_a_window_has_given_back_are_not_reported(runner):
    fields, _ = runner._step_arrays(np.array([40], np.int32), [2], [[np.array([5, 6, 7], np.int32)], [np.array([-1, -1, 9], np.int32)]], [])
    assert [s.tolist() for s in fields["slots"]] == [[120, 121], [152, 153]]
    runner.check_status()


def test_the_largest_layout():
    """As many requests as one call takes: their offsets fill the shared memory."""
    from coheryn_ai_studio_b200 import ops
    B, ps = ops.STEP_LAYOUT_REQUESTS, 16
    rng = np.random.default_rng(8)
    starts, q_lens = rng.integers(0, 60, B), rng.integers(0, 4, B)
    counts = -(-(starts + q_lens) // ps)
    page_cu = np.concatenate([[0], np.cumsum(counts)])
    pages = rng.permutation(int(page_cu[-1]))
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)      # noqa: E731
    T = int(q_lens.sum())
    slots, pos, req, table = (torch.empty(n, dtype=torch.int32, device=DEV) for n in (T, T, T, (B, 5)))
    cu, kv, status = (torch.empty(n, dtype=torch.int32, device=DEV) for n in (B + 1, B, 1))
    status.zero_()
    ops.step_layout(i32(starts), i32(q_lens), i32(page_cu), i32(pages), ps, table, slots, cu, kv, pos, req, status=status)
    want_req = np.repeat(np.arange(B), q_lens)
    want_cu = np.concatenate([[0], np.cumsum(q_lens)])
    want_pos = starts[want_req] + np.arange(T) - want_cu[want_req]
    want_table = np.full((B, 5), -1)
    for b in range(B):
        want_table[b, :counts[b]] = pages[page_cu[b]:page_cu[b + 1]]
    for got, want in ((req, want_req), (cu, want_cu), (pos, want_pos), (kv, starts + q_lens), (table, want_table),
                      (slots, want_table[want_req, want_pos // ps] * ps + want_pos % ps)):
        assert np.array_equal(got.cpu().numpy(), want)
    assert int(status) == 0
    with pytest.raises(ops.KernelError, match="requests"):
        ops.step_layout(*[torch.zeros(B + n, dtype=torch.int32, device=DEV) for n in (1, 1, 2)], i32([0]), ps, torch.zeros(B + 1, 1, dtype=torch.int32, device=DEV))


# ------------------------------------------------------------------------------------ a model with a window and an entry that reads another's cache
class Config(dict):
    def to_dict(self):
        return dict(self)


CONFIG = Config(architectures=["FourBitToyForCausalLM"], hidden_size=96, num_attention_heads=3, num_key_value_heads=1, head_dim=64,
                intermediate_size=128, vocab_size=400, rms_norm_eps=1e-5, rope_theta=1e4, max_position_embeddings=256, window=21)


def spec_of(c):
    from coheryn_ai_studio_b200.config import ModelSpec, PartSpec, ScheduleEntry, prenorm_layer
    H = c["hidden_size"]
    norm = PartSpec("rmsnorm", {"size": H, "eps": c["rms_norm_eps"]})
    rope = PartSpec("rope_rotate_half", {"head_dim": c["head_dim"], "rotary_dim": c["head_dim"], "theta": c["rope_theta"],
                                         "max_positions": c["max_position_embeddings"]})
    ff = PartSpec("gated_mlp", {"hidden_size": H, "intermediate_size": c["intermediate_size"], "activation": "silu"})
    layers = [prenorm_layer(f"model.layers.{i}", PartSpec("attention", {"hidden_size": H, "num_heads": c["num_attention_heads"],
                                                                       "num_kv_heads": c["num_key_value_heads"], "head_dim": c["head_dim"],
                                                                       "qkv_bias": True, "o_bias": False, "window": window,
                                                                       "scale": c["head_dim"] ** -0.5}), ff, norm, norm, rope)
              for i, window in enumerate((None, c["window"]))]
    return ModelSpec("FourBitToyForCausalLM", H, c["vocab_size"], c["max_position_embeddings"], "model.embed_tokens", layers,
                     [ScheduleEntry(0), ScheduleEntry(1), ScheduleEntry(0, cache_from=0)], norm, "model.norm", "lm_head")


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from coheryn_ai_studio_b200.config import register_architecture, unregister_architecture
    from coheryn_ai_studio_b200.engine import write_random_model
    from coheryn_ai_studio_b200.weights import InitPolicy
    register_architecture("FourBitToyForCausalLM", lambda obj: Config(obj), spec_of)
    d = str(tmp_path_factory.mktemp("kv4_serving") / "model")
    write_random_model(d, CONFIG, 11, InitPolicy(0.08, 0.2, 0.05))
    yield d
    unregister_architecture("FourBitToyForCausalLM")


def plain_forward(cfg, w, ids, keep=lambda x, n: x):
    """Logits of every place; ``keep`` is what the cache makes of keys and values."""
    nh, nkv, hd, positions, kept = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"], np.arange(len(ids)), {}
    x = plain.embedding(w["model.embed_tokens.weight"], ids)
    for entry, (i, window, source) in enumerate(((0, None, None), (1, cfg["window"], None), (0, None, 0))):
        p = f"model.layers.{i}."
        y = plain.rms_norm(x, w[p + "input_layernorm.weight"], cfg["rms_norm_eps"])
        made = [plain.linear(y, w[p + f"self_attn.{n}_proj.weight"], w[p + f"self_attn.{n}_proj.bias"]) for n in "qkv"]
        q, k = (plain.rope(t, positions, hd, cfg["rope_theta"]) for t in made[:2])
        if source is None:
            kept[entry] = (keep(k, nkv), keep(made[2], nkv))
        o = plain.attention(q, *kept[entry if source is None else source], nh, nkv, hd, window)
        x = (x + plain.linear(o, w[p + "self_attn.o_proj.weight"])).astype(np.float32)
        y = plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], cfg["rms_norm_eps"])
        a = plain.swiglu(plain.linear(y, w[p + "mlp.gate_proj.weight"]), plain.linear(y, w[p + "mlp.up_proj.weight"]))
        x = (x + plain.linear(a, w[p + "mlp.down_proj.weight"])).astype(np.float32)
    return plain.linear(plain.rms_norm(x, w["model.norm.weight"], cfg["rms_norm_eps"]), w["lm_head.weight"])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [False, True])
def test_a_padded_batch_of_a_model_with_a_window_and_a_shared_cache(folder, dtype, graphs):
    """Eleven requests (a captured width of sixteen), prompts in portions, then decoding until the window has given pages back, while
    requests end.  The yardstick is, as for decoding alone, what quantising every key and value moves the logits by: in float32 a value next
    to a border between two codes may fall to either side of it; in bfloat16 every rounded key may, besides the type's own rounding."""
    from coheryn_ai_studio_b200.engine import Engine, StepEntry
    cfg, w = plain.read_model(folder)
    rng = np.random.default_rng(5)
    eng = Engine.from_folder(folder, dtype, context=128, max_num_seqs=11, kv_bits=4, use_graphs=graphs)
    assert [len(g.entries) for g in eng.cache.groups] == [1, 1] and all(g.tensor.dtype == torch.uint8 for g in eng.cache.groups)
    seqs = {f"r{i}": rng.integers(0, cfg["vocab_size"], int(n)).tolist() for i, n in enumerate(rng.integers(40, 70, 11))}
    at = {r: 0 for r in seqs}
    got = {r: {} for r in seqs}

    def step(lens):
        entries = [StepEntry(r, seqs[r][at[r]:at[r] + n], [n - 1]) for r, n in lens.items()]
        for e, row in zip(entries, eng.runner.step(entries).cpu().numpy()):
            at[e.request_id] += len(e.tokens)
            got[e.request_id][at[e.request_id] - 1] = row
    for r in seqs:
        eng.cache.admit(r)
    step({r: int(rng.integers(1, 20)) for r in seqs})
    step({r: int(rng.integers(1, 12)) for r in list(seqs)[::2]})
    while any(at[r] < len(s) for r, s in seqs.items()):
        step({r: 1 for r, s in seqs.items() if at[r] < len(s)})
    eng.runner.check_status()
    if graphs:
        assert sorted(eng.runner._graphs)[-1] == 16
    assert eng.cache.block_table("r0", 1)[0] == -1 and eng.cache.block_table("r0", 0)[0] >= 0
    for r, ids in seqs.items():
        want, full = plain_forward(cfg, w, ids, held), plain_forward(cfg, w, ids)
        yard = float(np.abs(want - full).max())
        d = np.array([np.abs(row - want[p]).max() for p, row in got[r].items()])
        middle, most = (2e-3, 0.1) if dtype == "float32" else (1.0, 2.0)
        assert yard > 0.05 and np.median(d) < middle * yard and d.max() < most * yard, (r, yard, np.median(d), d.max())
        eng.cache.free(r)
    eng.cache.check()
