"""The attention over the 4-bit cache, each way against the bound of its own arithmetic (kv4_paths)."""
import numpy as np
import pytest
import torch

import kv4_paths as kp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def ops():
    from coheryn_ai_studio_b200 import ops as o
    return o


@pytest.fixture(autouse=True)
def no_status_left():
    yield
    torch.cuda.synchronize()
    word = ops().tc_status(torch.device(DEV))
    code = int(word.item())
    word.zero_()
    assert code == 0


def queries(seed, q_lens, heads, hd, spread=1.5, dtype=BF16):
    """[T, heads * hd]; ``spread`` one number, or one per request."""
    rng = np.random.default_rng(seed)
    by = np.repeat(np.broadcast_to(np.asarray(spread, np.float32), len(q_lens)), q_lens)[:, None]
    return torch.from_numpy(rng.standard_normal((sum(q_lens), heads * hd)).astype(np.float32) * by).to(dtype).to(DEV)


# ------------------------------------------------------------------------------------ rows that see nothing
@pytest.mark.parametrize("hd", [64, 96, 128, 192])
@pytest.mark.parametrize("window", [None, 30])
@pytest.mark.parametrize("lens", [(0, 0), (10, 0), (90, 40)])
def test_portions_longer_than_their_requests(hd, window, lens):
    """The first rows stand in front of position 0 and give zeros; the others as ever.  Also where no row of the call sees anything."""
    heads, nkv, q_lens = 4, 2, [90, 70]
    k, v = kp.random_rows(25, [90, 40], nkv, hd)
    rows = kp.Rows(k, v)
    rows.lens = list(lens)
    q = queries(26, q_lens, heads, hd)
    out = kp.attend(ops(), rows, q, q_lens, heads, window, kv_lens_host=list(lens))
    rows.k, rows.v = ([x[:n] for x, n in zip(y, lens)] for y in (k, v))
    at = 0
    for n, length in zip(q_lens, lens):
        assert (out[at:at + n - min(n, length)] == 0).all()
        at += n
    seen = [min(n, length) for n, length in zip(q_lens, lens)]
    part = lambda x: torch.cat([x[q_lens[0] - seen[0]:q_lens[0]], x[sum(q_lens) - seen[1]:]])        # noqa: E731
    kp.check(rows, part(q), part(out), seen, heads, BF16, window, simple=hd not in (64, 128), direct_rows=0)


def test_a_block_table_without_entries_is_refused():
    k, v = kp.random_rows(25, [90], 2, 96)
    for hd in (64, 96):
        rows = kp.Rows(*[[x[..., :hd] for x in y] for y in (k, v)])
        rows.table = rows.table[:, :0]
        with pytest.raises(ops().KernelError):
            kp.attend(ops(), rows, queries(27, [80], 4, hd), [80], 4)


# ------------------------------------------------------------------------------------ query rows and keys of zeros
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [None, 50])
@pytest.mark.parametrize("spread", [1e-4, 0.0])
def test_query_rows_of_zeros(hd, window, spread):
    """Scores of zero: the mean of the values that a row sees; over small keys, and over keys that are zeros."""
    heads, nkv, q_lens, lens = 4, 2, [130, 1, 70], [190, 33, 70]
    k, v = kp.random_rows(1, lens, nkv, hd, k_spread=spread)
    rows = kp.Rows(k, v)
    q = queries(2, q_lens, heads, hd)
    q[::3] = 0
    q[128:] = 0
    kp.check(rows, q, kp.attend(ops(), rows, q, q_lens, heads, window), q_lens, heads, BF16, window)


def test_a_zeroed_cache():
    heads, nkv, hd, q_lens, lens = 4, 1, 64, [140, 1], [300, 20]
    rows = kp.Rows(*[[np.zeros((n, nkv, hd), np.float32) for n in lens] for _ in range(2)])
    rows.k_cache.zero_(), rows.v_cache.zero_()
    for q in (queries(3, q_lens, heads, hd), torch.zeros(141, heads * hd, dtype=BF16, device=DEV)):
        assert (kp.attend(ops(), rows, q, q_lens, heads) == 0).all()


# ------------------------------------------------------------------------------------ magnitudes
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("k_spread,v_spread", [(1e36, 1e36), (1.0, 3e37), (1e-36, 1e-36), (1e36, 1e-36), (1.0, 1e-37)])
@pytest.mark.parametrize("context", [200, 2500])         # one CTA per pair of row tiles, and parts that are joined
def test_portions_of_any_magnitude(hd, k_spread, v_spread, context):
    heads, nkv, q_lens, lens = 4, 1, [70], [context]
    k, v = kp.random_rows(4, lens, nkv, hd, k_spread, v_spread)
    rows = kp.Rows(k, v)
    q = queries(5, q_lens, heads, hd, 1.5 / k_spread)
    kp.check(rows, q, kp.attend(ops(), rows, q, q_lens, heads), q_lens, heads, BF16)


@pytest.mark.parametrize("hd", [32, 64, 128, 160, 256])
@pytest.mark.parametrize("k_spread,v_spread", [(1e30, 1e29), (1e-30, 1e-30), (1.0, 1e-37)])
@pytest.mark.parametrize("q_lens,lens", [([1, 3], [700, 40]), ([1], [5000])])
def test_short_runs_of_any_magnitude(hd, k_spread, v_spread, q_lens, lens):
    k, v = kp.random_rows(32, lens, 2, hd, k_spread, v_spread)
    rows = kp.Rows(k, v)
    q = queries(33, q_lens, 4, hd, 1.5 / k_spread)
    kp.check(rows, q, kp.attend(ops(), rows, q, q_lens, 4), q_lens, 4, BF16)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("window", [None, 300])
@pytest.mark.parametrize("steps", ["up", "down", "zeros first", "one", "back and forth"])
def test_values_whose_magnitude_changes_along_the_context(hd, window, steps):
    """The power of two that the values are taken to follows the largest; what was added up before is scaled."""
    heads, nkv, q_lens, lens = 6, 2, [1, 4, 20], [900, 400, 130]
    k, v = kp.random_rows(34, lens, nkv, hd)
    for x in v:
        p = np.arange(len(x))
        by = {"up": 2.0 ** (p / 20), "down": 2.0 ** (-p / 20), "zeros first": np.where(p < 70, 0.0, 1.0), "one": np.where(p == 50, 2.0 ** 20, 1.0),
              "back and forth": 2.0 ** (10 * np.sin(p / 15.0))}[steps]
        x *= by[:, None, None].astype(np.float32)
        x[:, 1] *= np.float32(2.0 ** -12)
    rows = kp.Rows(k, v)
    q = queries(35, q_lens, heads, hd)
    kp.check(rows, q, kp.attend(ops(), rows, q, q_lens, heads, window), q_lens, heads, BF16, window)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,nkv", [(4, 1), (6, 2)])
def test_requests_of_one_call_keep_their_own_magnitudes(hd, heads, nkv):
    """A request's answer does not depend on what other requests, or other kv heads, hold."""
    q_lens, lens, spread = [70, 140, 1, 70], [200, 150, 40, 90], np.array([1e12, 1e-7, 1.0, 1e-3])
    parts = [kp.random_rows(10 + b, [n], nkv, hd, s, s) for b, (n, s) in enumerate(zip(lens, spread))]
    k, v = [p[0][0] for p in parts], [p[1][0] for p in parts]
    k[3][:, 0] *= np.float32(1e9)
    v[3][:, 0] *= np.float32(1e9)
    rows = kp.Rows(k, v)
    q = queries(6, q_lens, heads, hd, 1.5 / spread)
    q.view(-1, nkv, heads // nkv, hd)[sum(q_lens[:3]):, 0] *= 1e-9
    kp.check(rows, q, kp.attend(ops(), rows, q, q_lens, heads), q_lens, heads, BF16)
    alone = kp.Rows(k[1:2], v[1:2])
    again = kp.attend(ops(), alone, q[70:210], [140], heads)
    kp.check(alone, q[70:210], again, [140], heads, BF16)


@pytest.mark.parametrize("hd,top", [(64, 2.203125), (128, 1.5546875)])
@pytest.mark.parametrize("context", [600, 3000])
def test_many_keys_of_little_weight(hd, top, context):
    """One key in front of all others by 25.4 powers of two and a value of zero: what comes out is the others' share."""
    heads, nkv, q_lens, lens = 4, 1, [70], [context]
    k, v = np.zeros((context, nkv, hd), np.float32), np.ones((context, nkv, hd), np.float32)
    k[0], v[0] = top, 0
    rows = kp.Rows([k], [v])
    q = torch.ones(70, heads * hd, dtype=BF16, device=DEV)
    out = kp.attend(ops(), rows, q, q_lens, heads)
    # by hand: every p of the others is 2^-x of the first's
    p = np.exp(-top * hd ** 0.5)
    n = np.arange(context - 69, context + 1)[:, None] - 1.0
    want = n * p / (1 + n * p)
    # half a bfloat16 step, a float16 subnormal's step (2^-32 against p = 2^-25.4), float32 sums
    assert (np.abs(out.double().cpu().numpy() - want) <= want * (2.0 ** -8 + 2.0 ** -32 / p + context * 2.0 ** -22)).all()
    kp.check(rows, q, out, q_lens, heads, BF16)


# ------------------------------------------------------------------------------------ windows
@pytest.mark.parametrize("hd,page_size", [(64, 64), (128, 16), (128, 256), (96, 32), (64, 48)])
def test_what_lies_in_front_of_the_window(hd, page_size):
    """Values, and keys, that are not numbers at positions that no row of the request sees, in the page of the first that one does."""
    heads, nkv, window, q_lens, lens = 4, 1, 40, [70, 1, 66], [200, 90, 301]
    k, v = kp.random_rows(7, lens, nkv, hd)
    for b, (m, n) in enumerate(zip(q_lens, lens)):
        k[b][:n - m - window + 1] = np.nan
        v[b][:n - m - window + 1] = np.nan
    rows = kp.Rows(k, v, page_size)
    q = queries(8, q_lens, heads, hd)
    kp.check(rows, q, kp.attend(ops(), rows, q, q_lens, heads, window), q_lens, heads, BF16, window)


def temporaries(call):
    call()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("hd", [128, 96])
def test_a_window_bounds_the_expanded_pages(hd):
    """200 tokens at 16,384 positions that see 256 each: 456 positions of 8 kv heads in 16 bits are 1.9 MB at head size 128, all of them 67."""
    heads, nkv, window, q_lens, lens = 8, 8, 256, [200], [16384]
    rng = np.random.default_rng(9)
    k, v = [rng.standard_normal((lens[0], nkv, hd)).astype(np.float32) for _ in range(2)]
    rows = kp.Rows([k], [v])
    q = queries(9, q_lens, heads, hd)
    out = torch.zeros_like(q)
    assert temporaries(lambda: kp.attend(ops(), rows, q, q_lens, heads, window, out=out)) < 4 << 20
    kp.check(rows, q, out, q_lens, heads, BF16, window)


@pytest.mark.parametrize("hd", [64, 96])
def test_a_portion_beside_a_long_context_takes_its_own_pages(hd):
    """150 tokens beside a decoding request of 60,000 positions: 150 positions of 8 kv heads in 16 bits are 0.3 MB at head size 64, 60,000 123."""
    heads, nkv, q_lens, lens = 8, 8, [1, 150, 140], [60000, 150, 300]
    rng = np.random.default_rng(12)
    base = rng.standard_normal((500, nkv, hd)).astype(np.float32)
    k, v = kp.random_rows(12, lens[1:], nkv, hd)
    rows = kp.Rows([np.tile(base, (120, 1, 1))] + k, [np.tile(base[::-1], (120, 1, 1))] + v)
    q = queries(13, q_lens, heads, hd)
    out = torch.zeros_like(q)
    assert temporaries(lambda: kp.attend(ops(), rows, q, q_lens, heads, out=out, kv_lens_host=list(lens))) < 12 << 20
    kp.check(rows, q, out, q_lens, heads, BF16)


# ------------------------------------------------------------------------------------ block tables that end early
@pytest.mark.parametrize("hd", [32, 64, 96, 192])
def test_a_block_table_that_ends_before_its_request(hd):
    """Reported; nothing behind the table is read, and rows that see only pages that are there are right."""
    heads, nkv, q_lens, lens = 4, 2, [90, 70], [90, 200]
    k, v = kp.random_rows(28, lens, nkv, hd)
    rows = kp.Rows(k, v)
    rows.table = np.ascontiguousarray(rows.table[:, :8])
    q = queries(29, q_lens, heads, hd)
    out = kp.attend(ops(), rows, q, q_lens, heads)
    word = ops().tc_status(DEV)
    assert int(word.item()) == 41
    word.zero_()
    kp.check(rows, q[:90], out[:90], [90], heads, BF16, direct_rows=ops().kv4_direct_rows(hd))


# ------------------------------------------------------------------------------------ scales
@pytest.mark.parametrize("hd", [64, 128, 96, 256])
@pytest.mark.parametrize("scale", [-0.11, 0.0])
def test_scales_that_are_not_positive(hd, scale):
    heads, nkv, q_lens, lens = 4, 2, [90, 1, 70], [120, 33, 70]
    k, v = kp.random_rows(14, lens, nkv, hd)
    rows = kp.Rows(k, v)
    q = queries(15, q_lens, heads, hd)
    for lens_of_call in (q_lens, [1, 1, 2]):
        some = q[:sum(lens_of_call)]
        out = kp.attend(ops(), rows, some, lens_of_call, heads, scale=scale)
        direct = ops().kv4_direct_rows(hd) if max(lens_of_call) * 2 <= ops().kv4_direct_rows(hd) else 0         # all rows, or none
        kp.check(rows, some, out, lens_of_call, heads, BF16, scale=scale, direct_rows=direct)


# ------------------------------------------------------------------------------------ every way, every head size
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("heads,nkv,window", [(6, 2, None), (3, 1, 37), (4, 4, None)])
def test_runs_of_every_length(hd, heads, nkv, window):
    o = ops()
    limit = o.kv4_direct_rows(hd) // (heads // nkv)
    q_lens = [1, 5, limit, limit + 1, 0, limit + 40, 2]
    lens = [700, 5, limit + 30, limit + 1, 0, limit + 300, 90]
    k, v = kp.random_rows(16, lens, nkv, hd)
    rows = kp.Rows(k, v, 32)
    q = queries(17, q_lens, heads, hd)
    kp.check(rows, q, kp.attend(o, rows, q, q_lens, heads, window), q_lens, heads, BF16, window, direct_rows=o.kv4_direct_rows(hd))
    few = [1, 2, 0, 3, 0, 1, 1]
    for x, simple in ((q[:8], True), (q[:8].float(), False)):
        kp.check(rows, x, kp.attend(o, rows, x, few, heads, window, simple=simple), few, heads, x.dtype, window, simple=True)


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("hd,rot,heads,nkv,page_size", [(192, 192, 4, 2, 16), (192, 64, 3, 1, 48), (192, 0, 2, 2, 16), (224, 224, 2, 1, 32), (224, 30, 5, 1, 16),
                                                        (224, 0, 1, 3, 16), (96, 96, 2, 2, 16), (32, 10, 9, 3, 64)])
def test_writes_and_pages_of_other_head_sizes(dtype, hd, rot, heads, nkv, page_size):
    import test_kv4_gpu as base
    base.test_write_and_pages(dtype, hd, rot, heads, nkv, page_size)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q_lens,lens", [([1, 2], [2000, 40]), ([5, 1], [300, 5000]), ([70, 40], [200, 1500])])
def test_sharp_scores(hd, q_lens, lens):
    """Scores in the hundreds, where a key that has lost bits shows: a key rounded to bfloat16 moves them by tenths."""
    heads, nkv = 4, 1
    k, v = kp.random_rows(18, lens, nkv, hd, k_spread=6.0)
    rows = kp.Rows(k, v)
    q = queries(19, q_lens, heads, hd, 8.0)
    kp.check(rows, q, kp.attend(ops(), rows, q, q_lens, heads), q_lens, heads, BF16)
    some = q[:2].float()
    kp.check(rows, some, kp.attend(ops(), rows, some, [1, 1], heads), [1, 1], heads, torch.float32)


@pytest.mark.parametrize("hd", [64, 128])
def test_parts_joined_over_a_long_context(hd):
    heads, nkv, q_lens, lens = 8, 2, [33, 150], [3000, 2600]
    k, v = kp.random_rows(20, lens, nkv, hd)
    rows = kp.Rows(k, v)
    q = queries(21, q_lens, heads, hd)
    kp.check(rows, q, kp.attend(ops(), rows, q, q_lens, heads), q_lens, heads, BF16)


# ------------------------------------------------------------------------------------ rows behind the last request
@pytest.mark.parametrize("dtype,simple,scale", [(BF16, False, 0.125), (BF16, True, 0.125), (BF16, False, -0.125), (torch.float32, False, 0.125)])
@pytest.mark.parametrize("q_lens", [[3, 1], [80, 1], [0, 0]])
def test_rows_behind_the_last_request_stay(dtype, simple, scale, q_lens):
    """Whichever way the rows go; what a padded batch says about those rows is not read."""
    heads, nkv, hd, lens = 4, 2, 64, [90, 20]
    k, v = kp.random_rows(22, lens, nkv, hd)
    rows = kp.Rows(k, v)
    T = sum(q_lens)
    q = queries(23, [T + 5], heads, hd, dtype=dtype)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)      # noqa: E731
    req = np.concatenate([np.repeat([0, 1], q_lens), np.full(5, 9)])
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, q_lens)] + [np.full(5, 2 ** 30)])
    out = torch.full_like(q, 7.0)
    ops().attention_kv4_rows(q, out, rows.k_cache, rows.v_cache, i32(rows.table), i32(req), i32(pos), heads, nkv, hd, 16, None, scale,
                             cu_q=i32(np.concatenate([[0], np.cumsum(q_lens)])), kv_lens=i32(lens), q_lens=q_lens, max_kv_len=90, force_simple=simple)
    assert (out[T:] == 7).all()
    # (a scale that is not positive takes the whole call to the float32 kernel when a portion is in it)
    kp.check(rows, q[:T], out[:T], q_lens, heads, dtype, scale=scale, simple=simple or (scale < 0 and max(q_lens) > 64))


# ------------------------------------------------------------------------------------ operands checked in Python
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_calls_without_the_module_give_the_same(dtype, monkeypatch):
    """The four operators, with the module that checks their operands and without it: equal bits."""
    o = ops()
    heads, nkv, hd, q_lens, lens = 4, 2, 64, [3, 1], [90, 20]
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)      # noqa: E731
    qkv = queries(24, [110], heads + 2 * nkv, hd, dtype=dtype)
    table = torch.randn(200, hd // 2, 2, device=DEV)

    def run():
        entries, slots, pos, req = torch.full((2, 7), 5, dtype=torch.int32, device=DEV), i32(np.zeros(110)), i32(np.zeros(110)), i32(np.zeros(110))
        o.step_layout(i32([0, 0]), i32([90, 20]), i32([0, 6, 8]), i32([7, 3, 1, 0, 5, 2, 6, 4]), 16, entries, slots, positions=pos, token_req=req)
        caches = [torch.zeros((9,) + o.kv4_page_shape(nkv, 16, hd), dtype=torch.uint8, device=DEV) for _ in range(2)]
        q = o.rope_kv4_write(qkv, pos, table, slots, *caches, heads, nkv, hd, hd, 16)
        rows = torch.cat([q[87:90], q[109:]])
        out = torch.zeros_like(rows)
        o.attention_kv4_rows(rows, out, *caches, entries, i32([0, 0, 0, 1]), i32([87, 88, 89, 19]), heads, nkv, hd, 16, None, 0.125, cu_q=i32([0, 3, 4]),
                             kv_lens=i32(lens), q_lens=q_lens, max_kv_len=90)
        return [entries, slots, pos, req, *caches, q, out, *o.kv4_pages(*caches, i32([7, 4]), hd, 16, dtype)]
    module = run()
    called = []
    monkeypatch.setattr(o, "_calls_module", o._NoCalls)
    monkeypatch.setattr(o._NoCalls, "attention", staticmethod(lambda *operands: called.append(1)))
    for a, b in zip(module, run()):
        assert torch.equal(a, b)
    assert called


# ------------------------------------------------------------------------------------ refusals
def portion_call(q_lens=(80, 1), **more):
    k, v = kp.random_rows(22, [90, 20], 2, 64)
    rows = kp.Rows(k, v)
    q = queries(23, [81], 4, 64)
    return kp.attend(ops(), rows, q, list(q_lens), 4, **more)


def test_lengths_on_the_host_for_other_requests_are_refused():
    portion_call(kv_lens_host=[90, 20])
    with pytest.raises(ops().KernelError, match="lengths on the host"):
        portion_call(kv_lens_host=[90])


@pytest.mark.parametrize("q_lens", [(81, 1), (1, 81), (82, -1), (-1, 1), (2, -1)])
def test_lengths_that_do_not_fit_the_rows_are_refused(q_lens):
    """Refused on the host, before a kernel would follow such offsets (those on the device here are all zeros)."""
    k, v = kp.random_rows(22, [90, 20], 2, 64)
    rows = kp.Rows(k, v)
    q, none = queries(23, [81], 4, 64), torch.zeros(81, dtype=torch.int32, device=DEV)
    with pytest.raises(ops().KernelError, match="in 81 rows"):
        ops().attention_kv4_rows(q, torch.zeros_like(q), rows.k_cache, rows.v_cache, torch.from_numpy(rows.table).to(DEV), none, none, 4, 2, 64, 16, None,
                                 0.125, cu_q=none[:3], kv_lens=none[:2], q_lens=list(q_lens), max_kv_len=90)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_numbers_beyond_32_bits(dtype):
    """A window of more positions than there are is none; lengths and page sizes of that size are refused, not cut to 32 bits."""
    k, v = kp.random_rows(30, [90, 20], 2, 64)
    rows = kp.Rows(k, v)
    for q_lens in ([80, 1], [2, 1]):
        q = queries(31, q_lens, 4, 64, dtype=dtype)
        want = kp.attend(ops(), rows, q, q_lens, 4)
        for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 3, 2 ** 40 + 1):
            assert torch.equal(kp.attend(ops(), rows, q, q_lens, 4, window), want), window
        for more in (dict(max_kv_len=2 ** 32 + 90), dict(max_kv_len=-1), dict(kv_lens_host=[2 ** 32 + 90, 20]), dict(kv_lens_host=[-1, 20])):
            if "kv_lens_host" in more and (max(q_lens) == 2 or dtype == torch.float32):
                continue                                   # (not looked at where nothing is sized by it)
            with pytest.raises(ops().KernelError, match="on the host"):
                kp.attend(ops(), rows, q, q_lens, 4, **more)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    for page_size in (2 ** 32 + 16, -16, 0):
        with pytest.raises(ops().KernelError, match="pages|page size"):
            ops().step_layout(one, one, torch.zeros(2, dtype=torch.int32, device=DEV), one[:0], page_size, torch.zeros(1, 1, dtype=torch.int32, device=DEV))
