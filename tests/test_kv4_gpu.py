"""The 4-bit cache's kernels against its definition: write, pages as values, attention, the step's index arrays, alone and
together.  Tolerances are those that kv4_cases.bound derives; what is whole numbers or bytes is equal."""
import numpy as np
import pytest
import torch

import kv4_cases as kc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from coheryn_ai_studio_b200 import ops as o
    return o


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def no_status_left():
    yield
    torch.cuda.synchronize()
    word = ops().tc_status(torch.device(DEV))
    code = int(word.item())
    word.zero_()
    assert code == 0


def expect_status(code):
    word = ops().tc_status(torch.device(DEV))
    assert int(word.item()) == code
    word.zero_()


class Cache:
    """A pool whose pages hold noise, the rows of a few requests, and in every row that belongs to nobody pairs that are not numbers."""

    def __init__(self, seed, lens, nkv, hd, page_size=16, spare=3, spread=1.0):
        rng = np.random.default_rng(seed)
        self.page_size, self.nkv, self.hd = page_size, nkv, hd
        counts = [-(-max(n, 0) // page_size) for n in lens]
        total = sum(counts) + spare
        order = rng.permutation(total)
        self.k = [rng.standard_normal((n, nkv, hd)).astype(np.float32) * spread for n in lens]
        self.v = [(rng.standard_normal((n, nkv, hd)) + 0.25 * rng.standard_normal((nkv, hd))).astype(np.float32) for n in lens]
        rows = [np.full((total, nkv, page_size, hd), np.nan, np.float32) for _ in range(2)]
        width = max(max(counts, default=1), 1) + 1
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for b, n in enumerate(lens):
            for j in range(counts[b]):
                page = int(order[at]); at += 1
                self.table[b, j] = page
                part = slice(j * page_size, min(n, (j + 1) * page_size))
                for r, x in zip(rows, (self.k[b], self.v[b])):
                    r[page, :, :part.stop - part.start] = x[part].transpose(1, 0, 2)
        tiles = lambda x: x.reshape(total, nkv, page_size // 16, 16, hd)  # noqa: E731
        self.k_cache = torch.from_numpy(kc.pack(tiles(rows[0]), False)).to(DEV)
        self.v_cache = torch.from_numpy(kc.pack(tiles(rows[1]), True)).to(DEV)
        held = lambda x: x.astype(np.float64) if not len(x) else kc.unpack(kc.pack(np.concatenate([x, np.zeros((-len(x) % 16,) + x.shape[1:], np.float32)])      # noqa: E731
                                           .reshape(-1, 16, nkv, hd).transpose(0, 2, 1, 3), False), False).transpose(0, 2, 1, 3).reshape(-1, nkv, hd)[:len(x)]
        self.k64, self.v64 = [held(x) for x in self.k], [held(x) for x in self.v]


def run_attention(cache, q_lens, lens, heads, dtype, window=None, seed=0, pad=0, simple=False, runs=True, q_spread=1.5):
    o = ops()
    rng = np.random.default_rng(seed + 1000)
    T = sum(q_lens)
    hd = cache.hd
    q = torch.from_numpy(rng.standard_normal((T + pad, heads * hd)).astype(np.float32) * q_spread).to(dtype).to(DEV)
    out = torch.full((T + pad, heads * hd), 7.0, dtype=dtype, device=DEV)
    cu = np.concatenate([[0], np.cumsum(q_lens)])
    positions = np.concatenate([np.arange(n - k, n) for k, n in zip(q_lens, lens)] + [np.zeros(pad)])
    req = np.concatenate([np.full(k, b) for b, k in enumerate(q_lens)] + [np.zeros(pad)])
    table = cache.table.copy()
    if window:
        for b, (k, n) in enumerate(zip(q_lens, lens)):
            table[b, :max(0, n - k - window + 1) // cache.page_size] = -1
    kw = dict(cu_q=i32(cu), kv_lens=i32(lens), q_lens=list(q_lens), max_kv_len=max(lens)) if runs else {}
    rows = T if not runs else T + pad
    o.attention_kv4_rows(q[:rows], out[:rows], cache.k_cache, cache.v_cache, i32(table), i32(req[:rows]), i32(positions[:rows]), heads, cache.nkv, hd,
                         cache.page_size, window, hd ** -0.5, force_simple=simple, **kw)
    return q, out, cu


def check_attention(cache, q, out, cu, q_lens, lens, heads, dtype, window=None, rounded_keys=()):
    hd = cache.hd
    got = out.float().cpu().numpy().astype(np.float64)
    qh = q.float().cpu().numpy().reshape(-1, heads, hd)
    for b, (k, n) in enumerate(zip(q_lens, lens)):
        if not k:
            continue
        want, mass, most = kc.attend(qh[cu[b]:cu[b + 1]], cache.k64[b], cache.v64[b], n - k, hd ** -0.5, window)
        tol = kc.bound(want, mass, most, hd, n, dtype, rounded_keys=b in rounded_keys)
        err = np.abs(got[cu[b]:cu[b + 1]].reshape(k, heads, hd) - want)
        assert np.isfinite(got[cu[b]:cu[b + 1]]).all(), f"request {b}"
        assert (err <= tol).all(), f"request {b}: {float((err / tol).max()):.2f} of the bound"
    assert (got[cu[-1]:] == 7.0).all()          # rows behind the last request


# ------------------------------------------------------------------------------------ write and read back
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,rot,heads,nkv,page_size", [(32, 32, 3, 1, 16), (64, 64, 4, 2, 32), (96, 48, 2, 2, 16), (128, 128, 5, 1, 16),
                                                        (128, 20, 2, 2, 48), (256, 0, 4, 4, 16), (160, 160, 1, 1, 16), (64, 0, 0, 2, 16)])
def test_write_and_pages(dtype, hd, rot, heads, nkv, page_size):
    o = ops()
    rng = np.random.default_rng(hd + rot)
    T, pages = 37, 5
    wide = torch.from_numpy((rng.standard_normal((T, (heads + 2 * nkv) * hd + 8)) * np.exp(rng.standard_normal((T, 1)))).astype(np.float32)).to(dtype)
    wide[3, :] = 0.5                                        # constant groups
    qkv = wide[:, :-8].to(DEV) if hd == 64 else wide.to(DEV)[:, :-8]       # whole rows, and rows of a wider buffer
    before = qkv.clone()
    slots = rng.permutation(pages * page_size)[:T]
    slots[[5, 11]] = -1
    positions = rng.integers(0, 500, T)
    angle = np.arange(500)[:, None] * 1e4 ** (-np.arange(0, rot, 2) / max(rot, 1))
    table = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    kc_, vc = (torch.randint(0, 256, (pages,) + o.kv4_page_shape(nkv, page_size, hd), dtype=torch.uint8, device=DEV) for _ in range(2))
    old = [kc_.clone(), vc.clone()]
    q = o.rope_kv4_write(qkv, i32(positions) if rot else None, torch.from_numpy(table).to(DEV) if rot else None, i32(slots), kc_, vc, heads, nkv,
                         hd, rot, page_size)
    assert torch.equal(qkv, before)
    x = qkv.float().cpu().numpy().reshape(T, heads + 2 * nkv, hd)
    turned = x.copy()
    if rot:
        h = rot // 2
        c, s = table[positions][..., 0][:, None], table[positions][..., 1][:, None]
        a, b = x[:, :heads + nkv, :h], x[:, :heads + nkv, h:rot]
        turned[:, :heads + nkv, :h], turned[:, :heads + nkv, h:rot] = a * c - b * s, b * c + a * s
        if dtype == torch.bfloat16:
            turned = kc.bf16(turned)
    assert np.array_equal(q.float().cpu().numpy().reshape(T, heads, hd), turned[:, :heads])
    for cache, was, rows, values in ((kc_, old[0], turned[:, heads:heads + nkv], False), (vc, old[1], turned[:, heads + nkv:], True)):
        want = was.cpu().numpy().reshape(pages, nkv, -1, 10 * hd)
        nib, at_s, at_m = kc.places(hd, values)
        for t in range(T):
            if slots[t] < 0:
                continue
            page, row = divmod(int(slots[t]), page_size)
            code, sc, mn = kc.quantise(rows[t])
            tile = want[page, :, row // 16]
            r = row % 16
            for ch in range(hd):
                at, sh = nib[r, ch] // 2, 4 * (nib[r, ch] % 2)
                tile[:, at] = (tile[:, at] & ~np.uint8(15 << sh)) | code[:, ch] << sh
            for at, v in ((at_s, sc), (at_m, mn)):
                w = kc.bits16(v)
                tile[:, at[r, ::32]], tile[:, at[r, ::32] + 1] = w & 255, w >> 8
        assert np.array_equal(cache.cpu().numpy().reshape(want.shape), want)
    # read back: some pages, twice the same, one outside the pool
    numbers = [4, 0, 0, 3]
    k, v = o.kv4_pages(kc_, vc, i32(numbers), hd, page_size, dtype)
    for got, cache, values in ((k, kc_, False), (v, vc, True)):
        exact = kc.cache_rows(cache.cpu().numpy(), values)[numbers]
        with np.errstate(all="ignore"):
            rounded = torch.from_numpy(exact.astype(np.float32)).to(dtype).float().numpy()
        assert np.array_equal(got.float().cpu().numpy(), rounded, equal_nan=True)


def test_write_values_that_are_not_finite_and_extremes():
    o = ops()
    hd, nkv, ps = 64, 1, 16
    big = float(torch.finfo(torch.float32).max)
    rows = np.zeros((8, 2 * hd), np.float32)
    rng = np.random.default_rng(2)
    rows[:] = rng.standard_normal(rows.shape)
    rows[0, 5] = np.nan
    rows[1, 40] = np.inf
    rows[2, 3] = -np.inf
    rows[3, :32] = [big, -big] * 16                    # a range beyond float32
    rows[4, :32] = 1e-44                               # constant and tiny
    rows[5, :32] = np.arange(32) * 1e-41               # a scale that bfloat16 cannot tell from zero, or hardly
    rows[6, :32] = big
    rows[7, 32:64] = np.linspace(3e38, 3.3e38, 32)
    kcache, vcache = (torch.zeros((1,) + o.kv4_page_shape(nkv, ps, hd), dtype=torch.uint8, device=DEV) for _ in range(2))
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.from_numpy(rows).to(dtype)
        o.rope_kv4_write(x.to(DEV), None, None, i32(np.arange(8)), kcache, vcache, 0, nkv, hd, 0, ps)
        for cache, part, values in ((kcache, x[:, :hd], False), (vcache, x[:, hd:], True)):
            r = np.zeros((16, hd), np.float32)
            r[:8] = part.float().numpy()
            got, want = kc.unpack(cache.cpu().numpy()[0, 0, 0], values)[:8], kc.unpack(kc.pack(r, values), values)[:8]
            assert np.array_equal(got, want, equal_nan=True)
            finite = np.isfinite(r[:8]).reshape(8, -1, 32).all(-1)
            assert np.isnan(got.reshape(8, -1, 32))[~finite].all()


def test_slots_positions_and_pages_outside_are_left_out_and_reported():
    o = ops()
    hd, ps = 32, 16
    cache = [torch.full((2,) + o.kv4_page_shape(1, ps, hd), 3, dtype=torch.uint8, device=DEV) for _ in range(2)]
    was = cache[0].clone()
    qkv = torch.randn(3, 3 * hd, device=DEV)
    o.rope_kv4_write(qkv, None, None, i32([2 * ps, 2 ** 31 - 1, -5]), *cache, 1, 1, hd, 0, ps)
    assert torch.equal(cache[0], was) and torch.equal(cache[1], was)
    expect_status(41)
    cos_sin = torch.ones(4, hd // 2, 2, device=DEV)
    q = o.rope_kv4_write(qkv, i32([4, -1, 0]), cos_sin, i32([-1, -1, -1]), *cache, 1, 1, hd, hd, ps)
    assert torch.equal(q[:2], qkv[:2, :hd])           # rows whose position has no angles are not turned
    expect_status(41)
    k, v = o.kv4_pages(*cache, i32([0, 2, -1]), hd, ps, torch.float32)
    assert (k[1:] == 0).all() and (v[1:] == 0).all() and not (k[0] == 0).all()
    expect_status(41)


# ------------------------------------------------------------------------------------ attention
CASES = [
    # heads, kv heads, head size, page size, q_lens, lens
    (12, 2, 128, 16, [1], [1]),
    (12, 2, 128, 16, [1, 1, 1], [16, 17, 700]),
    (4, 4, 64, 16, [1, 1, 1, 1], [1, 15, 64, 65]),
    (8, 1, 32, 32, [1, 2], [129, 300]),
    (5, 1, 96, 16, [1, 3, 1], [40, 33, 511]),
    (16, 1, 128, 16, [1, 1], [257, 90]),
    (40, 8, 128, 16, [1] * 5, [3, 250, 1, 64, 128]),
    (2, 1, 256, 16, [1, 4], [200, 77]),
    (6, 2, 160, 48, [2, 1], [145, 50]),
    (28, 4, 128, 16, [9, 1, 0, 2], [300, 40, 0, 2]),
    (14, 2, 64, 16, [5, 20, 1], [64, 20, 9]),
    (1, 1, 32, 16, [1], [2000]),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("window", [None, 1, 33])
@pytest.mark.parametrize("dtype,simple", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_attention(case, window, dtype, simple):
    heads, nkv, hd, ps, q_lens, lens = CASES[case]
    cache = Cache(case, lens, nkv, hd, ps)
    q, out, cu = run_attention(cache, q_lens, lens, heads, dtype, window, case, pad=0 if simple or dtype == torch.float32 else 2,
                               simple=simple)
    limit = ops().KV4_DIRECT_ROWS // (heads // nkv)
    check_attention(cache, q, out, cu, q_lens, lens, heads, dtype, window,
                    rounded_keys=[b for b, n in enumerate(q_lens) if n > limit and not simple and dtype == torch.bfloat16])


@pytest.mark.parametrize("heads,nkv,hd,ps", [(4, 2, 64, 16), (7, 1, 128, 16), (3, 3, 32, 16), (2, 1, 96, 32), (2, 1, 256, 16)])
@pytest.mark.parametrize("window", [None, 50])
def test_attention_of_portions_beside_single_tokens(heads, nkv, hd, ps, window):
    q_lens, lens = [1, 130, 65, 1, 0, 90, 3], [90, 130, 250, 1, 0, 91, 140]
    cache = Cache(5, lens, nkv, hd, ps)
    q, out, cu = run_attention(cache, q_lens, lens, heads, torch.bfloat16, window, 3, pad=1)
    check_attention(cache, q, out, cu, q_lens, lens, heads, torch.bfloat16, window, rounded_keys=(1, 2, 5))


@pytest.mark.parametrize("rows", [1, 16])
def test_portions_in_pieces_and_direct_agree(rows, monkeypatch):
    """The choice between the direct kernel and expanded pages, and the bound on those, move results by rounding only."""
    q_lens, lens, heads, nkv, hd = [20, 9, 30], [200, 9, 64], 4, 2, 64
    cache = Cache(9, lens, nkv, hd)
    monkeypatch.setattr(ops(), "KV4_DIRECT_ROWS", rows)
    monkeypatch.setattr(ops(), "KV4_EXPAND_BYTES", 1)
    q, out, cu = run_attention(cache, q_lens, lens, heads, torch.bfloat16)
    check_attention(cache, q, out, cu, q_lens, lens, heads, torch.bfloat16, rounded_keys=(0, 1, 2))


@pytest.mark.parametrize("heads,nkv,hd,window", [(8, 2, 64, None), (5, 1, 128, None), (14, 2, 64, 1500), (2, 2, 128, 700), (8, 2, 64, 2300)])
def test_portions_late_in_long_prompts(heads, nkv, hd, window):
    """Few row tiles and many keys: the key tiles are cut into parts for a CTA each; pairs of row tiles whose first sees a key tile less."""
    q_lens, lens = [75, 1, 150], [3000, 40, 2049]
    cache = Cache(12, lens, nkv, hd)
    q, out, cu = run_attention(cache, q_lens, lens, heads, torch.bfloat16, window, 4, pad=1)
    parts = ops().kv4_lib(hd).coheryn_kv4_prompt_parts(heads, nkv, 1, 150, 150 * heads // nkv, 3000, window or 0)
    assert (parts > 1) == (window is None or window > 2000)          # eight key tiles per part at least
    check_attention(cache, q, out, cu, q_lens, lens, heads, torch.bfloat16, window)


@pytest.mark.parametrize("scale", [1e-9, 3e-3, 1e6, 1e20])
def test_keys_and_values_of_any_magnitude(scale):
    """The tensor cores see powers of two times keys, values and queries: exact, whatever their magnitude."""
    heads, nkv, hd, q_lens, lens = 4, 2, 64, [70, 1, 9], [200, 300, 30]
    cache = Cache(13, lens, nkv, hd)
    for t, values in ((cache.k_cache, False), (cache.v_cache, True)):
        rows = kc.cache_rows(t.cpu().numpy(), values)
        with np.errstate(invalid="ignore"):
            tiles = (rows * scale).astype(np.float32).reshape(t.shape[0], nkv, 1, 16, hd)
        t.copy_(torch.from_numpy(kc.pack(tiles, values)))
    held = [kc.cache_rows(t.cpu().numpy(), v) for t, v in ((cache.k_cache, False), (cache.v_cache, True))]
    for b, n in enumerate(lens):
        pages = [p for p in cache.table[b] if p >= 0]
        cache.k64[b], cache.v64[b] = (h[pages].transpose(0, 2, 1, 3).reshape(-1, nkv, hd)[:n] for h in held)
    q, out, cu = run_attention(cache, q_lens, lens, heads, torch.bfloat16, q_spread=1.5 / scale)
    check_attention(cache, q, out, cu, q_lens, lens, heads, torch.bfloat16)


def test_many_requests_of_all_lengths_share_the_cuts():
    """More lists than clusters would hold: the units of all of them in equal shares, lists that begin and end inside a share."""
    rng = np.random.default_rng(7)
    lens = [int(x) for x in rng.integers(1, 900, 60)] + [2500, 0, 1]
    q_lens = [1] * 60 + [1, 0, 1]
    for heads, nkv, hd, window in ((4, 2, 64, None), (16, 8, 128, 300), (2, 1, 256, None)):
        cache = Cache(20, lens, nkv, hd)
        q, out, cu = run_attention(cache, q_lens, lens, heads, torch.bfloat16, window)
        check_attention(cache, q, out, cu, q_lens, lens, heads, torch.bfloat16, window)


def test_rows_of_wider_buffers():
    heads, nkv, hd, lens, q_lens = 4, 2, 64, [300, 90], [1, 70]
    cache = Cache(2, lens, nkv, hd)
    wide = torch.randn(71, heads * hd + 64, device=DEV).to(torch.bfloat16)
    q, room = wide[:, 32:32 + heads * hd], torch.full((71, heads * hd + 16), 7.0, device=DEV, dtype=torch.bfloat16)
    out = room[:, 8:8 + heads * hd]
    cu = np.array([0, 1, 71])
    ops().attention_kv4_rows(q, out, cache.k_cache, cache.v_cache, i32(cache.table), i32([0] + [1] * 70), i32([299] + list(range(20, 90))), heads, nkv, hd,
                             16, None, hd ** -0.5, cu_q=i32(cu), kv_lens=i32(lens), q_lens=q_lens, max_kv_len=300)
    check_attention(cache, q, out, cu, q_lens, lens, heads, torch.bfloat16)
    assert (room[:, :8] == 7).all() and (room[:, 8 + heads * hd:] == 7).all()


def test_sharp_scores_and_a_long_context():
    """Scores in the hundreds (one key takes nearly all), over a context that is cut into many items."""
    lens, heads, nkv, hd = [9000, 5], 2, 1, 64
    cache = Cache(4, lens, nkv, hd, spread=8.0)
    for dtype in (torch.bfloat16, torch.float32):
        q, out, cu = run_attention(cache, [1, 1], lens, heads, dtype, q_spread=8.0)
        check_attention(cache, q, out, cu, [1, 1], lens, heads, dtype)


def test_rows_by_request_and_position_in_any_order():
    lens, heads, nkv, hd = [70, 33], 6, 2, 64
    cache = Cache(6, lens, nkv, hd)
    rng = np.random.default_rng(1)
    req, pos = [1, 0, 0, 1], [3, 69, 0, 32]
    q = torch.from_numpy(rng.standard_normal((4, heads * hd)).astype(np.float32)).to(DEV)
    wide = torch.zeros(4, heads * hd + 3, device=DEV)          # rows of any alignment
    out = wide[:, 3:]
    ops().attention_kv4_rows(q, out, cache.k_cache, cache.v_cache, i32(cache.table), i32(req), i32(pos), heads, nkv, hd, 16, None, hd ** -0.5)
    for i in range(4):
        want, mass, most = kc.attend(q[i:i + 1].cpu().numpy().reshape(1, heads, hd), cache.k64[req[i]], cache.v64[req[i]], pos[i], hd ** -0.5)
        tol = kc.bound(want, mass, most, hd, pos[i] + 1, torch.float32)
        assert (np.abs(out[i].cpu().numpy().reshape(1, heads, hd) - want) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_entries_outside_the_pool_are_left_out_and_reported(dtype):
    lens, heads, nkv, hd = [100], 4, 2, 64
    cache = Cache(8, lens, nkv, hd)
    cache.table[0, 2], cache.table[0, 4] = cache.k_cache.shape[0], -1
    q, out, cu = run_attention(cache, [1], lens, heads, dtype)
    expect_status(41)
    keep = np.r_[0:32, 48:64, 80:100]
    want, mass, most = kc.attend(q.float().cpu().numpy().reshape(1, heads, hd), cache.k64[0][keep], cache.v64[0][keep], len(keep) - 1, hd ** -0.5)
    tol = kc.bound(want, mass, most, hd, 100, dtype)
    assert (np.abs(out.float().cpu().numpy().reshape(1, heads, hd) - want) <= tol).all()


def test_a_row_without_keys_gives_zeros():
    cache = Cache(8, [40], 2, 64)
    q = torch.randn(2, 4 * 64, device=DEV, dtype=torch.bfloat16)
    out = torch.full_like(q, 7.0)
    # two rows of a request whose length is one: the first stands at position -1 and sees nothing
    ops().attention_kv4_rows(q, out, cache.k_cache, cache.v_cache, i32(cache.table), i32([0, 0]), i32([-1, 0]), 4, 2, 64, 16, None, 0.125,
                             cu_q=i32([0, 2]), kv_lens=i32([1]), q_lens=[2], max_kv_len=1)
    assert (out[0] == 0).all() and torch.isfinite(out).all() and not (out[1] == 0).all()
    other = torch.full_like(q, 7.0)
    ops().attention_kv4_rows(q, other, cache.k_cache, cache.v_cache, i32(cache.table), i32([0, 0]), i32([-1, 0]), 4, 2, 64, 16, None, 0.125)
    assert (other[0] == 0).all()


@pytest.mark.parametrize("longest", [1024, 8192])        # parts joined in clusters, and by a kernel of their own
def test_captured_and_replayed_with_other_lengths_and_on_another_stream(longest):
    o = ops()
    heads, nkv, hd, lens = 12, 2, 128, [900, 33, 400]
    cache = Cache(3, lens, nkv, hd)
    q = torch.randn(3, heads * hd, device=DEV).to(torch.bfloat16)
    table, cu, req = i32(cache.table), i32([0, 1, 2, 3]), i32([0, 1, 2])
    kv, pos, out = i32(lens), i32([n - 1 for n in lens]), torch.zeros_like(q)

    def call(to):
        o.attention_kv4_rows(q, to, cache.k_cache, cache.v_cache, table, req, pos, heads, nkv, hd, 16, None, hd ** -0.5, cu_q=cu, kv_lens=kv,
                             q_lens=[1, 1, 1], max_kv_len=longest)
    call(out)
    torch.cuda.synchronize()
    graphs, outs = [], [torch.zeros_like(q) for _ in range(2)]
    for to in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(to)
        graphs.append(g)
    for now in ([900, 33, 400], [1, 20, 399], [64, 1, 65]):
        kv.copy_(i32(now)); pos.copy_(i32([n - 1 for n in now]))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):          # two captured calls and an eager one at a time
            graphs[0].replay()
        graphs[1].replay()
        call(out)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], out) and torch.equal(outs[1], out)
        check_attention(Clipped(cache, now), q, out, [0, 1, 2, 3], [1, 1, 1], now, heads, torch.bfloat16)


@pytest.mark.parametrize("heads,nkv,hd", [(4, 2, 64), (7, 1, 128), (2, 1, 96)])
def test_portions_captured_and_replayed_over_other_pages(heads, nkv, hd):
    """Two captured calls of portions beside a single token, replayed at once over a cache that has changed in between."""
    o = ops()
    q_lens, lens = [150, 1, 200], [400, 77, 200]
    caches = [Cache(seed, lens, nkv, hd) for seed in (51, 51, 52)]
    kept = caches[0]
    q = torch.randn(351, heads * hd, device=DEV).to(torch.bfloat16)
    cu, kv = i32([0, 150, 151, 351]), i32(lens)
    req = i32(np.repeat([0, 1, 2], q_lens))
    pos = i32(np.concatenate([np.arange(n - m, n) for n, m in zip(lens, q_lens)]))
    table = i32(kept.table)
    outs = [torch.zeros_like(q) for _ in range(3)]
    call = lambda out: o.attention_kv4_rows(q, out, kept.k_cache, kept.v_cache, table, req, pos, heads, nkv, hd, 16, None, hd ** -0.5, cu_q=cu,  # noqa: E731
                                            kv_lens=kv, q_lens=q_lens, max_kv_len=400)
    call(outs[2])
    torch.cuda.synchronize()
    graphs = []
    for out in outs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(out)
        graphs.append(g)
    for other in (caches[2], caches[1]):
        kept.k_cache.copy_(other.k_cache); kept.v_cache.copy_(other.v_cache); table.copy_(i32(other.table))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        call(outs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2])
        check_attention(other, q, outs[2], [0, 150, 151, 351], q_lens, lens, heads, torch.bfloat16, rounded_keys=(0, 2))


class Clipped:
    def __init__(self, cache, lens):
        self.hd = cache.hd
        self.k64, self.v64 = ([x[:n] for x, n in zip(y, lens)] for y in (cache.k64, cache.v64))


# ------------------------------------------------------------------------------------ the step's index arrays
def plain_layout(starts, q_lens, lists, page_size, width):
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    pos, req, slots = [], [], []
    table = np.full((len(starts), width), -1, np.int32)
    for b, (s, q, pages) in enumerate(zip(starts, q_lens, lists)):
        table[b, :len(pages)] = pages
        for p in range(s, s + q):
            pos.append(p); req.append(b)
            slots.append(pages[p // page_size] * page_size + p % page_size if pages[p // page_size] >= 0 else -1)
    return cu, np.asarray(starts) + np.asarray(q_lens), np.array(pos, int), np.array(req, int), table, np.array(slots, int)


@pytest.mark.parametrize("B,page_size,most,spread", [(1, 16, 1, 40), (8, 16, 1, 4096), (300, 16, 1, 500), (5, 7, 900, 50), (2, 1, 60, 9), (1, 16, 5000, 1),
                                                     (1100, 32, 3, 40)])
def test_step_layout(B, page_size, most, spread):
    o = ops()
    rng = np.random.default_rng(B)
    starts, q_lens = rng.integers(0, spread, B), rng.integers(0 if B > 1 else most, most + 1, B)
    counts = [-(-(s + q) // page_size) + int(rng.integers(0, 2)) for s, q in zip(starts, q_lens)]
    order = rng.permutation(sum(counts) + 5)
    page_cu = np.concatenate([[0], np.cumsum(counts)])
    lists = [order[page_cu[b]:page_cu[b + 1]].copy() for b in range(B)]
    for b in range(0, B, 3):                     # pages that a window has given back
        lists[b][:starts[b] // page_size // 2] = -1
    pages = np.concatenate(lists) if sum(counts) else np.zeros(0, int)
    width = max(counts + [1]) + 2
    T = int(q_lens.sum())
    extra = 3
    out = {n: torch.full((size,), 77, dtype=torch.int32, device=DEV)
           for n, size in (("cu_q", B + 1), ("kv_lens", B), ("positions", T + extra), ("token_req", T + extra), ("slots", T + extra))}
    table = torch.full((B, width), 77, dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    o.step_layout(i32(starts), i32(q_lens), i32(page_cu), i32(pages), page_size, table, status=status, **out)
    cu, kv, pos, req, want, slots = plain_layout(starts, q_lens, lists, page_size, width)
    for name, x in (("cu_q", cu), ("kv_lens", kv)):
        assert np.array_equal(out[name].cpu().numpy(), x), name
    for name, x in (("positions", pos), ("token_req", req), ("slots", slots)):
        got = out[name].cpu().numpy()
        assert np.array_equal(got[:T], x), name
        assert (got[T:] == 77).all(), name
    assert np.array_equal(table.cpu().numpy(), want) and int(status) == 0
    # the table alone, then the same table grown by what each request gains
    again = torch.full((B, width), 55, dtype=torch.int32, device=DEV)
    kept = [len(l) - int(rng.integers(0, 2)) if len(l) else 0 for l in lists]
    o.step_layout(i32(starts), i32(np.zeros(B)), i32(np.concatenate([[0], np.cumsum(kept)])),
                  i32(np.concatenate([l[:n] for l, n in zip(lists, kept)]) if sum(kept) else np.zeros(0)), page_size, again)
    gain = [l[n:] for l, n in zip(lists, kept)]
    slots2 = torch.full((T,), 77, dtype=torch.int32, device=DEV)
    o.step_layout(i32(starts), i32(q_lens), i32(np.concatenate([[0], np.cumsum([len(g) for g in gain])])),
                  i32(np.concatenate(gain)), page_size, again, slots2, first=i32(kept), status=status)
    assert np.array_equal(again.cpu().numpy(), want) and np.array_equal(slots2.cpu().numpy(), slots) and int(status) == 0


def test_step_layout_of_lengths_that_do_not_fit():
    o = ops()

    def call(starts, q_lens, page_cu, pages, T, W=4, first=None):
        B = len(starts)
        got = [torch.full((T,), 77, dtype=torch.int32, device=DEV) for _ in range(3)]
        guard = torch.full((3, B, W), 77, dtype=torch.int32, device=DEV)
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        o.step_layout(i32(starts), i32(q_lens), i32(page_cu), i32(pages), 16, guard[1], got[0], positions=got[1], token_req=got[2],
                      first=None if first is None else i32(first), status=status)
        assert (guard[0] == 77).all() and (guard[2] == 77).all()
        return int(status), [g.cpu().tolist() for g in got], guard[1].cpu().tolist()
    code, (slots, pos, req), table = call([0, 3], [2, 4], [0, 1, 2], [5, 6], 4)         # more tokens than the arrays hold
    assert code == 51 and slots == [80, 81, 99, 100] and req == [0, 0, 1, 1]
    assert call([0, -3], [1, 1], [0, 1, 2], [5, 6], 2)[0] in (51, 52)                     # a negative length
    assert call([0], [-2], [0, 1], [5], 2)[0] == 51
    code, (slots, _, _), table = call([15], [3], [0, 1], [5], 3)                          # the second page is missing
    assert code == 52 and slots == [95, -1, -1] and table == [[5, -1, -1, -1]]
    code, _, table = call([0, 0], [1, 1], [0, 9, 2], [5, 6], 2)                           # offsets that leave the list
    assert code == 52 and table == [[-1] * 4] * 2
    code, _, table = call([0], [1], [0, 6], [1, 2, 3, 4, 5, 6], 1)                        # a list longer than the table
    assert code == 52 and table == [[1, 2, 3, 4]]
    code, (slots, _, _), _ = call([0], [1], [0, 1], [2 ** 31 - 1], 1)                     # a slot beyond 32 bits
    assert code == 52 and slots == [-1]
    assert call([0, 0], [2 ** 31 - 1] * 2, [0, 1, 2], [5, 6], 2)[0] == 51                # offsets beyond 32 bits
    table, status = torch.full((2, 3), 77, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    cu_q = torch.full((3,), 77, dtype=torch.int32, device=DEV)
    o.step_layout(i32([0, 3]), i32([2, 4]), i32([0, 1, 2]), i32([5, 6]), 16, table, cu_q=cu_q, status=status)      # no array of tokens
    assert int(status) == 0 and cu_q.tolist() == [0, 2, 6] and table.tolist() == [[5, -1, -1], [6, -1, -1]]
    with pytest.raises(o.KernelError, match="requests"):
        call([0] * 12000, [0] * 12000, [0] * 12001, [0], 0)


# ------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_steps_of_layout_write_and_attention(dtype):
    """A prompt in two portions, then single tokens, beside a second request, as a program strings the operators together; the
    attention reads what the writes left, against the rows quantised on the CPU."""
    o = ops()
    heads, nkv, hd, ps, pool = 4, 2, 64, 16, 24
    rng = np.random.default_rng(11)
    caches = [torch.full((pool,) + o.kv4_page_shape(nkv, ps, hd), 0xff, dtype=torch.uint8, device=DEV) for _ in range(2)]   # not-a-number everywhere
    free = list(rng.permutation(pool))
    held, k_rows, v_rows = [[], []], [np.zeros((0, nkv, hd))] * 2, [np.zeros((0, nkv, hd))] * 2
    steps = [[50, 3], [47, 1], [1, 1], [1, 20], [1, 1]]
    W = 8
    table = torch.full((2, W), -1, dtype=torch.int32, device=DEV)
    lens = [0, 0]
    for q_lens in steps:
        T = sum(q_lens)
        first = [len(h) for h in held]
        for b, n in enumerate(q_lens):
            while len(held[b]) * ps < lens[b] + n:
                held[b].append(int(free.pop()))
        gained = [h[f:] for h, f in zip(held, first)]
        out = {n: torch.empty(size, dtype=torch.int32, device=DEV) for n, size in (("cu_q", 3), ("kv_lens", 2), ("positions", T), ("token_req", T))}
        slots = torch.empty(T, dtype=torch.int32, device=DEV)
        o.step_layout(i32(lens), i32(q_lens), i32(np.concatenate([[0], np.cumsum([len(g) for g in gained])])), i32(sum(gained, [])), ps, table, slots,
                      first=i32(first), **out)
        qkv = torch.from_numpy(rng.standard_normal((T, (heads + 2 * nkv) * hd)).astype(np.float32)).to(dtype).to(DEV)
        q = o.rope_kv4_write(qkv, None, None, slots, *caches, heads, nkv, hd, 0, ps)
        got = torch.zeros(T, heads * hd, dtype=dtype, device=DEV)
        lens = [a + n for a, n in zip(lens, q_lens)]
        o.attention_kv4_rows(q, got, *caches, table, out["token_req"], out["positions"], heads, nkv, hd, ps, None, hd ** -0.5, cu_q=out["cu_q"],
                             kv_lens=out["kv_lens"], q_lens=q_lens, max_kv_len=max(lens))
        x = qkv.float().cpu().numpy().reshape(T, heads + 2 * nkv, hd)
        cu = np.concatenate([[0], np.cumsum(q_lens)])
        for b in range(2):
            part = x[cu[b]:cu[b + 1]]
            for rows, at in ((k_rows, heads), (v_rows, heads + nkv)):
                c, s, m = kc.quantise(part[:, at:at + nkv])
                rows[b] = np.concatenate([rows[b], (c.reshape(c.shape[:-1] + (-1, 32)) * s[..., None].astype(np.float64) + m[..., None]).reshape(c.shape)])
            want, mass, most = kc.attend(part[:, :heads], k_rows[b], v_rows[b], lens[b] - q_lens[b], hd ** -0.5)
            tol = kc.bound(want, mass, most, hd, lens[b], dtype, rounded_keys=q_lens[b] * heads // nkv > o.KV4_DIRECT_ROWS)
            err = np.abs(got[cu[b]:cu[b + 1]].float().cpu().numpy().reshape(want.shape) - want)
            assert (err <= tol).all(), (q_lens, b, float((err / tol).max()))


# How lists get their CTAs: clusters of 16, 8, 4 and 2 (also of three CTAs per SM), two row tiles, lists that end early, long ones beside short.
@pytest.mark.parametrize("requests,heads,nkv,hd,tokens,longest", [
    (1, 4, 2, 64, 1, 1500), (1, 14, 2, 128, 3, 1100), (3, 2, 1, 32, 1, 2048), (9, 8, 2, 64, 1, 900), (16, 8, 2, 128, 1, 700), (20, 8, 2, 32, 1, 1000),
    (24, 16, 4, 96, 1, 450), (26, 8, 4, 128, 1, 500), (40, 8, 4, 64, 1, 250), (70, 2, 2, 128, 1, 600), (3, 6, 2, 256, 2, 1000), (30, 4, 2, 160, 1, 500),
    (5, 12, 2, 64, 5, 700), (16, 7, 1, 128, 9, 300)])
@pytest.mark.parametrize("window", [None, 130])
def test_lists_of_clusters(requests, heads, nkv, hd, tokens, longest, window):
    rng = np.random.default_rng(requests * longest)
    q_lens = [int(x) for x in rng.integers(0, tokens + 1, requests)]
    q_lens[0] = tokens
    lens = [int(n + rng.integers(0, longest - n + 1)) for n in q_lens]
    lens[0], lens[-1] = longest, max(q_lens[-1], 1)
    cache = Cache(31, lens, nkv, hd)
    q, out, cu = run_attention(cache, q_lens, lens, heads, torch.bfloat16, window, 5, pad=1)
    check_attention(cache, q, out, cu, q_lens, lens, heads, torch.bfloat16, window)


# More units of 128 positions than CTAs: shares that begin and end inside lists, in front of their first unit too, and hold many short ones.
@pytest.mark.parametrize("requests,heads,nkv,hd,tokens,longest", [
    (200, 8, 4, 64, 1, 300), (150, 4, 4, 128, 1, 700), (10, 8, 8, 32, 2, 9000), (60, 10, 5, 96, 2, 1200), (90, 3, 3, 256, 1, 600), (40, 14, 2, 64, 4, 2500),
    (300, 8, 4, 64, 1, 120), (180, 12, 2, 128, 5, 128)])
@pytest.mark.parametrize("window", [None, 200])
def test_shares_across_lists(requests, heads, nkv, hd, tokens, longest, window):
    rng = np.random.default_rng(requests + longest)
    q_lens = [int(x) for x in rng.integers(0, tokens + 1, requests)]
    q_lens[-1] = tokens
    lens = [int(n + (longest - n) * rng.random() ** 3) for n in q_lens]
    lens[requests // 2] = longest
    cache = Cache(37, lens, nkv, hd)
    q, out, cu = run_attention(cache, q_lens, lens, heads, torch.bfloat16, window, 7, pad=1)
    check_attention(cache, q, out, cu, q_lens, lens, heads, torch.bfloat16, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_requests_that_are_not_there(dtype):
    o = ops()
    heads, nkv, hd = 4, 2, 64
    cache = Cache(3, [40, 70], nkv, hd)
    q = torch.randn(4, heads * hd, device=DEV).to(dtype)
    both = [torch.full_like(q, 7.0) for _ in range(2)]
    for out, req in zip(both, ([0, 0, 1, 1], [0, -1, 1, 2])):
        o.attention_kv4_rows(q, out, cache.k_cache, cache.v_cache, i32(cache.table), i32(req), i32([39, 20, 69, 5]), heads, nkv, hd, 16, None, hd ** -0.5, force_simple=True)
    expect_status(41)
    assert (both[1][[1, 3]] == 0).all() and torch.equal(both[0][[0, 2]], both[1][[0, 2]])


# ------------------------------------------------------------------------------------ refusals
def test_refusals():
    o = ops()
    ok = torch.zeros((2,) + o.kv4_page_shape(1, 16, 64), dtype=torch.uint8, device=DEV)
    qkv, slots = torch.zeros(2, 3 * 64, device=DEV), i32([0, 1])
    write = lambda **kw: o.rope_kv4_write(**{**dict(qkv=qkv, positions=None, cos_sin=None, slots=slots, k_cache=ok, v_cache=ok.clone(), num_heads=1,     # noqa: E731
                                                    num_kv_heads=1, head_dim=64, rotary_dim=0, page_size=16), **kw})
    for kw in (dict(head_dim=48), dict(page_size=8), dict(k_cache=ok.float()), dict(k_cache=ok[:, :, :, :320]), dict(v_cache=ok[:1]), dict(num_heads=2),
               dict(slots=i32([0])), dict(slots=slots.long()), dict(rotary_dim=64), dict(qkv=qkv.half()), dict(qkv=qkv.cpu()),
               dict(rotary_dim=64, positions=slots, cos_sin=torch.zeros(4, 16, 2, device=DEV)), dict(qkv=torch.zeros(2, 193, device=DEV)[:, 1:])):
        with pytest.raises(o.KernelError):
            write(**kw)
    q = torch.zeros(2, 64, device=DEV, dtype=torch.bfloat16)
    attend = lambda **kw: o.attention_kv4_rows(**{**dict(q=q, out=torch.zeros_like(q), k_cache=ok, v_cache=ok, block_tables=i32([[0]] * 2), token_req=slots,  # noqa: E731
                                                         positions=slots, num_heads=1, num_kv_heads=1, head_dim=64, page_size=16, window=None, scale=1.0,
                                                         cu_q=i32([0, 1, 2]), kv_lens=i32([1, 1]), q_lens=[1, 1], max_kv_len=1), **kw})
    for kw in (dict(num_heads=3, num_kv_heads=2), dict(out=torch.zeros(2, 64, device=DEV)), dict(q=q[:, :32]), dict(window=0), dict(kv_lens=i32([1])),
               dict(block_tables=i32([[0]])), dict(block_tables=i32([0])), dict(cu_q=i32([0, 1])), dict(q=q.half(), out=q.half())):
        with pytest.raises(o.KernelError):
            attend(**kw)
    with pytest.raises(o.KernelError):
        o.kv4_pages(ok, ok, slots, 64, 16, torch.float16)
    table = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    lay = lambda **kw: o.step_layout(**{**dict(starts=slots, q_lens=slots, page_cu=i32([0, 0, 0]), pages=i32([]), page_size=16, block_table=table), **kw})  # noqa: E731
    for kw in (dict(q_lens=i32([1])), dict(page_cu=i32([0, 0])), dict(block_table=table[:1]), dict(page_size=0), dict(slots=i32([0]), positions=slots),
               dict(block_table=table.t()), dict(starts=slots.float()), dict(cu_q=slots), dict(status=slots)):
        with pytest.raises(o.KernelError):
            lay(**kw)
