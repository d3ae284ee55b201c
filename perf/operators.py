"""The operators of a cache that keeps keys and values in 4 bits: the step's slot maps and block tables made on the GPU, the
rotation and write of a step's keys and values, and the attention over the cache's pages.

Layer sizes are those of the Qwen2.5 configurations that ``tests/test_real_sizes_gpu.py`` and ``bench.py`` have (1.5B: 12 heads
over 2; 7B: 28 over 4; 14B: 40 over 8; head size 128) and generic ones.

A page of ``page_size`` positions is, per kv head, ``page_size / 16`` tiles of ``10 * head_dim`` bytes; a tile holds 16 positions.
A row's channels are taken in groups of 32; a group has a scale and a minimum in bfloat16 and stands for scale * code + minimum.

* key tile: 16 rows of head_dim / 2 bytes; word (4 bytes) t * NG + u of a row (NG = head_dim / 32, t = 0..3, u = 0..NG-1) holds
  channels 32 u + 8 t + 0..7, the lowest 4 bits first; then 16 rows of NG pairs (scale, minimum).
* value tile: for every group u, for g = 0..7, t = 0..3, p = 0..1 a word: its low half has row 4 t + 2 p, its high half row
  4 t + 2 p + 1, each the channels 32 u + 4 g + 0..3, lowest bits first; then for every u and t the scales of rows 4 t .. 4 t + 3
  and their minima.
"""
import random

import torch

own = False
DEVICE = "cuda:0"
PAGE = 16
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # The headline's decode step: eight requests at contexts up to 4,096 (latency).
        dict(name="layout_decode_8", op="layout", batch=8, portions="", ctx_min=3600, ctx_max=4096, width=256, lens=1),
        # A serving batch of 256 requests whose contexts reach 32,768: tables of 2,048 entries.
        dict(name="layout_decode_256", op="layout", batch=256, portions="", ctx_min=100, ctx_max=32768, width=2048, lens=2),
        # A step of continuous batching: portions of three prompts beside 37 decoding requests.
        dict(name="layout_prompts", op="layout", batch=37, portions="8191 1337 403", ctx_min=1, ctx_max=8192, width=1024, lens=3),
        # Keys and values of one token for each of 64 requests, 7B layer sizes.
        dict(name="write_decode_64", op="write", batch=64, portions="", ctx_max=4096, heads=28, kv_heads=4, head_dim=128, rotary=128,
             dtype="bf16", lens=4),
        # A prompt of 2,048 tokens, continued from a place inside a page, 7B layer sizes.
        dict(name="write_prompt_2048", op="write", batch=0, portions="2048", ctx_max=4096, heads=28, kv_heads=4, head_dim=128, rotary=128,
             dtype="bf16", lens=5),
        # One user, a short conversation, 1.5B layer sizes (latency).
        dict(name="attend_decode_1", op="attend", batch=1, portions="", ctx_min=700, ctx_max=700, heads=12, kv_heads=2, head_dim=128,
             window=0, dtype="bf16", lens=6),
        # The headline of bench.py: eight requests at contexts up to 4,096.
        dict(name="attend_decode_8", op="attend", batch=8, portions="", ctx_min=3600, ctx_max=4096, heads=12, kv_heads=2, head_dim=128,
             window=0, dtype="bf16", lens=7),
        # A serving batch at the 14B sizes: 64 requests with contexts of every length up to 16,384.
        dict(name="attend_decode_64", op="attend", batch=64, portions="", ctx_min=17, ctx_max=16384, heads=40, kv_heads=8, head_dim=128,
             window=0, dtype="bf16", lens=8),
        # Two requests over whole books: what a cache in 4 bits is kept for.
        dict(name="attend_decode_131072", op="attend", batch=2, portions="", ctx_min=100003, ctx_max=131072, heads=28, kv_heads=4,
             head_dim=128, window=0, dtype="bf16", lens=9),
        # A prompt of 2,048 tokens from its start, 7B sizes.
        dict(name="attend_prompt_2048", op="attend", batch=0, portions="2048+0", ctx_min=0, ctx_max=0, heads=28, kv_heads=4, head_dim=128,
             window=0, dtype="bf16", lens=10),
        # Continuous batching: a portion late in a long prompt beside 15 decoding requests.
        dict(name="attend_mixed", op="attend", batch=15, portions="384+8191", ctx_min=33, ctx_max=4096, heads=28, kv_heads=4, head_dim=128,
             window=0, dtype="bf16", lens=11),
        # The 32-bit engine with a window: short runs of five requests, another head size.
        dict(name="attend_float32", op="attend", batch=2, portions="9+580 4+100 13+0", ctx_min=200, ctx_max=600, heads=14, kv_heads=2,
             head_dim=64, window=256, dtype="f32", lens=12),
    ]


HEADS = ((12, 2), (28, 4), (40, 8), (14, 2), (16, 16), (8, 1), (32, 8), (5, 1))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    while True:
        case = _drawn(rng)
        lens, w = _lengths(case), work(case)
        padded = len(lens) * max(q for _, q in lens) * case.get("heads", 0) * max(s + q for s, q in lens)
        if max(w["bytes"], w["flops"] / 50) <= 6e8 and padded <= 1.5e9:      # not above the largest listed ones
            return case


def _drawn(rng):
    op = rng.choice(("layout", "write", "attend", "attend"))
    lens = rng.randrange(1 << 30)
    if op == "layout":
        batch = _log(rng, 1, 256)
        ctx = _log(rng, 16, 32768)
        many = rng.choice((0, 0, 1, 3))
        portions = [_log(rng, 2, min(8192, ctx)) for _ in range(many)]
        return dict(op=op, batch=batch, portions=" ".join(map(str, portions)), ctx_min=1, ctx_max=ctx, width=-(-ctx // PAGE), lens=lens)
    heads, kv_heads = rng.choice(HEADS)
    head_dim = rng.choice((32, 64, 96, 128, 128, 256))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    if op == "write":
        portions = [_log(rng, 2, 1500) for _ in range(rng.choice((0, 1, 2)))]
        rotary = rng.choice((head_dim, head_dim, head_dim // 2, 0))
        return dict(op=op, batch=_log(rng, 1, 64), portions=" ".join(map(str, portions)), ctx_max=_log(rng, 1600, 8000), heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim, rotary=rotary, dtype=dtype, lens=lens)
    kind = rng.choice(("decode", "decode", "short", "portion"))
    if kind == "portion":
        q, before = _log(rng, 17, 1500 if dtype == "bf16" else 200), rng.choice((0, _log(rng, 1, 6000)))
        batch, ctx, portions = rng.choice((0, 0, _log(rng, 1, 8))), before + q, ["%d+%d" % (q, before)]
    elif kind == "short":
        batch, ctx = _log(rng, 1, 8), _log(rng, 20, 8192)
        portions = ["%d+%d" % (_log(rng, 2, 16), rng.randrange(ctx)) for _ in range(rng.randrange(1, 5))]
    else:
        batch, portions = _log(rng, 1, 64), []
        ctx = _log(rng, 1, 65536 if dtype == "bf16" else 8192)
    return dict(op=op, batch=batch, portions=" ".join(portions), ctx_min=1, ctx_max=ctx, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                window=rng.choice((0, 0, 0, _log(rng, 1, max(2, ctx)))), dtype=dtype, lens=lens)


def _lengths(case):
    """(positions a request holds already, tokens that it brings) of every request."""
    r = random.Random(case["lens"])
    got = []
    for p in case["portions"].split():
        q, _, before = p.partition("+")
        got.append((int(before) if before else r.randrange(max(1, case["ctx_max"] - int(q) + 1)), int(q)))
    if case["op"] != "write":
        got += [(r.randint(case["ctx_min"], case["ctx_max"]) - 1, 1) for _ in range(case["batch"])]
    else:
        got += [(r.randrange(case["ctx_max"]), 1) for _ in range(case["batch"])]
    return got


# ------------------------------------------------------------------------------------ inputs
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _pages(counts, gen, spare):
    """Page lists of every request: distinct pages of a pool in no order."""
    total = sum(counts)
    order = torch.randperm(total + spare, generator=gen, device=DEVICE)[:total].to(torch.int32)
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return order, cu, total + spare


def _pool(num_pages, case, gen):
    """Key and value pages as a cache holds them that has been in use: codes of every value, scales of rows of unit spread."""
    hd, nkv = case["head_dim"], case["kv_heads"]
    both = []
    for values in (False, True):
        tiles = torch.randint(0, 256, (num_pages, nkv, PAGE // 16, 10 * hd), generator=gen, device=DEVICE, dtype=torch.uint8)
        scale = (torch.randn(num_pages, nkv, PAGE // 16, hd // 2, generator=gen, device=DEVICE) * 0.15).exp() * 0.27
        least = -7.5 * scale + 0.3 * torch.randn(scale.shape, generator=gen, device=DEVICE)
        pair = torch.stack((scale, least), -1) if not values else torch.stack((scale.unflatten(-1, (-1, 4)), least.unflatten(-1, (-1, 4))), -2)
        tiles[..., 8 * hd:] = pair.to(torch.bfloat16).flatten(3).view(torch.uint8)
        both.append(tiles)
    return both


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    host = random.Random(seed)
    lens = _lengths(case)
    starts, q_lens = [s for s, _ in lens], [q for _, q in lens]
    T, B = sum(q_lens), len(lens)
    counts = [-(-(s + q) // PAGE) for s, q in lens]
    pages, page_cu, pool = _pages(counts, gen, 1 + host.randrange(8))
    if case["op"] == "layout":
        empty = lambda *shape: torch.empty(shape, dtype=torch.int32, device=DEVICE)  # noqa: E731
        return dict(case=case, T=T, W=case["width"], starts=_i32(starts), q_lens=_i32(q_lens), page_cu=_i32(page_cu), pages=pages,
                    cu_q=empty(B + 1), kv_lens=empty(B), positions=empty(T), token_req=empty(T), table=empty(B, case["width"]),
                    slots=empty(T), status=torch.zeros(1, dtype=torch.int32, device=DEVICE))
    dtype = TYPES[case["dtype"]]
    heads, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    k_cache, v_cache = _pool(pool, case, gen)
    flat = pages.tolist()
    positions = [s + i for s, q in lens for i in range(q)]
    cu = [0]
    for q in q_lens:
        cu.append(cu[-1] + q)
    state = dict(case=case, T=T, k_cache=k_cache, v_cache=v_cache, positions=_i32(positions))
    if case["op"] == "write":
        slots = [flat[page_cu[b] + p // PAGE] * PAGE + p % PAGE for b, (s, q) in enumerate(lens) for p in range(s, s + q)]
        channels = torch.randn((heads + 2 * nkv) * hd, generator=gen, device=DEVICE) * 0.5
        qkv = torch.randn(T, (heads + 2 * nkv) * hd, generator=gen, device=DEVICE) * (1 + channels.abs()) + channels
        touched = sorted(set(s // PAGE for s in slots))
        most, rot = max(positions) + 1, case["rotary"]
        state |= dict(qkv=qkv.to(dtype), slots=_i32(slots), pages=_i32(touched), cos_sin=None)
        if rot:
            angle = torch.arange(most, device=DEVICE, dtype=torch.float64)[:, None] * 1e6 ** (
                -torch.arange(0, rot, 2, device=DEVICE, dtype=torch.float64) / rot)
            state["cos_sin"] = torch.stack((angle.cos(), angle.sin()), -1).float()
        return state
    W = max(counts)
    table = torch.full((B, W), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        row = pages[page_cu[b]:page_cu[b] + n].cpu()
        if case["window"]:      # pages that every query has left behind are given back
            row[:max(0, starts[b] - case["window"] + 1) // PAGE] = -1
        table[b, :n] = row
    q = (torch.randn(T, heads * hd, generator=gen, device=DEVICE) * 1.5).to(dtype)
    return state | dict(q=q, out=torch.empty_like(q), table=table.to(DEVICE), cu_q=_i32(cu), kv_lens=_i32([s + n for s, n in lens]),
                        token_req=_i32([b for b, n in enumerate(q_lens) for _ in range(n)]), q_lens=q_lens, longest=max(s + n for s, n in lens))


# ------------------------------------------------------------------------------------ one pass
def run(state):
    return {"layout": _layout, "write": _write, "attend": _attend}[state["case"]["op"]](state)


def _layout(s):
    if own:
        from coheryn_ai_studio_b200 import ops
        ops.step_layout(s["starts"], s["q_lens"], s["page_cu"], s["pages"], PAGE, s["table"], s["slots"], cu_q=s["cu_q"],
                        kv_lens=s["kv_lens"], positions=s["positions"], token_req=s["token_req"], status=s["status"])
        return [s[k] for k in ("cu_q", "kv_lens", "positions", "token_req", "table", "slots")]
    starts, q_lens, cu_p, W, T = s["starts"], s["q_lens"], s["page_cu"], s["W"], s["T"]
    B = starts.numel()
    cu = torch.cat((torch.zeros(1, dtype=torch.int32, device=DEVICE), torch.cumsum(q_lens, 0).to(torch.int32)))
    req = torch.repeat_interleave(torch.arange(B, dtype=torch.int32, device=DEVICE), q_lens, output_size=T)
    pos = starts[req] + torch.arange(T, dtype=torch.int32, device=DEVICE) - cu[req]
    col = torch.arange(W, dtype=torch.int32, device=DEVICE)
    at = (cu_p[:-1, None] + col).clamp(max=s["pages"].numel() - 1)
    table = torch.where(col < (cu_p[1:] - cu_p[:-1])[:, None], s["pages"][at], -1)
    return [cu, starts + q_lens, pos, req, table, table[req, pos // PAGE] * PAGE + pos % PAGE]


def _key_values(tiles):
    """[..., 10 hd] bytes -> [..., 16, hd] float32."""
    hd = tiles.shape[-1] // 10
    codes = tiles[..., :8 * hd].unflatten(-1, (16, 4, hd // 32, 4))
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)          # [..., 16, t, u, 8]
    codes = codes.transpose(-3, -2).flatten(-2).float()                    # [..., 16, u, 32]
    pair = tiles[..., 8 * hd:].contiguous().view(torch.bfloat16).unflatten(-1, (16, hd // 32, 2)).float()
    return (codes * pair[..., 0:1] + pair[..., 1:2]).flatten(-2)


def _value_values(tiles):
    hd = tiles.shape[-1] // 10
    codes = tiles[..., :8 * hd].unflatten(-1, (hd // 32, 8, 4, 2, 2, 2))    # u g t p row-in-pair byte
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()  # u g t p e 4
    n = codes.dim() - 6
    codes = codes.permute(*range(n), n + 2, n + 3, n + 4, n, n + 1, n + 5)  # t p e u g 4
    codes = codes.flatten(n, n + 2).flatten(-2)                            # [..., 16, u, 32]
    pair = tiles[..., 8 * hd:].contiguous().view(torch.bfloat16).unflatten(-1, (hd // 32, 4, 2, 4)).float()
    scale, least = (pair.select(-2, i).flatten(-2).transpose(-2, -1) for i in (0, 1))                        # [..., 16, u]
    return (codes * scale[..., None] + least[..., None]).flatten(-2)


def _held(x):
    """What rows [..., hd] of a compute type become in 4 bits."""
    g = x.float().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) / torch.full((), 15.0, device=x.device)).to(torch.bfloat16).float()
    least = lo.to(torch.bfloat16).float()
    codes = torch.where(scale > 0, ((g - least) / scale).round().clamp(0, 15), 0.0)
    return (codes * scale + least).flatten(-2)


def _write(s):
    c = s["case"]
    heads, nkv, hd, rot = c["heads"], c["kv_heads"], c["head_dim"], c["rotary"]
    dtype = s["qkv"].dtype
    if own:
        from coheryn_ai_studio_b200 import ops
        q = ops.rope_kv4_write(s["qkv"], s["positions"], s["cos_sin"], s["slots"], s["k_cache"], s["v_cache"], heads, nkv, hd, rot, PAGE)
        return [q, *ops.kv4_pages(s["k_cache"], s["v_cache"], s["pages"], hd, PAGE, dtype)]
    qkv = s["qkv"].float().unflatten(-1, (-1, hd))
    turned = qkv[:, :heads + nkv]
    if rot:
        turn = s["cos_sin"][s["positions"]][:, None]
        cos, sin = turn[..., 0], turn[..., 1]
        a, b = turned[..., :rot // 2], turned[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin, turned[..., rot:]), -1)
    turned = turned.to(dtype)
    pages = s["pages"]
    place = torch.zeros(s["k_cache"].shape[0], dtype=torch.int32, device=DEVICE)
    place[pages] = torch.arange(pages.numel(), dtype=torch.int32, device=DEVICE)
    page, row = place[s["slots"] // PAGE], s["slots"] % PAGE
    k = _key_values(s["k_cache"][pages]).flatten(2, 3)
    v = _value_values(s["v_cache"][pages]).flatten(2, 3)
    k[page, :, row] = _held(turned[:, heads:])
    v[page, :, row] = _held(qkv[:, heads + nkv:])
    return [turned[:, :heads].flatten(1), k.to(dtype), v.to(dtype)]


def _attend(s):
    c = s["case"]
    heads, nkv, hd, window = c["heads"], c["kv_heads"], c["head_dim"], c["window"]
    if own:
        from coheryn_ai_studio_b200 import ops
        ops.attention_kv4_rows(s["q"], s["out"], s["k_cache"], s["v_cache"], s["table"], s["token_req"], s["positions"], heads, nkv, hd, PAGE,
                               window or None, hd ** -0.5, cu_q=s["cu_q"], kv_lens=s["kv_lens"], q_lens=s["q_lens"], max_kv_len=s["longest"])
        return s["out"]
    cu, lens, G, most = s["cu_q"], s["kv_lens"], heads // nkv, max(s["q_lens"])
    table = s["table"].clamp(min=0)
    k = _key_values(s["k_cache"][table]).movedim(2, 1).flatten(2, 4)        # [B, nkv, positions, hd]
    v = _value_values(s["v_cache"][table]).movedim(2, 1).flatten(2, 4)
    i = torch.arange(most, device=DEVICE)
    n = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + i).clamp(max=s["T"] - 1)                        # [B, most]
    q = s["q"].float()[rows].unflatten(-1, (nkv, G, hd)).permute(0, 2, 3, 1, 4).flatten(2, 3)     # [B, nkv, G most, hd]
    score = (q @ k.transpose(-1, -2)).unflatten(2, (G, most)) * hd ** -0.5
    place = (lens - n)[:, None] + i
    t = torch.arange(k.shape[2], device=DEVICE)
    seen = t <= place[..., None]
    if window:
        seen &= t > place[..., None] - window
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (G, most)).permute(0, 3, 1, 2, 4).flatten(2)           # [B, most, heads hd]
    return o[s["token_req"], torch.arange(s["T"], device=DEVICE) - cu[s["token_req"]]].to(s["q"].dtype)


# ------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    lens = _lengths(case)
    T, B = sum(q for _, q in lens), len(lens)
    pages = sum(-(-(s + q) // PAGE) for s, q in lens)
    if case["op"] == "layout":
        return {"bytes": 4.0 * (3 * B + 1 + pages + B + 1 + B + 3 * T + B * case["width"]), "flops": 0.0}
    e = 2 if case["dtype"] == "bf16" else 4
    heads, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    row = nkv * 2 * hd * 5 / 8                                              # bytes of a position's keys and values
    if case["op"] == "write":
        touched = sum((s + q - 1) // PAGE - s // PAGE + 1 for s, q in lens)
        q = T * heads * hd * e if case["rotary"] else 0
        return {"bytes": T * 2 * nkv * hd * e + 2 * q + T * row + touched * PAGE * (row + 2 * nkv * hd * e),
                "flops": T * (3.0 * (heads + nkv) * case["rotary"] + 6.0 * 2 * nkv * hd) + 2.0 * touched * PAGE * 2 * nkv * hd}
    w = case["window"]
    keys = pairs = 0
    for s, q in lens:
        keys += s + q - (max(0, s - w + 1) if w else 0)
        pairs += sum(min(p + 1, w) for p in range(s, s + q)) if w else q * s + q * (q + 1) // 2
    return {"bytes": 2 * T * heads * hd * e + keys * row, "flops": 4.0 * hd * heads * pairs}


# ------------------------------------------------------------------------------------ in 64 bits
def _at(tiles, values):
    """Every value of the tiles [..., 10 hd] as [..., 16, hd] in 64 bits: code and pair of each row and channel by its place."""
    hd = tiles.shape[-1] // 10
    r, c = torch.arange(16, device=DEVICE)[:, None], torch.arange(hd, device=DEVICE)[None]
    u = c // 32
    if not values:
        t, i = c % 32 // 8, c % 8
        nibble = (r * hd // 8 + t * (hd // 32) + u) * 8 + i
        scale = 8 * hd + (r * (hd // 32) + u) * 4
        least = scale + 2
    else:
        g, j = c % 32 // 4, c % 4
        nibble = (((u * 8 + g) * 4 + r // 4) * 2 + r % 4 // 2) * 8 + r % 2 * 4 + j
        scale = 8 * hd + ((u * 4 + r // 4) * 8 + r % 4) * 2
        least = scale + 8
    byte = lambda at: tiles[..., at.flatten()].unflatten(-1, at.shape).to(torch.int32)  # noqa: E731
    code = (byte(nibble // 2) >> (4 * (nibble % 2))) & 15
    wide = lambda at: (((byte(at + 1) << 24) | (byte(at) << 16)).view(torch.float32)).double()  # noqa: E731
    return code.double() * wide(scale) + wide(least)


def exact(case, seed):
    if case["op"] == "layout":
        return None          # whole numbers
    s = prepare(case, seed)
    return _exact_write(s) if case["op"] == "write" else _exact_attend(s)


def _exact_write(s):
    c = s["case"]
    heads, nkv, hd, rot, T = c["heads"], c["kv_heads"], c["head_dim"], c["rotary"], s["T"]
    x = s["qkv"].double().view(T, heads + 2 * nkv, hd).clone()
    if rot:
        z = torch.complex(x[:, :heads + nkv, :rot // 2], x[:, :heads + nkv, rot // 2:rot])
        turn = s["cos_sin"].double()[s["positions"].long()]
        z = z * torch.complex(turn[..., 0], turn[..., 1])[:, None]
        x[:, :heads + nkv, :rot // 2], x[:, :heads + nkv, rot // 2:rot] = z.real, z.imag
    q = x[:, :heads].reshape(T, -1)
    if s["qkv"].dtype == torch.float32:
        return [q, None, None]      # a value next to a border between two codes has no answer in more bits than the operator's
    x = x.to(torch.bfloat16).double()
    got = [q]
    for tiles, rows, values in ((s["k_cache"], x[:, heads:heads + nkv], False), (s["v_cache"], x[:, heads + nkv:], True)):
        group = rows.reshape(T, nkv, hd // 32, 32)
        least = group.min(-1, keepdim=True).values
        scale = ((group.max(-1, keepdim=True).values - least) / 15).float().to(torch.bfloat16).double()
        code = torch.where(scale == 0, torch.zeros_like(group), ((group - least) / scale).round().clamp(0, 15))
        kept = (least + scale * code).reshape(T, nkv, hd)
        pages = s["pages"].long()
        out = _at(tiles[pages], values).reshape(len(pages), nkv, PAGE, hd)
        which = torch.searchsorted(pages, s["slots"].long() // PAGE)
        out[which, :, s["slots"].long() % PAGE] = kept
        got.append(out)
    return got


def _exact_attend(s):
    c = s["case"]
    heads, nkv, hd, window = c["heads"], c["kv_heads"], c["head_dim"], c["window"]
    got, at = [], 0
    for b, n in enumerate(s["q_lens"]):
        length = int(s["kv_lens"][b])
        first = max(0, length - n - window + 1) // PAGE if window else 0
        pages = s["table"][b, first:-(-length // PAGE)].long()
        k, v = (_at(x[pages], which).permute(1, 0, 2, 3, 4).reshape(nkv, -1, hd)[:, :length - first * PAGE]
                for x, which in ((s["k_cache"], False), (s["v_cache"], True)))
        q = s["q"][at:at + n].double().reshape(n, nkv, heads // nkv, hd)
        score = torch.einsum("ngmd,gtd->gmnt", q, k) / hd ** 0.5
        t = torch.arange(first * PAGE, length, device=DEVICE)
        p = torch.arange(length - n, length, device=DEVICE)[:, None]
        hidden = t > p
        if window:
            hidden |= p - t >= window
        weight = torch.softmax(score.masked_fill(hidden, float("-inf")), -1)
        got.append(torch.einsum("gmnt,gtd->ngmd", weight, v).reshape(n, heads * hd))
        at += n
    return torch.cat(got)
