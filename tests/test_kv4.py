"""The 4-bit cache without a GPU: its format's restatement, the sizes it takes and refuses, how a user asks for it."""
import numpy as np
import pytest
import torch

import kv4_cases as kc
from coheryn_ai_studio_b200 import ops
from coheryn_ai_studio_b200.cache.manager import CacheManager
from coheryn_ai_studio_b200.cli import build_parser
from coheryn_ai_studio_b200.parts.base import PagedKV


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("values", [False, True])
def test_every_channel_has_a_place_of_its_own(hd, values):
    place, scale, minimum = kc.places(hd, values)
    assert sorted(place.ravel()) == list(range(16 * hd))
    pairs = np.unique(np.concatenate([scale.ravel(), minimum.ravel()]))
    assert len(pairs) == 2 * 16 * hd // 32 and pairs.min() == 8 * hd and pairs.max() == 10 * hd - 2


@pytest.mark.parametrize("values", [False, True])
def test_rows_come_back_within_half_a_step(values):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((5, 16, 64)) * 10.0 ** rng.integers(-3, 4, (5, 16, 1))).astype(np.float32)
    back = kc.unpack(kc.pack(x, values), values)
    g = x.reshape(5, 16, 2, 32)
    spread = (g.max(-1) - g.min(-1))[..., None]
    # half a step; the scale off by 2^-8 of itself over up to 15 steps, the minimum by 2^-8 of itself (and clamping to the last code)
    tol = spread / 30 + 2.0 ** -8 * (2 * spread + np.abs(g.min(-1))[..., None]) + 1e-30
    assert (np.abs(back.reshape(g.shape) - g) <= tol).all()


def test_values_that_are_not_finite_make_their_group_not_a_number():
    x = np.ones((1, 16, 64), np.float32)
    x[0, 3, 40], x[0, 7, 2] = np.inf, np.nan
    back = kc.unpack(kc.pack(x, True), True).reshape(16, 2, 32)
    bad = np.zeros((16, 2), bool)
    bad[3, 1] = bad[7, 0] = True
    assert np.isnan(back[bad]).all() and (back[~bad] == 1).all()


def test_page_shapes():
    assert ops.kv4_page_shape(8, 32, 128) == (8, 2, 1280)
    for args in ((8, 16, 48), (8, 16, 16), (8, 16, 288), (8, 24, 64), (8, 0, 64), (8, 8, 64)):
        with pytest.raises(ops.KernelError):
            ops.kv4_page_shape(*args)


def manager(*needs, kv_bits=4, page_size=16):
    return CacheManager(list(needs), [None] * len(needs), torch.bfloat16, "cpu", page_size=page_size, num_pages=3, max_requests=2, kv_bits=kv_bits)


def test_cache_of_four_bits():
    need = PagedKV(2, 64, None, four_bits=True)
    cache, plain = manager(need, need), manager(need, need, kv_bits=None)
    for c in cache.layer_caches():
        assert c.four_bits and c.k.dtype == torch.uint8 and tuple(c.k.shape[1:]) == ops.kv4_page_shape(2, 16, 64) and not c.k.any()
    assert not any(c.four_bits for c in plain.layer_caches())
    assert plain.bytes_per_token() * 5 == cache.bytes_per_token() * 16


@pytest.mark.parametrize("need,kw,message", [
    (PagedKV(2, 64, None, four_bits=True), dict(kv_bits=8), "not in 8"), (PagedKV(2, 64, None, four_bits=True), dict(page_size=24), "multiple of 16"),
    (PagedKV(2, 64, None), {}, "does not read"), (PagedKV(2, 48, None, four_bits=True), {}, "does not read"),
    (PagedKV(2, 64, None, v_head_dim=32, four_bits=True), {}, "does not read"), (PagedKV(2, 64, 32, keep_first=4, four_bits=True), {}, "does not read")])
def test_what_a_cache_of_four_bits_refuses(need, kw, message):
    with pytest.raises(ValueError, match=message):
        manager(need, **kw)


def test_command_line():
    assert build_parser().parse_args(["run", "m", "--tokens", "1", "--kv-bits", "4"]).kv_bits == 4
    assert build_parser().parse_args(["run", "m", "--tokens", "1"]).kv_bits is None
    with pytest.raises(SystemExit):
        build_parser().parse_args(["run", "m", "--tokens", "1", "--kv-bits", "8"])


def test_operands_on_the_host_are_refused():
    x = torch.zeros(2, 192, dtype=torch.bfloat16)
    words, pages = torch.zeros(2, dtype=torch.int32), torch.zeros((1,) + ops.kv4_page_shape(1, 16, 64), dtype=torch.uint8)
    with pytest.raises(ops.KernelError):
        ops.rope_kv4_write(x, None, None, words, pages, pages, 1, 1, 64, 0, 16)
    with pytest.raises(ops.KernelError):
        ops.kv4_pages(pages, pages, words, 64, 16, torch.bfloat16)
    with pytest.raises(ops.KernelError):
        ops.attention_kv4_rows(x[:, :64], torch.zeros(2, 64, dtype=torch.bfloat16), pages, pages, words[None], words, words, 1, 1, 64, 16, None, 1.0)
    with pytest.raises(ops.KernelError):
        ops.step_layout(words, words, torch.zeros(3, dtype=torch.int32), words, 16, torch.zeros(2, 3, dtype=torch.int32))
