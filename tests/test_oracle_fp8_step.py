"""The float64 oracle of the 8-bit serving step against known answers."""

from __future__ import annotations

import torch

from kernel_lab.kv_cache import build_paged_kv, quantize_fp8_pages
from oracle import fp8_step as ref
from oracle import reference


def test_e4m3_rounding_matches_torch_on_every_border():
    values = ref._MAGNITUDES
    mid = (values[1:] + values[:-1]) / 2  # ties, exact in float32
    x = torch.cat([values, mid, mid * (1 + 2.0**-22), mid * (1 - 2.0**-22), torch.tensor([464.0, 465.0, float("inf")])])
    x = torch.cat([x, -x, torch.tensor([float("nan")])]).float()
    want = x.to(torch.float8_e4m3fn).float().double()
    # torch rounds magnitudes up to 464 down to 448 and gives NaN beyond, as the oracle does.
    torch.testing.assert_close(ref.round_e4m3(x), want, rtol=0, atol=0, equal_nan=True)


def test_norm_known_answer():
    """A row of 3s and a 4 in unit weights: y = x / rms, the largest takes 448."""
    x = torch.tensor([[3.0, 4.0]])
    t, scale, _ = ref.norm_fp8(x, None, torch.ones(2), eps=0.0)
    rms = (12.5) ** 0.5
    torch.testing.assert_close(scale, torch.tensor([[4 / rms / 448]], dtype=torch.float64))
    torch.testing.assert_close(t, torch.tensor([[336.0, 448.0]], dtype=torch.float64))


def test_decode_with_equal_page_scales_is_decode_with_head_scales():
    g = torch.Generator().manual_seed(1)
    lens = [1, 16, 33]
    keys = [torch.randn(n, 2, 64, generator=g) for n in lens]
    kv = quantize_fp8_pages(build_paged_kv(keys, [k.flip(0) for k in keys], 16))
    q = torch.randn(3, 8, 64, generator=g)
    ks, vs = torch.tensor([0.01, 0.02]), torch.tensor([0.03, 0.005])
    pages = kv.k_cache.shape[0]
    got, _ = ref.decode(q, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens, ks.expand(pages, 2), vs.expand(pages, 2))
    want = reference.paged_decode_attention_fp8(q, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens, ks, vs, None)
    torch.testing.assert_close(got.float(), want, atol=2e-6, rtol=2e-6)


def test_append_then_decode_is_close_to_the_unrounded_attention():
    """Three appends to a page, the last one larger: the scale grows and the earlier codes are rounded again."""
    g = torch.Generator().manual_seed(2)
    cache = {n: torch.full((3, 16, 1, 64), float("nan"), dtype=torch.float64) for n in ("k", "v")}
    cache |= {"k_scale": torch.full((3, 1), float("nan")), "v_scale": torch.full((3, 1), float("nan")),
              "bounds": torch.zeros(3, 1, 2, 64, dtype=torch.float64), "block_table": torch.tensor([[2, 0]])}
    x = torch.randn(20, 1, 64, generator=g)
    x[10:] *= 3
    for i, (a, b) in enumerate([(0, 5), (5, 10), (10, 20)]):
        ref.append(x[a:b], -x[a:b], cache, torch.tensor([b]), torch.tensor([0, b - a]))
    back = torch.cat([cache["k"][2, :, 0] * cache["k_scale"][2, 0].double(), cache["k"][0, :4, 0] * cache["k_scale"][0, 0].double()])
    # Rounded at most three times, each within half a step (2^-4 of the value, or of the smallest normal code).
    off = (back - x[:, 0].double()).abs()
    assert bool((off <= 3 * (x[:, 0].double().abs() * 2.0**-4 + cache["k_scale"][2, 0].double() * 2.0**-10)).all())
    torch.testing.assert_close(cache["bounds"][2, 0, 0], cache["k"][2, :, 0].amin(0))
    torch.testing.assert_close(cache["bounds"][2, 0, 1], cache["k"][2, :, 0].amax(0))
    assert torch.isnan(cache["k"][1]).all() and torch.isnan(cache["k"][0, 4:]).all()


def test_selected_bounds_are_upper_bounds_and_ties_go_low():
    g = torch.Generator().manual_seed(3)
    keys = [torch.randn(16 * 9, 1, 64, generator=g)]
    kv = quantize_fp8_pages(build_paged_kv(keys, keys, 16))
    q = torch.randn(1, 2, 64, generator=g)
    table, lens = ref.select(q, kv.k_bounds, kv.k_scale, kv.block_table, kv.seq_lens, 4, 16)
    assert lens.tolist() == [[64]] and table[0, 0, 0] == kv.block_table[0, 0] and table[0, 0, 3] == kv.block_table[0, 8]
    flat = torch.zeros_like(q)  # every page scores 0
    table, _ = ref.select(flat, kv.k_bounds, kv.k_scale, kv.block_table, kv.seq_lens, 4, 16)
    assert table[0, 0].tolist() == kv.block_table[0, [0, 1, 2, 8]].tolist()


def test_norm_is_the_library_norm_before_its_rounding():
    g = torch.Generator().manual_seed(4)
    x, r, w = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 96), (5, 96), (96,)))
    t, scale, res = ref.norm_fp8(x.float(), r.float(), w, eps=1e-5, group=32)
    want = torch.nn.functional.rms_norm((x.float() + r.float()).double(), (96,), w, eps=1e-5)
    torch.testing.assert_close((t.reshape(5, 3, 32) * scale[..., None]).reshape(5, 96), want)
    torch.testing.assert_close(t.reshape(5, 3, 32).abs().amax(-1), torch.full((5, 3), 448.0, dtype=torch.float64))
    assert torch.equal(res, x.float() + r.float())


def test_append_to_empty_pages_is_the_quantised_cache():
    g = torch.Generator().manual_seed(5)
    lens = [16, 1, 40]
    keys = [torch.randn(n, 2, 64, generator=g) for n in lens]
    values = [3 * k.flip(0) for k in keys]
    want = quantize_fp8_pages(build_paged_kv(keys, values, 16))
    shape = want.k_cache.shape
    cache = {n: torch.full(shape, float("nan"), dtype=torch.float64) for n in ("k", "v")}
    cache |= {n + "_scale": torch.full(shape[::2], float("nan")) for n in ("k", "v")}
    cache |= {"bounds": torch.zeros(shape[0], 2, 2, 64, dtype=torch.float64), "block_table": want.block_table}
    ref.append(torch.cat(keys), torch.cat(values), cache, torch.tensor(lens), torch.tensor([0, 16, 17, 57]))
    for name, codes, scales in (("k", want.k_cache, want.k_scale), ("v", want.v_cache, want.v_scale)):
        torch.testing.assert_close(cache[name], codes.double(), rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(cache[name + "_scale"], scales, rtol=0, atol=0, equal_nan=True)
    held = torch.cat([want.block_table[b, : (n + 15) // 16] for b, n in enumerate(lens)]).long()
    torch.testing.assert_close(cache["bounds"][held], want.k_bounds.double()[held], rtol=0, atol=0)
