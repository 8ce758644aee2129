"""gfx950 append into the paged FP8 cache against the oracle, code for code.

The definition is a chain of single float32 roundings (a division for the scale, a product and a division for codes
rounded again, a division for new ones, then the rounding to E4M3), which the oracle takes one by one, so codes, scales
and bounds have to be equal.
"""

from __future__ import annotations

import pytest
import torch

from oracle import fp8_step as ref
from tests.conftest import DTYPES

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
POISON = 0x5B  # a finite code in slots that nothing has written


def make(lens, heads, dim, page, spare=3, seed=0, bounds=True):
    """An empty cache with room for `lens` tokens a sequence, on the GPU, and the oracle's copy of it."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max([*need, 1]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    codes = torch.full((pages, page, heads, dim), POISON, dtype=torch.uint8)
    scale = 0.001 + torch.rand(pages, heads, generator=g)
    dev = {
        "k": codes.cuda().view(F8), "v": codes.cuda().view(F8), "k_scale": scale.cuda(), "v_scale": scale.cuda().clone(),
        "bounds": torch.full((pages, heads, 2, dim), POISON, dtype=torch.uint8).cuda().view(F8) if bounds else None,
        "block_table": table.cuda(),
    }
    host = {n: None if t is None else t.cpu().float().double() if n in ("k", "v", "bounds") else t.cpu().clone() for n, t in dev.items()}
    return dev, host


def call(ops, k, v, dev, lens, offsets=None):
    ops.append_kv_fp8(k, v, dev["k"], dev["v"], dev["k_scale"], dev["v_scale"], dev["block_table"], lens.cuda(),
                      new_offsets=None if offsets is None else offsets.cuda(), k_bounds=dev["bounds"])


def same(dev, host):
    for name, want in host.items():
        if want is not None:
            got = dev[name].cpu()
            got = got.float().double() if got.dtype == F8 else got
            torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True, msg=lambda m, n=name: f"{n}: {m}")


def tokens(n, heads, dim, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, n, heads, dim, generator=g) * size * torch.exp(torch.randn(2, n, heads, 1, generator=g))
    return x.to(dtype)


def step(ops, dev, host, lens, news, heads, dim, dtype, seed, size=1.0, offsets=True):
    k, v = tokens(sum(news), heads, dim, dtype, seed, size)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    off = torch.tensor([0, *news]).cumsum(0).to(torch.int32) if offsets else None
    call(ops, k.cuda(), v.cuda(), dev, lens_t, off)
    ref.append(k, v, host, lens_t, off)
    same(dev, host)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("heads", "dim", "page"), [(8, 128, 16), (1, 64, 16), (2, 256, 32), (3, 128, 64), (1, 256, 128), (5, 64, 48)])
def test_chunks_then_single_tokens(gpu_ops, heads, dim, page, dtype):
    """A ragged first chunk, a second behind it, then single tokens, some of them larger than all before."""
    lens = [1, page - 1, page, page + 1, 3 * page + 5, 7]
    room = [n + 2 * page + 40 for n in lens]
    dev, host = make(room, heads, dim, page)
    step(gpu_ops, dev, host, lens, lens, heads, dim, dtype, 1)
    news = [page, 1, 2, page + 3, 3, 2 * page]
    lens = [a + b for a, b in zip(lens, news)]
    step(gpu_ops, dev, host, lens, news, heads, dim, dtype, 2, size=2.0)
    for i in range(4):
        lens = [n + 1 for n in lens]
        step(gpu_ops, dev, host, lens, [1] * len(lens), heads, dim, dtype, 3 + i, size=4.0**i, offsets=i % 2 == 0)


@pytest.mark.parametrize("page", [16, 64])
def test_long_ragged_chunks(gpu_ops, page):
    lens = [700, 1, 0, 333, 512, 15]
    dev, host = make([n + 3 for n in lens], 4, 128, page)
    step(gpu_ops, dev, host, lens, lens, 4, 128, torch.bfloat16, 5)


def test_without_bounds(gpu_ops):
    dev, host = make([50, 20], 2, 128, 16, bounds=False)
    step(gpu_ops, dev, host, [33, 20], [33, 20], 2, 128, torch.float16, 1)
    step(gpu_ops, dev, host, [34, 20], [1, 0], 2, 128, torch.float16, 2, size=3.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_unaligned_inputs(gpu_ops, dtype):
    """The keys and values of one fused projection, and rows that start at odd addresses."""
    heads, dim = 4, 128
    dev, host = make([40, 40], heads, dim, 16)
    qkv = torch.randn(37, 3 * heads, dim).to(dtype)
    k, v = qkv[:, heads : 2 * heads], qkv[:, 2 * heads :]
    lens, off = torch.tensor([17, 20], dtype=torch.int32), torch.tensor([0, 17, 37], dtype=torch.int32)
    on = qkv.cuda()
    call(gpu_ops, on[:, heads : 2 * heads], on[:, 2 * heads :], dev, lens, off)
    ref.append(k, v, host, lens, off)
    same(dev, host)
    flat = torch.randn(2 * (heads * dim + 1) + 3).to(dtype)
    odd = flat.as_strided((2, heads, dim), (heads * dim + 1, dim, 1), 1)
    turned = flat.as_strided((2, heads, dim), (dim, 2 * dim, 1), 3)  # heads outside tokens
    on = flat.cuda()
    lens = lens + 1
    call(gpu_ops, on.as_strided(odd.shape, odd.stride(), 1), on.as_strided(turned.shape, turned.stride(), 3), dev, lens)
    ref.append(odd, turned, host, lens)
    same(dev, host)


def test_values_that_are_not_finite_and_zeros(gpu_ops):
    dev, host = make([20, 20, 20], 1, 64, 16)
    k, v = tokens(15, 1, 64, torch.float32, 0)
    k[0, 0, 3], k[1, 0, 3], v[2, 0, 5], v[3, 0, 5] = float("nan"), float("inf"), float("-inf"), float("nan")
    k[5:10], v[5:10] = 0, 0  # a page of zeros, whose scale has to grow with the first value
    k[10:], v[10:] = k[10:] * 1e-42, v[10:] * 1e-37
    k[:5, 0, 9] = float("nan")  # a dimension without a number
    lens, off = torch.tensor([5, 5, 5], dtype=torch.int32), torch.tensor([0, 5, 10, 15], dtype=torch.int32)
    call(gpu_ops, k.cuda(), v.cuda(), dev, lens, off)
    ref.append(k, v, host, lens, off)
    same(dev, host)
    assert float(dev["k_scale"][int(dev["block_table"][1, 0]), 0]) == ref.MIN_SCALE
    k, v = tokens(3, 1, 64, torch.float32, 1)
    call(gpu_ops, k.cuda(), v.cuda(), dev, lens + 1)
    ref.append(k, v, host, lens + 1)
    same(dev, host)


def test_what_is_left_alone(gpu_ops):
    """Idle rows (length 0), lengths below the chunk, offsets outside the rows, columns and pages out of range."""
    heads, dim, page = 2, 64, 16
    dev, host = make([40] * 7, heads, dim, page, spare=2)
    table = host["block_table"]
    table[3, 0], table[4, 0] = -1, dev["k"].shape[0]
    dev["block_table"].copy_(table)
    width = table.shape[1] * page
    k, v = tokens(7, heads, dim, torch.bfloat16, 0)
    lens = torch.tensor([0, 1, 1, 1, 1, width + 1, width], dtype=torch.int32)
    call(gpu_ops, k.cuda(), v.cuda(), dev, lens)
    ref.append(k, v, host, lens)
    same(dev, host)
    off = torch.tensor([0, 2, 2, 9, 5, -1, 1, 7], dtype=torch.int32)
    lens = torch.tensor([1, 1, 30, 30, 30, 30, 6], dtype=torch.int32)
    call(gpu_ops, k.cuda(), v.cuda(), dev, lens, off)
    # Sequence 6 alone has rows 1 .. 6 and a length that holds them.
    only = torch.tensor([0, 0, 0, 0, 0, 0, 0, 6], dtype=torch.int32)
    ref.append(k[1:], v[1:], host, torch.tensor([0, 0, 0, 0, 0, 0, 6]), only)
    same(dev, host)


def test_a_page_in_the_middle_of_a_chunk_out_of_range(gpu_ops):
    dev, host = make([60], 1, 64, 16)
    host["block_table"][0, 1] = 1 << 20
    dev["block_table"].copy_(host["block_table"])
    step(gpu_ops, dev, host, [50], [50], 1, 64, torch.float16, 0)


def test_empty_calls(gpu_ops):
    dev, host = make([5], 1, 64, 16)
    none = torch.empty(0, 1, 64, device="cuda", dtype=torch.float16)
    call(gpu_ops, none, none, dev, torch.tensor([5], dtype=torch.int32), torch.tensor([0, 0], dtype=torch.int32))
    same(dev, host)
    dev["block_table"] = dev["block_table"][:0]
    call(gpu_ops, none, none, dev, torch.empty(0, dtype=torch.int32))
    host["block_table"] = host["block_table"][:0]
    same(dev, host)


def test_pages_far_into_a_large_cache(gpu_ops):
    """Page offsets past 2^32 bytes."""
    heads, dim, page = 8, 256, 128
    pages = (1 << 32) // (heads * dim * page) + 10
    k_cache = torch.zeros(pages, page, heads, dim, dtype=torch.uint8, device="cuda")
    v_cache = torch.zeros_like(k_cache)
    scale = torch.zeros(2, pages, heads, device="cuda")
    table = torch.tensor([[pages - 1], [2]], dtype=torch.int32, device="cuda")
    k, v = tokens(2, heads, dim, torch.bfloat16, 0)
    gpu_ops.append_kv_fp8(k.cuda(), v.cuda(), k_cache.view(F8), v_cache.view(F8), scale[0], scale[1], table,
                          torch.tensor([128, 1], dtype=torch.int32, device="cuda"))
    for b, (where, slot) in enumerate([(pages - 1, 127), (2, 0)]):
        want = ref.round_e4m3(k[b].float() / scale[0, where].cpu()[:, None])
        torch.testing.assert_close(k_cache[where, slot].view(F8).float().cpu().double(), want, rtol=0, atol=0)
    assert int((k_cache.view(torch.int64) != 0).sum()) <= 2 * heads * dim // 8


def test_refusals(gpu_ops):
    dev, _ = make([20, 20], 2, 64, 16)
    k, v = (t.cuda() for t in tokens(2, 2, 64, torch.float16, 0))
    lens = torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="one token per sequence"):
        call(gpu_ops, k[:1], v[:1], dev, lens)
    with pytest.raises(RuntimeError, match="of the cache"):
        call(gpu_ops, k[:, :1], v[:, :1], dev, lens)
    with pytest.raises(RuntimeError, match="share a dtype"):
        call(gpu_ops, k, v.float(), dev, lens)
    with pytest.raises(RuntimeError, match="dtype"):
        call(gpu_ops, k.double(), v.double(), dev, lens)
    with pytest.raises(RuntimeError, match="new_offsets"):
        call(gpu_ops, k, v, dev, lens, torch.tensor([0, 2], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="int32"):
        call(gpu_ops, k, v, dev, lens.long())
    for name, bad, match in [("k_scale", dev["k_scale"][:, :1], "k_scale"), ("v", dev["v"].view(torch.uint8), "float8"),
                             ("bounds", dev["bounds"][:, :, :1], "k_bounds"), ("k_scale", dev["k_scale"].half(), "k_scale")]:
        with pytest.raises((RuntimeError, ValueError), match=match):
            call(gpu_ops, k, v, {**dev, name: bad}, lens)
    small, _ = make([20, 20], 2, 64, 8)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        call(gpu_ops, k, v, small, lens)


def test_graph_replays(gpu_ops):
    """One captured call, replayed with new tokens and lengths, equals eager calls."""
    heads, dim = 8, 128
    dev, host = make([40] * 6, heads, dim, 16)
    k, v = (t.cuda() for t in tokens(6, heads, dim, torch.bfloat16, 0))
    lens = torch.zeros(6, dtype=torch.int32, device="cuda")
    run = lambda: gpu_ops.append_kv_fp8(k, v, dev["k"], dev["v"], dev["k_scale"], dev["v_scale"], dev["block_table"], lens,  # noqa: E731
                                        k_bounds=dev["bounds"])
    run()  # every row idle
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(5):
        new = tokens(6, heads, dim, torch.bfloat16, i, size=2.0**i)
        k.copy_(new[0])
        v.copy_(new[1])
        lens.copy_(torch.tensor([i + 1, i + 1, 16 + i, 0, 20 + i, i + 1], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        ref.append(new[0], new[1], host, lens.cpu())
        same(dev, host)
