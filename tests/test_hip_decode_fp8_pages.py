"""gfx950 decode over the FP8 cache with scales per page and KV head, and over block tables per KV head, against the
float64 oracle.

Tolerance, per output: half a step of the output's type, and 2^-15 of sum p |v|. The second term covers the weights'
bf16 pair (2^-17), the exponent's argument (scores of up to some tens in log2 units, summed in fp32: 2^-18 or so), the
hardware exponential and the fp32 sums.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from kernel_lab import _native
from kernel_lab.kv_cache import PagedFP8, build_paged_kv, quantize_fp8_pages
from oracle import fp8_step as ref
from tests.conftest import ulp_of

pytestmark = pytest.mark.gpu

QDTYPES = [torch.float16, torch.bfloat16]


def problem(lens, hq, hkv, d, dtype, page=16, seed=0, spread=1.0):
    """q and a cache whose pages differ in size by e^(spread N(0, 1)); lengths of 0 get no page of their own."""
    g = torch.Generator().manual_seed(seed)
    keys, values = [], []
    for n in lens:
        n = max(n, 1)
        size = torch.exp(spread * torch.randn(2, (n + page - 1) // page, hkv, generator=g)).repeat_interleave(page, 1)[:, :n]
        keys.append(torch.randn(n, hkv, d, generator=g) * size[0, ..., None])
        values.append(torch.randn(n, hkv, d, generator=g) * size[1, ..., None])
    kv = quantize_fp8_pages(build_paged_kv(keys, values, page, seed=seed))
    kv.seq_lens = torch.tensor(lens, dtype=torch.int32)
    q = torch.randn(len(lens), hq, d, generator=g).to(dtype)
    return q, kv


def on_gpu(kv):
    return PagedFP8(*(t.cuda() if isinstance(t, torch.Tensor) else t for t in vars(kv).values()))


def check(got, want, size, dtype):
    got = got.cpu()
    assert got.dtype == dtype and torch.isfinite(got).all(), "non-finite output: a NaN page, slot or scale leaked in"
    bound = 0.5 * ulp_of(want, dtype) + 2.0**-15 * size + 1e-30
    off = ((got.double() - want).abs() / bound).max()
    assert off <= 1, float(off)


def run(ops, q, kv, **kw):
    c = on_gpu(kv)
    return ops.paged_decode_attention(q.cuda(), c.k_cache, c.v_cache, kw.pop("table", c.block_table), kw.pop("lens", c.seq_lens),
                                      k_scale=c.k_scale, v_scale=c.v_scale, **kw)


def dense(ops, q, kv, scale=None, **kw):
    want = ref.decode(q, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens, kv.k_scale, kv.v_scale, scale)
    check(run(ops, q, kv, scale=scale, **kw), *want, q.dtype)


@pytest.mark.parametrize("dtype", QDTYPES)
@pytest.mark.parametrize(("hq", "hkv"), [(8, 8), (16, 4), (8, 1), (32, 8), (32, 1), (12, 4), (34, 2), (80, 2)])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_shapes(gpu_ops, hq, hkv, head_dim, dtype):
    dense(gpu_ops, *problem([1, 15, 16, 17, 300, 0], hq, hkv, head_dim, dtype))


@pytest.mark.parametrize("num_splits", [1, 3, 64, -1])
@pytest.mark.parametrize("dtype", QDTYPES)
@pytest.mark.parametrize(("hq", "hkv"), [(32, 8), (16, 1), (9, 3)])
def test_splits_and_balanced_schedule(gpu_ops, num_splits, dtype, hq, hkv):
    dense(gpu_ops, *problem([5000, 3, 700, 64], hq, hkv, 128, dtype, seed=2), num_splits=num_splits)


@pytest.mark.parametrize("num_splits", [0, 1, 2, -1])
@pytest.mark.parametrize(("hq", "hkv", "head_dim"), [(8, 2, 64), (32, 1, 64), (8, 2, 128), (32, 1, 128), (20, 5, 128), (4, 1, 256)])
def test_every_number_of_blocks(gpu_ops, hq, hkv, head_dim, num_splits):
    """Waves with every number of blocks up to some pipelines' length, alone and beside other sequences."""
    lens = [16 * n - n % 5 for n in range(1, 51)]
    q, kv = problem(lens, hq, hkv, head_dim, torch.bfloat16, seed=head_dim)
    dense(gpu_ops, q, kv, num_splits=num_splits)
    c = on_gpu(kv)
    want, size = ref.decode(q, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens, kv.k_scale, kv.v_scale)
    for b in (0, 1, 2, 6, 7, 8, 15, 16, 24, 31, 32, 49):
        got = gpu_ops.paged_decode_attention(q[b : b + 1].cuda(), c.k_cache, c.v_cache, c.block_table[b : b + 1], c.seq_lens[b : b + 1],
                                             k_scale=c.k_scale, v_scale=c.v_scale, num_splits=num_splits)
        check(got, want[b : b + 1], size[b : b + 1], q.dtype)


def test_pages_far_into_a_large_cache(gpu_ops):
    """Page offsets past 2^32 bytes, through a table of the sequence and through tables per head that were selected."""
    heads, dim, page, last = 8, 256, 128, 5
    pages = (1 << 32) // (heads * dim * page) + 10
    q, kv = problem([page * last - 3], 16, heads, dim, torch.bfloat16, page=page, seed=6)
    where = torch.arange(pages - last, pages)
    wide = {n: torch.zeros(pages, *getattr(kv, n).shape[1:], dtype=getattr(kv, n).dtype, device="cuda")
            for n in ("k_cache", "v_cache", "k_scale", "v_scale", "k_bounds")}
    held = kv.block_table[0, :last].long()
    for name, t in wide.items():
        bits = getattr(kv, name)[held]
        (t.view(torch.uint8) if t.element_size() == 1 else t)[where.cuda()] = (bits.view(torch.uint8) if t.element_size() == 1 else bits).cuda()
    table = where.to(torch.int32)[None].cuda()
    lens = kv.seq_lens.cuda()
    want = ref.decode(q, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens, kv.k_scale, kv.v_scale)
    got = gpu_ops.paged_decode_attention(q.cuda(), wide["k_cache"], wide["v_cache"], table, lens, k_scale=wide["k_scale"], v_scale=wide["v_scale"])
    check(got, *want, q.dtype)
    some = gpu_ops.select_pages(q.cuda(), wide["k_bounds"], wide["k_scale"], table, lens, 3, page)
    chosen = ref.select(q, kv.k_bounds, kv.k_scale, kv.block_table, kv.seq_lens, 3, page)
    place = {int(p): i for i, p in enumerate(held.tolist())}
    assert torch.equal(some[0].cpu() - (pages - last), chosen[0].apply_(lambda p: place[int(p)]))
    assert torch.equal(some[1].cpu(), chosen[1])
    got = gpu_ops.paged_decode_attention(q.cuda(), wide["k_cache"], wide["v_cache"], *some, k_scale=wide["k_scale"], v_scale=wide["v_scale"])
    back = held.to(torch.int32)[chosen[0].long()]
    check(got, *ref.decode(q, kv.k_cache, kv.v_cache, back, chosen[1], kv.k_scale, kv.v_scale), q.dtype)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("num_splits", [0, 2])
def test_page_sizes(gpu_ops, page, num_splits):
    dense(gpu_ops, *problem([100, 33, 1, 1000, page, page + 1], 16, 2, 128, torch.float16, page=page, seed=4), num_splits=num_splits)


@pytest.mark.parametrize("dtype", QDTYPES)
@pytest.mark.parametrize(("batch", "hq", "hkv", "head_dim"), [(70, 32, 8, 128), (64, 16, 8, 64), (300, 8, 1, 128), (40, 24, 8, 256)])
def test_full_batches(gpu_ops, batch, hq, hkv, head_dim, dtype):
    """Paired, wide and many-sequence schedules: even and ragged lengths."""
    g = torch.Generator().manual_seed(batch)
    dense(gpu_ops, *problem(torch.randint(0, 200, (batch,), generator=g).tolist(), hq, hkv, head_dim, dtype, seed=1))
    dense(gpu_ops, *problem([160] * batch, hq, hkv, head_dim, dtype, seed=2))


@pytest.mark.parametrize("dtype", QDTYPES)
@pytest.mark.parametrize("size", [1e-12, 1e9])
def test_scales_far_from_one(gpu_ops, size, dtype):
    """Values whose scale times a weight leaves fp16's range (the outputs of fp16 queries are kept in theirs)."""
    q, kv = problem([40, 200], 8, 2, 128, dtype, seed=3)
    kv.k_scale *= 0.5
    rest = kv.v_scale.clone()
    kv.v_scale = rest * (size if dtype == torch.bfloat16 else 1.0)
    dense(gpu_ops, q, kv)
    # One page of a sequence far above the others: its neighbours' values are lost beside it, not the other way round.
    kv.v_scale = rest.clone()
    kv.v_scale[int(kv.block_table[1, 3])] *= 300.0
    kv.v_scale[int(kv.block_table[1, 4])] *= 1e-9
    dense(gpu_ops, q, kv)


def test_a_zero_scale_and_a_custom_softmax_scale(gpu_ops):
    q, kv = problem([70, 9], 8, 2, 64, torch.bfloat16, seed=8)
    kv.k_scale[int(kv.block_table[0, 1])] = 0.0
    kv.v_scale[int(kv.block_table[0, 2])] = 0.0
    dense(gpu_ops, q, kv, scale=0.05)


def test_one_page_cache_and_equal_scales_equal_head_scales(gpu_ops):
    """Equal scales on every page are scales per head (to the rounding of where they enter)."""
    q, kv = problem([300, 17], 16, 4, 128, torch.bfloat16, seed=5)
    pages = kv.k_cache.shape[0]
    kv.k_scale, kv.v_scale = (torch.tensor(s).repeat(pages, 1) for s in ([0.01, 0.02, 0.03, 0.04], [0.02, 0.01, 0.05, 0.03]))
    dense(gpu_ops, q, kv)
    c = on_gpu(kv)
    by_head = gpu_ops.paged_decode_attention(q.cuda(), c.k_cache, c.v_cache, c.block_table, c.seq_lens, k_scale=c.k_scale[0], v_scale=c.v_scale[0])
    check(by_head, *ref.decode(q, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens, kv.k_scale, kv.v_scale), q.dtype)
    one = PagedFP8(kv.k_cache[:1], kv.v_cache[:1], kv.k_scale[:1], kv.v_scale[:1], kv.k_bounds[:1],
                   torch.zeros(2, 1, dtype=torch.int32), torch.tensor([1, 1], dtype=torch.int32), 16)
    one.k_cache = one.k_cache.float().nan_to_num(1.0).to(torch.float8_e4m3fn)
    one.v_cache = one.v_cache.float().nan_to_num(1.0).to(torch.float8_e4m3fn)
    dense(gpu_ops, q, one)
    lists = one.block_table[:, None].repeat(1, 4, 1), one.seq_lens[:, None].repeat(1, 4)
    got = run(gpu_ops, q, one, table=lists[0].cuda(), lens=lists[1].cuda())
    check(got, *ref.decode(q, one.k_cache, one.v_cache, *lists, one.k_scale, one.v_scale), q.dtype)


def lists_of(kv, heads, width, seed=0):
    """Random ascending choices of each sequence's pages, the last one among them; some of none, one and all."""
    g = torch.Generator().manual_seed(seed)
    batch, page = kv.block_table.shape[0], kv.page_size
    table = torch.zeros(batch, heads, width, dtype=torch.int32)
    lens = torch.zeros(batch, heads, dtype=torch.int32)
    for b in range(batch):
        n = int(kv.seq_lens[b])
        count = (n + page - 1) // page
        for h in range(heads):
            m = min(count, int(torch.randint(0, width + 1, (1,), generator=g)))
            if m == 0:
                continue
            some = torch.cat([torch.randperm(count - 1, generator=g)[: m - 1].sort().values, torch.tensor([count - 1])])
            table[b, h, :m] = kv.block_table[b, some]
            lens[b, h] = (m - 1) * page + n - (count - 1) * page
    return table, lens


@pytest.mark.parametrize("dtype", QDTYPES)
@pytest.mark.parametrize(("batch", "hq", "hkv", "head_dim", "page"),
                         [(1, 32, 8, 128, 16), (3, 8, 8, 64, 32), (5, 16, 2, 256, 16), (4, 32, 1, 128, 64), (66, 32, 8, 128, 16), (2, 40, 2, 128, 16)])
@pytest.mark.parametrize("num_splits", [0, -1, 3])
def test_block_tables_per_head(gpu_ops, batch, hq, hkv, head_dim, page, num_splits, dtype):
    g = torch.Generator().manual_seed(batch)
    seqs = torch.randint(1, 40 * page // 4, (batch,), generator=g).tolist()
    q, kv = problem(seqs, hq, hkv, head_dim, dtype, page=page, seed=6)
    table, lens = lists_of(kv, hkv, 9)
    got = run(gpu_ops, q, kv, table=table.cuda(), lens=lens.cuda(), num_splits=num_splits)
    check(got, *ref.decode(q, kv.k_cache, kv.v_cache, table, lens, kv.k_scale, kv.v_scale), dtype)


def test_long_lists(gpu_ops):
    """Lists cut into several segments a (sequence, KV head)."""
    q, kv = problem([9000, 4000], 16, 4, 128, torch.bfloat16, seed=7)
    table, lens = lists_of(kv, 4, 500)
    for splits in (0, -1, 5):
        got = run(gpu_ops, q, kv, table=table.cuda(), lens=lens.cuda(), num_splits=splits)
        check(got, *ref.decode(q, kv.k_cache, kv.v_cache, table, lens, kv.k_scale, kv.v_scale), torch.bfloat16)


def test_strided_block_table_and_max_seq_len(gpu_ops):
    q, kv = problem([100, 33], 8, 2, 128, torch.float16, seed=9)
    wide = torch.full((2, 40), 1 << 29, dtype=torch.int32)
    wide[:, : kv.block_table.shape[1]] = kv.block_table
    want = ref.decode(q, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens, kv.k_scale, kv.v_scale)
    check(run(gpu_ops, q, kv, table=wide.cuda()[:, : kv.block_table.shape[1]]), *want, q.dtype)
    check(run(gpu_ops, q, kv, table=wide.cuda(), max_seq_len=100), *want, q.dtype)
    lens = torch.tensor([100, 33]).clamp(max=32)
    want = ref.decode(q, kv.k_cache, kv.v_cache, kv.block_table, lens, kv.k_scale, kv.v_scale)
    check(run(gpu_ops, q, kv, max_seq_len=20), *want, q.dtype)  # two pages


def test_refusals(gpu_ops):
    q, kv = problem([20, 40], 8, 2, 64, torch.float16)
    c = on_gpu(kv)
    call = lambda q=q.cuda(), ks=c.k_scale, vs=c.v_scale, bt=c.block_table, sl=c.seq_lens: gpu_ops.paged_decode_attention(  # noqa: E731
        q, c.k_cache, c.v_cache, bt, sl, k_scale=ks, v_scale=vs)
    call()
    with pytest.raises(ValueError, match="both"):
        call(vs=c.v_scale[0])
    with pytest.raises(ValueError, match="scales"):
        call(ks=c.k_scale[:-1], vs=c.v_scale[:-1])
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        call(q=q.float().cuda())
    with pytest.raises(RuntimeError, match="k_scale"):
        call(ks=c.k_scale.half())
    lists = c.block_table[:, None].repeat(1, 2, 1), c.seq_lens[:, None].repeat(1, 2)
    with pytest.raises(ValueError, match="num_pages"):
        call(ks=c.k_scale[0], vs=c.v_scale[0], bt=lists[0], sl=lists[1])
    with pytest.raises(ValueError, match="num_pages"):
        call(ks=0.5, vs=0.5, bt=lists[0], sl=lists[1])
    with pytest.raises(RuntimeError, match="k_scale"):
        call(ks=c.k_scale[:-1], vs=c.v_scale[:-1], bt=lists[0], sl=lists[1])
    with pytest.raises(RuntimeError, match="v_cache"):
        gpu_ops.paged_decode_attention(q.cuda(), c.k_cache, c.v_cache[:-1], c.block_table, c.seq_lens, k_scale=c.k_scale, v_scale=c.v_scale)
    with pytest.raises(RuntimeError, match="per KV head"):
        call(bt=lists[0], sl=c.seq_lens)
    with pytest.raises(RuntimeError, match="per KV head"):
        call(bt=lists[0][:, :1], sl=lists[1][:, :1])
    q32, kv32 = problem([20], 8, 2, 32, torch.float16)
    with pytest.raises(RuntimeError, match="head_dim 64, 128 or 256"):
        run(gpu_ops, q32, kv32)
    q8, kv8 = problem([20], 8, 2, 64, torch.float16, page=8)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        run(gpu_ops, q8, kv8)


def test_a_query_with_a_history_and_a_given_output(gpu_ops):
    q, kv = problem([20, 40], 8, 2, 64, torch.float16)
    c = on_gpu(kv)
    args = c.k_cache, c.v_cache, c.block_table, c.seq_lens
    want = gpu_ops.paged_decode_attention(q.cuda(), *args, k_scale=c.k_scale, v_scale=c.v_scale)
    leaf = q.cuda().requires_grad_()
    got = gpu_ops.paged_decode_attention(leaf, *args, k_scale=c.k_scale, v_scale=c.v_scale)
    assert torch.equal(got, want) and not got.requires_grad
    out = torch.empty_like(want)
    assert gpu_ops.paged_decode_attention(q.cuda(), *args, k_scale=c.k_scale, v_scale=c.v_scale, out=out) is out
    assert torch.equal(out, want)
    every = torch.full((2,), 2, dtype=torch.int32)
    table, lens = gpu_ops.select_pages(leaf, c.k_bounds, c.k_scale, c.block_table, c.seq_lens, 2, 16)
    again = gpu_ops.select_pages(leaf.detach(), c.k_bounds, c.k_scale, c.block_table, c.seq_lens, 2, 16)
    assert torch.equal(table, again[0]) and torch.equal(lens, again[1]) and table.shape == (2, 2, int(every[0]))


@pytest.mark.parametrize("lists", [False, True])
def test_through_c_abi(gpu_ops, lists):
    lib = _native.core()
    q, kv = problem([7, 300, 33], 32, 8, 128, torch.bfloat16, seed=9)
    c, qd = on_gpu(kv), q.cuda()
    table, lens = lists_of(kv, 8, 6) if lists else (kv.block_table, kv.seq_lens)
    td, ld = table.cuda(), lens.cuda()
    code = _native.DTYPE_CODES[torch.bfloat16]
    width = table.shape[-1]
    splits, ws = ctypes.c_int(0), ctypes.c_size_t(0)
    shape = (24, 4, 1) if lists else (3, 32, 8)
    assert lib.kl_paged_decode_plan(code, *shape, 128, 16, width, 0, 0, ctypes.byref(splits), ctypes.byref(ws)) == 0
    workspace = torch.empty(max(ws.value, 1), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(qd)

    def call(ks=c.k_scale.data_ptr(), bytes_=ws.value):
        return lib.kl_paged_decode_attention_fp8_pages(
            code, out.data_ptr(), qd.data_ptr(), c.k_cache.data_ptr(), c.v_cache.data_ptr(), ks, c.v_scale.data_ptr(),
            td.data_ptr(), ld.data_ptr(), 3, 32, 8, 128, 16, width, width, int(lists), 128**-0.5, 0, workspace.data_ptr(),
            bytes_, torch.cuda.current_stream().cuda_stream)

    assert call() == 0, _native.last_error()
    torch.cuda.synchronize()
    check(out, *ref.decode(q, kv.k_cache, kv.v_cache, table, lens, kv.k_scale, kv.v_scale), q.dtype)
    assert call(ks=None) == 1
    if ws.value:
        assert call(bytes_=ws.value - 1) == 3
