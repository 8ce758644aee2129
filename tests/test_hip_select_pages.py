"""gfx950 page selection against the float64 oracle: tables and lengths have to be equal.

The scores' sums are exact in 64 bits for these inputs on both sides (a product of a query and a code has at most 15 bits
and the values' exponents span less than 30 binades), so their order does not matter, and both round once to float32.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from kernel_lab import _native
from oracle import fp8_step as ref

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def problem(lens, hq, hkv, dim, dtype, page, seed=0, spare=5):
    """Queries, bounds (smallest <= largest code, mixed signs), scales and a table of distinct pages."""
    g = torch.Generator().manual_seed(seed)
    need = [(max(n, 0) + page - 1) // page for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max([*need, 1]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    edges = (100 * torch.randn(total, hkv, 2, dim, generator=g)).clamp(-448, 448).sort(2).values.to(F8)
    scale = 0.01 * torch.exp(0.3 * torch.randn(total, hkv, generator=g))
    spare_ids = order[at:].long()
    edges.view(torch.uint8)[spare_ids] = 0x7F  # NaN
    scale[spare_ids] = float("nan")
    q = torch.randn(len(lens), hq, dim, generator=g).to(dtype)
    return q, edges, scale, table, torch.tensor(lens, dtype=torch.int32)


def check(ops, q, edges, scale, table, lens, keep, page, first=1, last=1):
    got = ops.select_pages(q.cuda(), edges.cuda(), scale.cuda(), table.cuda(), lens.cuda(), keep, page, first_pages=first, last_pages=last)
    want = ref.select(q, edges, scale, table, lens, keep, page, first, last)
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0]), (got[0].cpu() != want[0]).nonzero()[:5]
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("hq", "hkv"), [(8, 8), (16, 4), (8, 1), (32, 8), (32, 1), (12, 4), (80, 2)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_shapes(gpu_ops, hq, hkv, dim, dtype):
    lens = [1, 16, 17, 160, 161, 333, 0, 2000]
    check(gpu_ops, *problem(lens, hq, hkv, dim, dtype, 16, seed=dim), 10, 16)


@pytest.mark.parametrize("keep", [1, 2, 3, 7, 64, 255, 256, 257, 500, 700])
def test_keep_counts_on_long_tables(gpu_ops, keep):
    check(gpu_ops, *problem([16 * 600 - 3, 16 * 256, 16 * 257, 5, 16 * 300 + 1], 16, 2, 128, torch.bfloat16, 16), keep, 16, first=0)


@pytest.mark.parametrize(("first", "last"), [(0, 1), (1, 1), (0, 8), (7, 1), (4, 4), (3, 2)])
def test_pinned_pages(gpu_ops, first, last):
    check(gpu_ops, *problem([32 * 40, 32 * 8, 32 * 9, 32 * 3 + 1, 32], 8, 2, 64, torch.float16, 32, seed=3), 8, 32, first, last)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128])
def test_page_sizes(gpu_ops, page):
    check(gpu_ops, *problem([page * 33 + 7, page * 20, 3], 16, 4, 128, torch.bfloat16, page), 12, page)


def test_equal_scores_take_the_lowest_pages(gpu_ops):
    q, edges, scale, table, lens = problem([16 * 700], 8, 2, 128, torch.float16, 16)
    edges.copy_(edges[:1].float().nan_to_num(0).to(F8).expand_as(edges))
    scale.fill_(0.5)
    check(gpu_ops, q, edges, scale, table, lens, 100, 16)
    scale[table[0, 300:350].long()] = 0.75  # a run of better (or, below zero, worse) ones
    check(gpu_ops, q, edges, scale, table, lens, 100, 16)
    check(gpu_ops, -q, edges, scale, table, lens, 30, 16)
    check(gpu_ops, torch.zeros_like(q), edges, scale, table, lens, 300, 16)


def test_scores_below_zero_and_signed_zeros(gpu_ops):
    q, edges, scale, table, lens = problem([16 * 90], 4, 1, 64, torch.bfloat16, 16)
    q = q.abs()
    edges = (-edges.float().nan_to_num(0).abs()).to(F8)
    edges[:, :, 1] = edges[:, :, 0]
    edges[table[0, 10:20].long()] = 0
    edges.view(torch.uint8)[table[0, 20:30].long()] = 0x80  # -0
    check(gpu_ops, q, edges, scale, table, lens, 12, 16)
    check(gpu_ops, q, edges, scale, table, lens, 40, 16)


def test_scores_that_are_not_numbers(gpu_ops):
    """NaN and infinite scores count as the largest finite one; an infinite query, too."""
    q, edges, scale, table, lens = problem([16 * 64, 16 * 64], 8, 2, 64, torch.bfloat16, 16)
    scale[table[0, 20].long()] = float("nan")
    scale[table[0, 30].long()] = float("inf")
    edges.view(torch.uint8)[table[0, 40].long(), :, :, 5] = 0x7F
    check(gpu_ops, q, edges, scale, table, lens, 6, 16)
    q[1, 0, 3] = float("inf")
    q[1, 5, 3] = float("nan")
    check(gpu_ops, q, edges, scale, table, lens, 6, 16)


def test_dimensions_without_a_finite_key(gpu_ops):
    """Their bounds are 448 and -448, and lower the score."""
    q, edges, scale, table, lens = problem([16 * 64, 16 * 70], 8, 2, 64, torch.float16, 16, seed=9)
    for b, p in ((0, 3), (0, 21), (1, 5), (1, 40)):
        edges[table[b, p].long(), :, 0, 7] = 448.0
        edges[table[b, p].long(), :, 1, 7] = -448.0
    check(gpu_ops, q, edges, scale, table, lens, 30, 16)
    flat = edges[table[0, 0].long()].expand_as(edges).clone()  # equal scores but for one page's
    flat[table[0, 3].long(), :, 0, 7], flat[table[0, 3].long(), :, 1, 7] = 448.0, -448.0
    got, _ = check(gpu_ops, q, flat, torch.ones_like(scale), table, lens, 63, 16)
    assert not (got[0] == table[0, 3].item()).any()


def test_a_query_at_any_address(gpu_ops):
    q, edges, scale, table, lens = problem([16 * 64, 16 * 70], 8, 2, 64, torch.float16, 16, seed=9)
    store = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")
    shifted = store[1:].view(q.shape)
    shifted.copy_(q)
    got = gpu_ops.select_pages(shifted, edges.cuda(), scale.cuda(), table.cuda(), lens.cuda(), 30, 16)
    want = check(gpu_ops, q, edges, scale, table, lens, 30, 16)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_near_scores_are_told_apart(gpu_ops):
    """Pages whose scores differ only behind the 24 bits that a float32 sum keeps at its size, but not once rounded."""
    dim, pages = 128, 200
    q = torch.full((1, 1, dim), 1.0, dtype=torch.float16)
    q[..., 0] = 2.0**-14
    edges = torch.zeros(pages, 1, 2, dim)
    edges[..., 1:65], edges[..., 65:] = 448.0, -448.0  # they cancel
    g = torch.Generator().manual_seed(0)
    edges[..., 0] = torch.randint(1, 16, (pages, 1, 1), generator=g) * 1.0
    table = torch.arange(pages, dtype=torch.int32)[None]
    edges = edges.to(F8)
    check(gpu_ops, q, edges, torch.ones(pages, 1), table, torch.tensor([16 * pages], dtype=torch.int32), 20, 16, first=0)


@pytest.mark.parametrize(("dtype", "size"), [(torch.float16, 2.0**-20), (torch.float16, 2.0**-16), (torch.bfloat16, 1e-39), (torch.bfloat16, 1e-30),
                                             (torch.bfloat16, 1e30), (torch.float16, 1e4)])
def test_queries_far_from_one(gpu_ops, dtype, size):
    """Subnormal queries, and sums near the end of float32's range."""
    q, edges, scale, table, lens = problem([16 * 300, 16 * 90], 8, 2, 128, torch.float32, 16, seed=6)
    check(gpu_ops, (q * size).to(dtype), edges, scale, table, lens, 20, 16)


@pytest.mark.parametrize("pages", [300, 1500])
def test_many_pages_between(gpu_ops, pages):
    """Scores so near one another that the 16-bit matrix cores' sums cannot order them: hundreds are scored in 64 bits."""
    q, edges, scale, table, lens = problem([16 * pages], 8, 2, 128, torch.bfloat16, 16, seed=7)
    g = torch.Generator().manual_seed(1)
    edges.copy_(edges[:1].float().nan_to_num(1.0).to(F8).expand_as(edges))
    scale.copy_((1 + 1e-6 * torch.randn(scale.shape, generator=g)) * 0.01)
    check(gpu_ops, q, edges, scale, table, lens, 100, 16)
    edges[:, :, :, 3] = torch.rand(edges.shape[0], 2, 1, generator=g).expand(-1, -1, 2).to(F8)
    check(gpu_ops, q, edges, scale, table, lens, 100, 16)


def test_lengths_past_the_table_and_below_zero(gpu_ops):
    q, edges, scale, table, lens = problem([16 * 30, 16 * 30, 16 * 30], 8, 2, 64, torch.bfloat16, 16)
    lens = torch.tensor([16 * 30 + 100, -5, 2**31 - 1], dtype=torch.int32)
    check(gpu_ops, q, edges, scale, table, lens, 8, 16)


@pytest.mark.parametrize(("pages", "group"), [(2048, 4), (2049, 4), (2300, 8), (3000, 16), (2100, 40), (8192, 1), (9000, 2)])
def test_long_tables_of_few_sequences(gpu_ops, pages, group):
    """Past what one workgroup scores: the scores get a launch of their own; past its LDS, the keys stay in memory."""
    lens = [16 * pages - 3, 16 * 100, 5]
    args = problem(lens, group, 1, 64, torch.bfloat16, 16, seed=pages)
    check(gpu_ops, *args, 64, 16)
    check(gpu_ops, *args, 2047, 16, first=3, last=2)


def test_long_tables_of_a_full_batch(gpu_ops):
    """As many (sequence, KV head) pairs as compute units: one launch up to its LDS."""
    lens = torch.randint(0, 16 * 2500, (64,), generator=torch.Generator().manual_seed(2)).tolist()
    lens[3] = 16 * 2500
    args = problem(lens, 8, 4, 64, torch.float16, 16, seed=4)
    q, edges, scale, table, lens = args
    got = gpu_ops.select_pages(q.cuda(), edges.cuda(), scale.cuda(), table.cuda(), lens.cuda(), 40, 16)
    rows = [0, 3, 17, 63]
    want = ref.select(q[rows], edges, scale, table[rows], lens[rows], 40, 16)
    assert torch.equal(got[0].cpu()[rows], want[0]) and torch.equal(got[1].cpu()[rows], want[1])


def test_strided_table(gpu_ops):
    q, edges, scale, table, lens = problem([16 * 30, 40], 8, 2, 64, torch.bfloat16, 16)
    wide = torch.full((2, 50), 1 << 29, dtype=torch.int32)
    wide[:, : table.shape[1]] = table
    got = gpu_ops.select_pages(q.cuda(), edges.cuda(), scale.cuda(), wide.cuda()[:, : table.shape[1]], lens.cuda(), 8, 16)
    want = ref.select(q, edges, scale, table, lens, 8, 16)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_many_rows(gpu_ops):
    lens = torch.randint(0, 1500, (130,), generator=torch.Generator().manual_seed(1)).tolist()
    check(gpu_ops, *problem(lens, 32, 8, 64, torch.float16, 32), 16, 32, first=1, last=2)


def test_more_rows_than_a_grid_dimension(gpu_ops):
    """40,000 sequences, (sequence, KV head) pairs past the grid's second dimension."""
    batch, page, width = 40000, 16, 6
    g = torch.Generator().manual_seed(0)
    edges = torch.randn(50, 2, 2, 64, generator=g).mul(50).sort(2).values.to(F8)
    scale = 0.01 + torch.rand(50, 2, generator=g)
    table = torch.randint(0, 50, (batch, width), generator=g, dtype=torch.int32)
    lens = torch.randint(0, page * width + 1, (batch,), generator=g, dtype=torch.int32)
    q = torch.randn(batch, 4, 64, generator=g).to(torch.bfloat16)
    got = gpu_ops.select_pages(*(t.cuda() for t in (q, edges, scale, table, lens)), 3, page)
    rows = torch.tensor([0, 1, 16383, 16384, 20000, 32767, 32768, 39999])
    want = ref.select(q[rows], edges, scale, table[rows], lens[rows], 3, page)
    assert torch.equal(got[0].cpu()[rows], want[0]) and torch.equal(got[1].cpu()[rows], want[1])


def test_two_streams_at_once(gpu_ops):
    """Tables whose scores several workgroups share, on two streams: each has counters of its own."""
    args = [tuple(t.cuda() for t in problem([16 * 900, 16 * 500], 8, 2, 128, torch.bfloat16, 16, seed=s)) for s in range(2)]
    want = [gpu_ops.select_pages(*a, 40, 16) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(gpu_ops.select_pages(*args[i], 40, 16))
    torch.cuda.synchronize()
    for i in range(2):
        for table, lens in got[i]:
            assert torch.equal(table, want[i][0]) and torch.equal(lens, want[i][1])


def test_two_captured_graphs_at_once(gpu_ops):
    """Two graphs captured one after the other and replayed on two streams together."""
    args = [tuple(t.cuda() for t in problem([16 * 900, 16 * 500], 8, 2, 128, torch.float16, 16, seed=s)) for s in range(2)]
    want = [gpu_ops.select_pages(*a, 40, 16) for a in args]
    torch.cuda.synchronize()
    graphs, got = [], []
    for a in args:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(gpu_ops.select_pages(*a, 40, 16))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for t, n in got:
            t.zero_()
            n.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])


def test_empty_batch(gpu_ops):
    q, edges, scale, table, lens = problem([16], 8, 2, 64, torch.bfloat16, 16)
    got = gpu_ops.select_pages(q[:0].cuda(), edges.cuda(), scale.cuda(), table[:0].cuda(), lens[:0].cuda(), 8, 16)
    assert got[0].shape == (0, 2, 8) and got[1].shape == (0, 2)


def test_refusals(gpu_ops):
    q, edges, scale, table, lens = (t.cuda() for t in problem([16 * 30], 8, 2, 64, torch.bfloat16, 16))
    for bad in [{"first_pages": -1}, {"last_pages": 0}, {"first_pages": 5, "last_pages": 4}]:
        with pytest.raises(ValueError, match="must fit"):
            gpu_ops.select_pages(q, edges, scale, table, lens, 8, 16, **bad)
    with pytest.raises(ValueError, match="multiple"):
        gpu_ops.select_pages(q[:, :7], edges, scale, table, lens, 8, 16)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        gpu_ops.select_pages(q, edges, scale, table, lens, 8, 8)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        gpu_ops.select_pages(q.float(), edges, scale, table, lens, 8, 16)
    with pytest.raises(RuntimeError, match="k_scale"):
        gpu_ops.select_pages(q, edges, scale[:-1], table, lens, 8, 16)
    with pytest.raises(RuntimeError, match="k_bounds"):
        gpu_ops.select_pages(q, edges.view(torch.uint8), scale, table, lens, 8, 16)
    with pytest.raises(RuntimeError, match="one row per sequence"):
        gpu_ops.select_pages(q, edges, scale, table, lens.repeat(2), 8, 16)


def test_graph_replays(gpu_ops):
    q, edges, scale, table, lens = (t.cuda() for t in problem([16 * 90, 16 * 300, 3], 16, 4, 128, torch.bfloat16, 16))
    run = lambda: gpu_ops.select_pages(q, edges, scale, table, lens, 24, 16)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in range(4):
        new = problem([16 * 90, 16 * 300, 3], 16, 4, 128, torch.bfloat16, 16, seed=seed)
        for t, n in zip((q, edges, scale, table), new):
            t.copy_(n)
        lens.copy_(torch.tensor([16 * 90 - seed, 16 * (100 + seed), 3 + seed], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = ref.select(*(t.cpu() for t in (q, edges, scale, table, lens)), 24, 16)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("pages", [90, 2500])
def test_through_c_abi(gpu_ops, pages):
    """A table that one launch serves without a workspace, and one whose scores need it."""
    lib = _native.core()
    host = problem([16 * pages, 16 * 40 + 3], 16, 4, 128, torch.bfloat16, 16)
    q, edges, scale, table, lens = (t.cuda() for t in host)
    ws = ctypes.c_size_t(0)
    assert lib.kl_select_pages_workspace(2, 4, pages, ctypes.byref(ws)) == 0 and (ws.value == 0 if pages == 90 else ws.value >= 2 * 4 * pages * 4)
    work = torch.empty(max(1, ws.value), dtype=torch.uint8, device="cuda")
    out, out_lens = torch.empty(2, 4, 12, dtype=torch.int32, device="cuda"), torch.empty(2, 4, dtype=torch.int32, device="cuda")

    def call(bytes_=ws.value, first=1):
        return lib.kl_select_pages(2, out.data_ptr(), out_lens.data_ptr(), q.data_ptr(), edges.data_ptr(), scale.data_ptr(),
                                   table.data_ptr(), lens.data_ptr(), 2, 16, 4, 128, 16, pages, pages, 12, first, 1, work.data_ptr(),
                                   bytes_, torch.cuda.current_stream().cuda_stream)

    assert call() == 0, _native.last_error()
    torch.cuda.synchronize()
    want = ref.select(*host, 12, 16)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(out_lens.cpu(), want[1])
    if ws.value:
        assert call(bytes_=ws.value - 4) == 3
    assert call(first=12) == 1
