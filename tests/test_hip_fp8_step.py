"""The 8-bit serving step as a program runs it: norm into FP8, append, page selection, sparse and dense decode, several
tokens long, in eager calls and as one captured graph, against the oracle's steps."""

from __future__ import annotations

import pytest
import torch

from oracle import fp8_step as ref
from tests.conftest import ulp_of
from tests.test_hip_append_fp8 import make, same

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE, HIDDEN = 16, 4, 128, 16, 512


class Program:
    """One attention layer over an 8-bit stream: the projection's input is the norm's codes times their scales."""

    def __init__(self, ops, dev, batch, dtype):
        g = torch.Generator().manual_seed(0)
        self.ops, self.dev, self.dtype = ops, dev, dtype
        self.norm_w = torch.ones(HIDDEN, dtype=dtype, device="cuda")
        self.proj = (torch.randn(HIDDEN, (HQ + 2 * HKV) * D, generator=g) * HIDDEN**-0.5).cuda()
        self.x, self.res = (torch.zeros(batch, HIDDEN, dtype=dtype, device="cuda") for _ in range(2))
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def step(self):
        ops, c = self.ops, self.dev
        codes, scale = ops.fused_add_rms_norm_fp8_(self.x, self.res, self.norm_w, group_size=128)
        h = codes.float().reshape(len(self.x), -1, 128) * scale[..., None]
        qkv = (h.reshape(len(self.x), -1) @ self.proj).to(self.dtype).view(len(self.x), HQ + 2 * HKV, D)
        q, k, v = qkv[:, :HQ], qkv[:, HQ : HQ + HKV], qkv[:, HQ + HKV :]
        ops.append_kv_fp8(k, v, c["k"], c["v"], c["k_scale"], c["v_scale"], c["block_table"], self.lens, k_bounds=c["bounds"])
        table, lens = ops.select_pages(q, c["bounds"], c["k_scale"], c["block_table"], self.lens, 4, PAGE)
        sparse = ops.paged_decode_attention(q, c["k"], c["v"], table, lens, k_scale=c["k_scale"], v_scale=c["v_scale"])
        full = ops.paged_decode_attention(q, c["k"], c["v"], c["block_table"], self.lens, k_scale=c["k_scale"], v_scale=c["v_scale"])
        return qkv, table, lens, sparse, full


def close(got, want, size, dtype):
    bound = 0.5 * ulp_of(want, dtype) + 2.0**-15 * size + 1e-30
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_few_tokens(gpu_ops, dtype, captured):
    start = [100, 31, 0, 160, 15]
    batch = len(start)
    dev, host = make([n + 10 for n in start], HKV, D, PAGE)
    g = torch.Generator().manual_seed(7)
    k, v = torch.randn(2, sum(start), HKV, D, generator=g).to(dtype)
    off = torch.tensor([0, *start]).cumsum(0).to(torch.int32)
    lens = torch.tensor(start, dtype=torch.int32)
    gpu_ops.append_kv_fp8(k.cuda(), v.cuda(), dev["k"], dev["v"], dev["k_scale"], dev["v_scale"], dev["block_table"], lens.cuda(),
                          new_offsets=off.cuda(), k_bounds=dev["bounds"])
    ref.append(k, v, host, lens, off)
    same(dev, host)

    p = Program(gpu_ops, dev, batch, dtype)
    graph = None
    if captured:
        p.step()  # idle rows: lengths 0
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = p.step()
    for i in range(4):
        lens = lens + torch.tensor([1, 1, 0, 1, 1], dtype=torch.int32)  # sequence 2 stays idle
        p.x.copy_(torch.randn(batch, HIDDEN, generator=g))
        p.res.copy_(torch.randn(batch, HIDDEN, generator=g))
        p.lens.copy_(lens)
        if graph is not None:
            graph.replay()
        else:
            out = p.step()
        torch.cuda.synchronize()
        qkv, table, sel_lens, sparse, full = out
        qkv = qkv.cpu()
        q = qkv[:, :HQ]
        ref.append(qkv[:, HQ : HQ + HKV], qkv[:, HQ + HKV :], host, lens)
        same(dev, host)
        want = ref.select(q, dev["bounds"].cpu(), host["k_scale"], host["block_table"], lens, 4, PAGE)
        assert torch.equal(table.cpu(), want[0]) and torch.equal(sel_lens.cpu(), want[1])
        cache = dev["k"].cpu(), dev["v"].cpu()
        close(sparse, *ref.decode(q, *cache, *want, host["k_scale"], host["v_scale"]), dtype)
        close(full, *ref.decode(q, *cache, host["block_table"], lens, host["k_scale"], host["v_scale"]), dtype)
        assert float(full[2].abs().max()) == 0.0 and float(sparse[2].abs().max()) == 0.0


def test_compiled_and_on_a_stream_of_its_own(gpu_ops):
    """append, selection and both decodes under torch.compile(fullgraph=True), on a side stream."""
    batch, dtype = 3, torch.bfloat16
    dev, host = make([60, 40, 17], HKV, D, PAGE)
    lens = torch.tensor([50, 33, 16], dtype=torch.int32)
    k, v = torch.randn(2, batch, HKV, D, generator=torch.Generator().manual_seed(1)).to(dtype)
    q = torch.randn(batch, HQ, D, generator=torch.Generator().manual_seed(2)).to(dtype)
    full = torch.randn(2, 99, HKV, D, generator=torch.Generator().manual_seed(3)).to(dtype)
    off = torch.tensor([0, 50, 83, 99], dtype=torch.int32)
    gpu_ops.append_kv_fp8(full[0].cuda(), full[1].cuda(), dev["k"], dev["v"], dev["k_scale"], dev["v_scale"], dev["block_table"],
                          lens.cuda(), new_offsets=off.cuda(), k_bounds=dev["bounds"])
    ref.append(full[0], full[1], host, lens, off)

    def step(q, k, v, kc, vc, ks, vs, bounds, table, lens):
        gpu_ops.append_kv_fp8(k, v, kc, vc, ks, vs, table, lens, k_bounds=bounds)
        pages, some = gpu_ops.select_pages(q, bounds, ks, table, lens, 2, PAGE)
        return (pages, some, gpu_ops.paged_decode_attention(q, kc, vc, pages, some, k_scale=ks, v_scale=vs),
                gpu_ops.paged_decode_attention(q, kc, vc, table, lens, k_scale=ks, v_scale=vs))

    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    lens = lens + 1
    args = [t.cuda() for t in (q, k, v)] + [dev[n] for n in ("k", "v", "k_scale", "v_scale", "bounds", "block_table")] + [lens.cuda()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pages, some, sparse, dense = compiled(*args)
    torch.cuda.synchronize()
    ref.append(k, v, host, lens)
    same(dev, host)
    want = ref.select(q, dev["bounds"].cpu(), host["k_scale"], host["block_table"], lens, 2, PAGE)
    assert torch.equal(pages.cpu(), want[0]) and torch.equal(some.cpu(), want[1])
    cache = dev["k"].cpu(), dev["v"].cpu()
    close(sparse, *ref.decode(q, *cache, *want, host["k_scale"], host["v_scale"]), dtype)
    close(dense, *ref.decode(q, *cache, host["block_table"], lens, host["k_scale"], host["v_scale"]), dtype)


def test_two_captured_steps_at_once(gpu_ops):
    """Two graphs of append, selection and both decodes, each over a cache of its own, replayed together on two streams."""
    dtype, runs = torch.bfloat16, []
    for i, start in enumerate(([300, 90, 17, 700], [64, 515, 1, 33])):
        dev, host = make([n + 6 for n in start], HKV, D, PAGE)
        g = torch.Generator().manual_seed(20 + i)
        k, v = torch.randn(2, sum(start), HKV, D, generator=g).to(dtype)
        off = torch.tensor([0, *start]).cumsum(0).to(torch.int32)
        lens = torch.tensor(start, dtype=torch.int32)
        gpu_ops.append_kv_fp8(k.cuda(), v.cuda(), dev["k"], dev["v"], dev["k_scale"], dev["v_scale"], dev["block_table"], lens.cuda(),
                              new_offsets=off.cuda(), k_bounds=dev["bounds"])
        ref.append(k, v, host, lens, off)
        p = Program(gpu_ops, dev, len(start), dtype)
        p.step()
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = p.step()
        runs.append((p, dev, host, lens, g, stream, graph, out))
    for n in range(1, 5):
        for p, _, _, lens, g, _, _, _ in runs:
            p.x.copy_(torch.randn(p.x.shape, generator=g))
            p.res.copy_(torch.randn(p.res.shape, generator=g))
            p.lens.copy_(lens + n)
        torch.cuda.synchronize()
        for *_, stream, graph, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, dev, host, lens, _, _, _, (qkv, table, sel_lens, sparse, full) in runs:
            qkv = qkv.cpu()
            q = qkv[:, :HQ]
            ref.append(qkv[:, HQ : HQ + HKV], qkv[:, HQ + HKV :], host, lens + n)
            same(dev, host)
            want = ref.select(q, dev["bounds"].cpu(), host["k_scale"], host["block_table"], lens + n, 4, PAGE)
            assert torch.equal(table.cpu(), want[0]) and torch.equal(sel_lens.cpu(), want[1])
            cache = dev["k"].cpu(), dev["v"].cpu()
            close(sparse, *ref.decode(q, *cache, *want, host["k_scale"], host["v_scale"]), dtype)
            close(full, *ref.decode(q, *cache, host["block_table"], lens + n, host["k_scale"], host["v_scale"]), dtype)
