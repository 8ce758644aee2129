"""gfx950 RMSNorm with an FP8 output against the float64 oracle.

Tolerances. A code is the rounding of y / scale, which float32 has to about 2^-21 (the sum of squares, rstd, two
products, the scale and a reciprocal, each within a few 2^-24), so |code - y / scale| <= half a step + 2^-20 of the
value; half a step of E4M3 is 2^-4 of a normal value at most and 2^-10 below. A scale is within 2^-20 of the oracle's.
The new residual is bit-exact.
"""

from __future__ import annotations

import pytest
import torch

from oracle import fp8_step as ref
from tests.conftest import DTYPES

pytestmark = pytest.mark.gpu


def half_step(t: torch.Tensor) -> torch.Tensor:
    """Half the distance between the E4M3 values around t."""
    _, e = torch.frexp(t.abs())
    return torch.pow(2.0, (e - 1).clamp(min=-6).double() - 4)


def check(got, scales, x, residual, weight, group, eps=1e-6):
    t, want, res = ref.norm_fp8(x.cpu(), None if residual is None else residual.cpu(), weight.cpu(), eps, group)
    assert got.dtype == torch.float8_e4m3fn and got.shape == x.shape and scales.shape == want.shape
    scales = scales.cpu().double()
    assert bool(((scales - want).abs() <= want * 2.0**-20).all()), float(((scales - want).abs() / want).max())
    codes = got.cpu().float().double()
    bound = half_step(t) + t.abs() * 2.0**-20
    assert bool(((codes - t).abs() <= bound).all()), float(((codes - t).abs() / bound).max())
    return res


def inputs(shape, dtype, seed=0, big=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if big:
        x[..., :: max(1, shape[-1] // 3)] *= 20
    w = 1 + 0.2 * torch.randn(shape[-1], generator=g)
    return x.to(dtype).cuda(), torch.randn(*shape, generator=g).to(dtype).cuda(), w.to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hidden", [1, 2, 3, 7, 8, 31, 64, 65, 100, 128, 500, 512, 513, 1000, 1024, 4096, 5003, 8192, 16385, 20480])
def test_row_scales(gpu_ops, hidden, dtype):
    x, r, w = inputs((5, hidden), dtype, hidden)
    check(*gpu_ops.rms_norm_fp8(x, w), x, None, w, None)
    out, scales, res = gpu_ops.fused_add_rms_norm_fp8(x, r, w)
    assert torch.equal(res.cpu(), check(out, scales, x, r, w, None))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("groups", [1, 2, 3, 5, 16, 33, 80])
def test_group_scales(gpu_ops, group, groups, dtype):
    x, r, w = inputs((3, group * groups), dtype, groups)
    check(*gpu_ops.rms_norm_fp8(x, w, group_size=group), x, None, w, group)
    out, scales, res = gpu_ops.fused_add_rms_norm_fp8(x, r, w, group_size=group)
    assert torch.equal(res.cpu(), check(out, scales, x, r, w, group))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("hidden", "group"), [(40000, None), (65536, 128), (65664, 64), (70001, None), (131072, 256)])
def test_very_wide_rows(gpu_ops, hidden, group, dtype):
    x, r, w = inputs((2, hidden), dtype)
    out, scales, res = gpu_ops.fused_add_rms_norm_fp8(x, r, w, group_size=group)
    assert torch.equal(res.cpu(), check(out, scales, x, r, w, group))
    check(*gpu_ops.rms_norm_fp8(x, w, group_size=group), x, None, w, group)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 1000, 4097])
@pytest.mark.parametrize(("hidden", "group"), [(128, None), (128, 64), (2048, 128), (301, None)])
def test_row_counts(gpu_ops, rows, hidden, group):
    x, r, w = inputs((rows, hidden), torch.bfloat16, rows)
    out, scales, res = gpu_ops.fused_add_rms_norm_fp8(x, r, w, group_size=group)
    assert torch.equal(res.cpu(), check(out, scales, x, r, w, group))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("hidden", "group"), [(128, None), (128, 32), (1024, 128), (333, None), (4096, None)])
def test_strided_rows_and_heads(gpu_ops, hidden, group, dtype):
    """A column slice of wider rows (odd offset: unaligned rows), and the heads of a fused projection."""
    wide, _, w = inputs((9, hidden + 37), dtype)
    x, w = wide[:, 5 : 5 + hidden], w[:hidden]
    check(*gpu_ops.rms_norm_fp8(x, w, group_size=group), x, None, w, group)
    fused, _, _ = inputs((6, 7 * hidden), dtype, 1)
    heads = fused[:, : 4 * hidden].view(6, 4, hidden)
    out, scales = gpu_ops.rms_norm_fp8(heads, w, group_size=group)
    check(out, scales, heads, None, w, group)
    r = torch.randn(6, 4, hidden, device="cuda").to(dtype)
    out, scales, res = gpu_ops.fused_add_rms_norm_fp8(heads, r, w, group_size=group)
    assert torch.equal(res.cpu(), check(out, scales, heads, r, w, group))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("hidden", "group"), [(4096, None), (4096, 128), (333, None), (40004, None)])
def test_in_place_residual_equals_the_functional_form(gpu_ops, hidden, group, dtype):
    x, r, w = inputs((7, hidden), dtype)
    out, scales, res = gpu_ops.fused_add_rms_norm_fp8(x, r, w, group_size=group)
    before = r.clone()
    assert torch.equal(before, r)
    out2, scales2 = gpu_ops.fused_add_rms_norm_fp8_(x, r, w, group_size=group)
    assert torch.equal(r, res) and torch.equal(scales, scales2)
    assert torch.equal(out.view(torch.uint8), out2.view(torch.uint8))


@pytest.mark.parametrize("group", [None, 64])
def test_zero_rows_tiny_rows_and_zero_weights(gpu_ops, group):
    x = torch.zeros(4, 256, device="cuda")
    x[1] = 1e-30
    x[2] = torch.randn(256, device="cuda")
    x[3, 17] = 3.0
    w = torch.ones(256, device="cuda")
    w[64:128] = 0
    out, scales = gpu_ops.rms_norm_fp8(x, w, group_size=group)
    check(out, scales, x, None, w, group)
    assert torch.equal(out[0].float(), torch.zeros(256, device="cuda"))
    assert float(scales[0, 0]) == ref.MIN_SCALE


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("hidden", "group"), [(256, None), (256, 64), (4096, None), (4096, 128), (301, None)])
def test_values_that_are_not_finite(gpu_ops, hidden, group, dtype):
    """inf in x: rstd is 0, so the row's finite values give 0 and the inf a NaN code; a NaN makes its row NaN; an
    infinite weight makes its column NaN and does not touch the scale. Other rows are as without them."""
    x, _, w = inputs((4, hidden), dtype)
    clean, clean_scales = gpu_ops.rms_norm_fp8(x, w, group_size=group)
    x[1, 3] = float("inf")
    x[2, 7] = float("nan")
    out, scales = gpu_ops.rms_norm_fp8(x, w, group_size=group)
    for row in (0, 3):
        assert torch.equal(out[row].view(torch.uint8), clean[row].view(torch.uint8))
        assert torch.equal(scales[row], clean_scales[row])
    got = out[1].float()
    assert torch.isnan(got[3]) and float(got.nan_to_num(0).abs().max()) == 0.0
    assert torch.isnan(out[2].float()).all()
    assert torch.isfinite(scales).all() and float(scales[1:3].max()) == ref.MIN_SCALE
    w[5] = float("inf")
    x, _, _ = inputs((4, hidden), dtype)
    out, scales = gpu_ops.rms_norm_fp8(x, w, group_size=group)
    assert torch.isnan(out[:, 5].float()).all()
    keep = torch.arange(hidden, device="cuda") != 5
    t, want, _ = ref.norm_fp8(x.cpu(), None, torch.where(keep, w, 0).cpu(), 1e-6, group)
    assert bool(((scales.cpu().double() - want).abs() <= want * 2.0**-20).all())
    codes, t = out.cpu().float().double()[:, keep.cpu()], t[:, keep.cpu()]
    assert bool(((codes - t).abs() <= half_step(t) + t.abs() * 2.0**-20).all())


def test_refusals(gpu_ops):
    x, r, w = inputs((4, 256), torch.bfloat16)
    with pytest.raises(ValueError, match="does not match weight"):
        gpu_ops.rms_norm_fp8(x, w[:-1])
    with pytest.raises(ValueError, match="same shape"):
        gpu_ops.fused_add_rms_norm_fp8(x, r[:2], w)
    with pytest.raises(ValueError, match="group_size"):
        gpu_ops.rms_norm_fp8(x, w, group_size=48)
    with pytest.raises(ValueError, match="multiple"):
        gpu_ops.rms_norm_fp8(x[:, :200], w[:200], group_size=128)
    with pytest.raises(RuntimeError, match="dtype"):
        gpu_ops.rms_norm_fp8(x, w.float())
    with pytest.raises(RuntimeError, match="dtype"):
        gpu_ops.rms_norm_fp8(x.double(), w.double())
    with pytest.raises(RuntimeError, match="device|GPU"):
        gpu_ops.rms_norm_fp8(x, w.cpu())
    out = torch.empty(4, 256, dtype=torch.float8_e4m3fn, device="cuda")
    with pytest.raises(RuntimeError, match="scales"):
        torch.ops.kernel_lab.rms_norm_fp8(out, torch.empty(4, 3, device="cuda"), x, w, 1e-6, 64)
    with pytest.raises(RuntimeError, match="out"):
        torch.ops.kernel_lab.rms_norm_fp8(out[:2], torch.empty(4, 4, device="cuda"), x, w, 1e-6, 64)


def test_empty_inputs(gpu_ops):
    w = torch.ones(64, device="cuda")
    out, scales = gpu_ops.rms_norm_fp8(torch.empty(0, 64, device="cuda"), w, group_size=32)
    assert out.shape == (0, 64) and scales.shape == (0, 2)


@pytest.mark.parametrize("group", [None, 128])
def test_compiles(gpu_ops, group):
    """Under torch.compile(fullgraph=True): the functional and the in-place forms."""
    x, r, w = inputs((16, 1024), torch.bfloat16)

    def step(x, r, w):
        out, scales, new = gpu_ops.fused_add_rms_norm_fp8(x, r, w, group_size=group)
        plain, plain_scales = gpu_ops.rms_norm_fp8(new, w, group_size=group)
        return out, scales, new, plain, plain_scales

    want = step(x, r, w)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(x, r, w)
    for g, ok in zip(got, want):
        assert torch.equal(g.contiguous().view(torch.uint8), ok.contiguous().view(torch.uint8))


def test_inputs_with_a_history(gpu_ops):
    """Parameters and a residual in a graph give the same values; no gradient passes the codes."""
    x, r, w = inputs((4, 256), torch.float32)
    want = gpu_ops.fused_add_rms_norm_fp8(x, r, w)
    leaf, weight = r.clone().requires_grad_(), torch.nn.Parameter(w)
    out, scales, new = gpu_ops.fused_add_rms_norm_fp8(x, leaf * 1.0, weight)
    assert torch.equal(out.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])
    assert torch.equal(new.detach(), want[2]) and not out.requires_grad and not scales.requires_grad
    plain = gpu_ops.rms_norm_fp8(x, weight)
    assert torch.equal(plain[0].view(torch.uint8), gpu_ops.rms_norm_fp8(x, w)[0].view(torch.uint8))


def test_replays(gpu_ops):
    """Captured into a graph whose inputs change between replays."""
    x, r, w = inputs((16, 1024), torch.float16)
    want = gpu_ops.fused_add_rms_norm_fp8(x, r, w, group_size=128)
    out = torch.empty(16, 1024, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(16, 8, device="cuda")
    new = torch.empty_like(r)

    def step(x, r):
        torch.ops.kernel_lab.fused_add_rms_norm_fp8_new(out, scales, new, x, r, w, 1e-6, 128)

    graph = torch.cuda.CUDAGraph()
    step(x, r)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(x, r)
    for seed in range(3):
        x2, r2, _ = inputs((16, 1024), torch.float16, seed)
        x.copy_(x2)
        r.copy_(r2)
        graph.replay()
        torch.cuda.synchronize()
        want = gpu_ops.fused_add_rms_norm_fp8(x2, r2, w, group_size=128)
        for got, ok in zip((out, scales, new), want):
            assert torch.equal(got.view(torch.uint8), ok.view(torch.uint8))
