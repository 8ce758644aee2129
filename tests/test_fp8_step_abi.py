"""Refusals of the 8-bit serving step's C entry points, and their empty calls: every one of these returns before a launch, so
they run without a GPU."""

from __future__ import annotations

import ctypes

import pytest

from kernel_lab import _native

pytestmark = pytest.mark.skipif(not _native.loaded(), reason=_native.why_unavailable())

OK, ARGUMENT, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3
F32, F16, BF16 = 0, 1, 2


def call(name, args, want, match=""):
    lib = _native.core()
    assert getattr(lib, name)(*args) == want, (name, args, lib.kl_last_error())
    assert match in lib.kl_last_error().decode()


def norm(dtype=BF16, ptr=16, residual=None, residual_out=None, groups=1, rows=4, hidden=256, gs=0, rs=256, scale_group=0):
    return [dtype, ptr, ptr, ptr, residual, residual_out, ptr, groups, rows, hidden, gs, rs, scale_group, 1e-6, None]


@pytest.mark.parametrize(
    ("change", "want", "match"),
    [
        ({"rows": 0, "ptr": None}, OK, ""),
        ({"rows": -1}, ARGUMENT, ">= 0"),
        ({"ptr": None}, ARGUMENT, "non-null"),
        ({"residual": 16}, ARGUMENT, "go together"),
        ({"rs": 100}, ARGUMENT, "stride"),
        ({"scale_group": 48}, UNSUPPORTED, "scale_group"),
        ({"scale_group": 512}, UNSUPPORTED, "scale_group"),
        ({"scale_group": 128, "hidden": 192}, ARGUMENT, "multiple"),
        ({"dtype": 7}, UNSUPPORTED, "dtype"),
        ({"rows": 1 << 31}, UNSUPPORTED, "2^31"),
        ({"rows": 1 << 27, "hidden": 8192, "rs": 8192}, UNSUPPORTED, "too many rows"),
    ],
)
def test_norm(change, want, match):
    call("kl_rms_norm_fp8", norm(**change), want, match)


def append(dtype=BF16, cache=16, bounds=None, tokens=2, batch=2, heads=8, dim=128, page=16, pages=10, stride=4, width=4, offsets=None, ptr=16):
    return [dtype, cache, cache, ptr, ptr, bounds, ptr, ptr, heads * dim, dim, heads * dim, dim, ptr, ptr, offsets, tokens, batch,
            heads, dim, page, pages, stride, width, None]


@pytest.mark.parametrize(
    ("change", "want", "match"),
    [
        ({"tokens": 0, "batch": 0, "ptr": None}, OK, ""),
        ({"tokens": 0, "offsets": 16, "ptr": None}, OK, ""),
        ({"tokens": 3}, ARGUMENT, "one token"),
        ({"batch": -1}, ARGUMENT, "positive"),
        ({"heads": 0}, ARGUMENT, "positive"),
        ({"dim": 96}, UNSUPPORTED, "head_dim"),
        ({"page": 8}, UNSUPPORTED, "multiple of 16"),
        ({"ptr": None}, ARGUMENT, "non-null"),
        ({"stride": 3}, ARGUMENT, "stride"),
        ({"cache": 24}, ARGUMENT, "aligned"),
        ({"bounds": 24}, ARGUMENT, "aligned"),
        ({"tokens": 1 << 31, "offsets": 16}, UNSUPPORTED, "too many"),
        ({"dtype": 9}, UNSUPPORTED, "dtype"),
    ],
)
def test_append(change, want, match):
    call("kl_append_kv_fp8", append(**change), want, match)


def select(dtype=BF16, ptr=16, batch=2, hq=32, hkv=8, dim=128, page=16, stride=90, width=90, keep=12, first=1, last=1, bounds=16):
    return [dtype, ptr, ptr, ptr, bounds, ptr, ptr, ptr, batch, hq, hkv, dim, page, stride, width, keep, first, last, None, 0, None]


@pytest.mark.parametrize(
    ("change", "want", "match"),
    [
        ({"batch": 0, "ptr": None}, OK, ""),
        ({"batch": -1}, ARGUMENT, "positive"),
        ({"hq": 30}, ARGUMENT, "multiple"),
        ({"dtype": F32}, UNSUPPORTED, "fp16 or bf16"),
        ({"dim": 32}, UNSUPPORTED, "head_dim"),
        ({"page": 24}, UNSUPPORTED, "multiple of 16"),
        ({"first": -1}, ARGUMENT, "must fit"),
        ({"last": 0}, ARGUMENT, "must fit"),
        ({"first": 12}, ARGUMENT, "must fit"),
        ({"keep": 0}, ARGUMENT, "must fit"),
        ({"first": 2**31 - 1, "keep": 2**31 - 1, "last": 2**31 - 1}, ARGUMENT, "must fit"),
        ({"width": 0}, ARGUMENT, "max_pages"),
        ({"ptr": None}, ARGUMENT, "non-null"),
        ({"stride": 3}, ARGUMENT, "stride"),
        ({"bounds": 24}, ARGUMENT, "aligned"),
        ({"width": 1 << 28, "stride": 1 << 28}, UNSUPPORTED, "2^31"),
        ({"width": 9000, "stride": 9000}, WORKSPACE, "workspace"),
    ],
)
def test_select(change, want, match):
    call("kl_select_pages", select(**change), want, match)


def test_select_workspace():
    ws = ctypes.c_size_t(7)
    call("kl_select_pages_workspace", [2, 8, 90, ctypes.byref(ws)], OK)
    assert ws.value == 0
    call("kl_select_pages_workspace", [2, 8, 9000, ctypes.byref(ws)], OK)
    assert ws.value >= 2 * 8 * 9000 * 4
    call("kl_select_pages_workspace", [2, 0, 90, ctypes.byref(ws)], ARGUMENT, "positive")


def decode(dtype=BF16, ptr=16, scale=16, batch=2, hq=32, hkv=8, dim=128, page=16, stride=40, width=40, lists=0, splits=0):
    return [dtype, ptr, ptr, ptr, ptr, scale, scale, ptr, ptr, batch, hq, hkv, dim, page, stride, width, lists, 0.1, splits, None, 0, None]


@pytest.mark.parametrize("lists", [0, 1])
@pytest.mark.parametrize(
    ("change", "want", "match"),
    [
        ({"batch": 0, "ptr": None}, OK, ""),
        ({"batch": -1}, ARGUMENT, "positive"),
        ({"hq": 30}, ARGUMENT, "multiple"),
        ({"dtype": F32}, UNSUPPORTED, "fp16 or bf16"),
        ({"dim": 32}, UNSUPPORTED, "head_dim"),
        ({"page": 8}, UNSUPPORTED, "multiple of 16"),
        ({"scale": None}, ARGUMENT, "k_scale"),
        ({"ptr": None}, ARGUMENT, "non-null"),
        ({"stride": 3}, ARGUMENT, "stride"),
        ({"splits": -2}, ARGUMENT, "num_splits"),
        ({"splits": 4}, WORKSPACE, "workspace"),
        ({"ptr": 24}, ARGUMENT, "aligned"),
    ],
)
def test_decode(change, want, match, lists):
    call("kl_paged_decode_attention_fp8_pages", decode(lists=lists, **change), want, match)


def test_too_many_pairs():
    call("kl_paged_decode_attention_fp8_pages", decode(batch=2**29, lists=1), UNSUPPORTED, "pairs")
