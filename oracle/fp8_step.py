"""Ground truth of the 8-bit serving step, in float64 on the CPU: the norm with an
FP8 output, the paged FP8 cache with scales per page and KV head, the choice of
pages by key bounds, and decode over both.

Written as plain loops over sequences, heads and pages from the definitions in
include/kernel_lab.h; E4M3 rounding is a search in the table of its values, not
torch's conversion.
"""

from __future__ import annotations

import torch

E4M3_MAX = 448.0
MIN_SCALE = 2.0**-126


def _e4m3_magnitudes() -> torch.Tensor:
    """The 127 finite magnitudes in code order: code = 8 * exponent + mantissa."""
    code = torch.arange(127, dtype=torch.float64)
    exponent, mantissa = torch.div(code, 8, rounding_mode="floor"), code % 8
    return torch.where(exponent == 0, mantissa * 2.0**-9, (1 + mantissa / 8) * torch.pow(2.0, exponent - 7))


_MAGNITUDES = _e4m3_magnitudes()


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """x rounded to the nearest E4M3 value, ties to the even code, as float64.
    Magnitudes that round past 448 and values that are not finite give NaN."""
    x = x.double()
    mag = x.abs()
    hi = torch.searchsorted(_MAGNITUDES, mag.contiguous()).clamp(1, 126)
    lo = hi - 1
    below, above = mag - _MAGNITUDES[lo], _MAGNITUDES[hi] - mag
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    out = torch.copysign(_MAGNITUDES[torch.where(up, hi, lo)], x)
    return torch.where(torch.isfinite(x) & (mag <= 464.0), out, float("nan"))


def scale_of(x: torch.Tensor, dims) -> torch.Tensor:
    """max over the finite |x| / 448, at least 2^-126, rounded to float32."""
    mag = torch.where(torch.isfinite(x.double()), x.double().abs(), 0.0).amax(dims)
    return (mag.float() / torch.tensor(E4M3_MAX)).clamp(min=MIN_SCALE)


def norm_fp8(x, residual, weight, eps=1e-6, group=None):
    """(y / scale before its rounding, scale, new residual): float64, float64, x's dtype."""
    if residual is not None:
        x = (x.float() + residual.float()).to(x.dtype)
    wide = x.double()
    y = wide / torch.sqrt((wide * wide).mean(-1, keepdim=True) + eps) * weight.double()
    width = group or y.shape[-1]
    parts = y.reshape(*y.shape[:-1], -1, width)
    mag = torch.where(torch.isfinite(parts), parts.abs(), 0.0).amax(-1)
    scale = (mag / E4M3_MAX).clamp(min=MIN_SCALE)
    return (parts / scale[..., None]).reshape(y.shape), scale, x


def append(k, v, cache, seq_lens, new_offsets=None):
    """``cache``: dict of k, v (float64 code values), k_scale, v_scale (float32), bounds (float64 or None) and
    block_table, changed in place as ``append_kv_fp8`` defines."""
    pages, page = cache["k"].shape[:2]
    table = cache["block_table"]
    batch = len(seq_lens)
    offsets = list(range(batch + 1)) if new_offsets is None else new_offsets.tolist()
    for b, total in enumerate(seq_lens.tolist()):
        begin, end = offsets[b], offsets[b + 1]
        start = total - (end - begin)
        if start < 0 or end <= begin or begin < 0 or end > k.shape[0]:
            continue
        for col in range(start // page, (total + page - 1) // page):
            if col >= table.shape[1] or not 0 <= int(table[b, col]) < pages:
                continue
            where = int(table[b, col])
            t0, t1 = max(start - col * page, 0), min(total - col * page, page)
            row = begin + col * page + t0 - start
            for name, x in (("k", k), ("v", v)):
                codes, scales = cache[name], cache[name + "_scale"]
                for h in range(codes.shape[2]):
                    new = x[row : row + t1 - t0, h]
                    old, scale = scales[where, h].clone(), scale_of(new, (0, 1))
                    if t0 and not old < scale:
                        scale = old
                    # The kernel's float32 steps: a product and a division, each rounded once.
                    again = t0 > 0 and bool(scale > old)
                    if again:
                        codes[where, :t0, h] = round_e4m3(codes[where, :t0, h].float() * old / scale)
                    codes[where, t0:t1, h] = round_e4m3(new.float() / scale)
                    scales[where, h] = scale
                    if name == "k" and cache["bounds"] is not None:
                        edge = cache["bounds"][where, h]
                        now = codes[where, t0:t1, h]
                        lo, hi = now.nan_to_num(nan=E4M3_MAX).amin(0), now.nan_to_num(nan=-E4M3_MAX).amax(0)
                        if t0:
                            held = round_e4m3(edge.float() * old / scale) if again else edge.clone()
                            lo, hi = torch.minimum(lo, held[0]), torch.maximum(hi, held[1])
                        edge[0], edge[1] = lo, hi


def page_tokens(codes, scales, pages, head, n):
    """The first n tokens on the given pages of one head, float64 [n, D]."""
    x = codes[pages, :, head].float().double() * scales[pages, head].double()[:, None, None]
    return x.reshape(-1, codes.shape[3])[:n]


def decode(q, k, v, block_table, seq_lens, k_scale, v_scale, scale=None):
    """(output, sum of p |v|) in float64; block tables per sequence, or per (sequence, KV head)."""
    batch, hq, dim = q.shape
    heads, page = k.shape[2], k.shape[1]
    group = hq // heads
    scale = dim**-0.5 if scale is None else scale
    out, size = torch.zeros(2, batch, hq, dim, dtype=torch.float64)
    for b in range(batch):
        for h in range(heads):
            row, n = (block_table[b, h], seq_lens[b, h]) if block_table.dim() == 3 else (block_table[b], seq_lens[b])
            n = min(int(n), block_table.shape[-1] * page)
            if n <= 0:
                continue
            ids = row[: (n + page - 1) // page].long()
            kk, vv = page_tokens(k, k_scale, ids, h, n), page_tokens(v, v_scale, ids, h, n)
            for g in range(h * group, (h + 1) * group):
                p = torch.softmax((kk @ q[b, g].double()) * scale, 0)
                out[b, g], size[b, g] = p @ vv, p @ vv.abs()
    return out, size


def select(q, bounds, k_scale, block_table, seq_lens, num_pages, page, first=1, last=1):
    """(table, lens) as ``select_pages`` defines."""
    batch, hq, _ = q.shape
    heads = bounds.shape[1]
    group = hq // heads
    table = torch.zeros(batch, heads, num_pages, dtype=torch.int32)
    lens = torch.zeros(batch, heads, dtype=torch.int32)
    for b in range(batch):
        n = max(0, min(int(seq_lens[b]), block_table.shape[1] * page))
        count = (n + page - 1) // page
        for h in range(heads):
            ids = block_table[b, :count].long()
            lo, hi = bounds[ids, h].float().double().unbind(1)
            score = torch.full((count,), float("-inf"), dtype=torch.float64)
            for g in range(h * group, (h + 1) * group):
                x = q[b, g].double()
                score = torch.maximum(score, (x.clamp(max=0) * lo + x.clamp(min=0) * hi).sum(-1))
            score = (score * k_scale[ids, h].double()).float()
            most = torch.finfo(torch.float32).max
            score = score.nan_to_num(nan=most, posinf=most, neginf=float("-inf"))
            score[:first] = float("inf")
            score[max(0, count - last) :] = float("inf")
            rank = sorted(range(count), key=lambda i, s=score.tolist(): (-s[i], i))[:num_pages]
            kept = sorted(rank)
            table[b, h, : len(kept)] = block_table[b, kept] if kept else 0
            lens[b, h] = (len(kept) - 1) * page + n - (count - 1) * page if kept else 0
    return table, lens
