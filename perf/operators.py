"""Performance cases of the 8-bit serving step: norm, cache append, page selection and decode attention.

Four kinds of case, one pass each through ``kernel_lab.ops`` (``own``) or through elementary torch operations:

* ``attend``  decode attention over a paged FP8 cache with a scale per page and KV head;
* ``sparse``  the pages of each (sequence, KV head) are chosen by the bounds of their keys, then attended;
* ``append``  new keys and values are rounded into the pages of the cache;
* ``norm8``   RMSNorm (with the residual's addition) into FP8 with a scale per row or group of columns.

FP8 outputs are float8_e4m3fn tensors beside their float32 scales.
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
TINY = 2.0**-126  # smallest scale
DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
F8 = torch.float8_e4m3fn


# --------------------------------------------------------------------- cases


def _heads(q_heads, kv_heads, head_dim, page):
    return {"q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page}


def listed() -> list[dict]:
    return [
        # One user, a short conversation: the smallest call, where latency counts.
        {"name": "attend b1 ctx512", "kind": "attend", "dtype": "bf16", "batch": 1, "ctx": 512, "ragged": False,
         **_heads(32, 8, 128, 16)},
        # A full serving batch at its longest context.
        {"name": "attend b64 ctx4096", "kind": "attend", "dtype": "fp16", "batch": 64, "ctx": 4096, "ragged": False,
         **_heads(32, 8, 128, 16)},
        # One KV head for all query heads, lengths as users leave them, larger pages.
        {"name": "attend mqa ragged", "kind": "attend", "dtype": "bf16", "batch": 64, "ctx": 8192, "ragged": True,
         **_heads(32, 1, 128, 64)},
        # Few sequences of book length on a larger head layout.
        {"name": "attend b8 ctx32768", "kind": "attend", "dtype": "bf16", "batch": 8, "ctx": 32768, "ragged": False,
         **_heads(64, 8, 128, 32)},
        # One user with a long document, 2,048 of its tokens attended.
        {"name": "sparse b1 ctx32768", "kind": "sparse", "dtype": "bf16", "batch": 1, "ctx": 32768, "ragged": False,
         "keep": 64, "first": 1, "last": 2, **_heads(32, 8, 128, 32)},
        # A serving batch of long, mixed contexts on small pages.
        {"name": "sparse b32 ragged 16384", "kind": "sparse", "dtype": "fp16", "batch": 32, "ctx": 16384,
         "ragged": True, "keep": 128, "first": 1, "last": 4, **_heads(32, 8, 128, 16)},
        # Eight book-length contexts, larger head layout and pages.
        {"name": "sparse b8 ctx65536", "kind": "sparse", "dtype": "bf16", "batch": 8, "ctx": 65536, "ragged": False,
         "keep": 64, "first": 1, "last": 1, **_heads(64, 8, 128, 64)},
        # A decode step of one user.
        {"name": "append b1 token", "kind": "append", "dtype": "bf16", "batch": 1, "ctx": 1024, "new": 1,
         "ragged": False, "bounds": True, **_heads(32, 8, 128, 16)},
        # A decode step of a full batch: one token each, at mixed places of their pages.
        {"name": "append b64 token", "kind": "append", "dtype": "fp16", "batch": 64, "ctx": 1024, "new": 1,
         "ragged": True, "bounds": True, **_heads(32, 8, 128, 16)},
        # Chunks of eight prompts, written behind what their sequences hold already.
        {"name": "append prompts", "kind": "append", "dtype": "bf16", "batch": 8, "ctx": 1024, "new": 4096,
         "ragged": True, "bounds": True, **_heads(32, 8, 128, 16)},
        # Pre-norm step of prefill ahead of an 8-bit projection with a scale per token.
        {"name": "norm8 4096x8192", "kind": "norm8", "dtype": "bf16", "rows": 4096, "hidden": 8192, "group": 0,
         "residual": True},
        # Pre-norm step of a small decode batch, a scale for each 128 columns.
        {"name": "norm8 16x4096 groups", "kind": "norm8", "dtype": "fp16", "rows": 16, "hidden": 4096, "group": 128,
         "residual": True},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


# Bytes of K and V codes of the largest listed case of a kind.
_MOST = {"attend": 2 * 8 * 32768 * 8 * 128, "sparse": 2 * 8 * 65536 * 8 * 128}


def draw(rng: random.Random) -> dict:
    """One more case: kinds in about the proportions of listed(), sizes over their whole ranges."""
    kind = rng.choice(["attend", "attend", "attend", "sparse", "sparse", "append", "append", "norm8", "norm8"])
    if kind == "norm8":
        rows = _log_int(rng, 1, 4096)
        # Model widths are multiples of 64; other widths are rarer, and have one scale a row.
        hidden = 64 * _log_int(rng, 2, 128) if rng.random() < 0.8 else _log_int(rng, 100, 8192)
        dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
        rows = max(1, min(rows, (32 << 20) // (hidden * (2 if dtype == "fp32" else 1))))
        groups = [0] + [g for g in (32, 64, 128, 256) if hidden % g == 0]
        return {"kind": kind, "dtype": dtype, "rows": rows, "hidden": hidden, "group": rng.choice(groups),
                "residual": rng.random() < 0.7}
    q_heads, kv_heads = rng.choice([(32, 8), (32, 8), (64, 8), (16, 4), (8, 8), (32, 1), (8, 1)])
    shape = _heads(q_heads, kv_heads, rng.choice([64, 128, 128, 256]), rng.choice([16, 16, 32, 64]))
    row = kv_heads * shape["head_dim"]
    ragged = rng.random() < 0.6
    if kind == "append":
        batch = _log_int(rng, 1, 128)
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 4096)
        new = max(1, min(new, (1 << 25) // (batch * row)))
        ctx = max(new, min(_log_int(rng, 16, 4096), (1 << 26) // (batch * row)))
        return {"kind": kind, "dtype": rng.choice(["fp16", "bf16", "bf16", "fp32"]), "batch": batch, "ctx": ctx,
                "new": new, "ragged": ragged, "bounds": rng.random() < 0.7, **shape}
    batch = _log_int(rng, 1, 128 if kind == "attend" else 64)
    ctx = _log_int(rng, 64 if kind == "attend" else 1024, 32768 if kind == "attend" else 131072)
    ctx = max(16, min(ctx, _MOST[kind] // (2 * batch * row)))
    case = {"kind": kind, "dtype": rng.choice(["fp16", "bf16"]), "batch": batch, "ctx": ctx, "ragged": ragged, **shape}
    if kind == "sparse":
        case.update(keep=_log_int(rng, 8, max(8, 4096 // shape["page"])), first=rng.choice([0, 1, 1]),
                    last=rng.choice([1, 1, 2, 4]))
    return case


# -------------------------------------------------------------------- inputs


def _lens(case: dict, seed: int) -> list[int]:
    """The batch's lengths. Ragged ones are uniform on [1, ctx]: which lengths there are depends on the case alone,
    their order in the batch on the seed. A cache to append to holds these tokens before the call."""
    batch, ctx = case["batch"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * batch
    rng = random.Random(batch * 1000003 + ctx)
    lens = [rng.randint(1, ctx) for _ in range(batch)]
    random.Random(seed).shuffle(lens)
    return lens


def _news(case: dict, seed: int) -> list[int]:
    """New tokens of each sequence: one each, or (ragged chunks) from half of ``new`` to all of it."""
    batch, new = case["batch"], case["new"]
    if new == 1 or not case["ragged"]:
        return [new] * batch
    rng = random.Random(batch * 1000003 + new)
    news = [rng.randint((new + 1) // 2, new) for _ in range(batch)]
    random.Random(seed + 1).shuffle(news)
    return news


def _pages(n: int, page: int) -> int:
    return (n + page - 1) // page


def _round_pages(x: torch.Tensor, live: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of pages [n, P, H, D] whose tokens `live` [n, P] count; the others' codes are NaN."""
    on = live[:, :, None, None]
    scale = (torch.where(on, x, 0.0).abs().amax((1, 3)) / E4M3_MAX).clamp(min=TINY)
    codes = (x / scale[:, None, :, None]).to(F8)
    return torch.where(on, codes.float(), float("nan")).to(F8), scale


def _cache(case: dict, lens: list[int], spare: list[int], gen: torch.Generator) -> dict:
    """A paged cache holding `lens` tokens a sequence, with room for `spare` tokens more; pages lie in random order.
    Keys and values are normal, their size differing from page to page and (keys) from dimension to dimension."""
    page, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    need = [_pages(n + m, page) for n, m in zip(lens, spare)]
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device=DEVICE)
    rows = torch.arange(len(lens), device=DEVICE)
    counts = torch.tensor(need, device=DEVICE)
    width = max(need)
    col = torch.arange(width, device=DEVICE)
    used = col[None, :] < counts[:, None]
    table = torch.zeros(len(lens), width, dtype=torch.int32, device=DEVICE)
    table[used] = order[: sum(need)].to(torch.int32)
    held = torch.zeros(total, dtype=torch.int64, device=DEVICE)  # tokens on each page
    tokens = torch.tensor(lens, device=DEVICE)
    on_page = (tokens[:, None] - col[None, :] * page).clamp(0, page)
    held[table[used].long()] = on_page[used]
    live = torch.arange(page, device=DEVICE)[None, :] < held[:, None]
    s = {"table": table, "lens": tokens.to(torch.int32), "rows": rows}
    channel = torch.exp(0.7 * torch.randn(heads, dim, generator=gen, device=DEVICE))
    for name in ("k", "v"):
        codes = torch.empty(total, page, heads, dim, dtype=F8, device=DEVICE)
        scale = torch.empty(total, heads, device=DEVICE)
        step = max(1, (1 << 27) // (page * heads * dim))
        for i in range(0, total, step):
            n = min(step, total - i)
            x = torch.randn(n, page, heads, dim, generator=gen, device=DEVICE)
            x *= torch.exp(0.4 * torch.randn(n, 1, heads, 1, generator=gen, device=DEVICE))
            if name == "k":
                x *= channel
                # What a page's tokens have in common, by which pages differ.
                x += 0.5 * channel * torch.randn(n, 1, heads, dim, generator=gen, device=DEVICE)
            c, scale[i : i + n] = _round_pages(x, live[i : i + n])
            codes[i : i + n] = c
        s[name], s[name + "_scale"] = codes, scale
    if case["kind"] == "sparse" or case.get("bounds"):
        bounds = torch.empty(total, heads, 2, dim, dtype=F8, device=DEVICE)
        for i in range(0, total, step):
            c = s["k"][i : i + step].float()
            bounds[i : i + step, :, 0] = c.nan_to_num(nan=E4M3_MAX).amin(1).to(F8)
            bounds[i : i + step, :, 1] = c.nan_to_num(nan=-E4M3_MAX).amax(1).to(F8)
        s["bounds"] = bounds
    return s


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def rand(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)

    if case["kind"] == "norm8":
        rows, hidden = case["rows"], case["hidden"]
        s = {"case": case, "x": rand(rows, hidden), "group": case["group"] or None}
        # A stream with a few columns much larger than the others, as trained models have.
        s["x"][:, :: max(1, hidden // 5)] *= 8
        s["residual"] = rand(rows, hidden) if case["residual"] else None
        s["weight"] = (1 + 0.1 * torch.randn(hidden, generator=gen, device=DEVICE)).to(dtype)
        return s
    lens = _lens(case, seed)
    news = _news(case, seed) if case["kind"] == "append" else [0] * len(lens)
    s = {"case": case, **_cache(case, lens, news, gen)}
    if case["kind"] == "append":
        total = sum(news)
        # Keys and values as one projection of queries, keys and values leaves them.
        heads, dim = case["q_heads"] + 2 * case["kv_heads"], case["head_dim"]
        kv = rand(total, heads, dim)
        kv *= torch.exp(0.4 * torch.randn(total, heads, 1, generator=gen, device=DEVICE)).to(dtype)
        s["k_new"] = kv[:, case["q_heads"] : case["q_heads"] + case["kv_heads"]]
        s["v_new"] = kv[:, case["q_heads"] + case["kv_heads"] :]
        s["lens"] = s["lens"] + torch.tensor(news, dtype=torch.int32, device=DEVICE)
        s["offsets"] = None
        if case["new"] > 1:
            s["offsets"] = torch.tensor([0, *news], device=DEVICE).cumsum(0).to(torch.int32)
        return s
    s["q"] = rand(case["batch"], case["q_heads"], case["head_dim"])
    return s


# --------------------------------------------------------------- plain forms


def _plain_norm8(x, residual, weight, group):
    if residual is not None:
        residual = (x.float() + residual.float()).to(x.dtype)
        x = residual
    f = x.float()
    y = f / torch.sqrt((f * f).mean(-1, keepdim=True) + EPS) * weight.float()
    g = y.reshape(*y.shape[:-1], -1, group or y.shape[-1])
    scale = (g.abs().amax(-1) / E4M3_MAX).clamp(min=TINY)
    codes = (g / scale[..., None]).reshape(y.shape).to(F8)
    return {"out": codes, "scale": scale, "residual": residual}


def _plain_attend(q, codes_k, codes_v, scale_k, scale_v, live):
    """q [B, H, G, D]; codes [B, H or 1, N, P, D]; scales [B, H, N]; live [B, H or 1, N * P]."""
    b, h, g, d = q.shape
    k = (codes_k.float() * scale_k[..., None, None]).reshape(b, h, -1, d)
    v = (codes_v.float() * scale_v[..., None, None]).reshape(b, h, -1, d)
    k = torch.where(live[..., None], k, 0.0)
    v = torch.where(live[..., None], v, 0.0)
    s = torch.matmul(k, q.float().transpose(2, 3).contiguous()) * d**-0.5  # [B, H, L, G]
    s = torch.where(live[..., None], s, float("-inf"))
    m = s.amax(2, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    total = p.sum(2)  # [B, H, G]
    o = torch.matmul(p.transpose(2, 3).contiguous(), v)
    o = o / torch.where(total > 0, total, 1.0)[..., None]
    return o.to(q.dtype).reshape(b, h * g, d)


def _plain_dense(s):
    case, table = s["case"], s["table"].long()
    b, heads, dim = case["batch"], case["kv_heads"], case["head_dim"]
    q = s["q"].reshape(b, heads, -1, dim)
    k, v = (s[c].view(torch.uint8)[table].view(F8).permute(0, 3, 1, 2, 4) for c in ("k", "v"))
    ks, vs = (s[c][table].transpose(1, 2) for c in ("k_scale", "v_scale"))
    at = torch.arange(table.shape[1] * case["page"], device=table.device)
    live = (at[None, :] < s["lens"][:, None])[:, None, :]
    return _plain_attend(q, k, v, ks, vs, live)


def _plain_sparse(s):
    case, table, page = s["case"], s["table"].long(), s["case"]["page"]
    b, heads, dim = case["batch"], case["kv_heads"], case["head_dim"]
    q = s["q"].reshape(b, heads, -1, dim)
    width = table.shape[1]
    bounds = s["bounds"].view(torch.uint8)[table].view(F8).double().permute(3, 0, 2, 1, 4)  # [2, B, H, N, D]
    wide = q.double().transpose(2, 3).contiguous()
    score = torch.matmul(bounds[0].contiguous(), wide.clamp(max=0)) + torch.matmul(bounds[1].contiguous(), wide.clamp(min=0))
    score = (score.amax(-1) * s["k_scale"][table].transpose(1, 2).double()).float()  # [B, H, N]
    count = ((s["lens"] + page - 1) // page).long()[:, None, None]
    at = torch.arange(width, device=table.device)
    pinned = (at < case["first"]) | (at >= count - case["last"])
    score = torch.where(pinned, float("inf"), score)
    score = torch.where(at < count, score, float("-inf"))
    keep = min(case["keep"], width)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = count.clamp(max=keep)  # [B, 1, 1]
    rank = torch.arange(keep, device=table.device)
    best = torch.where(rank < kept, best, width).sort(-1).values
    chosen = torch.where(rank < kept, table[:, None, :].expand(b, heads, width).gather(2, best.clamp(max=width - 1)), 0)
    tail = s["lens"].long()[:, None, None] - (count - 1) * page
    lens = torch.where(kept > 0, (kept - 1) * page + tail, 0).expand(b, heads, 1)[..., 0]
    padded = torch.zeros(b, heads, case["keep"], dtype=torch.int32, device=table.device)
    padded[..., :keep] = chosen.to(torch.int32)
    head = torch.arange(heads, device=table.device)[None, :, None]
    k, v = (s[c].view(torch.uint8)[chosen, :, head].view(F8) for c in ("k", "v"))  # [B, H, n, P, D]
    live = torch.arange(keep * page, device=table.device) < lens[..., None]
    out = _plain_attend(q, k, v, s["k_scale"][chosen, head], s["v_scale"][chosen, head], live)
    return {"table": padded, "lens": lens.to(torch.int32), "out": out}


def _plain_append_one(x, codes, scale, table, start, phys, slot):
    """Rounds the tokens x [T, H, D] into their pages; returns the old scales and which pages held tokens before."""
    page, heads = codes.shape[1], codes.shape[2]
    f = x.float()
    amax = torch.where(torch.isfinite(f), f, 0.0).abs().amax(-1)  # [T, H]
    new = torch.full_like(scale, -1.0).scatter_reduce(0, phys[:, None].expand(-1, heads), amax / E4M3_MAX, "amax")
    touched = new >= 0
    new = new.clamp(min=TINY)
    # A sequence's first touched page may hold tokens already; the others start empty.
    first = table.gather(1, (start // page).clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    held = start % page  # [B]
    holds = torch.zeros(scale.shape[0], dtype=torch.bool, device=scale.device)
    holds[first[held > 0]] = True
    old = scale.clone()
    scale.copy_(torch.where(touched, torch.where(holds[:, None], torch.maximum(old, new), new), old))
    ratio_old, ratio_new = old[first], scale[first]  # [B, H]
    mine = codes.view(torch.uint8)[first].view(F8)  # [B, P, H, D]
    again = (mine.float() * ratio_old[:, None, :, None] / ratio_new[:, None, :, None]).to(F8)
    at = torch.arange(page, device=scale.device)[None, :, None, None]
    grown = (at < held[:, None, None, None]) & (ratio_new > ratio_old)[:, None, :, None]
    raw = codes.view(torch.uint8)
    raw[first] = torch.where(grown, again.view(torch.uint8), mine.view(torch.uint8))
    raw[phys, slot] = (f / scale[phys][..., None]).to(F8).view(torch.uint8)
    return old, holds, touched


def _plain_append(s):
    case, table = s["case"], s["table"].long()
    page, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    t = s["k_new"].shape[0]
    offsets = torch.arange(case["batch"] + 1, device=table.device) if s["offsets"] is None else s["offsets"].long()
    n = offsets[1:] - offsets[:-1]
    seq = torch.repeat_interleave(s["rows"], n, output_size=t)
    start = s["lens"].long() - n
    pos = start[seq] + torch.arange(t, device=table.device) - offsets[seq]
    phys, slot = table[seq, pos // page], pos % page
    old, holds, touched = _plain_append_one(s["k_new"], s["k"], s["k_scale"], table, start, phys, slot)
    _plain_append_one(s["v_new"], s["v"], s["v_scale"], table, start, phys, slot)
    out = {c: s[c] for c in ("k", "v", "k_scale", "v_scale")}
    if case["bounds"]:
        b = s["bounds"].float()
        grown = (s["k_scale"] > old)[..., None, None]
        b_held = torch.where(grown, (b * old[..., None, None] / s["k_scale"][..., None, None]).to(F8).float(), b)
        codes = s["k"].view(torch.uint8)[phys, slot].view(F8).float()  # [T, H, D]
        at = phys[:, None, None].expand(-1, heads, dim)
        kept = holds[:, None, None]
        lo = torch.where(kept, b_held[:, :, 0], E4M3_MAX).scatter_reduce(0, at, codes, "amin")
        hi = torch.where(kept, b_held[:, :, 1], -E4M3_MAX).scatter_reduce(0, at, codes, "amax")
        fresh = torch.where(touched[..., None, None], torch.stack([lo, hi], 2), b)
        s["bounds"].copy_(fresh.to(F8))
        out["bounds"] = s["bounds"]
    return out


# ----------------------------------------------------------------------- run


@functools.lru_cache(maxsize=1)
def _ops():
    path = str(Path(__file__).resolve().parent.parent / "kernel-lab_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from kernel_lab import ops

    return ops


def _own_run(s):
    ops, kind = _ops(), s["case"]["kind"]
    if kind == "norm8":
        if s["residual"] is None:
            out, scale = ops.rms_norm_fp8(s["x"], s["weight"], EPS, group_size=s["group"])
            return {"out": out, "scale": scale, "residual": None}
        out, scale, residual = ops.fused_add_rms_norm_fp8(s["x"], s["residual"], s["weight"], EPS, group_size=s["group"])
        return {"out": out, "scale": scale, "residual": residual}
    if kind == "attend":
        return ops.paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], k_scale=s["k_scale"],
                                          v_scale=s["v_scale"])
    if kind == "sparse":
        case = s["case"]
        table, lens = ops.select_pages(s["q"], s["bounds"], s["k_scale"], s["table"], s["lens"], case["keep"],
                                       page_size=case["page"], first_pages=case["first"], last_pages=case["last"])
        out = ops.paged_decode_attention(s["q"], s["k"], s["v"], table, lens, k_scale=s["k_scale"],
                                         v_scale=s["v_scale"])
        return {"table": table, "lens": lens, "out": out}
    ops.append_kv_fp8(s["k_new"], s["v_new"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["lens"],
                      new_offsets=s["offsets"], k_bounds=s.get("bounds"))
    return {c: s[c] for c in ("k", "v", "k_scale", "v_scale", "bounds") if c in s}


def run(s: dict):
    if own:
        return _own_run(s)
    kind = s["case"]["kind"]
    if kind == "norm8":
        return _plain_norm8(s["x"], s["residual"], s["weight"], s["group"])
    return {"attend": _plain_dense, "sparse": _plain_sparse, "append": _plain_append}[kind](s)


def work(case: dict) -> dict:
    """Each input that the operator needs read once, each output written once."""
    size, kind = SIZES[case["dtype"]], case["kind"]
    if kind == "norm8":
        n = case["rows"] * case["hidden"]
        scales = case["rows"] * (case["hidden"] // case["group"] if case["group"] else 1)
        moved = (3 if case["residual"] else 1) * size + 1
        return {"bytes": moved * n + case["hidden"] * size + 4 * scales, "flops": 7 * n}
    heads, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    lens = _lens(case, 0)
    if kind == "append":
        tokens = sum(_news(case, 0))
        pages = sum(_pages(n + m, page) - n // page for n, m in zip(lens, _news(case, 0)))
        side = 2 * 4 + (2 * dim if case["bounds"] else 0)
        return {"bytes": 2 * tokens * heads * dim * (size + 1) + pages * heads * side,
                "flops": 4 * tokens * heads * dim}
    rows = 2 * case["batch"] * case["q_heads"] * dim * size
    per_page = 4 + 8 * heads  # table entry, scales
    if kind == "attend":
        pages = sum(_pages(n, page) for n in lens)
        return {"bytes": 2 * sum(lens) * heads * dim + pages * per_page + rows,
                "flops": 4 * sum(lens) * case["q_heads"] * dim}
    pages = sum(_pages(n, page) for n in lens)
    kept = sum(min(_pages(n, page), case["keep"]) for n in lens)
    tokens = sum(n - page * max(0, _pages(n, page) - case["keep"]) for n in lens)
    scored = pages * (2 * heads * dim + 4 * heads + 4)
    return {"bytes": scored + 2 * tokens * heads * dim + kept * heads * 16 + rows + case["batch"] * heads * 8,
            "flops": 4 * pages * case["q_heads"] * dim + 4 * tokens * case["q_heads"] * dim}


# ------------------------------------------------------------------ in 64 bits


def _wide_attention(q, k, v):
    """Softmax attention of q [H, G, D] over k, v [H, n, D] in 64 bits."""
    if k.shape[1] == 0:
        return torch.zeros_like(q).reshape(-1, q.shape[-1])
    w = torch.softmax(torch.bmm(q, k.transpose(1, 2).contiguous()) * q.shape[-1] ** -0.5, -1)
    return torch.bmm(w, v).reshape(-1, q.shape[-1])


def _exact_attend(s, case):
    q, page, heads = s["q"].double(), case["page"], case["kv_heads"]
    out = torch.empty_like(q)
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, : _pages(n, page)].long()
        kv = []
        for c in ("k", "v"):
            x = s[c].view(torch.uint8)[pages].view(F8).double() * s[c + "_scale"][pages].double()[:, None, :, None]
            kv.append(x.reshape(-1, heads, case["head_dim"])[:n].transpose(0, 1).contiguous())
        out[b] = _wide_attention(q[b].reshape(heads, -1, case["head_dim"]), *kv)
    return out


def _exact_sparse(s, case):
    q, page, heads, dim, keep = s["q"].double(), case["page"], case["kv_heads"], case["head_dim"], case["keep"]
    out = torch.zeros_like(q)
    for b, n in enumerate(s["lens"].tolist()):
        count = _pages(n, page)
        if count == 0:
            continue
        pages = s["table"][b, :count].long()
        edge = s["bounds"].view(torch.uint8)[pages].view(F8).double()  # [N, H, 2, D]
        qb = q[b].reshape(heads, -1, dim)
        kv = [[], []]
        for h in range(heads):
            # The largest q.k that a key between the bounds can have.
            best = [torch.where(x >= 0, x * edge[:, h, 1], x * edge[:, h, 0]).sum(-1) for x in qb[h]]
            score = (torch.stack(best).amax(0) * s["k_scale"][pages, h].double()).float().cpu()
            score[: case["first"]] = math.inf
            score[max(0, count - case["last"]) :] = math.inf
            order = sorted(range(count), key=lambda i, v=score.tolist(): (-v[i], i))
            mine = pages[torch.tensor(sorted(order[:keep]), device=pages.device)]
            tokens = (mine.numel() - 1) * page + n - (count - 1) * page
            for c, to in (("k", kv[0]), ("v", kv[1])):
                x = s[c].view(torch.uint8)[mine, :, h].view(F8).double() * s[c + "_scale"][mine, h].double()[:, None, None]
                to.append(x.reshape(-1, dim)[:tokens])
        out[b] = _wide_attention(qb, torch.stack(kv[0]), torch.stack(kv[1]))
    return {"table": None, "lens": None, "out": out}


def _exact_append(s, case):
    """Before the codes' rounding: what each code stands for, over its scale."""
    page = case["page"]
    lens = s["lens"].tolist()
    ends = s["offsets"].tolist()[1:] if s["offsets"] is not None else list(range(1, len(lens) + 1))
    table = s["table"].tolist()
    out = {}
    for c in ("k", "v"):
        codes, scale = s[c].double(), s[c + "_scale"].double()
        bounds = s["bounds"].double() if c == "k" and case["bounds"] else None
        begin = 0
        for b, (total, end) in enumerate(zip(lens, ends)):
            x = s[c + "_new"][begin:end].double()
            pos = total - (end - begin)
            begin = end
            while x.shape[0]:
                slot, where = pos % page, table[b][pos // page]
                part = x[: page - slot]
                x, pos = x[part.shape[0] :], pos + part.shape[0]
                new = (part.abs().amax((0, 2)) / E4M3_MAX).clamp(min=TINY)
                if slot:
                    before = scale[where].clone()
                    new = torch.maximum(before, new)
                    codes[where, :slot] *= (before / new)[:, None]
                scale[where] = new
                codes[where, slot : slot + part.shape[0]] = part / new[:, None]
                if bounds is not None:
                    now = codes[where, : slot + part.shape[0]]
                    bounds[where, :, 0], bounds[where, :, 1] = now.amin(0), now.amax(0)
        out[c], out[c + "_scale"] = codes, scale
        if bounds is not None:
            out["bounds"] = bounds
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(s, case)
    if case["kind"] == "sparse":
        return _exact_sparse(s, case)
    if case["kind"] == "append":
        return _exact_append(s, case)
    x = s["x"]
    if s["residual"] is not None:
        # The residual stream is kept in its type, and that rounded value is normalised.
        x = (x.float() + s["residual"].float()).to(x.dtype)
    wide = x.double()
    y = wide * (wide.pow(2).sum(-1, keepdim=True) / wide.shape[-1] + EPS).rsqrt() * s["weight"].double()
    width = case["group"] or case["hidden"]
    scale = torch.stack([part.abs().amax(-1) for part in y.split(width, -1)], -1) / E4M3_MAX
    # The codes before their rounding.
    return {"out": y / scale.repeat_interleave(width, -1), "scale": scale,
            "residual": wide if s["residual"] is not None else None}
