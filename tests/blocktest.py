"""The attention block's operators in 64 bits, and the bounds that the kernels are held to."""
from __future__ import annotations

import math

import torch

import dynalm_amd as dq

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KINDS = {torch.float32: dq.F32, torch.float16: dq.F16, torch.bfloat16: dq.BF16}
U = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}      # half a unit in the last place, relative
TINY = {"f32": 2.0**-149, "f16": 2.0**-24, "bf16": 2.0**-133}  # and the smallest step
F32U = 2.0**-24


def heads(x: torch.Tensor) -> dq.Heads:
    """x: [tokens, heads, dim], a head's values contiguous."""
    assert x.stride(2) == 1
    return dq.Heads(x.data_ptr(), KINDS[x.dtype], x.shape[1], x.stride(0), x.stride(1))


def kv_cache(k: torch.Tensor, v: torch.Tensor) -> dq.KvCache:
    """k, v: [pages, page, kv_heads, dim], strided alike."""
    assert k.stride() == v.stride() and k.stride(3) == 1
    return dq.KvCache(k.data_ptr(), v.data_ptr(), KINDS[k.dtype], k.shape[2], k.shape[3], k.shape[1], k.shape[0], k.stride(0),
                      k.stride(1), k.stride(2))


def rope_table(longest: int, rot: int):
    a = torch.arange(longest, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    return a.cos().float(), a.sin().float()


def norm_rope(x, weight, eps, tables, positions, rot: int, halves: bool):
    """(values, bound without the last rounding) of norm and rotation of x [tokens, heads, dim]."""
    x = x.double()
    y = x
    # the sum of squares: log2(dim) + a few roundings of non-negative terms; root, quotient and two products
    u = 0.0
    if weight is not None:
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
        u = 24 * F32U
    if tables is None:
        return y, u * y.abs()
    cos, sin = tables[0].double(), tables[1].double()
    inside = (positions >= 0) & (positions < cos.shape[0])
    at = torch.where(inside, positions, 0).long()
    c, s = cos[at][:, None], sin[at][:, None]
    c = torch.where(inside[:, None, None], c, math.nan)
    s = torch.where(inside[:, None, None], s, math.nan)
    out, bound = y.clone(), u * y.abs()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if halves else (slice(0, rot, 2), slice(1, rot, 2))
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    size = (y[..., a] * c).abs() + (y[..., b] * s).abs(), (y[..., b] * c).abs() + (y[..., a] * s).abs()
    bound[..., a], bound[..., b] = (u + 3 * F32U) * size[0], (u + 3 * F32U) * size[1]
    return out, bound


def close(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, type: str) -> None:
    """got (of `type`) is within bound, and one rounding, of want; NaN and infinite in the same places."""
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    room = bound + U[type] * (want.abs() + bound) + TINY[type]
    over = ((got - want).abs() - room)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"over the bound by {over.max():.3g} (of {room[fine].max():.3g})"


def attention(q, ks, vs, lens_q, lens, prefix: int, scale: float, type: str, cache_type: str):
    """(out, lse, bound of out, bound of lse) for q [tokens, heads, dim] and a list of each
    sequence's keys and values [prefix + own, kv_heads, dim] in 64 bits."""
    tokens, nh, dim = q.shape
    out = torch.zeros((tokens, nh, dim), dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((tokens, nh), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros_like(lse)
    start = 0
    ut = 0.0 if type == "f32" else U[cache_type]
    for b, n in enumerate(lens_q):
        k, v = ks[b].double(), vs[b].double()
        group = nh // k.shape[1]
        for i in range(n):
            seen = prefix + max(0, min(lens[b], lens[b] - n + i + 1))
            if seen == 0:
                continue
            for h in range(nh):
                kk, vv = k[:seen, h // group], v[:seen, h // group]
                qq = q[start + i, h].double()
                s = kk @ qq * scale
                z = torch.logsumexp(s, 0)
                p = torch.exp(s - z)
                pv = p @ vv
                size = p @ vv.abs()
                # a score: dim products and sums in fp32 (and, split in parts, as much again), scaled, and
                # its distance to the maximum rounded
                d = ((dim + 16) * 2 * F32U * (kk.abs() @ qq.abs()).max() * scale + 4 * F32U * (s.abs().max() + 16)).item()
                # the weights' exponential, the sums over keys, the joins of parts; 16-bit weights: one rounding
                # (below f16's normal range: half its smallest step of the largest weight)
                e = 2 * d + (64 + seen / 8) * F32U + ut
                out[start + i, h] = pv
                bound[start + i, h] = e * size + (2.0**-25 * vv.abs().sum(0) * p.max() if type == "f16" else 0.0)
                lse[start + i, h] = z
                lse_bound[start + i, h] = d + (64 + seen / 8) * F32U + 2 * F32U * abs(z.item())
        start += n
    return out, lse, bound, lse_bound


def attention_by_heads(q, ks, vs, lens_q, lens, prefix: int, scale: float, type: str, cache_type: str):
    """`attention` for many rows: the same values and bounds, a sequence's head at a time, on q's device."""
    tokens, nh, dim = q.shape
    out = torch.zeros((tokens, nh, dim), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lse = torch.full((tokens, nh), -math.inf, dtype=torch.float64, device=q.device)
    lse_bound = torch.zeros_like(lse)
    start = 0
    ut = 0.0 if type == "f32" else U[cache_type]
    for b, n in enumerate(lens_q):
        k, v = ks[b].to(q.device).double(), vs[b].to(q.device).double()
        group = nh // k.shape[1]
        seen = prefix + torch.clamp(lens[b] - n + 1 + torch.arange(n, device=q.device), 0, lens[b])
        hidden = torch.arange(k.shape[0], device=q.device)[None, :] >= seen[:, None]
        some = seen > 0
        rows = slice(start, start + n)
        for h in range(nh if n and k.shape[0] else 0):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[rows, h].double()
            s = (qq @ kk.t().contiguous() * scale).masked_fill(hidden, -math.inf)
            z = torch.logsumexp(s, 1)
            p = torch.where(some[:, None], torch.exp(s - z[:, None]), 0.0)
            size = p @ vv.abs()
            most = (qq.abs() @ kk.abs().t().contiguous()).masked_fill(hidden, 0.0).amax(1)
            d = (dim + 16) * 2 * F32U * most * scale + 4 * F32U * (s.masked_fill(hidden, 0.0).abs().amax(1) + 16)
            steps = (64 + seen / 8) * F32U
            low = 2.0**-25 * ((~hidden).double() @ vv.abs()) * p.amax(1, keepdim=True) if type == "f16" else 0.0
            out[rows, h] = p @ vv
            bound[rows, h] = (2 * d + steps + ut)[:, None] * size + low
            lse[rows, h] = z
            lse_bound[rows, h] = torch.where(some, d + steps + 2 * F32U * z.abs(), 0.0)
        start += n
    return out.cpu(), lse.cpu(), bound.cpu(), lse_bound.cpu()
