"""The long caches' operators in 64 bits, built by sequence and row, and the bounds that the kernels are held to."""
from __future__ import annotations

import math

import torch

import blocktest as B
import dynalm_amd as dq
from blocktest import F32U, TYPES, U

KINDS = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


def stream() -> int:
    return torch.cuda.current_stream().cuda_stream


class Call:
    """A batch's tensors: places and page numbers that nothing may read hold NaN and numbers outside the cache."""

    def __init__(self, seed, new, lens, hq, hk, dim, type, cache, page, heads_first=False, spread=1.0, tail=0, odd=False):
        gen = torch.Generator().manual_seed(seed)
        self.new, self.lens, self.hq, self.hk, self.dim, self.type, self.cache, self.page = new, lens, hq, hk, dim, type, cache, page
        self.most, self.max_q = max(lens + [0]), max(new + [1])
        each = -(-self.most // page)
        total = each * len(new) + 1
        shape = (total, hk, page, dim) if heads_first else (total, page, hk, dim)
        pools = [torch.full(shape, math.nan, dtype=TYPES[cache]) for _ in range(2)]
        order = torch.randperm(total - 1, generator=gen).to(torch.int32)
        table = torch.full((len(new), each + 2), 2**31 - 1, dtype=torch.int32)
        self.ks, self.vs = [], []
        for b, n in enumerate(lens):
            mine = order[b * each : b * each + -(-n // page)].long()
            table[b, : len(mine)] = mine.to(torch.int32)
            own = [torch.randn((n, hk, dim), generator=gen).to(TYPES[cache]) for _ in range(2)]
            for pool, x in zip(pools, own):
                at = mine[torch.arange(n) // page], torch.arange(n) % page
                (pool.transpose(1, 2) if heads_first else pool)[at] = x
            self.ks.append(own[0])
            self.vs.append(own[1])
        offsets = [0]
        for n in new:
            offsets.append(offsets[-1] + n)
        self.offsets, self.rows, self.tokens = offsets, offsets[-1], offsets[-1] + tail
        q = torch.randn((self.tokens, hq, dim), generator=gen) * spread
        wide = torch.zeros((self.tokens, hq, dim + 3), dtype=TYPES[type])
        wide[..., 1 : dim + 1] = q.to(TYPES[type])
        wide = wide.cuda()
        self.q = wide[..., 1 : dim + 1] if odd else wide[..., 1 : dim + 1].contiguous()
        self.kc, self.vc = (p.cuda().transpose(1, 2) if heads_first else p.cuda() for p in pools)
        self.table, self.lens_d = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
        self.offsets_d = torch.tensor(offsets, dtype=torch.int32).cuda()
        self.scale = 1.0 / math.sqrt(dim)
        self.pages = each

    def c(self):
        return B.kv_cache(self.kc, self.vc)

    def seqs(self, no_offsets=False, max_len=None, max_q=None):
        return dq.Sequences(len(self.new), self.tokens, None if no_offsets else self.offsets_d.data_ptr(),
                            self.max_q if max_q is None else max_q, self.table.data_ptr(), self.table.stride(0), self.lens_d.data_ptr(),
                            self.most if max_len is None else max_len)

    def row(self, t):
        """The sequence of row t and the keys that it sees."""
        b = next(b for b in range(len(self.new)) if self.offsets[b] <= t < self.offsets[b + 1])
        return b, min(max(self.lens[b] - self.new[b] + t - self.offsets[b] + 1, 0), self.lens[b])

    def workspace(self, need):
        """`need` bytes of NaN, and behind them a guard."""
        assert 0 <= need <= dq.ATTENTION_WORKSPACE_BYTES
        return torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------ bounds


def page_bounds(call: Call, start=None, old=None):
    """Bounds of the pages of keys from start[b] on, on top of `old` [pages, kv_heads, 2, dim]."""
    out = old.clone()
    for b, n in enumerate(call.lens):
        first = 0 if start is None else min(max(start[b], 0), n)
        for p in range(first // call.page, -(-n // call.page)) if first < n else ():
            x = call.ks[b][p * call.page : min(n, (p + 1) * call.page)].double()
            lo, hi = x.amin(0), x.amax(0)  # (NaN if one is)
            out[int(call.table[b, p])] = torch.stack((lo, hi), 1).to(out.dtype)
    return out


def run_bounds(call: Call, start=None, max_new=None, old=None, **kw):
    bounds = torch.full((call.kc.shape[0], call.hk, 2, call.dim), 55.0, dtype=call.kc.dtype, device="cuda") if old is None else old.clone()
    f = None if start is None else torch.tensor(start, dtype=torch.int32, device="cuda")
    dq.page_bounds(call.c(), call.seqs(**kw), f, call.most if max_new is None else max_new, bounds, stream())
    return bounds


def same(got, want):
    """Equal values; NaN in the same places."""
    got, want = got.cpu().double(), want.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(want, 7.0))


# ------------------------------------------------------------------ the choice


def choose(call: Call, bounds, first, last, count):
    out = torch.full((call.tokens, call.hk, count), 77, dtype=torch.int32)
    group, bounds, q = call.hq // call.hk, bounds.cpu().double(), call.q.cpu().double()
    for t in range(call.rows):
        b, sees = call.row(t)
        pages = -(-sees // call.page)
        for h in range(call.hk):
            out[t, h] = -1
            ids = call.table[b, :pages].cpu().long()
            ok = (ids >= 0) & (ids < bounds.shape[0])
            near = bounds[torch.where(ok, ids, 0), h]
            score = torch.full((pages,), -math.inf, dtype=torch.float64)
            for i in range(h * group, (h + 1) * group):
                x = torch.where(q[t, i] > 0, near[:, 1], near[:, 0])
                score = torch.maximum(score, (x * q[t, i]).sum(-1))  # (NaN if one is)
            score[~ok] = math.nan
            rank = sorted(range(pages), key=lambda p: (not (p < first or p >= pages - last), not math.isnan(score[p]), -score[p].item()
                                                       if not math.isnan(score[p]) else 0.0, p))
            best = sorted(rank[:count])
            out[t, h, : len(best)] = torch.tensor(best, dtype=torch.int32)
    return out


def run_choose(call: Call, bounds, first, last, count, workspace=None, **kw):
    chosen = torch.full((call.tokens, call.hk, count), 77, dtype=torch.int32, device="cuda")
    s = call.seqs(**kw)
    need = dq.choose_pages_workspace(call.c(), s)
    work = call.workspace(need) if workspace is None else workspace
    dq.choose_pages(call.c(), s, B.heads(call.q), bounds, first, last, count, chosen, work, need, stream())
    assert workspace is not None or torch.all(work[need:] == 0xFF)
    return chosen


# ------------------------------------------------------------------ attention over chosen pages


def page_attention(call: Call, chosen):
    """(out, lse, bound of out, bound of lse) of the rows, from the formula in 64 bits."""
    tokens, group, dim = call.rows, call.hq // call.hk, call.dim
    out = torch.zeros((tokens, call.hq, dim), dtype=torch.float64)
    bound, lse = torch.zeros_like(out), torch.full((tokens, call.hq), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros_like(lse)
    chosen, q = chosen.cpu(), call.q.cpu().double()
    ut = 0.0 if call.type == "f32" else U[call.cache]
    for t in range(tokens):
        b, sees = call.row(t)
        for h in range(call.hk):
            keys = [j for p in chosen[t, h].tolist() if 0 <= p * call.page < sees and p >= 0 for j in range(p * call.page, min(sees, (p + 1) * call.page))]
            if not keys:
                continue
            kk, vv = call.ks[b][keys, h].double(), call.vs[b][keys, h].double()
            for i in range(h * group, (h + 1) * group):
                s = kk @ q[t, i] * call.scale
                z = torch.logsumexp(s, 0)
                p = torch.exp(s - z)
                # a score: dim products and sums in fp32 (and, split in parts, as much again), scaled, and its
                # distance to the maximum rounded; the weights' exponential, their sums over keys and the joins of parts;
                # 16-bit weights: one rounding (below f16's normal range: half its smallest step of the largest weight)
                d = ((dim + 16) * 2 * F32U * (kk.abs() @ q[t, i].abs()).max() * call.scale + 4 * F32U * (s.abs().max() + 16)).item()
                e = 2 * d + (64 + len(keys) / 8) * F32U + ut
                out[t, i], lse[t, i] = p @ vv, z
                bound[t, i] = e * (p @ vv.abs()) + (2.0**-25 * vv.abs().sum(0) * p.max() if call.type == "f16" else 0.0)
                lse_bound[t, i] = d + (64 + len(keys) / 8) * F32U + 2 * F32U * abs(z.item())
    return out, lse, bound, lse_bound


def run_attention(call: Call, chosen, out=None, lse=None, workspace=None, **kw):
    out = torch.full((call.tokens, call.hq, call.dim), 55.0, dtype=call.q.dtype, device="cuda") if out is None else out
    s, q, count = call.seqs(**kw), B.heads(call.q), chosen.shape[2]
    need = dq.page_attention_workspace(call.c(), s, q, count)
    work = call.workspace(need) if workspace is None else workspace
    dq.page_attention(call.c(), s, q, B.heads(out), lse, chosen, count, call.scale, work, need, stream())
    assert workspace is not None or torch.all(work[need:] == 0xFF)
    return out


def check_attention(call: Call, chosen, **kw):
    lse = torch.full((call.tokens, call.hq), 33.0, device="cuda")
    out = run_attention(call, chosen.cuda(), lse=lse, **kw)
    n = call.rows
    want, want_lse, bound, lse_bound = page_attention(call, chosen)
    B.close(out[:n], want, bound, call.type)
    assert torch.all(out[n:] == 55.0) and torch.all(lse[n:] == 33.0)  # rows of no sequence
    B.close(lse[:n], want_lse, lse_bound, "f32")
    return out


def some_pages(call: Call, count, seed=0, shuffled=False):
    """Lists of up to `count` pages that hold visible keys, -1 behind (or between, shuffled)."""
    gen = torch.Generator().manual_seed(seed)
    chosen = torch.full((call.tokens, call.hk, count), -1, dtype=torch.int32)
    for t in range(call.rows):
        b, sees = call.row(t)
        pages = -(-sees // call.page)
        for h in range(call.hk):
            mine = torch.randperm(pages, generator=gen)[: max(1, count - (t + h) % 3)].sort().values.to(torch.int32)
            chosen[t, h, : min(len(mine), count)] = mine[:count]
            if shuffled:
                chosen[t, h] = chosen[t, h, torch.randperm(count, generator=gen)]
    return chosen


# ------------------------------------------------------------------ weights


def mass(call: Call, lse, old, decay):
    """(mass, bound) [batch, kv_heads, width] from the formula in 64 bits; lse: float tensor."""
    out, q = old.double().cpu().clone(), call.q.cpu().double()
    bound = torch.zeros_like(out)
    group, dim, lse = call.hq // call.hk, call.dim, lse.cpu().double()
    for b, (n, k) in enumerate(zip(call.new, call.lens)):
        for h in range(call.hk):
            x = call.ks[b][:, h].double()
            total, err = torch.zeros(k, dtype=torch.float64), torch.zeros(k, dtype=torch.float64)
            for t in range(call.offsets[b], call.offsets[b] + n):
                sees = call.row(t)[1]
                for i in range(h * group, (h + 1) * group):
                    if sees == 0 or lse[t, i] == -math.inf:
                        continue
                    s = x[:sees] @ q[t, i] * call.scale
                    w = torch.exp(s - lse[t, i])
                    # a score as in the attention; its difference to lse in powers of two
                    d = (dim + 16) * 2 * F32U * (x[:sees].abs() @ q[t, i].abs()) * call.scale + 4 * F32U * (s.abs() + lse[t, i].abs() + 16)
                    total[:sees] += w
                    err[:sees] += w * 2 * d
            old_k = max(0, k - n)
            before = torch.zeros(k, dtype=torch.float64)
            if decay != 0:
                before[:old_k] = decay * out[b, h, :old_k]
            # (sums over rows: one after the other in a lane, then lanes and ranges)
            bound[b, h, :k] = err + (64 + n * group / 4) * F32U * total + 3 * F32U * before.abs()
            out[b, h, :k] = before + total
    return out, bound


def run_mass(call: Call, lse, out, decay, workspace=None, **kw):
    s, q = call.seqs(**kw), B.heads(call.q)
    need = dq.attention_mass_workspace(call.c(), s, q)
    work = call.workspace(need) if workspace is None else workspace
    dq.attention_mass(call.c(), s, q, lse, call.scale, decay, out, out.stride(0), out.stride(1), work, need, stream())
    assert workspace is not None or torch.all(work[need:] == 0xFF)
    return out


# ------------------------------------------------------------------ the keys that stay


def keep(weights, lens, first, last, budget):
    """kept [batch, kv_heads, budget]; weights: [batch, kv_heads, width]."""
    weights = weights.cpu()
    out = torch.full((len(lens), weights.shape[1], budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(weights.shape[1]):
            w = weights[b, h, :n].tolist()
            rank = sorted(range(n), key=lambda j: (not (j < first or j >= n - last), math.isnan(w[j]), 0.0 if math.isnan(w[j]) else -w[j], j))
            best = sorted(rank[:budget])
            out[b, h, : len(best)] = torch.tensor(best, dtype=torch.int32)
    return out


def run_keep(call_or_lens, weights, first, last, budget, max_len=None):
    lens = call_or_lens
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept = torch.full((len(lens), weights.shape[1], budget), 77, dtype=torch.int32, device="cuda")
    kept_lens = torch.full((len(lens),), 77, dtype=torch.int32, device="cuda")
    s = dq.Sequences(len(lens), 0, None, 1, None, 0, lens_d.data_ptr(), max(lens + [0]) if max_len is None else max_len)
    dq.kv_keep(s, weights.shape[1], weights, weights.stride(0), weights.stride(1), first, last, budget, kept, kept_lens, stream())
    return kept, kept_lens
