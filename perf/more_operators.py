"""The operators of long caches whose time is measured, each as a user's program calls it.

A decode step over a long paged cache need not read every key, and a cache need not keep every
key. `page_bounds` writes the smallest and the largest value of each channel over a page's keys,
`choose_pages` bounds with them what a query can score on a page and lists the pages that it
reads, `page_attention` attends to the keys of those pages, `attention_mass` adds up the attention
weight that each key gathers, and `kv_keep` with `kv_compact` leaves the keys of largest
weight in the cache. The listed cases are decode steps and prompts of models with the head
shapes of the benchmark's layers; `draw` spreads sequences, lengths, heads, head sizes, types and
pages over the same ranges.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
WORKSPACE_BYTES = 128 << 20

# batch sequences of up to `keys` keys each in pages of `page` tokens; heads_first: pages are
# [heads][tokens][dim], else [tokens][heads][dim]. queries: a sequence's rows (new tokens), at most.
# kind "bounds": the pages of the last `new` keys (0: of all).
# kind "choose": `count` pages a row and kv head, the `first` first and `last` last among them.
# kind "attend": over `count` such pages.
# kind "mass": the weights of the rows, on top of decay times what the keys had.
# kind "evict": `budget` keys stay in each kv head, the `first` first and `last` last among them; moved: into
#   pages of their own, else to the front of the sequence's.


def listed() -> list[dict]:
    return [
        # one decode step of 64 sequences: the page of the new key, all latency
        dict(name="bounds_step_64", kind="bounds", batch=64, keys=4096, new=1, kv_heads=8, dim=128, cache="bf16", page=64,
             heads_first=True),
        # after prompts, or after an eviction: every page
        dict(name="bounds_prompts", kind="bounds", batch=8, keys=16384, new=0, kv_heads=8, dim=128, cache="f16", page=16,
             heads_first=False),
        # two sequences of a small model, fp32 rows as this framework's matmuls write them
        dict(name="choose_step_2", kind="choose", batch=2, keys=8192, queries=1, heads=12, kv_heads=2, dim=128, type="f32",
             cache="bf16", page=16, first=1, last=2, count=64),
        # a serving batch over long documents
        dict(name="choose_decode_32", kind="choose", batch=32, keys=32768, queries=1, heads=32, kv_heads=8, dim=128, type="bf16",
             cache="bf16", page=64, first=1, last=2, count=64),
        # a question of some hundred tokens behind a document
        dict(name="choose_chunk", kind="choose", batch=1, queries=512, keys=16384, heads=32, kv_heads=4, dim=128, type="f16",
             cache="f16", page=32, first=1, last=4, count=32),
        # a few sequences: the smallest attention call
        dict(name="attend_step_4", kind="attend", batch=4, keys=16384, queries=1, heads=32, kv_heads=8, dim=128, type="f32",
             cache="f16", page=16, heads_first=False, count=64, lse=False),
        # the serving batch: an eighth of its keys
        dict(name="attend_decode_32", kind="attend", batch=32, keys=32768, queries=1, heads=32, kv_heads=8, dim=128, type="bf16",
             cache="bf16", page=64, heads_first=True, count=64, lse=False),
        # questions behind documents, each row with pages of its own
        dict(name="attend_chunk", kind="attend", batch=2, keys=8192, queries=256, heads=32, kv_heads=8, dim=128, type="bf16",
             cache="bf16", page=64, heads_first=True, count=16, lse=True),
        # a decode step's weights on top of the earlier ones
        dict(name="mass_decode_32", kind="mass", batch=32, keys=8192, queries=1, heads=32, kv_heads=8, dim=128, type="bf16",
             cache="bf16", page=64, heads_first=True, decay=0.99),
        # a whole prompt's weights
        dict(name="mass_prompt", kind="mass", batch=1, keys=4096, queries=4096, heads=32, kv_heads=8, dim=128, type="f16",
             cache="f16", page=64, heads_first=True, decay=0.0),
        # odd sizes, into pages of their own
        dict(name="evict_odd", kind="evict", batch=3, keys=5001, kv_heads=5, dim=80, cache="f16", page=48, heads_first=False,
             first=4, last=33, budget=1001, moved=True),
        # a serving batch whose documents shrink to a quarter in their own pages
        dict(name="evict_32", kind="evict", batch=32, keys=16384, kv_heads=8, dim=128, cache="bf16", page=64, heads_first=True,
             first=4, last=128, budget=4096, moved=False),
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(("bounds", "choose", "attend", "mass", "evict"))
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
    cache = rng.choice(("f16", "bf16"))
    c = dict(kind=kind, kv_heads=kv_heads, dim=rng.choice((64, 80, 96, 128, 128, 256)), cache=cache,
             page=rng.choice((16, 32, 48, 64, 128)), batch=_log(rng, 1, 24), keys=_log(rng, 100, 10000))
    if kind == "choose":
        c.update(heads=heads, type=rng.choice(("f32", cache)), queries=rng.choice((1, 1, 2, _log(rng, 1, 60))),
                 first=rng.choice((0, 1, 2)), last=rng.choice((1, 2, 4)))
        c["keys"] = max(c["keys"], 600)
        c["page"] = c["page"] if c["keys"] // 2 // c["page"] >= 12 else 16
        c["count"] = _log(rng, 8, c["keys"] // 2 // c["page"] - 2)  # (fewer than the shortest sequence's pages)
        c["batch"] = min(c["batch"], max(1, 64 // c["queries"]))
        return c
    c["heads_first"] = rng.random() < 0.5
    if kind == "bounds":
        c["new"] = rng.choice((0, 1, min(c["keys"], _log(rng, 1, 2000))))
    elif kind == "attend":
        c.update(heads=heads, type=rng.choice(("f32", cache)), queries=rng.choice((1, 1, 2, _log(rng, 1, 60))),
                 count=_log(rng, 4, 2000 // c["page"]), lse=rng.random() < 0.3)
        c["keys"] = max(c["keys"], 2 * c["queries"])
        c["batch"] = min(c["batch"], max(1, 64 // c["queries"]))
    elif kind == "mass":
        c.update(heads=heads, type=rng.choice(("f32", cache)), queries=rng.choice((1, 1, 2, 32, _log(rng, 1, 400))),
                 decay=rng.choice((0.0, 0.9, 1.0)))
        c["keys"] = max(c["keys"], c["queries"])
        c["batch"] = min(c["batch"], max(1, 400 // c["queries"]))
    else:
        c["budget"] = min(c["keys"], _log(rng, 64, 4096))
        c["first"] = rng.choice((0, 4, 16))
        c["last"] = rng.choice((0, 1, 32, 45))
        c["moved"] = rng.random() < 0.5
    return c


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """The sequences' rows and keys: the case's at most, keys spread down to half."""
    most = case.get("queries", 1)
    new = [most - (b * 7919) % (most // 2 + 1) for b in range(case["batch"])]
    return new, [max(n, case["keys"] - (b * 6007) % (case["keys"] // 2 + 1)) for b, n in enumerate(new)]


def _pool(case: dict, pages: int, gen) -> torch.Tensor:
    """Keys or values [pages, page, kv_heads, dim], with strides that go by heads_first; channels have
    sizes and offsets of their own, as those of a trained projection do."""
    first = case.get("heads_first", True)
    shape = (pages, case["kv_heads"], case["page"], case["dim"]) if first else (pages, case["page"], case["kv_heads"], case["dim"])
    channel = (1, case["kv_heads"], 1, case["dim"]) if first else (1, 1, case["kv_heads"], case["dim"])
    x = torch.randn(shape, generator=gen, device="cuda")
    x.mul_(0.5 + torch.rand(channel, generator=gen, device="cuda")).add_(0.5 * torch.randn(channel, generator=gen, device="cuda"))
    x = x.to(TYPES[case["cache"]])
    return x.transpose(1, 2) if first else x


def _limits(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Each row's sequence and the keys that it sees."""
    n_new = (s["offsets"][1:] - s["offsets"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n_new.numel(), device="cuda"), n_new, output_size=s["tokens"])
    at = torch.arange(s["tokens"], device="cuda") - s["offsets"][:-1].long()[seq]
    return seq, s["keys"].long()[seq] - n_new[seq] + at + 1


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s, c = {"case": case}, case
    kind, kv, dim, page = c["kind"], c["kv_heads"], c["dim"], c["page"]
    new, keys = _lengths(c)
    each = -(-max(keys) // page)
    total = each * c["batch"]
    moved = -(-c["budget"] // page) if c.get("moved") else 0
    order = torch.randperm(total + moved * c["batch"], generator=gen, device="cuda").to(torch.int32)
    s["pages"] = order[:total].reshape(c["batch"], each).contiguous()
    s["keys"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
    s["most_keys"], s["most_new"], s["n_pages"] = max(keys), max(new), order.numel()
    s["strides"] = (page * kv * dim, dim, page * dim) if c.get("heads_first", True) else (page * kv * dim, kv * dim, dim)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    s["tokens"], s["offsets"] = offsets[-1], torch.tensor(offsets, dtype=torch.int32, device="cuda")
    if kind != "choose":  # (which reads the pages' bounds alone)
        s["k_cache"] = _pool(c, order.numel(), gen)
    if kind in ("attend", "evict"):
        s["v_cache"] = _pool(c, order.numel(), gen)
    if "queries" in c:
        size = 0.5 + torch.rand((c["heads"], 1), generator=gen, device="cuda")
        s["q"] = (torch.randn((s["tokens"], c["heads"], dim), generator=gen, device="cuda") * size).to(TYPES[c["type"]])
        s["scale"] = 1.0 / math.sqrt(dim)
        s["workspace"] = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    if kind == "bounds":
        s["from"] = torch.tensor([max(0, k - c["new"]) for k in keys], dtype=torch.int32, device="cuda") if c["new"] else None
        s["bounds"] = torch.zeros((order.numel(), kv, 2, dim), dtype=TYPES[c["cache"]], device="cuda")
    elif kind == "choose":
        middle = torch.randn((order.numel(), kv, 1, dim), generator=gen, device="cuda") * 0.7
        reach = 1.5 + torch.rand((order.numel(), kv, 1, dim), generator=gen, device="cuda")
        s["bounds"] = torch.cat((middle - reach, middle + reach), 2).to(TYPES[c["cache"]])
        s["chosen"] = torch.empty((s["tokens"], kv, c["count"]), dtype=torch.int32, device="cuda")
    elif kind == "attend":
        # any pages, the row's last among them
        seq, sees = _limits(s)
        last = (sees - 1) // page
        score = torch.rand((s["tokens"], kv, each), generator=gen, device="cuda")
        at = torch.arange(each, device="cuda")
        score = torch.where(at > last[:, None, None], -1.0, torch.where(at == last[:, None, None], 2.0, score))
        best, which = score.topk(min(c["count"], each), -1)
        which = torch.where(best < 0, each, which).sort(-1).values
        chosen = torch.full((s["tokens"], kv, c["count"]), -1, dtype=torch.int32, device="cuda")
        chosen[..., : which.shape[-1]] = torch.where(which == each, -1, which).to(torch.int32)
        s["chosen"] = chosen
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((s["tokens"], c["heads"]), dtype=torch.float32, device="cuda") if c["lse"] else None
    else:
        width = max(keys)
        s["mass"] = torch.exp(1.5 * torch.randn((c["batch"], kv, width), generator=gen, device="cuda") - 4.0)
        if kind == "mass":
            s["lse"] = _plain_lse(s)
        else:
            s["mass_out"] = torch.zeros_like(s["mass"])
            s["kept"] = torch.empty((c["batch"], kv, c["budget"]), dtype=torch.int32, device="cuda")
            s["kept_lens"] = torch.empty(c["batch"], dtype=torch.int32, device="cuda")
            s["to_pages"] = order[total:].reshape(c["batch"], moved).contiguous() if moved else None
    return s


# ---------------------------------------------------------------- the framework's operators


def _run_own(s: dict):
    import dynalm_amd as dq

    c = s["case"]
    kind = c["kind"]
    stream = torch.cuda.current_stream().cuda_stream
    kinds = {torch.float32: dq.F32, torch.float16: dq.F16, torch.bfloat16: dq.BF16}
    k, v = s.get("k_cache"), s.get("v_cache")
    cache = dq.KvCache(k.data_ptr() if k is not None else None, v.data_ptr() if v is not None else None, kinds[TYPES[c["cache"]]],
                       c["kv_heads"], c["dim"], c["page"], s["n_pages"], *s["strides"])
    seqs = dq.Sequences(c["batch"], s["tokens"], s["offsets"].data_ptr() if s["most_new"] > 1 else None, s["most_new"],
                        s["pages"].data_ptr(), s["pages"].stride(0), s["keys"].data_ptr(), s["most_keys"])
    if kind == "bounds":
        dq.page_bounds(cache, seqs, s["from"], c["new"] or s["most_keys"], s["bounds"], stream)
        return s["bounds"]
    if kind == "evict":
        mass, out = s["mass"], s["mass_out"]
        strides = mass.stride()[:2]
        dq.kv_keep(seqs, c["kv_heads"], mass, *strides, c["first"], c["last"], c["budget"], s["kept"], s["kept_lens"], stream)
        to = s["to_pages"]
        dq.kv_compact(cache, seqs, s["kept"], c["budget"], to, to.stride(0) if to is not None else 0, mass, out, *strides, stream)
        return s["kept"], s["kept_lens"], k, v, out
    q = dq.Heads(s["q"].data_ptr(), kinds[s["q"].dtype], c["heads"], s["q"].stride(0), s["q"].stride(1))
    if kind == "choose":
        dq.choose_pages(cache, seqs, q, s["bounds"], c["first"], c["last"], c["count"], s["chosen"], s["workspace"], WORKSPACE_BYTES,
                        stream)
        return s["chosen"]
    if kind == "mass":
        dq.attention_mass(cache, seqs, q, s["lse"], s["scale"], c["decay"], s["mass"], *s["mass"].stride()[:2], s["workspace"],
                          WORKSPACE_BYTES, stream)
        return s["mass"]
    out = dq.Heads(s["out"].data_ptr(), kinds[s["out"].dtype], c["heads"], s["out"].stride(0), s["out"].stride(1))
    dq.page_attention(cache, seqs, q, out, s["lse"], s["chosen"], c["count"], s["scale"], s["workspace"], WORKSPACE_BYTES, stream)
    return (s["out"], s["lse"]) if c["lse"] else s["out"]


# ---------------------------------------------------------------- their plain form


def _by_sequence(s: dict, pool: torch.Tensor) -> torch.Tensor:
    """A sequence's places one after another: [batch, kv_heads, places, dim] in fp32."""
    return pool[s["pages"].long()].flatten(1, 2).permute(0, 2, 1, 3).float()


def _rows(s: dict, dtype=torch.float32):
    """q as [batch, kv, group, new, dim], with each row's token (0 where there is none) and whether there is one."""
    c = s["case"]
    step = torch.arange(s["most_new"], device="cuda")
    real = step[None, :] < (s["offsets"][1:] - s["offsets"][:-1])[:, None]
    at = torch.where(real, s["offsets"][:-1, None] + step, 0).long()
    q = s["q"].to(dtype)[at].unflatten(2, (c["kv_heads"], -1)).permute(0, 2, 3, 1, 4).contiguous()
    return q, at, real


def _scores(s: dict) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Scaled scores [batch, kv, group, new, places] with -inf where a row does not see a key."""
    q, at, real = _rows(s)
    b, kv, group, new, dim = q.shape
    k = _by_sequence(s, s["k_cache"]).transpose(2, 3).contiguous()
    scores = torch.matmul(q.reshape(b, kv, group * new, dim) * s["scale"], k).reshape(b, kv, group, new, -1)
    n_new = s["offsets"][1:] - s["offsets"][:-1]
    sees = (s["keys"] - n_new)[:, None] + torch.arange(new, device="cuda")[None, :] + 1
    sees = torch.where(real, sees, 0)
    hidden = torch.arange(k.shape[-1], device="cuda") >= sees[:, None, None, :, None]
    return scores.masked_fill_(hidden, -math.inf), at, real


def _plain_lse(s: dict) -> torch.Tensor:
    """log of the sum of exp of a row's scores, [tokens, heads], as the attention before it gives it."""
    scores, at, real = _scores(s)
    lse = torch.logsumexp(scores, -1).permute(0, 3, 1, 2).flatten(2)  # [batch, new, heads]
    return lse[real].contiguous()


def _plain_mass(s: dict):
    c, mass = s["case"], s["mass"]
    scores, at, real = _scores(s)
    lse = s["lse"][at].unflatten(2, (c["kv_heads"], -1)).permute(0, 2, 3, 1)[..., None]  # [batch, kv, group, new, 1]
    gained = torch.exp(scores - lse).sum((2, 3))[..., : mass.shape[2]]
    n_new = s["offsets"][1:] - s["offsets"][:-1]
    key = torch.arange(mass.shape[2], device="cuda")
    before = torch.where((key[None, :] < (s["keys"] - n_new)[:, None])[:, None], mass * c["decay"], 0.0)
    mass.copy_(torch.where((key[None, :] < s["keys"][:, None])[:, None], before + gained, mass))
    return mass


def _plain_bounds(s: dict):
    c, bounds, page = s["case"], s["bounds"], s["case"]["page"]
    start = s["from"] if s["from"] is not None else torch.zeros_like(s["keys"])
    most = min(s["pages"].shape[1], (c["new"] or s["most_keys"]) // page + 2)
    which = torch.div(start, page, rounding_mode="floor")[:, None] + torch.arange(most, device="cuda")   # [batch, most]
    written = which * page < s["keys"][:, None]
    at = s["pages"].long().gather(1, which.clamp(max=s["pages"].shape[1] - 1).long())
    keys = s["k_cache"][at].float()                                             # [batch, most, page, kv, dim]
    place = which[..., None] * page + torch.arange(page, device="cuda")
    hidden = (place >= s["keys"][:, None, None])[..., None, None]
    low = keys.masked_fill(hidden, math.inf).amin(2)
    high = keys.masked_fill(hidden, -math.inf).amax(2)
    bounds[at[written]] = torch.stack((low, high), 3)[written].to(bounds.dtype)
    return bounds


def _plain_choose(s: dict):
    c = s["case"]
    page, count = c["page"], c["count"]
    q, at, real = _rows(s, torch.float64)
    b, kv, group, new, dim = q.shape
    near = s["bounds"][s["pages"].long()].double().permute(0, 2, 3, 4, 1)      # [batch, kv, 2, dim, each]
    low, high = near[:, :, 0].contiguous(), near[:, :, 1].contiguous()
    rows = q.reshape(b, kv, group * new, dim)
    score = torch.matmul(rows.clamp(min=0), high) + torch.matmul(rows.clamp(max=0), low)
    score = score.reshape(b, kv, group, new, -1).amax(2).permute(0, 2, 1, 3)[real]   # [tokens, kv, each]
    seq, sees = _limits(s)
    visible = ((sees + page - 1) // page)[:, None, None]
    at = torch.arange(score.shape[-1], device="cuda")
    score = score.masked_fill((at < c["first"]) | (at >= visible - c["last"]), math.inf).masked_fill(at >= visible, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :count]
    best = torch.where(best < visible, best, score.shape[-1]).sort(-1).values
    chosen = s["chosen"].fill_(-1)
    chosen[..., : best.shape[-1]] = torch.where(best < score.shape[-1], best, -1).to(torch.int32)
    return chosen


def _plain_attend(s: dict):
    c = s["case"]
    page, kv, dim, group = c["page"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    seq, sees = _limits(s)
    chosen = s["chosen"].long()
    at = s["pages"].long()[seq[:, None, None], chosen.clamp(min=0)]             # [tokens, kv, count]
    head = torch.arange(kv, device="cuda")[None, :, None]
    k = s["k_cache"].permute(0, 2, 1, 3)[at, head].flatten(2, 3).float()        # [tokens, kv, count * page, dim]
    v = s["v_cache"].permute(0, 2, 1, 3)[at, head].flatten(2, 3).float()
    key = (chosen[..., None] * page + torch.arange(page, device="cuda")).flatten(2)
    seen = (key >= 0) & (key < sees[:, None, None])
    q = s["q"].float().unflatten(1, (kv, group)) * s["scale"]
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).masked_fill_(~seen[:, :, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    weights = torch.exp(scores - most)
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, torch.where(seen[..., None], v, 0.0))
    out = torch.where(total > 0, out / total, 0.0).flatten(1, 2).to(s["q"].dtype)
    return (out, (most + torch.log(total)).reshape(-1, c["heads"])) if c["lse"] else out


def _plain_evict(s: dict):
    c = s["case"]
    page, budget, mass = c["page"], c["budget"], s["mass"]
    place = torch.arange(mass.shape[2], device="cuda")
    lens = s["keys"].long()[:, None, None]
    rank = mass.masked_fill((place < c["first"]) | (place >= lens - c["last"]), math.inf).masked_fill(place >= lens, -math.inf)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.where(best < lens, best, mass.shape[2]).sort(-1).values
    real = kept < mass.shape[2]
    s["kept"].copy_(torch.where(real, kept, -1))
    s["kept_lens"].copy_(real[:, 0].sum(-1))
    to = (s["to_pages"] if s["to_pages"] is not None else s["pages"]).long()
    b = torch.arange(c["batch"], device="cuda")[:, None, None]
    h = torch.arange(c["kv_heads"], device="cuda")[None, :, None]
    i = torch.arange(budget, device="cuda").expand_as(kept)
    kept = torch.where(real, kept, 0)
    source = (s["pages"].long()[b, kept // page], kept % page, h.expand_as(kept))
    k, v, m = s["k_cache"][source], s["v_cache"][source], mass[b, h, kept]
    target = (to[b, i // page][real], (i % page)[real], h.expand_as(kept)[real])
    s["k_cache"][target] = k[real]
    s["v_cache"][target] = v[real]
    s["mass_out"][..., :budget] = torch.where(real, m, s["mass_out"][..., :budget])
    return s["kept"], s["kept_lens"], s["k_cache"], s["v_cache"], s["mass_out"]


_PLAIN = {"bounds": _plain_bounds, "choose": _plain_choose, "attend": _plain_attend, "mass": _plain_mass, "evict": _plain_evict}


def run(s: dict):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


# ---------------------------------------------------------------- the work and the values in 64 bits


def work(case: dict) -> dict:
    c = case
    kind, kv, dim, page = c["kind"], c["kv_heads"], c["dim"], c["page"]
    new, keys = _lengths(c)
    pages = [-(-k // page) for k in keys]
    if kind == "bounds":
        start = [max(0, k - c["new"]) // page if c["new"] else 0 for k in keys]
        read = sum(k - f * page for k, f in zip(keys, start)) * kv * dim
        return {"bytes": 2 * read + 4 * sum(p - f for p, f in zip(pages, start)) * kv * dim, "flops": 2 * read}
    if kind == "evict":
        stay = sum(min(k, c["budget"]) for k in keys) * kv
        return {"bytes": 4 * sum(keys) * kv + stay * (4 + 8 + 8 * dim), "flops": sum(keys) * kv}
    rows = sum(new) * c["heads"] * dim * BYTES[c["type"]]
    if kind == "choose":
        return {"bytes": rows + 4 * sum(pages) * kv * dim + 4 * sum(new) * kv * c["count"],
                "flops": 2 * dim * c["heads"] * sum(n * p for n, p in zip(new, pages))}
    if kind == "mass":
        seen = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(new, keys))
        return {"bytes": rows + 2 * sum(keys) * kv * dim + 8 * sum(keys) * kv, "flops": 2 * dim * c["heads"] * seen}
    # a sequence's rows together read none of its keys twice
    some = sum(min(n * min(c["count"], p) * page, k) for n, p, k in zip(new, pages, keys))
    seen = sum(n * min(c["count"] * page, k) for n, k in zip(new, keys))
    return {"bytes": 2 * rows + 4 * some * kv * dim + 4 * sum(new) * kv * c["count"], "flops": 4 * dim * c["heads"] * seen}


def _sequence(pool: torch.Tensor, pages: torch.Tensor, count: int) -> torch.Tensor:
    return pool[pages.long()].reshape(-1, *pool.shape[2:])[:count]


def exact(case: dict, seed: int):
    s, c = prepare(case, seed), case
    kind, kv, dim, page = c["kind"], c["kv_heads"], c["dim"], c["page"]
    new, keys = _lengths(c)
    if kind == "choose":
        return None  # whole numbers
    if kind == "bounds":
        out = s["bounds"].double()
        for b, k in enumerate(keys):
            x = _sequence(s["k_cache"], s["pages"][b], k).double()
            first = max(0, k - c["new"]) // page if c["new"] else 0
            whole = k // page
            if whole > first:
                y = x[first * page : whole * page].unflatten(0, (-1, page))
                out[s["pages"][b, first:whole].long()] = torch.stack((-(-y).max(1).values, -(-y).min(1).values), 2)
            if k % page:
                y = x[whole * page :]
                out[s["pages"][b, whole].long()] = torch.stack((-(-y).max(0).values, -(-y).min(0).values), 1)
        return out
    if kind == "evict":
        kc, vc, out = s["k_cache"].double(), s["v_cache"].double(), s["mass_out"].double()
        for b, k in enumerate(keys):
            ks, vs = _sequence(s["k_cache"], s["pages"][b], k), _sequence(s["v_cache"], s["pages"][b], k)
            to = s["to_pages"][b] if s["to_pages"] is not None else s["pages"][b]
            for h in range(kv):
                m = s["mass"][b, h, :k].double().clone()
                m[: c["first"]] = math.inf
                m[max(0, k - c["last"]) :] = math.inf
                # (largest first; of equal ones the lower place)
                order = torch.argsort(-m, stable=True)[: c["budget"]].sort().values
                i = torch.arange(order.numel(), device="cuda")
                at = to.long()[i // page]
                kc[at, i % page, h], vc[at, i % page, h] = ks[order, h].double(), vs[order, h].double()
                out[b, h, : order.numel()] = s["mass"][b, h, order].double()
        return None, None, kc, vc, out
    group = c["heads"] // kv
    start = 0
    if kind == "mass":
        out = s["mass"].double()
        for b, (n, k) in enumerate(zip(new, keys)):
            x = _sequence(s["k_cache"], s["pages"][b], k).double()
            seen = torch.arange(k, device="cuda")[None, :] <= (k - n + torch.arange(n, device="cuda"))[:, None]
            out[b, :, : k - n] *= c["decay"]
            out[b, :, k - n : k] = 0
            for h in range(c["heads"]):
                p = s["q"][start : start + n, h].double() @ x[:, h // group].t().contiguous() / math.sqrt(dim)
                out[b, h // group, :k] += torch.where(seen, torch.exp(p - s["lse"][start : start + n, h, None].double()), 0.0).sum(0)
            start += n
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], c["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, (n, k) in enumerate(zip(new, keys)):
        ks, vs = _sequence(s["k_cache"], s["pages"][b], k), _sequence(s["v_cache"], s["pages"][b], k)
        last = k - n + torch.arange(n, device="cuda")
        pages = s["chosen"][start : start + n].long()
        rows = slice(start, start + n)
        for h in range(kv):
            # a row's keys among all of the sequence's
            reads = torch.zeros((n, -(-k // page) + 1), dtype=torch.bool, device="cuda")
            reads.scatter_(1, torch.where(pages[:, h] < 0, reads.shape[1] - 1, pages[:, h]), True)
            reads = reads[:, :-1].repeat_interleave(page, 1)[:, :k] & (torch.arange(k, device="cuda") <= last[:, None])
            x, y = ks[:, h].double(), vs[:, h].double()
            for g in range(h * group, (h + 1) * group):
                p = (s["q"][rows, g].double() @ x.t().contiguous() / math.sqrt(dim)).masked_fill(~reads, -math.inf)
                lse[rows, g] = torch.logsumexp(p, -1)
                out[rows, g] = torch.softmax(p, -1) @ y
        start += n
    return (out, lse) if c["lse"] else out
