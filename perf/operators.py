"""The attention block's operators whose time is measured, each as a user's program calls it.

Between a decoder layer's matmuls an inference program normalizes and rotates the heads of its
queries and keys (`qk_norm_rope`), appends the new keys and values to a paged cache
(`kv_append`), and lets a batch of sequences attend to a prefix that all of them share (a
system prompt, a document) and to their own tokens after it (`shared_attention`). The listed
cases are decode steps and prompts of models with the head shapes of the benchmark's layers;
`draw` spreads tokens, heads, head sizes, types, pages and lengths over the same ranges.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
THETA = 500000.0
WORKSPACE_BYTES = 128 << 20

# kind "norm_rope": tokens of heads query heads and kv_heads key heads of dim values, type to
#   out; rot: rotated values of a head; halves: pairs (i, i + rot / 2), else (2i, 2i + 1); fused:
#   q and k are parts of one row of q, k and v, as a fused projection writes them.
# kind "append": tokens appended to a cache of type out with pages of `page` tokens; norm: k is
#   normalized on the way; heads_first: pages are [heads][tokens][dim], else [tokens][heads][dim].
# kind "attention": batch sequences of up to `queries` new tokens each, a shared prefix of
#   `prefix` keys and up to `own_keys` own ones (the new tokens among them).


def listed() -> list[dict]:
    return [
        # one token of one sequence: the smallest call, all latency
        dict(name="norm_rope_one_token", kind="norm_rope", tokens=1, heads=32, kv_heads=8, dim=128, rot=128, type="f32",
             out="f32", halves=True, fused=False),
        # a prompt's rows as a fused projection leaves them
        dict(name="norm_rope_prompt", kind="norm_rope", tokens=8192, heads=32, kv_heads=8, dim=128, rot=128, type="bf16",
             out="bf16", halves=True, fused=True),
        # an odd number of rows, half of each head rotated in neighbouring pairs
        dict(name="norm_rope_odd", kind="norm_rope", tokens=1023, heads=14, kv_heads=2, dim=96, rot=48, type="f32",
             out="f16", halves=False, fused=False),
        # one decode step of 64 sequences, k normalized and rotated on its way into the cache
        dict(name="append_decode_64", kind="append", tokens=64, kv_heads=8, dim=128, rot=128, type="f32", out="bf16",
             halves=True, norm=True, page=16, heads_first=False),
        # prompts of a batch
        dict(name="append_prompt", kind="append", tokens=16384, kv_heads=8, dim=128, rot=128, type="bf16", out="bf16",
             halves=True, norm=False, page=64, heads_first=True),
        # a few sequences at the start of their answers: the smallest attention call
        dict(name="attn_decode_4", kind="attention", batch=4, queries=1, heads=32, kv_heads=8, dim=128, prefix=1024,
             own_keys=64, type="f32", cache="f16", page=16, heads_first=False, lse=False),
        # a serving batch behind one system prompt
        dict(name="attn_decode_64", kind="attention", batch=64, queries=1, heads=32, kv_heads=8, dim=128, prefix=8192,
             own_keys=512, type="bf16", cache="bf16", page=64, heads_first=True, lse=False),
        # many questions on one long document
        dict(name="attn_decode_long", kind="attention", batch=128, queries=1, heads=32, kv_heads=4, dim=128, prefix=32768,
             own_keys=2048, type="bf16", cache="bf16", page=128, heads_first=True, lse=False),
        # fp32 rows, as this framework's matmuls write and read them, of a small model
        dict(name="attn_decode_f32", kind="attention", batch=32, queries=1, heads=12, kv_heads=2, dim=128, prefix=4096,
             own_keys=300, type="f32", cache="bf16", page=16, heads_first=False, lse=False),
        # questions of some hundred tokens each, prefilled behind the shared prompt
        dict(name="attn_prefill_shared", kind="attention", batch=8, queries=512, heads=32, kv_heads=8, dim=128, prefix=8192,
             own_keys=512, type="bf16", cache="bf16", page=64, heads_first=True, lse=False),
        # one prompt, nothing shared
        dict(name="attn_prompt_4096", kind="attention", batch=1, queries=4096, heads=32, kv_heads=8, dim=128, prefix=0,
             own_keys=4096, type="f16", cache="f16", page=64, heads_first=True, lse=False),
        # a few proposed tokens for each of seven sequences, odd sizes, pages that end inside tiles
        dict(name="attn_proposed_odd", kind="attention", batch=7, queries=5, heads=15, kv_heads=5, dim=80, prefix=1111,
             own_keys=201, type="f16", cache="f16", page=48, heads_first=False, lse=True),
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(("norm_rope", "append", "attention", "attention"))
    dim = rng.choice((64, 80, 96, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    rot = rng.choice((dim, dim, dim // 2))
    if kind == "norm_rope":
        return dict(kind=kind, tokens=_log(rng, 1, 8000), heads=kv_heads * rng.choice((1, 2, 4)), kv_heads=kv_heads, dim=dim, rot=rot,
                    type=rng.choice(("f32", "f16", "bf16")), out=rng.choice(("f32", "f16", "bf16")),
                    halves=rng.random() < 0.6, fused=rng.random() < 0.5)
    if kind == "append":
        return dict(kind=kind, tokens=_log(rng, 1, 16000), kv_heads=kv_heads, dim=dim, rot=rot,
                    type=rng.choice(("f32", "f16", "bf16")), out=rng.choice(("f16", "bf16")), halves=rng.random() < 0.6,
                    norm=rng.random() < 0.5, page=rng.choice((16, 32, 48, 64, 256)), heads_first=rng.random() < 0.5)
    heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
    cache = rng.choice(("f16", "bf16"))
    long = rng.random() < 0.4
    queries = _log(rng, 16, 512) if long else rng.choice((1, 1, 1, 2, 5))
    batch = _log(rng, 1, 6) if long else _log(rng, 2, 100)
    prefix = rng.choice((0, 1, 1)) * _log(rng, 100, 8000)
    return dict(kind=kind, batch=batch, queries=queries, heads=heads, kv_heads=kv_heads, dim=dim, prefix=prefix,
                own_keys=queries + _log(rng, 1, 1000), type=rng.choice(("f32", cache)), cache=cache,
                page=rng.choice((16, 32, 48, 64, 256)), heads_first=rng.random() < 0.5, lse=rng.random() < 0.3)


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """The sequences' new tokens and own keys: the case's at most, spread down to half."""
    new, keys = [], []
    for b in range(case["batch"]):
        n = case["queries"] - (b * 7919) % (case["queries"] // 2 + 1)
        new.append(n)
        keys.append(max(n, case["own_keys"] - (b * 6007) % (case["own_keys"] // 2 + 1)))
    return new, keys


def _rows(gen, tokens: int, heads: int, dim: int, type: str, width: int = 0, at: int = 0, base=None) -> torch.Tensor:
    # each head has its own size, as heads of a trained projection do
    size = 0.5 + torch.rand((heads, 1), generator=gen, device="cuda") * 1.5
    x = (torch.randn((tokens, heads, dim), generator=gen, device="cuda") * size).to(TYPES[type])
    if base is None:
        return x
    part = base[:, at : at + heads * dim].unflatten(1, (heads, dim))
    part.copy_(x)
    return part


def _rope_tables(case: dict, longest: int) -> tuple[torch.Tensor, torch.Tensor]:
    half = case["rot"] // 2
    angle = torch.arange(longest, device="cuda", dtype=torch.float64)[:, None] * THETA ** (
        -torch.arange(half, device="cuda", dtype=torch.float64) / half)[None, :]
    return angle.cos().float(), angle.sin().float()


def _cache(case: dict, pages: int, gen, type: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [pages, page, kv_heads, dim], with strides that go by heads_first."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"]) if case["heads_first"] else (
        pages, case["page"], case["kv_heads"], case["dim"])
    k = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(TYPES[type])
    v = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(TYPES[type])
    return (k.transpose(1, 2), v.transpose(1, 2)) if case["heads_first"] else (k, v)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    dim = case["dim"]
    if case["kind"] == "attention":
        new, keys = _lengths(case)
        page = case["page"]
        shared = -(-case["prefix"] // page)
        each = -(-max(keys) // page)
        total = shared + each * case["batch"]
        s["k_cache"], s["v_cache"] = _cache(case, total, gen, case["cache"])
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        s["prefix_pages"] = order[:shared].contiguous()
        s["pages"] = order[shared:].reshape(case["batch"], each).contiguous()
        s["keys"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
        offsets = [0]
        for n in new:
            offsets.append(offsets[-1] + n)
        s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        s["tokens"], s["most_new"], s["most_keys"] = offsets[-1], max(new), max(keys)
        s["q"] = _rows(gen, offsets[-1], case["heads"], dim, case["type"])
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((offsets[-1], case["heads"]), dtype=torch.float32, device="cuda") if case["lse"] else None
        s["scale"] = 1.0 / math.sqrt(dim)
        s["workspace"] = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    else:
        tokens = case["tokens"]
        longest = 2 * tokens + 1000
        s["cos"], s["sin"] = _rope_tables(case, longest)
        s["positions"] = torch.randint(0, longest, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
        s["k_weight"] = 1.0 + 0.2 * torch.randn(dim, generator=gen, device="cuda")
        if case["kind"] == "norm_rope":
            s["q_weight"] = 1.0 + 0.2 * torch.randn(dim, generator=gen, device="cuda")
            heads, kv = case["heads"], case["kv_heads"]
            base = torch.empty((tokens, (heads + 2 * kv) * dim), dtype=TYPES[case["type"]], device="cuda") if case["fused"] else None
            s["q"] = _rows(gen, tokens, heads, dim, case["type"], at=0, base=base)
            s["k"] = _rows(gen, tokens, kv, dim, case["type"], at=heads * dim, base=base)
            s["q_out"] = torch.empty((tokens, heads, dim), dtype=TYPES[case["out"]], device="cuda")
            s["k_out"] = torch.empty((tokens, kv, dim), dtype=TYPES[case["out"]], device="cuda")
        else:
            pages = -(-tokens * 5 // (4 * case["page"])) + 1
            s["k_cache"], s["v_cache"] = _cache(case, pages, gen, case["out"])
            s["k"] = _rows(gen, tokens, case["kv_heads"], dim, case["type"])
            s["v"] = _rows(gen, tokens, case["kv_heads"], dim, case["type"])
            # a prompt fills its pages in order, the pages lie anywhere
            order = torch.randperm(pages, generator=gen, device="cuda")
            places = (order[:, None] * case["page"] + torch.arange(case["page"], device="cuda")[None, :]).reshape(-1)
            s["slots"] = places[:tokens].to(torch.int64).contiguous()
    return s


# ---------------------------------------------------------------- the framework's operators


def _heads(dq, x: torch.Tensor):
    kinds = {torch.float32: dq.F32, torch.float16: dq.F16, torch.bfloat16: dq.BF16}
    return dq.Heads(x.data_ptr(), kinds[x.dtype], x.shape[1], x.stride(0), x.stride(1))


def _rope(dq, s: dict):
    c = s["case"]
    return dq.Rope(s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], c["rot"],
                   dq.ROPE_HALVES if c["halves"] else dq.ROPE_PAIRS)


def _kv(dq, s: dict):
    k, v = s["k_cache"], s["v_cache"]
    kinds = {torch.float16: dq.F16, torch.bfloat16: dq.BF16}
    return dq.KvCache(k.data_ptr(), v.data_ptr(), kinds[k.dtype], k.shape[2], k.shape[3], k.shape[1], k.shape[0], k.stride(0),
                      k.stride(1), k.stride(2))


def _run_own(s: dict):
    import dynalm_amd as dq

    c = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] == "norm_rope":
        dq.qk_norm_rope(c["tokens"], c["dim"], _heads(dq, s["q"]), _heads(dq, s["q_out"]), s["q_weight"], _heads(dq, s["k"]),
                        _heads(dq, s["k_out"]), s["k_weight"], EPS, _rope(dq, s), s["positions"], stream)
        return s["q_out"], s["k_out"]
    if c["kind"] == "append":
        dq.kv_append(_kv(dq, s), c["tokens"], _heads(dq, s["k"]), _heads(dq, s["v"]), s["slots"], s["k_weight"] if c["norm"] else None,
                     EPS, _rope(dq, s), s["positions"], stream)
        return s["k_cache"], s["v_cache"]
    dq.shared_attention(_kv(dq, s), _heads(dq, s["q"]), _heads(dq, s["out"]), s["lse"], s["tokens"], c["batch"], s["offsets"],
                        s["most_new"], s["prefix_pages"] if c["prefix"] else None, c["prefix"], s["pages"], s["pages"].stride(0), s["keys"],
                        s["most_keys"], s["scale"], s["workspace"], WORKSPACE_BYTES, stream)
    return (s["out"], s["lse"]) if c["lse"] else s["out"]


# ---------------------------------------------------------------- their plain form


def _plain_norm_rope(x, weight, cos, sin, rot: int, halves: bool):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    r = x[..., :rot]
    a, b = (r[..., : rot // 2], r[..., rot // 2 :]) if halves else (r[..., 0::2], r[..., 1::2])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.cat((ra, rb), -1) if halves else torch.stack((ra, rb), -1).flatten(-2)
    return torch.cat((r, x[..., rot:]), -1)


def _plain_attention(s: dict):
    c = s["case"]
    batch, heads, kv, dim, prefix = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["prefix"]
    group, new, keys = heads // kv, s["most_new"], s["most_keys"]
    dev = s["q"].device
    n_new = s["offsets"][1:] - s["offsets"][:-1]
    step = torch.arange(new, device=dev)
    real = step[None, :] < n_new[:, None]                                    # [batch, new]
    at = torch.where(real, s["offsets"][:-1, None] + step, 0).long()
    # queries as [batch, kv, group * new, dim]
    q = s["q"].float()[at].reshape(batch, new, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * new, dim) * s["scale"]
    own_k = s["k_cache"][s["pages"].long()].flatten(1, 2)[:, :keys].float().permute(0, 2, 1, 3).contiguous()
    own_v = s["v_cache"][s["pages"].long()].flatten(1, 2)[:, :keys].float().permute(0, 2, 1, 3).contiguous()
    key = torch.arange(keys, device=dev)
    own_v = torch.where((key[None, :] < s["keys"][:, None])[:, None, :, None], own_v, 0.0)
    sees = key[None, None, :] <= (s["keys"] - n_new)[:, None, None] + step[None, :, None]
    sees = (sees & real[:, :, None])[:, None, None].expand(batch, 1, group, new, keys).reshape(batch, 1, group * new, keys)
    scores = torch.matmul(q, own_k.transpose(2, 3).contiguous()).masked_fill_(~sees, -math.inf)
    most = scores.amax(-1, keepdim=True)
    if prefix:
        first_k = s["k_cache"][s["prefix_pages"].long()].flatten(0, 1)[:prefix].float().permute(1, 2, 0).contiguous()
        first_v = s["v_cache"][s["prefix_pages"].long()].flatten(0, 1)[:prefix].float().permute(1, 0, 2).contiguous()
        qp = q.transpose(0, 1).reshape(kv, batch * group * new, dim)
        first = torch.matmul(qp, first_k).reshape(kv, batch, group * new, prefix).transpose(0, 1)
        most = torch.maximum(most, first.amax(-1, keepdim=True))
    most = torch.where(most == -math.inf, 0.0, most)
    scores = torch.exp(scores - most)
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores, own_v)
    if prefix:
        first = torch.exp(first - most)
        total = total + first.sum(-1, keepdim=True)
        out = out + torch.matmul(first.transpose(0, 1).reshape(kv, batch * group * new, prefix), first_v).reshape(
            kv, batch, group * new, dim).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (most + torch.log(total)).reshape(batch, kv, group, new).permute(0, 3, 1, 2).reshape(batch, new, heads)[real]
    out = out.reshape(batch, kv, group, new, dim).permute(0, 3, 1, 2, 4).reshape(batch, new, heads, dim)[real]
    out = out.to(s["q"].dtype)
    return (out, lse) if c["lse"] else out


def _run_plain(s: dict):
    c = s["case"]
    if c["kind"] == "attention":
        return _plain_attention(s)
    cos, sin = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]
    if c["kind"] == "norm_rope":
        return (_plain_norm_rope(s["q"], s["q_weight"], cos, sin, c["rot"], c["halves"]).to(TYPES[c["out"]]),
                _plain_norm_rope(s["k"], s["k_weight"], cos, sin, c["rot"], c["halves"]).to(TYPES[c["out"]]))
    k = _plain_norm_rope(s["k"], s["k_weight"] if c["norm"] else None, cos, sin, c["rot"], c["halves"])
    page, place = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k_cache"][page, place] = k.to(TYPES[c["out"]])
    s["v_cache"][page, place] = s["v"].float().to(TYPES[c["out"]])
    return s["k_cache"], s["v_cache"]


def run(s: dict):
    return _run_own(s) if own else _run_plain(s)


# ---------------------------------------------------------------- the work and the values in 64 bits


def work(case: dict) -> dict:
    dim, kv = case["dim"], case["kv_heads"]
    if case["kind"] == "attention":
        new, keys = _lengths(case)
        q_bytes = 2 * sum(new) * case["heads"] * dim * BYTES[case["type"]]
        kv_bytes = 2 * (case["prefix"] + sum(keys)) * kv * dim * 2
        seen = sum(n * (case["prefix"] + k - n) + n * (n + 1) // 2 for n, k in zip(new, keys))
        return {"bytes": q_bytes + kv_bytes + (sum(new) * case["heads"] * 4 if case["lse"] else 0),
                "flops": 4 * dim * case["heads"] * seen}
    values = case["tokens"] * dim * (case["heads"] + kv if case["kind"] == "norm_rope" else 2 * kv)
    table = case["tokens"] * (case["rot"] * 4 + 4)
    return {"bytes": values * (BYTES[case["type"]] + BYTES[case["out"]]) + table, "flops": 6 * values}


def _exact_turn(x, weight, cos, sin, positions, rot: int, halves: bool):
    """Norm as a division by the root, rotation as a product of complex numbers."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + EPS) * weight.double()
    turn = torch.complex(cos[positions.long()].double(), sin[positions.long()].double())[:, None, :]
    y = x.clone()
    if halves:
        z = torch.complex(x[..., : rot // 2].contiguous(), x[..., rot // 2 : rot].contiguous()) * turn
        y[..., : rot // 2], y[..., rot // 2 : rot] = z.real, z.imag
    else:
        z = torch.view_as_complex(x[..., :rot].unflatten(-1, (rot // 2, 2)).contiguous()) * turn
        y[..., :rot] = torch.view_as_real(z).flatten(-2)
    return y


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "norm_rope":
        return tuple(_exact_turn(s[n], s[n + "_weight"], s["cos"], s["sin"], s["positions"], c["rot"], c["halves"]) for n in ("q", "k"))
    if c["kind"] == "append":
        k = _exact_turn(s["k"], s["k_weight"] if c["norm"] else None, s["cos"], s["sin"], s["positions"], c["rot"], c["halves"])
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        page, place = torch.div(s["slots"], c["page"], rounding_mode="floor"), torch.remainder(s["slots"], c["page"])
        kc.index_put_((page, place), k)
        vc.index_put_((page, place), s["v"].double())
        return kc, vc
    new, keys = _lengths(c)
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros((s["tokens"], c["heads"], c["dim"]), dtype=torch.float64, device="cuda")
    lse = torch.full((s["tokens"], c["heads"]), -math.inf, dtype=torch.float64, device="cuda")

    def gather(pool, pages, count):
        return pool[pages.long()].reshape(-1, c["kv_heads"], c["dim"])[:count]

    start = 0
    for b, (n, k) in enumerate(zip(new, keys)):
        ks = torch.cat([gather(s["k_cache"], s["prefix_pages"], c["prefix"]), gather(s["k_cache"], s["pages"][b], k)]).double()
        vs = torch.cat([gather(s["v_cache"], s["prefix_pages"], c["prefix"]), gather(s["v_cache"], s["pages"][b], k)]).double()
        last = c["prefix"] + k - n + torch.arange(n, device="cuda")
        hidden = torch.arange(c["prefix"] + k, device="cuda")[None, :] > last[:, None]
        for h in range(c["heads"]):
            g = h // group
            p = (s["q"][start : start + n, h].double() @ ks[:, g].t().contiguous()) / math.sqrt(c["dim"])
            p[hidden] = -math.inf
            z = torch.logsumexp(p, -1)
            out[start : start + n, h] = torch.exp(p - z[:, None]) @ vs[:, g]
            lse[start : start + n, h] = z
        start += n
    return (out, lse) if c["lse"] else out
