"""The attention block's kernels: head norms and rotation, the append to a paged cache and
attention over a shared prefix, against their formulas in 64 bits."""
from __future__ import annotations

import math

import pytest

import dynalm_amd as dq

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import blocktest as B  # noqa: E402


def stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def rows(gen, tokens, heads, dim, type, odd=False, fused=0):
    """[tokens, heads, dim] on the GPU: contiguous, starting at an odd value, or part of wider rows."""
    x = torch.randn((tokens, heads, dim), generator=gen)
    t = B.TYPES[type]
    if fused:
        wide = torch.zeros((tokens, heads * dim + fused), dtype=t, device="cuda")
        y = wide[:, fused // 2 : fused // 2 + heads * dim].unflatten(1, (heads, dim))
    elif odd:
        y = torch.zeros(tokens * heads * dim + 1, dtype=t, device="cuda")[1:].view(tokens, heads, dim)
    else:
        y = torch.empty((tokens, heads, dim), dtype=t, device="cuda")
    y.copy_(x)
    return y


NORM_ROPE = [
    # tokens, q heads, k heads, dim, rot, halves, norm, in, out, odd, fused
    (1, 32, 8, 128, 128, True, True, "f32", "f32", False, 0),
    (1, 1, 1, 8, 2, False, True, "f32", "bf16", False, 0),
    (5, 4, 2, 64, 64, False, True, "f16", "f16", False, 0),
    (7, 3, 1, 80, 40, True, True, "bf16", "bf16", False, 0),
    (33, 14, 2, 96, 48, False, True, "f32", "f16", False, 16),
    (9, 5, 5, 72, 10, True, True, "f32", "f32", True, 0),
    (9, 5, 5, 72, 10, False, True, "bf16", "f32", True, 0),
    (3, 2, 0, 256, 256, True, True, "f32", "f32", False, 8),
    (3, 2, 1, 256, 64, False, False, "f16", "bf16", False, 3),
    (300, 2, 2, 200, 200, True, True, "bf16", "f16", False, 24),
    (6, 2, 2, 128, 0, True, True, "f32", "f32", False, 0),
    (6, 2, 2, 128, 0, True, False, "f32", "bf16", False, 0),
    (1027, 16, 4, 128, 128, True, True, "bf16", "bf16", False, 1024),
    # two heads a lane group (an odd number of heads among them), and outputs past 32 MB
    (2500, 13, 3, 64, 32, True, True, "f32", "bf16", False, 8),
    (7001, 5, 1, 72, 64, False, True, "f16", "f16", False, 0),
    (9000, 13, 2, 128, 128, True, True, "bf16", "bf16", False, 256),
    (2300, 13, 2, 256, 128, False, True, "f32", "f32", False, 0),
]


@pytest.mark.parametrize("tokens,hq,hk,dim,rot,halves,norm,ti,to,odd,fused", NORM_ROPE)
def test_norm_rope(cuda, tokens, hq, hk, dim, rot, halves, norm, ti, to, odd, fused):
    gen = torch.Generator().manual_seed(tokens * 1000 + dim)
    tables = B.rope_table(500, rot) if rot else None
    pos = torch.randint(0, 500, (tokens,), generator=gen, dtype=torch.int32)
    if tokens > 4:
        pos[1], pos[3] = -1, 500  # outside the tables
    sides = [(hq, 1.0), (hk, 3.0)] if hk else [(hq, 1.0)]
    x = [rows(gen, tokens, h, dim, ti, odd, fused) for h, _ in sides]
    w = [(1 + 0.3 * torch.randn(dim, generator=gen)) if norm else None for _ in sides]
    out = [torch.full((tokens, h, dim + 8), 77.0, dtype=B.TYPES[to], device="cuda")[:, :, :dim] for h, _ in sides]
    td = [t.cuda() for t in tables] if tables else None
    rope = dq.Rope(td[0].data_ptr(), td[1].data_ptr(), 500, rot, dq.ROPE_HALVES if halves else dq.ROPE_PAIRS) if rot else None
    wd = [t.cuda() if t is not None else None for t in w] + [None]
    dq.qk_norm_rope(tokens, dim, B.heads(x[0]), B.heads(out[0]), wd[0], B.heads(x[1]) if hk else None,
                    B.heads(out[1]) if hk else None, wd[1], 1e-6, rope, pos.cuda() if rot else None, stream())
    for xs, ws, o in zip(x, w, out):
        want, bound = B.norm_rope(xs.cpu(), ws, 1e-6, tables, pos, rot, halves)
        B.close(o, want, bound, to)
        assert torch.all(o.as_strided((tokens, o.shape[1], 8), o.stride(), dim) == 77.0)  # nothing past a head


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,rot,halves", [(128, 128, True), (128, 64, False), (40, 6, True)])
def test_norm_rope_in_place_gives_the_same_bits(cuda, type, dim, rot, halves):
    gen = torch.Generator().manual_seed(dim)
    q, k = rows(gen, 21, 6, dim, type), rows(gen, 21, 2, dim, type)
    td = [t.cuda() for t in B.rope_table(64, rot)]
    pos = torch.arange(21, dtype=torch.int32, device="cuda")
    w = torch.rand(dim, generator=gen).cuda()
    rope = dq.Rope(td[0].data_ptr(), td[1].data_ptr(), 64, rot, dq.ROPE_HALVES if halves else dq.ROPE_PAIRS)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    dq.qk_norm_rope(21, dim, B.heads(q), B.heads(qo), w, B.heads(k), B.heads(ko), w, 1e-5, rope, pos, stream())
    dq.qk_norm_rope(21, dim, B.heads(q), B.heads(q), w, B.heads(k), B.heads(k), w, 1e-5, rope, pos, stream())
    assert torch.equal(q, qo) and torch.equal(k, ko)


def test_norm_of_zeros_and_large_rows(cuda):
    x = torch.zeros((3, 1, 64), device="cuda")
    x[1] = 1e15
    x[2, 0, 0] = math.inf
    w = torch.ones(64, device="cuda")
    out = torch.empty_like(x)
    dq.qk_norm_rope(3, 64, B.heads(x), B.heads(out), w, eps=1e-6, stream=stream())
    want, bound = B.norm_rope(x.cpu(), w.cpu(), 1e-6, None, None, 0, True)
    B.close(out[:2], want[:2], bound[:2], "f32")
    assert torch.isnan(out[2, 0, 0]) and torch.all(out[2, 0, 1:] == 0)


APPEND = [
    # tokens, kv heads, dim, rot, halves, norm, in, cache, page, heads first, odd
    (1, 8, 128, 128, True, True, "f32", "bf16", 16, False, False),
    (1, 1, 8, 0, True, False, "f32", "f16", 16, False, False),
    (64, 8, 128, 128, True, True, "f32", "bf16", 16, True, False),
    (77, 5, 80, 40, False, True, "f16", "f16", 48, False, False),
    (300, 2, 256, 256, True, False, "bf16", "bf16", 32, True, False),
    (45, 3, 72, 8, False, True, "f32", "f16", 16, True, True),
    (45, 3, 72, 72, True, False, "bf16", "f16", 80, False, True),
    (513, 4, 64, 64, False, False, "f16", "bf16", 256, True, False),
    (19, 2, 200, 0, True, True, "f32", "f16", 16, False, False),
    (6000, 3, 96, 48, False, True, "bf16", "bf16", 48, True, False),
]


@pytest.mark.parametrize("tokens,hk,dim,rot,halves,norm,ti,tc,page,heads_first,odd", APPEND)
def test_append(cuda, tokens, hk, dim, rot, halves, norm, ti, tc, page, heads_first, odd):
    gen = torch.Generator().manual_seed(tokens * 100 + dim)
    pages = -(-tokens // page) + 2
    shape = (pages, hk, page, dim) if heads_first else (pages, page, hk, dim)
    pools = [torch.randn(shape, generator=gen).to(B.TYPES[tc]).cuda() for _ in range(2)]
    kc, vc = (p.transpose(1, 2) if heads_first else p for p in pools)
    before = [kc.cpu().clone(), vc.cpu().clone()]
    k, v = rows(gen, tokens, hk, dim, ti, odd), rows(gen, tokens, hk, dim, ti, odd)
    slots = torch.randperm(pages * page, generator=gen)[:tokens].to(torch.int64)
    if tokens > 4:
        slots[0], slots[2], slots[4] = -1, pages * page, -(2**40)  # left out
    tables = B.rope_table(300, rot) if rot else None
    pos = torch.randint(0, 300, (tokens,), generator=gen, dtype=torch.int32)
    if tokens > 4:
        pos[3] = 300
    td = [t.cuda() for t in tables] if rot else None
    rope = dq.Rope(td[0].data_ptr(), td[1].data_ptr(), 300, rot, dq.ROPE_HALVES if halves else dq.ROPE_PAIRS) if rot else None
    w = 1 + 0.3 * torch.randn(dim, generator=gen) if norm else None
    dq.kv_append(B.kv_cache(kc, vc), tokens, B.heads(k), B.heads(v), slots.cuda(), w.cuda() if norm else None, 1e-5, rope,
                 pos.cuda() if rot else None, stream())
    want_k, bound = B.norm_rope(k.cpu(), w, 1e-5, tables, pos, rot, halves)
    kept = torch.ones(pages * page, dtype=torch.bool)
    inside = (slots >= 0) & (slots < pages * page)
    at = slots[inside]
    kept[at] = False
    B.close(kc.cpu()[at // page, at % page], want_k[inside], bound[inside], tc)
    assert torch.equal(vc.cpu()[at // page, at % page], v.cpu()[inside].to(B.TYPES[tc]))
    for new, old in zip((kc.cpu(), vc.cpu()), before):
        assert torch.equal(new.reshape(pages * page, hk, dim)[kept], old.reshape(pages * page, hk, dim)[kept])


# ------------------------------------------------------------------ attention


def build(seed, new, lens, prefix, hq, hk, dim, type, cache, page, heads_first=False, odd=False, tail=0, spread=1.0, fused=0):
    """A call's tensors: places and page numbers that no row reads hold NaN and numbers outside the cache."""
    gen = torch.Generator().manual_seed(seed)
    most = max(lens + [0])
    shared, each = -(-prefix // page), -(-most // page)
    total = shared + each * len(new) + 1
    shape = (total, hk, page, dim) if heads_first else (total, page, hk, dim)
    kc, vc = (torch.full(shape, math.nan, dtype=B.TYPES[cache]) for _ in range(2))
    k4, v4 = (p.transpose(1, 2) if heads_first else p for p in (kc, vc))
    order = torch.randperm(total - 1, generator=gen).to(torch.int32)
    prefix_pages = order[:shared].clone()
    table = torch.full((len(new), each + 2), 2**31 - 1, dtype=torch.int32)
    first = [torch.randn((prefix, hk, dim), generator=gen).to(B.TYPES[cache]) for _ in range(2)]
    for j in range(prefix):
        for pool, x in zip((k4, v4), first):
            pool[int(prefix_pages[j // page]), j % page] = x[j]
    ks, vs = [], []
    for b, n in enumerate(lens):
        mine = order[shared + b * each : shared + b * each + -(-n // page)]
        table[b, : len(mine)] = mine
        own = [torch.randn((n, hk, dim), generator=gen).to(B.TYPES[cache]) for _ in range(2)]
        for j in range(n):
            for pool, x in zip((k4, v4), own):
                pool[int(mine[j // page]), j % page] = x[j]
        ks.append(torch.cat([first[0], own[0]]))
        vs.append(torch.cat([first[1], own[1]]))
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    tokens = offsets[-1] + tail
    q = rows(gen, tokens, hq, dim, type, odd, fused)
    q.mul_(spread)
    return dict(new=new, lens=lens, prefix=prefix, tokens=tokens, q=q, ks=ks, vs=vs, kc=k4.cuda() if not heads_first else kc.cuda().transpose(1, 2),
                vc=v4.cuda() if not heads_first else vc.cuda().transpose(1, 2), prefix_pages=prefix_pages.cuda(), table=table.cuda(),
                offsets=torch.tensor(offsets, dtype=torch.int32).cuda(), lens_d=torch.tensor(lens, dtype=torch.int32).cuda(),
                type=type, cache=cache, scale=1.0 / math.sqrt(dim), most=most, max_q=max(new + [1]))


def call(c, out=None, lse=None, workspace=None, no_offsets=False, max_len=None, max_q=None):
    out = torch.full_like(c["q"], 55.0) if out is None else out
    cache, q, o = B.kv_cache(c["kc"], c["vc"]), B.heads(c["q"]), B.heads(out)
    max_len = c["most"] if max_len is None else max_len
    max_q = c["max_q"] if max_q is None else max_q
    need = dq.shared_attention_workspace(cache, q, o, c["tokens"], len(c["new"]), max_q, c["prefix"], c["table"].stride(0),
                                         max_len, c["scale"])
    assert 0 <= need <= dq.ATTENTION_WORKSPACE_BYTES
    if workspace is None:
        workspace = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN, and beyond it a guard
        guard = workspace[need:]
    else:
        guard = None
    dq.shared_attention(cache, q, o, lse, c["tokens"], len(c["new"]), None if no_offsets else c["offsets"], max_q,
                        c["prefix_pages"] if c["prefix"] else None, c["prefix"], c["table"], c["table"].stride(0), c["lens_d"],
                        max_len, c["scale"], workspace, need, stream())
    if guard is not None:
        assert torch.all(guard == 0xFF)
    return out


def check(c, **kw):
    lse = torch.full((c["tokens"], c["q"].shape[1]), 33.0, device="cuda")
    out = call(c, lse=lse, **kw)
    n = sum(c["new"])
    want, want_lse, bound, lse_bound = B.attention(c["q"].cpu()[:n], c["ks"], c["vs"], c["new"], c["lens"], c["prefix"], c["scale"],
                                                   c["type"], c["cache"])
    B.close(out[:n], want, bound, c["type"])
    assert torch.all(out[n:] == 55.0) and torch.all(lse[n:] == 33.0)  # rows of no sequence
    B.close(lse[:n], want_lse, lse_bound, "f32")
    return out


KINDS = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]

SHAPES = [
    # new tokens, own lens, prefix, q heads, kv heads, dim, page, heads first
    pytest.param([1], [1], 0, 1, 1, 8, 16, False, id="one key"),
    pytest.param([1], [0], 0, 2, 1, 64, 16, False, id="no key"),
    pytest.param([1, 1, 1], [0, 5, 0], 17, 4, 2, 64, 16, True, id="prefix alone"),
    pytest.param([1, 1], [0, 40], 0, 4, 4, 128, 32, False, id="an empty row beside one"),
    pytest.param([1] * 5, [1, 15, 16, 17, 130], 33, 8, 2, 128, 16, True, id="decode"),
    pytest.param([1] * 19, [7 + 3 * i for i in range(19)], 300, 8, 1, 80, 48, False, id="decode, odd head size"),
    pytest.param([1] * 3, [600, 1, 259], 1500, 17, 1, 64, 64, True, id="17 heads a kv head"),
    pytest.param([1] * 2, [65, 64], 63, 6, 6, 256, 16, False, id="one head each"),
    pytest.param([1] * 40, [33] * 40, 129, 4, 2, 96, 32, True, id="many rows on a short prefix"),
    pytest.param([3, 0, 5, 1], [3, 9, 5, 77], 40, 6, 2, 72, 16, False, id="proposed tokens"),
    pytest.param([4, 6], [2, 3], 11, 2, 1, 40, 16, False, id="rows before the first key"),
    pytest.param([4, 6], [2, 3], 0, 2, 1, 128, 16, False, id="rows that see nothing"),
    pytest.param([70, 33], [70, 200], 50, 4, 2, 128, 16, True, id="prompts behind a prefix"),
    pytest.param([131], [131], 0, 3, 1, 200, 32, False, id="one prompt"),
    pytest.param([1], [77], 1300, 8, 2, 128, 16, False, id="one sequence behind a prefix"),
    pytest.param([3], [3], 1023, 15, 3, 96, 48, False, id="one sequence, no own keys before"),
    pytest.param([40], [300], 900, 4, 2, 256, 32, True, id="one prompt behind a prefix"),
    pytest.param([6, 2, 5], [700, 2, 300], 260, 10, 2, 128, 64, True, id="own keys in several ranges"),
    pytest.param([i % 3 for i in range(150)], [i % 3 + i % 40 for i in range(150)], 35, 2, 1, 64, 16, False, id="150 sequences"),
    pytest.param([33, 40], [90, 70], 140, 4, 2, 192, 16, True, id="heads of 192"),
    pytest.param([33, 40], [90, 70], 140, 4, 2, 160, 32, False, id="heads of 160"),
    pytest.param([33, 40], [90, 170], 140, 8, 2, 96, 16, True, id="prompts in heads of 96"),
    pytest.param([64, 1, 17], [64, 500, 17], 100, 8, 8, 64, 64, True, id="prompts and a decode step"),
]


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,lens,prefix,hq,hk,dim,page,heads_first", SHAPES)
def test_attention(cuda, new, lens, prefix, hq, hk, dim, page, heads_first, type, cache):
    check(build(dim + prefix, new, lens, prefix, hq, hk, dim, type, cache, page, heads_first))


@pytest.mark.parametrize("type,cache", KINDS)
def test_attention_rows_of_other_strides(cuda, type, cache):
    for kw in ({"odd": True}, {"fused": 24}, {"tail": 5}):
        check(build(3, [1, 2, 4], [30, 2, 50], 70, 4, 2, 64, type, cache, 16, **kw))
    c = build(3, [1, 2, 4], [30, 2, 50], 70, 4, 2, 64, type, cache, 16)
    wide = torch.full((4, c["tokens"], 80), 55.0, dtype=c["q"].dtype, device="cuda")
    check(c, out=wide.transpose(0, 1)[:, :, 3:67])  # [heads][tokens], heads at odd values
    assert torch.all(wide[:, :, :3] == 55.0) and torch.all(wide[:, :, 67:] == 55.0)


@pytest.mark.parametrize("type,cache", KINDS)
def test_attention_peaked_scores(cuda, type, cache):
    """Scores far apart: one key takes nearly all, the running maximum moves often."""
    check(build(5, [1, 9], [200, 140], 90, 4, 2, 128, type, cache, 16, spread=30.0))


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,lens,prefix", [([3], [40], 20), ([90], [90], 0), ([40, 50], [70, 50], 64)])
def test_nan_in_masked_places(cuda, type, cache, new, lens, prefix):
    """A key and value that only the last row sees are infinite or NaN: the other rows do not change."""
    c = build(7, new, lens, prefix, 4, 2, 64, type, cache, 16)
    clean = call(c)
    page = c["kc"].shape[1]
    at = int(c["table"][0, (lens[0] - 1) // page]), (lens[0] - 1) % page
    for bad in (math.nan, math.inf, -math.inf):
        c["kc"][at], c["vc"][at] = bad, bad
        out = call(c)
        last = new[0] - 1
        seen = torch.ones(c["tokens"], dtype=torch.bool)
        seen[last] = False
        assert torch.equal(out[seen.cuda()], clean[seen.cuda()])
        assert torch.isnan(out[last]).any()


def test_attention_page_numbers_outside_the_cache(cuda):
    c = build(11, [1, 1, 1], [40, 40, 40], 20, 4, 2, 64, "f32", "f16", 16)
    clean = call(c)
    c["table"][1, 1] = -1
    out = call(c)
    assert torch.isnan(out[1]).all() and torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
    c["table"][1, 1] = c["kc"].shape[0]
    assert torch.isnan(call(c)[1]).all()
    c["prefix_pages"][1] = 2**31 - 1
    assert torch.isnan(call(c)).all()


def test_attention_lengths_beyond_the_bounds_are_cut(cuda):
    """Lengths over max_len count as max_len, negative ones as none."""
    c = build(13, [1, 1], [48, 48], 20, 4, 2, 64, "f32", "f16", 16)
    clean = call(c)
    c["lens_d"].copy_(torch.tensor([1 << 30, -5], dtype=torch.int32))
    out = call(c)
    assert torch.equal(out[0], clean[0])
    short = build(13, [1, 1], [48, 48], 20, 4, 2, 64, "f32", "f16", 16)
    short["lens_d"][1] = 0
    assert torch.equal(call(short)[1], out[1])


@pytest.mark.parametrize("type,cache", KINDS)
def test_attention_bounds_above_the_lengths(cuda, type, cache):
    """max_len and max_q may be above what the sequences have: the same values within the bounds."""
    c = build(17, [1, 3, 2], [30, 41, 2], 100, 8, 2, 128, type, cache, 16)
    wide = torch.full((3, 200), 2**31 - 1, dtype=torch.int32, device="cuda")
    wide[:, : c["table"].shape[1]] = c["table"]
    c["table"] = wide
    check(c, max_len=3000, max_q=64)


def test_one_token_each_without_offsets(cuda):
    c = build(19, [1] * 7, [9, 1, 33, 0, 5, 70, 2], 50, 8, 2, 128, "bf16", "bf16", 16)
    a, b = call(c), call(c, no_offsets=True)
    assert torch.equal(a, b)


@pytest.mark.parametrize("new,lens,prefix", [([1] * 6, [60] * 6, 700), ([33, 40], [50, 40], 300)])
def test_attention_gives_the_same_bits_again(cuda, new, lens, prefix):
    c = build(23, new, lens, prefix, 8, 2, 128, "f32", "bf16", 16)
    first = call(c)
    for _ in range(4):
        assert torch.equal(call(c), first)


def test_attention_more_rows_than_the_workspace_holds(cuda):
    """Parts of 4,100 sequences would take over 128 MB: every sequence then takes the prefix itself."""
    n, dim = 4100, 256
    c = build(37, [1] * n, [1 + i % 3 for i in range(n)], 40, 16, 1, dim, "bf16", "bf16", 16)
    cache, q = B.kv_cache(c["kc"], c["vc"]), B.heads(c["q"])
    assert dq.shared_attention_workspace(cache, q, q, n, n, 1, 40, 3, 3) == 0
    assert dq.shared_attention_workspace(cache, q, q, n - 1000, n - 1000, 1, 40, 3, 3) == 2 * (n - 1000) * 16 * (dim + 2) * 4
    out = call(c)
    some = list(range(0, n, 97))
    want, _, bound, _ = B.attention(c["q"].cpu()[some], [c["ks"][i] for i in some], [c["vs"][i] for i in some], [1] * len(some),
                                    [c["lens"][i] for i in some], 40, c["scale"], "bf16", "bf16")
    B.close(out[some], want, bound, "bf16")


def test_long_cache_offsets(cuda):
    """Pages more than 2^32 bytes and values apart."""
    hk, dim, page = 2, 64, 16
    far = (1 << 32) + 4096
    pool = torch.empty(far * 2 + page * hk * dim * 2, dtype=torch.float16, device="cuda")
    k = pool.as_strided((3, page, hk, dim), (far, 2 * hk * dim, dim, 1))
    v = pool.as_strided((3, page, hk, dim), (far, 2 * hk * dim, dim, 1), hk * dim)
    gen = torch.Generator().manual_seed(1)
    kk, vv = torch.randn((2, 40, hk, dim), generator=gen).half().cuda()
    slots = torch.cat([torch.arange(32, 48), torch.arange(0, 16), torch.arange(16, 24)]).cuda()
    dq.kv_append(B.kv_cache(k, v), 40, B.heads(kk), B.heads(vv), slots, stream=stream())
    assert torch.equal(k[2], kk[:16]) and torch.equal(v[0], vv[16:32]) and torch.equal(k[1, :8], kk[32:])
    c = build(1, [1, 2], [8, 8], 32, 4, hk, dim, "f32", "f16", page)
    c |= dict(kc=k, vc=v, prefix_pages=torch.tensor([2, 0], dtype=torch.int32).cuda(),
              table=torch.tensor([[1], [1]], dtype=torch.int32).cuda(), ks=[kk.cpu()] * 2, vs=[vv.cpu()] * 2)
    check(c)


def test_calls_run_on_their_stream(cuda):
    """On a stream of their own, behind work that it waits for, with a workspace of its own."""
    c = build(29, [1] * 4, [100, 20, 300, 77], 600, 8, 2, 128, "bf16", "bf16", 16)
    want = call(c)
    q = c["q"].clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        c["q"].zero_()
        big = torch.randn((4096, 4096), device="cuda")
        for _ in range(20):
            big = big @ big * 1e-4
        c["q"].copy_(q)
        out = call(c)
    side.synchronize()
    assert torch.equal(out, want)


def test_block_in_a_graph(cuda):
    """Norm, append and attention of a decode step captured once, replayed with other data."""
    hq, hk, dim, page, n = 8, 2, 128, 16, 5
    gen = torch.Generator().manual_seed(31)
    c = build(31, [1] * n, [20, 33, 16, 47, 2], 200, hq, hk, dim, "f32", "bf16", page)
    k, v = rows(gen, n, hk, dim, "f32"), rows(gen, n, hk, dim, "f32")
    td = [t.cuda() for t in B.rope_table(400, dim)]
    rope = dq.Rope(td[0].data_ptr(), td[1].data_ptr(), 400, dim, dq.ROPE_HALVES)
    pos = c["lens_d"] + 199
    w = torch.rand(dim, generator=gen).cuda()
    last = (c["lens_d"] - 1).long()
    slots = c["table"][torch.arange(n, device="cuda"), last // page].long() * page + last % page
    turned, out = torch.empty_like(c["q"]), torch.empty_like(c["q"])
    raw = c["q"]
    workspace = torch.empty(dq.ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")

    def step():
        dq.qk_norm_rope(n, dim, B.heads(raw), B.heads(turned), w, eps=1e-5, rope=rope, positions=pos, stream=stream())
        dq.kv_append(B.kv_cache(c["kc"], c["vc"]), n, B.heads(k), B.heads(v), slots, w, 1e-5, rope, pos, stream())
        call(c | {"q": turned}, out=out, workspace=workspace)

    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        raw.normal_()
        k.normal_()
        step()
        torch.cuda.synchronize()
        want = out.clone()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def check_by_heads(c, repeats=0, every=1, **kw):
    """`check` for calls of many rows (every `every`th sequence of them); every further call gives the same bits."""
    lse = torch.full((c["tokens"], c["q"].shape[1]), 33.0, device="cuda")
    out = call(c, lse=lse, **kw)
    at, start = [], 0
    for b, n in enumerate(c["new"]):
        at += range(start, start + n) if b % every == 0 else ()
        start += n
    want, want_lse, bound, lse_bound = B.attention_by_heads(c["q"][at], c["ks"][::every], c["vs"][::every], c["new"][::every],
                                                            c["lens"][::every], c["prefix"], c["scale"], c["type"], c["cache"])
    B.close(out[at], want, bound, c["type"])
    B.close(lse[at], want_lse, lse_bound, "f32")
    for _ in range(repeats):
        assert torch.equal(call(c, **kw), out)


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("new,lens,prefix", [([256] * 8, [300] * 8, 200), ([1] * 96, [130] * 96, 2000)], ids=["prompts", "decode"])
def test_attention_with_every_cu_taken(cuda, type, cache, dim, new, lens, prefix):
    """Tiles of several keys' worth on all CUs, two workgroups each, whose waves run apart: keys are loaded over
    those of two tiles before only once all waves have read them."""
    check_by_heads(build(41, new, lens, prefix, 32, 8, dim, type, cache, 16, True), repeats=10)


def put(c, pool, b, j, head, column, value):
    """Sets a value of key j (the prefix's before the own ones) of sequence b in the cache."""
    page = pool.shape[1]
    if j < c["prefix"]:
        pool[int(c["prefix_pages"][j // page]), j % page, head, column] = value
    else:
        j -= c["prefix"]
        pool[int(c["table"][b, j // page]), j % page, head, column] = value


# (few rows and tiles, with and without a prefix, one item a row and several)
SPLITS = [([1], [700], 600), ([3, 2], [40, 30], 900), ([90], [1500], 0), ([12] * 3, [60] * 3, 1100)]
IDS = ["few rows", "prefix shared", "tiles", "prefix shared by tiles"]


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("new,lens,prefix", SPLITS + [([2], [20], 0), ([70], [70], 0)], ids=IDS + ["few rows, one item", "tiles, one item"])
def test_rows_whose_scores_are_all_minus_infinity(cuda, type, new, lens, prefix):
    """They get zeros whatever the values, as rows without keys do."""
    c = build(47, new, lens, prefix, 2, 1, 64, type, type, 16)
    keys = torch.isfinite(c["kc"][..., 0])
    c["kc"][..., 0] = torch.where(keys, -math.inf, c["kc"][..., 0])
    c["q"][:, :, 0] = c["q"][:, :, 0].abs() + 1
    lse = torch.full((c["tokens"], 2), 33.0, device="cuda")
    for value in (0.5, math.inf, math.nan):
        for j in {0, prefix // 2, prefix + lens[0] - new[0], prefix + lens[0] - 1}:
            put(c, c["vc"], 0, j, 0, 9, value)
        assert torch.all(call(c, lse=lse) == 0), value
        assert torch.all(lse == -math.inf)


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,lens,prefix", SPLITS, ids=IDS)
def test_a_nan_value_is_seen_whatever_its_weight(cuda, type, cache, new, lens, prefix):
    """A visible key's NaN makes its column NaN, also where the key's weight rounds to 0 beside another
    range's: it does not depend on how the keys are split."""
    c = build(43, new, lens, prefix, 2, 1, 64, type, cache, 16)
    c["q"][:, :, 0] = 40.0
    last = prefix + lens[0] - new[0]
    for b in range(len(new)):
        put(c, c["kc"], b, prefix + lens[b] - new[b], 0, 0, 120.0)  # 600 above all others, seen by all rows
    clean = call(c)
    assert torch.isfinite(clean).all()
    for at in {0, last // 2, last - 1}:
        c2 = c | {"vc": c["vc"].clone()}
        put(c2, c2["vc"], 0, at, 0, 5, math.nan)
        out = call(c2)
        want = torch.zeros_like(out, dtype=torch.bool)
        want[: new[0] if at >= prefix else None, :, 5] = True
        assert torch.equal(torch.isnan(out), want), at
        assert torch.equal(out[~want], clean[~want])


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("dim", [64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("new,lens,prefix", SPLITS + [([5], [40], 20), ([90], [90], 0), ([40, 50], [70, 50], 64), ([70], [200], 130)])
def test_infinite_values_reach_the_rows_that_see_them(cuda, type, cache, dim, new, lens, prefix):
    """Values alone are infinite or NaN, the keys finite: their columns in the rows that see them are what the
    sum makes of them, everything else keeps its bits."""
    heads, kv = 4, 2
    c = build(53 + dim, new, lens, prefix, heads, kv, dim, type, cache, 16)
    clean = call(c)
    n, own = new[0], prefix + lens[0] - new[0]  # own: the key of row 0
    want = torch.zeros((c["tokens"], heads, dim), dtype=torch.float64)
    bad = [(own + n - 1, 0, 0, math.inf), (own + n - 1, 1, dim - 1, -math.inf), (own + n // 2, 0, 3, math.nan), (own + n // 2, 1, 1, math.inf),
           (own + n - 1, 1, 1, -math.inf), (own, 0, dim - 2, -math.inf), (own + n // 3, 0, dim // 2 + 1, math.inf),
           (max(0, own - 1), 1, dim // 2, math.inf), (0, 1, 7, -math.inf), (prefix // 2, 0, 7, math.nan)]
    for (j, head, column), value in {b[:3]: b[3] for b in bad}.items():
        put(c, c["vc"], 0, j, head, column, value)
        rows = slice(None) if j < prefix else slice(max(0, j - own), n)
        want[rows, 2 * head : 2 * head + 2, column] += value
    out = call(c).cpu()
    same = want == 0
    assert torch.equal(out[same], clean.cpu()[same])
    if type == "f32":  # (a weight's parts times an infinity: of both signs, or NaN)
        assert not torch.isfinite(out[~same]).any()
    else:
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(out[torch.isinf(want)].double(), want[torch.isinf(want)])


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 80, 96, 128])
@pytest.mark.parametrize("new,lens", [([1] * 40, [1 + 9 * i % 200 for i in range(40)]), ([3 - i % 3 for i in range(20)], [3 + 31 * i for i in range(20)])],
                         ids=["one token", "proposed tokens"])
def test_shared_tiles_of_128_rows(cuda, type, dim, new, lens):
    """A prefix so long that its items take 128 rows, own keys beside them in tiles of 16 and of 64 rows."""
    check_by_heads(build(59, new, lens, 10001, 64, 8, dim, type, type, 16, dim == 96), repeats=2, every=7)


@pytest.mark.parametrize("rot", [0, 2])
def test_more_rows_than_a_launch_has_threads_for(cuda, rot):
    """2^26 head rows and some, a wave each: in several launches, the same bits as in calls of fewer tokens. (Half of a
    rotation of 2 is less than a chunk of 8 values; heads at odd values are no chunks either.)"""
    tokens, heads, dim, part = (1 << 23) + 5, 8, 8, 1 << 20
    x = torch.randn(tokens * heads * dim + 1, device="cuda", dtype=torch.float16)[1:].view(tokens, heads, dim)
    td = [t.cuda() for t in B.rope_table(64, 2)]
    rope = dq.Rope(td[0].data_ptr(), td[1].data_ptr(), 64, 2, dq.ROPE_HALVES) if rot else None
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda") % 64
    w = 1 + torch.rand(dim, device="cuda")
    out = torch.full_like(x, math.nan)
    dq.qk_norm_rope(tokens, dim, B.heads(x), B.heads(out), w, eps=1e-5, rope=rope, positions=pos, stream=stream())
    for t0 in range(0, tokens, part):
        n = min(part, tokens - t0)
        want = torch.full_like(x[t0 : t0 + n], 55.0)
        dq.qk_norm_rope(n, dim, B.heads(x[t0 : t0 + n]), B.heads(want), w, eps=1e-5, rope=rope, positions=pos[t0 : t0 + n], stream=stream())
        assert torch.equal(out[t0 : t0 + n], want), t0
    pages = (tokens + 15) // 16
    k, v = (torch.zeros((pages, 16, heads, dim), device="cuda", dtype=torch.float16) for _ in range(2))
    slots = tokens - 1 - torch.arange(tokens, device="cuda")
    dq.kv_append(B.kv_cache(k, v), tokens, B.heads(x), B.heads(x), slots, w, 1e-5, rope, pos, stream())
    assert torch.equal(k.view(-1, heads, dim)[:tokens].flip(0), out) and torch.equal(v.view(-1, heads, dim)[:tokens].flip(0), x)


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,hq,hk,dim,tail", [([1] * 4100, 32, 8, 128, 0), ([i % 9 for i in range(1300)], 16, 4, 256, 3), ([1] * 8200, 16, 16, 128, 0)],
                         ids=["one token", "up to 8 tokens", "one token, 3 slices"])
def test_large_batches_run_in_slices(cuda, type, cache, new, hq, hk, dim, tail):
    """More rows than the workspace holds parts of: slices of the batch share the prefix, each row is its sequence's."""
    lens = [n + i % 5 for i, n in enumerate(new)]
    c = build(61, new, lens, 300, hq, hk, dim, type, cache, 16, tail=tail)
    out, lse = torch.full_like(c["q"], 55.0), torch.full((c["tokens"], hq), 33.0, device="cuda")
    call(c, out=out, lse=lse)
    n, at, start = sum(new), [], 0
    every = len(new) // 23
    for b, k in enumerate(new):
        at += range(start, start + k) if b % every == 0 else ()
        start += k
    want, want_lse, bound, lse_bound = B.attention_by_heads(c["q"][at], c["ks"][::every], c["vs"][::every], new[::every], lens[::every], 300,
                                                            c["scale"], type, cache)
    B.close(out[at], want, bound, type)
    B.close(lse[at], want_lse, lse_bound, "f32")
    assert torch.all(out[n:] == 55.0) and torch.all(lse[n:] == 33.0) and torch.isfinite(out).all() and torch.isfinite(lse).all()
    if max(new) == 1:
        assert torch.equal(call(c, out=torch.empty_like(out), no_offsets=True), out)


@pytest.mark.parametrize("offsets", [True, False])
def test_more_items_than_a_launch_has_threads_for(cuda, offsets):
    """2^24 items and some, in several launches: each of 2^21 sequences has one key, whose value it gets as it is."""
    n, heads, dim, page = (1 << 21) + 3, 8, 8, 16
    k, v = (torch.randn((64, page, heads, dim), device="cuda").half() for _ in range(2))
    q = torch.randn((n, heads, dim), device="cuda").half()
    out, lens = torch.full_like(q, math.nan), torch.ones(n, dtype=torch.int32, device="cuda")
    pages = torch.randint(0, 64, (n, 1), dtype=torch.int32, device="cuda")
    at = torch.arange(n + 1, dtype=torch.int32, device="cuda") if offsets else None
    dq.shared_attention(B.kv_cache(k, v), B.heads(q), B.heads(out), None, n, n, at, 1, None, 0, pages, 1, lens, 1, 1.0, None, 0, stream())
    assert torch.equal(out, v[pages[:, 0].long(), 0])


@pytest.mark.parametrize("new,max_q", [([3, 0, 5, 1, 2, 4, 2], 6), ([40, 33, 20, 1, 2, 4, 30], 64), ([1 + i % 2 for i in range(3000)], 2)],
                         ids=["few rows", "tiles", "slices"])
def test_offsets_of_any_values_stay_inside_the_tensors(cuda, new, max_q):
    """Offsets that decrease or leave the tokens: rows past the tensors' ends and the workspace's are not touched."""
    c = build(67, new, [n + 20 for n in new], 300, 32, 8, 128, "bf16", "bf16", 16)
    gen = torch.Generator().manual_seed(5)
    wide = torch.full((c["tokens"] + 20, 32, 128), 55.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((c["tokens"] + 20, 32), 33.0, device="cuda")
    q = torch.zeros_like(wide)
    q[10:-10] = c["q"]
    c["q"] = q[10:-10]
    for low, high in ((-(2**31), 2**31 - 1), (-5, c["tokens"] + 5)):
        c["offsets"] = torch.randint(low, high, (len(new) + 1,), generator=gen).to(torch.int32).cuda()
        call(c, out=wide[10:-10], lse=lse[10:-10], max_q=max_q)
        for x, value in ((wide, 55.0), (lse, 33.0)):
            assert torch.all(x[:10] == value) and torch.all(x[-10:] == value)
