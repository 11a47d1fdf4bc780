"""The long caches' kernels against the formulas in 64 bits (tests/longtest.py)."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import blocktest as B  # noqa: E402
import dynalm_amd as dq  # noqa: E402
import longtest as L  # noqa: E402
from longtest import KINDS, Call, stream  # noqa: E402

# ------------------------------------------------------------------ bounds of pages

LENS = [0, 1, 15, 16, 17, 130]


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 24, 64, 80, 128, 136, 256])
@pytest.mark.parametrize("page,heads_first", [(16, False), (48, True), (128, False)])
def test_bounds(cuda, cache, dim, page, heads_first):
    c = Call(dim, [1] * len(LENS), LENS, 2, 2, dim, "f32", cache, page, heads_first)
    got = L.run_bounds(c)
    L.same(got, L.page_bounds(c, None, torch.full_like(got, 55.0).cpu()))


@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_bounds_of_new_keys(cuda, cache):
    """Only the pages that hold a new key are written; starts outside the sequence are cut."""
    c = Call(1, [1] * 7, [0, 1, 16, 17, 100, 130, 130], 2, 2, 64, "f32", cache, 16)
    for start, most in (([0, 0, 15, 16, 99, 129, 100], 30), ([-5, 1, 16, 0, 200, 130, 113], 17), ([0, 0, 0, 0, 80, 128, 111], 20)):
        got = L.run_bounds(c, start, most)
        L.same(got, L.page_bounds(c, start, torch.full_like(got, 55.0).cpu()))


@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_bounds_of_infinite_and_nan_keys(cuda, cache):
    c = Call(2, [1, 1], [40, 33], 2, 2, 64, "f32", cache, 16)
    bad = [(0, 3, 0, 5, math.nan), (0, 17, 1, 9, math.inf), (0, 18, 1, 9, -math.inf), (1, 32, 0, 63, -math.nan), (1, 2, 0, 0, -math.inf),
           (0, 39, 1, 2, -math.nan), (1, 5, 1, 1, 0.0), (1, 6, 1, 1, -0.0)]
    for b, j, h, d, x in bad:
        c.ks[b][j, h, d] = x
        c.kc[int(c.table[b, j // 16]), j % 16, h, d] = x
    got = L.run_bounds(c)
    L.same(got, L.page_bounds(c, None, torch.full_like(got, 55.0).cpu()))


def test_bounds_of_pages_outside_the_cache(cuda):
    """Page numbers outside the cache are left out."""
    c = Call(3, [1, 1], [40, 40], 2, 2, 64, "f32", "f16", 16)
    want = L.page_bounds(c, None, torch.full((c.kc.shape[0], 2, 2, 64), 55.0, dtype=torch.float16))
    for b, p, number in ((0, 1, -1), (1, 2, c.kc.shape[0])):
        want[int(c.table[b, p])] = 55.0
        c.table[b, p] = number
    L.same(L.run_bounds(c), want)


# ------------------------------------------------------------------ the choice of pages

CHOICES = [
    # new, lens, q heads, kv heads, dim, page, first, last, count
    pytest.param([1], [1], 1, 1, 8, 16, 0, 1, 1, id="one key"),
    pytest.param([1, 1], [0, 40], 2, 1, 64, 16, 0, 1, 2, id="no key"),
    pytest.param([1] * 4, [16, 160, 161, 1000], 8, 2, 128, 16, 1, 2, 10, id="decode"),
    pytest.param([1] * 3, [900, 64, 701], 17, 1, 80, 48, 0, 1, 1, id="the last page alone"),
    pytest.param([1] * 2, [1500, 1100], 6, 6, 256, 16, 3, 1, 17, id="one head each"),
    pytest.param([5, 0, 2, 1], [70, 33, 2, 400], 6, 2, 72, 16, 1, 1, 4, id="proposed tokens"),
    pytest.param([40], [700], 14, 2, 96, 16, 2, 3, 9, id="prompt behind keys"),
    pytest.param([4, 6], [2, 3], 2, 1, 40, 16, 0, 1, 3, id="rows before the first key"),
    pytest.param([1, 1], [16 * 512, 16 * 513], 2, 2, 24, 16, 1, 1, 100, id="513 pages"),
    pytest.param([1, 1], [16 * 2048 + 1, 16 * 100], 2, 1, 16, 16, 1, 1, 300, id="2,049 pages"),
]


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,lens,hq,hk,dim,page,first,last,count", CHOICES)
def test_choice(cuda, new, lens, hq, hk, dim, page, first, last, count, type, cache):
    c = Call(dim + count, new, lens, hq, hk, dim, type, cache, page, heads_first=dim == 80, odd=dim == 72, tail=dim % 5)
    bounds = L.run_bounds(c)
    assert torch.equal(L.run_choose(c, bounds, first, last, count).cpu(), L.choose(c, bounds, first, last, count))


MANY_CHOICES = [
    # new, lens, q heads, kv heads, dim, page, first, last, count
    pytest.param([150], [16 * 520 + 5], 40, 2, 24, 16, 1, 1, 40, id="20 heads a kv head, 521 pages"),
    pytest.param([90, 0, 61], [16 * 640, 3, 61], 28, 14, 96, 16, 1, 2, 30, id="two heads a kv head, 640 pages"),
    pytest.param([70, 40], [70, 1200], 100, 20, 136, 16, 0, 1, 5, id="five heads a kv head, heads of 136"),
    pytest.param([33, 300, 9], [16 * 70, 300, 16 * 130 + 1], 9, 3, 64, 16, 2, 2, 11, id="ragged prompts"),
]


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,lens,hq,hk,dim,page,first,last,count", MANY_CHOICES)
def test_choice_of_many_rows(cuda, new, lens, hq, hk, dim, page, first, last, count, type, cache):
    """Scores in a launch of their own: a workgroup's waves go through many rows together."""
    c = Call(dim + count, new, lens, hq, hk, dim, type, cache, page, heads_first=dim == 96, odd=dim == 24, tail=dim % 5)
    bounds = L.run_bounds(c)
    assert torch.equal(L.run_choose(c, bounds, first, last, count).cpu(), L.choose(c, bounds, first, last, count))


def test_choice_of_equal_scores(cuda):
    """Of equal pages the lower ones; a page of zeros ties with one of minus zeros."""
    c = Call(4, [1, 1], [40 * 16, 33 * 16], 4, 2, 64, "f32", "bf16", 16)
    for values in ([0.0, -0.0], [1.0], [1.0, 2.0, 1.0, 1.0]):
        bounds = torch.empty((c.kc.shape[0], 2, 2, 64), dtype=torch.bfloat16, device="cuda")
        for b in range(2):
            for p in range(-(-c.lens[b] // 16)):
                bounds[int(c.table[b, p])] = values[p % len(values)]
        for count in (3, 8, 32):
            assert torch.equal(L.run_choose(c, bounds, 1, 1, count).cpu(), L.choose(c, bounds, 1, 1, count))


@pytest.mark.parametrize("pages,count", [(200, 70), (700, 65), (9000, 1000)])
@pytest.mark.parametrize("type,cache", KINDS)
def test_choice_where_many_pages_meet_at_the_border(cuda, pages, count, type, cache):
    """Hundreds of pages with one score, or with two, and some apart: all are told apart exactly, ties go to the lower ones."""
    c = Call(61, [1, 1], [pages * 16, pages * 16 - 300], 2, 1, 16, type, cache, 16)
    gen = torch.Generator().manual_seed(pages)
    bounds = torch.zeros((c.kc.shape[0], 1, 2, 16), dtype=c.kc.dtype, device="cuda")
    # (NaN keys elsewhere would make intervals without ends: the bounds alone count here)
    for kind in range(4):
        if kind == 0:
            c.q.zero_()
        else:
            c.q.copy_(torch.randn(c.q.shape, generator=gen))
            bounds.copy_(torch.randn((1, 1, 1, 16), generator=gen).expand(bounds.shape))
        if kind == 2:
            bounds[torch.rand(bounds.shape[0], generator=gen).cuda() < 0.5] *= 1.0078125
        if kind == 3:
            some = torch.rand(bounds.shape[0], generator=gen).cuda() < 0.02
            bounds[some] = torch.randn((int(some.sum()), 1, 2, 16), generator=gen).to(bounds.dtype).cuda() * 3
            bounds[int(c.table[0, 5]), 0, 1, 3] = math.inf
            bounds[int(c.table[0, 9]), 0, 0, 2] = math.nan
        assert torch.equal(L.run_choose(c, bounds, 2, 3, count).cpu(), L.choose(c, bounds, 2, 3, count)), kind


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e30])
@pytest.mark.parametrize("mixed", [False, True])
def test_choice_of_queries_of_any_size(cuda, type, cache, size, mixed):
    """Large and small queries, and heads whose values lie many orders of magnitude apart."""
    if type == "f16":
        size = min(max(size, 1e-6), 1e3)
    c = Call(62, [1, 2], [300 * 16, 250 * 16], 6, 2, 64, type, cache, 16)
    bounds = L.run_bounds(c)
    scale = torch.full((64,), size)
    if mixed:
        scale = scale * 2.0 ** -torch.randint(0, 12 if type == "f16" else 40, (64,), generator=torch.Generator().manual_seed(1))
    c.q.copy_((c.q.float().cpu() * scale).to(c.q.dtype))
    assert torch.equal(L.run_choose(c, bounds, 1, 1, 20).cpu(), L.choose(c, bounds, 1, 1, 20))


def test_choice_tells_scores_apart_that_differ_by_little(cuda):
    """Scores that differ by 2^-40 of their size are no tie."""
    c = Call(5, [1], [64 * 16], 1, 1, 64, "f32", "bf16", 16)
    c.q.fill_(0.0)
    c.q[..., 0], c.q[..., 1] = 2.0**20, 2.0**-20
    bounds = torch.zeros((c.kc.shape[0], 1, 2, 64), dtype=torch.bfloat16, device="cuda")
    order = torch.randperm(64, generator=torch.Generator().manual_seed(1)).tolist()
    for rank, p in enumerate(order):
        bounds[int(c.table[0, p]), 0, :, 0] = 1.0
        bounds[int(c.table[0, p]), 0, :, 1] = 1.0 + rank / 64
    got = L.run_choose(c, bounds, 0, 1, 10).cpu()
    assert got[0, 0].tolist() == sorted([63] + [p for p in reversed(order) if p != 63][:9])


def test_choice_of_infinite_and_nan_scores(cuda):
    """NaN above all, then infinity; minus infinity below all; page numbers outside the cache count as NaN."""
    c = Call(6, [1], [50 * 16], 2, 1, 64, "f32", "f16", 16)
    bounds = L.run_bounds(c)
    c.q[..., 3] = 1.0
    for p, x in ((7, math.nan), (30, math.inf), (12, -math.inf), (45, math.nan), (46, math.inf)):
        bounds[int(c.table[0, p]), 0, :, 3] = x
    c.table[0, 20] = -1
    c.table[0, 21] = c.kc.shape[0]
    for count in (1, 2, 3, 5, 7, 49):
        assert torch.equal(L.run_choose(c, bounds, 0, 1, count).cpu(), L.choose(c, bounds, 0, 1, count))


def test_choice_in_slices(cuda):
    """More scores than the workspace holds: several launches, the same pages as row by row."""
    n, keys, page = 3000, 16 * 800, 16
    c = Call(7, [1] * 2, [keys, keys - 5], 8, 8, 8, "bf16", "bf16", page)
    bounds = L.run_bounds(c)
    few = L.run_choose(c, bounds, 1, 1, 5)
    wide = Call(7, [1] * 2, [keys, keys - 5], 8, 8, 8, "bf16", "bf16", page)
    wide.kc, wide.vc = c.kc, c.vc
    wide.new = [1] * n
    wide.tokens = wide.rows = n
    wide.q = c.q.repeat(n // 2, 1, 1)
    wide.table, wide.lens_d = c.table.repeat(n // 2, 1), c.lens_d.repeat(n // 2)
    wide.offsets_d = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    got = L.run_choose(wide, bounds, 1, 1, 5)
    assert torch.equal(got, few.repeat(n // 2, 1, 1))
    assert torch.equal(L.run_choose(wide, bounds, 1, 1, 5, no_offsets=True), got)


# ------------------------------------------------------------------ attention over chosen pages

SHAPES = [
    # new, lens, q heads, kv heads, dim, page, count
    pytest.param([1], [1], 1, 1, 8, 16, 1, id="one key"),
    pytest.param([1, 1], [0, 40], 4, 4, 64, 16, 2, id="no key"),
    pytest.param([1] * 5, [1, 15, 16, 17, 530], 8, 2, 128, 16, 9, id="decode"),
    pytest.param([1] * 3, [600, 1, 259], 17, 1, 64, 64, 5, id="17 heads a kv head"),
    pytest.param([1] * 2, [65, 640], 6, 6, 256, 16, 30, id="one head each"),
    pytest.param([3, 0, 5, 1], [3, 9, 95, 377], 6, 2, 72, 48, 3, id="proposed tokens"),
    pytest.param([40], [300], 3, 1, 200, 32, 4, id="prompt"),
    pytest.param([4, 6], [2, 3], 2, 1, 40, 16, 3, id="rows before the first key"),
    pytest.param([1], [3000], 8, 2, 96, 16, 150, id="one sequence, several ranges"),
    pytest.param([2], [2600], 40, 1, 128, 128, 20, id="40 heads, several ranges"),
    pytest.param([1] * 3, [700, 16 * 77, 5], 4, 2, 128, 16, 200, id="lists longer than the pages"),
]


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,lens,hq,hk,dim,page,count", SHAPES)
def test_attention(cuda, new, lens, hq, hk, dim, page, count, type, cache):
    c = Call(dim + count, new, lens, hq, hk, dim, type, cache, page, heads_first=dim in (64, 96), odd=dim == 72, tail=dim % 5)
    out = L.check_attention(c, L.some_pages(c, count))
    for _ in range(2):
        assert torch.equal(L.run_attention(c, L.some_pages(c, count).cuda()), out)


@pytest.mark.parametrize("type,cache", KINDS)
def test_attention_lists_of_any_order(cuda, type, cache):
    """Entries in any order, some -1 or past the sequence or its visible keys, one twice."""
    c = Call(9, [1, 3], [400, 250], 4, 2, 64, type, cache, 16)
    chosen = L.some_pages(c, 12, shuffled=True)
    chosen[0, 0, :3] = torch.tensor([24, 25, 2**31 - 1], dtype=torch.int32)
    chosen[1, 1, 2:6] = torch.tensor([3, -(2**31), 3, 3], dtype=torch.int32)
    L.check_attention(c, chosen)


@pytest.mark.parametrize("type,cache", KINDS)
def test_attention_peaked_scores(cuda, type, cache):
    """Scores far apart: one key takes nearly all, the running maximum moves often."""
    c = Call(10, [1, 4], [900, 340], 4, 2, 128, type, cache, 16, spread=30.0)
    L.check_attention(c, L.some_pages(c, 20))


@pytest.mark.parametrize("type,cache", KINDS)
def test_attention_over_all_pages_is_dense(cuda, type, cache):
    """With every page chosen a row is dq_shared_attention's, within both bounds."""
    c = Call(11, [1, 3, 1], [200, 77, 0], 4, 2, 64, type, cache, 16)
    chosen = torch.arange(c.pages, dtype=torch.int32).repeat(c.tokens, 2, 1)
    out = L.check_attention(c, chosen)
    dense = torch.full_like(out, 55.0)
    work = torch.empty(dq.ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    dq.shared_attention(c.c(), B.heads(c.q), B.heads(dense), None, c.tokens, 3, c.offsets_d, c.max_q, None, 0, c.table, c.table.stride(0),
                        c.lens_d, c.most, c.scale, work, work.numel(), stream())
    want, _, bound, _ = L.page_attention(c, chosen)
    B.close(dense, want, bound, type)


@pytest.mark.parametrize("type,cache", KINDS)
def test_attention_places_that_a_row_does_not_see(cuda, type, cache):
    """Infinite and NaN keys and values past a row's keys, and on pages not chosen, change no bit."""
    c = Call(12, [3], [120], 4, 2, 64, type, cache, 16)
    chosen = L.some_pages(c, 4, seed=3)
    chosen[:, :, 0] = -1
    chosen[:, :, 3] = 7
    clean = L.run_attention(c, chosen.cuda())
    for x in (math.nan, math.inf, -math.inf):
        for pool in (c.kc, c.vc):
            pool[int(c.table[0, 7]), 119 % 16] = x  # (the last row's own key)
            for p in range(7):
                if not (chosen == p).any():
                    pool[int(c.table[0, p])] = x
        out = L.run_attention(c, chosen.cuda())
        assert torch.equal(out[:2], clean[:2]) and torch.isnan(out[2]).any()


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("count", [3, 90])
def test_attention_infinite_values(cuda, type, cache, count):
    """A visible key's infinite or NaN value reaches its column, whatever its weight; nothing else changes."""
    c = Call(13, [1], [1600], 4, 2, 64, type, cache, 16)
    chosen = L.some_pages(c, count)
    clean = L.run_attention(c, chosen.cuda())
    p = int(chosen[0, 1, 1])
    for x in (math.nan, math.inf, -math.inf):
        c.vc[int(c.table[0, p]), 5, 1, 9] = x
        out = L.run_attention(c, chosen.cuda())
        assert not torch.isfinite(out[0, 2:, 9]).any()
        out[0, 2:, 9] = clean[0, 2:, 9]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("new,lens,hq,hk,dim,page,count", [([1] * 3, [700, 333, 64], 8, 2, 128, 16, 12), ([1], [3000], 8, 2, 96, 16, 150),
                                                           ([40, 2], [300, 700], 6, 2, 64, 32, 5), ([1] * 2, [600, 1], 17, 1, 256, 64, 8)])
def test_attention_weights_of_16_bit_rows(cuda, new, lens, hq, hk, dim, page, count, type):
    """The output is off by its own rounding and little else: the softmax weights are not rounded to 16 bits."""
    c = Call(dim + 1, new, lens, hq, hk, dim, type, type, page)
    chosen = L.some_pages(c, count)
    out = L.run_attention(c, chosen.cuda())
    c.type = "f32"  # (the bound without a rounding of weights)
    want, _, bound, _ = L.page_attention(c, chosen)
    values, c.vs = c.vs, [v.abs() for v in c.vs]
    size = L.page_attention(c, chosen)[0]
    # weights in two parts: 2^-16 of each for bf16; for f16 2^-22, and 2^-24 of weights whose largest is 2^6 or more
    most = max(v.abs().max().item() for v in values if v.numel())
    part = 2.0**-16 * size if type == "bf16" else 2.0**-22 * size + 2.0**-30 * count * page * most
    B.close(out[: c.rows], want, bound + part, type)


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_attention_an_infinite_value_keeps_its_sign(cuda, type):
    """Of keys that have a weight, whatever its bits."""
    c = Call(16, [1], [400], 4, 2, 64, type, type, 16)
    c.q.mul_(0.1)
    chosen = L.some_pages(c, 6)
    p = int(chosen[0, 0, 2])
    c.kc[int(c.table[0, p]), 2, 0] = 0.0  # (one score of 0 beside the others)
    for j in range(4):
        for x in (math.inf, -math.inf):
            c.vc[int(c.table[0, p]), j, 0, 9 + j] = x
            out = L.run_attention(c, chosen.cuda())
            assert torch.all(out[0, :2, 9 + j] == x)


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("count", [2, 80])
def test_attention_scores_of_minus_infinity(cuda, type, count):
    """Rows whose every score is -inf get zeros whatever the values."""
    c = Call(14, [1], [1500], 2, 1, 64, type, type, 16)
    c.kc[..., 0] = torch.where(torch.isfinite(c.kc[..., 0]), -math.inf, c.kc[..., 0])
    c.q[:, :, 0] = c.q[:, :, 0].abs() + 1
    chosen = L.some_pages(c, count)
    lse = torch.full((1, 2), 33.0, device="cuda")
    for x in (0.5, math.inf, math.nan):
        c.vc[int(c.table[0, int(chosen[0, 0, 0])]), 3, 0, 9] = x
        assert torch.all(L.run_attention(c, chosen.cuda(), lse=lse) == 0)
        assert torch.all(lse == -math.inf)


def test_attention_page_numbers_outside_the_cache(cuda):
    """A row that would read one gets NaN; one whose list leaves it out does not."""
    c = Call(15, [1, 1, 1], [400, 400, 400], 4, 2, 64, "f32", "f16", 16)
    chosen = L.some_pages(c, 6)
    chosen[1, :, 2] = 9
    chosen[2][chosen[2] == 9] = -1
    clean = L.run_attention(c, chosen.cuda())
    for number in (-1, c.kc.shape[0], 2**31 - 1):
        c.table[1, 9] = c.table[2, 9] = number
        out = L.run_attention(c, chosen.cuda())
        assert torch.isnan(out[1]).all() and torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])


# ------------------------------------------------------------------ the weight that keys gather

MASSES = [
    # new, lens, q heads, kv heads, dim, page
    pytest.param([1], [1], 1, 1, 8, 16, id="one key"),
    pytest.param([1, 1, 1], [0, 40, 257], 4, 4, 64, 16, id="decode"),
    pytest.param([1] * 3, [600, 1, 259], 17, 1, 80, 48, id="17 heads a kv head"),
    pytest.param([3, 0, 5, 1], [3, 9, 95, 377], 6, 2, 72, 16, id="proposed tokens"),
    pytest.param([70], [300], 4, 2, 128, 64, id="prompt"),
    pytest.param([33, 64], [33, 70], 2, 2, 256, 16, id="prompts"),
    pytest.param([4, 6], [2, 3], 2, 1, 40, 16, id="rows before the first key"),
    pytest.param([300], [300], 4, 1, 96, 32, id="several ranges of rows"),
    pytest.param([130, 3, 90], [700, 300, 90], 6, 2, 136, 48, id="prompts, heads of 136"),
    pytest.param([200], [650], 7, 1, 48, 16, id="prompt, 7 heads a kv head"),
]


def weights(c, width=None, heads_far=False):
    """Earlier weights [batch, kv_heads, width], with NaN where none are read."""
    shape = (c.hk, len(c.new), width or c.most + 3) if heads_far else (len(c.new), c.hk, width or c.most + 3)
    x = torch.rand(shape, generator=torch.Generator().manual_seed(c.dim)).cuda()
    x = x.transpose(0, 1) if heads_far else x
    for b, (n, k) in enumerate(zip(c.new, c.lens)):
        x[b, :, max(0, k - n) : k] = math.nan
    return x


def own_lse(c, spread=0.0):
    """lse of the rows over all keys that they see, as the attention writes it."""
    q, lse = c.q.cpu().double(), torch.full((c.tokens, c.hq), 5.0)
    for t in range(c.rows):
        b, sees = c.row(t)
        for h in range(c.hq):
            lse[t, h] = torch.logsumexp(c.ks[b][:sees, h // (c.hq // c.hk)].double() @ q[t, h] * c.scale, 0)
    return lse.cuda()


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("decay", [0.0, 0.75, 1.0])
@pytest.mark.parametrize("new,lens,hq,hk,dim,page", MASSES)
def test_mass(cuda, new, lens, hq, hk, dim, page, decay, type, cache):
    c = Call(dim, new, lens, hq, hk, dim, type, cache, page, heads_first=dim == 128, odd=dim == 72, tail=dim % 5)
    lse, old = own_lse(c), weights(c, heads_far=decay == 0.75)
    if decay == 0:
        old.fill_(math.nan)
    before = old.clone()
    got = L.run_mass(c, lse, old, decay)
    want, bound = L.mass(c, lse, before, decay)
    for b, k in enumerate(lens):
        B.close(got[b, :, :k], want[b, :, :k], bound[b, :, :k], "f32")
        rest = got[b, :, k:]
        assert torch.equal(torch.nan_to_num(rest, 9.0), torch.nan_to_num(before[b, :, k:], 9.0))
    again = before.clone()
    assert torch.equal(torch.nan_to_num(L.run_mass(c, lse, again, decay), 9.0), torch.nan_to_num(got, 9.0))


def test_mass_of_a_row_adds_up_to_one(cuda):
    """With lse from dq_shared_attention the weights of a sequence's rows add up to their number."""
    c = Call(21, [1, 40, 7], [900, 300, 7], 8, 2, 128, "bf16", "bf16", 16)
    out, lse = torch.empty_like(c.q), torch.full((c.tokens, 8), 33.0, device="cuda")
    work = torch.empty(dq.ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    dq.shared_attention(c.c(), B.heads(c.q), B.heads(out), lse, c.tokens, 3, c.offsets_d, c.max_q, None, 0, c.table, c.table.stride(0),
                        c.lens_d, c.most, c.scale, work, work.numel(), stream())
    mass = L.run_mass(c, lse, torch.zeros((3, 2, c.most), device="cuda"), 0.0)
    want = torch.tensor(c.new, dtype=torch.float64)[:, None].expand(3, 2) * 4
    # lse's bound and the weights' (their largest score distance is below 30, sums of up to 160 rows)
    assert torch.all((mass.double().sum(-1).cpu() - want).abs() <= want * 2e-5)


def test_mass_lse_of_any_value(cuda):
    """-inf adds nothing, +inf nothing either, NaN makes what the row sees NaN; large ones stay in their row."""
    c = Call(22, [4], [60], 2, 1, 64, "f32", "f16", 16)
    lse = own_lse(c)
    lse[0, 0], lse[1, 1], lse[2, 0], lse[2, 1] = -math.inf, math.inf, 3e38, 1e30
    got = L.run_mass(c, lse, torch.zeros((1, 1, 60), device="cuda"), 0.0)
    some = torch.where(lse.abs() > 1e20, -math.inf, lse)
    want, bound = L.mass(c, some, torch.zeros((1, 1, 60)), 0.0)
    B.close(got, want, bound, "f32")
    lse[1, 0] = math.nan
    got = L.run_mass(c, lse, torch.zeros((1, 1, 60), device="cuda"), 0.0)
    assert torch.isnan(got[..., :58]).all() and torch.isfinite(got[..., 58:]).all()


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,lens", [([4], [60]), ([150], [300])])
def test_mass_lse_of_large_size(cuda, new, lens, type, cache):
    """A row whose lse is far above its scores adds 0 to each key that it sees, one whose lse is far below them infinity, whatever
    lse's bits; by few rows and by many."""
    c = Call(24, new, lens, 4, 2, 64, type, cache, 16)
    start = own_lse(c)
    large = [3e9, 5e9, 1e10, 1.1e10, 1e11, 1e15, 1.5e15, 1e30, 3e30, 7e33, 2e38]
    for first in range(3):
        lse = start.clone()
        for i, t in enumerate(range(0, new[0], 3)):
            lse[t, (t + first) % 4] = large[(i + 4 * first) % len(large)]
        got = L.run_mass(c, lse, torch.zeros((1, 2, lens[0]), device="cuda"), 0.0)
        want, bound = L.mass(c, lse, torch.zeros((1, 2, lens[0])), 0.0)
        B.close(got, want, bound, "f32")
    for x in large:
        lse = start.clone()
        lse[1, 0] = -x
        got = L.run_mass(c, lse, torch.zeros((1, 2, lens[0]), device="cuda"), 0.0)
        sees = c.row(1)[1]
        assert torch.all(got[0, 0, :sees] == math.inf) and torch.isfinite(got[0, 0, sees:]).all() and torch.isfinite(got[0, 1]).all()


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("group,dim,new,lens", [(3, 64, 150, 300), (5, 256, 70, 200), (7, 128, 60, 400), (22, 96, 20, 90), (4, 128, 100, 300), (3, 64, 5, 60)])
def test_mass_of_infinite_keys(cuda, group, dim, new, lens, type, cache):
    """A key on which every row scores -inf gathers 0, by few rows and by many, whatever the number of heads a kv head; the others what
    they gather beside it. (With fp32 rows, whose products are summed in parts, that key's may be NaN.)"""
    c = Call(25, [new], [lens], 2 * group, 2, dim, type, cache, 16)
    c.q[..., 5] = c.q[..., 5].abs() + 0.5
    for j, h in ((20, 0), (33, 1)):
        c.ks[0][j, h, 5] = -math.inf
        c.kc[int(c.table[0, j // 16]), j % 16, h, 5] = -math.inf
    lse = own_lse(c)
    got = L.run_mass(c, lse, torch.zeros((1, 2, lens), device="cuda"), 0.0)
    want, bound = L.mass(c, lse, torch.zeros((1, 2, lens)), 0.0)
    bound = torch.nan_to_num(bound, 0.0, 0.0, 0.0)  # (of the two keys: exactly 0)
    for j, h in ((20, 0), (33, 1)):
        assert want[0, h, j] == 0
        if type == "f32" and torch.isnan(got[0, h, j]):
            got[0, h, j] = 0.0
    B.close(got, want, bound, "f32")


@pytest.mark.parametrize("type,cache", KINDS)
@pytest.mark.parametrize("new,lens", [(5, 60), (150, 300)])
def test_mass_of_rows_without_weights(cuda, new, lens, type, cache):
    """A row whose lse is -inf adds nothing, whatever it scores: infinite and NaN keys and queries among them."""
    c = Call(26, [new], [lens], 4, 2, 64, type, cache, 16)
    dead = torch.zeros((c.tokens, 4), dtype=torch.bool)
    dead[torch.arange(1, new, 3), torch.arange(1, new, 3) % 4] = True
    dead[2] = True
    # the live rows score -inf on one key, the others +inf; one of the others is NaN itself
    c.q[..., 5] = torch.where(dead.cuda(), -1.0, 1.0) * (c.q[..., 5].abs() + 0.5)
    c.ks[0][20, 0, 5] = -math.inf
    c.kc[int(c.table[0, 1]), 4, 0, 5] = -math.inf
    lse = own_lse(c)
    lse[dead.cuda()] = -math.inf
    c.q[2, 3, 7] = math.nan
    c.q[2, 1, 9] = math.inf
    got = L.run_mass(c, lse, torch.zeros((1, 2, lens), device="cuda"), 0.0)
    want, bound = L.mass(c, lse, torch.zeros((1, 2, lens)), 0.0)
    bound = torch.nan_to_num(bound, 0.0, 0.0, 0.0)
    assert want[0, 0, 20] == 0 and torch.isfinite(want).all()
    if type == "f32" and torch.isnan(got[0, 0, 20]):
        got[0, 0, 20] = 0.0
    B.close(got, want, bound, "f32")
    # all of them
    lse.fill_(-math.inf)
    c.kc[int(c.table[0, 0]), 3, 1] = math.nan
    assert torch.all(L.run_mass(c, lse, torch.ones((1, 2, lens), device="cuda"), 0.0) == 0)


def test_mass_of_infinite_and_hidden_keys(cuda):
    """A NaN key's weight is NaN, no other's; places past the keys hold NaN and are not read into any."""
    c = Call(23, [2, 1], [50, 33], 2, 1, 64, "bf16", "bf16", 16)
    lse = own_lse(c)
    clean = L.run_mass(c, lse, torch.zeros((2, 1, 50), device="cuda"), 0.0)
    c.kc[int(c.table[0, 1]), 4, 0, 7] = math.nan
    got = L.run_mass(c, lse, torch.zeros((2, 1, 50), device="cuda"), 0.0)
    assert torch.isnan(got[0, 0, 20])
    got[0, 0, 20] = clean[0, 0, 20]
    assert torch.equal(got, clean)
    c.table[1, 1] = -1
    got = L.run_mass(c, lse, torch.zeros((2, 1, 50), device="cuda"), 0.0)
    assert torch.isnan(got[1, 0, 16:32]).all() and torch.equal(got[1, 0, :16], clean[1, 0, :16]) and torch.equal(got[1, 0, 32:], clean[1, 0, 32:])


# ------------------------------------------------------------------ the keys that stay

KEEPS = [([1], 1, 0, 0, 1), ([0, 5, 100], 2, 4, 8, 20), ([100, 64, 65], 3, 0, 0, 64), ([1000, 999, 3], 2, 16, 45, 61), ([5000, 4097], 2, 4, 32, 1001),
         ([20000, 16385], 1, 0, 1, 4096), ([70000, 66000], 1, 5, 7, 300), ([300], 4, 0, 0, 299)]


@pytest.mark.parametrize("lens,heads,first,last,budget", KEEPS)
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_keep(cuda, lens, heads, first, last, budget, kind):
    gen = torch.Generator().manual_seed(budget)
    w = torch.exp(2 * torch.randn((len(lens), heads, max(lens) + 5), generator=gen))
    if kind == "ties":
        w = torch.randint(0, 3, w.shape, generator=gen).float()
    if kind == "odd":
        odd = torch.tensor([math.nan, math.inf, -math.inf, -0.0, 0.0, -1.0, 1e-42, math.nan])
        w = torch.where(torch.rand(w.shape, generator=gen) < 0.8, odd[torch.randint(0, 8, w.shape, generator=gen)], w)
    kept, kept_lens = L.run_keep(lens, w.cuda(), first, last, budget)
    assert torch.equal(kept.cpu(), L.keep(w, lens, first, last, budget))
    assert kept_lens.tolist() == [min(n, budget) for n in lens]


@pytest.mark.parametrize("lens,heads,first,last,budget", [([8193, 16384, 12000], 2, 4, 128, 4096), ([4097, 8192], 1, 0, 3, 4), ([16385], 1, 3, 0, 16384),
                                                          ([65536, 16500], 1, 1, 1, 5000), ([65537], 1, 0, 0, 65536)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd", "near"])
def test_keep_of_every_length(cuda, lens, heads, first, last, budget, kind):
    """Around the lengths at which a lane holds more places, up to those that are read again."""
    gen = torch.Generator().manual_seed(budget)
    w = torch.exp(2 * torch.randn((len(lens), heads, max(lens) + 5), generator=gen))
    if kind == "ties":
        w = torch.randint(0, 3, w.shape, generator=gen).float()
    if kind == "odd":
        odd = torch.tensor([math.nan, math.inf, -math.inf, -0.0, 0.0, -1.0, 1e-42, math.nan])
        w = torch.where(torch.rand(w.shape, generator=gen) < 0.8, odd[torch.randint(0, 8, w.shape, generator=gen)], w)
    if kind == "near":  # (neighbours among the floats: every pass over the bins counts)
        w = (torch.randint(0, 1 << 16, w.shape, generator=gen, dtype=torch.int32) + 0x3F000000).view(torch.float32)
        w[..., 0], w[..., 1] = 1e30, 1e-30
    kept, kept_lens = L.run_keep(lens, w.cuda(), first, last, budget)
    assert torch.equal(kept.cpu(), L.keep(w, lens, first, last, budget))
    assert kept_lens.tolist() == [min(n, budget) for n in lens]


def test_keep_lengths_beyond_the_bounds_are_cut(cuda):
    w = torch.rand((3, 1, 40), device="cuda")
    lens = torch.tensor([1 << 30, -5, 40], dtype=torch.int32, device="cuda")
    kept, kept_lens = (torch.full(n, 77, dtype=torch.int32, device="cuda") for n in ((3, 1, 10), (3,)))
    s = dq.Sequences(3, 0, None, 1, None, 0, lens.data_ptr(), 40)
    dq.kv_keep(s, 1, w, 40, 40, 1, 1, 10, kept, kept_lens, stream())
    assert torch.equal(kept.cpu(), L.keep(w, [40, 0, 40], 1, 1, 10)) and kept_lens.tolist() == [10, 0, 10]


# ------------------------------------------------------------------ their move


def lists(c, budget, seed=0):
    """Ascending places of each kv head, -1 behind."""
    gen = torch.Generator().manual_seed(seed)
    kept = torch.full((len(c.new), c.hk, budget), -1, dtype=torch.int32)
    for b, n in enumerate(c.lens):
        for h in range(c.hk):
            mine = torch.randperm(n, generator=gen)[:budget].sort().values.to(torch.int32)
            kept[b, h, : len(mine)] = mine
    return kept


MOVES = [([5], 1, 8, 16, 3), ([0, 1, 100], 2, 64, 16, 40), ([700, 301], 3, 128, 48, 200), ([2500, 2000], 2, 80, 16, 1999), ([300, 150], 2, 256, 32, 500),
         ([3000], 1, 24, 128, 2900)]


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("lens,hk,dim,page,budget", MOVES)
@pytest.mark.parametrize("moved", [False, True])
def test_compact(cuda, cache, lens, hk, dim, page, budget, moved):
    c = Call(dim, [1] * len(lens), lens, hk, hk, dim, "f32", cache, page, heads_first=dim in (80, 128))
    kept = lists(c, budget)
    w = torch.rand((len(lens), hk, c.most), generator=torch.Generator().manual_seed(3)).cuda()
    before = [p.cpu().clone() for p in (c.kc, c.vc)]
    table = c.table.cpu().long()
    to = None
    if moved:
        each = -(-min(budget, c.most) // page)
        pools = [torch.cat((p, torch.full((each * len(lens), *p.shape[1:]), 44.0, dtype=p.dtype, device="cuda"))) for p in (c.kc, c.vc)]
        if c.kc.stride(2) > c.kc.stride(1):
            pools = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in pools]
        to = (c.kc.shape[0] + torch.randperm(each * len(lens), generator=torch.Generator().manual_seed(1))).to(torch.int32).view(len(lens), each)
        c.kc, c.vc = pools
        before = [p.cpu().clone() for p in pools]
    want = [p.clone() for p in before]
    target = to.long() if moved else table
    want_w = w.cpu().clone()
    for b in range(len(lens)):
        for h in range(hk):
            mine = kept[b, h][kept[b, h] >= 0].long()
            i = torch.arange(len(mine))
            for pool, old in zip(want, before):
                pool[target[b, i // page], i % page, h] = old[table[b, mine // page], mine % page, h]
            want_w[b, h, : len(mine)] = w[b, h].cpu()[mine]
    dq.kv_compact(c.c(), c.seqs(), kept.cuda(), budget, to.cuda() if moved else None, to.stride(0) if moved else 0, w, w, *w.stride()[:2], stream())
    for got, x in zip((c.kc, c.vc), want):
        L.same(got, x)
    assert torch.equal(w.cpu(), want_w)


def test_compact_lists_of_any_values_stay_inside(cuda):
    """Entries outside the sequence and pages outside the cache are left out; other sequences' pages keep their bits."""
    c = Call(31, [1, 1], [90, 90], 2, 2, 64, "f32", "f16", 16)
    gen = torch.Generator().manual_seed(2)
    kept = torch.randint(-(2**31), 2**31 - 1, (2, 2, 120), generator=gen, dtype=torch.int64).to(torch.int32)
    kept[0, :, ::3] = torch.randint(-5, 100, (2, 40), generator=gen).to(torch.int32)
    c.table[0, 3] = -7
    c.table[0, 1] = c.kc.shape[0]
    before = c.kc.clone(), c.vc.clone()
    dq.kv_compact(c.c(), c.seqs(), kept.cuda(), 120, stream=stream())
    mine = c.table[0, [0, 2, 4, 5]].long()
    others = torch.ones(c.kc.shape[0], dtype=torch.bool)
    others[mine.cpu()] = False
    for got, x in zip((c.kc, c.vc), before):
        L.same(got[others.cuda()], x[others.cuda()])


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("dim,page,heads_first,weights_in_place", [(64, 16, False, True), (80, 48, True, False), (256, 64, True, True), (8, 16, False, None)])
def test_compact_many_sequences_in_place(cuda, cache, dim, page, heads_first, weights_in_place):
    """A serving batch: 32 sequences of 4 heads, some of which keep more than a list's part of 2,048 places."""
    hk, budget = 4, 2500
    lens = [5000, 2501, 0, 2100, 1, 4097] + [17 + 31 * i for i in range(26)]
    c = Call(34, [1] * 32, lens, hk, hk, dim, "f32", cache, page, heads_first=heads_first)
    kept = lists(c, budget)
    w = torch.rand((32, hk, c.most), generator=torch.Generator().manual_seed(3)).cuda()
    out = None if weights_in_place is None else w if weights_in_place else torch.full_like(w, 33.0)
    want, table = [p.cpu().clone() for p in (c.kc, c.vc)], c.table.cpu().long()
    want_w = None if out is None else out.cpu().clone()
    for b in range(32):
        for h in range(hk):
            mine = kept[b, h][kept[b, h] >= 0].long()
            i = torch.arange(len(mine))
            for pool, own in zip(want, (c.ks, c.vs)):
                pool[table[b, i // page], i % page, h] = own[b][mine, h]
            if out is not None:
                want_w[b, h, : len(mine)] = w[b, h].cpu()[mine]
    dq.kv_compact(c.c(), c.seqs(), kept.cuda(), budget, None, 0, None if out is None else w, out, *w.stride()[:2], stream())
    for got, x in zip((c.kc, c.vc), want):
        L.same(got, x)
    assert out is None or torch.equal(out.cpu(), want_w)


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("lens,hk,dim,budget", [([9, 0, 40], 2, 64, 40), ([300, 100], 1, 80, 5000), ([700, 3000], 2, 24, 2900)])
def test_compact_lists_with_gaps(cuda, cache, lens, hk, dim, budget):
    """Into pages of their own: places in any order, some twice, some left out, lists longer than the sequence; weights beside them."""
    page = 16
    c = Call(33, [1] * len(lens), lens, hk, hk, dim, "f32", cache, page)
    most, gen = min(budget, c.most), torch.Generator().manual_seed(7)
    each = -(-most // page)
    kept = torch.full((len(lens), hk, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        kept[b] = torch.randint(-(n // 3) - 1, n + n // 3 + 1, (hk, budget), generator=gen).to(torch.int32)
    first = c.kc.shape[0]
    c.kc, c.vc = (torch.cat((p, torch.full((each * len(lens), *p.shape[1:]), 44.0, dtype=p.dtype, device="cuda"))) for p in (c.kc, c.vc))
    to = (first + torch.randperm(each * len(lens), generator=gen)).to(torch.int32).view(len(lens), each)
    w = torch.rand((len(lens), hk, c.most), generator=gen).cuda()
    out = torch.full_like(w, 33.0)
    want, want_w = [p.cpu().clone() for p in (c.kc, c.vc)], out.cpu().clone()
    for b, n in enumerate(lens):
        for h in range(hk):
            place = kept[b, h, :most].long()
            i = torch.arange(most)[(place >= 0) & (place < n)]
            for pool, own in zip(want, (c.ks, c.vs)):
                pool[to[b, i // page].long(), i % page, h] = own[b][place[i], h]
            want_w[b, h, i] = w[b, h].cpu()[place[i]]
    dq.kv_compact(c.c(), c.seqs(), kept.cuda(), budget, to.cuda(), each, w, out, *w.stride()[:2], stream())
    for got, x in zip((c.kc, c.vc), want):
        L.same(got, x)
    assert torch.equal(out.cpu(), want_w)


def test_compact_weights_alone_in_place(cuda):
    """Keys into pages of their own, weights in place: a long list moves as a whole."""
    c = Call(32, [1], [9000], 1, 1, 8, "f32", "f16", 16)
    kept = lists(c, 8000)
    each = 500
    kc, vc = (torch.cat((p, torch.zeros((each, *p.shape[1:]), dtype=p.dtype, device="cuda"))) for p in (c.kc, c.vc))
    c.kc, c.vc = kc, vc
    to = torch.arange(kc.shape[0] - each, kc.shape[0], dtype=torch.int32, device="cuda")[None]
    w = torch.rand((1, 1, 9000), device="cuda")
    want = w.clone()
    want[0, 0, :8000] = w[0, 0, kept[0, 0].long().cuda()]
    dq.kv_compact(c.c(), c.seqs(), kept.cuda(), 8000, to, each, w, w, 9000, 9000, stream())
    assert torch.equal(w, want)


# ------------------------------------------------------------------ far strides, streams, graphs, the whole


def test_long_cache_offsets(cuda):
    """Pages more than 2^32 bytes and values apart, through all calls."""
    hk, dim, page = 2, 64, 16
    far = (1 << 32) + 4096
    c = Call(41, [1, 2], [40, 33], 4, hk, dim, "f32", "f16", page)
    pool = torch.empty(far * 2 + page * hk * dim * 2, dtype=torch.float16, device="cuda")
    k = pool.as_strided((3, page, hk, dim), (far, 2 * hk * dim, dim, 1))
    v = pool.as_strided((3, page, hk, dim), (far, 2 * hk * dim, dim, 1), hk * dim)
    kk, vv = (torch.randn((40, hk, dim), generator=torch.Generator().manual_seed(1)).half() for _ in range(2))
    c.ks, c.vs = [kk, kk[:33]], [vv, vv[:33]]
    for p, number in enumerate((2, 0, 1)):
        n = min(16, 40 - 16 * p)
        k[number, :n], v[number, :n] = kk[16 * p : 16 * p + n].cuda(), vv[16 * p : 16 * p + n].cuda()
    c.kc, c.vc = k, v
    c.table = torch.tensor([[2, 0, 1], [2, 0, 1]], dtype=torch.int32).cuda()
    first = Call(41, [1, 2], [40, 33], 4, hk, dim, "f32", "f16", page)
    first.kc, first.vc, first.table, first.ks, first.lens = k, v, c.table[:1].repeat(2, 1), [kk, kk], [40, 40]
    first.lens_d = torch.tensor([40, 40], dtype=torch.int32).cuda()
    bounds = L.run_bounds(first)
    L.same(bounds, L.page_bounds(first, None, bounds.cpu()))
    chosen = L.run_choose(c, bounds, 0, 1, 2)
    assert torch.equal(chosen.cpu(), L.choose(c, bounds, 0, 1, 2))
    L.check_attention(c, chosen)
    lse = own_lse(c)
    got = L.run_mass(c, lse, torch.zeros((2, hk, 40), device="cuda"), 0.0)
    want, bound = L.mass(c, lse, torch.zeros((2, hk, 40)), 0.0)
    B.close(got, want, bound, "f32")
    kept = torch.tensor([3, 20, 30, 33, 39], dtype=torch.int32).cuda().repeat(1, hk, 1)
    one = dq.Sequences(1, 0, None, 1, c.table.data_ptr(), 3, c.lens_d.data_ptr(), 40)
    dq.kv_compact(c.c(), one, kept, 5, stream=stream())
    assert torch.equal(k[2, :5].cpu(), kk[[3, 20, 30, 33, 39]]) and torch.equal(v[2, :5].cpu(), vv[[3, 20, 30, 33, 39]])


class Cycle:
    """A decode step's calls and an eviction, as a program makes them."""

    def __init__(self, seed, type, cache):
        self.c = c = Call(seed, [1] * 3, [700, 333, 64], 8, 2, 128, type, cache, 16)
        self.bounds = torch.zeros((c.kc.shape[0], 2, 2, 128), dtype=c.kc.dtype, device="cuda")
        self.chosen = torch.empty((3, 2, 12), dtype=torch.int32, device="cuda")
        self.out, self.dense = torch.empty_like(c.q), torch.empty_like(c.q)
        self.lse, self.page_lse = (torch.empty((3, 8), device="cuda") for _ in range(2))
        self.mass, self.mass_out = (torch.zeros((3, 2, 700), device="cuda") for _ in range(2))
        self.kept = torch.empty((3, 2, 200), dtype=torch.int32, device="cuda")
        self.kept_lens = torch.empty(3, dtype=torch.int32, device="cuda")
        self.work = torch.empty(dq.ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")

    def run(self):
        c, w, n = self.c, self.work, self.work.numel()
        cache, s, q = c.c(), c.seqs(), B.heads(c.q)
        dq.page_bounds(cache, s, None, 0, self.bounds, stream())
        dq.choose_pages(cache, s, q, self.bounds, 1, 2, 12, self.chosen, w, n, stream())
        dq.page_attention(cache, s, q, B.heads(self.out), self.page_lse, self.chosen, 12, c.scale, w, n, stream())
        dq.shared_attention(cache, q, B.heads(self.dense), self.lse, 3, 3, None, 1, None, 0, c.table, c.table.stride(0), c.lens_d, c.most,
                            c.scale, w, n, stream())
        dq.attention_mass(cache, s, q, self.lse, c.scale, 0.5, self.mass, 1400, 700, w, n, stream())
        dq.kv_keep(s, 2, self.mass, 1400, 700, 2, 5, 200, self.kept, self.kept_lens, stream())
        dq.kv_compact(cache, s, self.kept, 200, None, 0, self.mass, self.mass_out, 1400, 700, stream())

    def results(self):
        c = self.c
        return [x.clone() for x in (self.bounds, self.chosen, self.out, self.page_lse, self.mass, self.kept, self.kept_lens, self.mass_out, c.kc, c.vc)]


def assert_same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(torch.nan_to_num(x.float(), 7.0), torch.nan_to_num(y.float(), 7.0))


@pytest.mark.parametrize("type,cache", KINDS)
def test_the_calls_together(cuda, type, cache):
    """Each call's result from the one before it, against the formulas; then attention over what stayed."""
    y = Cycle(51, type, cache)
    c = y.c
    old = c.kc.cpu().clone(), c.vc.cpu().clone()
    y.run()
    L.same(y.bounds, L.page_bounds(c, None, torch.zeros_like(y.bounds).cpu()))
    assert torch.equal(y.chosen.cpu(), L.choose(c, y.bounds, 1, 2, 12))
    want, want_lse, bound, lse_bound = L.page_attention(c, y.chosen)
    B.close(y.out, want, bound, type)
    B.close(y.page_lse, want_lse, lse_bound, "f32")
    want, bound = L.mass(c, y.lse, torch.zeros((3, 2, 700)), 0.5)
    B.close(y.mass, want, bound, "f32")
    kept = L.keep(y.mass, c.lens, 2, 5, 200)
    assert torch.equal(y.kept.cpu(), kept) and y.kept_lens.tolist() == [200, 200, 64]
    ks, vs = [], []
    for b, n in enumerate(y.kept_lens.tolist()):
        ks.append(torch.stack([c.ks[b][kept[b, h, :n].long(), h] for h in range(2)], 1))
        vs.append(torch.stack([c.vs[b][kept[b, h, :n].long(), h] for h in range(2)], 1))
    out = torch.empty_like(c.q)
    dq.shared_attention(c.c(), B.heads(c.q), B.heads(out), None, 3, 3, None, 1, None, 0, c.table, c.table.stride(0), y.kept_lens, 200,
                        c.scale, y.work, y.work.numel(), stream())
    want, _, bound, _ = B.attention(c.q.cpu(), ks, vs, [1, 1, 1], [200, 200, 64], 0, c.scale, type, cache)
    B.close(out, want, bound, type)
    # what lay behind the kept keys is as it was
    table = c.table.cpu().long()
    for b, n in enumerate(c.lens):
        j = torch.arange(min(n, 200), n)
        for pool, x in zip((c.kc, c.vc), old):
            assert torch.equal(pool.cpu()[table[b, j // 16], j % 16], x[table[b, j // 16], j % 16])


def test_the_calls_in_a_graph(cuda):
    """All calls captured once, replayed with other data and lengths; eager work between the replays."""
    y = Cycle(52, "f32", "bf16")
    c = y.c
    start = c.kc.clone(), c.vc.clone()
    y.run()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y.run()
    for i in range(4):
        c.q.normal_()
        c.lens_d.copy_(torch.tensor([700 - 31 * i, 333 - i, 64 - 20 * i], dtype=torch.int32))
        got = []
        for go in (y.run, graph.replay):
            c.kc.copy_(start[0])
            c.vc.copy_(start[1])
            y.mass.fill_(0.25)
            y.mass_out.zero_()
            y.bounds.zero_()
            torch.cuda.synchronize()
            go()
            torch.cuda.synchronize()
            got.append(y.results())
        assert_same(*got)


@pytest.mark.parametrize("type,cache", KINDS)
def test_prompts_in_a_graph(cuda, type, cache):
    """The calls over many rows captured once, replayed with other queries, an infinite key and rows without weights among them."""
    c = Call(56, [150, 40], [700, 333], 6, 2, 128, type, cache, 16)
    bounds = torch.zeros((c.kc.shape[0], 2, 2, 128), dtype=c.kc.dtype, device="cuda")
    chosen = torch.empty((c.tokens, 2, 12), dtype=torch.int32, device="cuda")
    out, dense = torch.empty_like(c.q), torch.empty_like(c.q)
    lse, page_lse = (torch.empty((c.tokens, 6), device="cuda") for _ in range(2))
    mass = torch.zeros((2, 2, 700), device="cuda")
    work = torch.empty(dq.ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    dead = torch.zeros((c.tokens, 6), dtype=torch.bool, device="cuda")
    dead[::7, 1] = True

    def run():
        kv, s, q = c.c(), c.seqs(), B.heads(c.q)
        dq.page_bounds(kv, s, None, 0, bounds, stream())
        dq.choose_pages(kv, s, q, bounds, 1, 2, 12, chosen, work, work.numel(), stream())
        dq.page_attention(kv, s, q, B.heads(out), page_lse, chosen, 12, c.scale, work, work.numel(), stream())
        dq.shared_attention(kv, q, B.heads(dense), lse, c.tokens, 2, c.offsets_d, c.max_q, None, 0, c.table, c.table.stride(0), c.lens_d, c.most,
                            c.scale, work, work.numel(), stream())
        lse.masked_fill_(dead, -math.inf)
        dq.attention_mass(kv, s, q, lse, c.scale, 0.5, mass, 1400, 700, work, work.numel(), stream())

    run()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        run()
    for i in range(4):
        c.q.normal_()
        if i == 2:  # (every row scores -inf on it)
            c.q[..., 3] = c.q[..., 3].abs() + 0.5
            c.kc[int(c.table[0, 2]), 1, 0, 3] = -math.inf
        got = []
        for go in (run, graph.replay):
            mass.fill_(0.25)
            torch.cuda.synchronize()
            go()
            torch.cuda.synchronize()
            got.append([x.clone() for x in (bounds, chosen, out, page_lse, mass)])
        assert_same(*got)


def test_calls_run_on_their_stream(cuda):
    """On a stream of their own, behind work that it waits for; another cycle on another stream at the same time."""
    plain = Cycle(53, "bf16", "bf16")
    plain.run()
    want = plain.results()
    sides = [torch.cuda.Stream() for _ in range(2)]
    cycles = [Cycle(53, "bf16", "bf16") for _ in range(2)]
    queries = [y.c.q.clone() for y in cycles]
    torch.cuda.synchronize()
    for y, q, side in zip(cycles, queries, sides):
        with torch.cuda.stream(side):
            y.c.q.zero_()
            big = torch.randn((4096, 4096), device="cuda")
            for _ in range(20):
                big = big @ big * 1e-4
            y.c.q.copy_(q)
            y.run()
    for side in sides:
        side.synchronize()
    for y in cycles:
        assert_same(y.results(), want)


def test_bounds_above_the_lengths(cuda):
    """max_len and max_q may be above what the sequences have."""
    c = Call(54, [1, 3, 2], [30, 141, 2], 8, 2, 128, "f16", "f16", 16)
    wide = torch.full((3, 200), 2**31 - 1, dtype=torch.int32, device="cuda")
    wide[:, : c.table.shape[1]] = c.table
    c.table = wide
    kw = dict(max_len=3000, max_q=64)
    bounds = L.run_bounds(c, max_new=3000, **kw)
    L.same(bounds, L.page_bounds(c, None, torch.full_like(bounds, 55.0).cpu()))
    chosen = L.run_choose(c, bounds, 1, 1, 5, **kw)
    assert torch.equal(chosen.cpu(), L.choose(c, bounds, 1, 1, 5))
    L.check_attention(c, chosen, **kw)
    lse = own_lse(c)
    got = L.run_mass(c, lse, torch.zeros((3, 2, 3000), device="cuda"), 0.0, **kw)
    want, bound = L.mass(c, lse, torch.zeros((3, 2, 3000)), 0.0)
    B.close(got, want, bound, "f32")


def test_offsets_and_lengths_of_any_values_stay_inside(cuda):
    """Offsets that decrease or leave the tokens, lengths of any value: nothing past the tensors' ends is touched."""
    c = Call(55, [3, 0, 5, 1, 2, 4, 2], [n + 40 for n in [3, 0, 5, 1, 2, 4, 2]], 8, 2, 64, "bf16", "bf16", 16)
    gen = torch.Generator().manual_seed(5)
    c.table = torch.randint(-3, c.kc.shape[0] + 3, c.table.shape, generator=gen).to(torch.int32).cuda()
    t, wide = c.tokens, torch.full((c.tokens + 20, 8, 64), 55.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((t + 20, 8), 33.0, device="cuda")
    lists = torch.full((t + 20, 2, 4), 77, dtype=torch.int32, device="cuda")
    mass = torch.full((9, 2, 50), 33.0, device="cuda")
    bounds = torch.full((c.kc.shape[0] + 2, 2, 2, 64), 44.0, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros_like(wide)
    q[10:-10] = c.q
    c.q = q[10:-10]
    work = torch.empty(dq.ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    for low, high in ((-(2**31), 2**31 - 1), (-5, t + 5)):
        c.offsets_d = torch.randint(low, high, (8,), generator=gen).to(torch.int32).cuda()
        c.lens_d = torch.randint(low, high, (7,), generator=gen).to(torch.int32).cuda()
        cache, s, heads = c.c(), c.seqs(max_len=44), B.heads(c.q)
        from_ = torch.randint(low, high, (7,), generator=gen).to(torch.int32).cuda()
        dq.page_bounds(cache, s, from_, 9, bounds[1:-1], stream())
        dq.choose_pages(cache, s, heads, bounds[1:-1], 0, 1, 2, lists[10:-10].view(-1)[: t * 4], work, work.numel(), stream())
        lists[10:-10].random_(-4, 6)
        dq.page_attention(cache, s, heads, B.heads(wide[10:-10]), lse[10:-10], lists[10:-10], 4, 0.1, work, work.numel(), stream())
        dq.attention_mass(cache, s, heads, lse[10:-10], 0.1, 0.5, mass[1:-1], 100, 50, work, work.numel(), stream())
        torch.cuda.synchronize()
        for x, value, n in ((wide, 55.0, 10), (lse, 33.0, 10), (lists, 77, 10), (mass, 33.0, 1), (bounds, 44.0, 1)):
            assert torch.all(x[:n] == value) and torch.all(x[-n:] == value)
        assert torch.all(mass[..., 44:] == 33.0)


@pytest.mark.parametrize("count", [1, 3])
def test_no_keys_at_all(cuda, count):
    """max_len 0 and a cache without pages: no page is chosen, rows are zeros, nothing is kept."""
    cache = dq.KvCache(None, None, dq.F16, 2, 64, 16, 0, 0, 64, 64)
    s = dq.Sequences(3, 3, None, 1, None, 0, None, 0)
    q, out = torch.randn((3, 4, 64), device="cuda"), torch.full((3, 4, 64), 55.0, device="cuda")
    lse, chosen = torch.full((3, 4), 33.0, device="cuda"), torch.full((3, 2, count), 77, dtype=torch.int32, device="cuda")
    kept, kept_lens = torch.full((3, 2, 5), 77, dtype=torch.int32, device="cuda"), torch.full((3,), 77, dtype=torch.int32, device="cuda")
    dq.page_bounds(cache, s, None, 0, None, stream())
    dq.choose_pages(cache, s, B.heads(q), None, 0, 1, count, chosen, None, 0, stream())
    dq.page_attention(cache, s, B.heads(q), B.heads(out), lse, chosen, count, 0.1, None, 0, stream())
    dq.attention_mass(cache, s, B.heads(q), lse, 0.1, 0.5, None, 0, 0, None, 0, stream())
    dq.kv_keep(s, 2, None, 0, 0, 1, 1, 5, kept, kept_lens, stream())
    dq.kv_compact(cache, s, kept, 5, stream=stream())
    assert torch.all(chosen == -1) and torch.all(out == 0) and torch.all(lse == -math.inf)
    assert torch.all(kept == -1) and torch.all(kept_lens == 0)


def test_a_list_that_ends_with_the_last_sequence(cuda):
    """Of the last sequence only the page numbers that hold keys need exist: what lies behind the list changes nothing."""
    c = Call(71, [1, 1], [900, 200], 4, 2, 64, "f16", "f16", 16)
    stride = c.table.stride(0)
    flat = torch.full((stride + 13 + 64,), 2**31 - 1, dtype=torch.int32, device="cuda")
    flat[: stride + 13] = c.table.reshape(-1)[: stride + 13]
    c.table = flat.as_strided((2, 13), (stride, 1))
    bounds = L.run_bounds(c)
    chosen = L.run_choose(c, bounds, 1, 1, 6)
    flat[stride + 13 :] = 0
    again = L.run_choose(c, bounds, 1, 1, 6)
    first = Call(71, [1, 1], [900, 200], 4, 2, 64, "f16", "f16", 16)
    assert torch.equal(chosen, again) and torch.equal(chosen.cpu(), L.choose(first, bounds, 1, 1, 6))


def test_decay_of_sequences_without_rows(cuda):
    """No rows at all: every key's weight decays."""
    c = Call(72, [0, 0], [50, 20], 2, 1, 64, "f32", "f16", 16)
    old = torch.rand((2, 1, 50), device="cuda")
    s = dq.Sequences(2, 0, c.offsets_d.data_ptr(), 1, c.table.data_ptr(), c.table.stride(0), c.lens_d.data_ptr(), 50)
    got = old.clone()
    q = dq.Heads(None, dq.F32, 2, 128, 64)
    dq.attention_mass(c.c(), s, q, None, 0.1, 0.5, got, 50, 50, None, 0, stream())
    want = old.clone()
    want[0] *= 0.5
    want[1, :, :20] *= 0.5
    assert torch.equal(got, want)


@pytest.mark.parametrize("type,cache", KINDS)
def test_pages_of_more_keys_than_any_sequence(cuda, type, cache):
    """A page holds a sequence's whole cache, most of it never written."""
    hk, dim, page = 2, 64, 1 << 16
    c = Call(73, [1, 2, 1], [40, 33, 700], 4, hk, dim, type, cache, page)
    assert c.kc.shape[0] == 4 and c.pages == 1
    bounds = L.run_bounds(c)
    L.same(bounds, L.page_bounds(c, None, torch.full_like(bounds, 55.0).cpu()))
    chosen = L.run_choose(c, bounds, 0, 1, 2)
    assert chosen.tolist() == [[[0, -1]] * hk] * 4
    L.check_attention(c, chosen)
    L.check_attention(c, torch.tensor([0, -1, 0, 5], dtype=torch.int32).repeat(4, hk, 1))
    lse = own_lse(c)
    got = L.run_mass(c, lse, torch.zeros((3, hk, 700), device="cuda"), 0.0)
    want, bound = L.mass(c, lse, torch.zeros((3, hk, 700)), 0.0)
    B.close(got, want, bound, "f32")
    kept = lists(c, 30)
    dq.kv_compact(c.c(), c.seqs(), kept.cuda(), 30, stream=stream())
    for b in range(3):
        for h in range(hk):
            assert torch.equal(c.kc[int(c.table[b, 0]), :30, h].cpu(), c.ks[b][kept[b, h].long(), h])
