"""The long caches' refusals and workspaces: arguments are checked before any GPU work (CPU only)."""
from __future__ import annotations

import ctypes as C

import pytest

import dynalm_amd as dq
from test_attention_block import AT, cache, heads, refused

BAD, NO = "invalid_argument", "unsupported"


def seqs(**kw):
    return dq.Sequences(**{"batch": 3, "tokens": 3, "q_offsets": AT, "max_q": 1, "pages": AT, "pages_stride": 4, "lens": AT, "max_len": 40, **kw})


def test_struct_size_is_the_headers():
    assert C.sizeof(dq.Sequences) == 64


def bounds(c=None, s=None, from_=AT, max_new=5, out=AT):
    dq.page_bounds(c or cache(), s or seqs(), from_, max_new, out)


def choose(c=None, s=None, q=None, bounds=AT, first=0, last=1, count=2, chosen=AT, workspace=AT, bytes=128 << 20):
    dq.choose_pages(c or cache(), s or seqs(), q or heads(), bounds, first, last, count, chosen, workspace, bytes)


def attend(c=None, s=None, q=None, out=None, lse=None, chosen=AT, count=2, scale=0.125, workspace=AT, bytes=128 << 20):
    dq.page_attention(c or cache(), s or seqs(), q or heads(), out or heads(), lse, chosen, count, scale, workspace, bytes)


def mass(c=None, s=None, q=None, lse=AT, scale=0.125, decay=0.5, out=AT, seq=80, head=40, workspace=AT, bytes=128 << 20):
    dq.attention_mass(c or cache(), s or seqs(), q or heads(), lse, scale, decay, out, seq, head, workspace, bytes)


def keep(s=None, kv=2, weights=AT, seq=80, head=40, first=0, last=0, budget=10, kept=AT, lens=None):
    dq.kv_keep(s or seqs(), kv, weights, seq, head, first, last, budget, kept, lens)


def compact(c=None, s=None, kept=AT, budget=10, to=None, to_stride=0, weights=AT, out=AT, seq=80, head=40):
    dq.kv_compact(c or cache(v=AT + 2 * 8 * 2048), s or seqs(), kept, budget, to, to_stride, weights, out, seq, head)


ALL = [bounds, choose, attend, mass, keep, compact]


@pytest.mark.parametrize("call", ALL)
def test_no_sequences_are_no_work(call):
    call(s=seqs(batch=0, tokens=0, max_len=0))


@pytest.mark.parametrize("call", ALL)
def test_sequences_that_are_refused(call):
    for kw in ({"batch": -1}, {"batch": 1 << 31}, {"max_len": -1}, {"max_len": (1 << 29) + 1, "pages_stride": 1 << 29}, {"lens": None}):
        refused(BAD, call, s=seqs(**kw))
    if call is not keep:
        for kw in ({"pages": None}, {"pages_stride": 2}, {"max_len": 65}, {"pages_stride": 1 << 30}):
            refused(BAD, call, s=seqs(**kw))
        for kw in ({"page_size": 8}, {"page_size": 24}, {"head_dim": 60}, {"kv_heads": 0}, {"token_stride": -8}, {"n_pages": -1}, {"n_pages": 0}):
            refused(BAD, call, c=cache(**{"v": AT + 2 * 8 * 2048, **kw}))
        refused(NO, call, c=cache(dtype=dq.F32, v=AT + 2 * 8 * 2048))
    if call in (choose, attend, mass):
        for kw in ({"tokens": -1}, {"max_q": 0}, {"q_offsets": None, "tokens": 4}, {"q_offsets": None, "max_q": 2}):
            refused(BAD, call, s=seqs(**kw))
        refused(BAD, call, q=heads(heads=3))
        refused(BAD, call, q=heads(p=None))
        refused(BAD, call, q=heads(p=AT + 2))
        refused(NO, call, q=heads(dtype=dq.BF16))  # (the cache is f16)
        refused(NO, call, q=heads(dtype=7))


@pytest.mark.parametrize("call", [bounds, choose, attend, mass, keep, compact])
def test_null_sequences_and_caches(call):
    class Null:
        def __bool__(self):
            return True

    with pytest.raises((dq.DqError, C.ArgumentError)):
        call(s=Null())


def test_bounds_refusals():
    bounds(max_new=0)  # no new keys
    refused(BAD, bounds, max_new=-1)
    refused(BAD, bounds, out=None)
    refused(BAD, bounds, out=AT + 8)
    refused(BAD, bounds, c=cache(k=None))
    refused(BAD, bounds, c=cache(k=AT + 8))


def test_choose_refusals():
    for kw in ({"bounds": None}, {"bounds": AT + 8}, {"first": -1}, {"last": 0}, {"count": 0}, {"first": 2, "last": 1}, {"last": 3}, {"chosen": None},
               {"workspace": None}, {"workspace": AT + 8}, {"first": 1 << 62, "last": 1 << 62}, {"count": 1 << 40}):
        refused(BAD, choose, **kw)
    refused("resource_exhausted", choose, bytes=3 * 2 * 3 * 8 - 1)
    # one row's scores of a launch: 2^26 pages of 2 heads in 64 bits are over the workspace
    refused(NO, choose, s=seqs(max_len=1 << 29, pages_stride=1 << 29))


def test_attend_refusals():
    for kw in ({"out": heads(p=None)}, {"out": heads(token_stride=100)}, {"out": heads(heads=2)}, {"chosen": None}, {"count": 0}, {"count": -5},
               {"scale": 0.0}, {"scale": float("nan")}, {"scale": float("inf")}, {"c": cache(v=None)}, {"c": cache(v=AT + 8)}):
        refused(BAD, attend, **kw)
    refused(NO, attend, out=heads(dtype=dq.F16))
    refused(NO, attend, c=cache(token_stride=1 << 26))
    refused(NO, attend, c=cache(page_size=(1 << 24) + 16, page_stride=1 << 31))
    refused(NO, attend, s=seqs(tokens=1 << 29, batch=1 << 29))
    refused(NO, attend, s=seqs(tokens=1 << 24, batch=1 << 24), q=heads(heads=2), out=heads(heads=2))
    many = {"s": seqs(max_len=3000, pages_stride=200), "count": 100}
    for kw, status in (({"workspace": None}, BAD), ({"workspace": AT + 8}, BAD), ({"bytes": 1000}, "resource_exhausted")):
        refused(status, attend, **many, **kw)


def test_mass_refusals():
    for kw in ({"lse": None}, {"scale": -1.0}, {"decay": -0.1}, {"decay": 1.5}, {"decay": float("nan")}, {"out": None}, {"out": AT + 2}, {"seq": 39, "head": 40},
               {"seq": 79}, {"head": 39}, {"seq": -80}, {"seq": 40, "head": 119}, {"head": 1 << 60}, {"c": cache(k=None)}, {"c": cache(k=AT + 8)}):
        refused(BAD, mass, **kw)
    refused(NO, mass, c=cache(token_stride=1 << 26))
    refused(NO, mass, s=seqs(batch=1 << 23, max_len=1 << 10, pages_stride=64, tokens=4), seq=1 << 11, head=1 << 10)
    prompt = {"s": seqs(tokens=3000, max_q=1000, max_len=3000, pages_stride=200), "seq": 6000, "head": 3000}
    for kw, status in (({"workspace": None}, BAD), ({"workspace": AT + 8}, BAD), ({"bytes": 1000}, "resource_exhausted")):
        refused(status, mass, **prompt, **kw)


def test_keep_refusals():
    for kw in ({"kv": 0}, {"weights": None}, {"weights": AT + 1}, {"first": -1}, {"last": -1}, {"budget": 0}, {"first": 6, "last": 5}, {"kept": None},
               {"seq": 79}, {"first": 1 << 62, "last": 1 << 62}):
        refused(BAD, keep, **kw)
    refused(NO, keep, kv=1 << 22, seq=1 << 40)


def test_compact_refusals():
    for kw in ({"kept": None}, {"budget": 0}, {"to": AT, "to_stride": 0}, {"budget": 40, "to": AT, "to_stride": 2}, {"weights": None}, {"out": None},
               {"weights": AT + 2}, {"out": AT + 2}, {"seq": 79}, {"c": cache(k=None)}, {"c": cache(v=None)}, {"c": cache(v=AT + 8)}):
        refused(BAD, compact, **kw)
    refused(BAD, compact, c=cache(v=AT + 64))  # keys and values overlap
    refused(BAD, compact, c=cache(head_stride=0, v=AT + 2 * 8 * 2048))


def test_workspaces_have_a_bound():
    for batch, tokens, max_q in ((1, 1, 1), (64, 64, 1), (1, 4096, 4096), (7, 300, 100), (40, 20000, 512)):
        for dim in (64, 256):
            for most in (1, 100, 16384, 1 << 20):
                for kv, group in ((1, 1), (8, 4), (2, 40)):
                    c = cache(k=None, v=None, kv_heads=kv, head_dim=dim, token_stride=kv * dim, head_stride=dim, page_stride=16 * kv * dim)
                    s = seqs(batch=batch, tokens=tokens, max_q=max_q, max_len=most, pages_stride=1 << 17, q_offsets=None, pages=None, lens=None)
                    q = heads(p=None, heads=kv * group, token_stride=kv * group * dim, head_stride=dim)
                    for n in (dq.choose_pages_workspace(c, s), dq.attention_mass_workspace(c, s, q),
                              *(dq.page_attention_workspace(c, s, q, count) for count in (1, 64, 100000))):
                        assert 0 <= n <= dq.ATTENTION_WORKSPACE_BYTES


def test_the_workspace_queries_are_refused_with_the_calls_status():
    c, s, q = cache(), seqs(max_len=65), heads(dtype=7)
    refused(BAD, dq.choose_pages_workspace, c, s)
    refused(BAD, dq.page_attention_workspace, c, s, heads(), 2)
    refused(BAD, dq.attention_mass_workspace, c, s, heads())
    refused(NO, dq.page_attention_workspace, c, seqs(), q, 2)
    refused(NO, dq.attention_mass_workspace, c, seqs(), q)
