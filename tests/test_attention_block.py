"""The attention block's refusals: arguments are checked before any GPU work (CPU only)."""
from __future__ import annotations

import ctypes as C

import pytest

import dynalm_amd as dq

AT = 1 << 20  # a device address that no call here reads


def heads(**kw):
    return dq.Heads(**{"p": AT, "dtype": dq.F32, "heads": 4, "token_stride": 4 * 64, "head_stride": 64, **kw})


def cache(**kw):
    return dq.KvCache(**{"k": AT, "v": AT, "dtype": dq.F16, "kv_heads": 2, "head_dim": 64, "page_size": 16, "n_pages": 8,
                         "page_stride": 16 * 128, "token_stride": 128, "head_stride": 64, **kw})


def rope(**kw):
    return dq.Rope(**{"cos": AT, "sin": AT, "max_pos": 100, "rot_dim": 64, "style": dq.ROPE_HALVES, **kw})


def refused(status, call, *a, **kw):
    with pytest.raises(dq.DqError) as e:
        call(*a, **kw)
    assert e.value.status == status, e.value
    assert str(e.value).split(": ", 1)[1]


def test_struct_sizes_are_the_headers():
    assert (C.sizeof(dq.Heads), C.sizeof(dq.Rope), C.sizeof(dq.KvCache), C.sizeof(dq.Attention)) == (32, 32, 64, 112)


def test_norm_rope_refusals():
    f = dq.qk_norm_rope
    f(0, 64, heads(p=None), heads(p=None))  # no tokens: nothing is read
    bad = "invalid_argument"
    refused(bad, f, -1, 64, heads(), heads())
    refused(bad, f, 2, 60, heads(), heads())
    refused(bad, f, 2, 0, heads(), heads())
    refused("unsupported", f, 2, 264, heads(token_stride=2000, head_stride=264), heads(token_stride=2000, head_stride=264))
    refused(bad, f, 2, 64, None, heads())
    refused(bad, f, 2, 64, heads(), None)
    refused(bad, f, 2, 64, heads(), heads(), None, heads(), None)
    refused(bad, f, 2, 64, heads(p=None), heads())
    refused(bad, f, 2, 64, heads(p=AT + 2), heads())
    refused(bad, f, 2, 64, heads(heads=0), heads(heads=0))
    refused(bad, f, 2, 64, heads(), heads(heads=3))
    refused(bad, f, 2, 64, heads(token_stride=-1), heads())
    refused(bad, f, 2, 64, heads(), heads(head_stride=63))
    refused(bad, f, 2, 64, heads(), heads(token_stride=200))  # outputs that overlap
    refused("unsupported", f, 2, 64, heads(dtype=7), heads())
    refused("unsupported", f, 2, 64, heads(), heads(), None, heads(dtype=dq.F16), heads())
    refused("unsupported", f, 1 << 40, 64, heads(), heads())
    refused(bad, f, 2, 64, heads(), heads(), AT, eps=float("nan"))
    refused(bad, f, 2, 64, heads(), heads(), AT, eps=-1.0)
    for r in (rope(rot_dim=66), rope(rot_dim=0), rope(rot_dim=7), rope(style=2), rope(max_pos=-1), rope(cos=None)):
        refused(bad, f, 2, 64, heads(), heads(), rope=r, positions=AT)
    refused(bad, f, 2, 64, heads(), heads(), rope=rope())  # no positions


def test_append_refusals():
    f = dq.kv_append
    kv = heads(heads=2, token_stride=128)
    f(cache(), 0, kv, kv, None)
    bad = "invalid_argument"
    refused(bad, f, None, 2, kv, kv, AT)
    refused(bad, f, cache(), -1, kv, kv, AT)
    refused(bad, f, cache(), 2, heads(heads=3), kv, AT)
    refused(bad, f, cache(), 2, kv, None, AT)
    refused(bad, f, cache(), 2, kv, kv, None)
    refused("unsupported", f, cache(), 2, kv, heads(heads=2, dtype=dq.F16), AT)
    refused("unsupported", f, cache(dtype=dq.F32), 2, kv, kv, AT)
    for c in (cache(k=None), cache(v=AT + 8), cache(page_size=24), cache(page_size=0), cache(head_dim=60), cache(n_pages=-1),
              cache(token_stride=132), cache(page_stride=-8), cache(kv_heads=0), cache(head_stride=56), cache(token_stride=0)):
        refused(bad, f, c, 2, kv, kv, AT)
    refused(bad, f, cache(), 2, kv, kv, AT, AT, float("inf"))
    refused(bad, f, cache(), 2, kv, kv, AT, rope=rope())


def attend(c=None, q=None, out=None, **kw):
    a = {"lse": None, "tokens": 3, "batch": 3, "q_offsets": AT, "max_q": 1, "prefix_pages": AT, "prefix_len": 20, "pages": AT,
         "pages_stride": 4, "lens": AT, "max_len": 40, "scale": 0.125, "workspace": AT, "workspace_bytes": 128 << 20, **kw}
    dq.shared_attention(c if c is not None else cache(), q if q is not None else heads(), out if out is not None else heads(), *a.values())


def test_attention_refusals():
    attend(tokens=0, batch=0)  # nothing to do
    bad = "invalid_argument"
    for kw in ({"tokens": -1}, {"batch": -1}, {"max_q": 0}, {"prefix_len": -1}, {"prefix_pages": None}, {"pages": None},
               {"lens": None}, {"pages_stride": 2}, {"max_len": -1}, {"max_len": 65}, {"scale": 0.0}, {"scale": -1.0},
               {"scale": float("inf")}, {"scale": float("nan")}, {"q_offsets": None, "tokens": 4}, {"q_offsets": None, "max_q": 2}):
        refused(bad, attend, **kw)
    refused(bad, attend, q=heads(heads=3), out=heads(heads=3))  # not a multiple of the kv heads
    refused(bad, attend, q=heads(heads=2))
    refused(bad, attend, q=heads(p=None))
    refused(bad, attend, out=heads(p=None))
    refused(bad, attend, out=heads(token_stride=100))
    refused("unsupported", attend, q=heads(dtype=dq.F16), out=heads())
    refused("unsupported", attend, q=heads(dtype=dq.BF16), out=heads(dtype=dq.BF16))
    refused(bad, attend, c=cache(page_size=8))
    refused(bad, attend, c=cache(n_pages=0))
    refused(bad, attend, workspace=None)
    refused(bad, attend, workspace=AT + 8)
    refused("resource_exhausted", attend, workspace_bytes=1000)
    refused("unsupported", attend, c=cache(token_stride=1 << 26))
    refused("unsupported", attend, tokens=1 << 29, batch=1, max_q=1)
    refused("unsupported", attend, batch=1 << 30)


def test_workspace_needs_no_pointers_and_has_a_bound():
    for tokens, batch, max_q in ((1, 1, 1), (64, 64, 1), (4096, 1, 4096), (300, 7, 100), (20000, 40, 512)):
        for dim in (64, 128, 256):
            for type in (dq.F32, dq.F16):
                for prefix, most in ((0, 1), (100, 0), (8192, 512), (1 << 20, 1 << 16)):
                    c = cache(k=None, v=None, head_dim=dim, token_stride=2 * dim, head_stride=dim, page_stride=32 * dim)
                    q = heads(p=None, dtype=type, token_stride=4 * dim, head_stride=dim)
                    n = dq.shared_attention_workspace(c, q, q, tokens, batch, max_q, prefix, 1 << 20, most)
                    assert 0 <= n <= dq.ATTENTION_WORKSPACE_BYTES
    with pytest.raises(dq.DqError):
        dq.shared_attention_workspace(cache(), heads(), heads(), 1, 1, 0, 0, 1, 1)


def test_heads_of_a_token_run_in_one_launch():
    """A launch counts its threads in 32 bits: 2^26 heads of one token are over that, refused and not tried."""
    many = {"heads": 1 << 26, "token_stride": 64 << 26}
    refused("unsupported", dq.qk_norm_rope, 1, 64, heads(**many), heads(**many))
    kv = heads(**{"heads": 1 << 25, "token_stride": 64 << 25})
    refused("unsupported", dq.kv_append, cache(kv_heads=1 << 25, token_stride=64 << 25, page_stride=64 << 29), 1, kv, kv, AT)


def test_append_refuses_caches_whose_places_overlap():
    """Two rows would be written to one address; which layouts are apart is counted place by place."""

    def apart(c):
        base = [c.k // 2 + p * c.page_stride + i * c.token_stride + h * c.head_stride
                for p in range(c.n_pages) for i in range(c.page_size) for h in range(c.kv_heads)]
        at = sorted(base + [x + (c.v - c.k) // 2 for x in base])
        return all(b - a >= c.head_dim for a, b in zip(at, at[1:]))

    n, kinds = 3 * 16 * 2 * 64, set()
    for kv, page, token, head in ((2, 16 * 128, 128, 64), (2, 16 * 128, 64, 1024), (2, 64, 3 * 128, 3 * 64), (2, 64, 192, 192 * 16),
                                  (2, 2048, 64, 64), (2, 1024, 128, 64), (2, 16 * 128, 96, 64), (1, 16 * 64, 64, 8), (1, 16 * 64, 64, 64),
                                  (2, 16 * 256, 256, 64), (2, 16 * 256, 256, 128), (2, 64, 64, 64), (2, 2040, 128, 64), (2, 2 * 2048, 128, 64)):
        for d in (n, 2 * n + 8, 0, 8, 56, 64, 128, 2048, -2048, 1024, -64, -n, 2048 + 64, 4 * n, 192):
            c = cache(v=AT + 2 * d, kv_heads=kv, n_pages=3, page_stride=page, token_stride=token, head_stride=head)
            rows = heads(heads=kv, token_stride=128)
            with pytest.raises(dq.DqError) as e:
                dq.kv_append(c, 1, rows, rows, None)  # (a layout that passes is refused for its slots)
            assert ("slots" if apart(c) else "overlap") in str(e.value), (page, token, head, d)
            assert e.value.status == "invalid_argument"
            kinds.add(apart(c))
    assert kinds == {True, False}


def test_large_batches_go_on_sharing_the_prefix():
    """More rows than the workspace holds parts of: the batch runs in slices, whose parts are counted here (32 / 8 heads
    of 128; two parts a row of 32 x 130 floats)."""
    c = cache(k=None, v=None, kv_heads=8, head_dim=128, token_stride=1024, head_stride=128, page_stride=1 << 14)
    q = heads(p=None, dtype=dq.F16, heads=32, token_stride=4096, head_stride=128)
    for tokens, batch, max_q, a_slice in ((4000, 4000, 1, 4000), (4096, 4096, 1, 2048), (4096, 1024, 4, 2048), (4096, 512, 8, 2048),
                                          (20000, 20000, 1, 4000), (5000, 1500, 7, 500 * 7)):
        n = dq.shared_attention_workspace(c, q, q, tokens, batch, max_q, 8192, 64, 512)
        assert n == 2 * a_slice * 32 * 130 * 4 <= dq.ATTENTION_WORKSPACE_BYTES, (tokens, batch, max_q, n)


def test_a_sequence_runs_in_one_launch():
    """2^24 workgroups have more threads than a launch counts: 128 tokens of 2^23 kv heads are refused, not tried."""
    kv = 1 << 23
    c = cache(kv_heads=kv, token_stride=64, head_stride=1024, page_stride=1024 * kv)
    q = heads(dtype=dq.F16, heads=kv, token_stride=64 * kv)
    with pytest.raises(dq.DqError, match="too many for a launch"):
        dq.shared_attention_workspace(c, q, q, 128, 1, 128, 0, 8, 128)


def test_the_workspace_query_is_refused_with_the_calls_status():
    def ask(q=heads(), most=16):
        return dq.shared_attention_workspace(cache(), q, q, 1, 1, 1, 0, 1, most)

    assert ask() == 0
    refused("invalid_argument", ask, most=17)
    refused("unsupported", ask, q=heads(dtype=7))
