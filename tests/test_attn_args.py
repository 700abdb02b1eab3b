"""What the cache, attention and adapter entry points refuse: every call here is
rejected on the host, before any launch, so this runs without a GPU."""
import ctypes as C

import pytest

import qfm

P = 1 << 20                                          # an aligned address that nothing follows


@pytest.fixture
def lib():
    lib = qfm.load()
    lib.qfm_last_error()
    return lib


def _cache(**kw):
    a = dict(k=P, v=P, ks=P, vs=P, n_pages=8, page=16, kv_heads=2, head_dim=128, fmt=0)
    a.update(kw)
    return qfm.QfmKvCache(*a.values())


def _seqs(**kw):
    a = dict(table=P, n_seq=2, max_pages=3)
    a.update(kw)
    return qfm.QfmKvSeqs(*a.values())


BAD_CACHES = [dict(k=None), dict(v=None), dict(ks=None), dict(vs=None), dict(n_pages=0), dict(n_pages=-1), dict(page=8),
              dict(page=48), dict(page=512), dict(page=0), dict(page=-16), dict(kv_heads=0), dict(kv_heads=1025), dict(head_dim=96),
              dict(head_dim=512), dict(head_dim=0), dict(fmt=2), dict(fmt=-1), dict(k=P + 8), dict(v=P + 1), dict(ks=P + 4), dict(vs=P + 2)]
BAD_SEQS = [dict(table=None), dict(n_seq=0), dict(n_seq=65536), dict(max_pages=0)]


def _rows_call(lib, name, cache, seqs, **kw):
    a = dict(k=P, v=P, dtype=1, rs=256, hs=128, seq=P, pos=P, T=4)
    a.update(kw)
    rc = getattr(lib, name)(C.byref(cache) if cache else None, C.byref(seqs) if seqs else None, *a.values(), None)
    return rc, lib.qfm_last_error()


@pytest.mark.parametrize("name", ["qfm_kv_write", "qfm_kv_read"])
def test_rows_refuse(lib, name):
    for bad in BAD_CACHES:
        rc, msg = _rows_call(lib, name, _cache(**bad), _seqs())
        assert rc == -1 and name.encode() in msg, bad
    for bad in BAD_SEQS:
        rc, msg = _rows_call(lib, name, _cache(), _seqs(**bad))
        assert rc == -1 and name.encode() in msg, bad
    for bad in (dict(dtype=3), dict(dtype=-1), dict(rs=-8), dict(hs=-8), dict(rs=252), dict(hs=129), dict(seq=None),
                dict(pos=None), dict(T=-1), dict(T=(1 << 24) + 1), dict(k=P + 8), dict(v=P + 2), dict(k=None, v=None)):
        rc, msg = _rows_call(lib, name, _cache(), _seqs(), **bad)
        assert rc == -1 and name.encode() in msg, bad
    for c, s in ((None, _seqs()), (_cache(), None)):
        assert _rows_call(lib, name, c, s)[0] == -1
    assert _rows_call(lib, name, _cache(), _seqs(), T=0)[0] == 0      # nothing to do


def test_write_needs_both_rows_and_read_rows_apart(lib):
    assert _rows_call(lib, "qfm_kv_write", _cache(), _seqs(), k=None)[0] == -1
    assert _rows_call(lib, "qfm_kv_write", _cache(), _seqs(), v=None)[0] == -1
    # results that would lie on each other
    assert _rows_call(lib, "qfm_kv_read", _cache(), _seqs(), rs=0)[0] == -1
    assert _rows_call(lib, "qfm_kv_read", _cache(), _seqs(), hs=120)[0] == -1


def test_struct_layouts():
    assert C.sizeof(qfm.QfmKvCache) == 56 and qfm.QfmKvCache.fmt.offset == 48
    assert C.sizeof(qfm.QfmKvSeqs) == 16


def _attn_call(lib, cache=None, seqs=None, **kw):
    a = dict(q=P, out=P, dtype=1, q_heads=8, qrs=1024, qhs=128, ors=1024, ohs=128, start=P, ctx=P, tree=P, T=4, nodes=2,
             max_ctx=100, scale=0.1, ws=P, wsb=1 << 40)
    a.update(kw)
    rc = lib.qfm_tree_attn(C.byref(cache or _cache()), C.byref(seqs or _seqs()), *a.values(), None)
    return rc, lib.qfm_last_error()


def test_attention_refuses(lib):
    for bad in BAD_CACHES:
        rc, msg = _attn_call(lib, _cache(**bad))
        assert rc == -1 and b"qfm_tree_attn" in msg, bad
    for bad in BAD_SEQS:
        rc, msg = _attn_call(lib, seqs=_seqs(**bad))
        assert rc == -1 and b"qfm_tree_attn" in msg, bad
    for bad in (dict(q=None), dict(out=None), dict(start=None), dict(ctx=None), dict(q=P + 8), dict(out=P + 2), dict(tree=P + 4),
                dict(dtype=3), dict(q_heads=0), dict(q_heads=7), dict(q_heads=4098), dict(qrs=-8), dict(qhs=4), dict(ors=120),
                dict(ohs=0), dict(ohs=129), dict(T=-1), dict(T=(1 << 22) + 1), dict(nodes=0), dict(nodes=65), dict(max_ctx=-1),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        rc, msg = _attn_call(lib, **bad)
        assert rc == -1 and b"qfm_tree_attn" in msg, bad
    assert _attn_call(lib, T=0)[0] == 0


def test_attention_asks_for_its_workspace(lib):
    c = _cache()
    need = lib.qfm_tree_attn_ws_bytes(C.byref(c), 2, 4, 8, 2, 8000)
    assert need > 0 and lib.qfm_tree_attn_ws_bytes(C.byref(c), 2, 4, 8, 2, 0) == 0
    for bad in (dict(ws=None), dict(wsb=need - 1), dict(ws=P + 8), dict(wsb=0)):
        rc, msg = _attn_call(lib, max_ctx=8000, **bad)
        assert rc == -1 and b"workspace" in msg, bad
    for args in ((0, 4, 8, 2, 10), (2, -1, 8, 2, 10), (2, 4, 7, 2, 10), (2, 4, 8, 65, 10), (2, 4, 8, 0, 10), (2, 4, 8, 2, -1)):
        assert lib.qfm_tree_attn_ws_bytes(C.byref(c), *args) == 0
    assert lib.qfm_tree_attn_ws_bytes(None, 2, 4, 8, 2, 10) == 0


def _lora(**kw):
    l = qfm.QfmLora()
    l.n, l.K, l.R, l.slots, l.dtype, l.rank, l.scale = 2, 128, 16, 4, 1, P, P
    for i in range(2):
        l.a[i], l.b[i], l.base[i], l.y[i], l.rows[i] = P, P, P, P, 64
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(l, k)[v[0]] = v[1]
        else:
            setattr(l, k, v)
    return l


def _lora_call(lib, l, x=P, xs=128, slot=P, T=4, ws=P, wsb=1 << 30):
    return lib.qfm_lora_rows(C.byref(l) if l else None, x, xs, slot, T, ws, wsb, None), lib.qfm_last_error()


def test_adapters_refuse(lib):
    assert C.sizeof(qfm.QfmLora) == 184
    for bad in (dict(n=0), dict(n=5), dict(K=0), dict(K=96), dict(K=1 << 17), dict(R=0), dict(R=12), dict(R=136), dict(slots=0),
                dict(dtype=0), dict(dtype=3), dict(rank=None), dict(scale=None), dict(a=(1, None)), dict(b=(0, None)), dict(y=(1, None)),
                dict(rows=(0, 0)), dict(rows=(1, -5)), dict(rows=(0, (1 << 20) + 1)), dict(a=(0, P + 8)), dict(y=(0, P + 4)),
                dict(base=(1, P + 4))):
        rc, msg = _lora_call(lib, _lora(**bad))
        assert rc == -1 and b"qfm_lora_rows" in msg, bad
    for bad in (dict(x=None), dict(x=P + 2), dict(xs=-8), dict(xs=132), dict(slot=None), dict(T=-1), dict(T=(1 << 20) + 1),
                dict(ws=None), dict(wsb=4 * 2 * 16 * 4 - 1), dict(ws=P + 4)):
        rc, msg = _lora_call(lib, _lora(), **bad)
        assert rc == -1 and b"qfm_lora_rows" in msg, bad
    assert _lora_call(lib, None)[0] == -1
    assert _lora_call(lib, _lora(), T=0)[0] == 0
    l = _lora()
    assert lib.qfm_lora_ws_bytes(C.byref(l), 4) == 4 * 2 * 16 * 4 and lib.qfm_lora_ws_bytes(None, 4) == 0
    assert lib.qfm_lora_ws_bytes(C.byref(_lora(R=12)), 4) == 0
