"""GPU: the quantised key/value cache (qfm_kv_write, qfm_kv_read) against numpy,
codes and scales for equality and the whole pool, so that what no row names
stays as it was."""
import numpy as np
import pytest

import qfm
import _kv
from _kv import E4M3, INT8

pytestmark = pytest.mark.gpu


def _say(*a):
    print("[kv]", *a, flush=True)


def _rows(rng, T, H, D):
    x = rng.standard_normal((T, H, D)).astype(np.float32) * np.exp(rng.uniform(-3, 3, (T, H, 1))).astype(np.float32)
    x[:, :, :: max(1, D // 4)] *= 10
    return x


def _case(rng, T, n_seq, page, H, D, fmt, dt, layout):
    max_pages = -(-(T + 40) // page)
    c = _kv.Cache(n_seq * max_pages + 3, page, H, D, fmt, _kv.tables(rng, n_seq, max_pages, n_seq * max_pages + 3), rng)
    seq = np.sort(rng.integers(0, n_seq, T)).astype(np.int32)
    first = rng.integers(0, 40, n_seq)
    pos = np.array([first[s] + (seq[:t] == s).sum() for t, s in enumerate(seq)], np.int32)
    kb, k = _kv.to_dtype(_rows(rng, T, H, D), dt)
    vb, v = _kv.to_dtype(_rows(rng, T, H, D), dt)
    n, rs, hs = _kv.strided(T, H, D, layout)
    return c, seq, pos, (kb, k), (vb, v), n, rs, hs


def _write(lib, c, refs, kb, vb, n, rs, hs, dt, seq, pos, st):
    d = [qfm.DevBuf.from_array(_kv.scatter(b, n, rs, hs)[0]) for b in (kb, vb)] + [qfm.DevBuf.from_array(a) for a in (seq, pos)]
    qfm.check(lib.qfm_kv_write(*refs, d[0].ptr, d[1].ptr, qfm.QFM_DT[dt], rs, hs, d[2].ptr, d[3].ptr, len(seq), st.h), "write")
    st.sync()
    return d


def _same(c):
    for name, got in c.download().items():
        want = getattr(c, name)
        same = got.view(np.uint32) == want.view(np.uint32) if got.dtype == np.float32 else got == want
        same |= np.isnan(got) & np.isnan(want) if got.dtype == np.float32 else False
        assert same.all(), (name, int((~same).sum()), np.argwhere(~same)[:4].tolist())


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("T,n_seq,page,H,D,dt,layout", [
    (1, 1, 16, 1, 64, "f32", "rows"), (8, 1, 16, 2, 256, "f32", "rows"), (37, 5, 32, 4, 128, "bf16", "heads"),
    (133, 3, 64, 3, 64, "f16", "wide"), (301, 2, 256, 2, 128, "f16", "heads"), (64, 64, 128, 1, 256, "bf16", "wide"),
    (515, 1, 16, 5, 64, "f32", "wide")])
def test_write_and_read(fmt, T, n_seq, page, H, D, dt, layout):
    _say("fmt", fmt, "T", T, "seqs", n_seq, "page", page, "heads", H, "D", D, dt, layout)
    lib, rng, st = qfm.load(), np.random.default_rng(T * 7 + D + fmt), qfm.Stream()
    c, seq, pos, (kb, k), (vb, v), n, rs, hs = _case(rng, T, n_seq, page, H, D, fmt, dt, layout)
    refs = c.upload()
    d = _write(lib, c, refs, kb, vb, n, rs, hs, dt, seq, pos, st)
    c.put(k, v, seq, pos)
    _same(c)
    # back in every type, into a buffer whose other elements stay
    for out in ("f32", "bf16", "f16"):
        fill = _kv.to_dtype(np.float32(7.0), out)[0]
        bufs = [qfm.DevBuf.from_array(np.full(n, fill, _kv.NP[out])) for _ in range(2)]
        qfm.check(lib.qfm_kv_read(*refs, bufs[0].ptr, bufs[1].ptr, qfm.QFM_DT[out], rs, hs, d[2].ptr, d[3].ptr, T, st.h), "read")
        st.sync()
        rows = [c.row(int(s), int(p)) for s, p in zip(seq, pos)]
        for i in range(2):
            want64 = np.stack([r[i] for r in rows])
            want = _kv.to_dtype(want64.astype(np.float32), out)[0]       # code * scale has 32 bits at most: one rounding
            got = bufs[i].download(_kv.NP[out], n)
            flat, at = _kv.scatter(want, n, rs, hs, fill)
            assert np.array_equal(got, flat), (out, i)
    st.destroy()


@pytest.mark.parametrize("fmt", [INT8, E4M3])
def test_rows_that_do_not_exist_are_passed_over(fmt):
    lib, rng, st = qfm.load(), np.random.default_rng(5), qfm.Stream()
    page, H, D, T = 16, 2, 64, 24
    table = np.array([[3, 1, 99], [-1, 2, 0]], np.int32)                 # pages 99 and -1 are none of the 5
    c = _kv.Cache(5, page, H, D, fmt, table, rng)
    refs = c.upload()
    seq = np.array([0, 0, 0, 0, 1, 1, 1, 2, -1, 1 << 30] * 3, np.int32)[:T]
    pos = np.array([0, 47, 15, 48, 3, 17, -1, 0, 0, 0] * 3, np.int32)[:T]
    pos[10:] += np.where(pos[10:] >= 0, 1, 0)
    pos[20:] = [1 << 30, (1 << 31) - 1, -(1 << 31), 31]
    k, v = _rows(rng, T, H, D), _rows(rng, T, H, D)
    d = _write(lib, c, refs, k, v, T * H * D, H * D, D, "f32", seq, pos, st)
    c.put(k, v, seq, pos)
    _same(c)
    out = qfm.DevBuf.from_array(np.full((T, H, D), 3.0, np.float32))
    for which in (0, 1):                                                # keys alone, values alone
        args = (out.ptr, None) if which == 0 else (None, out.ptr)
        qfm.check(lib.qfm_kv_read(*refs, *args, 0, H * D, D, d[2].ptr, d[3].ptr, T, st.h), "read")
        st.sync()
        got = out.download(np.float32, (T, H, D))
        for t in range(T):
            r = c.row(int(seq[t]), int(pos[t]))
            want = np.full((H, D), 3.0) if r is None else r[which].astype(np.float32)
            assert np.array_equal(got[t], want), (which, t)
        out.upload(np.full((T, H, D), 3.0, np.float32))
    assert lib.qfm_kv_write(*refs, out.ptr, out.ptr, 0, H * D, D, d[2].ptr, d[3].ptr, 0, st.h) == 0     # no rows
    st.sync()
    _same(c)
    st.destroy()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fmt", [INT8, E4M3])
def test_values_at_the_ends_of_the_range(fmt, dt):
    """Zeros, the smallest and largest magnitudes, one value alone, NaN and infinities in a row."""
    lib, rng, st = qfm.load(), np.random.default_rng(11), qfm.Stream()
    D, H = 64, 1
    big = {"f32": 3.4e38, "bf16": 3.3e38, "f16": 65504.0}[dt]
    small = {"f32": 1.5e-45, "bf16": 1e-40, "f16": 6e-8}[dt]
    rows = [np.zeros(D), np.full(D, small), np.full(D, big), np.where(np.arange(D) == 5, -big, small), np.linspace(-1, 1, D),
            np.where(np.arange(D) == 63, np.nan, 1.0), np.where(np.arange(D) == 0, np.inf, 1.0),
            np.where(np.arange(D) == 9, -np.inf, np.nan), np.full(D, -0.0), np.arange(D) - 31.5, (np.arange(D) + 0.5) / 63.5 * 127,
            rng.standard_normal(D) * small * 50]
    with np.errstate(over="ignore"):
        bits, vals = _kv.to_dtype(np.array(rows, np.float32)[:, None, :], dt)
    T = len(rows)
    c = _kv.Cache(2, 16, H, D, fmt, np.array([[1]], np.int32), rng)
    refs = c.upload()
    seq, pos = np.zeros(T, np.int32), np.arange(T, dtype=np.int32)
    d = _write(lib, c, refs, bits, bits, T * D, D, D, dt, seq, pos, st)
    c.put(vals, vals, seq, pos)
    if fmt == E4M3:                                                    # -0.0 and 0 are the same value
        for x in (c.k, c.v):
            x[x == 128] = 0
        got = c.download()
        for n in ("k", "v"):
            g = got[n].copy()
            g[g == 128] = 0
            assert np.array_equal(g, getattr(c, n)), n
    else:
        _same(c)
    got = c.download()
    for n in ("ks", "vs"):
        a, b = got[n][1, 0, :T], getattr(c, n)[1, 0, :T]
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)]), n
    out = qfm.DevBuf(T * D * 4)
    qfm.check(lib.qfm_kv_read(*refs, out.ptr, None, 0, D, D, d[2].ptr, d[3].ptr, T, st.h), "read")
    st.sync()
    o = out.download(np.float32, (T, D))
    assert np.isnan(o[5:8]).all() and np.isfinite(np.delete(o, [5, 6, 7], 0)).all()
    st.destroy()


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_runs_of_every_length_and_alignment(fmt, D):
    """Rows whose positions begin and break anywhere: four tokens of a channel share a word of the value codes."""
    lib, rng, st = qfm.load(), np.random.default_rng(D + fmt), qfm.Stream()
    page, H, n_seq = 16, 2, 3
    for trial in range(6):
        seq, pos, at = [], [], [0] * n_seq
        while len(seq) < 61 + 5 * trial:
            s, n = int(rng.integers(0, n_seq)), int(rng.integers(1, 12))
            at[s] += int(rng.integers(0, 3))
            if rng.random() < 0.2:
                seq, pos = seq + [s], pos + [-1]                          # a row between that goes nowhere
            for i in range(n):
                seq, pos = seq + [s], pos + [at[s]]
                at[s] += 1
        if trial == 5:                                                    # backwards: no row continues another
            seq, pos = seq[::-1], pos[::-1]
        T = len(seq)
        seq, pos = np.array(seq, np.int32), np.array(pos, np.int32)
        max_pages = -(-max(at) // page)
        c = _kv.Cache(n_seq * max_pages, page, H, D, fmt, _kv.tables(rng, n_seq, max_pages, n_seq * max_pages), rng)
        if trial == 4:
            c.table[1, :] = -1
        refs = c.upload()
        k, v = _rows(rng, T, H, D), _rows(rng, T, H, D)
        v[5], k[9] = np.nan, np.inf
        _write(lib, c, refs, k, v, T * H * D, H * D, D, "f32", seq, pos, st)
        c.put(k, v, seq, pos)
        _same(c)
    st.destroy()


def test_pages_behind_four_gigabytes():
    """Codes whose offset needs more than 32 bits: the last pages of a pool of 4.4e9 bytes."""
    lib, rng, st = qfm.load(), np.random.default_rng(3), qfm.Stream()
    page, H, D, pages = 256, 8, 256, 8300
    per = page * H * D
    assert pages * per > 1 << 32
    k, v, ks, vs = (qfm.DevBuf(pages * n) for n in (per, per, page * H * 4, page * H * 4))
    table = qfm.DevBuf.from_array(np.array([[pages - 1, pages - 2]], np.int32))
    cc, sq = qfm.QfmKvCache(k.ptr, v.ptr, ks.ptr, vs.ptr, pages, page, H, D, INT8), qfm.QfmKvSeqs(table.ptr, 1, 2)
    T = 9
    x, seq, pos = _rows(rng, T, H, D), np.zeros(T, np.int32), np.arange(T, dtype=np.int32) + 251
    d = [qfm.DevBuf.from_array(a) for a in (x, seq, pos)]
    refs = (qfm.C.byref(cc), qfm.C.byref(sq))
    qfm.check(lib.qfm_kv_write(*refs, d[0].ptr, d[0].ptr, 0, H * D, D, d[1].ptr, d[2].ptr, T, st.h), "write")
    out = [qfm.DevBuf(T * H * D * 4) for _ in range(2)]
    qfm.check(lib.qfm_kv_read(*refs, out[0].ptr, out[1].ptr, 0, H * D, D, d[1].ptr, d[2].ptr, T, st.h), "read")
    st.sync()
    code, s = _kv.quantise(x, INT8)
    want = (_kv.CODE_VALUE[INT8][code] * s.astype(np.float64)[..., None]).astype(np.float32)
    for o in out:
        assert np.array_equal(o.download(np.float32, (T, H, D)), want)
    # rows 0..4 at the end of the last page, the others at the start of the one before it
    got = k.download(np.uint8, (H, page, D), (pages - 1) * per)
    assert np.array_equal(got[:, 251:], code[:5].transpose(1, 0, 2)) and not got[:, :251].any()
    got = v.download(np.uint8, (H, page // 4, D, 4), (pages - 2) * per)
    assert np.array_equal(got[:, 0].transpose(2, 0, 1), code[5:9])
    assert not k.download(np.uint8, (per,), 0).any()                   # where a 32-bit offset would have landed
    st.destroy()


def test_replayed_writes_and_reads():
    """A captured write and read over five replays, with other rows in the same buffers before each."""
    lib, rng, st = qfm.load(), np.random.default_rng(9), qfm.Stream()
    T, H, D, page = 21, 2, 128, 32
    c = _kv.Cache(4, page, H, D, INT8, np.array([[2, 0]], np.int32), rng)
    refs = c.upload()
    seq, pos = np.zeros(T, np.int32), np.arange(T, dtype=np.int32) + 17
    d = [qfm.DevBuf(T * H * D * 2), qfm.DevBuf.from_array(seq), qfm.DevBuf.from_array(pos), qfm.DevBuf(T * H * D * 4)]

    def calls():
        qfm.check(lib.qfm_kv_write(*refs, d[0].ptr, d[0].ptr, qfm.QFM_DT["bf16"], H * D, D, d[1].ptr, d[2].ptr, T, st.h), "write")
        qfm.check(lib.qfm_kv_read(*refs, None, d[3].ptr, 0, H * D, D, d[1].ptr, d[2].ptr, T, st.h), "read")

    qfm.check(lib.qfm_graph_capture_begin(st.h), "capture")
    calls()
    g = lib.qfm_graph_capture_end(st.h)
    assert g, lib.qfm_last_error().decode()
    for rep in range(5):
        bits, x = _kv.to_dtype(_rows(rng, T, H, D), "bf16")
        d[0].upload(bits)
        qfm.check(lib.qfm_graph_launch(g, st.h), "launch")
        st.sync()
        c.put(x, x, seq, pos)
        _same(c)
        a = d[3].download(np.float32, (T, H, D))
        calls()
        st.sync()
        assert np.array_equal(a, d[3].download(np.float32, (T, H, D))), rep
    assert lib.qfm_graph_destroy(g) == 0
    st.destroy()
