"""GPU: attention of drafted rows over the quantised cache (qfm_tree_attn)
against numpy in 64 bits. What no sequence holds (the ends of pages, pages of
nobody) is filled with NaN scales and codes that E4M3 reads as NaN."""
import numpy as np
import pytest

import qfm
import _kv
from _kv import E4M3, INT8

pytestmark = pytest.mark.gpu


def _say(*a):
    print("[attn]", *a, flush=True)


def _pool(rng, lens, page, H, D, fmt, spare=2):
    max_pages = max(1, max(-(-n // page) for n in lens))
    pages = len(lens) * max_pages + spare
    c = _kv.Cache(pages, page, H, D, fmt, _kv.tables(rng, len(lens), max_pages, pages), rng, fill=0x7F)
    for s, n in enumerate(lens):
        _kv.fill_rows(c, s, n, rng)
    return c


class Call:
    """One call's buffers, with out filled with 5 so that what is left can be seen."""

    def __init__(self, c, q_bits, dt, counts, ctx, tree, scale, layout="rows", T=None, max_ctx=None, max_nodes=None):
        self.lib, self.c, self.dt, self.st = qfm.load(), c, dt, qfm.Stream()
        T, Hq, D = q_bits.shape
        self.n, self.rs, self.hs = _kv.strided(T, Hq, D, layout)
        flat, self.at = _kv.scatter(q_bits, self.n, self.rs, self.hs)
        start = np.cumsum([0] + list(counts)).astype(np.int32)
        self.shape, self.fill = q_bits.shape, _kv.to_dtype(np.float32(5.0), dt)[0]
        self.b = {"q": qfm.DevBuf.from_array(flat), "start": qfm.DevBuf.from_array(start),
                  "ctx": qfm.DevBuf.from_array(np.asarray(ctx, np.int32)),
                  "out": qfm.DevBuf.from_array(np.full(self.n, self.fill, _kv.NP[dt]))}
        if tree is not None:
            self.b["tree"] = qfm.DevBuf.from_array(np.asarray(tree, np.uint64))
        refs = c.upload()
        mc, mn = max(ctx) if max_ctx is None else max_ctx, max_nodes or max(counts)
        wsb = self.lib.qfm_tree_attn_ws_bytes(refs[0], len(ctx), T, Hq, mn, mc)
        self.ws = qfm.DevBuf.from_array(np.full(max(16, wsb), 0xFF, np.uint8))     # NaN everywhere
        self.args = (*refs, self.b["q"].ptr, self.b["out"].ptr, qfm.QFM_DT[dt], Hq, self.rs, self.hs, self.rs, self.hs,
                     self.b["start"].ptr, self.b["ctx"].ptr, self.b["tree"].ptr if tree is not None else None, T, mn, mc, scale,
                     self.ws.ptr, wsb)

    def __call__(self):
        qfm.check(self.lib.qfm_tree_attn(*self.args, self.st.h), "qfm_tree_attn")

    def result(self):
        self.st.sync()
        flat = self.b["out"].download(_kv.NP[self.dt], self.n)
        rest = np.ones(self.n, bool)
        rest[self.at.ravel()] = False
        assert (flat[rest] == self.fill).all()                          # between the rows
        return flat[self.at]


def _check(got_bits, dt, want, tol, fill):
    got = _kv.from_bits(got_bits, dt).astype(np.float64)
    left = (tol == -1).all((1, 2))
    assert (got_bits[left] == fill).all()                               # rows of no sequence
    live = ~left
    bad = np.isnan(want[live])
    assert np.array_equal(np.isnan(got[live]), bad), "NaN where there is none, or the reverse"
    err = np.abs(got[live] - want[live])[~bad]
    over = err - tol[live][~bad]
    _say("  largest error", f"{err.max(initial=0):.2e}", "of its tolerance", f"{(err / np.maximum(tol[live][~bad], 1e-30)).max(initial=0):.2f}")
    assert (over <= 0).all(), (float(err.max()), float(over.max()))


def _run(rng, c, counts, ctx, Hq, dt, tree=True, layout="rows", extra=0, scale=None, q_scale=1.0, **kw):
    T, D = sum(counts) + extra, c.dim
    bits, q = _kv.to_dtype((rng.standard_normal((T, Hq, D)) * q_scale).astype(np.float32), dt)
    masks = _kv.tree_masks(list(counts) + [extra] * (extra > 0), rng) if tree is True else tree
    scale = D ** -0.5 if scale is None else scale
    call = Call(c, bits, dt, counts, ctx, masks, scale, layout, **kw)
    call()
    start = np.cumsum([0] + list(counts))
    want, tol = _kv.attention(c, q, start, ctx, masks, np.float32(scale), dt)
    _check(call.result(), dt, want, tol, call.fill)
    return call, want, tol


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("counts,ctx,Hq,H,D,page,layout", [
    ([1], [0], 1, 1, 64, 16, "rows"),                       # a token that sees itself alone
    ([1], [1], 8, 2, 64, 16, "heads"),
    ([1, 1, 1, 1], [31, 32, 33, 15], 4, 1, 128, 32, "wide"),
    ([1, 1, 1], [0, 500, 129], 16, 2, 256, 16, "rows"),
    ([8], [1021], 16, 2, 256, 16, "rows"),                  # fork rows, keys split over workgroups
    ([3, 7, 1], [64, 0, 300], 7, 1, 128, 64, "wide"),       # seven heads on one
    ([2, 5], [40, 17], 8, 8, 64, 128, "heads"),             # every head its own
    ([64, 33], [95, 160], 8, 2, 128, 32, "rows"),           # the widest trees, several row blocks
    ([64], [7], 12, 4, 256, 256, "heads"),
    ([64, 1, 20], [200, 3, 0], 16, 4, 64, 16, "rows"),
    ([20, 17], [700, 33], 16, 4, 128, 32, "wide"),          # 65 to 128 rows of a head
    ([9, 1], [333, 1300], 16, 2, 256, 16, "rows"),
    ([33, 30], [64, 900], 8, 2, 64, 64, "heads"),
    ([41], [2100], 12, 4, 128, 16, "rows"),                 # more, keys split over workgroups
    ([10, 16, 3], [50, 0, 40], 8, 2, 128, 32, "rows")])     # 33 to 64
def test_against_64_bits(fmt, dt, counts, ctx, Hq, H, D, page, layout):
    _say("fmt", fmt, dt, "rows", counts, "ctx", ctx, "heads", Hq, H, "D", D, "page", page, layout)
    rng = np.random.default_rng(sum(ctx) + Hq * D + fmt)
    c = _pool(rng, [a + b for a, b in zip(ctx, counts)], page, H, D, fmt)
    _run(rng, c, counts, ctx, Hq, dt, layout=layout)


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("seqs,m,Hq,H,max_ctx", [
    (9, 3, 16, 1, 0),                                       # one workgroup a block of rows
    (3, 17, 8, 8, 5000),                                    # 32 rows a wave, the keys in a few splits
    (1, 8, 16, 1, 400000),                                  # in as many as there are
    (3, 64, 32, 2, 8000),                                   # 256 rows and more a head
    (2, 8, 32, 2, 100000),
    (33, 17, 8, 8, 1300),
    (40, 40, 16, 1, 0)])
def test_every_layout(seqs, m, Hq, H, max_ctx, D, dt, fmt):
    """The host's bound of the contexts chooses the layout: each form, over short sequences of many lengths (so that
    splits without keys, waves without rows and sequences of fewer rows than planned are all there)."""
    _say("fmt", fmt, dt, "D", D, "sequences", seqs, "nodes", m, "heads", Hq, H, "planned for", max_ctx)
    rng = np.random.default_rng(seqs * m + Hq + D)
    counts = [m] + [int(x) for x in rng.integers(0, m + 1, seqs - 1)]
    ctx = [int(x) for x in rng.integers(0, 90, seqs)]
    if seqs > 2:
        ctx[1], counts[2] = 0, 1
    c = _pool(rng, [a + b for a, b in zip(ctx, counts)], 16, H, D, fmt)
    _run(rng, c, counts, ctx, Hq, dt, max_ctx=max_ctx, max_nodes=m, extra=1)


@pytest.mark.parametrize("seqs,long_one,Hq,H,D,dt,max_ctx", [
    (2, 3000, 8, 2, 64, "bf16", 3000), (5, 4000, 16, 1, 128, "f16", 4000), (37, 2500, 8, 4, 64, "f32", 131071),
    (70, 2000, 4, 2, 128, "bf16", 4000),                    # more sequences than lanes
    (200, 1500, 4, 1, 64, "bf16", 100000), (256, 700, 4, 1, 256, "f32", 100000),
    (257, 700, 4, 1, 64, "f16", 100000), (300, 300, 2, 1, 64, "bf16", 9000)])
def test_one_long_sequence_among_short_ones(seqs, long_one, Hq, H, D, dt, max_ctx):
    """The keys are dealt out by length: sequences in one part, in several and without rows beside each other, the long
    one anywhere; and a batch in which nobody has rows."""
    _say(seqs, "sequences, one of", long_one, "heads", Hq, H, "D", D, dt, "planned for", max_ctx)
    rng = np.random.default_rng(seqs)
    for at in (0, seqs // 2, seqs - 1):
        ctx = [int(x) for x in rng.integers(0, 40, seqs)]
        counts = [int(x) for x in rng.integers(0, 3, seqs)]
        ctx[at], counts[at] = long_one, 3
        ctx[(at + 1) % seqs] = long_one // 2
        c = _pool(rng, [a + b for a, b in zip(ctx, counts)], 16, H, D, E4M3)
        _run(rng, c, counts, ctx, Hq, dt, max_ctx=max_ctx, max_nodes=4, extra=2)
    c = _pool(rng, [1] * seqs, 16, H, D, INT8)
    _run(rng, c, [0] * seqs, [0] * seqs, Hq, dt, max_ctx=max_ctx, max_nodes=4, extra=3)


@pytest.mark.parametrize("D,dt", [(128, "bf16"), (256, "f16"), (64, "f32")])
def test_chain_and_rows_of_no_sequence(D, dt):
    """No masks: a chain. Rows behind the last sequence, and a sequence without rows, are left alone."""
    rng = np.random.default_rng(D)
    counts, ctx = [5, 0, 9], [70, 30, 2]
    c = _pool(rng, [a + b for a, b in zip(ctx, counts)], 16, 2, D, E4M3)
    _run(rng, c, counts, ctx, 6, dt, tree=None, extra=4)


def test_masks_that_leave_rows_empty():
    """Masks of nothing, of other nodes only, and bits of nodes that do not exist."""
    rng = np.random.default_rng(4)
    for ctx in ([0, 0], [0, 33]):
        counts = [4, 3]
        c = _pool(rng, [a + b for a, b in zip(ctx, counts)], 16, 1, 64, INT8)
        tree = np.array([0, 1 << 3, (1 << 64) - 1, 0xF0, 0, 1 << 63, 0b101], np.uint64)
        for dt in ("bf16", "f32"):
            _run(rng, c, counts, ctx, 2, dt, tree=tree)


@pytest.mark.parametrize("fmt", [INT8, E4M3])
def test_rows_lost_to_nan_reach_only_those_that_see_them(fmt):
    """A drafted token whose keys or values are NaN: its own row and its descendants' are NaN, its siblings' are not."""
    rng = np.random.default_rng(8)
    ctx, m, H, D = 50, 6, 1, 64
    for lost in ("k", "v", "both"):
        c = _pool(rng, [ctx + m], 16, H, D, fmt)
        bad, p = np.full((1, H, D), np.nan, np.float32), ctx + 2
        g, o = c.place(0, p)
        code, s = _kv.quantise(bad[0], fmt)
        if lost != "v":
            c.k[g, :, o], c.ks[g, :, o] = code, s
        if lost != "k":
            c.v[g, :, o // 4, :, o % 4], c.vs[g, :, o] = code, s
        tree = np.array([0b1, 0b11, 0b101, 0b1101, 0b10011, 0b100000], np.uint64)
        call, want, _ = _run(rng, c, [m], [ctx], 4, "f16", tree=tree)
        assert np.isnan(want[2:4]).all() and np.isfinite(np.delete(want, [2, 3], 0)).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_queries_that_are_not_finite(dt):
    """An infinity or a NaN in a row of q: NaN for that row and head alone, whatever the signs of its keys; zeros where it
    sees nothing."""
    rng = np.random.default_rng(18)
    for counts, ctx, tree in (([3], [0], [1, 2, 0]), ([5, 40], [33, 200], None)):
        T, Hq, H, D = sum(counts), 4, 1, 64
        c = _pool(rng, [a + b for a, b in zip(ctx, counts)], 16, H, D, INT8)
        c.k[:, :, :, 7] = 0x85                                          # one channel negative in every key
        x = rng.standard_normal((T, Hq, D)).astype(np.float32)
        x[0, 0, 7], x[1, 1, 9], x[1, 2, 7], x[2, 3, 3] = np.inf, -np.inf, np.nan, np.inf
        bits, q = _kv.to_dtype(x, dt)
        tree = None if tree is None else np.array(tree, np.uint64)
        call = Call(c, bits, dt, counts, ctx, tree, D ** -0.5)
        call()
        with np.errstate(invalid="ignore"):
            want, tol = _kv.attention(c, q, np.cumsum([0] + counts), ctx, tree, np.float32(D ** -0.5), dt)
        assert np.isnan(want[0, 0]).all() and np.isfinite(want[0, 1:]).all()
        _check(call.result(), dt, want, tol, call.fill)


@pytest.mark.parametrize("fmt", [INT8, E4M3])
def test_pages_that_do_not_exist_are_not_seen(fmt):
    rng = np.random.default_rng(12)
    counts, ctx = [3, 2], [70, 100]
    c = _pool(rng, [a + b for a, b in zip(ctx, counts)], 16, 2, 128, fmt)
    c.table[0, 1], c.table[0, 4], c.table[1, 0], c.table[1, 6] = -1, 1 << 30, c.pages, -(1 << 31)
    _run(rng, c, counts, ctx, 4, "bf16")
    # positions beyond the table, and contexts that are no lengths
    for far in ([1 << 30, (1 << 31) - 1], [-5, 112]):
        _run(rng, c, counts, far, 4, "bf16", max_ctx=100)


def test_host_bound_of_contexts_only_plans():
    """max_ctx far too small or far too large: the same results."""
    rng = np.random.default_rng(13)
    counts, ctx = [4, 1], [777, 20]
    c = _pool(rng, [a + b for a, b in zip(ctx, counts)], 64, 2, 128, INT8)
    for max_ctx in (0, 1 << 20):
        _run(rng, c, counts, ctx, 8, "f32", max_ctx=max_ctx, max_nodes=64)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("fmt", [INT8, E4M3])
def test_scores_and_scales_far_apart(fmt, dt):
    """Scores in the thousands with the largest last, rows of Q 2^40 apart, value scales over eight decades in any order."""
    rng = np.random.default_rng(14)
    counts, ctx, H, D = [6], [600], 1, 64
    c = _pool(rng, [606], 32, H, D, fmt)
    order = np.exp(rng.uniform(np.log(1e-4), np.log(1e4), 606)).astype(np.float32)
    for p in range(606):
        g, o = c.place(0, p)
        c.vs[g, :, o] *= order[p]
        c.ks[g, :, o] *= np.float32(0.2 + 30.0 * p / 606)
    T = 6
    bits, q = _kv.to_dtype((rng.standard_normal((T, 2, D)) * np.array([1, 2.0 ** -20, 2.0 ** 20, 8, 0, 2.0 ** -30])[:, None, None]).astype(np.float32), dt)
    call = Call(c, bits, dt, counts, ctx, None, D ** -0.5)
    call()
    want, tol = _kv.attention(c, q, [0, T], ctx, None, np.float32(D ** -0.5), dt)
    _check(call.result(), dt, want, tol, call.fill)


def test_replays_with_growing_contexts():
    """One captured call over replays whose contexts, masks and rows change in place; eager calls between."""
    rng, lib = np.random.default_rng(15), qfm.load()
    counts, top, D, Hq, H = [2, 3], [900, 400], 128, 8, 2
    c = _pool(rng, [a + b for a, b in zip(top, counts)], 32, H, D, INT8)
    tree = _kv.tree_masks(counts, rng)
    bits, _ = _kv.to_dtype(rng.standard_normal((5, Hq, D)).astype(np.float32), "bf16")
    call = Call(c, bits, "bf16", counts, top, tree, D ** -0.5)
    qfm.check(lib.qfm_graph_capture_begin(call.st.h), "capture")
    call()
    g = lib.qfm_graph_capture_end(call.st.h)
    assert g, lib.qfm_last_error().decode()
    for rep, ctx in enumerate([[900, 400], [0, 399], [513, 1], [31, 32], [899, 0]]):
        bits, q = _kv.to_dtype(rng.standard_normal((5, Hq, D)).astype(np.float32), "bf16")
        call.b["q"].upload(bits)
        call.b["ctx"].upload(np.array(ctx, np.int32))
        qfm.check(lib.qfm_graph_launch(g, call.st.h), "launch")
        got = call.result()
        want, tol = _kv.attention(c, q, [0, 2, 5], ctx, tree, np.float32(D ** -0.5), "bf16")
        _check(got, "bf16", want, tol, call.fill)
        call()
        assert np.array_equal(call.result(), got), rep                  # and the same bits eagerly
    assert lib.qfm_graph_destroy(g) == 0


def test_two_graphs_share_a_workspace():
    """Two captured calls of different shapes on one workspace, replayed in turn on one stream: each as by itself."""
    rng, lib = np.random.default_rng(19), qfm.load()
    calls, want = [], []
    for counts, ctx, Hq, H, D, dt in (([3, 1], [900, 40], 8, 2, 128, "bf16"), ([20], [2100], 16, 2, 64, "f32")):
        c = _pool(rng, [a + b for a, b in zip(ctx, counts)], 32, H, D, INT8)
        bits, q = _kv.to_dtype(rng.standard_normal((sum(counts), Hq, D)).astype(np.float32), dt)
        calls.append(Call(c, bits, dt, counts, ctx, None, D ** -0.5))
        want.append(_kv.attention(c, q, np.cumsum([0] + counts), ctx, None, np.float32(D ** -0.5), dt))
    sizes = [c.args[-1] for c in calls]
    assert min(sizes) > 0
    ws, st = qfm.DevBuf.from_array(np.full(max(sizes), 0xFF, np.uint8)), calls[0].st
    graphs = []
    for c, size in zip(calls, sizes):
        c.args, c.st = (*c.args[:-2], ws.ptr, size), st
        qfm.check(lib.qfm_graph_capture_begin(st.h), "capture")
        c()
        graphs.append(lib.qfm_graph_capture_end(st.h))
        assert graphs[-1], lib.qfm_last_error().decode()
    first = None
    for rep in range(4):
        for c in calls:
            c.b["out"].upload(np.full(c.n, c.fill, _kv.NP[c.dt]))
        for g in graphs:
            qfm.check(lib.qfm_graph_launch(g, st.h), "launch")
        got = [c.result() for c in calls]
        for c, y, (w, tol) in zip(calls, got, want):
            _check(y, c.dt, w, tol, c.fill)
        assert first is None or all(np.array_equal(a, b) for a, b in zip(got, first))
        first = got
        calls[rep % 2]()                                                # an eager one on the same workspace between
    for g in graphs:
        assert lib.qfm_graph_destroy(g) == 0


def test_pages_behind_four_gigabytes():
    rng, lib = np.random.default_rng(16), qfm.load()
    page, H, D, pages, ctx, m, Hq = 256, 8, 256, 8300, 300, 2, 8
    per = page * H * D
    small = _pool(rng, [ctx + m], page, H, D, INT8, spare=0)            # two pages, put at the end of a large pool
    bufs = {n: qfm.DevBuf(pages * b) for n, b in (("k", per), ("v", per), ("ks", page * H * 4), ("vs", page * H * 4))}
    for n, b in (("k", per), ("v", per), ("ks", page * H * 4), ("vs", page * H * 4)):
        a = np.ascontiguousarray(getattr(small, n))
        qfm.check(lib.qfm_memcpy_h2d(bufs[n].ptr + (pages - 2) * b, a.ctypes.data, a.nbytes), "h2d")
    bits, q = _kv.to_dtype(rng.standard_normal((m, Hq, D)).astype(np.float32), "bf16")
    call = Call(small, bits, "bf16", [m], [ctx], None, D ** -0.5)
    small.d["table"].upload(small.table + (pages - 2))
    small.c.k, small.c.v, small.c.ks, small.c.vs = (bufs[n].ptr for n in ("k", "v", "ks", "vs"))
    small.c.n_pages = pages
    call()
    want, tol = _kv.attention(small, q, [0, m], [ctx], None, np.float32(D ** -0.5), "bf16")
    _check(call.result(), "bf16", want, tol, call.fill)
