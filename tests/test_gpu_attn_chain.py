"""GPU: the cache, the attention, the adapters and the INT8 projections as a
decode program runs them together. Rows of several users' draft trees go through
X8 -> projections -> adapters in place -> cache write -> attention -> X8 ->
output projection; the accepted nodes' keys and values are then written again
behind the context, and the next round's rows see them. Every stage is compared
with numpy on the GPU's own inputs to it, and a captured round with the eager
one."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

import _kv
import _oracle as orc
import qfm
import test_gpu_lora as lora

pytestmark = pytest.mark.gpu

K, HQ, H, D, NO, R, SLOTS, PAGE = 2560, 8, 2, 64, 100, 16, 3, 16
STAGE = 2e-5                                # of the largest output, as for the projections by themselves


def _say(*a):
    print("[chain]", *a, flush=True)


class Mat:
    def __init__(self, rng, rows, k, scale):
        self.q = rng.integers(-127, 128, (rows, k)).astype(np.int8)
        self.s = (rng.uniform(0.5, 1.5, rows) * scale / np.sqrt(k)).astype(np.float32)
        self.dq, self.ds = qfm.DevBuf.from_array(self.q), qfm.DevBuf.from_array(self.s)
        self.m = qfm.Qf8I8Mat(self.dq.ptr, self.ds.ptr, rows, k)


def _multi(mats, ys):
    mm = qfm.Qf8I8Multi()
    mm.n = len(mats)
    for i, (m, y) in enumerate(zip(mats, ys)):
        mm.m[i], mm.y[i], mm.act[i] = C.pointer(m.m), y.ptr, 0
    return mm


class Round:
    """A layer's decode step for draft trees of counts[s] nodes behind ctx[s] tokens, on the caller's buffers."""

    def __init__(self, rng, fmt, counts, ctx, max_ctx):
        self.lib, self.st, self.T, self.fmt = qfm.load(), qfm.Stream(), sum(counts), fmt
        qfm.init(2560, 640, 512, 10, 1, 1)
        T, n, self.counts = self.T, len(counts), counts
        self.start = np.cumsum([0] + counts).astype(np.int32)
        self.seq = np.repeat(np.arange(n), counts).astype(np.int32)
        pages = n * (-(-(max_ctx + 64) // PAGE)) + 3
        self.cache = _kv.Cache(pages, PAGE, H, D, fmt, _kv.tables(rng, n, (pages - 3) // n, pages), rng, fill=0x7F)
        for s in range(n):
            _kv.fill_rows(self.cache, s, ctx[s], rng)
        self.refs = self.cache.upload()
        self.mats = [Mat(rng, HQ * D, K, 0.02), Mat(rng, H * D, K, 0.02), Mat(rng, H * D, K, 0.02)]
        self.out_mat = Mat(rng, NO, HQ * D, 0.02)
        self.slot = np.array([s % (SLOTS + 1) - 1 for s in self.seq], np.int32)       # the first user has none
        b = self.b = {n_: qfm.DevBuf(nb) for n_, nb in
                      (("x", T * K * 4), ("xh", T * K * 2), ("xq", T * K), ("xs", T * K // 8), ("q", T * HQ * D * 4),
                       ("k", T * H * D * 4), ("v", T * H * D * 4), ("o", T * HQ * D * 4), ("oq", T * HQ * D),
                       ("os", T * HQ * D // 8), ("y", T * NO * 4), ("pos", T * 4), ("pos2", T * 4), ("ctx", n * 4), ("tree", T * 8))}
        b["seq"], b["start"], b["slot"] = (qfm.DevBuf.from_array(a) for a in (self.seq, self.start, self.slot))
        self.rank = np.array([R, 3, 9], np.int32)
        self.scale = np.array([0.5, 1.0, 2.0], np.float32)
        b["rank"], b["scale"] = qfm.DevBuf.from_array(self.rank), qfm.DevBuf.from_array(self.scale)
        l = self.l = qfm.QfmLora()
        l.n, l.K, l.R, l.slots, l.dtype, l.rank, l.scale = 3, K, R, SLOTS, qfm.QFM_DT["bf16"], b["rank"].ptr, b["scale"].ptr
        self.A, self.B = [], []
        for i, (m, y) in enumerate(zip(self.mats, ("q", "k", "v"))):
            rows = m.q.shape[0]
            ab, a = _kv.to_dtype((rng.standard_normal((SLOTS, R, K)) / np.sqrt(K)).astype(np.float32), "bf16")
            bb, w = _kv.to_dtype((rng.standard_normal((SLOTS, rows, R)) * 0.2).astype(np.float32), "bf16")
            past = np.arange(R) >= self.rank[:, None]
            self.A.append(np.where(past[..., None], 0, a))
            self.B.append(np.where(past[:, None, :], 0, w))
            b[f"a{i}"], b[f"b{i}"] = qfm.DevBuf.from_array(ab), qfm.DevBuf.from_array(bb)
            l.a[i], l.b[i], l.rows[i], l.y[i], l.base[i] = b[f"a{i}"].ptr, b[f"b{i}"].ptr, rows, b[y].ptr, b[y].ptr
        self.mm, self.mo = _multi(self.mats, [b["q"], b["k"], b["v"]]), _multi([self.out_mat], [b["y"]])
        self.lws = self.lib.qfm_lora_ws_bytes(C.byref(l), T)
        self.max_ctx, self.m = max_ctx, max(counts)
        self.aws = self.lib.qfm_tree_attn_ws_bytes(self.refs[0], n, T, HQ, self.m, max_ctx)
        b["ws"] = qfm.DevBuf.from_array(np.full(max(self.lws, self.aws, 16), 0xFF, np.uint8))   # one after the other: shared

    def load(self, rng, ctx):
        """New rows, masks and contexts, in place."""
        self.ctx = list(ctx)
        self.pos = np.array([self.ctx[s] + i for s, m in enumerate(self.counts) for i in range(m)], np.int32)
        self.tree = _kv.tree_masks(self.counts, rng)
        bits, x = _kv.to_dtype(rng.standard_normal((self.T, K)).astype(np.float32), "bf16")
        self.x = x
        for n, a in (("x", x), ("xh", bits), ("pos", self.pos), ("ctx", np.array(ctx, np.int32)), ("tree", self.tree)):
            self.b[n].upload(a)

    def stages(self):
        lib, b, T, s, dt = self.lib, self.b, self.T, self.st.h, qfm.QFM_DT["f32"]
        ok = lambda rc: qfm.check(rc, "stage")
        return [
            ("x8", lambda: ok(lib.qf8_i8_x8_ex(b["x"].ptr, b["xq"].ptr, b["xs"].ptr, T * K, s))),
            ("project", lambda: ok(lib.qf8_i8_gemv_rows(C.byref(self.mm), b["xq"].ptr, b["xs"].ptr, T, s))),
            ("adapt", lambda: ok(lib.qfm_lora_rows(C.byref(self.l), b["xh"].ptr, K, b["slot"].ptr, T, b["ws"].ptr, self.lws, s))),
            ("write", lambda: ok(lib.qfm_kv_write(*self.refs, b["k"].ptr, b["v"].ptr, dt, H * D, D, b["seq"].ptr, b["pos"].ptr, T, s))),
            ("attend", lambda: ok(lib.qfm_tree_attn(*self.refs, b["q"].ptr, b["o"].ptr, dt, HQ, HQ * D, D, HQ * D, D, b["start"].ptr,
                                                    b["ctx"].ptr, b["tree"].ptr, T, self.m, self.max_ctx, D ** -0.5, b["ws"].ptr,
                                                    self.aws, s))),
            ("x8 out", lambda: ok(lib.qf8_i8_x8_ex(b["o"].ptr, b["oq"].ptr, b["os"].ptr, T * HQ * D, s))),
            ("project out", lambda: ok(lib.qf8_i8_gemv_rows(C.byref(self.mo), b["oq"].ptr, b["os"].ptr, T, s)))]

    def get(self, n, shape, t=np.float32):
        return self.b[n].download(t, shape)

    def cache_state(self):
        d = self.cache.download()
        self.cache.k, self.cache.v, self.cache.ks, self.cache.vs = d["k"], d["v"], d["ks"], d["vs"]
        return d

    def check_write(self, before, pos):
        """The rows of k and v that lie in the buffers now, at pos: their codes and scales, and nothing else changed."""
        want = _kv.Cache.__new__(_kv.Cache)
        want.__dict__.update(self.cache.__dict__)
        want.k, want.v, want.ks, want.vs = (before[n].copy() for n in ("k", "v", "ks", "vs"))
        want.put(self.get("k", (self.T, H, D)), self.get("v", (self.T, H, D)), self.seq, pos)
        after = self.cache_state()
        for n in ("k", "v", "ks", "vs"):
            assert np.array_equal(after[n].view(np.uint8), getattr(want, n).view(np.uint8)), n

    def check_round(self):
        """Runs the stages one by one, each against numpy on what the GPU had before it."""
        T, before = self.T, self.cache_state()
        for name, run in self.stages():
            base = [self.get(n, (T, m.q.shape[0])) for n, m in zip("qkv", self.mats)] if name == "adapt" else None
            run()
            self.st.sync()
            if name == "x8":
                xq, xs = self.get("xq", (T, K), np.int8), self.get("xs", (T, K // 32))
                for t in range(T):
                    q, s = orc.x8_quant(self.x[t])
                    assert np.array_equal(q, xq[t]) and np.array_equal(s, xs[t])
            elif name == "project":
                for n, m in zip("qkv", self.mats):
                    y = self.get(n, (T, m.q.shape[0]))
                    for t in range(T):
                        ref = orc.i8_gemv(m.q, m.s, xq[t], xs[t], 0)
                        assert np.abs(y[t] - ref).max() <= STAGE * np.abs(ref).max()
            elif name == "adapt":
                want = lora.Case.want(SimpleNamespace(a=self.A, b=self.B, base=base, slot=self.slot, scale=self.scale, x=self.x, dt="bf16"))
                for n, m, (y, tol) in zip("qkv", self.mats, want):
                    assert (np.abs(self.get(n, (T, m.q.shape[0])) - y) <= tol).all(), n
            elif name == "write":
                self.check_write(before, self.pos)
            elif name == "attend":
                want, tol = _kv.attention(self.cache, self.get("q", (T, HQ, D)), self.start, self.ctx, self.tree,
                                          np.float32(D ** -0.5), "f32")
                assert (np.abs(self.get("o", (T, HQ, D)) - want) <= tol).all()
            elif name == "x8 out":
                oq, os_, o = self.get("oq", (T, HQ * D), np.int8), self.get("os", (T, HQ * D // 32)), self.get("o", (T, HQ * D))
                for t in range(T):
                    q, s = orc.x8_quant(o[t])
                    assert np.array_equal(q, oq[t]) and np.array_equal(s, os_[t])
            else:
                y = self.get("y", (T, NO))
                for t in range(T):
                    ref = orc.i8_gemv(self.out_mat.q, self.out_mat.s, oq[t], os_[t], 0)
                    assert np.abs(y[t] - ref).max() <= STAGE * np.abs(ref).max()
                assert y.any()
                return y

    def accept(self, rng):
        """Each sequence accepts a path of its tree: those rows again at the positions behind the context."""
        pos, ctx = np.full(self.T, -1, np.int32), []
        for s, m in enumerate(self.counts):
            r0 = int(self.start[s])
            mask = int(self.tree[r0 + int(rng.integers(m))])
            path = [i for i in range(m) if mask >> i & 1]
            pos[[r0 + i for i in path]] = self.ctx[s] + np.arange(len(path))
            ctx.append(self.ctx[s] + len(path))
        before = self.cache_state()
        self.b["pos2"].upload(pos)
        qfm.check(self.lib.qfm_kv_write(*self.refs, self.b["k"].ptr, self.b["v"].ptr, qfm.QFM_DT["f32"], H * D, D,
                                        self.b["seq"].ptr, self.b["pos2"].ptr, self.T, self.st.h), "accept")
        self.st.sync()
        self.check_write(before, pos)
        return ctx


@pytest.mark.parametrize("fmt", [_kv.INT8, _kv.E4M3])
@pytest.mark.parametrize("counts,ctx,max_ctx", [([7, 1, 4], [30, 0, 200], 300), ([40, 33], [100, 17], 4000)])
def test_rounds_of_drafting_and_accepting(fmt, counts, ctx, max_ctx):
    rng = np.random.default_rng(len(counts) + fmt)
    r = Round(rng, fmt, counts, ctx, max_ctx)
    for i in range(3):
        _say("fmt", fmt, "round", i, "contexts", ctx)
        r.load(rng, ctx)
        r.check_round()
        ctx = r.accept(rng)


def test_captured_round():
    """A whole round captured once and replayed over growing contexts, eager rounds between: the same bits."""
    rng, counts, ctx = np.random.default_rng(3), [6, 2, 1], [12, 0, 150]
    r = Round(rng, _kv.INT8, counts, ctx, 400)
    r.load(rng, ctx)
    r.check_round()
    qfm.check(r.lib.qfm_graph_capture_begin(r.st.h), "capture")
    for _, run in r.stages():
        run()
    g = r.lib.qfm_graph_capture_end(r.st.h)
    assert g, r.lib.qfm_last_error().decode()
    for i in range(4):
        ctx = r.accept(rng)
        _say("replay", i, "contexts", ctx)
        r.load(rng, ctx)
        y = r.check_round()
        state, o = r.cache_state(), r.get("o", (r.T, HQ, D))
        for n in ("q", "k", "v", "o", "y"):
            r.b[n].upload(np.full(r.b[n].nbytes, 0xA5, np.uint8))
        qfm.check(r.lib.qfm_graph_launch(g, r.st.h), "launch")
        r.st.sync()
        assert np.array_equal(r.get("y", (r.T, NO)), y) and np.array_equal(r.get("o", (r.T, HQ, D)), o)
        again = r.cache_state()
        assert all(np.array_equal(again[n].view(np.uint8), state[n].view(np.uint8)) for n in state)
    assert r.lib.qfm_graph_destroy(g) == 0


def test_two_rounds_at_once():
    """Two users' rounds on streams and workspaces of their own, queued without a wait between them: as by themselves."""
    rounds = []
    for seed in (5, 6):
        rng = np.random.default_rng(seed)
        ctx = [40 * seed, 3]
        r = Round(rng, _kv.E4M3, [20, 5], ctx, 300)
        r.load(rng, ctx)
        rounds.append((r, r.check_round()))
    for _ in range(5):
        for r, _y in rounds:
            for n in ("q", "k", "v", "o", "y"):
                r.b[n].upload(np.full(r.b[n].nbytes, 0xA5, np.uint8))
        for pair in zip(*(r.stages() for r, _ in rounds)):
            for _, run in pair:
                run()
        for r, y in rounds:
            r.st.sync()
            assert np.array_equal(r.get("y", (r.T, NO)), y)
