"""GPU: low-rank adapters of many requests (qfm_lora_rows) against numpy in 64
bits. Ranks below R: the rows and columns behind them are NaN and do not count."""
import ctypes as C

import numpy as np
import pytest

import qfm
import _kv

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _say(*a):
    print("[lora]", *a, flush=True)


class Case:
    def __init__(self, rng, T, slots, R, K, ns, dt, slot, base="rows", x_stride=None):
        self.lib, self.st, self.dt, self.T, self.ns = qfm.load(), qfm.Stream(), dt, T, ns
        self.slot = np.asarray(slot, np.int32)
        self.rank = rng.integers(1, R + 1, slots).astype(np.int32)
        self.rank[0] = R
        self.scale = rng.uniform(0.5, 2, slots).astype(np.float32)
        xs = x_stride or K
        xb, x = _kv.to_dtype(rng.standard_normal((T, xs)).astype(np.float32), dt)
        self.x = x[:, :K]
        self.a, self.b, self.base, bufs = [], [], [], {}
        l = self.l = qfm.QfmLora()
        l.n, l.K, l.R, l.slots, l.dtype = len(ns), K, R, slots, qfm.QFM_DT[dt]
        past = np.arange(R) >= self.rank[:, None]                            # [slots][R]
        for i, n in enumerate(ns):
            ab, a = _kv.to_dtype((rng.standard_normal((slots, R, K)) / np.sqrt(K)).astype(np.float32), dt)
            bb, b = _kv.to_dtype((rng.standard_normal((slots, n, R)) * 0.3).astype(np.float32), dt)
            nan = _kv.to_dtype(np.float32(np.nan), dt)[0]
            ab[past] = nan
            bb[np.broadcast_to(past[:, None, :], bb.shape)] = nan
            self.a.append(np.where(past[..., None], 0, a))
            self.b.append(np.where(past[:, None, :], 0, b))
            base_i = rng.standard_normal((T, n)).astype(np.float32)
            self.base.append(base_i if base != "none" else np.zeros_like(base_i))
            bufs[f"a{i}"], bufs[f"b{i}"] = qfm.DevBuf.from_array(ab), qfm.DevBuf.from_array(bb)
            bufs[f"y{i}"] = qfm.DevBuf.from_array(base_i if base == "in place" else np.full((T, n), 9.0, np.float32))
            bufs[f"base{i}"] = qfm.DevBuf.from_array(base_i)
            l.a[i], l.b[i], l.rows[i], l.y[i] = bufs[f"a{i}"].ptr, bufs[f"b{i}"].ptr, n, bufs[f"y{i}"].ptr
            l.base[i] = {"rows": bufs[f"base{i}"].ptr, "none": None, "in place": bufs[f"y{i}"].ptr}[base]
        for n, v in (("rank", self.rank), ("scale", self.scale), ("slot", self.slot), ("x", xb)):
            bufs[n] = qfm.DevBuf.from_array(v)
        l.rank, l.scale = bufs["rank"].ptr, bufs["scale"].ptr
        self.wsb = self.lib.qfm_lora_ws_bytes(C.byref(l), T)
        bufs["ws"] = qfm.DevBuf.from_array(np.full(max(16, self.wsb), 0xFF, np.uint8))
        self.bufs, self.xs = bufs, xs

    def __call__(self):
        b = self.bufs
        qfm.check(self.lib.qfm_lora_rows(C.byref(self.l), b["x"].ptr, self.xs, b["slot"].ptr, self.T, b["ws"].ptr, self.wsb,
                                         self.st.h), "qfm_lora_rows")

    def result(self):
        self.st.sync()
        return [self.bufs[f"y{i}"].download(np.float32, (self.T, n)) for i, n in enumerate(self.ns)]

    def want(self):
        """(y, tolerance) of each projection. h: K products summed in fp32 (6 sqrt(K) u of their magnitudes), kept as
        three bf16 numbers (2^-24 of a value) or two fp16 ones (2^-22 of a value, 2^-38 of the row's largest); the second
        product's R terms (at most 3 R additions) 6 sqrt(3 R) u; the factor, its product and the sum, a rounding each."""
        out = []
        for a, b, base in zip(self.a, self.b, self.base):
            y, tol = base.astype(np.float64), np.zeros(base.shape)
            for t, e in enumerate(self.slot):
                if not 0 <= e < len(self.scale):
                    continue
                x, ae, be, f = self.x[t].astype(np.float64), a[e].astype(np.float64), b[e].astype(np.float64), float(self.scale[e])
                h = ae @ x
                dh = 6 * np.sqrt(x.size) * U * (np.abs(ae) @ np.abs(x)) + np.abs(h) * (2.0 ** -24 if self.dt == "bf16" else 2.0 ** -22)
                dh += 2.0 ** -38 * np.abs(h).max()
                d = be @ h
                y[t] += f * d
                tol[t] = f * (np.abs(be) @ (dh + np.abs(h) * 6 * np.sqrt(3 * h.size) * U)) + 4 * U * (np.abs(f * d) + np.abs(base[t]))
            out.append((y, tol))
        return out

    def check(self, got):
        for i, (g, (y, tol)) in enumerate(zip(got, self.want())):
            err = np.abs(g - y)
            _say("  projection", i, "largest error", f"{err.max():.2e}", "of its tolerance", f"{(err / np.maximum(tol, 1e-30)).max():.2f}"
                 if tol.max() else "-")
            assert (err <= tol).all(), (i, float(err.max()))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("T,slots,R,K,ns,kind", [
    (1, 1, 8, 64, [1], "any"), (1, 5, 16, 2048, [4096, 512, 512], "any"), (8, 3, 16, 2560, [640, 640], "any"),
    (37, 24, 32, 512, [1021], "any"), (16, 16, 128, 128, [256], "each"), (17, 4, 24, 320, [63, 64, 65, 2], "any"),
    (256, 9, 64, 192, [130], "any"), (257, 9, 64, 192, [130], "any"), (700, 6, 40, 256, [512, 33], "runs"),
    (530, 40, 8, 64, [100], "any"), (300, 2, 128, 1024, [128], "runs"),
    # both products in one launch: ranks and K at its ends, ragged rows and outputs, and one beyond each bound
    (16, 5, 64, 2048, [33], "any"), (37, 24, 8, 64, [255, 2], "any"), (5, 2, 40, 3200, [600], "any"), (1, 1, 24, 4096, [7, 300], "any"),
    (250, 2, 16, 576, [256, 256], "any"), (3, 3, 72, 512, [64], "each"), (2, 2, 64, 2112, [64], "each"), (2, 9, 8, 4160, [64], "each")])
def test_against_64_bits(dt, T, slots, R, K, ns, kind):
    _say(dt, "rows", T, "slots", slots, "R", R, "K", K, "outputs", ns, kind)
    rng = np.random.default_rng(T * 31 + R + K)
    slot = {"any": lambda: rng.integers(-1, slots, T), "each": lambda: rng.permutation(slots)[:T],
            "runs": lambda: np.repeat(rng.integers(0, slots, 7), -(-T // 7))[:T]}[kind]()
    for base in ("rows", "none", "in place"):
        c = Case(rng, T, slots, R, K, ns, dt, slot, base, x_stride=K + 8 if base == "none" else None)
        c()
        c.check(c.result())


@pytest.mark.parametrize("T", [40, 400])
def test_slots_that_do_not_exist_and_ranks_out_of_range(T):
    """Rows of no slot keep base; ranks below 0 count as 0, above R as R."""
    rng = np.random.default_rng(T)
    slot = rng.integers(-3, 9, T)
    slot[3], slot[5] = 1 << 30, -(1 << 31)
    c = Case(rng, T, 5, 16, 128, [48], "bf16", slot)
    c()
    got = c.result()
    c.check(got)
    none = (slot < 0) | (slot >= 5)
    assert np.array_equal(got[0][none], c.base[0][none])
    rank = np.array([16, 0, -4, 99, 1], np.int32)
    c.bufs["rank"].upload(rank)
    for e, r in ((1, 0), (2, 0), (4, 1)):
        c.a[0][e, r:] = 0
        c.b[0][e, :, r:] = 0
    # slot 3 has its whole rank now: what lay behind the old one was NaN
    full, col = _kv.to_dtype(rng.standard_normal((16, 128)).astype(np.float32), "bf16"), _kv.to_dtype(rng.standard_normal((48, 16)).astype(np.float32), "bf16")
    for name, i, (bits, val), dst in (("a0", 3, full, c.a[0]), ("b0", 3, col, c.b[0])):
        qfm.check(c.lib.qfm_memcpy_h2d(c.bufs[name].ptr + i * bits.nbytes, bits.ctypes.data, bits.nbytes), "h2d")
        dst[i] = val
    c()
    c.check(c.result())


@pytest.mark.parametrize("T", [12, 300])
def test_rows_and_adapters_that_are_not_finite_stay_alone(T):
    """A row of NaN, a row with an infinity and an adapter with infinite weights reach their own rows only."""
    rng = np.random.default_rng(1)
    slot = np.arange(T) % 3
    for dt in ("bf16", "f16"):
        c = Case(rng, T, 3, 8, 64, [40], dt, slot)
        c()
        before = c.result()[0]
        x = c.bufs["x"].download(_kv.NP[dt], (T, 64))
        x[1, 5], x[4, 0] = _kv.to_dtype(np.float32(np.nan), dt)[0], _kv.to_dtype(np.float32(np.inf), dt)[0]
        c.bufs["x"].upload(x)
        b = c.bufs["b0"].download(_kv.NP[dt], (3, 40, 8))
        b[2, :, 0] = _kv.to_dtype(np.float32(np.inf), dt)[0]
        c.bufs["b0"].upload(b)
        c()
        y = c.result()[0]
        lost = (np.arange(T) == 1) | (np.arange(T) == 4) | (slot == 2)
        assert not np.isfinite(y[lost]).any()
        assert np.array_equal(y[~lost], before[~lost])


def test_replays_with_other_rows_and_slots():
    rng, lib = np.random.default_rng(2), qfm.load()
    T = 45
    c = Case(rng, T, 6, 16, 256, [96, 20], "bf16", rng.integers(-1, 6, T))
    qfm.check(lib.qfm_graph_capture_begin(c.st.h), "capture")
    c()
    g = lib.qfm_graph_capture_end(c.st.h)
    assert g, lib.qfm_last_error().decode()
    for rep in range(4):
        bits, c.x = _kv.to_dtype(rng.standard_normal((T, 256)).astype(np.float32), "bf16")
        c.slot = rng.integers(-1, 6, T).astype(np.int32)
        c.bufs["x"].upload(bits)
        c.bufs["slot"].upload(c.slot)
        qfm.check(lib.qfm_graph_launch(g, c.st.h), "launch")
        got = c.result()
        c.check(got)
        c()
        assert all(np.array_equal(p, q) for p, q in zip(got, c.result())), rep
    assert lib.qfm_graph_destroy(g) == 0
