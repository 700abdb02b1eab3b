"""The cache, attention and adapters in plain numpy: what the tests of
include/qf_attn.h and of the adapters compare against. Quantisation follows the
header's rule with one fp32 operation a step (so codes and scales are compared
for equality); everything after it is 64-bit."""
import ctypes as C

import numpy as np

import qfm

INT8, E4M3 = qfm.QFM_KV_INT8, qfm.QFM_KV_E4M3
EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}      # half a step, relative to the value


def _e4m3_table():
    b = np.arange(128)
    e, m = b >> 3, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[127] = np.nan
    return v


E4M3_POS = _e4m3_table()
CODE_VALUE = {INT8: np.arange(256).astype(np.uint8).view(np.int8).astype(np.float64),
              E4M3: np.concatenate([E4M3_POS, -E4M3_POS])}


def e4m3_encode(q):
    """The nearest E4M3 byte (ties to the even code) of finite values within +-448."""
    a = np.abs(q).astype(np.float64)
    hi = np.clip(np.searchsorted(E4M3_POS[:127], a, "left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - E4M3_POS[lo], E4M3_POS[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (code | np.where(np.signbit(q), 128, 0)).astype(np.uint8)


def quantise(x, fmt):
    """fp32 rows [..., D] -> (code bytes, fp32 scales), the header's rule."""
    x = np.asarray(x, np.float32)
    fine = np.isfinite(x).all(-1)
    y = np.where(fine[..., None], x, np.float32(0))
    s = np.abs(y).max(-1) * (np.float32(1) / np.float32(127 if fmt == INT8 else 448))
    s = np.where(s == 0, np.float32(1), s).astype(np.float32)
    q = y / s[..., None]
    assert q.dtype == np.float32
    if fmt == INT8:
        code = np.clip(np.rint(q), -127, 127).astype(np.int8).view(np.uint8)
    else:
        code = e4m3_encode(np.clip(q, -448, 448))
    code = np.where(fine[..., None], code, np.uint8(0))
    return code, np.where(fine, s, np.float32(np.nan)).astype(np.float32)


def bf16_bits(a):
    u = np.asarray(a, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def to_dtype(a, dt):
    """Values as the bits of a row type, and the fp32 values that those bits are."""
    a = np.asarray(a, np.float32)
    if dt == "f32":
        return a, a
    if dt == "bf16":
        b = bf16_bits(a)
        return b, (b.astype(np.uint32) << 16).view(np.float32)
    with np.errstate(over="ignore"):
        h = a.astype(np.float16)
    return h, h.astype(np.float32)


def from_bits(b, dt):
    return b if dt == "f32" else (b.astype(np.uint32) << 16).view(np.float32) if dt == "bf16" else b.astype(np.float32)


NP = {"f32": np.float32, "bf16": np.uint16, "f16": np.float16}


class Cache:
    """A pool of pages in numpy and on the device."""

    def __init__(self, pages, page, heads, dim, fmt, table, rng, fill=0xA5):
        self.pages, self.page, self.heads, self.dim, self.fmt = pages, page, heads, dim, fmt
        self.table = np.ascontiguousarray(table, np.int32)
        self.k = np.full((pages, heads, page, dim), fill, np.uint8)
        self.v = np.full((pages, heads, page // 4, dim, 4), fill, np.uint8)
        self.ks = np.full((pages, heads, page), np.nan, np.float32)
        self.vs = np.full((pages, heads, page), np.nan, np.float32)

    def place(self, s, p):
        """(page, token) of position p of sequence s, or None."""
        if not 0 <= s < self.table.shape[0] or p < 0 or p // self.page >= self.table.shape[1]:
            return None
        g = int(self.table[s, p // self.page])
        return (g, p % self.page) if 0 <= g < self.pages else None

    def put(self, k, v, seq, pos):
        """The header's write, row by row: k, v [T][heads][dim] fp32."""
        kc, ks = quantise(k, self.fmt)
        vc, vs = quantise(v, self.fmt)
        for t, (s, p) in enumerate(zip(seq, pos)):
            at = self.place(int(s), int(p))
            if at is not None:
                g, o = at
                self.k[g, :, o], self.ks[g, :, o] = kc[t], ks[t]
                self.v[g, :, o // 4, :, o % 4], self.vs[g, :, o] = vc[t], vs[t]

    def row(self, s, p):
        """(k, v) [heads][dim] in 64 bits, or None."""
        at = self.place(s, p)
        if at is None:
            return None
        g, o = at
        val = CODE_VALUE[self.fmt]
        return (val[self.k[g, :, o]] * self.ks[g, :, o].astype(np.float64)[:, None],
                val[self.v[g, :, o // 4, :, o % 4]] * self.vs[g, :, o].astype(np.float64)[:, None])

    def upload(self):
        self.d = {n: qfm.DevBuf.from_array(getattr(self, n)) for n in ("k", "v", "ks", "vs", "table")}
        self.c = qfm.QfmKvCache(self.d["k"].ptr, self.d["v"].ptr, self.d["ks"].ptr, self.d["vs"].ptr, self.pages, self.page,
                                self.heads, self.dim, self.fmt)
        self.s = qfm.QfmKvSeqs(self.d["table"].ptr, self.table.shape[0], self.table.shape[1])
        return C.byref(self.c), C.byref(self.s)

    def download(self):
        return {n: self.d[n].download(getattr(self, n).dtype, getattr(self, n).shape) for n in ("k", "v", "ks", "vs")}


def tables(rng, n_seq, max_pages, pages):
    """Distinct random pages for every sequence."""
    return rng.permutation(pages)[:n_seq * max_pages].reshape(n_seq, max_pages).astype(np.int32)


def strided(T, heads, dim, layout):
    """(elements, row stride, head stride) of rows laid out as [T][heads][dim], [heads][T][dim] or in a wider row."""
    if layout == "rows":
        return T * heads * dim, heads * dim, dim
    if layout == "heads":
        return T * heads * dim, dim, T * dim
    return T * (heads + 3) * (dim + 8), (heads + 3) * (dim + 8), dim + 8


def scatter(a, n, rs, hs, fill=0):
    """[T][H][D] as a flat buffer of n elements with the given strides."""
    T, H, D = a.shape
    out = np.full(n, fill, a.dtype)
    at = np.arange(T)[:, None, None] * rs + np.arange(H)[None, :, None] * hs + np.arange(D)
    out[at.ravel()] = a.ravel()
    return out, at


# ---- attention ----------------------------------------------------------------------
def fill_rows(c, s, n, rng, spread=0.5):
    """Positions 0..n-1 of sequence s: codes and scales as a writer leaves them (pages that exist only)."""
    pos = np.arange(n)
    inside = pos // c.page < c.table.shape[1]
    pos = pos[inside]
    g = c.table[s, pos // c.page]
    ok = (g >= 0) & (g < c.pages)
    g, o = g[ok], pos[ok] % c.page
    for name, sc in (("k", "ks"), ("v", "vs")):
        x = rng.standard_normal((len(g), c.heads, c.dim)).astype(np.float32)
        x *= np.exp(rng.normal(0, spread, (len(g), c.heads, 1))).astype(np.float32)
        code, scale = quantise(x, c.fmt)
        if name == "k":
            c.k[g, :, o] = code
        else:
            c.v[g, :, o // 4, :, o % 4] = code
        getattr(c, sc)[g, :, o] = scale


def tree_masks(counts, rng):
    """Masks of random trees, a node's ancestors and itself, [sum counts] uint64."""
    out = []
    for m in counts:
        t = []
        for j in range(m):
            up = int(rng.integers(-1, j)) if j else -1
            t.append((t[up] if up >= 0 else 0) | 1 << j)
        out += t
    return np.array(out, np.uint64)


def attention(c, q, row_start, ctx, tree, scale, dt):
    """(out, tolerance) in 64 bits, [T][q_heads][dim]; the tolerance of rows that no sequence has is -1.

    The tolerance, element by element, with A = sum p |v| / sum p and u = 2^-24:
      the result's own rounding, EPS[dt] |out|;
      p times the value scale in fp16 (2^-11 relative; two numbers, 2^-22, for f32), and below fp16's normal range
      half a step of 2^-24, where the largest value scale is kept at 2^6: 2^-24 of it a position at most;
      scores: a sum of D products in fp32, 6 sqrt(D) u sum |q k| (roundings that are independent pass it once in
      1e7), q as two fp16 numbers 2^-22 of it for f32, three more roundings of the scaled score and one of its
      exponent: relative errors of p, twice (numerator and sum);
      the sums over n positions in fp32, 6 sqrt(n) u each, and the joins of up to 4 waves and 128 splits, 10
      roundings each.
    """
    T, Hq, D = q.shape
    G, u = Hq // c.heads, 2.0 ** -24
    out, tol = np.full(q.shape, np.nan), np.full(q.shape, -1.0)
    val, q = CODE_VALUE[c.fmt], q.astype(np.float64)
    cap = c.table.shape[1] * c.page
    for s in range(len(ctx)):
        r0, r1 = int(row_start[s]), min(int(row_start[s + 1]), T)
        m, cx = max(r1 - r0, 0), min(max(int(ctx[s]), 0), cap)
        pos = np.arange(min(cx + m, cap))
        g = c.table[s, pos // c.page]
        ok = (g >= 0) & (g < c.pages)
        pos, g = pos[ok], g[ok]
        o = pos % c.page
        k = val[c.k[g, :, o]] * c.ks[g, :, o].astype(np.float64)[..., None]
        v = val[c.v[g, :, o // 4, :, o % 4]] * c.vs[g, :, o].astype(np.float64)[..., None]
        for i in range(m):
            bits = int(tree[r0 + i]) if tree is not None else (2 << i) - 1
            see = np.array([p < cx or bool(bits >> int(p - cx) & 1) for p in pos], bool)
            for h in range(Hq):
                kk, vv, n = k[see, h // G], v[see, h // G], int(see.sum())
                if not n:
                    out[r0 + i, h], tol[r0 + i, h] = 0.0, 0.0
                    continue
                x = kk @ q[r0 + i, h] * scale
                p = np.exp(x - x.max())
                a = p @ np.abs(vv) / p.sum()
                out[r0 + i, h] = p @ vv / p.sum()
                mag = (np.abs(kk) @ np.abs(q[r0 + i, h])).max() * scale
                eq, ep = (2.0 ** -22, 2.0 ** -22) if dt == "f32" else (0.0, 2.0 ** -11)
                dx = mag * (6 * D ** 0.5 * u + eq) + (np.abs(x).max() + 1) * 4 * u
                tol[r0 + i, h] = (EPS[dt] * np.abs(out[r0 + i, h]) + a * (ep + 2 * dx + (12 * n ** 0.5 + 20) * u) +
                                  n * 2.0 ** -24 * c.vs[g][:, h // G].max(initial=0, where=np.isfinite(c.vs[g][:, h // G])))
    return out, tol
