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
