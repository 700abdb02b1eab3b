"""The measured cases of the cache, attention and adapter operators.

What a decode program asks of this library beside its MoE layers, on torch
device memory that the program owns:

  write   qfm_kv_write: key and value rows quantised into a paged cache
  read    qfm_kv_read: rows of that cache back as values
  attn    qfm_tree_attn: the drafted tokens (fork rows, a draft tree, one
          token) of several sequences over their cached keys and values
  lora    qfm_lora_rows: each row's own low-rank adapter added beside the
          projections that all rows share

`own` false: the same results from elementary torch operations in 32 bits.
"""
import ctypes as C
import math
import os
import random
import sys

import numpy as np
import torch

own = False

INT8, E4M3 = "int8", "e4m3"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOP = {INT8: 127.0, E4M3: 448.0}


# ---- cases --------------------------------------------------------------------------
def _write(name, rows, seqs, kv_heads, dim, page, fmt, dt):
    case = {"name": name} if name else {}
    case.update(kind="write", rows=rows, seqs=seqs, kv_heads=kv_heads, dim=dim, page=page, fmt=fmt, dt=dt)
    return case


def _read(name, rows, seqs, kv_heads, dim, page, fmt, dt):
    return {**_write(name, rows, seqs, kv_heads, dim, page, fmt, dt), "kind": "read"}


def _attn(name, seqs, ctx, nodes, heads, kv_heads, dim, page, fmt, dt, even):
    """Contexts of ctx tokens where `even`, else of ctx/2 to ctx; draft trees of up to `nodes` tokens."""
    case = {"name": name} if name else {}
    case.update(kind="attn", seqs=seqs, ctx=ctx, nodes=nodes, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                fmt=fmt, dt=dt, even=even)
    return case


def _lora(name, rows, slots, rank, k, n0, n1, n2, dt, runs):
    """Up to three projections of n0, n1, n2 outputs; the rows' adapters in `runs` runs of neighbours (0: any order)."""
    case = {"name": name} if name else {}
    case.update(kind="lora", rows=rows, slots=slots, rank=rank, k=k, n0=n0, n1=n1, n2=n2, dt=dt, runs=runs)
    return case


def listed():
    return [
        # the eight fork rows of one conversation, as the INT8 projections leave them (fp32)
        _write("write_forks8", 8, 1, 2, 256, 16, INT8, "f32"),
        # a whole prompt's keys and values
        _write("write_prompt8038", 8038, 1, 8, 128, 64, INT8, "bf16"),
        # an odd chunk read back, and a long prefix handed on
        _read("read_chunk129", 129, 1, 4, 64, 32, E4M3, "f16"),
        _read("read_prefix8038", 8038, 3, 8, 128, 64, INT8, "bf16"),
        # one token of one user, a middling context
        _attn("attn_one_1021", 1, 1021, 1, 16, 2, 256, 16, INT8, "bf16", True),
        # the fork rows of one conversation
        _attn("attn_forks8_8038", 1, 8038, 8, 16, 2, 256, 16, INT8, "bf16", True),
        # a batch of users decoding together
        _attn("attn_batch37", 37, 4099, 1, 32, 4, 128, 64, E4M3, "f16", False),
        # wide draft trees of a few users
        _attn("attn_tree61", 5, 8038, 61, 32, 8, 128, 32, INT8, "bf16", False),
        # three drafted tokens behind a book, results in the projections' own fp32
        _attn("attn_long131071", 1, 131071, 3, 16, 2, 256, 64, E4M3, "f32", True),
        # one token with an adapter on its query, key and value projections
        _lora("lora_one", 1, 8, 16, 2048, 4096, 512, 512, "bf16", 0),
        # a batch whose requests bring many adapters
        _lora("lora_batch37", 37, 24, 32, 2560, 2560, 0, 0, "f16", 0),
        # prompts of a few requests in one call
        _lora("lora_prompt2050", 2050, 6, 64, 2048, 4096, 512, 512, "bf16", 5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges: lengths over the logarithm, every head layout, format and type."""
    kind = rng.choice(["write", "read", "attn", "attn", "attn", "lora", "lora"])
    fmt, dt, page = rng.choice([INT8, E4M3]), rng.choice(["f32", "bf16", "f16"]), rng.choice([16, 32, 64, 128])
    heads, kv_heads, dim = rng.choice([(16, 2, 256), (32, 4, 128), (32, 8, 128), (16, 4, 64), (8, 8, 64), (12, 4, 128),
                                       (7, 1, 128), (8, 1, 256)])
    if kind in ("write", "read"):
        rows = _log_int(rng, 1, 8000)
        return (_write if kind == "write" else _read)(None, rows, rng.randint(1, min(rows, 9)), kv_heads, dim, page, fmt, dt)
    if kind == "attn":
        ctx, nodes = _log_int(rng, 1, 58000), _log_int(rng, 1, 64)
        # within the largest listed cases: cached values, and products of wide trees
        nodes = max(1, min(nodes, int(6e9 / (ctx * heads * dim))))
        most = min(64.0, 6e7 / (ctx * kv_heads * dim), 6e9 / (nodes * ctx * heads * dim))
        return _attn(None, _log_int(rng, 1, max(1, int(most))), ctx, nodes, heads, kv_heads, dim, page, fmt, dt, rng.random() < 0.3)
    rows = _log_int(rng, 1, 2000)
    slots = rng.randint(1, 24 if rows <= 128 else 6)
    n0, n1, n2 = rng.choice([(4096, 512, 512), (2048, 0, 0), (2560, 0, 0), (1021, 0, 0), (2048, 256, 256), (640, 640, 0)])
    return _lora(None, rows, slots, rng.choice([8, 16, 24, 32, 64]), rng.choice([512, 2048, 2560]), n0, n1, n2,
                 rng.choice(["bf16", "f16"]), rng.choice([0, 0, 1, 3, 7]) if rows <= 128 else rng.randint(1, 6))


# ---- inputs -------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(a):
    return torch.from_numpy(np.asarray(a, np.int32)).cuda()


def _lens(case):
    """Context length and draft length of each sequence."""
    r = random.Random("%(seqs)d %(ctx)d %(nodes)d" % case)
    return [(case["ctx"] if case["even"] else r.randint((case["ctx"] + 1) // 2, case["ctx"]),
             case["nodes"] if case["even"] else r.randint((case["nodes"] + 1) // 2, case["nodes"])) for _ in range(case["seqs"])]


def _normal_rows(g, rows, heads, dim, dt):
    """Rows as projections leave them: a few channels an order of magnitude over the others."""
    x = torch.randn((rows, heads, dim), device="cuda", generator=g)
    return (x * (1.0 + 9.0 * (torch.rand((heads, dim), device="cuda", generator=g) < 0.03))).to(dt)


def _codes(v, fmt):
    """A cache row's codes and scale (elementary torch, 32 bits): codes as int8, or as float8 values."""
    amax = v.abs().amax(-1)
    s = torch.where(amax > 0, amax / TOP[fmt], torch.ones_like(amax))
    q = v / s.unsqueeze(-1)
    return (q.round().clamp(-127, 127).to(torch.int8) if fmt == INT8 else q.clamp(-448, 448).to(torch.float8_e4m3fn)), s


def _cache(case, tokens, g, filled):
    """The pool of pages, with a third more pages than the sequences hold, in any order."""
    H, D, P = case["kv_heads"], case["dim"], case["page"]
    per = [-(-t // P) for t in tokens]
    pages = sum(per) + sum(per) // 3 + 1
    order = torch.randperm(pages, device="cuda", generator=g, dtype=torch.int32)
    table = torch.full((len(per), max(per)), -1, dtype=torch.int32, device="cuda")
    at = np.cumsum([0] + per)
    for i, n in enumerate(per):
        table[i, :n] = order[at[i]:at[i + 1]]
    ct = torch.int8 if case["fmt"] == INT8 else torch.float8_e4m3fn
    t = {"table": table, "k": torch.zeros((pages, H, P, D), dtype=ct, device="cuda"),
         "v": torch.zeros((pages, H, P // 4, D, 4), dtype=ct, device="cuda"),
         "ks": torch.zeros((pages, H, P), device="cuda"), "vs": torch.zeros((pages, H, P), device="cuda")}
    if filled:
        for p0 in range(0, pages, 512):
            p1 = min(pages, p0 + 512)
            x = _normal_rows(g, (p1 - p0) * P, H, D, torch.float32).reshape(p1 - p0, P, H, D).transpose(1, 2)
            t["k"][p0:p1], t["ks"][p0:p1] = _codes(x, case["fmt"])
            x = torch.randn((p1 - p0, H, P, D), device="cuda", generator=g)
            q, t["vs"][p0:p1] = _codes(x, case["fmt"])
            t["v"][p0:p1] = q.view(torch.int8).reshape(p1 - p0, H, P // 4, 4, D).transpose(3, 4).contiguous().view(ct)
    return t


def _places(case):
    """Sequence and position of each row: runs of neighbours, each behind a context of its own."""
    n, T = case["seqs"], case["rows"]
    r = random.Random("%(seqs)d %(rows)d %(page)d" % case)
    cut = [T * i // n for i in range(n + 1)]
    first = [0 if T > 64 and i == 0 else r.randint(0, 300) for i in range(n)]
    seq = np.repeat(np.arange(n), np.diff(cut))
    pos = np.concatenate([first[i] + np.arange(cut[i + 1] - cut[i]) for i in range(n)])
    return seq, pos, [int(first[i] + cut[i + 1] - cut[i]) for i in range(n)]


def _rows_inputs(case, g):
    seq, pos, tokens = _places(case)
    t = _cache(case, tokens, g, case["kind"] == "read")
    t["seq"], t["pos"] = _i32(seq), _i32(pos)
    shape, dt = (case["rows"], case["kv_heads"], case["dim"]), DT[case["dt"]]
    if case["kind"] == "write":
        t["kx"], t["vx"] = _normal_rows(g, *shape, dt), torch.randn(shape, device="cuda", generator=g).to(dt)
    else:
        t["ko"], t["vo"] = torch.zeros(shape, dtype=dt, device="cuda"), torch.zeros(shape, dtype=dt, device="cuda")
    return t


def _attn_inputs(case, g):
    lens = _lens(case)
    t = _cache(case, [c + m for c, m in lens], g, True)
    T = sum(m for _, m in lens)
    t["ctx"], t["start"] = _i32([c for c, _ in lens]), _i32(np.cumsum([0] + [m for _, m in lens]))
    r, words = np.random.RandomState(len(lens) * 1000 + T), []
    for _, m in lens:                                 # each drafted token sees its ancestors and itself
        tree = []
        for j in range(m):
            up = int(r.randint(-1, j)) if j else -1
            tree.append((tree[up] if up >= 0 else 0) | 1 << j)
        words += tree
    t["tree"] = torch.from_numpy(np.array(words, np.uint64).view(np.int64)).cuda()
    t["q"] = torch.randn((T, case["heads"], case["dim"]), device="cuda", generator=g).to(DT[case["dt"]])
    t["out"] = torch.zeros_like(t["q"])
    return t


def _lora_inputs(case, g):
    T, S, R, K, dt = case["rows"], case["slots"], case["rank"], case["k"], DT[case["dt"]]
    ns = [n for n in (case["n0"], case["n1"], case["n2"]) if n]
    r = np.random.RandomState(T * 100 + S)
    if case["runs"]:                                  # prompts: neighbours share an adapter
        slot = r.randint(0, S, case["runs"])[np.arange(T) * case["runs"] // T]
    else:                                             # a batch: any order, some rows without
        slot = r.randint(-1 if T > 1 else 0, S, T)
    t = {"slot": _i32(slot), "rank": _i32(np.maximum(1, R - r.randint(0, 2, S) * (R // 2))),
         "scale": 0.5 + torch.rand(S, device="cuda", generator=g),
         "x": torch.randn((T, K), device="cuda", generator=g).to(dt)}
    t["a"] = [(torch.randn((S, R, K), device="cuda", generator=g) / math.sqrt(K)).to(dt) for _ in ns]
    t["b"] = [(torch.randn((S, n, R), device="cuda", generator=g) * 0.05).to(dt) for n in ns]
    t["base"] = [torch.randn((T, n), device="cuda", generator=g) for n in ns]
    t["y"] = [torch.zeros((T, n), device="cuda") for n in ns]
    return t


def _inputs(case, seed):
    g = _gen(seed)
    return {"write": _rows_inputs, "read": _rows_inputs, "attn": _attn_inputs, "lora": _lora_inputs}[case["kind"]](case, g)


class State:
    """What the program keeps: its tensors, and the library's handles on them."""


def prepare(case, seed):
    st = State()
    st.case, st.t = dict(case), _inputs(case, seed)
    if own:
        _bind(st)
    return st


# ---- the framework's calls ----------------------------------------------------------
def _bind(st):
    """The structs and the argument list that a program builds once for its buffers."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-3-ocho_amd"))
    import qfm
    lib, c, t = qfm.load(), st.case, st.t
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] == "lora":
        st.l = l = qfm.QfmLora()
        l.n, l.K, l.R, l.slots = len(t["a"]), c["k"], c["rank"], c["slots"]
        l.dtype, l.rank, l.scale = qfm.QFM_DT[c["dt"]], t["rank"].data_ptr(), t["scale"].data_ptr()
        for i, b in enumerate(t["b"]):
            l.a[i], l.b[i], l.rows[i] = t["a"][i].data_ptr(), b.data_ptr(), b.shape[1]
            l.base[i], l.y[i] = t["base"][i].data_ptr(), t["y"][i].data_ptr()
        st.ws = torch.empty(max(1, lib.qfm_lora_ws_bytes(C.byref(l), c["rows"])), dtype=torch.uint8, device="cuda")
        st.args = (C.byref(l), t["x"].data_ptr(), c["k"], t["slot"].data_ptr(), c["rows"], st.ws.data_ptr(), st.ws.numel(), stream)
        st.call, st.out = lib.qfm_lora_rows, t["y"]
        return
    H, D, P = c["kv_heads"], c["dim"], c["page"]
    st.c = qfm.QfmKvCache(t["k"].data_ptr(), t["v"].data_ptr(), t["ks"].data_ptr(), t["vs"].data_ptr(), t["k"].shape[0], P, H,
                          D, qfm.QFM_KV_INT8 if c["fmt"] == INT8 else qfm.QFM_KV_E4M3)
    st.s = qfm.QfmKvSeqs(t["table"].data_ptr(), t["table"].shape[0], t["table"].shape[1])
    cache, seqs, dt = C.byref(st.c), C.byref(st.s), qfm.QFM_DT[c["dt"]]
    if c["kind"] == "attn":
        Hq, T = c["heads"], t["q"].shape[0]
        wsb = lib.qfm_tree_attn_ws_bytes(cache, c["seqs"], T, Hq, c["nodes"], c["ctx"])
        st.ws = torch.zeros(max(1, wsb), dtype=torch.uint8, device="cuda")
        st.args = (cache, seqs, t["q"].data_ptr(), t["out"].data_ptr(), dt, Hq, Hq * D, D, Hq * D, D, t["start"].data_ptr(),
                   t["ctx"].data_ptr(), t["tree"].data_ptr(), T, c["nodes"], c["ctx"], D ** -0.5, st.ws.data_ptr(), wsb, stream)
        st.call, st.out = lib.qfm_tree_attn, t["out"]
        return
    x = ("kx", "vx") if c["kind"] == "write" else ("ko", "vo")
    st.args = (cache, seqs, t[x[0]].data_ptr(), t[x[1]].data_ptr(), dt, H * D, D, t["seq"].data_ptr(), t["pos"].data_ptr(),
               c["rows"], stream)
    st.call = lib.qfm_kv_write if c["kind"] == "write" else lib.qfm_kv_read
    st.out = [t[n] for n in ("k", "ks", "v", "vs")] if c["kind"] == "write" else [t["ko"], t["vo"]]


# ---- the plain forms ----------------------------------------------------------------
def _plain_write(c, t):
    P = c["page"]
    page, off = t["table"][t["seq"].long(), t["pos"].long() // P].long(), t["pos"].long() % P
    kq, t["ks"][page, :, off] = _codes(t["kx"].float(), c["fmt"])
    vq, t["vs"][page, :, off] = _codes(t["vx"].float(), c["fmt"])
    t["k"].view(torch.int8)[page, :, off] = kq.view(torch.int8)
    t["v"].view(torch.int8)[page, :, off // 4, :, off % 4] = vq.view(torch.int8)
    return [t["k"], t["ks"], t["v"], t["vs"]]


def _plain_read(c, t):
    P, dt = c["page"], DT[c["dt"]]
    page, off = t["table"][t["seq"].long(), t["pos"].long() // P].long(), t["pos"].long() % P
    k = t["k"].view(torch.int8)[page, :, off].view(t["k"].dtype).float() * t["ks"][page, :, off].unsqueeze(-1)
    v = t["v"].view(torch.int8)[page, :, off // 4, :, off % 4].view(t["v"].dtype).float() * t["vs"][page, :, off].unsqueeze(-1)
    return [k.to(dt), v.to(dt)]


def _plain_attn(c, t):
    P, H, D, Hq = c["page"], c["kv_heads"], c["dim"], c["heads"]
    n, G, M = c["seqs"], c["heads"] // c["kv_heads"], c["nodes"]
    pages = t["table"].long().clamp(min=0)
    L = pages.shape[1] * P
    k = t["k"].view(torch.int8)[pages].view(t["k"].dtype).float() * t["ks"][pages].unsqueeze(-1)      # [n][pages][H][P][D]
    k = k.transpose(1, 2).reshape(n, H, L, D)
    v = t["v"].view(torch.int8)[pages].view(t["v"].dtype).float().transpose(4, 5).reshape(n, -1, H, P, D)
    v = (v * t["vs"][pages].unsqueeze(-1)).transpose(1, 2).reshape(n, H, L, D)
    start, ctx = t["start"].long(), t["ctx"].long()
    row = start[:-1, None] + torch.arange(M, device="cuda")
    real = row < start[1:, None]
    row = row.clamp(max=t["q"].shape[0] - 1)
    q = t["q"].float()[row].reshape(n, M, H, G, D).permute(0, 2, 3, 1, 4).reshape(n, H, G * M, D)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5).reshape(n, H, G, M, L)
    node = torch.arange(L, device="cuda") - ctx[:, None]                                            # [n][L]
    bit = (t["tree"][row][:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1                         # [n][M][L]
    seen = (node < 0)[:, None, :] | ((node >= 0) & (node < 64) & (node < (start[1:] - start[:-1])[:, None]))[:, None, :] & (bit > 0)
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(n, H, G * M, L), v).reshape(n, H, G, M, D) / l
    o = o.permute(0, 3, 1, 2, 4).reshape(n, M, Hq, D)
    return o[real].to(DT[c["dt"]])


def _plain_lora(c, t):
    S, R, K = c["slots"], c["rank"], c["k"]
    x = t["x"].float()
    mine = t["slot"].long()[:, None] == torch.arange(S, device="cuda")                              # [T][S]
    keep = mine[:, :, None] & (torch.arange(R, device="cuda") < t["rank"][:, None])                 # [T][S][R]
    w = torch.where(keep, t["scale"][:, None], torch.zeros((), device="cuda")).reshape(-1, S * R)
    return [base + ((x @ a.float().reshape(S * R, K).T) * w) @ b.float().transpose(1, 2).reshape(S * R, -1)
            for a, b, base in zip(t["a"], t["b"], t["base"])]


_PLAIN = {"write": _plain_write, "read": _plain_read, "attn": _plain_attn, "lora": _plain_lora}


def run(state):
    if own:
        if state.call(*state.args):
            raise RuntimeError("the call was refused")
        return state.out
    return _PLAIN[state.case["kind"]](state.case, state.t)


# ---- work ---------------------------------------------------------------------------
def work(case):
    """Bytes: codes, scales, rows and weights that the pass reaches, once each; operations: two a product."""
    if case["kind"] == "lora":
        T, S, R, K = case["rows"], case["slots"], case["rank"], case["k"]
        N, n = case["n0"] + case["n1"] + case["n2"], sum(1 for i in range(3) if case["n%d" % i])
        used = S * (1.0 - (1.0 - 1.0 / S) ** (case["runs"] or T))
        return {"bytes": used * R * (n * K + N) * 2.0 + T * (2.0 * K + 8.0 * N), "flops": 2.0 * T * R * (n * K + N)}
    D, H, size = case["dim"], case["kv_heads"], 4 if case["dt"] == "f32" else 2
    if case["kind"] != "attn":
        return {"bytes": float(case["rows"] * (2 * H * (D * (1 + size) + 4) + 8)), "flops": 0.0}
    lens, Hq = _lens(case), case["heads"]
    return {"bytes": float(sum((c + m) * 2 * H * (D + 4) + m * 2 * Hq * D * size for c, m in lens)),
            "flops": float(sum(4 * m * (c + m) * Hq * D for c, m in lens))}


# ---- exact --------------------------------------------------------------------------
def _e4m3_64(q):
    """The nearest E4M3 number (ties to the even one) of values within +-448."""
    e = torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(q / step) * step


def _exact_write(case, t):
    """Scales in 64 bits; codes of the definition, which divides by the 32-bit scale and rounds the quotient to 32 bits."""
    P, out = case["page"], []
    seq, pos = t["seq"].tolist(), t["pos"].tolist()
    page = torch.tensor([int(p) for p in t["table"].cpu()[seq, [x // P for x in pos]]], device="cuda")
    off = torch.tensor([x % P for x in pos], device="cuda")
    for name in ("k", "v"):
        x = t[name + "x"].double()
        s = x.abs().amax(-1) / TOP[case["fmt"]]
        s32 = s.float().double()
        q = (x / s32.unsqueeze(-1)).float().double()
        q = torch.round(q) if case["fmt"] == INT8 else _e4m3_64(q)
        code = torch.zeros(t[name].shape, dtype=torch.float64, device="cuda")
        if name == "k":
            code[page, :, off] = q
        else:
            code[page, :, off // 4, :, off % 4] = q
        scale = torch.zeros(t[name + "s"].shape, dtype=torch.float64, device="cuda")
        scale[page, :, off] = s
        out += [code, scale]
    return out


def _exact_rows(case, t, seq, pos):
    """Rows (seq, pos) of the cache in 64 bits, [rows][heads][dim]."""
    P = case["page"]
    page, off = t["table"][seq, pos // P].long(), pos % P
    k = t["k"].view(torch.int8)[page, :, off].view(t["k"].dtype).double() * t["ks"][page, :, off].double().unsqueeze(2)
    v = t["v"].view(torch.int8)[page, :, off // 4, :, off % 4].view(t["v"].dtype).double()
    return k, v * t["vs"][page, :, off].double().unsqueeze(2)


def _exact_attn(case, t):
    G, D, out, at = case["heads"] // case["kv_heads"], case["dim"], [], 0
    tree = t["tree"].cpu().numpy().view(np.uint64).tolist()
    for s, (ctx, m) in enumerate(_lens(case)):
        pos = torch.arange(ctx + m, device="cuda")
        k, v = _exact_rows(case, t, torch.full_like(pos, s), pos)
        see = torch.ones((m, ctx + m), dtype=torch.bool)
        for i in range(m):
            see[i, ctx:] = torch.tensor([bool(tree[at + i] >> j & 1) for j in range(m)])
        see = see.cuda()
        q = t["q"][at:at + m].double()
        o = torch.empty_like(q)
        for h in range(case["heads"]):
            w = (q[:, h] @ k[:, h // G].T.contiguous() / math.sqrt(D)).masked_fill(~see, -math.inf)
            o[:, h] = torch.softmax(w, 1) @ v[:, h // G].contiguous()
        out.append(o)
        at += m
    return torch.cat(out)


def _exact_lora(case, t):
    out = []
    for a, b, base in zip(t["a"], t["b"], t["base"]):
        y = base.double()
        for s in range(case["slots"]):
            rows, r = (t["slot"] == s).nonzero()[:, 0], int(t["rank"][s])
            if len(rows):
                h = t["x"][rows].double() @ a[s, :r].double().T.contiguous()
                y[rows] += float(t["scale"][s]) * (h @ b[s, :, :r].double().T.contiguous())
        out.append(y)
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "write":
        return _exact_write(case, t)
    if case["kind"] == "read":
        return list(_exact_rows(case, t, t["seq"].long(), t["pos"].long()))
    return (_exact_attn if case["kind"] == "attn" else _exact_lora)(case, t)
