"""Operators over a paged KV cache, as a serving loop with many sequences calls
them, as cases that can be timed and compared:

  append  per-head norms of queries and keys, the position rotation and the store
          of keys and values into pages (kv_paged_append)
  chunk   the same into pages of 8 bits, quantised as they are written, and the
          whole context read back for the chunk's attention (kv_paged_append,
          kv_paged_read)
  read    cached sequences gathered out of their pages, 8 bits dequantised
          (kv_paged_read)
  paged   attention of new tokens over the pages, 16 or 8 bits (sdpa_paged)

Shapes are those of the package's decoder (32 query and 8 KV heads of 64, and 14
and 2) and generic ones around them; sequences of a batch have lengths of their
own, and their pages lie anywhere in the pool.

``own`` False computes each operator with elementary torch operations in 32 bits
(64 for angles, and for keys next to a quantisation border), ``own`` True calls the
package.  ``exact`` is the definition in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
PAGES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}
EPS = 1e-6
# the largest listed cases: a long batch's attention, and a batch of prompts appended
MOST_FLOPS = 4.0e9
MOST_BYTES = 4.6e8


def listed():
    return [
        # one token of one sequence of the package's decoder: latency
        dict(name="append_1x1", kind="append", n=1, t=1, s=600, hq=32, hkv=8, hd=64, page=16, norm=False, cache="same", dtype="bf16"),
        # one token for each of a full batch, queries and keys normed
        dict(name="append_64x1_norm_f16", kind="append", n=64, t=1, s=900, hq=32, hkv=8, hd=128, page=32, norm=True, cache="same", dtype="f16"),
        # the largest: a batch of ragged prompts
        dict(name="append_4x4001_norm", kind="append", n=4, t=4001, s=4001, hq=32, hkv=8, hd=128, page=64, norm=True, cache="same", dtype="bf16"),
        # a piece of a prompt behind its first pieces, 8 bits
        dict(name="chunk_2x256_int8", kind="chunk", n=2, t=256, s=1277, hq=32, hkv=8, hd=64, page=16, norm=False, cache="int8", dtype="bf16"),
        # long pieces of a batch, normed, the other 8-bit type
        dict(name="chunk_8x1024_e4m3", kind="chunk", n=8, t=1024, s=4096, hq=32, hkv=8, hd=128, page=64, norm=True, cache="e4m3", dtype="bf16"),
        # a shared prefix gathered for one prompt
        dict(name="read_1x500", kind="read", n=1, s=500, hq=14, hkv=2, hd=64, page=16, cache="same", dtype="bf16"),
        # long cached contexts of a batch dequantised
        dict(name="read_8x8000_int8", kind="read", n=8, s=8000, hq=32, hkv=8, hd=128, page=32, cache="int8", dtype="bf16"),
        # one decoded token of one sequence of the package's decoder: latency
        dict(name="paged_1x1_600", kind="paged", n=1, l=1, s=600, hq=32, hkv=8, hd=64, page=16, cache="same", dtype="bf16"),
        # a decoding step of a serving batch
        dict(name="paged_16x1_4000", kind="paged", n=16, l=1, s=4000, hq=32, hkv=8, hd=128, page=64, cache="same", dtype="bf16"),
        # one sequence with a very long context in 8 bits
        dict(name="paged_1x1_60000_int8", kind="paged", n=1, l=1, s=60001, hq=32, hkv=8, hd=128, page=32, cache="int8", dtype="bf16"),
        # a few drafted tokens at once, no shared heads
        dict(name="paged_8x4_3000_f16", kind="paged", n=8, l=4, s=3003, hq=32, hkv=32, hd=64, page=128, cache="same", dtype="f16"),
        # the largest: a full batch with long contexts in 8 bits
        dict(name="paged_32x1_8000_e4m3", kind="paged", n=32, l=1, s=8000, hq=32, hkv=8, hd=128, page=16, cache="e4m3", dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(("append", "append", "chunk", "read", "paged", "paged", "paged"))
        hq = rng.choice((8, 14, 16, 32, 40))
        case = dict(kind=kind, n=_log(rng, 1, 64), hq=hq, hkv=rng.choice([h for h in (2, 8, hq) if hq % h == 0]),
                    hd=rng.choice((64, 128)), page=rng.choice((16, 32, 48, 64, 128)), dtype=rng.choice(("bf16", "bf16", "f16")),
                    cache=rng.choice(("int8", "e4m3") if kind == "chunk" else ("same", "int8", "e4m3")))
        if kind == "append":
            # single tokens, drafted ones, whole prompts
            t = rng.choice((1, 1, _log(rng, 1, 16), _log(rng, 16, 8000)))
            case.update(t=t, s=t + _log(rng, 1, 1000), norm=rng.random() < 0.5, cache="same")
        elif kind == "chunk":
            t = _log(rng, 1, 2048)
            case.update(t=t, s=t + _log(rng, 1, 8000), norm=rng.random() < 0.5)
        elif kind == "read":
            case.update(s=_log(rng, 16, 30000))
        else:
            l = rng.choice((1, 1, 1, _log(rng, 1, 8)))
            case.update(l=l, s=l + _log(rng, 1, 60000))
        w = work(case)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and _held(case) <= 1.5e9:
            return case


def _held(case):
    """Bytes of the pages that a state holds, about."""
    return case["n"] * case["hkv"] * (case["s"] + case["page"]) * case["hd"] * 4


def _lens(case):
    """Keys of each sequence: the first has all s, the others down to half of it."""
    least = max(case.get("t", 1), case.get("l", 1))
    return [max(least, int(case["s"] * (1 - 0.5 * (b * 0.618034 % 1.0)))) for b in range(case["n"])]


def _tokens(case):
    """Tokens appended to each sequence: the first has all t, the others down to half of it."""
    return [max(1, int(case["t"] * (1 - 0.5 * (b * 0.381966 % 1.0)))) for b in range(case["n"])]


def work(case):
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    keys = sum(_lens(case)) * hkv
    one = 2 if case["cache"] == "same" else 1
    row = 2 * hd * one + (0 if one == 2 else 8)          # a key and its value, and their scales
    if case["kind"] == "paged":
        rows = case["n"] * hq * case["l"]
        return dict(bytes=keys * row + rows * (4 * hd + 4), flops=4 * keys * (hq // hkv) * case["l"] * hd)
    read = dict(bytes=keys * (row + 4 * hd), flops=2 * keys * hd)
    if case["kind"] == "read":
        return read
    tokens = sum(_tokens(case))
    # the rows of q, k and v read, q and the cache's rows written; norm and rotation of q and k
    got = dict(bytes=tokens * (2 * (hq + 2 * hkv) * hd + 2 * hq * hd + hkv * row), flops=10 * tokens * (hq + hkv) * hd)
    if case["kind"] == "chunk":
        got = {k: got[k] + read[k] for k in got}
    return got


# ------------------------------------------------------------------ inputs

def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, device=DEV, generator=g) * std).to(dtype)


def _filled(case, g, pages):
    """Pages of one cache with everything in them: (pages, scales or None)."""
    x = _randn(g, (pages, case["hkv"], case["page"], case["hd"]), DTYPES[case["dtype"]])
    if case["cache"] == "same":
        return x, None
    top = x.float().abs().amax(-1, keepdim=True)
    y = x.float() * LARGEST[case["cache"]] / top
    y = y.round().to(torch.int8) if case["cache"] == "int8" else y.to(torch.float8_e4m3fn)
    return y, (top / LARGEST[case["cache"]])[..., 0].contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, n, page, dt = case["kind"], case["n"], case["page"], DTYPES[case["dtype"]]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    lens = _lens(case)
    need = [-(-L // page) for L in lens]
    pool = sum(need) + 3
    st = dict(case, kv_len=torch.tensor(lens, dtype=torch.int32, device=DEV))
    # every sequence's pages lie anywhere in the pool, and its table is longer than they are
    order = torch.randperm(pool, device=DEV, generator=g).to(torch.int32)
    table = torch.full((n, max(need) + 2), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    st["table"] = table
    st["k"], st["ks"] = _filled(case, g, pool)
    st["v"], st["vs"] = _filled(case, g, pool)
    if kind == "paged":
        # as the projections leave them: [n, l, heads, hd], seen through a transposed view
        st["q"] = _randn(g, (n, case["l"], hq, hd), dt).transpose(1, 2)
    if kind in ("append", "chunk"):
        tokens = _tokens(case)
        st["qkv"] = _randn(g, (n, case["t"], (hq + 2 * hkv) * hd), dt)
        st["lens"] = torch.tensor(tokens, dtype=torch.int32, device=DEV)
        st["pos0"] = torch.tensor([L - t for L, t in zip(lens, tokens)], dtype=torch.int32, device=DEV)
        st["inv_freq"] = (10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)).float()
        # the norms' weights as training leaves them, around one
        st["qw"], st["kw"] = (1 + _randn(g, (hd,), torch.float32, 0.2)).to(dt), (1 + _randn(g, (hd,), torch.float32, 0.2)).to(dt)
        if not case["norm"]:
            st["qw"] = st["kw"] = None
    return st


# ------------------------------------------------------------- the package

def _run_own(st):
    from kuillm_amd import ops
    scales = dict(k_scale=st["ks"], v_scale=st["vs"])
    if st["kind"] == "paged":
        out, lse = ops.sdpa_paged(st["q"], st["k"], st["v"], st["table"], st["kv_len"], return_lse=True, **scales)
        return dict(out=out, lse=lse)
    got = {}
    if st["kind"] != "read":
        got["q"] = ops.kv_paged_append(st["qkv"], st["inv_freq"], st["pos0"], st["k"], st["v"], st["table"], lens=st["lens"],
                                       q_norm=st["qw"], k_norm=st["kw"], eps=EPS, **scales)
        if st["kind"] == "append":
            return dict(got, k=st["k"], v=st["v"])
    k, v = ops.kv_paged_read(st["k"], st["v"], st["table"], st["kv_len"], length=st["s"], dtype=DTYPES[st["dtype"]], **scales)
    return dict(got, k=k, v=v)


# --------------------------------------------------------- the plain forms

def _gathered(pages, scale, table, s):
    """Values in 32 bits [n, hkv, s, hd] of the first s slots (absent pages' are whatever page 0 holds)."""
    P, hkv, page, hd = pages.shape
    j = torch.arange(s, device=DEV)
    at = table.long().clamp(min=0)[:, j // page]                                    # [n, s]
    x = pages[at, :, j % page].float()                                              # [n, s, hkv, hd]
    if scale is not None:
        x = x * scale[at, :, j % page][..., None]
    return x.transpose(1, 2)


def _quantised(x, cache):
    """(values of the cache's type, scales) of rows in 64 bits."""
    top = x.abs().amax(-1, keepdim=True)
    y = x * LARGEST[cache] / torch.where(top > 0, top, 1.0)
    y = y.round().to(torch.int8) if cache == "int8" else y.to(torch.float8_e4m3fn)
    return y, (top[..., 0] / LARGEST[cache]).float()


def _plain_append(st):
    n, t, hq, hkv, hd, page = (st[x] for x in ("n", "t", "hq", "hkv", "hd", "page"))
    i = torch.arange(t, device=DEV)
    pos = st["pos0"].long()[:, None] + i                                             # [n, t]
    ang = pos.double()[..., None] * st["inv_freq"].double()
    cos, sin = ang.cos()[:, :, None], ang.sin()[:, :, None]
    x = st["qkv"].view(n, t, hq + 2 * hkv, hd)
    q, k, v = x[:, :, :hq].float(), x[:, :, hq:hq + hkv], x[:, :, hq + hkv:]
    k = k.float() if st["cache"] == "same" else k.double()
    rotated = []
    for y, w in ((q, st["qw"]), (k, st["kw"])):
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.to(y.dtype)
        a, b = y[..., :hd // 2], y[..., hd // 2:]
        c, s = cos.to(y.dtype), sin.to(y.dtype)
        rotated.append(torch.cat([a * c - b * s, b * c + a * s], -1))
    q, k = rotated
    there = i < st["lens"][:, None]
    q = torch.where(there[:, :, None, None], q, 0.0).to(st["qkv"].dtype).transpose(1, 2)
    b, i = there.nonzero(as_tuple=True)
    where = pos[b, i]
    at = st["table"].long()[b, where // page]
    for row, pages, scale in ((k, st["k"], st["ks"]), (v, st["v"], st["vs"])):
        row = row[b, i]
        if scale is None:
            pages[at, :, where % page] = row.to(pages.dtype)
        else:
            pages[at, :, where % page], scale[at, :, where % page] = _quantised(row.double(), st["cache"])
    return q


def _plain_read(st):
    behind = torch.arange(st["s"], device=DEV) >= st["kv_len"][:, None]
    got = []
    for pages, scale in ((st["k"], st["ks"]), (st["v"], st["vs"])):
        x = _gathered(pages, scale, st["table"], st["s"])
        got.append(torch.where(behind[:, None, :, None], 0.0, x).to(DTYPES[st["dtype"]]))
    return dict(k=got[0], v=got[1])


def _plain_paged(st):
    q, l, s, hkv = st["q"].float(), st["l"], st["s"], st["hkv"]
    n, hq, _, hd = q.shape
    k, v = (_gathered(p, sc, st["table"], s).contiguous() for p, sc in ((st["k"], st["ks"]), (st["v"], st["vs"])))
    last = st["kv_len"].long()[:, None] - l + torch.arange(l, device=DEV)
    seen = torch.arange(s, device=DEV) <= last[:, :, None]                           # [n, l, s]
    x = torch.matmul(q.reshape(n, hkv, hq // hkv * l, hd), k.transpose(2, 3).contiguous()) / math.sqrt(hd)
    x = x.view(n, hkv, hq // hkv, l, s).masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-3e38)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    lse = (top + total.log()).view(n, hq, l)
    x = x.div_(torch.where(total > 0, total, 1.0))
    out = torch.matmul(x.view(n, hkv, hq // hkv * l, s), v)
    return dict(out=out.view(n, hq, l, hd).to(st["q"].dtype), lse=lse)


def run(state):
    if own:
        return _run_own(state)
    if state["kind"] == "paged":
        return _plain_paged(state)
    if state["kind"] == "read":
        return _plain_read(state)
    q = _plain_append(state)
    if state["kind"] == "append":
        return dict(q=q, k=state["k"], v=state["v"])
    return dict(_plain_read(state), q=q)


# ------------------------------------------------------ definitions, 64 bits

def _to_grid(y, cache):
    """The nearest value of the 8-bit type, ties to the even one."""
    if cache == "int8":
        return y.round()
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (y / step).round() * step


def _rows(st, name, b, L):
    """One sequence's rows [hkv, L, hd] as numbers."""
    page = st["page"]
    pages, scale = st[name], st[name + "s"]
    got = []
    for j, p in enumerate(st["table"][b, :-(-L // page)].tolist()):
        m = min(page, L - j * page)
        x = pages[p, :, :m].double()
        got.append(x if scale is None else x * scale[p, :, :m, None].double())
    return torch.cat(got, 1)


def exact(case, seed):
    st = prepare(case, seed)
    kind, n, hq, hkv, hd, s = (case[x] for x in ("kind", "n", "hq", "hkv", "hd", "s"))
    lens, group = _lens(case), case["hq"] // case["hkv"]
    if kind == "paged":
        l, outs, lses = case["l"], [], []
        for b, L in enumerate(lens):
            k, v = _rows(st, "k", b, L), _rows(st, "v", b, L)
            seen = torch.ones(l, L, dtype=torch.bool, device=DEV).tril(L - l)
            for h in range(hq):
                x = (st["q"][b, h].double() @ k[h // group].t().contiguous()) / math.sqrt(hd)
                x = torch.where(seen, x, -math.inf)
                lses.append(torch.logsumexp(x, 1))
                outs.append(torch.softmax(x, 1) @ v[h // group])
        return dict(out=torch.stack(outs).view(n, hq, l, hd), lse=torch.stack(lses).view(n, hq, l))
    new = {}
    if kind != "read":
        t, tokens, page = case["t"], _tokens(case), case["page"]
        qs = torch.zeros(n, hq, t, hd, dtype=torch.float64, device=DEV)
        for b, m in enumerate(tokens):
            x = st["qkv"][b, :m].double().view(m, hq + 2 * hkv, hd).transpose(0, 1)
            turn = torch.arange(lens[b] - m, lens[b], device=DEV).double()[:, None] * st["inv_freq"].double()
            turn = torch.polar(torch.ones_like(turn), turn)

            def placed(y, w):
                if w is not None:
                    y = w.double() * y / ((y ** 2).mean(-1, keepdim=True) + EPS).sqrt()
                z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous()) * turn
                return torch.cat([z.real, z.imag], -1)

            qs[b, :, :m] = placed(x[:hq], st["qw"])
            new[b] = placed(x[hq:hq + hkv], st["kw"]), x[hq + hkv:]
        if kind == "append":
            k, v = st["k"].double(), st["v"].double()
            for b, m in enumerate(tokens):
                for i in range(0, lens[b] // page + 1):
                    lo, hi = max(lens[b] - m, i * page), min(lens[b], (i + 1) * page)
                    if lo < hi:
                        p = int(st["table"][b, i])
                        for c, rows in ((k, new[b][0]), (v, new[b][1])):
                            c[p, :, lo - i * page:hi - i * page] = rows[:, lo - lens[b] + m:hi - lens[b] + m]
            return dict(q=qs, k=k, v=v)
    got = {}
    for x, name in enumerate("kv"):
        got[name] = torch.zeros(n, hkv, s, hd, dtype=torch.float64, device=DEV)
        for b, L in enumerate(lens):
            got[name][b, :, :L] = _rows(st, name, b, L)
            if kind == "chunk":
                rows = new[b][x]
                top = rows.abs().amax(-1, keepdim=True)
                unit = torch.where(top > 0, top, 1.0) / LARGEST[case["cache"]]
                got[name][b, :, L - rows.shape[1]:L] = _to_grid(rows * LARGEST[case["cache"]] / torch.where(top > 0, top, 1.0), case["cache"]) * unit
    if kind == "chunk":
        got["q"] = qs
    return got
