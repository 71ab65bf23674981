"""Operators over a KV cache that a serving loop with drafted tokens and a
bounded cache calls, as cases that can be timed and compared:

  tree    attention of a tree of drafted tokens over the cache (sdpa_tree)
  commit  greedy acceptance of a drafted branch and the move of its cache rows
          behind the context, for every layer (tree_accept, kv_tree_commit)
  accum   attention that adds every key's weight to a running sum, for single
          tokens and for prompts (sdpa_decode_accum)
  evict   a cache cut down to a budget by those sums (kv_evict)

Shapes are those of the package's decoder (32 query and 8 KV heads of 64) and
generic ones around them; sequences of a batch have lengths of their own.

``own`` False computes each operator with elementary torch operations in 32
bits, ``own`` True calls the package.  ``exact`` is the definition in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# the largest listed cases: the 64-node trees of 16 sequences
MOST_FLOPS = 1.4e11
MOST_BYTES = 7.0e8
VOCAB = 32000


def listed():
    return [
        # one sequence of the package's decoder, a small tree, a short context: latency
        dict(name="tree_1x8_500", kind="tree", n=1, hq=32, hkv=8, hd=64, t=8, s=508, dtype="bf16"),
        # no shared heads, a narrow tree, f16
        dict(name="tree_4x13_2000_f16", kind="tree", n=4, hq=32, hkv=32, hd=128, t=13, s=2013, dtype="f16"),
        # a serving batch with middling trees
        dict(name="tree_8x26_4000", kind="tree", n=8, hq=32, hkv=8, hd=128, t=26, s=4026, dtype="bf16"),
        # one sequence with a very long context and a wide tree
        dict(name="tree_1x64_60000", kind="tree", n=1, hq=32, hkv=8, hd=128, t=64, s=60001, dtype="bf16"),
        # the largest: a batch of 16 with wide trees
        dict(name="tree_16x64_8000", kind="tree", n=16, hq=32, hkv=8, hd=128, t=64, s=8064, dtype="bf16"),
        # the branch accepted for one sequence, the decoder's 16 layers
        dict(name="commit_1x8", kind="commit", n=1, layers=16, hkv=8, hd=64, t=8, s=508, dtype="bf16"),
        # the branches accepted for a batch of 16, wide trees
        dict(name="commit_16x64", kind="commit", n=16, layers=16, hkv=8, hd=128, t=64, s=700, dtype="bf16"),
        # one decoded token of one sequence of the package's decoder: latency
        dict(name="accum_1x1_600", kind="accum", n=1, hq=32, hkv=8, hd=64, l=1, s=600, dtype="bf16"),
        # one decoded token for each of 16 sequences with long caches
        dict(name="accum_16x1_4000", kind="accum", n=16, hq=32, hkv=8, hd=128, l=1, s=4000, dtype="bf16"),
        # a whole prompt, its weights summed for the first cut
        dict(name="accum_prompt_1999_f16", kind="accum", n=1, hq=32, hkv=8, hd=64, l=1999, s=1999, dtype="f16"),
        # the regular cut of one sequence: 64 tokens over the budget
        dict(name="evict_1x576", kind="evict", n=1, hkv=8, hd=64, s=576, budget=512, recent=64, fresh=False, dtype="bf16"),
        # the first cut after long prompts of a batch
        dict(name="evict_8x8000", kind="evict", n=8, hkv=8, hd=128, s=8000, budget=2048, recent=128, fresh=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(("tree", "tree", "tree", "commit", "accum", "accum", "evict"))
        hq = rng.choice((8, 14, 16, 32, 40))
        case = dict(kind=kind, n=_log(rng, 1, 32), hkv=rng.choice([h for h in (2, 8, hq) if hq % h == 0]),
                    hd=rng.choice((64, 128)), dtype=rng.choice(("bf16", "bf16", "f16")))
        if kind == "tree":
            t = _log(rng, 1, 128)
            case.update(hq=hq, t=t, s=t + _log(rng, 16, 60000))
        elif kind == "commit":
            t = _log(rng, 1, 128)
            case.update(layers=_log(rng, 1, 32), t=t, s=t + _log(rng, 16, 1000))
        elif kind == "accum":
            # single tokens, pieces of a prompt, whole prompts
            s = _log(rng, 16, 30000)
            l = rng.choice((1, 1, _log(rng, 1, min(s, 2048)), min(s, 3000)))
            case.update(hq=hq, l=l, s=s)
        else:
            s = _log(rng, 64, 16000)
            budget = max(1, int(s * rng.uniform(0.1, 1.0)))
            case.update(s=s, budget=budget, recent=rng.randrange(0, budget // 2 + 1), fresh=rng.random() < 0.5)
        w = work(case)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and _held(case) <= 6e9:
            return case


def _held(case):
    """Bytes of the caches that a state holds."""
    return case["n"] * case.get("layers", 1) * case["hkv"] * _capacity(case) * case["hd"] * 4


def _capacity(case):
    return case["s"] + 37


def _lens(case):
    """Keys of each sequence: the first has all s, the others down to half of it."""
    least = max(case.get("t", 1), case.get("l", 1))
    return [max(least, int(case["s"] * (1 - 0.5 * (b * 0.618034 % 1.0)))) for b in range(case["n"])]


def _evicted(case, L):
    """About how many rows of a KV head move: the kept ones behind the budget."""
    over = L - case["budget"]
    if over <= 0:
        return 0
    r = min(case["recent"], over)
    return r + (case["budget"] - case["recent"]) * (over - r) / max(1, L - case["recent"])


def work(case):
    n, hkv, hd = case["n"], case["hkv"], case["hd"]
    lens = _lens(case)
    row = 2 * hd * 2                                     # bytes of one key and its value
    if case["kind"] == "tree":
        hq, t = case["hq"], case["t"]
        return dict(bytes=sum(lens) * hkv * row + n * hq * t * (4 * hd + 4), flops=4 * hq * t * hd * sum(lens))
    if case["kind"] == "commit":
        # about two nodes of a branch are accepted, whose rows are read and written
        return dict(bytes=n * case["t"] * 20 + n * case["layers"] * hkv * 2 * row * 2, flops=0)
    if case["kind"] == "accum":
        hq, l = case["hq"], case["l"]
        seen = sum(l * (L - l) + l * (l + 1) // 2 for L in lens)     # pairs of a query and a key
        return dict(bytes=sum(lens) * hkv * (row + 8) + n * hq * l * (4 * hd + 4), flops=4 * hq * hd * seen)
    moved = sum(_evicted(case, L) for L in lens)
    return dict(bytes=sum(lens) * hkv * 8 + n * hkv * _capacity(case) * 8 + moved * hkv * 2 * row, flops=0)


# ------------------------------------------------------------------ inputs

def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, device=DEV, generator=g) * std).to(dtype)


def _trees(case, g):
    """Drafted trees: node 0 is the root, every other hangs on an earlier one;
    the sequences behind the first have fewer nodes (the others are absent)."""
    n, t = case["n"], case["t"]
    i = torch.arange(t, device=DEV)
    parent = (torch.rand(n, t, device=DEV, generator=g) * i).long().clamp(max=t - 1)
    parent = torch.minimum(parent, (i - 1).clamp(min=0))
    parent[:, 0] = -1
    nodes = torch.tensor([max(1, t - b % 3) for b in range(n)], device=DEV)
    return torch.where(i < nodes[:, None], parent, -2).to(torch.int32)


def _drafts(case, g, parent):
    """Drafted tokens, and the model's choice at every node: mostly a child's token."""
    n, t = parent.shape
    tokens = torch.randint(0, VOCAB, (n, t), device=DEV, generator=g)
    child = parent.long()[:, None, :] == torch.arange(t, device=DEV)[None, :, None]       # [n, node, child]
    likes = torch.rand(n, t, t, device=DEV, generator=g) * child
    follow = child.any(2) & (torch.rand(n, t, device=DEV, generator=g) < 0.8)
    other = torch.randint(0, VOCAB, (n, t), device=DEV, generator=g)
    return tokens, torch.where(follow, tokens.gather(1, likes.argmax(2)), other)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, n, hkv, hd, dt = case["kind"], case["n"], case["hkv"], case["hd"], DTYPES[case["dtype"]]
    cap = _capacity(case)
    st = dict(case, kv_len=torch.tensor(_lens(case), dtype=torch.int32, device=DEV))
    batch = n * case.get("layers", 1)
    st["k"] = _randn(g, (batch, hkv, cap, hd), dt)
    st["v"] = _randn(g, (batch, hkv, cap, hd), dt)
    if kind in ("tree", "accum"):
        rows = case["t" if kind == "tree" else "l"]
        # as the projections leave them: [n, rows, heads, hd], seen through a transposed view
        st["q"] = _randn(g, (n, rows, case["hq"], hd), dt).transpose(1, 2)
    if kind in ("tree", "commit"):
        st["parent"] = _trees(case, g)
    if kind == "commit":
        st["tokens"], st["target"] = _drafts(case, g, st["parent"])
    if kind == "accum":
        st["acc"] = torch.rand(n, hkv, cap, device=DEV, generator=g)
    if kind == "evict":
        # sums of earlier attention: a few keys weigh much, some nothing, the first most
        acc = torch.exp(1.5 * torch.randn(n, hkv, cap, device=DEV, generator=g))
        acc *= torch.rand(n, hkv, cap, device=DEV, generator=g) > 0.05
        acc[:, :, :4] += 100.0
        pos = torch.arange(cap, device=DEV).expand(n, hkv, cap)
        if not case["fresh"]:
            # cut before: the slots under the budget hold earlier positions in any order
            m = min(case["budget"], cap)
            order = torch.rand(n, hkv, m, device=DEV, generator=g).argsort(-1)
            pos = torch.cat([order, pos[:, :, m:]], 2) + 1000
        st["acc"], st["pos"] = acc, pos.to(torch.int32).contiguous()
        st["acc_out"], st["pos_out"] = torch.empty_like(acc), torch.empty_like(st["pos"])
        st["len_out"] = torch.empty_like(st["kv_len"])
    return st


# ------------------------------------------------------------- the package

def _run_own(st):
    from kuillm_amd import ops
    if st["kind"] == "tree":
        out, lse = ops.sdpa_tree(st["q"], st["k"], st["v"], st["parent"], kv_len=st["kv_len"], return_lse=True)
        return dict(out=out, lse=lse)
    if st["kind"] == "commit":
        path, count, follow = ops.tree_accept(st["tokens"], st["parent"], st["target"])
        kv_len = ops.kv_tree_commit(st["k"], st["v"], path, st["kv_len"], st["t"])
        return dict(k=st["k"], v=st["v"], path=path, count=count, follow=follow, kv_len=kv_len)
    if st["kind"] == "accum":
        out, lse = ops.sdpa_decode_accum(st["q"], st["k"], st["v"], st["acc"], kv_len=st["kv_len"], return_lse=True)
        return dict(out=out, lse=lse, acc=st["acc"])
    ops.kv_evict(st["k"], st["v"], st["acc"], st["pos"], st["kv_len"], st["budget"], st["recent"],
                 acc_out=st["acc_out"], pos_out=st["pos_out"], len_out=st["len_out"])
    return dict(k=st["k"], v=st["v"], acc=st["acc_out"], pos=st["pos_out"], kv_len=st["len_out"])


# --------------------------------------------------------- the plain forms

def _ancestors(parent):
    """(seen [n, t, t]: node j is i or an ancestor of it, present [n, t])."""
    n, t = parent.shape
    i = torch.arange(t, device=DEV)
    sound = (parent >= -1) & (parent < i)
    up = ((parent[:, :, None] == i) & sound[:, :, None]).double()
    seen = torch.linalg.matrix_power(up + torch.eye(t, dtype=torch.float64, device=DEV), t) > 0
    present = ~(seen & ~sound[:, None, :]).any(2)
    return seen & present[:, :, None], present


def _weights(q, k, visible):
    """Softmax weights in 32 bits [n, hkv, G, l, s] of the visible keys, and the LSE."""
    n, hq, l, e = q.shape
    hkv, s = k.shape[1], k.shape[2]
    qf = q.float().reshape(n, hkv, hq // hkv * l, e)
    x = torch.matmul(qf, k.float().transpose(2, 3).contiguous()) / math.sqrt(e)
    x = x.view(n, hkv, hq // hkv, l, s).masked_fill_(~visible[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-3e38)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    lse = (top + total.log()).view(n, hq, l)
    return x.div_(torch.where(total > 0, total, 1.0)), lse


def _mix(p, v, dtype):
    n, hkv, G, l, s = p.shape
    o = torch.matmul(p.view(n, hkv, G * l, s), v.float())
    return o.view(n, hkv * G, l, v.shape[-1]).to(dtype)


def _plain_tree(st):
    q, L, t, s = st["q"], st["kv_len"].long(), st["t"], st["s"]
    seen, present = _ancestors(st["parent"])
    j = torch.arange(s, device=DEV)
    node = j - (L[:, None] - t)                              # [n, s]: the tree's node of a key
    tree = seen.gather(2, node.clamp(0, t - 1)[:, None, :].expand(-1, t, -1)) & (node < t)[:, None, :]
    visible = torch.where((node < 0)[:, None, :], present[:, :, None], tree)
    p, lse = _weights(q, st["k"][:, :, :s], visible)
    return dict(out=_mix(p, st["v"][:, :, :s], q.dtype), lse=lse)


def _plain_accum(st):
    q, L, l, s = st["q"], st["kv_len"].long(), st["l"], st["s"]
    last = L[:, None] - l + torch.arange(l, device=DEV)
    visible = torch.arange(s, device=DEV) <= last[:, :, None]
    p, lse = _weights(q, st["k"][:, :, :s], visible)
    st["acc"][:, :, :s] += p.sum((2, 3))
    return dict(out=_mix(p, st["v"][:, :, :s], q.dtype), lse=lse, acc=st["acc"])


def _plain_commit(st):
    parent, tokens, target = st["parent"].long(), st["tokens"], st["target"]
    n, t = parent.shape
    i = torch.arange(t, device=DEV)
    seen, present = _ancestors(st["parent"])
    up = parent.clamp(min=0)
    hit = present & (parent >= 0) & (tokens == target.gather(1, up))
    same = (parent[:, :, None] == parent[:, None, :]) & (tokens[:, :, None] == tokens[:, None, :]) & present[:, None, :]
    first = ~(same & (i[:, None] > i)).any(2)
    chosen = (hit & first) | ((i == 0) & present)
    taken = present & seen[:, :, 0] & ~(seen & ~chosen[:, None, :]).any(2)
    count = taken.sum(1)
    path = torch.where(taken, i, t).sort(1).values
    follow = target.gather(1, torch.where(path < t, path, -1).amax(1).clamp(min=0)[:, None])[:, 0]
    follow = torch.where(count > 0, follow, -1)
    path = torch.where(path < t, path, -1).to(torch.int32)
    base = (st["kv_len"].long() - t)[:, None]
    src = base + torch.where(path >= 0, path.long(), i)
    for c in (st["k"], st["v"]):
        where = [x.repeat(st["layers"], 1)[:, None, :, None].expand(-1, c.shape[1], -1, c.shape[3]) for x in (src, base + i)]
        c.scatter_(2, where[1], c.gather(2, where[0]))
    kv_len = (base[:, 0] + count).to(torch.int32)
    return dict(k=st["k"], v=st["v"], path=path, count=count.to(torch.int32), follow=follow, kv_len=kv_len)


def _plain_evict(st):
    acc, pos, L, m = st["acc"], st["pos"].long(), st["kv_len"].long()[:, None, None], st["budget"]
    n, hkv, cap = acc.shape
    j = torch.arange(cap, device=DEV)
    inside = j < L
    newest = torch.where(inside, pos, -(1 << 40)).amax(2, keepdim=True)
    key = torch.where(pos > newest - st["recent"], math.inf, acc)
    key = torch.where(inside, key, -math.inf)
    rank = torch.empty_like(pos).scatter_(2, key.sort(dim=2, descending=True, stable=True).indices, j.expand_as(pos))
    kept = inside & (rank < m)
    # the slot whose row each slot ends with: itself, or for the freed ones below the budget the next kept one behind it
    hole, far = ~kept & (j < m) & (L > m), kept & (j >= m)
    source = far.to(torch.int8).sort(dim=2, descending=True, stable=True).indices
    take = torch.where(hole, source.gather(2, (hole.cumsum(2) - 1).clamp(min=0)), j)
    for c in (st["k"], st["v"]):
        h = min(m, cap)
        c[:, :, :h] = c.gather(2, take[:, :, :h, None].expand(-1, -1, -1, c.shape[3]))
    kv_len = torch.clamp(st["kv_len"], max=m)
    stays = j < kv_len[:, None, None]
    acc = torch.where(stays, acc.gather(2, take), 0.0)
    pos = torch.where(stays, pos.gather(2, take), -1).to(torch.int32)
    return dict(k=st["k"], v=st["v"], acc=acc, pos=pos, kv_len=kv_len)


_PLAIN = dict(tree=_plain_tree, commit=_plain_commit, accum=_plain_accum, evict=_plain_evict)


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["kind"]](state)


# ------------------------------------------------------ definitions, 64 bits

def _walk(parent):
    """Per node: the nodes that it sees (none if it is absent)."""
    sees = []
    for i, p in enumerate(parent):
        up = [] if p == -1 else sees[p] if 0 <= p < i else None
        sees.append(up + [i] if up is not None and (up or p == -1) else [])
    return sees


def _attend(q, k, v, visible):
    """One sequence: q [hq, l, e], k / v [hkv, L, e], visible [l, L] -> (out, lse, weights summed per KV head)."""
    hq, l, e = q.shape
    outs, lses, sums = [], [], []
    for g, (kg, vg) in enumerate(zip(k, v)):
        total = torch.zeros(k.shape[1], dtype=torch.float64, device=DEV)
        for h in range(g * (hq // len(k)), (g + 1) * (hq // len(k))):
            x = (q[h].double() @ kg.double().t()) / math.sqrt(e)
            x = torch.where(visible, x, -math.inf)
            lse = torch.logsumexp(x, 1)
            w = torch.where(visible, (x - torch.where(lse > -math.inf, lse, 0.0)[:, None]).exp(), 0.0)
            outs.append(w @ vg.double())
            lses.append(lse)
            total += w.sum(0)
        sums.append(total)
    return torch.stack(outs), torch.stack(lses), torch.stack(sums)


def exact(case, seed):
    st = prepare(case, seed)
    kind, n, lens = case["kind"], case["n"], _lens(case)
    if kind in ("tree", "accum"):
        q, k, v = st["q"], st["k"], st["v"]
        got = []
        for b, L in enumerate(lens):
            if kind == "tree":
                t = case["t"]
                visible = torch.zeros(t, L, dtype=torch.bool)
                for i, nodes in enumerate(_walk(st["parent"][b].tolist())):
                    if nodes:
                        visible[i, :L - t] = True
                        visible[i, [L - t + c for c in nodes]] = True
                visible = visible.to(DEV)
            else:
                l = case["l"]
                visible = torch.ones(l, L, dtype=torch.bool, device=DEV).tril(L - l)
            got.append(_attend(q[b], k[b, :, :L], v[b, :, :L], visible))
        res = dict(out=torch.stack([x[0] for x in got]), lse=torch.stack([x[1] for x in got]))
        if kind == "accum":
            res["acc"] = st["acc"].double()
            for b, L in enumerate(lens):
                res["acc"][b, :, :L] += got[b][2]
        return res
    k, v = st["k"].clone(), st["v"].clone()
    if kind == "commit":
        t, paths, counts, follows, ends = case["t"], [], [], [], []
        for b, L in enumerate(lens):
            parent, tokens, target = (st[x][b].tolist() for x in ("parent", "tokens", "target"))
            sees, path = _walk(parent), []
            at = 0 if sees[0] else None
            while at is not None:
                path.append(at)
                at = next((i for i in range(at + 1, t) if sees[i] and parent[i] == path[-1] and tokens[i] == target[path[-1]]), None)
            for c, old in ((k, st["k"]), (v, st["v"])):
                for z in range(case["layers"]):
                    for i, node in enumerate(path):
                        c[z * n + b, :, L - t + i] = old[z * n + b, :, L - t + node]
            paths.append(path + [-1] * (t - len(path)))
            counts.append(len(path))
            follows.append(target[path[-1]] if path else -1)
            ends.append(L - t + len(path))
        return dict(k=k, v=v, path=torch.tensor(paths, dtype=torch.int32), count=torch.tensor(counts, dtype=torch.int32),
                    follow=torch.tensor(follows), kv_len=torch.tensor(ends, dtype=torch.int32))
    acc, pos, m = st["acc"].cpu(), st["pos"].cpu(), case["budget"]
    acc_out, pos_out = torch.zeros_like(acc), torch.full_like(pos, -1)
    for b, L in enumerate(lens):
        for g in range(case["hkv"]):
            a, x = acc[b, g, :L].tolist(), pos[b, g, :L].tolist()
            new = max(x) - case["recent"]
            order = sorted(range(L), key=lambda i: (x[i] <= new, -a[i] if x[i] <= new else 0.0, i))
            kept = set(order[:m])
            slots = list(range(min(L, m)))
            far = iter([i for i in range(m, L) if i in kept])
            if L > m:
                slots = [i if i in kept else next(far) for i in slots]
            src = torch.tensor(slots, dtype=torch.long)
            acc_out[b, g, :len(slots)], pos_out[b, g, :len(slots)] = acc[b, g, src], pos[b, g, src]
            k[b, g, :len(slots)], v[b, g, :len(slots)] = st["k"][b, g, src.to(DEV)], st["v"][b, g, src.to(DEV)]
    return dict(k=k, v=v, acc=acc_out, pos=pos_out, kv_len=st["kv_len"].clamp(max=m))
