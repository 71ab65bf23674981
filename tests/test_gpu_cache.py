"""Drafted trees and bounded caches on the GPU against the fp64 oracle.

Tolerances.  u = eps / 2 is half a step of the output type.  An output rounds
once: u |out|.  A probability that is multiplied as one 16-bit value rounds by
u, as the sum of two by 2^-16 (bf16: 8 + 8 bits; f16: 11 + 11): at most that
much of the sum A of the absolute terms p |v|.  Scores are fp32 sums of e exact
products, off by at most ds = e 2^-23 S, S the sum of their absolute terms, and
by three roundings of the score (scale, product, exponent: 2^-22 S); p and the
sums of p move by 2 ds + the fp32 exponential's 2^-22."""
import math

import numpy as np
import pytest
import torch

from kuillm_amd import ops
from oracle import kuiops_oracle as O

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def npy(t):
    return t.detach().double().cpu().numpy()


def gen(shape, dtype=BF, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def score_error(e, terms):
    return (e * 2.0 ** -23 + 2.0 ** -21) * terms


def close_out(out, ref, size, terms, e, one_part):
    u = torch.finfo(out.dtype).eps / 2
    ds = score_error(e, terms)
    p = (u if one_part else 2.0 ** -16) + 4 * ds + 2.0 ** -20
    # (values near 0 round to f16's smallest step)
    tol = u * np.abs(ref) + p * (1 + u) * size + (2.0 ** -25 if out.dtype == HF else 0)
    err = np.abs(npy(out) - ref) - tol
    assert np.isfinite(npy(out)).all() and err.max() <= 0, f"max excess {err.max():.3e}"


def close_lse(lse, ref, terms, e):
    ds = score_error(e, terms)
    got = npy(lse)
    assert (np.isneginf(got) == np.isneginf(ref)).all()
    f = np.isfinite(ref)
    assert (np.abs(got[f] - ref[f]) <= ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(ref[f])).all()


def trees(n, t, seed, absent=0):
    g = np.random.default_rng(seed)
    p = np.array([[-1] + [int(g.integers(-1 if i % 7 == 3 else 0, i)) for i in range(1, t)] for _ in range(n)], np.int32)
    for b in range(n):
        for i in range(absent):
            p[b, int(g.integers(0, t))] = (-2, t, -100)[i % 3]
    return p


def wide_capacity(n, hq, hkv, rows, e, ev):
    """A cache capacity with which a call of more than 16 rows runs on the
    128-row kernel (whose probabilities are single 16-bit values); the smaller
    ones of these tests run on the 16-row kernel."""
    groups = n * hkv * -(-(hq // hkv * rows) // 16)
    return 2 ** 25 // ((64 if max(e, ev) <= 64 else 128) * groups) + 64


def padded(x, cap):
    """x with its third axis padded to the capacity with NaN."""
    return torch.cat([x, torch.full((*x.shape[:2], cap - x.shape[2], x.shape[3]), math.nan, dtype=x.dtype)], 2)


TREES = [  # n, hq, hkv, t, s, e, ev, lens, absent, chain
    (1, 1, 1, 1, 1, 64, 64, None, 0, False),                    # one node, nothing before it
    (1, 4, 2, 5, 5, 128, 128, None, 0, False),                  # nothing before the tree
    (2, 4, 2, 7, 100, 64, 64, (100, 33), 2, False),             # shared heads, ragged, absent nodes
    (3, 8, 8, 3, 70, 128, 128, (3, 2, 0), 0, False),            # a tree alone, one cut off, an empty cache
    (2, 8, 2, 13, 400, 64, 64, (400, 129), 1, True),            # a chain (with a hole)
    (1, 14, 2, 9, 260, 64, 64, (257,), 0, False),               # 63 rows
    (1, 16, 2, 8, 260, 128, 128, (255,), 0, False),             # 64 rows
    (1, 16, 1, 5, 300, 128, 128, (300,), 3, False),             # 80 rows
    (2, 8, 2, 64, 500, 128, 128, (500, 64), 4, False),          # 256 rows, one tree from the start
    (1, 4, 4, 65, 200, 64, 64, (190,), 5, False),               # 65 nodes: a second word of bits
    (1, 2, 1, 256, 700, 128, 128, (700,), 9, False),            # the largest tree
    (1, 2, 1, 256, 300, 64, 64, (299,), 0, True),               # the deepest
    (2, 6, 2, 6, 150, 80, 96, (150, 90), 0, False),             # head dims of their own
    (1, 4, 2, 6, 150, 256, 256, (149,), 1, False),
    (1, 4, 4, 20, 150, 8, 200, (150,), 0, False),
    (2, 40, 2, 4, 330, 128, 128, (330, 301), 0, False),
]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,t,s,e,ev,lens,absent,chain", TREES)
def test_sdpa_tree(cuda, n, hq, hkv, t, s, e, ev, lens, absent, chain, dtype, wide):
    q, k, v = gen((n, hq, t, e), dtype, 1), gen((n, hkv, s, e), dtype, 2), gen((n, hkv, s, ev), dtype, 3)
    if wide:
        if hq // hkv * t <= 16 or max(e, ev) > 128:
            return      # these have the 16-row kernel alone
        lens = lens or (s,) * n
    parent = trees(n, t, 4, absent)
    if chain:
        parent = np.where(parent >= -1, np.arange(t) - 1, parent).astype(np.int32)
    ref, lref, size, terms = O.sdpa_tree(npy(q), npy(k), npy(v), parent, lens)
    kv_len = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=cuda)
    if wide:
        cap = wide_capacity(n, hq, hkv, t, e, ev)
        k, v = padded(k, cap), padded(v, cap)
    out, lse = ops.sdpa_tree(q.to(cuda), k.to(cuda), v.to(cuda), torch.from_numpy(parent).to(cuda), kv_len, return_lse=True)
    assert out.dtype == dtype and lse.dtype == torch.float32
    close_out(out, ref, size, terms, e, wide)
    close_lse(lse, lref, terms, e)


def test_sdpa_tree_long_cache_splits(cuda):
    # one sequence, few heads: the keys are split over work-groups; the tree's keys end inside a tile
    q, k, v = gen((1, 2, 6, 64), BF, 1), gen((1, 1, 9001, 64), BF, 2), gen((1, 1, 9001, 64), BF, 3)
    parent = trees(1, 6, 4)
    for L in (9001, 8999, 4100, 129, 6):
        ref, lref, size, terms = O.sdpa_tree(npy(q), npy(k), npy(v), parent, (L,))
        out, lse = ops.sdpa_tree(q.to(cuda), k.to(cuda), v.to(cuda), torch.from_numpy(parent).to(cuda),
                                 torch.tensor([L], dtype=torch.int32, device=cuda), return_lse=True)
        close_out(out, ref, size, terms, 64, False)
        close_lse(lse, lref, terms, 64)


@pytest.mark.parametrize("n,hq,hkv,t,s,e,ev,lens,absent,chain", [x for x in TREES if x[1] // x[2] * x[3] > 16 and max(x[5], x[6]) <= 128])
def test_sdpa_tree_key_groups(cuda, n, hq, hkv, t, s, e, ev, lens, absent, chain):
    # 128-row kernel with at least 1536 keys a work-group: two groups of waves share them
    q, k, v = gen((n, hq, t, e), BF, 1), gen((n, hkv, s, e), BF, 2), gen((n, hkv, s, ev), BF, 3)
    parent = trees(n, t, 4, absent)
    if chain:           # an infinite value that only the last node sees
        parent = np.where(parent >= -1, np.arange(t) - 1, parent).astype(np.int32)
        v[0, 0, (lens or (s,))[0] - 1] = math.inf
    lens = lens or (s,) * n
    ref, lref, size, terms = O.sdpa_tree(npy(q), npy(k), npy(v), parent, lens)
    cap = max(wide_capacity(n, hq, hkv, t, e, ev), 1536 * min(64, 256 // (n * hkv * -(-(hq // hkv * t) // 128))) + 31)
    out, lse = ops.sdpa_tree(q.to(cuda), padded(k, cap).to(cuda), padded(v, cap).to(cuda), torch.from_numpy(parent).to(cuda),
                             torch.tensor(lens, dtype=torch.int32, device=cuda), return_lse=True)
    ok = np.isfinite(ref)
    assert chain or ok.all()
    assert (npy(out)[~ok] == math.inf).all()
    out = torch.where(torch.from_numpy(ok).to(cuda), out, torch.zeros_like(out))
    close_out(out, np.where(ok, ref, 0), np.where(ok, size, 0), terms, e, True)
    close_lse(lse, lref, terms, e)


@pytest.mark.parametrize("L", [7, 63, 64, 65, 200, 1000, 4097])
def test_sdpa_tree_splits_of_the_wide_kernel(cuda, L):
    # 128-row kernel, the keys over several work-groups, the tree across block ends
    n, hq, hkv, t, e = 1, 16, 2, 7, 64
    q, k, v = gen((n, hq, t, e), BF, 1), gen((n, hkv, L, e), BF, 2), gen((n, hkv, L, e), BF, 3)
    parent = trees(n, t, 4)
    ref, lref, size, terms = O.sdpa_tree(npy(q), npy(k), npy(v), parent, (L,))
    cap = wide_capacity(n, hq, hkv, t, e, e)
    out, lse = ops.sdpa_tree(q.to(cuda), padded(k, cap).to(cuda), padded(v, cap).to(cuda), torch.from_numpy(parent).to(cuda),
                             torch.tensor([L], dtype=torch.int32, device=cuda), return_lse=True)
    close_out(out, ref, size, terms, e, True)
    close_lse(lse, lref, terms, e)


def test_sdpa_tree_layouts(cuda):
    # queries as the projection leaves them, caches as (n, s, h, e), one parent list for all, output in place
    n, hq, hkv, t, s, e = 2, 8, 2, 6, 90, 64
    q, k, v = gen((n, t, hq, e), BF, 1), gen((n, s, hkv, e), BF, 2), gen((n, s, hkv, e), BF, 3)
    parent = trees(1, t, 4)
    ref, _, size, terms = O.sdpa_tree(npy(q).transpose(0, 2, 1, 3), npy(k).transpose(0, 2, 1, 3), npy(v).transpose(0, 2, 1, 3),
                                      np.repeat(parent, n, 0))
    buf = torch.full((n, t, hq, e), 7.0, dtype=BF, device=cuda)
    got, lse = ops.sdpa_tree(q.to(cuda).transpose(1, 2), k.to(cuda).transpose(1, 2), v.to(cuda).transpose(1, 2),
                             torch.from_numpy(parent[0]).to(cuda), out=buf.transpose(1, 2))
    assert lse is None and got.data_ptr() == buf.data_ptr()
    close_out(got, ref, size, terms, e, False)
    # queries in rows that cannot be read in place
    odd = torch.zeros(n, t, hq, e + 1, dtype=BF, device=cuda)[..., 1:]
    odd.copy_(q)
    got, _ = ops.sdpa_tree(odd.transpose(1, 2), k.to(cuda).transpose(1, 2), v.to(cuda).transpose(1, 2), torch.from_numpy(parent[0]).to(cuda))
    close_out(got, ref, size, terms, e, False)


@pytest.mark.parametrize("e", [64, 128])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_sdpa_tree_values_that_are_not_finite_where_no_query_looks(cuda, dtype, wide, e):
    n, hq, hkv, t, s, L = 1, 24, 2, 6, 120, 100
    q, k, v = gen((n, hq, t, e), dtype, 1), gen((n, hkv, s, e), dtype, 2), gen((n, hkv, s, e), dtype, 3)
    parent = np.array([[-1, 0, 0, 1, -2, 4]], np.int32)
    ref, lref, size, terms = O.sdpa_tree(npy(q), npy(k), npy(v), parent, (L,))
    # behind the length, at absent nodes, and in an absent node's query
    for j in list(range(L, s)) + [L - 2, L - 1]:
        k[:, :, j], v[:, :, j] = (math.nan, math.inf) if j % 2 else (-math.inf, math.nan)
    q[:, :, 4:] = math.nan
    if wide:
        cap = wide_capacity(n, hq, hkv, t, e, e)
        k, v = padded(k, cap), padded(v, cap)
    args = k.to(cuda), v.to(cuda), torch.from_numpy(parent).to(cuda), torch.tensor([L], dtype=torch.int32, device=cuda)
    out, lse = ops.sdpa_tree(q.to(cuda), *args, return_lse=True)
    close_out(out, ref, size, terms, e, wide)
    close_lse(lse, lref, terms, e)
    # node 2's value: seen by node 2 alone
    v[:, :, L - t + 2, 5], v[:, :, L - t + 2, 6], v[:, :, L - t + 2, 7] = math.inf, -math.inf, math.nan
    out, _ = ops.sdpa_tree(q.to(cuda), k.to(cuda), v.to(cuda), *args[2:], return_lse=True)
    got = npy(out)
    assert (got[:, :, 2, 5] == math.inf).all() and (got[:, :, 2, 6] == -math.inf).all() and np.isnan(got[:, :, 2, 7]).all()
    got[:, :, 2, 5:8] = ref[:, :, 2, 5:8]
    close_out(torch.from_numpy(got).to(dtype), ref, size, terms, e, wide)


def test_sdpa_tree_an_infinite_value_of_the_context_reaches_every_row(cuda):
    q, k, v = gen((1, 4, 5, 128), BF, 1), gen((1, 2, 300, 128), BF, 2), gen((1, 2, 300, 128), BF, 3)
    v[:, :, 17, 3] = math.inf
    out, _ = ops.sdpa_tree(q.to(cuda), k.to(cuda), v.to(cuda), torch.from_numpy(trees(1, 5, 4)).to(cuda))
    got = npy(out)
    assert (got[..., 3] == math.inf).all()
    assert np.isfinite(np.delete(got, 3, -1)).all()


def test_sdpa_tree_equals_itself(cuda):
    # no order of work-groups shows in the result
    q, k, v = gen((1, 8, 7, 128), BF, 1).to(cuda), gen((1, 2, 6000, 128), BF, 2).to(cuda), gen((1, 2, 6000, 128), BF, 3).to(cuda)
    parent = torch.from_numpy(trees(1, 7, 4)).to(cuda)
    first, lse = ops.sdpa_tree(q, k, v, parent, return_lse=True)
    for _ in range(5):
        out, l2 = ops.sdpa_tree(q, k, v, parent, return_lse=True)
        assert torch.equal(out, first) and torch.equal(lse, l2)


def test_sdpa_tree_cache_past_32_bit_offsets(cuda):
    # 2.2e9 elements of K and of V between the first and the last key; written where they are read
    s, stride = 33000, 1 << 16
    k = torch.zeros(s * stride, dtype=BF, device=cuda).as_strided((1, 1, s, 64), (0, 0, stride, 1))
    data = gen((1, 1, s, 64), BF, 2)
    k.copy_(data.to(cuda))
    q, v = gen((1, 2, 3, 64), BF, 1), gen((1, 1, s, 64), BF, 3)
    parent = np.array([[-1, 0, 0]], np.int32)
    ref, lref, size, terms = O.sdpa_tree(npy(q), npy(data), npy(v), parent)
    out, lse = ops.sdpa_tree(q.to(cuda), k, v.to(cuda), torch.from_numpy(parent).to(cuda), return_lse=True)
    close_out(out, ref, size, terms, 64, False)
    close_lse(lse, lref, terms, 64)


# ------------------------------------------------------------------- accum

ACCUM = [  # n, hq, hkv, l, s, e, ev, lens, causal
    (1, 1, 1, 1, 1, 64, 64, None, True),
    (2, 8, 2, 1, 130, 64, 64, (130, 37), True),
    (3, 4, 4, 1, 90, 128, 128, (90, 1, 0), True),
    (1, 40, 2, 1, 600, 128, 128, (555,), True),
    (2, 4, 2, 7, 60, 64, 64, (60, 9), True),
    (2, 4, 2, 7, 60, 64, 64, (60, 9), False),
    (1, 4, 2, 7, 60, 64, 64, (4,), True),                 # queries before the first key see nothing
    (1, 8, 2, 150, 150, 64, 64, None, True),              # a prompt
    (2, 4, 1, 70, 333, 128, 128, (333, 70), True),        # a piece of one
    (1, 4, 2, 33, 90, 80, 40, (90,), True),
    (1, 2, 2, 3, 90, 256, 256, (90,), True),
    (1, 2, 1, 60, 130, 256, 192, (130,), True),
    (1, 8, 4, 1000, 1000, 64, 64, None, True),            # row groups that end with a head
    (1, 4, 1, 897, 1500, 128, 128, (1400,), True),
    (2, 8, 4, 20, 70, 64, 64, (70, 25), True),
    (3, 4, 2, 1540, 1600, 64, 64, (1600, 1541, 700), True),     # paired row groups with two key groups
    (1, 2, 1, 700, 700, 256, 256, None, True),            # a tile's rows over two work-groups
]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,l,s,e,ev,lens,causal", ACCUM)
def test_sdpa_decode_accum(cuda, n, hq, hkv, l, s, e, ev, lens, causal, dtype, wide):
    q, k, v = gen((n, hq, l, e), dtype, 1), gen((n, hkv, s, e), dtype, 2), gen((n, hkv, s, ev), dtype, 3)
    if wide:
        if hq // hkv * l <= 16 or max(e, ev) > 128:
            return      # these have the 16-row kernel alone
        lens = lens or (s,) * n
        cap = max(s, wide_capacity(n, hq, hkv, l, e, ev))
        k, v = padded(k, cap), padded(v, cap)
    acc = torch.rand(n, hkv, k.shape[2], generator=torch.Generator().manual_seed(4))
    ref, lref, aref, size, terms = O.sdpa_decode_accum(npy(q), npy(k), npy(v), npy(acc), lens, causal=causal)
    kv_len = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=cuda)
    got = acc.to(cuda)
    out, lse = ops.sdpa_decode_accum(q.to(cuda), k.to(cuda), v.to(cuda), got, kv_len, causal=causal, return_lse=True)
    close_out(out, ref, size, terms, e, wide or 2 ** 25 // 128 < n * hkv * -(-(hq // hkv * l) // 16) * s)
    close_lse(lse, lref, terms, e)
    rows = hq // hkv * l
    grown = aref - npy(acc)
    tol = grown * (4 * score_error(e, terms) + 2.0 ** -19 + rows * 2.0 ** -24) + 2.0 ** -23 * aref
    assert (np.abs(npy(got) - aref) <= tol).all()
    # keys behind the length keep their sums, to the bit
    for b in range(n):
        L = k.shape[2] if lens is None else lens[b]
        assert torch.equal(got[b, :, L:].cpu(), acc[b, :, L:])


def test_sdpa_decode_accum_ignores_what_lies_behind(cuda):
    q, k, v = gen((2, 4, 1, 64), BF, 1), gen((2, 2, 80, 64), BF, 2), gen((2, 2, 80, 64), BF, 3)
    lens = (50, 33)
    ref, lref, aref, size, terms = O.sdpa_decode_accum(npy(q), npy(k), npy(v), np.zeros((2, 2, 80)), lens)
    for b, L in enumerate(lens):
        k[b, :, L:], v[b, :, L:] = math.nan, math.inf
    big = torch.zeros(2, 3, 100, device=cuda)
    out, lse = ops.sdpa_decode_accum(q.to(cuda), k.to(cuda), v.to(cuda), big[:, 1:, 7:87], torch.tensor(lens, dtype=torch.int32, device=cuda),
                                     return_lse=True)
    close_out(out, ref, size, terms, 64, False)
    close_lse(lse, lref, terms, 64)
    assert (big[:, 0] == 0).all() and (big[..., :7] == 0).all() and (big[..., 87:] == 0).all()
    assert (np.abs(npy(big[:, 1:, 7:87]) - aref) <= aref * (4 * score_error(64, terms) + 2.0 ** -18)).all()


# ----------------------------------------------------------- exact operators

@pytest.mark.parametrize("t", [1, 2, 9, 64, 65, 256])
def test_tree_accept(cuda, t):
    n = 40
    g = np.random.default_rng(t)
    parent = trees(n, t, t, absent=1 if t > 1 else 0)
    parent[: n // 2, 0] = -1
    tokens, target = g.integers(0, 3, (n, t)), g.integers(0, 3, (n, t))
    if t > 1:
        parent[0], tokens[0], target[0] = np.arange(t) - 1, 1, 1            # a chain, accepted whole
    ref = O.tree_accept(tokens, parent, target)
    got = ops.tree_accept(torch.from_numpy(tokens).to(cuda), torch.from_numpy(parent).to(cuda), torch.from_numpy(target).to(cuda))
    for a, r in zip(got, ref):
        np.testing.assert_array_equal(a.cpu().numpy(), r)


@pytest.mark.parametrize("n,layers,hkv,cap,e,ev,t,dtype", [
    (1, 1, 1, 9, 64, 64, 1, BF), (3, 2, 2, 40, 64, 128, 9, BF), (2, 1, 3, 300, 128, 128, 256, HF),
    (2, 3, 1, 50, 8, 24, 7, torch.float32), (1, 1, 2, 64, 512, 1024, 40, BF), (1, 2, 1, 33, 16, 16, 5, torch.uint8),
])
def test_kv_tree_commit(cuda, n, layers, hkv, cap, e, ev, t, dtype):
    g = np.random.default_rng(t)
    k = torch.randint(0, 100, (layers * n, hkv, cap, e), generator=torch.Generator().manual_seed(1)).to(dtype)
    v = torch.randint(0, 100, (layers * n, hkv, cap, ev), generator=torch.Generator().manual_seed(2)).to(dtype)
    for path in (np.sort(np.stack([g.permutation(t) for _ in range(n)])[:, : (t + 1) // 2], 1), np.stack([g.permutation(t) for _ in range(n)])):
        path = path.astype(np.int32)
        for b in range(n):
            path[b, int(g.integers(0, path.shape[1] + 1)):] = -1 if b % 2 else t
        lens = np.array([cap if b == 0 else t + b for b in range(n)], np.int32)
        ref = O.kv_tree_commit(npy(k), npy(v), path, lens, t)
        kd, vd = k.to(cuda), v.to(cuda)
        ends = ops.kv_tree_commit(kd, vd, torch.from_numpy(path).to(cuda), torch.from_numpy(lens).to(cuda), t)
        for a, r in zip((kd, vd, ends), ref):
            np.testing.assert_array_equal(npy(a), r)


def test_kv_tree_commit_short_caches_and_views(cuda):
    # fewer keys than nodes: nothing moves; keys past the capacity: the path ends there; a view of a larger buffer
    base = torch.randn(4, 20, 3, 64).to(BF)
    path = torch.tensor([[1, 2, -1], [0, 2, 2], [2, 0, 1], [-1, 0, 0]], dtype=torch.int32)
    lens = torch.tensor([2, 21, 12, 9], dtype=torch.int32)
    view = base.transpose(1, 2)[:, 1:]
    ref = O.kv_tree_commit(npy(view), npy(view), path.numpy(), lens.numpy(), 3)
    kd, vd = base.to(cuda), base.to(cuda)
    ends = ops.kv_tree_commit(kd.transpose(1, 2)[:, 1:], vd.transpose(1, 2)[:, 1:], path.to(cuda), lens.to(cuda), 3)
    np.testing.assert_array_equal(npy(kd.transpose(1, 2)[:, 1:]), ref[0])
    np.testing.assert_array_equal(npy(vd.transpose(1, 2)[:, 1:]), ref[1])
    assert torch.equal(kd[:, :, 0].cpu(), base[:, :, 0]) and ends.tolist() == ref[2].tolist() == [2, 19, 12, 6]


EVICT = [  # n, hkv, cap, lens, budget, recent, kind of weights
    (1, 1, 1, (1,), 1, 0, "random"), (2, 2, 70, (70, 33), 20, 5, "random"), (3, 1, 50, (0, 20, 21), 20, 20, "random"),
    (1, 2, 3000, (2900,), 1024, 64, "random"), (1, 1, 5000, (5000,), 1, 1, "random"), (1, 1, 2048, (2048,), 2047, 0, "ties"),
    (2, 2, 1500, (1500, 1025), 700, 0, "ties"), (1, 2, 1200, (1100,), 300, 10, "odd"), (1, 1, 64, (64,), 100, 50, "random"),
    (1, 1, 90, (90,), 30, 30, "same positions"), (2, 8, 40000, (40000, 12345), 9000, 1000, "random"),
]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("n,hkv,cap,lens,budget,recent,kind", EVICT)
def test_kv_evict(cuda, n, hkv, cap, lens, budget, recent, kind, inplace):
    g = np.random.default_rng(cap)
    acc = (g.random((n, hkv, cap)) ** 4 * 10).astype(np.float32)
    pos = np.stack([[g.permutation(cap) for _ in range(hkv)] for _ in range(n)]).astype(np.int32)
    if kind == "ties":
        acc = np.floor(acc)
        acc[acc == 1] = -0.0
    if kind == "odd":
        acc[..., ::7], acc[..., 1::9], acc[..., 2::11], acc[..., 3::13] = np.nan, np.inf, -np.inf, -1.5
    if kind == "same positions":
        pos[:] = 5
    if cap > 10000:
        pos = np.sort(pos, -1)
    k, v = g.integers(0, 99, (n, hkv, cap, 8)).astype(np.float32), g.integers(0, 99, (n, hkv, cap, 16)).astype(np.float32)
    ref = O.kv_evict(k, v, acc, pos, lens, budget, recent)
    d = [torch.from_numpy(x).to(cuda) for x in (k, v, acc, pos, np.array(lens, np.int32))]
    outs = {} if inplace else dict(acc_out=torch.full_like(d[2], 7), pos_out=torch.full_like(d[3], 7), len_out=torch.full_like(d[4], 7))
    got = ops.kv_evict(*d, budget, recent, **outs)
    if inplace:
        assert all(a is b for a, b in zip(got, d[2:]))
    else:
        np.testing.assert_array_equal(d[2].cpu().numpy(), acc)
        np.testing.assert_array_equal(d[3].cpu().numpy(), pos)
        assert d[4].tolist() == list(lens)
    for a, r in zip((d[0], d[1], *got), ref):
        np.testing.assert_array_equal(a.cpu().numpy(), r)


def test_kv_evict_lengths_past_the_capacity_and_below_zero(cuda):
    k = torch.randn(2, 1, 12, 64, device=cuda).to(BF)
    acc, pos = torch.rand(2, 1, 12, device=cuda), torch.arange(12, dtype=torch.int32, device=cuda).repeat(2, 1, 1).contiguous()
    ref = O.kv_evict(npy(k), npy(k), acc.cpu().numpy(), pos.cpu().numpy(), (40, -3), 5, 2)
    kd, vd = k.clone(), k.clone()
    got = ops.kv_evict(kd, vd, acc, pos, torch.tensor([40, -3], dtype=torch.int32, device=cuda), 5, 2)
    for a, r in zip((kd, vd, *got), ref):
        np.testing.assert_array_equal(npy(a), r)


# --------------------------------------------------------- a run of them all

def rounds(cuda, steps, seed=0):
    """State of a serving loop: two sequences, one layer, a budget of 48 keys."""
    n, hq, hkv, e, cap, t = 2, 4, 2, 64, 96, 7
    d = dict(k=torch.zeros(n, hkv, cap, e, dtype=BF), v=torch.zeros(n, hkv, cap, e, dtype=BF), acc=torch.zeros(n, hkv, cap),
             pos=torch.full((n, hkv, cap), -1, dtype=torch.int32), kv_len=torch.tensor([40, 33], dtype=torch.int32),
             seen=torch.tensor([40, 33], dtype=torch.int32))
    for b, L in enumerate((40, 33)):
        d["k"][b, :, :L], d["v"][b, :, :L] = gen((hkv, L, e), BF, seed + b), gen((hkv, L, e), BF, seed + b + 9)
        d["pos"][b, :, :L] = torch.arange(L, dtype=torch.int32)
        d["acc"][b, :, :L] = torch.rand(hkv, L, generator=torch.Generator().manual_seed(seed))
    feed = []
    for i in range(steps):
        r = np.random.default_rng(seed + i)
        feed.append(dict(q=gen((n, hq, t, e), BF, seed + 100 + i), nk=gen((n, hkv, t, e), BF, seed + 200 + i),
                         nv=gen((n, hkv, t, e), BF, seed + 300 + i), parent=torch.from_numpy(trees(n, t, seed + i)),
                         tokens=torch.from_numpy(r.integers(0, 2, (n, t))), target=torch.from_numpy(r.integers(0, 2, (n, t))),
                         q1=gen((n, hq, 1, e), BF, seed + 400 + i)))
    return {x: y.to(cuda) for x, y in d.items()}, [{x: y.to(cuda) for x, y in f.items()} for f in feed], t


def one_round(d, f, t):
    """Drafted keys into the cache, tree attention, acceptance, commit, a token with summed weights, eviction: no host sync."""
    cap = d["k"].shape[2]
    slot = torch.arange(cap, device=d["k"].device)
    first = d["kv_len"][:, None]
    mine = (slot >= first) & (slot < first + t)
    node = (slot - first).clamp(0, t - 1).long()
    for c, new in (("k", "nk"), ("v", "nv")):
        rows = f[new].gather(2, node[:, None, :, None].expand(-1, d[c].shape[1], -1, d[c].shape[3]))
        d[c].copy_(torch.where(mine[:, None, :, None], rows, d[c]))
    drafted = d["kv_len"] + t
    out, _ = ops.sdpa_tree(f["q"], d["k"], d["v"], f["parent"], drafted)
    path, count, follow = ops.tree_accept(f["tokens"], f["parent"], f["target"])
    ends = ops.kv_tree_commit(d["k"], d["v"], path, drafted, t)
    fresh = (slot >= first) & (slot < ends[:, None])
    d["pos"].copy_(torch.where(fresh[:, None], (d["seen"][:, None] + slot - first)[:, None].int(), d["pos"]))
    d["seen"] += count
    d["kv_len"].copy_(ends)
    one, _ = ops.sdpa_decode_accum(f["q1"], d["k"], d["v"], d["acc"], d["kv_len"])
    ops.kv_evict(d["k"], d["v"], d["acc"], d["pos"], d["kv_len"], 48, 8)
    return out, one, path, count, follow


def test_serving_rounds_against_the_oracle(cuda):
    d, feed, t = rounds(cuda, 4)
    for f in feed:
        before = {x: y.clone() for x, y in d.items()}
        out, one, path, count, follow = one_round(d, f, t)
        k, v, lens = npy(before["k"]), npy(before["v"]), before["kv_len"].tolist()
        for b, L in enumerate(lens):
            k[b, :, L:L + t], v[b, :, L:L + t] = npy(f["nk"])[b], npy(f["nv"])[b]
        drafted = [L + t for L in lens]
        parent = f["parent"].cpu().numpy()
        ref, _, size, terms = O.sdpa_tree(npy(f["q"]), k, v, parent, drafted)
        close_out(out, ref, size, terms, 64, False)
        rp, rc, rf = O.tree_accept(f["tokens"].cpu().numpy(), parent, f["target"].cpu().numpy())
        for a, r in zip((path, count, follow), (rp, rc, rf)):
            np.testing.assert_array_equal(a.cpu().numpy(), r)
        k, v, ends = O.kv_tree_commit(k, v, rp, drafted, t)
        ref, _, acc, size, terms = O.sdpa_decode_accum(npy(f["q1"]), k, v, npy(before["acc"]), ends)
        close_out(one, ref, size, terms, 64, False)
        pos = before["pos"].cpu().numpy()
        for b, L in enumerate(lens):
            pos[b, :, L:ends[b]] = int(before["seen"][b]) + np.arange(ends[b] - L)
        ref = O.kv_evict(k, v, acc, pos, ends, 48, 8)
        # (random weights 2^-10 apart at least where the budget cuts: checked, else the choice could differ)
        for b in range(2):
            for g in range(2):
                w = np.sort(acc[b, g, :ends[b]])
                assert np.diff(w).min() > 1e-6
        np.testing.assert_array_equal(npy(d["k"]), ref[0])
        np.testing.assert_array_equal(npy(d["v"]), ref[1])
        np.testing.assert_allclose(npy(d["acc"]), ref[2], rtol=1e-4, atol=1e-6)
        np.testing.assert_array_equal(d["pos"].cpu().numpy(), ref[3])
        assert d["kv_len"].tolist() == ref[4].tolist()


def test_serving_rounds_in_graphs(cuda):
    # two graphs of the same calls, captured with no eager call before, replayed in turn with eager work between
    sides = []
    for seed in (0, 50):
        d, feed, t = rounds(cuda, 1, seed)
        start = {x: y.clone() for x, y in d.items()}
        eager = {x: y.clone() for x, y in d.items()}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = one_round(d, feed[0], t)
        sides.append((graph, d, feed[0], start, eager, outs, t))
    for d, start in ((s[1], s[3]) for s in sides):
        for x in d:
            d[x].copy_(start[x])
    for _ in range(4):
        for graph, *_ in sides:
            graph.replay()
        torch.cuda.synchronize()
        for _, d, f, _, eager, outs, t in sides:
            refs = one_round(eager, f, t)
            torch.cuda.synchronize()
            for a, r in zip(outs, refs):
                assert torch.equal(a, r)
            for x in d:
                assert torch.equal(d[x], eager[x]), x


def test_calls_on_two_streams_at_once(cuda):
    sides = []
    for seed in (1, 2):
        q, k, v = (x.to(cuda) for x in (gen((1, 8, 5, 128), BF, seed), gen((1, 2, 8000, 128), BF, seed + 10), gen((1, 2, 8000, 128), BF, seed + 20)))
        parent = torch.from_numpy(trees(1, 5, seed)).to(cuda)
        acc = torch.zeros(1, 2, 8000, device=cuda)
        alone = ops.sdpa_tree(q, k, v, parent)[0], ops.sdpa_decode_accum(q[:, :, :1], k, v, acc.clone())[0]
        sides.append((torch.cuda.Stream(), (q, k, v, parent, acc), alone))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, (st, (q, k, v, parent, acc), _) in enumerate(sides):
            with torch.cuda.stream(st):
                got[i].append((ops.sdpa_tree(q, k, v, parent)[0], ops.sdpa_decode_accum(q[:, :, :1], k, v, acc)[0]))
    torch.cuda.synchronize()
    for (_, _, alone), results in zip(sides, got):
        for r in results:
            assert torch.equal(r[0], alone[0]) and torch.equal(r[1], alone[1])


def test_empty_calls(cuda):
    z = dict(device=cuda, dtype=BF)
    out, lse = ops.sdpa_tree(torch.zeros(0, 4, 3, 64, **z), torch.zeros(0, 2, 9, 64, **z), torch.zeros(0, 2, 9, 64, **z),
                             torch.zeros(0, 3, dtype=torch.int32, device=cuda), return_lse=True)
    assert out.shape == (0, 4, 3, 64) and lse.shape == (0, 4, 3)
    out, _ = ops.sdpa_tree(torch.zeros(1, 4, 0, 64, **z), torch.zeros(1, 2, 9, 64, **z), torch.zeros(1, 2, 9, 64, **z),
                           torch.zeros(1, 0, dtype=torch.int32, device=cuda))
    assert out.shape == (1, 4, 0, 64)
    out, lse = ops.sdpa_decode_accum(torch.ones(1, 4, 2, 64, **z), torch.zeros(1, 2, 0, 64, **z), torch.zeros(1, 2, 0, 64, **z),
                                     torch.zeros(1, 2, 0, device=cuda), causal=False, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    k = torch.zeros(1, 2, 0, 64, **z)
    got = ops.kv_evict(k, k.clone(), torch.zeros(1, 2, 0, device=cuda), torch.zeros(1, 2, 0, dtype=torch.int32, device=cuda),
                       torch.zeros(1, dtype=torch.int32, device=cuda), 4)
    assert got[2].tolist() == [0]


def test_custom_ops_run_the_same_kernels(cuda):
    from kuillm_amd import library  # noqa: F401
    op = torch.ops.kuiops
    q, k, v = (x.to(cuda) for x in (gen((2, 4, 5, 64), BF, 1), gen((2, 2, 60, 64), BF, 2), gen((2, 2, 60, 64), BF, 3)))
    parent, lens = torch.from_numpy(trees(2, 5, 4)).to(cuda), torch.tensor([60, 33], dtype=torch.int32, device=cuda)
    for a, b in zip(op.sdpa_tree(q, k, v, parent, lens), ops.sdpa_tree(q, k, v, parent, lens, return_lse=True)):
        assert torch.equal(a, b)
    tok = torch.randint(0, 2, (2, 5), device=cuda)
    path, count, follow = op.tree_accept(tok, parent, tok.flip(0).contiguous())
    for a, b in zip((path, count, follow), ops.tree_accept(tok, parent, tok.flip(0))):
        assert torch.equal(a, b)
    sides = [[k.clone(), v.clone()] for _ in range(2)]
    assert torch.equal(op.kv_tree_commit(*sides[0], path, lens, 5), ops.kv_tree_commit(*sides[1], path, lens, 5))
    accs = [torch.zeros(2, 2, 60, device=cuda) for _ in range(2)]
    for a, b in zip(op.sdpa_decode_accum(q, k, v, accs[0], lens), ops.sdpa_decode_accum(q, k, v, accs[1], lens, return_lse=True)):
        assert torch.equal(a, b)
    pos = [torch.arange(60, dtype=torch.int32, device=cuda).repeat(2, 2, 1) for _ in range(2)]
    ends = [lens.clone(), lens.clone()]
    op.kv_evict(*sides[0], accs[0], pos[0], ends[0], 20, 4)
    ops.kv_evict(*sides[1], accs[1], pos[1], ends[1], 20, 4)
    for a, b in zip((*sides[0], accs[0], pos[0], ends[0]), (*sides[1], accs[1], pos[1], ends[1])):
        assert torch.equal(a, b)
    assert ends[0].tolist() == [20, 20]


def test_another_current_device_or_stream_is_not_used(cuda):
    # a side stream's call runs behind that stream's own work
    q, k, v = (x.to(cuda) for x in (gen((1, 4, 5, 64), BF, 1), gen((1, 2, 600, 64), BF, 2), gen((1, 2, 600, 64), BF, 3)))
    parent = torch.from_numpy(trees(1, 5, 4)).to(cuda)
    ref, _ = ops.sdpa_tree(q, k, v, parent)
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=cuda)
        for _ in range(10):
            big = big @ big * 1e-4
        late.copy_(q)
        got, _ = ops.sdpa_tree(late, k, v, parent)
    side.synchronize()
    assert torch.equal(got, ref)
