"""Forms of the cache operators that a call reaches by its sizes alone, against
the fp64 oracle; tolerances as tests/test_gpu_cache.py counts them."""
import math

import numpy as np
import pytest
import torch

from kuillm_amd import ops
from oracle import kuiops_oracle as O
from test_gpu_cache import (ACCUM, BF, HF, TREES, close_lse, close_out, gen, npy, padded, score_error, trees,
                            wide_capacity)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens", [(3100,) * 16, tuple(3100 - 64 * b for b in range(16))])
def test_sdpa_tree_last_block_of_the_second_key_group_past_the_cache(cuda, dtype, lens):
    # 128-row kernel, two splits of 1664 keys at most, two key groups with blocks of 64 keys in turn: the
    # last split has 1436 keys, 28 past a whole turn, so the second group's last block begins past the last
    # key; with full caches, past the end of the last sequence's memory too
    n, h, t, s, e = 16, 8, 20, 3100, 64
    q, k, v = gen((n, h, t, e), dtype, 1), gen((n, h, s, e), dtype, 2), gen((n, h, s, e), dtype, 3)
    parent = trees(n, t, 4)
    out, lse = ops.sdpa_tree(q.to(cuda), k.to(cuda), v.to(cuda), torch.from_numpy(parent).to(cuda),
                             torch.tensor(lens, dtype=torch.int32, device=cuda), return_lse=True)
    for b in (0, 1, 7, 15):
        ref, lref, size, terms = O.sdpa_tree(npy(q[b:b + 1]), npy(k[b:b + 1]), npy(v[b:b + 1]), parent[b:b + 1], lens[b:b + 1])
        close_out(out[b:b + 1], ref, size, terms, e, True)
        close_lse(lse[b:b + 1], lref, terms, e)


def bits_case(dtype, n, hq, hkv, t, e, L=24):
    """Rows whose weights have to keep fp32's bits: a key of weight about 1 with value 0, and two keys of about
    e^-1 each whose values are 1 and -1 and whose scores are 2^-13 apart, so what is left of their weights is
    about 2^-13 of them.  Scores are single exact products: row r's query is 1 + r / 128 in its first column."""
    rows = torch.arange(hq * t).view(1, hq, t).remainder(128) / 128 + 1
    q = torch.zeros(n, hq, t, e)
    q[..., 0] = rows
    k, v = torch.zeros(n, hkv, L, e), torch.zeros(n, hkv, L, e)
    k[..., 0] = -2048.0
    b = 1 + torch.randint(0, 120, (n, hkv), generator=torch.Generator().manual_seed(5)) / 128
    k[:, :, 0, 0], k[:, :, 3, 0], k[:, :, 9, 0] = 64.0, b, b + 1 / 128
    v[:, :, 3], v[:, :, 9] = 1.0, -1.0
    return q.to(dtype), k.to(dtype), v.to(dtype)


def close_bits(out, ref, size):
    """A weight's relative error: the exponent's rounding (below 8: 2^-22 ln 2), the scale's (2^-24 of a difference of
    at most 2) and the exponential's unit 2^-23, 2^-21.2 in all; six fp32 additions of 2^-24 each on half of the terms'
    sum, 2^-22.4.  Together below 2^-20 of the terms; the output's own rounding and f16's smallest step."""
    u = torch.finfo(out.dtype).eps / 2
    err = np.abs(npy(out) - ref) - (u * np.abs(ref) + 2.0 ** -20 * size + (2.0 ** -25 if out.dtype == HF else 0))
    assert err.max() <= 0, f"max excess {err.max():.3e}, {(err > 0).mean():.3f} of them"


BITS = [  # n, hq, hkv, t, e, kernel
    (4, 8, 2, 4, 64, "16 rows"), (2, 8, 2, 4, 128, "16 rows"), (2, 8, 2, 6, 256, "16 rows"),
    (4, 8, 2, 8, 64, "128 rows"), (2, 8, 2, 20, 128, "128 rows"),
    (4, 8, 2, 8, 64, "two key groups"), (2, 8, 2, 20, 128, "two key groups"),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,t,e,kernel", BITS)
def test_weights_keep_the_bits_of_fp32(cuda, n, hq, hkv, t, e, kernel, dtype):
    q, k, v = bits_case(dtype, n, hq, hkv, t, e)
    L, parent, scale = k.shape[2], np.repeat(np.arange(t, dtype=np.int32)[None] - 1, n, 0), 2.0 ** -6
    cap = L
    if kernel != "16 rows":
        cap = wide_capacity(n, hq, hkv, t, e, e)
    if kernel == "two key groups":
        cap = max(cap, 1536 * min(64, 256 // (n * hkv * -(-(hq // hkv * t) // 128))) + 31)
    q, k, v = q.to(cuda), padded(k, cap).to(cuda), padded(v, cap).to(cuda)
    lens, ends = (L,) * n, torch.full((n,), L, dtype=torch.int32, device=cuda)
    ref, _, size, _ = O.sdpa_tree(npy(q), npy(k[:, :, :L]), npy(v[:, :, :L]), parent, lens, scale)
    out, _ = ops.sdpa_tree(q, k, v, torch.from_numpy(parent).to(cuda), ends, scale=scale)
    close_bits(out, ref, size)
    # and as the rows of decode attention
    acc = torch.zeros(n, hkv, cap, device=cuda)
    ref, _, _, size, _ = O.sdpa_decode_accum(npy(q), npy(k[:, :, :L]), npy(v[:, :, :L]), np.zeros((n, hkv, L)), lens, scale)
    out, _ = ops.sdpa_decode_accum(q, k, v, acc, ends, scale=scale)
    close_bits(out, ref, size)
    if kernel == "16 rows" and e < 256:        # what sdpa_decode gives for the same rows
        same, _ = ops.sdpa_decode(q, k, v, scale=scale, kv_len=ends)
        close_bits(same, ref, size)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,l,e", [(8, 5, 64), (8, 9, 128), (8, 100, 64), (2, 300, 256)])
def test_sdpa_decode_accum_of_an_empty_cache(cuda, hq, l, e, dtype):
    # 20, 36, 400 and 300 rows a KV head that see no key
    q, k = gen((2, hq, l, e), dtype, 1).to(cuda), torch.zeros(2, 2, 0, e, dtype=dtype, device=cuda)
    out, lse = ops.sdpa_decode_accum(q, k, k.clone(), torch.zeros(2, 2, 0, device=cuda), causal=False, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,l,s,e,bad", [
    (1, 2, 2, 5, 90, 64, 1),          # one launch: a work-group has all rows and keys of its KV head
    (2, 4, 2, 8, 1500, 64, 3),        # kept scores, several splits
    (1, 4, 2, 12, 150, 128, 0),       # kept scores of two row groups
    (1, 8, 2, 50, 200, 64, 17),       # scores computed again
    (1, 4, 4, 300, 300, 64, 100),
    (1, 2, 1, 70, 130, 256, 69),
    (40, 8, 8, 40, 800, 64, 20),      # tiles of 64 keys
])
def test_sdpa_decode_accum_a_row_of_nan_reaches_the_keys_that_it_sees_alone(cuda, n, hq, hkv, l, s, e, bad, dtype):
    q, k, v = gen((n, hq, l, e), dtype, 1), gen((n, hkv, s, e), dtype, 2), gen((n, hkv, s, e), dtype, 3)
    head, L = hq - 1, s - 3                       # the last head's row at position `bad`, in sequence 0
    lens = torch.full((n,), L, dtype=torch.int32, device=cuda)
    acc = torch.rand(n, hkv, s, generator=torch.Generator().manual_seed(4)).to(cuda)
    args = k.to(cuda), v.to(cuda)
    clean, dirty = acc.clone(), acc.clone()
    ref, _ = ops.sdpa_decode_accum(q.to(cuda), *args, clean, lens)
    clean_q = q.clone()
    q[0, head, bad] = math.nan
    out, lse = ops.sdpa_decode_accum(q.to(cuda), *args, dirty, lens, return_lse=True)
    assert out[0, head, bad].isnan().all() and lse[0, head, bad].isnan()
    out[0, head, bad] = ref[0, head, bad]
    # (a wave with a row of NaN sums its rows again, value by value: other roundings of the same fp32 sums)
    want, _, _, size, terms = O.sdpa_decode_accum(npy(clean_q[:1]), npy(k[:1]), npy(v[:1]), np.zeros((1, hkv, s)), (L,))
    close_out(out[:1], want, size, terms, e, False)
    assert torch.equal(out[1:], ref[1:])
    sees = L - l + bad + 1
    assert dirty[0, -1, :sees].isnan().all()
    # the keys behind lose this row's weight, which is none, and nothing else
    assert torch.equal(dirty[0, -1, sees:], clean[0, -1, sees:])
    dirty[0, -1, :sees] = clean[0, -1, :sees]
    assert torch.equal(dirty, clean)


# The lists of test_gpu_cache.py on the 128-row kernel, at the tolerance of weights that keep fp32's bits.

def wide_cases(cases):
    return [c for c in cases if c[1] // c[2] * c[3] > 16 and max(c[5], c[6]) <= 128]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,t,s,e,ev,lens,absent,chain", wide_cases(TREES))
def test_sdpa_tree_128_rows(cuda, n, hq, hkv, t, s, e, ev, lens, absent, chain, dtype):
    q, k, v = gen((n, hq, t, e), dtype, 1), gen((n, hkv, s, e), dtype, 2), gen((n, hkv, s, ev), dtype, 3)
    parent, lens = trees(n, t, 4, absent), lens or (s,) * n
    ref, lref, size, terms = O.sdpa_tree(npy(q), npy(k), npy(v), parent, lens)
    cap = wide_capacity(n, hq, hkv, t, e, ev)
    out, lse = ops.sdpa_tree(q.to(cuda), padded(k, cap).to(cuda), padded(v, cap).to(cuda), torch.from_numpy(parent).to(cuda),
                             torch.tensor(lens, dtype=torch.int32, device=cuda), return_lse=True)
    close_out(out, ref, size, terms, e, False)
    close_lse(lse, lref, terms, e)


def close_sums(got, ref, start, rows, terms, e):
    grown = ref - start
    tol = grown * (4 * score_error(e, terms) + 2.0 ** -19 + rows * 2.0 ** -24) + 2.0 ** -23 * np.abs(ref)
    assert (np.abs(npy(got) - ref) <= tol).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,l,s,e,ev,lens,causal", wide_cases(ACCUM))
def test_sdpa_decode_accum_128_rows(cuda, n, hq, hkv, l, s, e, ev, lens, causal, dtype):
    q, k, v = gen((n, hq, l, e), dtype, 1), gen((n, hkv, s, e), dtype, 2), gen((n, hkv, s, ev), dtype, 3)
    lens, cap = lens or (s,) * n, max(s, wide_capacity(n, hq, hkv, l, e, ev))
    k, v = padded(k, cap), padded(v, cap)
    acc = torch.rand(n, hkv, cap, generator=torch.Generator().manual_seed(4))
    got = acc.to(cuda)
    out, lse = ops.sdpa_decode_accum(q.to(cuda), k.to(cuda), v.to(cuda), got, torch.tensor(lens, dtype=torch.int32, device=cuda),
                                     causal=causal, return_lse=True)
    ref, lref, aref, size, terms = O.sdpa_decode_accum(npy(q), npy(k), npy(v), npy(acc), lens, causal=causal)
    close_out(out, ref, size, terms, e, False)
    close_lse(lse, lref, terms, e)
    close_sums(got, aref, npy(acc), hq // hkv * l, terms, e)
    for b in range(n):
        assert torch.equal(got[b, :, lens[b]:].cpu(), acc[b, :, lens[b]:])


def head_on_device(q, k, v, causal):
    """One KV head in 64 bits on the device: q (G, l, e), k / v (L, e) -> out, lse, sums of the weights per key, sums
    of absolute output terms, the largest sum of absolute score terms."""
    G, l, e = q.shape
    rows, L = q.double().reshape(G * l, e), k.shape[0]
    x = rows @ k.double().t().contiguous() / math.sqrt(e)
    terms = float((rows.abs() @ k.double().abs().t().contiguous()).max()) / math.sqrt(e) if L else 0.0
    if causal:
        at = torch.arange(l, device=q.device).repeat(G)[:, None] + L - l
        x.masked_fill_(torch.arange(L, device=q.device)[None] > at, -math.inf)
    lse = torch.logsumexp(x, 1)
    w = (x - torch.where(lse > -math.inf, lse, 0.0)[:, None]).exp_()
    return ((w @ v.double()).view(G, l, -1), lse.view(G, l), w.sum(0), (w @ v.double().abs()).view(G, l, -1), terms)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,l,s,e,lens,causal", [
    # paired row groups, one group of waves: 3 groups (the middle one alone), and 4
    (8, 8, 8, 320, 450, 64, (450, 449, 320, 385, 1, 400, 333, 384), True),
    (8, 8, 8, 400, 460, 128, (460, 459, 400, 385, 384, 123, 0, 257), True),
    # the same at 1600 keys, with as many work-groups as keep one group of waves; two prompts, by heads
    (14, 8, 8, 513, 1600, 64, tuple(1600 - 91 * b for b in range(14)), True),
    (2, 32, 8, 1999, 2036, 64, (1999, 2001), True),
    # paired row groups, two groups of waves, and 64-key tiles whose rows two work-groups share
    (1, 32, 8, 1999, 2036, 128, (1999,), True),
    (1, 32, 1, 128, 16384, 128, (15001,), True),
    # 32-key tiles whose rows three work-groups share
    (1, 32, 8, 512, 550, 64, (540,), True),
    # 64-key tiles, both of a work-group's live: 5 and 3 tiles, the middle one alone
    (16, 8, 8, 40, 260, 64, (260, 257, 256, 193, 192, 129, 128, 65, 64, 40, 3, 0, 100, 200, 250, 259), True),
    (22, 8, 8, 33, 190, 128, tuple(190 - 8 * b for b in range(22)), False),
])
def test_sdpa_decode_accum_forms(cuda, n, hq, hkv, l, s, e, lens, causal, dtype):
    q, k, v = (gen(x, dtype, i).to(cuda) for i, x in enumerate(((n, hq, l, e), (n, hkv, s, e), (n, hkv, s, e))))
    acc = torch.rand(n, hkv, s, generator=torch.Generator().manual_seed(4)).to(cuda)
    got, G = acc.clone(), hq // hkv
    out, lse = ops.sdpa_decode_accum(q, k, v, got, torch.tensor(lens, dtype=torch.int32, device=cuda), causal=causal, return_lse=True)
    for b, L in enumerate(lens):
        for h in range(hkv):
            heads = slice(h * G, (h + 1) * G)
            ref, lref, sums, size, terms = head_on_device(q[b, heads], k[b, h, :L], v[b, h, :L], causal)
            close_out(out[b, heads], npy(ref), npy(size), terms, e, False)
            close_lse(lse[b, heads], npy(lref), terms, e)
            want = acc[b, h].double()
            want[:L] += sums
            close_sums(got[b, h], npy(want), npy(acc[b, h]), G * l, terms, e)
            assert torch.equal(got[b, h, L:], acc[b, h, L:])


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("kind", ["random", "ties"])
@pytest.mark.parametrize("cap,lens,budget,recent", [
    (8192, (8192, 5000), 2048, 64), (8193, (8193, 8192), 4000, 0), (12000, (11999, 9000), 1000, 1000),
    (16384, (16384, 16383), 8192, 128), (16384, (16384, 16384), 1, 0), (16385, (16385, 16000), 8192, 128), (20000, (20000, 600), 333, 7),
])
def test_kv_evict_of_long_caches(cuda, cap, lens, budget, recent, kind, inplace):
    # 8 and 16 slots a thread in registers, and slots read again in every pass
    n, hkv, g = 2, 2, np.random.default_rng(cap)
    acc = (g.random((n, hkv, cap)) ** 4 * 10).astype(np.float32)
    if kind == "ties":
        acc = np.floor(acc)
        acc[acc == 1] = -0.0
    pos = np.stack([[g.permutation(cap) for _ in range(hkv)] for _ in range(n)]).astype(np.int32)
    k, v = g.integers(0, 99, (n, hkv, cap, 8)).astype(np.float32), g.integers(0, 99, (n, hkv, cap, 16)).astype(np.float32)
    ref = O.kv_evict(k, v, acc, pos, lens, budget, recent)
    d = [torch.from_numpy(x).to(cuda) for x in (k, v, acc, pos, np.array(lens, np.int32))]
    outs = {} if inplace else dict(acc_out=torch.full_like(d[2], 7), pos_out=torch.full_like(d[3], 7), len_out=torch.full_like(d[4], 7))
    got = ops.kv_evict(*d, budget, recent, **outs)
    for a, r in zip((d[0], d[1], *got), ref):
        np.testing.assert_array_equal(a.cpu().numpy(), r)


def test_in_place_operators_through_a_compiled_function(cuda):
    # functionalised by the tracer: what the calls change has to come out as the direct calls leave it
    from kuillm_amd import library  # noqa: F401
    op = torch.ops.kuiops

    def serve(q, k, v, acc, pos, lens, path):
        ends = op.kv_tree_commit(k, v, path, lens, 5)
        out, lse = op.sdpa_decode_accum(q, k, v, acc, ends)
        op.kv_evict(k, v, acc, pos, ends, 20, 4)
        return out, lse, ends, acc * 2

    def state():
        q, k, v = (x.to(cuda) for x in (gen((2, 4, 1, 64), BF, 1), gen((2, 2, 60, 64), BF, 2), gen((2, 2, 60, 64), BF, 3)))
        acc = torch.rand(2, 2, 60, generator=torch.Generator().manual_seed(4)).to(cuda)
        pos = torch.arange(60, dtype=torch.int32, device=cuda).repeat(2, 2, 1)
        path = torch.tensor([[0, 2, 4, -1, -1], [0, 1, -1, -1, -1]], dtype=torch.int32, device=cuda)
        return q, k, v, acc, pos, torch.tensor([60, 33], dtype=torch.int32, device=cuda), path
    traced = torch.compile(serve, backend="aot_eager", fullgraph=True)
    for _ in range(2):
        mine, theirs = state(), state()
        for a, b in zip(serve(*mine), traced(*theirs)):
            assert torch.equal(a, b)
        for a, b in zip(mine, theirs):
            assert torch.equal(a, b)


def test_kv_tree_commit_of_a_path_without_entries(cuda):
    k = torch.randn(2, 2, 30, 64, device=cuda).to(BF)
    kd, vd = k.clone(), k.clone()
    lens = torch.tensor([20, 3], dtype=torch.int32, device=cuda)
    ends = ops.kv_tree_commit(kd, vd, torch.zeros(2, 0, dtype=torch.int32, device=cuda), lens, 7)
    assert ends.tolist() == [13, 3] and torch.equal(kd, k) and torch.equal(vd, k)
