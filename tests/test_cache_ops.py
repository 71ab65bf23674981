"""Drafted trees and bounded caches without a GPU: the oracle against closed
forms, and what the entry points refuse before anything is enqueued."""
import ctypes

import numpy as np
import pytest
import torch

from kuillm_amd import _lib, compile as _compile, config as C, ops
from oracle import kuiops_oracle as O

BF = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not C.LIB_PATH.exists():
        _compile.build_library()
    return _lib.load()


# ------------------------------------------------------------------ oracle

def test_tree_sees():
    assert O.tree_sees([-1, 0, 0, 1, -1, 4]) == [[0], [0, 1], [0, 2], [0, 1, 3], [4], [4, 5]]
    # absent: below -1, not an earlier node, and what hangs on such a node
    assert O.tree_sees([-1, -2, 1, 3, 0, 9]) == [[0], [], [], [], [0, 4], []]


def test_a_chain_is_causal_decode_attention():
    r = np.random.default_rng(0)
    q, k, v = (r.standard_normal(s) for s in ((2, 4, 5, 8), (2, 2, 11, 8), (2, 2, 11, 8)))
    out, lse, _, _ = O.sdpa_tree(q, k, v, [np.arange(5) - 1] * 2)
    ref, lref, acc, _, _ = O.sdpa_decode_accum(q, k, v, np.zeros((2, 2, 11)))
    np.testing.assert_allclose(out, ref, rtol=1e-12)
    np.testing.assert_allclose(lse, lref, rtol=1e-12)
    np.testing.assert_allclose(acc.sum(), 2 * 4 * 5)           # every row's weights sum to 1
    # one query over one key: that key's value, all its weight
    out, lse, acc, _, _ = O.sdpa_decode_accum(q[:, :, :1], k[:, :, :1], v[:, :, :1], np.zeros((2, 2, 1)))
    np.testing.assert_allclose(out[:, :, 0], np.repeat(v[:, :, 0], 2, 1))
    np.testing.assert_allclose(acc, 2.0)


def test_the_attention_is_torchs():
    r = np.random.default_rng(1)
    q, k, v = (r.standard_normal(s) for s in ((2, 4, 9, 8), (2, 2, 9, 8), (2, 2, 9, 6)))
    wide = [torch.from_numpy(np.repeat(x, 2, 1)) for x in (k, v)]
    ref = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q), *wide, is_causal=True)
    np.testing.assert_allclose(O.sdpa_decode_accum(q, k, v, np.zeros((2, 2, 9)))[0], ref.numpy(), rtol=1e-10)
    # a tree's rows: its nodes' keys alone behind the context
    parent = [-1, 0, 0, 1, -1]
    mask = torch.zeros(5, 9, dtype=torch.bool)
    mask[:, :4] = True
    for i, seen in enumerate(O.tree_sees(parent)):
        mask[i, [4 + j for j in seen]] = True
    ref = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q[:, :, :5]), *wide, attn_mask=mask)
    np.testing.assert_allclose(O.sdpa_tree(q[:, :, :5], k, v, [parent] * 2)[0], ref.numpy(), rtol=1e-10)


def test_accept_and_commit_by_hand():
    #      0 -> 1, 2; 1 -> 3; 2 -> 4, 5
    parent, tokens, target = [-1, 0, 0, 1, 2, 2], [7, 8, 9, 5, 5, 6], [9, 1, 6, 1, 1, 3]
    path, count, follow = O.tree_accept([tokens], [parent], [target])
    assert path[0].tolist() == [0, 2, 5, -1, -1, -1] and count[0] == 3 and follow[0] == 3
    k = np.arange(9.0)[None, None, :, None] + np.zeros((1, 1, 9, 2))
    k2, v2, ends = O.kv_tree_commit(k, -k, path, [8], 6)
    assert k2[0, 0, :, 0].tolist() == [0, 1, 2, 4, 7, 5, 6, 7, 8] and ends.tolist() == [5]
    np.testing.assert_array_equal(v2, -k2)


def test_evict_by_hand():
    acc = np.array([[[5, 1, 9, 1, 7, 3, 99, 0]]], np.float32)
    pos = np.arange(8, dtype=np.int32)[None, None]
    k = np.arange(8.0)[None, None, :, None] + np.zeros((1, 1, 8, 2))
    k2, _, a2, p2, ends = O.kv_evict(k, k, acc, pos, [6], 4, 1)      # slot 6 lies behind the length
    # position 5 is the newest; then 9, 7 and 5: slots 0, 2, 4, 5; 4 and 5 move into 1 and 3
    assert p2[0, 0].tolist() == [0, 4, 2, 5, -1, -1, -1, -1] and ends.tolist() == [4]
    assert a2[0, 0].tolist() == [5, 7, 9, 3, 0, 0, 0, 0]
    assert k2[0, 0, :, 0].tolist() == [0, 4, 2, 5, 4, 5, 6, 7]


# ---------------------------------------------------------------- refusals

def attn(n=2, hq=4, hkv=2, l=3, s=10, e=64, ev=64, dtype=BF):
    return (torch.zeros(n, hq, l, e, dtype=dtype), torch.zeros(n, hkv, s, e, dtype=dtype),
            torch.zeros(n, hkv, s, ev, dtype=dtype))


def tree(n=2, t=3):
    return torch.arange(-1, t - 1, dtype=torch.int32).expand(n, t).contiguous()


INVALID, UNSUPPORTED = _lib.E_INVALID, _lib.E_UNSUPPORTED


def refuses(status, fn, *args, **kw):
    with pytest.raises(_lib.KuiopsError) as err:
        fn(*args, **kw)
    assert err.value.status == status


@pytest.mark.parametrize("change, status", [
    (lambda q, k, v, p, o: dict(q=q[0]), INVALID),                                   # rank
    (lambda q, k, v, p, o: dict(q=q.half()), INVALID),                               # mixed types
    (lambda q, k, v, p, o: dict(q=q.float(), k=k.float(), v=v.float()), UNSUPPORTED),
    (lambda q, k, v, p, o: dict(k=k[:1]), INVALID),                                  # batches differ
    (lambda q, k, v, p, o: dict(k=k[..., :32]), INVALID),                            # head dims differ
    (lambda q, k, v, p, o: dict(v=v[:, :, :9]), INVALID),                            # lengths differ
    (lambda q, k, v, p, o: dict(q=q[:, :3]), INVALID),                               # 3 heads over 2
    (lambda q, k, v, p, o: dict(k=k.transpose(2, 3).contiguous().transpose(2, 3)), UNSUPPORTED),
    (lambda q, k, v, p, o: dict(parent=p.long()), INVALID),
    (lambda q, k, v, p, o: dict(parent=p[:, :2]), INVALID),
    (lambda q, k, v, p, o: dict(k=k[:, :, :2], v=v[:, :, :2]), INVALID),             # more nodes than keys
    (lambda q, k, v, p, o: dict(kv_len=torch.zeros(2, dtype=torch.int64)), INVALID),
    (lambda q, k, v, p, o: dict(kv_len=torch.zeros(3, dtype=torch.int32)), INVALID),
    (lambda q, k, v, p, o: dict(kv_len=torch.zeros(4, dtype=torch.int32)[::2]), INVALID),
    (lambda q, k, v, p, o: dict(out=o.float()), INVALID),
    (lambda q, k, v, p, o: dict(out=o[:, :, :2]), INVALID),
    (lambda q, k, v, p, o: dict(out=o[:, :, :1].expand(-1, -1, 3, -1)), INVALID),    # rows on one another
    (lambda q, k, v, p, o: dict(out=q), INVALID),
    (lambda q, k, v, p, o: dict(), UNSUPPORTED),                                     # not on a GPU
])
def test_sdpa_tree_refuses(change, status):
    q, k, v = attn()
    kw = dict(q=q, k=k, v=v, parent=tree())
    kw.update(change(q, k, v, kw["parent"], torch.zeros(2, 4, 3, 64, dtype=BF)))
    refuses(status, ops.sdpa_tree, **kw)


@pytest.mark.parametrize("change, status", [
    (dict(acc=torch.zeros(2, 2, 10, dtype=torch.float64)), INVALID),
    (dict(acc=torch.zeros(2, 2, 9)), INVALID),
    (dict(acc=torch.zeros(2, 1, 10).expand(2, 2, 10)), INVALID),          # heads on one another
    (dict(acc=torch.zeros(2, 2, 20)[..., ::2]), INVALID),
    (dict(), UNSUPPORTED),
])
def test_sdpa_decode_accum_refuses(change, status):
    q, k, v = attn()
    refuses(status, ops.sdpa_decode_accum, **{**dict(q=q, k=k, v=v, acc=torch.zeros(2, 2, 10)), **change})


def test_sdpa_decode_accum_refuses_more_causal_queries_than_keys():
    q, k, v = attn(l=11)
    refuses(INVALID, ops.sdpa_decode_accum, q, k, v, torch.zeros(2, 2, 10))


def test_tree_accept_refuses():
    tok = torch.zeros(2, 3, dtype=torch.int64)
    for args in ((tok.int(), tree(), tok), (tok, tree().long(), tok), (tok, tree(), tok.float()), (tok[0], tree(), tok),
                 (tok, tree(2, 4), tok), (tok, tree(), tok[:1]), (tok[:, :0], tree(2, 0), tok[:, :0])):
        refuses(INVALID, ops.tree_accept, *args)
    refuses(UNSUPPORTED, ops.tree_accept, tok, tree(), tok)


def test_kv_tree_commit_refuses():
    _, k, v = attn()
    path, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for args in ((k[0], v[0], path, n, 3), (k, v[:, :, :9], path, n, 3), (k, v, path.long(), n, 3), (k, v, path, n.long(), 3),
                 (k, v, path[:1], n, 3), (k, v, path, n, 0), (k, v, path, n, 2),           # a path longer than the tree
                 (torch.cat([k, k[:1]]), torch.cat([v, v[:1]]), path, n, 3),               # 3 entries of 2 sequences
                 (k, k, path, n, 3),                                                       # one cache for both
                 (k[:, :, :1].expand(-1, -1, 10, -1), v, path, n, 3)):                     # rows on one another
        refuses(INVALID, ops.kv_tree_commit, *args)
    refuses(UNSUPPORTED, ops.kv_tree_commit, k.transpose(2, 3).contiguous().transpose(2, 3), v, path, n, 3)
    refuses(UNSUPPORTED, ops.kv_tree_commit, k, v, path, n, 3)


def test_kv_evict_refuses():
    _, k, v = attn()
    acc, pos, n = torch.zeros(2, 2, 10), torch.zeros(2, 2, 10, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    both = torch.zeros(2, 2, 12)
    for kw in (dict(budget=0), dict(recent=-1), dict(recent=5), dict(acc=acc.double()), dict(pos=pos.long()), dict(acc=acc[..., :9]),
               dict(kv_len=n.long()), dict(kv_len=n[:1]), dict(acc_out=acc.half()), dict(pos_out=pos[:1]), dict(len_out=n.long()),
               dict(acc_out=both[..., 1:11], acc=both[..., :10]), dict(pos_out=pos.view(-1)[:40].view(2, 2, 10).transpose(0, 1)), dict(k=k[:, :, :1].expand(-1, -1, 10, -1)), dict(v=v[:, :1])):
        refuses(INVALID, ops.kv_evict, **{**dict(k=k, v=v, acc=acc, pos=pos, kv_len=n, budget=4), **kw})
    refuses(UNSUPPORTED, ops.kv_evict, k, v, acc, pos, n, 4)
    # another part of the same buffer is another buffer
    refuses(UNSUPPORTED, ops.kv_evict, k, v, torch.zeros(2, 2, 2, 10)[0], pos, n, 4, acc_out=torch.zeros(2, 2, 2, 10)[1])
    pair = torch.zeros(2, 2, 2, 10)
    refuses(UNSUPPORTED, ops.kv_evict, k, v, pair[0], pos, n, 4, acc_out=pair[1])


def test_c_entries_refuse_on_the_host(lib):
    p, null = ctypes.c_void_p(1 << 20), None
    s3 = _lib.strides3(0, 0, 64)

    def tree_call(n=1, hq=2, hkv=2, t=4, s=40, e=64, ev=64, dt=_lib.BF16, q=p, sk=s3, lse=null, scale=0.1, parent=p, ws=p, nb=1 << 30):
        return lib.kuiops_sdpa_tree(n, hq, hkv, t, s, e, ev, dt, q, s3, p, sk, p, s3, p, s3, lse, scale, parent, null, ws, nb, null)
    assert tree_call(hq=3) == tree_call(hkv=0) == tree_call(e=0) == tree_call(q=null) == tree_call(parent=null) == INVALID
    assert tree_call(t=41) == INVALID
    assert tree_call(dt=_lib.F32) == tree_call(e=60) == tree_call(e=264) == tree_call(t=257, s=300) == UNSUPPORTED
    assert tree_call(scale=0.0) == tree_call(scale=-1.0) == tree_call(scale=float("nan")) == tree_call(scale=float("inf")) == UNSUPPORTED
    assert tree_call(q=ctypes.c_void_p((1 << 20) + 8)) == tree_call(sk=_lib.strides3(0, 0, 60)) == UNSUPPORTED
    assert tree_call(sk=_lib.strides3(0, 0, -64)) == UNSUPPORTED
    # a split's keys end past 31-bit offsets
    assert tree_call(s=1 << 29, sk=_lib.strides3(0, 0, 1 << 12)) == UNSUPPORTED
    assert tree_call(n=0) == tree_call(t=0) == _lib.OK
    # splits need their workspace
    need = lib.kuiops_sdpa_tree_workspace(1, 2, 2, 4, 4000, 64, 64)
    assert need > 0 and tree_call(s=4000, ws=null, nb=0) == tree_call(s=4000, nb=need - 1) == _lib.E_WORKSPACE

    def accum_call(l=1, s=40, lse=p, acc=p, sa=_lib.strides3(0, 0, 0)):
        return lib.kuiops_sdpa_decode_accum(1, 2, 2, l, s, 64, 64, _lib.BF16, p, s3, p, s3, p, s3, p, s3, lse, 0.1, 1, null, acc, sa,
                                            p, 1 << 30, null)
    assert accum_call(lse=null) == accum_call(acc=null) == accum_call(sa=null) == accum_call(l=41) == INVALID

    assert lib.kuiops_tree_accept(1, 0, p, p, p, p, p, p, null) == lib.kuiops_tree_accept(1, 4, null, p, p, p, p, p, null) == INVALID
    assert lib.kuiops_tree_accept(1, 257, p, p, p, p, p, p, null) == UNSUPPORTED
    assert lib.kuiops_tree_accept(0, 4, null, null, null, null, null, null, null) == _lib.OK

    r3, q = _lib.strides3(0, 0, 128), ctypes.c_void_p(1 << 21)

    def commit(batch=2, n=2, krow=128, sk=r3, np=3, t=4, ln=p, out=q, vp=q):
        return lib.kuiops_kv_tree_commit(batch, n, 2, 40, krow, 128, p, sk, vp, r3, np, p, t, ln, out, null)
    assert commit(vp=p) == commit(batch=3) == commit(np=5) == commit(t=0) == commit(out=p) == commit(ln=null) == INVALID
    assert commit(krow=120) == commit(sk=_lib.strides3(0, 0, 64)) == commit(sk=_lib.strides3(0, 8, 128)) == commit(np=257, t=300) == UNSUPPORTED

    s2 = _lib.strides3(0, 0, 0)

    def evict(budget=8, recent=2, krow=128, acc=p, ws=p, nb=1 << 20):
        return lib.kuiops_kv_evict(1, 2, 40, krow, 128, p, r3, p, r3, acc, s2, p, s2, p, budget, recent, p, s2, p, s2, p, ws, nb, null)
    assert evict(budget=0) == evict(recent=9) == evict(recent=-1) == evict(acc=null) == INVALID
    assert evict(krow=8) == UNSUPPORTED
    assert evict(ws=null) == evict(nb=lib.kuiops_kv_evict_workspace(1, 2, 8) - 1) == _lib.E_WORKSPACE


def test_c_entries_refuse_launches_of_2_32_threads(lib):
    p, null, s3 = ctypes.c_void_p(1 << 20), None, _lib.strides3(0, 0, 512)
    assert lib.kuiops_sdpa_tree(128, 1 << 15, 1, 256, 300, 256, 256, _lib.BF16, p, s3, p, s3, p, s3, p, s3, null, 0.1, p, null,
                                null, 0, null) == UNSUPPORTED
    assert lib.kuiops_tree_accept(1 << 26, 1, p, p, p, p, p, p, null) == UNSUPPORTED
    assert lib.kuiops_kv_tree_commit(65535, 1, 65535, 40, 512, 512, p, s3, ctypes.c_void_p(1 << 21), _lib.strides3(0, 0, 512), 3, p,
                                     4, p, ctypes.c_void_p(1 << 22), null) == UNSUPPORTED


# ------------------------------------------------------------- custom ops

def test_custom_ops_trace_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from kuillm_amd import library  # noqa: F401
    with FakeTensorMode():
        q, k, v = attn()
        par, n = tree(), torch.zeros(2, dtype=torch.int32)
        op = torch.ops.kuiops
        out, lse = op.sdpa_tree(q, k, v, par, n)
        assert out.shape == (2, 4, 3, 64) and out.dtype == BF and lse.shape == (2, 4, 3) and lse.dtype == torch.float32
        tok = torch.zeros(2, 3, dtype=torch.int64)
        path, count, follow = op.tree_accept(tok, par, tok)
        assert path.shape == (2, 3) and path.dtype == count.dtype == torch.int32 and follow.shape == (2,) and follow.dtype == torch.int64
        assert op.kv_tree_commit(k, v, path, n, 3).shape == (2,)
        acc = torch.zeros(2, 2, 10)
        out, lse = op.sdpa_decode_accum(q, k, v, acc, n)
        assert out.shape == (2, 4, 3, 64) and lse.shape == (2, 4, 3)
        assert op.kv_evict(k, v, acc, torch.zeros(2, 2, 10, dtype=torch.int32), n, 4) is None
    for name, changed in (("kv_tree_commit", 2), ("sdpa_decode_accum", 1), ("kv_evict", 5), ("sdpa_tree", 0), ("tree_accept", 0)):
        schema = getattr(torch.ops.kuiops, name).default._schema
        assert sum(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments) == changed


def test_custom_ops_have_no_cpu_kernel():
    from kuillm_amd import library  # noqa: F401
    q, k, v = attn()
    with pytest.raises(NotImplementedError):
        torch.ops.kuiops.sdpa_tree(q, k, v, tree())


# ------------------------------------------------------------ empty caches

def test_an_empty_cache_has_a_plan(lib):
    # rows per KV head below 16, up to 32 (whose maxima and sums are kept, 8 bytes each) and beyond: no
    # division by the cache's tiles
    for l, held in ((1, 0), (4, 0), (8, 32 * 8 * 8), (16, 0), (100, 0), (2000, 0)):
        assert lib.kuiops_sdpa_decode_accum_workspace(1, 32, 8, l, 0, 64, 64) == held
        assert lib.kuiops_sdpa_tree_workspace(1, 32, 8, l, 0, 64, 64) == 0


@pytest.mark.parametrize("l", [1, 8, 16, 100])
def test_sdpa_decode_accum_of_an_empty_cache_refuses_causal_queries(l):
    q, k, v = attn(n=1, hq=32, hkv=8, l=l, s=0)
    refuses(INVALID, ops.sdpa_decode_accum, q, k, v, torch.zeros(1, 8, 0))
    refuses(UNSUPPORTED, ops.sdpa_decode_accum, q, k, v, torch.zeros(1, 8, 0), causal=False)        # not on a GPU


# ------------------------------------------------------------ largest caches

@pytest.mark.parametrize("e", [64, 128, 256])
def test_weights_of_caches_past_a_launch_are_refused_before_anything_runs(lib, e):
    # rows of 8 read as heads of e: pairs of 32- or 64-key tiles, 512 threads each, or 256 at head dim 256: 2^24 of
    # those for 2^30 - 1 keys (one less, and a launch that fits, for 2^30 - 64)
    p, null, s3, s2 = ctypes.c_void_p(1 << 20), None, _lib.strides3(0, 0, 8), _lib.strides3(0, 0, 0)
    for l in (40, 100):
        got = lib.kuiops_sdpa_decode_accum(1, 1, 1, l, (1 << 30) - 1, e, e, _lib.BF16, p, s3, p, s3, p, s3, p, s3, p, 0.1, 1, null, p, s2,
                                           p, 1 << 50, null)
        assert got == UNSUPPORTED


def test_kv_tree_commit_of_a_path_without_entries(lib):
    # nothing was accepted: no path to read, so none is asked for; the call goes as far as the device
    p, q, null, r3 = ctypes.c_void_p(1 << 20), ctypes.c_void_p(1 << 21), None, _lib.strides3(0, 0, 128)
    for entries, status in ((3, INVALID), (0, UNSUPPORTED)):
        # (rows of 120 bytes: refused behind the check of the path)
        assert lib.kuiops_kv_tree_commit(1, 1, 2, 40, 120, 128, p, r3, q, r3, entries, null, 4, p, q, null) == status
    _, k, v = attn()
    refuses(UNSUPPORTED, ops.kv_tree_commit, k, v, torch.zeros(2, 0, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 3)
