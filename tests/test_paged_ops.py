"""Paged KV caches without a GPU: the oracle against closed forms, where the kernels
look for a slot (compiled for the host), and what the entry points refuse before
anything is enqueued."""
import ctypes
import shutil
import subprocess

import numpy as np
import pytest
import torch

from kuillm_amd import _lib, compile as _compile, config as C, ops
from oracle import kuiops_oracle as O

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
INVALID, UNSUPPORTED = _lib.E_INVALID, _lib.E_UNSUPPORTED


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not C.LIB_PATH.exists():
        _compile.build_library()
    return _lib.load()


# ------------------------------------------------------------------ oracle

def test_slots_by_hand():
    row = [3, -1, 0, 7]
    assert O.paged_slot(row, 16, 5, 0) == (3, 0) and O.paged_slot(row, 16, 5, 47) == (0, 15)
    for slot in (-1, 16, 31, 48, 64):                # before, no page, one past the pool, past the table
        assert O.paged_slot(row, 16, 5, slot) is None


def test_e4m3_rounds_as_torch_does():
    r = np.random.default_rng(0)
    y = np.concatenate([r.uniform(-448, 448, 4000), r.standard_normal(4000) * 0.02, [0, 448, -448, 2.0 ** -10, 2.0 ** -9 * 1.5, 17, 19, 2.0 ** -6 * 0.99]])
    y = y.astype(np.float32)
    np.testing.assert_array_equal(O.nearest_e4m3(y), torch.from_numpy(y).to(F8).double().numpy())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_quantised_rows_by_hand(kind):
    M = 127 if kind == "int8" else 448
    x = np.array([[0.0, 1.0, -2.0, 0.5], [0, 0, 0, 0], [1, np.inf, 0, 0], [np.nan, 1, 2, 3]])
    stored, scale, _ = O.quantise_rows(x, kind)
    assert stored[0].tolist() == ([0, 64, -127, 32] if kind == "int8" else [0, 224, -448, 112])      # 63.5 and 31.75 of 127
    assert scale[:2].tolist() == [2 / M, 0] and np.isnan(scale[2:]).all() and not stored[1:].any()
    # within half a step of the row
    r = np.random.default_rng(0).standard_normal((50, 64))
    stored, scale, off = O.quantise_rows(r, kind)
    step = 0.5 if kind == "int8" else 16.0
    assert (np.abs(stored * scale[:, None] - r) <= step * scale[:, None] * 1.0000001).all() and (off <= 0.5).all()


def test_norm_and_rotation_by_hand():
    x = np.array([3.0, 0, 4, 0])
    y, _ = O.norm_rope(x, None, 0, 0, [1.0, 0.5])
    assert y.tolist() == x.tolist()
    y, _ = O.norm_rope(x, [1, 1, 1, 1], 0, 2, [np.pi / 4, 0.5])          # a quarter turn of the pair (3, 4) / rms
    np.testing.assert_allclose(y, np.array([-4.0, 0, 3, 0]) / 2.5, atol=1e-15)


def test_a_full_table_is_a_cache():
    r = np.random.default_rng(1)
    k, v, q = r.standard_normal((1, 2, 48, 8)), r.standard_normal((1, 2, 48, 8)), r.standard_normal((1, 4, 3, 8))
    pages = [x[0].reshape(2, 3, 16, 8).transpose(1, 0, 2, 3)[[2, 0, 1]] for x in (k, v)]
    out, lse, _, _ = O.sdpa_paged(q, *pages, [[1, 2, 0]], [41])
    ref, lref, _, _, _ = O.sdpa_decode_accum(q, k, v, np.zeros((1, 2, 48)), [41])
    np.testing.assert_allclose(out, ref, rtol=1e-12)
    np.testing.assert_allclose(lse, lref, rtol=1e-12)


def test_queries_keep_their_slots_past_the_table():
    r = np.random.default_rng(2)
    k, v, q = r.standard_normal((3, 1, 16, 8)), r.standard_normal((3, 1, 16, 8)), r.standard_normal((1, 2, 4, 8))
    whole, _, _, _ = O.sdpa_paged(q, k, v, [[0, 1, 2]], [34])                # slots 30 .. 33
    out, _, _, _ = O.sdpa_paged(q, k, v, [[0, 1]], [34])
    np.testing.assert_array_equal(out[:, :, :2], whole[:, :, :2])
    without, _, _, _ = O.sdpa_paged(q, k, v, [[0, 1, -1]], [34])
    np.testing.assert_array_equal(out, without)


# ------------------------------------------------- the kernels' arithmetic, on the host

@pytest.fixture(scope="module")
def index(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    at = tmp_path_factory.mktemp("index")
    (at / "index.cpp").write_text('#include "paged_index.hpp"\nextern "C" {\n'
                                  "int slots(int a, int b, int c) { return kuiops::paged_slots(a, b, c); }\n"
                                  "int rows16(int a, int b, int c) { return kuiops::paged_rows16(a, b, c); }\n"
                                  "int find(const int32_t *r, int w, int p, int n, int s, int *at) { return kuiops::paged_find(r, w, p, kuiops::paged_div(p / 16), n, s, *at); }\n"
                                  "int entry(int s, int p, int *at) { return kuiops::paged_entry(s, p, kuiops::paged_div(p / 16), *at); }\n"
                                  "int id(int e, int n) { return kuiops::paged_id(e, n); }\n"
                                  "int quotient(int x, int d) { return kuiops::paged_quotient(x, kuiops::paged_div(d)); }\n}\n")
    subprocess.run([gxx, "-std=c++17", "-shared", "-fPIC", f"-I{C.CSRC}", "-o", str(at / "index.so"), str(at / "index.cpp")], check=True)
    return ctypes.CDLL(str(at / "index.so"))


BAD = [-1, -2, -2 ** 31, 2 ** 31 - 1]


@pytest.mark.parametrize("page,width,pages", [(16, 5, 7), (48, 3, 1), (1024, 2, 3), (16, 1, 0), (32, 40, 64), (1 << 20, 3, 2)])
def test_every_slot_lies_in_the_pool_or_nowhere(index, page, width, pages):
    g = np.random.default_rng(page + width)
    row = g.integers(0, max(pages, 1), width).astype(np.int32)
    hit = g.random(width) < 0.4
    row[hit] = g.choice(BAD + [pages, pages + 1], hit.sum())
    # (entries on both sides of the row are pages that a read outside of it would take)
    buf = np.concatenate([np.zeros(4, np.int32), row, np.zeros(4, np.int32)])
    ptr = ctypes.c_void_p(buf.ctypes.data + 16)
    at = ctypes.c_int()
    slots = sorted(set(g.integers(0, width * page, 300).tolist()) | {0, page - 1, page, width * page - 1, width * page, width * page + 5, -1, -page})
    for slot in slots:
        ref = O.paged_slot(row, page, pages, slot)
        got = index.find(ptr, width, page, pages, slot, ctypes.byref(at))
        assert (got, at.value) == ref if ref is not None else got == -1
    for length in (-5, 0, 1, 15, 16, 17, page, width * page, width * page + 1, 2 ** 31 - 1):
        end = index.slots(length, width, page)
        assert end == min(max(length, 0), width * page)
        for slot in [s // 16 * 16 for s in slots]:
            # (as the attention does: the entry of a slot at or behind the end is not fetched)
            p = index.entry(max(slot, 0), page, ctypes.byref(at))
            got = index.id(int(row[p]), pages) if 0 <= slot < end else -1
            n = index.rows16(got, slot, end)
            assert 0 <= n <= 16
            if got >= 0:
                assert 0 <= slot < end and n > 0 and at.value % 16 == 0
            for i in range(n):
                assert O.paged_slot(row, page, pages, slot + i) == (got, at.value + i) and slot + i < end
            for i in range(n, 16):          # the others have no page or lie behind the sequence
                assert slot + i >= end or slot < 0 or O.paged_slot(row, page, pages, slot + i) is None


def test_the_quotient_is_exact(index):
    # below 2^26 (2^30 slots in groups of 16), by up to 2^16 groups of a page
    g = np.random.default_rng(0)
    for d in [1, 2, 3, 5, 7, 31, 32, 33, 1000, 4095, 4097, 32768, 32769, 65535, 65536] + g.integers(1, 65537, 200).tolist():
        top = 2 ** 26 - 1
        for x in [0, 1, d - 1, d, d + 1, top, top // d * d, top // d * d - 1] + g.integers(0, top + 1, 50).tolist():
            if 0 <= x <= top:
                assert index.quotient(x, d) == x // d, (x, d)


# ---------------------------------------------------------------- refusals

def refuses(status, fn, *args, **kw):
    with pytest.raises(_lib.KuiopsError) as err:
        fn(*args, **kw)
    assert err.value.status == status


def cache(dtype=BF, pages=6, hkv=2, page=16, hd=64, n=2, width=3):
    kw = dict(k_pages=torch.zeros(pages, hkv, page, hd, dtype=dtype), v_pages=torch.zeros(pages, hkv, page, hd, dtype=dtype),
              table=torch.zeros(n, width, dtype=torch.int32))
    if dtype in (torch.int8, F8):
        kw.update(k_scale=torch.zeros(pages, hkv, page), v_scale=torch.zeros(pages, hkv, page))
    return kw


def append_args(dtype=BF, **kw):
    return dict(qkv=torch.zeros(2, 3, 8 * 64, dtype=BF), inv_freq=torch.ones(32), pos0=torch.zeros(2, dtype=torch.int32), **cache(dtype, **kw))


def read_args(dtype=BF, **kw):
    return dict(kv_len=torch.zeros(2, dtype=torch.int32), **cache(dtype, **kw))


def attn_args(dtype=BF, **kw):
    return dict(q=torch.zeros(2, 4, 1, 64, dtype=BF), **read_args(dtype, **kw))


ENTRIES = [(ops.kv_paged_append, append_args), (ops.kv_paged_read, read_args), (ops.sdpa_paged, attn_args)]


@pytest.mark.parametrize("fn, args", ENTRIES)
@pytest.mark.parametrize("dtype, change, status", [
    (BF, lambda a: dict(k_pages=a["k_pages"][0]), INVALID),                                   # rank
    (BF, lambda a: dict(v_pages=a["v_pages"][:5]), INVALID),                                  # pools differ
    (BF, lambda a: dict(v_pages=a["v_pages"].half()), INVALID),
    (BF, lambda a: dict(k_pages=a["k_pages"].float(), v_pages=a["v_pages"].float()), UNSUPPORTED),
    (BF, lambda a: dict(table=a["table"].long()), INVALID),
    (BF, lambda a: dict(table=a["table"][0]), INVALID),
    (BF, lambda a: dict(table=a["table"].repeat(1, 2)[:, ::2]), UNSUPPORTED),                 # entries apart
    (BF, lambda a: dict(table=a["table"][:1]), INVALID),                                      # a sequence without a row
    (BF, lambda a: dict(k_scale=torch.zeros(6, 2, 16), v_scale=torch.zeros(6, 2, 16)), INVALID),      # 16-bit pages have none
    (BF, lambda a: dict(k_pages=a["k_pages"][:1].expand(6, -1, -1, -1)), INVALID),            # pages on one another
    (BF, lambda a: dict(k_pages=a["k_pages"].transpose(2, 3).contiguous().transpose(2, 3)), INVALID),
    (torch.int8, lambda a: dict(k_scale=None), INVALID),
    (torch.int8, lambda a: dict(v_scale=a["v_scale"].half()), INVALID),
    (torch.int8, lambda a: dict(v_scale=a["v_scale"][:, :1]), INVALID),
    (F8, lambda a: dict(k_scale=torch.zeros(6, 2, 32)[:, :, ::2]), INVALID),
    (BF, lambda a: {}, UNSUPPORTED),                                                          # not on a GPU
    (torch.int8, lambda a: {}, UNSUPPORTED),
    (F8, lambda a: {}, UNSUPPORTED),
])
def test_caches_that_are_refused(fn, args, dtype, change, status):
    a = args(dtype)
    a.update(change(a))
    refuses(status, fn, **a)


@pytest.mark.parametrize("change, status", [
    (dict(qkv=torch.zeros(2, 512, dtype=BF)), INVALID),
    (dict(qkv=torch.zeros(2, 3, 500, dtype=BF)), INVALID),                    # not whole heads
    (dict(qkv=torch.zeros(2, 3, 192, dtype=BF)), INVALID),                    # fewer than the cache's
    (dict(qkv=torch.zeros(3, 3, 512, dtype=BF)), INVALID),                    # a sequence more
    (dict(qkv=torch.zeros(2, 3, 512)), UNSUPPORTED),
    (dict(qkv=torch.zeros(2, 3, 512, dtype=torch.half)), INVALID),            # not the pages' type
    (dict(inv_freq=torch.ones(64)), INVALID),
    (dict(inv_freq=torch.ones(32, dtype=torch.float64)), INVALID),
    (dict(pos0=torch.zeros(2, dtype=torch.int64)), INVALID),
    (dict(pos0=torch.zeros(1, dtype=torch.int32)), INVALID),
    (dict(lens=torch.zeros(4, dtype=torch.int32)[::2]), INVALID),
    (dict(q_norm=torch.ones(64)), INVALID),
    (dict(k_norm=torch.ones(32, dtype=BF)), INVALID),
    (dict(q_out=torch.zeros(2, 4, 3, 64)), INVALID),
    (dict(q_out=torch.zeros(2, 4, 2, 64, dtype=BF)), INVALID),
    (dict(q_out=torch.zeros(2, 1, 3, 64, dtype=BF).expand(2, 4, 3, 64)), INVALID),
])
def test_kv_paged_append_refuses(change, status):
    refuses(status, ops.kv_paged_append, **{**append_args(), **change})


def test_kv_paged_append_refuses_one_pool_for_both():
    a = append_args()
    refuses(INVALID, ops.kv_paged_append, **{**a, "v_pages": a["k_pages"]})


@pytest.mark.parametrize("change, status", [
    (dict(kv_len=torch.zeros(2, dtype=torch.int64)), INVALID),
    (dict(kv_len=torch.zeros(3, dtype=torch.int32)), INVALID),
    (dict(length=-1), INVALID),
    (dict(dtype=torch.half), UNSUPPORTED),                                    # 16-bit pages come as they are
    (dict(dtype=torch.float32), UNSUPPORTED),
    (dict(k_out=torch.zeros(2, 2, 48, 64, dtype=BF)), INVALID),               # one of the two
    (dict(k_out=torch.zeros(2, 2, 48, 64, dtype=BF), v_out=torch.zeros(2, 2, 47, 64, dtype=BF)), INVALID),
    (dict(k_out=torch.zeros(2, 2, 48, 64, dtype=BF), v_out=torch.zeros(2, 1, 48, 64, dtype=BF).expand(2, 2, 48, 64)), INVALID),
])
def test_kv_paged_read_refuses(change, status):
    refuses(status, ops.kv_paged_read, **{**read_args(), **change})
    out = torch.zeros(2, 2, 48, 64, dtype=BF)
    refuses(INVALID, ops.kv_paged_read, **read_args(), k_out=out, v_out=out)


@pytest.mark.parametrize("change, status", [
    (dict(q=torch.zeros(4, 1, 64, dtype=BF)), INVALID),
    (dict(q=torch.zeros(2, 3, 1, 64, dtype=BF)), INVALID),                    # 3 heads over 2
    (dict(q=torch.zeros(2, 4, 1, 32, dtype=BF)), INVALID),
    (dict(q=torch.zeros(3, 4, 1, 64, dtype=BF)), INVALID),
    (dict(q=torch.zeros(2, 4, 1, 64, dtype=torch.half)), INVALID),
    (dict(q=torch.zeros(2, 4, 1, 64)), UNSUPPORTED),
    (dict(kv_len=torch.zeros(2, dtype=torch.int64)), INVALID),
    (dict(out=torch.zeros(2, 4, 1, 64)), INVALID),
    (dict(out=torch.zeros(2, 4, 2, 64, dtype=BF)), INVALID),
])
def test_sdpa_paged_refuses(change, status):
    refuses(status, ops.sdpa_paged, **{**attn_args(), **change})


def test_sdpa_paged_refuses_its_query_as_output():
    a = attn_args()
    refuses(INVALID, ops.sdpa_paged, **a, out=a["q"])


def test_what_shares_memory():
    # against the sets of bytes, over small layouts of any strides
    g = np.random.default_rng(5)

    def some():
        size = int(g.choice([1, 2, 4]))
        shape = tuple(int(x) for x in g.integers(1, 4, g.integers(1, 4)))
        return shape, tuple(int(x) for x in g.integers(0, 9, len(shape))), {1: torch.int8, 2: BF, 4: torch.float32}[size]

    def places(x, at):
        own = {0}
        for count, st in zip(*x[:2]):
            own = {o + i * st for o in own for i in range(count)}
        return {at + o * x[2].itemsize + i for o in own for i in range(x[2].itemsize)}
    seen = [0, 0]
    for _ in range(4000):
        a, b, to = some(), some(), int(g.integers(-30, 40))
        shared = bool(places(a, 0) & places(b, to))
        assert ops._apart(100, ops._extent(a), 100 + to, ops._extent(b)) != shared, (a, b, to)
        seen[shared] += 1
    assert min(seen) > 500
    empty = ops._extent(((3, 0), (4, 1), BF))
    assert ops._apart(0, empty, 0, ops._extent(((4,), (1,), BF))) and ops._apart(0, None, 0, empty)
    # strides that do not nest, as large as tensors are: an answer, and soon
    x = ops._extent(((1 << 20, 1 << 20), (7, 3), BF))
    assert not ops._apart(0, x, 1, x)


def takes(fn, **a):
    refuses(UNSUPPORTED, fn, **a)              # all that is left to refuse: it is not on a GPU


def test_kv_paged_append_refuses_shared_scales_and_pools_that_overlap():
    for dtype in (torch.int8, F8):
        a = append_args(dtype)
        refuses(INVALID, ops.kv_paged_append, **{**a, "v_scale": a["k_scale"]})
        scales = torch.zeros(7, 2, 16)
        refuses(INVALID, ops.kv_paged_append, **{**a, "k_scale": scales[:6], "v_scale": scales[1:]})
        both = torch.zeros(6, 2, 2, 16)
        takes(ops.kv_paged_append, **{**a, "k_scale": both[:, 0], "v_scale": both[:, 1]})
    a = append_args()
    pool = torch.zeros(12, 2, 16, 64, dtype=BF)
    refuses(INVALID, ops.kv_paged_append, **{**a, "k_pages": pool[:6], "v_pages": pool[1:7]})
    refuses(INVALID, ops.kv_paged_append, **{**a, "k_pages": pool[5:11], "v_pages": pool[:6]})
    takes(ops.kv_paged_append, **{**a, "k_pages": pool[:6], "v_pages": pool[6:]})
    takes(ops.kv_paged_append, **{**a, "k_pages": pool[::2], "v_pages": pool[1::2]})
    heads = torch.zeros(6, 4, 16, 64, dtype=BF)
    takes(ops.kv_paged_append, **{**a, "k_pages": heads[:, :2], "v_pages": heads[:, 2:]})
    refuses(INVALID, ops.kv_paged_append, **{**a, "k_pages": heads[:, :2], "v_pages": heads[:, 1:3]})
    rows = torch.zeros(6, 2, 16, 128, dtype=BF)
    takes(ops.kv_paged_append, **{**a, "k_pages": rows[..., 64:], "v_pages": rows[..., :64]})
    # halves of the same rows, the heads of one in the order of the other's slots
    rows = torch.zeros(6, 64, 2, 128, dtype=BF)
    mixed = rows.view(6, 2, 64, 128)
    for page in (16, 64):
        k, v = rows[:, :page, :, :64].transpose(1, 2), mixed[:, :, :page, 64:]
        takes(ops.kv_paged_append, **{**a, "k_pages": k, "v_pages": v})
        refuses(INVALID, ops.kv_paged_append, **{**a, "k_pages": k, "v_pages": mixed[:, :, :page, 63:127]})
    large = torch.empty(10, 4096, 8, 256, dtype=BF, device="meta")
    k, v = (ops._extent(ops._meta(x)) for x in (large[..., :128].transpose(1, 2), large.view(10, 8, 4096, 256)[..., 128:]))
    assert ops._apart(0, k, 256, v) and not ops._apart(0, k, 254, v)
    # one pool to read keys and values from is no mistake
    for fn, args in ENTRIES[1:]:
        b = args()
        takes(fn, **{**b, "v_pages": b["k_pages"]})


def test_kv_paged_append_refuses_a_query_output_on_its_inputs():
    a = append_args()
    wide = torch.zeros(2, 3, 800, dtype=BF)
    a["qkv"] = wide[..., :512]
    for first, fn in ((0, refuses), (256, refuses), (511, refuses), (512, None), (544, None)):
        view = wide[..., first:first + 256].view(2, 3, 4, 64).transpose(1, 2)
        takes(ops.kv_paged_append, **a, q_out=view) if fn is None else fn(INVALID, ops.kv_paged_append, **a, q_out=view)
    for pool in (a["k_pages"], a["v_pages"]):
        refuses(INVALID, ops.kv_paged_append, **a, q_out=pool.view(-1)[-2 * 4 * 3 * 64:].view(2, 4, 3, 64))
    a = append_args(torch.int8)
    scales = torch.zeros(1000)
    refuses(INVALID, ops.kv_paged_append, **{**a, "v_scale": scales[:192].view(6, 2, 16)},
            q_out=scales.view(BF)[380:380 + 1536].view(2, 4, 3, 64))


def test_kv_paged_read_refuses_outputs_that_overlap():
    a = read_args()
    out = torch.zeros(2, 2, 97, 64, dtype=BF)
    refuses(INVALID, ops.kv_paged_read, **a, k_out=out[:, :, :48], v_out=out[:, :, 47:95])
    takes(ops.kv_paged_read, **a, k_out=out[:, :, :48], v_out=out[:, :, 48:96])
    for dtype in (BF, torch.int8):
        a = read_args(dtype)
        far = torch.zeros(2, 2, 8, 64, dtype=BF)
        for name in ("k_pages", "v_pages") + (("k_scale", "v_scale") if dtype != BF else ()):
            base = torch.zeros(64 << 10, dtype=torch.uint8)
            x = a[name]
            b = {**a, name: base[:x.numel() * x.element_size()].view(x.dtype).view(x.shape)}
            at = x.numel() * x.element_size() - 16
            on, off = (base[i:i + 4096].view(BF).view(2, 2, 8, 64) for i in (at, at + 16))
            for outs in ((on, far), (far, on)):
                refuses(INVALID, ops.kv_paged_read, **b, k_out=outs[0], v_out=outs[1])
            takes(ops.kv_paged_read, **b, k_out=off, v_out=far)


def test_sdpa_paged_refuses_an_output_on_its_inputs():
    a = attn_args()
    buf = torch.zeros(2, 8, 1, 64, dtype=BF)
    refuses(INVALID, ops.sdpa_paged, **{**a, "q": buf[:, :4]}, out=buf[:, 1:5])
    takes(ops.sdpa_paged, **{**a, "q": buf[:, :4]}, out=buf[:, 4:])
    for name in ("k_pages", "v_pages"):
        refuses(INVALID, ops.sdpa_paged, **a, out=a[name].view(-1)[-512:].view(2, 4, 1, 64))
    b = attn_args(F8)
    scales = torch.zeros(512)
    refuses(INVALID, ops.sdpa_paged, **{**b, "k_scale": scales[:192].view(6, 2, 16)}, out=scales.view(BF)[382:894].view(2, 4, 1, 64))
    takes(ops.sdpa_paged, **{**b, "k_scale": scales[:192].view(6, 2, 16)}, out=scales.view(BF)[384:896].view(2, 4, 1, 64))


def layout(pages=6, page=16, hkv=2, hd=64, width=3, dtype=_lib.BF16, row=64, scale=16):
    at = _lib.PagedLayout(pages=pages, page=page, hkv=hkv, hd=hd, width=width, ld_table=width, dtype=dtype)
    at.sk[:] = at.sv[:] = (hkv * page * row, page * row, row)
    at.sks[:] = at.svs[:] = (hkv * scale, scale)
    return at


def test_c_entries_refuse_on_the_host(lib):
    p, null, s3 = ctypes.c_void_p(1 << 20), None, _lib.strides3(0, 0, 64)
    off = ctypes.c_void_p((1 << 20) + 8)

    def attn(n=2, hq=4, l=1, dt=_lib.BF16, q=p, at=None, k=p, ks=null, tb=p, ln=p, sq=s3, sm=0.1, ws=p, nb=1 << 30, **kw):
        return lib.kuiops_sdpa_paged(n, hq, l, dt, q, sq, at or layout(**kw), k, p, ks, ks, tb, ln, p, s3, null, sm, ws, nb, null)

    def append(n=2, t=3, hq=4, dt=_lib.BF16, x=p, ld=512, f=p, w=null, eps=1e-6, at=None, k=p, ks=null, tb=p, **kw):
        return lib.kuiops_kv_paged_append(n, t, hq, dt, x, ld, 3 * 512, null, null, f, w, w, eps, p, s3, at or layout(**kw), k, p, ks, ks, tb, null)

    def read(n=2, s=40, dt=_lib.BF16, at=None, k=p, ks=null, tb=p, ln=p, out=p, so=s3, **kw):
        return lib.kuiops_kv_paged_read(n, s, dt, at or layout(**kw), k, p, ks, ks, tb, ln, out, so, p, s3, 0, null)

    for call in (attn, append, read):
        assert call(n=-1) == call(k=null) == call(tb=null) == call(page=0) == call(pages=-1) == call(width=-1) == call(hkv=0) == INVALID
        assert call(dt=_lib.F16) == INVALID                                   # not the pages' type
        assert call(dtype=_lib.I8) == INVALID                                 # no scales
        assert call(hd=72) == call(hd=144, row=144) == call(page=24) == call(page=8) == UNSUPPORTED
        assert call(page=1 << 21) == call(width=1 << 26) == UNSUPPORTED       # 2^30 slots
        assert call(k=off) == call(row=60) == call(row=32) == call(row=1 << 24) == UNSUPPORTED
        assert call(dtype=_lib.I8, ks=off) == call(dtype=_lib.F8E4M3, ks=p, row=72) == call(dtype=_lib.I8, ks=p, scale=18) == UNSUPPORTED
        assert call(dtype=_lib.F32) == call(dtype=_lib.I32) == UNSUPPORTED
        bad = layout()
        bad.sk[0] = -64
        assert call(at=bad) == UNSUPPORTED
        assert call(n=0) == _lib.OK
    assert attn(dt=_lib.F32) == append(dt=_lib.F32) == UNSUPPORTED
    assert read(dt=_lib.F32) == UNSUPPORTED                                   # 16-bit pages as fp32
    assert attn(hq=3) == attn(q=null) == attn(ln=null) == INVALID
    assert attn(sm=0.0) == attn(sm=-1.0) == attn(sm=float("nan")) == attn(sm=float("inf")) == UNSUPPORTED
    assert attn(q=off) == attn(sq=_lib.strides3(0, 0, 60)) == UNSUPPORTED
    assert attn(n=1 << 19) == attn(n=1 << 18, width=1 << 16) == attn(l=1 << 24) == attn(hq=1 << 20, l=1 << 10) == UNSUPPORTED
    assert attn(l=0) == attn(hq=0) == append(t=0) == read(s=0) == _lib.OK
    assert append(x=null) == append(f=null) == append(eps=-1.0) == append(eps=float("nan")) == append(eps=float("inf")) == INVALID
    assert append(ld=500) == append(x=off) == append(w=off) == append(n=1 << 16) == append(t=1 << 24) == UNSUPPORTED
    assert read(ln=null) == read(out=null) == INVALID
    assert read(out=off) == read(so=_lib.strides3(0, 0, 60)) == read(s=1 << 30) == read(n=1 << 16) == read(n=1 << 15, s=1 << 15) == UNSUPPORTED
    # splits need their workspace
    need = lib.kuiops_sdpa_paged_workspace(2, 4, 2, 1, 4800, 64)
    assert need > 0
    assert attn(width=300, ws=null, nb=0) == attn(width=300, nb=need - 1) == attn(width=300, ws=off) == _lib.E_WORKSPACE


def test_pages_of_one_row_are_refused_whatever_their_strides(lib):
    # (torch lets the stride of an axis of one entry be anything; the layout has 0 for it)
    p, null, s3 = ctypes.c_void_p(1 << 20), None, _lib.strides3(0, 0, 64)
    for row in (0, 64, 128):
        at = layout(page=1)
        at.sk[2] = at.sv[2] = row
        assert lib.kuiops_kv_paged_read(2, 40, _lib.BF16, at, p, p, null, null, p, p, p, s3, p, s3, 0, null) == UNSUPPORTED
        assert lib.kuiops_sdpa_paged(2, 4, 1, _lib.BF16, p, s3, at, p, p, null, null, p, p, p, s3, null, 0.1, p, 1 << 30, null) == UNSUPPORTED


def test_workspace_sizes(lib):
    assert f"#define KUIOPS_SDPA_PAGED_ZEROED {_lib.SDPA_PAGED_ZEROED}\n" in (C.INCLUDE / "kuiops.h").read_text()
    f = lib.kuiops_sdpa_paged_workspace
    for args in ((0, 4, 2, 1, 48, 64), (2, 4, 2, 1, 0, 64), (2, 3, 2, 1, 48, 64), (2, 4, 0, 1, 48, 64), (1, 4, 1, 1, 32, 64)):
        assert f(*args) == 0
    assert f(1, 32, 8, 1, 1 << 20, 128) <= 10 << 20


def test_many_query_rows_need_no_workspace(lib):
    # a piece of a work-group for each 16 rows of a KV head: from 129 groups of rows on a work-group has all
    # keys, nothing is split, and the states' space does not grow with the rows
    f = lib.kuiops_sdpa_paged_workspace
    assert f(1, 16, 1, 128, 8000, 128) > 0
    for l in (129, 300, 8192, 1 << 20):
        assert f(1, 16, 1, l, 8000, 128) == f(2, 128, 8, l, 1 << 20, 128) == 0
    most = max(f(n, 16 * g, g, l, 1 << 16, 128) for n in (1, 2, 16, 64, 300) for g in (1, 8) for l in (1, 2, 5, 16, 100, 128, 129, 1000))
    assert most <= 40 << 20


# ------------------------------------------------------------- custom ops

def test_custom_ops_trace_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from kuillm_amd import library  # noqa: F401
    op = torch.ops.kuiops
    with FakeTensorMode():
        for dtype in (BF, torch.int8, F8):
            q = op.kv_paged_append(**append_args(dtype))
            assert q.shape == (2, 4, 3, 64) and q.dtype == BF
            k, v = op.kv_paged_read(**read_args(dtype), length=40)
            assert k.shape == v.shape == (2, 2, 40, 64) and k.dtype == v.dtype == BF
            out, lse = op.sdpa_paged(**attn_args(dtype))
            assert out.shape == (2, 4, 1, 64) and out.dtype == BF and lse.shape == (2, 4, 1) and lse.dtype == torch.float32
        assert op.kv_paged_read(**read_args(F8), length=40, dtype=torch.float32)[0].dtype == torch.float32
    for name, changed in (("kv_paged_append", 4), ("kv_paged_read", 0), ("sdpa_paged", 0)):
        schema = getattr(op, name).default._schema
        assert sum(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments) == changed


def test_custom_ops_have_no_cpu_kernel():
    from kuillm_amd import library  # noqa: F401
    with pytest.raises(NotImplementedError):
        torch.ops.kuiops.sdpa_paged(**attn_args())
