"""Paged KV caches on the GPU against the fp64 oracle.

Tolerances.  u = eps / 2 is half a step of the output type.

Attention: as for the contiguous cache's operators (probabilities keep 2^-16 and more;
scores, scaled by 8-bit pages' scales or not, are fp32 sums of hd exact products).

Queries and 16-bit keys: fp32, one rounding u at the end.  The sum of squares is off by
(hd / 8 + 4) 2^-24 at most (relative; 16 values a lane and 3 lane steps), its mean, eps,
root, quotient and the weight by 5 2^-24, cos and sin by 2^-24, the rotation's products and
sum by 3 2^-24: (hd / 16 + 11) 2^-24 < hd 2^-24 / 4 + 2^-20 of the sum S of its absolute terms.

8-bit rows: 64 bits, errors below (hd + 40) 2^-52 of |x| < 2^-43, at most 127 2^-43 < 2^-36 steps of
int8, 2^-36 of e4m3's too: equal where no border is nearer than 2^-30 steps."""
import math

import numpy as np
import pytest
import torch

from kuillm_amd import ops
from oracle import kuiops_oracle as O
from test_gpu_cache import BF, HF, close_lse, close_out, gen, npy

pytestmark = pytest.mark.gpu
F8, I8 = torch.float8_e4m3fn, torch.int8
NAN = float("nan")


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


class Cache:
    """A paged cache with everything filled, its pages dealt to the sequences in any order."""

    def __init__(self, device, dtype, kind, n, hkv, hd, page, width, seed=0, spare=2):
        g = np.random.default_rng(seed)
        P = n * width + spare
        self.table = g.permutation(P)[:n * width].reshape(n, width).astype(np.int32)
        self.device, self.dtype, self.kind = device, dtype, kind
        self.pages, self.scales = [], []
        for i in range(2):
            x = gen((P, hkv, page, hd), dtype, 10 * seed + i)
            if kind == "same":
                self.pages.append(x.to(device))
                self.scales.append(None)
            else:
                stored, scale, _ = O.quantise_rows(npy(x), kind)
                self.pages.append(torch.from_numpy(stored).to(I8 if kind == "int8" else F8).to(device))
                self.scales.append(torch.from_numpy(scale).float().to(device))

    def args(self):
        return dict(k_pages=self.pages[0], v_pages=self.pages[1], table=torch.from_numpy(self.table).to(self.device),
                    k_scale=self.scales[0], v_scale=self.scales[1])

    def numbers(self):
        return [npy(p) for p in self.pages], [None if s is None else npy(s) for s in self.scales]

    def attention(self, q, lens, scale=None):
        (k, v), (ks, vs) = self.numbers()
        return O.sdpa_paged(npy(q), k, v, self.table, lens, ks, vs, scale)


def attends(c, q, lens, scale=None):
    ref, lref, size, terms = c.attention(q, lens, scale)
    out, lse = ops.sdpa_paged(q.to(c.device), **c.args(), kv_len=ints(lens, c.device), scale=scale, return_lse=True)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    close_out(out, ref, size, terms, q.shape[-1], False)
    close_lse(lse, lref, terms, q.shape[-1])
    return out, lse


KINDS = ["same", "int8", "e4m3"]
SHAPES = [  # n, hq, hkv, l, hd, page, lens
    (1, 1, 1, 1, 64, 16, (1,)),
    (1, 4, 2, 1, 128, 16, (0,)),                             # an empty sequence
    (3, 8, 2, 1, 64, 32, (33, 0, 600)),                      # ragged, one empty
    (2, 14, 2, 1, 64, 48, (100, 47)),                        # pages of no power of two
    (2, 40, 2, 1, 128, 16, (130, 129)),                      # 20 rows: two row groups
    (1, 32, 8, 4, 128, 64, (515,)),                          # drafted tokens, a page that ends inside a tile
    (2, 8, 8, 3, 64, 128, (3, 2)),                           # as many queries as keys, and more
    (1, 16, 1, 20, 128, 16, (300,)),                         # 320 rows
    (1, 4, 4, 1, 16, 16, (50,)),                             # head dims of their own
    (1, 6, 2, 2, 96, 32, (77,)),
    (2, 4, 1, 1, 112, 16, (31, 32)),
    (1, 3, 1, 1, 48, 64, (64,)),
    (1, 8, 1, 1, 128, 1024, (2100,)),                        # large pages, splits
    (1, 2, 2, 1, 64, 16, (4097,)),                           # many splits, the last of one key
    (17, 2, 1, 1, 64, 16, tuple(range(0, 17 * 9, 9))),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,l,hd,page,lens", SHAPES)
def test_sdpa_paged(cuda, n, hq, hkv, l, hd, page, lens, dtype, kind):
    c = Cache(cuda, dtype, kind, n, hkv, hd, page, max(1, -(-max(lens) // page)) + 1, seed=3)
    attends(c, gen((n, hq, l, hd), dtype, 1), lens)


def some_of(c, q, lens, picked):
    """Attention of all sequences, checked for the picked ones."""
    out, lse = ops.sdpa_paged(q.to(c.device), **c.args(), kv_len=ints(lens, c.device), return_lse=True)
    for b in picked:
        own = torch.from_numpy(c.table[b].astype(np.int64)).to(c.device)
        k, v, ks, vs = (None if x is None else npy(x[own]) for x in c.pages + c.scales)
        ref, lref, size, terms = O.sdpa_paged(npy(q[b:b + 1]), k, v, [np.arange(len(own))], lens[b:b + 1], ks, vs)
        close_out(out[b:b + 1], ref, size, terms, q.shape[-1], False)
        close_lse(lse[b:b + 1], lref, terms, q.shape[-1])


@pytest.mark.parametrize("kind", KINDS)
def test_sdpa_paged_over_turns_of_page_numbers(cuda, kind):
    # the numbers of 32 turns (4096 slots) of a work-group are fetched at once: 70 sequences' heads leave one split
    c = Cache(cuda, BF, kind, 70, 4, 64, 16, 536, seed=4)
    g = np.random.default_rng(0)
    lens = [int(x) for x in g.integers(1, 200, 70)]
    lens[0], lens[1], lens[69] = 8561, 4096, 4129
    some_of(c, gen((70, 4, 1, 64), BF, 1), lens, (0, 1, 5, 69))


# From 16 tiles of 32 slots a work-group on (256 of them over the 16-row groups) the tiles of all
# sequences and KV heads are one list: pieces end anywhere in a sequence, units of one tile and
# empty sequences lie between others.
EVEN = [  # n, hq, hkv, l, hd, page, lens, checked
    (9, 8, 8, 1, 64, 64, (3200, 0, 1, 3199, 2377, 33, 2800, 3200, 2900), (0, 1, 2, 3, 4, 5, 8)),
    (2, 16, 16, 1, 128, 48, (6000, 5000), (0, 1)),
    (1, 20, 1, 2, 64, 16, (50000,), (0,)),                          # three row groups of 40 rows
    (130, 2, 2, 1, 64, 32, tuple(700 - 3 * (b % 90) for b in range(130)), (0, 1, 63, 64, 65, 127, 128, 129)),    # past 64 sequences
    (70, 8, 8, 1, 64, 16, tuple(1300 - b * (b % 3) for b in range(70)), (0, 2, 40, 64, 69)),                     # two units a work-group and more
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,hq,hkv,l,hd,page,lens,checked", EVEN)
def test_sdpa_paged_even_pieces(cuda, n, hq, hkv, l, hd, page, lens, checked, kind):
    row_groups = -(-(hq // hkv * l) // 16)
    tiles = hkv * sum(max(1, -(-x // 32)) for x in lens)
    assert tiles >= (16 if n * hkv < 512 // row_groups else 64) * (256 // row_groups)
    c = Cache(cuda, BF, kind, n, hkv, hd, page, -(-max(lens) // page), seed=31)
    some_of(c, gen((n, hq, l, hd), BF, 1), lens, checked)


def longest_piece(lens, hkv, row_groups):
    """Tiles of 32 slots of the longest piece that a work-group has, for lengths that make one list
    of all tiles (a unit, a sequence's KV head, begins with 12 places that no tile has)."""
    groups, switch = max(1, 256 // row_groups), 12
    tiles = [max(1, -(-x // 32)) for x in lens for _ in range(hkv)]
    assert sum(tiles) >= (16 if len(tiles) < 2 * groups else 64) * groups
    per = max(switch + 16, int((sum(tiles) + len(tiles) * switch) / groups) + 1)
    best, at = 0, 0
    for t in tiles:
        first, end = at + switch, at + switch + t
        best = max([best] + [min(end, (w + 1) * per) - max(first, w * per) for w in range(first // per, (end - 1) // per + 1)])
        at = end
    return best


# A wave takes every fourth tile of a piece; where its tiles lie is fetched for 32 of them at a time,
# so a piece of 128 tiles and more goes on to the next 32 (many rows a KV head leave few work-groups
# for the tiles, so long pieces need no large cache)
TURNS = [  # n, hq, hkv, l, hd, page, lens
    (1, 16, 1, 129, 64, 16, (9000,)),                       # one work-group a row group: 282 tiles
    (3, 16, 1, 64, 64, 48, (9000, 3, 9001)),                # four: pieces that end anywhere, and another behind them
    (2, 16, 2, 129, 128, 32, (4097, 4480)),                 # three: two units of 129 tiles and two of 140
]


def rows_of(q, lens, first, count):
    """(the queries first .. first + count - 1, the lengths with which they are the last ones)"""
    return q[:, :, first:first + count], [L - q.shape[2] + first + count for L in lens]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,hq,hkv,l,hd,page,lens", TURNS)
def test_sdpa_paged_goes_on_to_more_page_numbers(cuda, n, hq, hkv, l, hd, page, lens, kind):
    assert longest_piece(lens, hkv, -(-(hq // hkv * l) // 16)) > 128
    c = Cache(cuda, BF, kind, n, hkv, hd, page, -(-max(lens) // page), seed=46)
    q = gen((n, hq, l, hd), BF, 1)
    out, lse = ops.sdpa_paged(q.to(cuda), **c.args(), kv_len=ints(lens, cuda), return_lse=True)
    for first in (0, l - 2):
        some, ends = rows_of(q, lens, first, 2)
        ref, lref, size, terms = c.attention(some, ends)
        close_out(out[:, :, first:first + 2], ref, size, terms, hd, False)
        close_lse(lse[:, :, first:first + 2], lref, terms, hd)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,hq,hkv,l,hd,page,lens", TURNS)
def test_masked_nan_behind_more_page_numbers(cuda, n, hq, hkv, l, hd, page, lens, kind):
    # the newest slot of each sequence holds a NaN: the wave that has it goes over all its tiles again
    # for the queries that do not see it
    c = Cache(cuda, BF, kind, n, hkv, hd, page, -(-max(lens) // page), seed=47)
    q = gen((n, hq, l, hd), BF, 1)
    some, ends = rows_of(q, lens, l - 3, 2)
    ref, lref, size, terms = c.attention(some, ends)
    for b, L in enumerate(lens):
        p, r = O.paged_slot(c.table[b], page, c.pages[1].shape[0], L - 1)
        if kind == "same":
            c.pages[1][p, :, r] = NAN
        else:
            c.scales[1][p, :, r] = NAN
    out, lse = ops.sdpa_paged(q.to(cuda), **c.args(), kv_len=ints(lens, cuda), return_lse=True)
    close_out(out[:, :, l - 3:l - 1], ref, size, terms, hd, False)
    close_lse(lse[:, :, l - 3:l - 1], lref, terms, hd)
    assert torch.isnan(out[:, :, l - 1]).all() and torch.isfinite(out[:, :, :l - 1]).all()


def test_large_pools_pass_by_the_caches(cuda):
    # (pools of 120 MB and more are read with other loads)
    for kind, dtype, hd, n in (("same", BF, 128, 8), ("int8", HF, 64, 32), ("e4m3", BF, 128, 16), ("same", HF, 64, 16)):
        page, width, hkv = 64, 66 if n < 32 else 62, 8
        lens = [width * page - 31 * b for b in range(n)]
        bytes_ = 2 * n * width * page * hkv * hd * (2 if kind == "same" else 1)
        c = Cache(cuda, dtype, kind, n, hkv, hd, page, width, seed=32)
        assert bytes_ >= 120 << 20
        some_of(c, gen((n, hkv, 1, hd), dtype, 1), lens, (0, n - 1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_absent_pages_are_not_seen(cuda, dtype, kind):
    c = Cache(cuda, dtype, kind, 4, 2, 64, 16, 40, seed=5)
    P = c.pages[0].shape[0]
    c.table[0, [0, 3, 4, 17, 30]] = (-1, P, 2 ** 31 - 1, -2 ** 31, -7)
    c.table[1, :] = -1                                     # none at all
    c.table[2, 38:] = P + 5                                # the last ones: the queries do not see themselves
    c.table[3, 1:] = -1
    attends(c, gen((4, 4, 2, 64), dtype, 2), (600, 640, 635, 500))


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_that_share_pages(cuda, kind):
    # a prefix in pages that all tables name, and one page over and over
    c = Cache(cuda, HF, kind, 5, 2, 128, 32, 40, seed=43)
    c.table[:, :30] = c.table[0, :30]
    c.table[4] = 7
    lens = (1000, 1280, 961, 5, 1279)
    attends(c, gen((5, 8, 2, 128), HF, 2), lens)
    k, v = ops.kv_paged_read(**c.args(), kv_len=ints(lens, cuda))
    assert torch.equal(k[0, :, :960], k[2, :, :960]) and torch.equal(v[4, :, :32], v[4, :, 1216:1248])


def test_more_rows_than_work_groups(cuda):
    # 300 groups of 16 rows: each has the whole sequence
    c = Cache(cuda, BF, "same", 1, 1, 64, 16, 50, seed=44)
    attends(c, gen((1, 16, 300, 64), BF, 2), (777,))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width,l", [(3, 4), (3, 20), (200, 5)])
def test_drafted_tokens_that_pass_the_table(cuda, width, l, kind):
    # the queries of slots that the table has keep them, whatever lies past its end
    end = 16 * width
    c = Cache(cuda, BF, kind, 6, 2, 64, 16, width, seed=41)
    attends(c, gen((6, 4, l, 64), BF, 2), (end, end + 1, end + 3, end + l, end + l + 7, 2 ** 31 - 1))
    attends(c, gen((6, 4, l, 64), BF, 3), (end + 2, 3, -1, end + 1, 0, -2 ** 31))


def test_lengths_outside_the_table(cuda):
    c = Cache(cuda, BF, "same", 4, 2, 64, 16, 3, seed=6)
    attends(c, gen((4, 4, 1, 64), BF, 2), (49, -1, 2 ** 31 - 1, -2 ** 31))
    # no table, no pages, no sequences
    q = gen((2, 4, 1, 64), BF).to(cuda)
    a = c.args()
    out, lse = ops.sdpa_paged(q, **{**a, "table": a["table"][:2, :0]}, kv_len=ints([5, 0], cuda), return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()
    empty = dict(k_pages=a["k_pages"][:0], v_pages=a["v_pages"][:0], table=a["table"][:2])
    out, lse = ops.sdpa_paged(q, **empty, kv_len=ints([40, 1], cuda), return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()
    k, v = ops.kv_paged_read(**empty, kv_len=ints([40, 1], cuda))
    assert k.shape == (2, 2, 48, 64) and not k.any() and not v.any()
    assert ops.sdpa_paged(q[:0], **{**a, "table": a["table"][:0]}, kv_len=ints([], cuda))[0].shape == (0, 4, 1, 64)
    assert ops.sdpa_paged(q[:, :, :0], **{**a, "table": a["table"][:2]}, kv_len=ints([5, 0], cuda))[0].shape == (2, 4, 0, 64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("l", [1, 3])
def test_what_is_not_seen_stays_out(cuda, kind, l):
    # NaN and infinities behind the sequences, in pages of nobody and behind pages' last rows
    lens = (601, 130)
    c = Cache(cuda, BF, kind, 2, 2, 128, 32, 20, seed=7, spare=5)
    q = gen((2, 8, l, 128), BF, 1)
    plain = ops.sdpa_paged(q.to(cuda), **c.args(), kv_len=ints(lens, cuda), return_lse=True)
    used = np.zeros((c.pages[0].shape[0], 32), bool)
    for b, L in enumerate(lens):
        for s in range(L):
            used[O.paged_slot(c.table[b], 32, used.shape[0], s)] = True
    where = torch.from_numpy(~used).to(cuda)[:, None].expand(-1, 2, -1)
    for i in range(2):
        if kind == "same":
            c.pages[i][where] = (math.inf, NAN)[i]
        else:
            c.scales[i][where] = (NAN, math.inf)[i]
            c.pages[i].view(torch.uint8)[where] = 0x7f
    spoilt = ops.sdpa_paged(q.to(cuda), **c.args(), kv_len=ints(lens, cuda), return_lse=True)
    assert torch.equal(plain[0], spoilt[0]) and torch.equal(plain[1], spoilt[1])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_infinite_and_nan_values(cuda, dtype):
    lens = (700, 65)
    c = Cache(cuda, dtype, "same", 2, 1, 64, 16, 44, seed=8)
    v = c.pages[1]

    def at(b, slot):
        return O.paged_slot(c.table[b], 16, v.shape[0], slot)
    p, r = at(0, 300)
    v[p, 0, r, 5] = math.inf                    # seen by all queries
    p, r = at(0, 699)
    v[p, 0, r, 7] = -math.inf                   # by the last query alone
    v[p, 0, r, 9] = NAN
    p, r = at(1, 3)
    c.pages[0][p, 0, r, 0] = NAN                # a key
    q = gen((2, 4, 2, 64), dtype, 1)
    out, lse = ops.sdpa_paged(q.to(cuda), **c.args(), kv_len=ints(lens, cuda), return_lse=True)
    ref, lref, size, terms = c.attention(q, lens)
    out, ref = npy(out), ref
    assert np.isposinf(out[0, :, :, 5]).all() and np.isneginf(out[0, :, 1, 7]).all() and np.isnan(out[0, :, 1, 9]).all()
    assert np.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    fine = np.isfinite(ref)
    fine[1] = False
    assert np.isfinite(out[0][fine[0]]).all() and fine[0].sum() == 4 * 2 * 64 - 4 * (2 + 2)
    terms = 64 * 20                             # (above any |q k| here: gaussians)
    u = torch.finfo(dtype).eps / 2
    tol = u * np.abs(ref) + 2.0 ** -12 * size + 2.0 ** -25
    assert (np.abs(out - ref)[fine] <= tol[fine]).all()


def test_a_nan_row_of_8_bit_pages_reads_as_nan(cuda):
    for kind in ("int8", "e4m3"):
        c = Cache(cuda, BF, kind, 1, 1, 64, 16, 4, seed=9)
        p, r = O.paged_slot(c.table[0], 16, 6, 20)
        c.scales[1][p, 0, r] = NAN
        q = gen((1, 2, 1, 64), BF, 1).to(cuda)
        out, lse = ops.sdpa_paged(q, **c.args(), kv_len=ints([30], cuda), return_lse=True)
        assert torch.isnan(out).all() and torch.isfinite(lse).all()
        assert torch.isfinite(ops.sdpa_paged(q, **c.args(), kv_len=ints([20], cuda))[0]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_layouts(cuda, kind):
    # keys and values in one buffer, pages token by token, tables in a wider one, a query and an output of other strides
    n, hq, hkv, l, hd, page, lens = 2, 6, 3, 2, 64, 16, (77, 40)
    c = Cache(cuda, HF, kind, n, hkv, hd, page, 5, seed=11)
    q = gen((n, hq, l, hd), HF, 1)
    want = ops.sdpa_paged(q.to(cuda), **c.args(), kv_len=ints(lens, cuda), return_lse=True)
    P = c.pages[0].shape[0]
    both = torch.zeros(P, 2, page, hkv, 2 * hd, device=cuda, dtype=c.pages[0].dtype)
    a = c.args()
    wide = torch.full((n, 9), -1, dtype=torch.int32, device=cuda)
    wide[:, 2:7] = a["table"]
    a["table"] = wide[:, 2:7]
    for i, name in enumerate(("k_pages", "v_pages")):
        view = both[:, i].transpose(1, 2)[..., :hd]
        view.copy_(a[name])
        a[name] = view
    if kind != "same":
        scales = torch.zeros(2, P, hkv + 1, page, device=cuda)
        for i, name in enumerate(("k_scale", "v_scale")):
            scales[i, :, 1:] = a[name]
            a[name] = scales[i, :, 1:]
    queries = [q.to(cuda).transpose(1, 2).contiguous().transpose(1, 2), torch.cat([q, q], -1).to(cuda)[..., :hd]]
    odd = torch.zeros(n, hq, l, hd + 1, dtype=HF, device=cuda)
    odd[..., 1:] = q.to(cuda)
    queries.append(odd[..., 1:])                           # rows that start anywhere
    for x in queries:
        big = torch.full((n, l, hq, hd + 8), 3.0, dtype=HF, device=cuda)
        out = big[..., :hd].transpose(1, 2)
        got = ops.sdpa_paged(x, **a, kv_len=ints(lens, cuda), return_lse=True, out=out)
        assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1]) and (big[..., hd:] == 3).all()
    k, v = ops.kv_paged_read(**a, kv_len=ints(lens, cuda), dtype=HF)
    k2, v2 = ops.kv_paged_read(**c.args(), kv_len=ints(lens, cuda), dtype=HF)
    assert torch.equal(k, k2) and torch.equal(v, v2)


def test_scale_and_large_scores(cuda):
    c = Cache(cuda, BF, "same", 1, 2, 64, 16, 40, seed=12)
    attends(c, gen((1, 4, 1, 64), BF, 1), (640,), scale=0.5)
    attends(c, gen((1, 4, 1, 64), BF, 1, std=30.0), (640,))        # one key takes nearly all
    # rising scores: the running maximum moves in every tile
    (k, _), _ = c.numbers()
    for s in range(640):
        p, r = O.paged_slot(c.table[0], 16, k.shape[0], s)
        c.pages[0][p, :, r] = s / 64
    attends(c, torch.ones(1, 4, 1, 64, dtype=BF), (640,))


def test_pools_past_32_bits(cuda):
    # 4.6e9 bytes of keys, and as many of values: the last pages
    P = 70000
    k, v = (torch.empty(P, 8, 64, 128, dtype=I8, device=cuda) for _ in range(2))
    ks, vs = (torch.ones(P, 8, 64, device=cuda) for _ in range(2))
    table = np.array([[P - 1, P - 4, P - 2]], np.int32)
    for i, x in enumerate((k, v)):
        x[P - 4:] = torch.randint(-127, 128, (4, 8, 64, 128), generator=torch.Generator().manual_seed(i)).to(I8).to(cuda)
    scale = 0.02 / math.sqrt(128)
    q = gen((1, 16, 1, 128), BF, 1)
    a = dict(k_pages=k, v_pages=v, table=torch.from_numpy(table).to(cuda), k_scale=ks, v_scale=vs)
    out, lse = ops.sdpa_paged(q.to(cuda), **a, kv_len=ints([170], cuda), scale=scale, return_lse=True)
    ref, lref, size, terms = O.sdpa_paged(npy(q), npy(k[P - 4:]), npy(v[P - 4:]), table - (P - 4), [170], scale=scale)
    close_out(out, ref, size, terms, 128, False)
    close_lse(lse, lref, terms, 128)
    got, _ = ops.kv_paged_read(**a, kv_len=ints([170], cuda), length=170)
    want, _ = O.paged_rows(npy(k[P - 4:]), None, table - (P - 4), 170)
    np.testing.assert_array_equal(npy(got), want)
    qkv = gen((1, 3, 32 * 128), BF, 2).to(cuda)
    ops.kv_paged_append(qkv, torch.ones(64, device=cuda), ints([166], cuda), **a)
    np.testing.assert_array_equal(npy(v[P - 2, :, 38:41]), O.quantise_rows(npy(qkv[0].view(3, 32, 128)[:, 24:].transpose(0, 1)), "int8")[0])


def test_the_same_bits_every_time(cuda):
    c = Cache(cuda, BF, "e4m3", 2, 4, 128, 16, 300, seed=13)
    q, lens = gen((2, 16, 1, 128), BF, 1).to(cuda), ints([4700, 3000], cuda)
    first = ops.sdpa_paged(q, **c.args(), kv_len=lens, return_lse=True)
    for _ in range(20):
        again = ops.sdpa_paged(q, **c.args(), kv_len=lens, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_a_workspace_serves_calls_of_all_sizes(cuda):
    # one stream's workspace: what a call leaves is no other's counter
    small, large = Cache(cuda, BF, "same", 1, 1, 64, 16, 20, seed=14), Cache(cuda, BF, "same", 3, 8, 128, 16, 200, seed=15)
    for lens in ((3200, 900, 128), (129, 3000, 2000)):
        attends(small, gen((1, 16, 1, 64), BF, 1), (300,))
        attends(large, gen((3, 8, 1, 128), BF, 2), lens)
    attends(small, gen((1, 3, 1, 64), BF, 1), (310,))


def test_streams_and_graphs(cuda):
    c, d = (Cache(cuda, BF, kind, 2, 2, 64, 16, 130, seed=16) for kind in ("same", "int8"))
    q, lens = gen((2, 8, 1, 64), BF, 1).to(cuda), ints([2000, 700], cuda)
    a, b = c.args(), d.args()

    def both():
        return ops.sdpa_paged(q, **a, kv_len=lens)[0], ops.sdpa_paged(q, **b, kv_len=lens)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = both()
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, both()))
    for step in range(4):
        lens.copy_(ints([2000 - 321 * step, 700 + 400 * step], cuda))
        q.mul_(0.9)
        want = both()
        torch.cuda.synchronize()
        # two graphs of the same calls at the same time
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(x, y) for x, y in zip(want, got)), step


# ------------------------------------------------------------------ append

def heads_of(qkv, hq, hkv, hd):
    x = npy(qkv).reshape(*qkv.shape[:2], hq + 2 * hkv, hd)
    return x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:]


def rotated_tolerance(ref, terms, dtype, hd):
    u = torch.finfo(dtype).eps / 2
    return u * np.abs(ref) * 1.001 + (hd * 2.0 ** -26 + 2.0 ** -20) * terms + (2.0 ** -25 if dtype == HF else 0)


def appends(c, qkv, hq, hkv, hd, freq, pos0, lens=None, wq=None, wk=None, eps=1e-6, **kw):
    """Calls kv_paged_append and checks q and every row of the pool."""
    dev, dtype = c.device, qkv.dtype
    n, t, _ = qkv.shape
    before = [p.clone() for p in c.pages], [None if s is None else s.clone() for s in c.scales]
    q = ops.kv_paged_append(qkv if qkv.is_cuda else qkv.to(dev), freq.to(dev), None if pos0 is None else ints(pos0, dev), **c.args(),
                            lens=None if lens is None else ints(lens, dev), q_norm=None if wq is None else wq.to(dev),
                            k_norm=None if wk is None else wk.to(dev), eps=eps, **kw)
    got = npy(q)
    xq, xk, xv = heads_of(qkv, hq, hkv, hd)
    pages, scales = [npy(p) for p in c.pages], [None if s is None else npy(s) for s in c.scales]
    want = [npy(p) for p in before[0]], [None if s is None else npy(s) for s in before[1]]
    P, page = c.pages[0].shape[0], c.pages[0].shape[2]
    for b in range(n):
        for i in range(t):
            if lens is not None and i >= lens[b]:
                assert not got[b, :, i].any()
                continue
            pos = (0 if pos0 is None else pos0[b]) + i
            ref, terms = O.norm_rope(xq[b, i], None if wq is None else npy(wq), eps, pos, freq.double().numpy())
            err = np.abs(got[b, :, i] - ref) - rotated_tolerance(ref, terms, dtype, hd)
            assert (err <= 0).all(), f"token {b}, {i}: {err.max():.3e}"
            at = O.paged_slot(c.table[b], page, P, pos)
            if at is None:
                continue
            ref, terms = O.norm_rope(xk[b, i], None if wk is None else npy(wk), eps, pos, freq.double().numpy())
            for x, rows, S in ((0, ref, terms), (1, xv[b, i], None)):
                where = (at[0], slice(None), at[1])
                if c.kind == "same":
                    if x:
                        np.testing.assert_array_equal(pages[1][where], rows)
                    else:
                        assert (np.abs(pages[0][where] - rows) <= rotated_tolerance(rows, S, dtype, hd)).all()
                    want[0][x][where] = pages[x][where]
                else:
                    stored, scale, off = O.quantise_rows(rows, c.kind)
                    near = off < 2.0 ** -30
                    assert ((pages[x][where] == stored) | near).all()
                    assert near.sum() <= 2 or x                   # (values' ties are exact, and go to even)
                    if x:
                        np.testing.assert_array_equal(pages[x][where], stored)
                    # one rounding of 64 bits
                    ok = np.isnan(scale) & np.isnan(scales[x][where]) | (np.abs(scales[x][where] - scale) <= 2.0 ** -23 * scale)
                    assert ok.all()
                    want[0][x][where], want[1][x][where] = pages[x][where], scales[x][where]
    for x in range(2):          # nothing else was written
        np.testing.assert_array_equal(pages[x], want[0][x])
        if scales[x] is not None:
            np.testing.assert_array_equal(scales[x], want[1][x])
    return q


def frequencies(hd, base=10000.0):
    return (base ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float()


APPENDS = [  # n, t, hq, hkv, hd, page, width, pos0, lens, norm
    (1, 1, 32, 8, 64, 16, 4, (37,), None, False),
    (3, 1, 4, 2, 128, 32, 3, (0, 31, 95), None, True),             # first slot, a page's last, the table's last
    (2, 5, 4, 2, 64, 16, 3, (45, -2), None, True),                 # slots past the table and before the first are dropped
    (2, 19, 14, 2, 64, 48, 2, (3, 0), (19, 7), False),             # ragged
    (2, 3, 6, 3, 96, 16, 2, None, (0, 5), True),                   # nothing there; more than t is t
    (1, 4, 2, 1, 16, 16, 2, (1,), None, True),
    (2, 2, 3, 1, 112, 16, 2, (1, 17), None, False),
    (1, 2, 0, 2, 64, 16, 2, (4,), None, False),                    # no queries
    (2, 700, 2, 1, 128, 64, 12, (5, 60), (700, 501), True),        # a work-group per 4 tokens
    (1, 1030, 3, 1, 64, 16, 65, (7,), (1027,), False),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,t,hq,hkv,hd,page,width,pos0,lens,norm", APPENDS)
def test_kv_paged_append(cuda, n, t, hq, hkv, hd, page, width, pos0, lens, norm, dtype, kind):
    c = Cache(cuda, dtype, kind, n, hkv, hd, page, width, seed=20)
    qkv = gen((n, t, (hq + 2 * hkv) * hd), dtype, 1)
    w = [(1 + gen((hd,), torch.float32, 2 + i, 0.3)).to(dtype) if norm else None for i in range(2)]
    appends(c, qkv, hq, hkv, hd, frequencies(hd), pos0, lens, *w)


@pytest.mark.parametrize("kind", KINDS)
def test_append_far_positions(cuda, kind):
    # angles up to 8.4e6: 64 bits (slots past the table: q alone), and rows at 65536 through one page
    c = Cache(cuda, HF, kind, 2, 1, 64, 16384, 5, seed=21, spare=0)
    c.table[:, :4] = -1
    qkv = gen((2, 3, 4 * 64), HF, 1)
    appends(c, qkv, 2, 1, 64, torch.ones(32) * 1.0078125, (65534, 8388600))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_of_rows_that_are_zero_tiny_or_not_finite(cuda, kind):
    c = Cache(cuda, BF, kind, 1, 1, 64, 16, 1, seed=22)
    qkv = gen((1, 6, 3 * 64), BF, 1)
    qkv[0, 0] = 0
    qkv[0, 1] *= 2.0 ** -120
    qkv[0, 2] *= 2.0 ** 115
    qkv[0, 3, 64 + 5] = NAN                # a key
    qkv[0, 4, 128 + 63] = -math.inf        # a value
    freq = torch.zeros(32)                 # no turn: keys are exact
    ops.kv_paged_append(qkv.to(cuda), freq.to(cuda), None, **c.args())
    k, v = ops.kv_paged_read(**c.args(), kv_len=ints([6], cuda), length=6, dtype=torch.float32)
    x = npy(qkv)[0].reshape(6, 3, 64)
    for row, got in ((1, npy(k)[0, 0]), (2, npy(v)[0, 0])):
        stored, scale, _ = O.quantise_rows(x[:, row], kind)
        ref = stored * scale[:, None]
        assert (np.isnan(got) == np.isnan(ref)).all()
        fine = np.isfinite(scale)
        # the scale's rounding and the product's; 2^-120's rows have scales near 2^-127, below fp32's normal ones
        assert (np.abs(got - ref)[fine] <= 2.0 ** -22 * np.abs(ref[fine]) + 448 * 2.0 ** -149).all()
    assert torch.isnan(k[0, 0, 3]).all() and torch.isnan(v[0, 0, 4]).all()
    assert torch.isfinite(k[0, 0, [0, 1, 2, 4, 5]]).all() and torch.isfinite(v[0, 0, [0, 1, 2, 3, 5]]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6, 1e12])
def test_append_norms_rows_of_any_size(cuda, eps, hd, kind):
    # squares past fp32's range on both sides, rows of different sizes in one wave
    c = Cache(cuda, BF, kind, 1, 2, hd, 16, 1, seed=26)
    sizes = (-75, -70, -64, -40, 0, 50, 62, 64, 70, 115)
    qkv = gen((1, len(sizes), 7 * hd), BF, 1) * 2.0 ** torch.tensor(sizes, dtype=torch.float32).to(BF)[:, None]
    qkv[0, :, hd:2 * hd] = gen((len(sizes), hd), BF, 4)          # one head of each as it mostly is
    w = [(1 + gen((hd,), torch.float32, 2 + i, 0.3)).to(BF) for i in range(2)]
    appends(c, qkv, 3, 2, hd, frequencies(hd), (3,), None, *w, eps=eps)


def test_append_norms_the_smallest_and_largest(cuda, monkeypatch):
    # bf16's denormals; an eps past fp32's range beside large rows.  Below 2^-126 bf16's step is 2^-126 2^-7
    # whatever the value, so that half a step, what a rounding is off by, is 2^-134 there, not u |ref|.
    relative = rotated_tolerance
    monkeypatch.setitem(globals(), "rotated_tolerance", lambda *a: relative(*a) + 2.0 ** -134)
    c = Cache(cuda, BF, "same", 1, 1, 64, 16, 1, seed=27)
    w = torch.ones(64, dtype=BF)
    for size, eps in ((2.0 ** -128, 0.0), (2.0 ** -128, 1e-6), (2.0 ** 64, 1e40), (2.0 ** 110, 1e60)):
        appends(c, gen((1, 3, 3 * 64), BF, 1) * size, 1, 1, 64, frequencies(64), (3,), None, w, w, eps=eps)


def test_append_norms_of_rows_that_are_not_finite(cuda):
    # as the formula gives: a number over an infinite root is 0, an infinity over it NaN; with a NaN all are
    c = Cache(cuda, BF, "same", 1, 1, 64, 16, 1, seed=28)
    qkv = gen((1, 3, 3 * 64), BF, 1)
    for at in (0, 64):                      # the query, the key
        qkv[0, 0, at + 5], qkv[0, 1, at + 40] = math.inf, NAN
    w = torch.ones(64, dtype=BF, device=cuda)
    fine = ops.kv_paged_append(qkv[:, 2:].to(cuda), frequencies(64).to(cuda), ints([2], cuda), **c.args(), q_norm=w, k_norm=w)
    q = ops.kv_paged_append(qkv.to(cuda), frequencies(64).to(cuda), None, **c.args(), q_norm=w, k_norm=w)
    k = c.pages[0][int(c.table[0, 0]), 0, :3]
    for x in (q[0, 0], k):
        assert torch.isnan(x[0, [5, 37]]).all() and x[0].isnan().sum() == 2 and (x[0, [*range(5), *range(6, 37), *range(38, 64)]] == 0).all()
        assert torch.isnan(x[1]).all() and torch.isfinite(x[2]).all()
    assert torch.equal(q[:, :, 2:], fine)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_norms_of_rows_that_are_not_finite_in_8_bits(cuda, kind):
    c = Cache(cuda, BF, kind, 1, 1, 128, 16, 1, seed=29)
    qkv = gen((1, 4, 3 * 128), BF, 1)
    for at in (0, 128):                     # the query, the key
        qkv[0, 0, at + 5], qkv[0, 1, at + 70] = -math.inf, NAN
        qkv[0, 2, at:at + 128] *= 2.0 ** 100
    w, freq = torch.ones(128, dtype=BF, device=cuda), frequencies(128).to(cuda)
    q = ops.kv_paged_append(qkv.to(cuda), freq, None, **c.args(), q_norm=w, k_norm=w)
    k, v = ops.kv_paged_read(**c.args(), kv_len=ints([4], cuda), length=4)
    assert torch.isnan(k[0, 0, :2]).all() and torch.isfinite(k[0, 0, 2:]).all() and torch.isfinite(v).all()
    assert torch.isnan(q[0, 0, 0, [5, 69]]).all() and q[0, 0, 0].isnan().sum() == 2 and torch.isnan(q[0, 0, 1]).all()
    # a normed row's mean square is 1: values off by 2^-4 (e4m3) and less, their squares by (1 + 2^-4)^2 - 1 < 0.13
    for x in (q[0, 0, 2:], k[0, 0, 2:]):
        assert ((x.float().square().mean(-1) - 1).abs() < 0.13).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_ties_go_to_even(cuda, kind):
    # values at every border of the type (x / 2 of its largest and so on): exact in bf16
    c = Cache(cuda, BF, kind, 1, 1, 128, 16, 1, seed=23)
    x = torch.zeros(1, 2, 3 * 128, dtype=BF)
    M = 127 if kind == "int8" else 448
    x[0, :, 256] = M
    x[0, 0, 257:] = torch.arange(127) + 0.5 if kind == "int8" else torch.arange(127) / 16 + 2
    x[0, 1, 257:] = -(torch.arange(127) + 0.5) if kind == "int8" else torch.arange(127) * 2.0 ** -11
    x[0, :, 128:256] = x[0, :, 256:]
    ops.kv_paged_append(x.to(cuda), torch.zeros(64, device=cuda), None, **c.args())
    stored, scale, _ = O.quantise_rows(npy(x)[0, :, 256:], kind)
    assert (scale == 1).all()
    for pages, scales in zip(c.pages, c.scales):
        np.testing.assert_array_equal(npy(pages)[c.table[0, 0], 0, :2], stored)
        assert (npy(scales)[c.table[0, 0], 0, :2] == 1).all()


def test_append_layouts(cuda):
    n, t, hq, hkv, hd = 2, 3, 4, 2, 64
    qkv = gen((n, t, (hq + 2 * hkv) * hd), BF, 1)
    freq = frequencies(hd)
    c = Cache(cuda, BF, "int8", n, hkv, hd, 16, 3, seed=24)
    wide = torch.zeros(t, n, (hq + 2 * hkv) * hd + 8, dtype=BF, device=cuda)
    wide[..., :-8] = qkv.to(cuda).transpose(0, 1)
    q_out = torch.full((n, t, hq, hd + 8), 5.0, dtype=BF, device=cuda)
    view = q_out[..., :hd].transpose(1, 2)
    q = appends(c, wide[..., :-8].transpose(0, 1), hq, hkv, hd, freq, (3, 40), q_out=view)
    assert q is view and (q_out[..., hd:] == 5).all()
    # rows that start anywhere
    odd = torch.zeros(n, t, (hq + 2 * hkv) * hd + 1, dtype=BF, device=cuda)
    odd[..., 1:] = qkv.to(cuda)
    d = Cache(cuda, BF, "int8", n, hkv, hd, 16, 3, seed=24)
    assert torch.equal(appends(d, odd[..., 1:], hq, hkv, hd, freq, (3, 40)), q)


def test_pieces_of_a_prompt_are_the_prompt(cuda):
    for kind in KINDS:
        c, d = (Cache(cuda, BF, kind, 1, 2, 64, 32, 42, seed=25) for _ in range(2))
        qkv, freq = gen((1, 1300, 6 * 64), BF, 1).to(cuda), frequencies(64).to(cuda)
        w = (1 + gen((64,), torch.float32, 2, 0.3)).to(BF).to(cuda)
        whole = ops.kv_paged_append(qkv, freq, None, **c.args(), q_norm=w, k_norm=w)
        parts, at = [], 0
        for m in (1, 700, 33, 1, 565):
            parts.append(ops.kv_paged_append(qkv[:, at:at + m], freq, ints([at], cuda), **d.args(), q_norm=w, k_norm=w))
            at += m
        assert torch.equal(whole, torch.cat(parts, 2))
        for x, y in zip(c.pages + c.scales, d.pages + d.scales):
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# -------------------------------------------------------------------- read

READS = [  # n, hkv, hd, page, width, lens, length
    (1, 2, 64, 16, 4, (1,), None),
    (3, 2, 128, 32, 9, (33, 0, 288), None),
    (2, 8, 64, 48, 7, (300, 129), 200),              # cut off
    (2, 1, 96, 16, 3, (48, 5), 100),                 # longer than the table
    (1, 3, 16, 16, 20, (317,), 317),
    (2, 2, 48, 64, 3, (-4, 2 ** 31 - 1), None),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("n,hkv,hd,page,width,lens,length", READS)
def test_kv_paged_read(cuda, n, hkv, hd, page, width, lens, length, dtype, kind):
    if kind == "same" and dtype == torch.float32:
        return          # (16-bit pages come as they are)
    c = Cache(cuda, BF if dtype == torch.float32 else dtype, kind, n, hkv, hd, page, width, seed=30)
    c.table[0, width // 2] = -1
    rows = width * page if length is None else length
    a = c.args()
    got = ops.kv_paged_read(**a, kv_len=ints(lens, cuda), length=length, dtype=dtype)
    outs = [torch.full((n, rows, hkv, hd + 8), 7.0, dtype=dtype, device=cuda) for _ in range(2)]
    views = [o[..., :hd].transpose(1, 2) for o in outs]
    assert ops.kv_paged_read(**a, kv_len=ints(lens, cuda), k_out=views[0], v_out=views[1])[0] is views[0]
    P = c.pages[0].shape[0]
    for x in range(2):
        assert got[x].shape == (n, hkv, rows, hd) and got[x].dtype == dtype
        numbers = c.pages[x].float() * c.scales[x][..., None] if kind != "same" else c.pages[x]
        numbers = numbers.to(dtype)
        for b in range(n):
            for s in range(rows):
                at = O.paged_slot(c.table[b], page, P, s) if s < lens[b] else None
                want = 0 if at is None else numbers[at[0], :, at[1]]
                assert (got[x][b, :, s] == want).all(), (x, b, s)
        end = [min(max(m, 0), width * page, rows) for m in lens]
        for b in range(n):
            assert torch.equal(views[x][b, :, :end[b]], got[x][b, :, :end[b]]) and (views[x][b, :, end[b]:] == 7).all()
        assert (outs[x][..., hd:] == 7).all()


# ---------------------------------------------------------- used together

@pytest.mark.parametrize("kind", KINDS)
def test_a_server_of_three_sequences(cuda, kind):
    """Prompts in pieces, then decoding in a graph: every step's attention is that over what
    the cache holds, and 16-bit pages give what a contiguous cache does."""
    n, hq, hkv, hd, page, width = 3, 8, 2, 64, 16, 12
    c = Cache(cuda, BF, kind, n, hkv, hd, page, width, seed=40)
    a, freq = c.args(), frequencies(hd).to(cuda)
    w = (1 + gen((hd,), torch.float32, 2, 0.3)).to(BF).to(cuda)
    prompt, lens = gen((n, 90, (hq + 2 * hkv) * hd), BF, 1).to(cuda), ints([90, 17, 64], cuda)
    q = ops.kv_paged_append(prompt, freq, None, **a, q_norm=w, k_norm=w, lens=lens)
    k, v = ops.kv_paged_read(**a, kv_len=lens, length=90)
    first = [ops.sdpa_decode_accum(q[b:b + 1, :, :m], k[b:b + 1, :, :m], v[b:b + 1, :, :m], torch.zeros(1, hkv, m, device=cuda))[0]
             for b, m in enumerate((90, 17, 64))]
    for b, m in enumerate((90, 17, 64)):
        ref, _, _, size, terms = O.sdpa_decode_accum(npy(q[b:b + 1, :, :m]), npy(k[b:b + 1, :, :m]), npy(v[b:b + 1, :, :m]), np.zeros((1, hkv, m)))
        close_out(first[b], ref, size, terms, hd, False)
    # decoding: append, attend, count, as one graph
    x = torch.zeros(n, 1, (hq + 2 * hkv) * hd, dtype=BF, device=cuda)
    pos, ends = lens.clone(), lens + 1
    tokens = gen((20, n, 1, (hq + 2 * hkv) * hd), BF, 3).to(cuda)

    def step():
        q = ops.kv_paged_append(x, freq, pos, **a, q_norm=w, k_norm=w)
        out, lse = ops.sdpa_paged(q, **a, kv_len=ends, return_lse=True)
        pos.add_(1)
        ends.add_(1)
        return q, out, lse
    graph = None
    for i in range(20):
        x.copy_(tokens[i])
        if i == 0:
            q, out, lse = step()
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    q, out, lse = step()
            graph.replay()
        if i in (0, 1, 2, 19):
            torch.cuda.synchronize()
            now = [90 + i + 1, 17 + i + 1, 64 + i + 1]
            ref, lref, size, terms = c.attention(q, now)
            close_out(out, ref, size, terms, hd, False)
            close_lse(lse, lref, terms, hd)
            if kind == "same":
                k, v = ops.kv_paged_read(**a, kv_len=ints(now, cuda))
                flat, _ = ops.sdpa_decode(q, k, v, kv_len=ints(now, cuda))
                close_out(flat, ref, size, terms, hd, False)
    assert pos.tolist() == [110, 37, 84]


@pytest.mark.parametrize("kind", KINDS)
def test_drafted_tokens_of_a_padded_batch(cuda, kind):
    """Fewer drafted tokens than others have: with kv_len = pos0 + t each token sees what it
    sees alone, whatever lies in the slots of the padding (or past the table's end)."""
    n, t, hq, hkv, hd, page, width = 5, 4, 8, 2, 64, 16, 6
    pos0, lens = (90, 95, 0, 33, 92), (4, 1, 2, 0, 3)
    c = Cache(cuda, BF, kind, n, hkv, hd, page, width, seed=42)
    for b, (p, m) in enumerate(zip(pos0, lens)):        # not finite where the padding would be
        for s in range(p + m, min(p + t, page * width)):
            at = c.table[b, s // page], slice(None), s % page
            for x in (c.pages if kind == "same" else c.scales):
                x[at] = NAN
    a, freq = c.args(), frequencies(hd).to(cuda)
    qkv = gen((n, t, (hq + 2 * hkv) * hd), BF, 1).to(cuda)
    start = ints(pos0, cuda)
    q = ops.kv_paged_append(qkv, freq, start, **a, lens=ints(lens, cuda))
    out, lse = ops.sdpa_paged(q, **a, kv_len=start + t, return_lse=True)
    for b, m in enumerate(lens):
        if m:
            one = Cache.__new__(Cache)
            one.__dict__.update(c.__dict__, table=c.table[b:b + 1])
            ref, lref, size, terms = one.attention(q[b:b + 1, :, :m], [pos0[b] + m])
            close_out(out[b:b + 1, :, :m], ref, size, terms, hd, False)
            close_lse(lse[b:b + 1, :, :m], lref, terms, hd)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t,hd", [(24, 64), (130, 128)])
def test_prompt_pieces_of_a_padded_batch(cuda, t, hd, dtype, kind):
    """Append, read back with kv_len = pos0 + lens and attend to the slots up to each token's, all
    sequences in one call: each token sees what it sees alone, whatever the pages hold behind it."""
    n, hq, hkv, page, width = 4, 8, 2, 16, 8 if t < 100 else 16
    pos0, lens = (0, 40, 7, 16 * width - 25), (t, 5, 0, min(t, 25))        # the last one's padding passes the table
    c = Cache(cuda, dtype, kind, n, hkv, hd, page, width, seed=45)
    for b, (p, m) in enumerate(zip(pos0, lens)):
        for s in range(p + m, min(p + t, page * width)):
            at = c.table[b, s // page], slice(None), s % page
            for x in (c.pages if kind == "same" else c.scales):
                x[at] = NAN
    a, freq = c.args(), frequencies(hd).to(cuda)
    qkv, w = gen((n, t, (hq + 2 * hkv) * hd), dtype, 1).to(cuda), (1 + gen((hd,), torch.float32, 2, 0.3)).to(dtype).to(cuda)
    start, there = ints(pos0, cuda), ints(lens, cuda)
    longest = max(pos0) + t
    q = ops.kv_paged_append(qkv, freq, start, **a, q_norm=w, k_norm=w, lens=there)
    k, v = ops.kv_paged_read(**a, kv_len=start + there, length=longest, dtype=dtype)
    acc = torch.zeros(n, hkv, longest, device=cuda)
    seen = torch.arange(longest, device=cuda) <= (start[:, None] + torch.arange(t, device=cuda))[:, :, None]
    mask = torch.where(seen, 0.0, -math.inf).to(dtype)[:, None]
    calls = [(True, ops.sdpa(q, k, v, bias=mask)), (False, ops.sdpa_decode(q, k, v, kv_len=start + t, return_lse=True)),
             (False, ops.sdpa_decode_accum(q, k, v, acc, start + t, return_lse=True))]
    for b, (p, m) in enumerate(zip(pos0, lens)):
        if m:
            kk, vv = npy(k[b:b + 1, :, :p + m]), npy(v[b:b + 1, :, :p + m])
            ref, lref, _, size, terms = O.sdpa_decode_accum(npy(q[b:b + 1, :, :m]), kk, vv, np.zeros((1, hkv, p + m)))
            for one_part, (out, lse) in calls:
                close_out(out[b:b + 1, :, :m], ref, size, terms, hd, one_part)
                close_lse(lse[b:b + 1, :, :m], lref, terms, hd)


def test_custom_ops_on_the_gpu(cuda):
    from kuillm_amd import library  # noqa: F401
    op = torch.ops.kuiops
    c = Cache(cuda, BF, "int8", 2, 2, 64, 16, 3, seed=41)
    a, freq = c.args(), frequencies(64).to(cuda)
    qkv = gen((2, 3, 8 * 64), BF, 1).to(cuda)
    q = op.kv_paged_append(qkv, freq, ints([4, 9], cuda), **a)
    assert torch.equal(q, ops.kv_paged_append(qkv, freq, ints([4, 9], cuda), **a))
    ends = ints([7, 12], cuda)
    for got, want in ((op.sdpa_paged(q, **a, kv_len=ends), ops.sdpa_paged(q, **a, kv_len=ends, return_lse=True)),
                      (op.kv_paged_read(**a, kv_len=ends, length=20), ops.kv_paged_read(**a, kv_len=ends, length=20))):
        assert all(torch.equal(x, y) for x, y in zip(got, want))
