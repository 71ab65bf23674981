"""Forms of the cache operators that a call reaches by its sizes alone, against
the fp64 oracle; tolerances as tests/test_gpu_cache.py counts them."""
import math

import numpy as np
import pytest
import torch

from kuillm_amd import ops
from oracle import kuiops_oracle as O
from test_gpu_cache import BF, HF, close_lse, close_out, gen, npy, padded, trees, wide_capacity

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
