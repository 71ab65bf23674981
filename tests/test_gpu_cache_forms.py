"""Forms of the cache operators that a call reaches by its sizes alone, against
the fp64 oracle; tolerances as tests/test_gpu_cache.py counts them."""
import numpy as np
import pytest
import torch

from kuillm_amd import ops
from oracle import kuiops_oracle as O
from test_gpu_cache import BF, HF, close_lse, close_out, gen, npy, trees

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
