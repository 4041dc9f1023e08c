"""Bounds that a caller does not know well (max_rows, max_keys far above any sequence's) change neither results nor
the order of a call's time (needs a B200)."""
import time

import numpy as np
import pytest
import torch

from test_gpu_operators import check_append, check_attention, finite_codes, gen, ints, kill_tail, make_cache, ops, ref_append  # noqa: F401

pytestmark = pytest.mark.gpu

INT_MAX = 2**31 - 1


@pytest.mark.parametrize("n_q,n_rows,max_rows", [(4, 1, 1), (4, 200, 200), (2, 64, 64)])
def test_workspace_grows_with_the_bound_of_the_keys(ops, n_q, n_rows, max_rows):  # noqa: F811
    c = make_cache(ops, 1, 2, 64, 16, 4)
    need = [ops.kv_attention_workspace(c, n_q=n_q, n_rows=n_rows, max_rows=max_rows, max_keys=m) for m in (1 << 20, 1 << 30, INT_MAX - 64, INT_MAX - 63, INT_MAX)]
    assert need == sorted(need) and need[-1] > 0


@pytest.mark.parametrize("n_seq,count,keys", [(1, 1, 300), (1, 70, 500), (400, 3, 200), (2000, 1, 40)])
def test_attention_loose_bounds(ops, n_seq, count, keys):  # noqa: F811
    n_kv, n_q, hd = 8, 8, 64
    lens, off = [keys - i % 7 for i in range(n_seq)], np.arange(0, n_seq * count + 1, count).tolist()
    c = kill_tail(make_cache(ops, n_seq, n_kv, hd, 64, -(-keys // 64), seed=3), lens)
    q = torch.randn((n_seq * count, n_q, hd), generator=gen(4), device="cuda").half()
    for max_rows, max_keys in ((count, INT_MAX), (n_seq * count, keys), (1 << 26, keys), (1 << 27, INT_MAX)):
        took = []
        for _ in range(3):  # (the first may load the kernel)
            torch.cuda.synchronize()
            t = time.perf_counter()
            ops.kv_attention(c, q, ints(off), ints(lens), max_rows=max_rows, max_keys=max_keys)
            torch.cuda.synchronize()
            took.append(time.perf_counter() - t)
        assert min(took) < 0.5  # (a loop over all tiles that 2^26 rows could have takes seconds)
        check_attention(ops, c, q, off, lens, max_rows=max_rows, max_keys=max_keys)


def test_append_loose_bounds(ops):  # noqa: F811
    c = finite_codes(make_cache(ops, 2, 2, 64, 16, 9))
    k, v = (torch.randn((7, 2, 64), generator=gen(s), device="cuda") for s in (1, 2))
    want = ref_append(c, k, v, [0, 4, 7], [30, 100], None, None)
    status = ints([0])
    ops.kv_append(c, k, v, ints([0, 4, 7]), ints([30, 100]), max_rows=INT_MAX, status=status)
    check_append(c, want)
    assert int(status) == 0
