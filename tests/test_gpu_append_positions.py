"""kv_append with positions that cannot all be stored: what is left out leaves no trace, what is stored is
what the same call without the left-out rows stores, no row that does not lie above the row before it is
stored, and no position twice (needs a B200)."""
import random

import pytest
import torch

from test_gpu_operators import check_append, finite_codes, gen, ints, make_cache, ops, ref_append  # noqa: F401

pytestmark = pytest.mark.gpu

SENTINEL = 77.0


def ascending(pos, cap):
    """Rows above the row before them and within the table."""
    return [i for i, p in enumerate(pos) if 0 <= p < cap and (i == 0 or p > pos[i - 1])]


def run(ops, seqs, lens, page, max_pages, dtype=torch.float32):  # noqa: F811
    """Rows stored of each sequence, after the cache has been compared with what storing those rows alone gives."""
    hd, n_kv, n_q = 64, 2, 3
    off = [0]
    for p in seqs:
        off.append(off[-1] + len(p))
    n = off[-1]
    g = gen(n)
    k, v = (torch.randn((n, n_kv, hd), generator=g, device="cuda").to(dtype) for _ in range(2))
    k[n // 2] *= 50
    q = torch.randn((n, n_q, hd), generator=g, device="cuda").to(dtype)
    q_out = torch.full_like(q, SENTINEL)
    c = finite_codes(make_cache(ops, len(seqs), n_kv, hd, page, max_pages))
    before = ops.PagedKV(c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone(), c.pages)
    status = ints([0])
    ops.kv_append(c, k, v, ints(off), ints(lens), max_rows=max(map(len, seqs)), pos=ints([p for s in seqs for p in s]), q=q, q_out=q_out,
                  status=status)
    wrote = (q_out != SENTINEL).all(-1).all(-1)
    assert bool(((q_out == SENTINEL).all(-1).all(-1) | wrote).all())
    assert bool((q_out[wrote] == q[wrote]).all())
    kept = [[i for i in range(len(s)) if bool(wrote[off[j] + i])] for j, s in enumerate(seqs)]
    rows = [off[j] + i for j, x in enumerate(kept) for i in x]
    new_off = [0]
    for x in kept:
        new_off.append(new_off[-1] + len(x))
    want = ref_append(before, k[rows], v[rows], new_off, lens, [seqs[j][i] for j, x in enumerate(kept) for i in x], None)
    check_append(c, want)
    for s, x in zip(seqs, kept):
        assert set(x) <= set(ascending(s, page * max_pages)), (s, x)
        assert len({s[i] for i in x}) == len(x), (s, x)
    bad = any(p < 0 or p >= page * max_pages for s in seqs for p in s) or any(b <= a for s in seqs for a, b in zip(s, s[1:]))
    assert int(status) == (ops.STAT_POSITION if bad else 0)
    return kept


@pytest.mark.parametrize("pos,kept", [
    ([0, 1, 2, 2, 3, 4, 5, 6], [0, 1, 2, 4, 5, 6, 7]),
    ([0, 5, 4, 6, 7, 8, 9, 10], [0, 1, 3, 4, 5, 6, 7]),
    ([-2, 0, 1, 2, 3, 4, 5, 6], [1, 2, 3, 4, 5, 6, 7]),
    ([0, 1, 2, 3, 4, 5, 6, 40], [0, 1, 2, 3, 4, 5, 6]),
    ([2**31 - 1] * 8, []),
    ([-(2**31)] * 8, []),
    ([3, 1, 3, 4, 5, 6, 7, 8], [0, 3, 4, 5, 6, 7]),     # a position again, not next to its first row
    ([3, 4, 5, 3, 4, 5, 6, 7], [0, 1, 2, 6, 7]),        # several again
    ([0, 5, 1, 2, 6, 7, 8, 9], [0, 1, 3, 4, 5, 6, 7]),  # backwards, to positions that no other row names
    ([15, 14, 13, 12, 11, 10, 9, 8], [0]),
    ([7] * 8, [0]),
])
@pytest.mark.parametrize("filled", [0, 20])
def test_bad_positions_leave_no_trace(ops, pos, kept, filled):  # noqa: F811
    assert run(ops, [pos], [filled], 16, 2) == [kept]


@pytest.mark.parametrize("page,dtype", [(16, torch.float32), (32, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16)])
def test_positions_out_of_order(ops, page, dtype):  # noqa: F811
    """Ascending positions with a few rows moved, repeated or sent out of the table, in several sequences."""
    rng = random.Random(page)
    for _ in range(25):
        seqs, lens = [], []
        for _ in range(rng.randint(1, 4)):
            cap = 4 * page
            p = sorted(rng.sample(range(cap), rng.randint(0, min(cap, 150))))
            for _ in range(rng.choice([0, 1, 1, 3])):
                if p:
                    i = rng.randrange(len(p))
                    p[i] = rng.choice([p[rng.randrange(len(p))], rng.randrange(cap), -3, cap + 5])
            seqs.append(p)
            lens.append(rng.randint(0, cap))
        if not any(seqs):
            continue
        got = run(ops, seqs, lens, page, 4, dtype)
        for s, x in zip(seqs, got):
            if s == sorted(set(s)):  # nothing out of order: all that fit
                assert x == ascending(s, 4 * page)
