"""Outputs whose rows share elements are refused, for every layout and no other (no GPU needed: the check comes
before the device is looked up)."""
import ctypes as C
import itertools
import random

import pytest

from test_operators_refusals import ARG, P, attn, cache, rows


def refused(pkg, what, n, tok, heads, head, hd):
    ops = pkg.ops
    c = cache(ops, head_dim=hd, n_kv=1)
    if what == "out":
        s = attn(ops, n_q=heads, n_rows=n, max_rows=n, q_tok=0, q_head=0, out_tok=tok, out_head=head)
        rc = ops._fn("dfb_kv_attention")(C.addressof(c), C.addressof(s), None, 0, None, None)
    else:
        s = rows(ops, n_q=heads, n_rows=n, max_rows=n, q_tok=0, q_head=0, k_tok=0, k_head=0, v_tok=0, v_head=0, q_out_tok=tok, q_out_head=head)
        rc = ops._fn("dfb_kv_append")(C.addressof(c), C.addressof(s), None, None)
    message = pkg.native()[0].dfb_last_error().decode()
    hit = "overlap" in message
    assert rc != 0 and (not hit or (rc == ARG and what in message))  # (no device here: every call ends in an error)
    return hit


def overlap(n, tok, heads, head, hd):
    at = sorted(i * tok + h * head for i in range(n) for h in range(heads))
    return any(b - a < hd for a, b in itertools.pairwise(at))


@pytest.mark.parametrize("what", ["out", "q_out"])
def test_every_layout(pkg, what):
    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        hd, n, heads = rng.choice([64, 128]), rng.randint(1, 6), rng.randint(1, 6)
        tok, head = (rng.choice([0, 1, hd - 1, hd, hd + 1, 2 * hd, 3 * hd, 5 * hd, heads * hd, n * hd, rng.randint(0, 8 * hd)]) for _ in range(2))
        want = overlap(n, tok, heads, head, hd)
        assert refused(pkg, what, n, tok, heads, head, hd) == want, (hd, n, tok, heads, head)
        seen[want] += 1
    assert min(seen.values()) > 500


@pytest.mark.parametrize("what", ["out", "q_out"])
@pytest.mark.parametrize("n,tok,heads,head,want", [
    (100000, 0, 28, 128, True), (100000, 28 * 128, 28, 0, True), (100000, 28 * 128, 28, 128, False), (100000, 128, 28, 12800000, False),
    (1, 0, 28, 128, False), (100000, 128, 1, 0, False), (1000, 128, 28, 128, True), (100000, 1 << 62, 28, 128, False),
    (5, 1 << 62, 28, 1 << 62, True)])
def test_large_layouts(pkg, what, n, tok, heads, head, want):
    assert refused(pkg, what, n, tok, heads, head, 128) == want
