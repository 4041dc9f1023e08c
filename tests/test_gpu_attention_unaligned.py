"""Query rows that no 16-byte copy can take (odd strides, odd starts), in the large row tiles, give the same bits as
the same rows in a dense tensor: those are moved by other instructions, into the same operands (needs a B200)."""
import numpy as np
import pytest
import torch

from test_gpu_operators import FAR, gen, ints, kill_tail, make_cache, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("split", [True, False], ids=["split", "whole"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [0.1, -0.1])
def test_unaligned_queries(ops, split, dtype, hd, scale):  # noqa: F811
    n_kv, n_q = 2, 6
    n_seq, counts, keys = (3, [150, 1, 97], [700, 1000, 130]) if split else (90, [70, 3, 41] * 30, [300, 40, 129] * 30)
    c = kill_tail(make_cache(ops, n_seq, n_kv, hd, 64, 16, seed=31), keys)
    n = sum(counts)
    off = ints(np.cumsum([0] + counts).tolist())
    q = torch.randn((n, n_q, hd), generator=gen(32), device="cuda").to(dtype)
    kw = dict(max_rows=max(counts), max_keys=FAR if split else max(keys), scale=scale, return_lse=True)
    want = ops.kv_attention(c, q, off, ints(keys), **kw)
    for tok, head, at in ((n_q * (hd + 1), hd + 1, 0), (hd + 3, n * (hd + 3), 1), (n_q * hd, hd, 3)):
        base = torch.full((n * n_q * (hd + 3) + at + 8,), float("nan"), dtype=dtype, device="cuda")
        odd = base.as_strided((n, n_q, hd), (tok, head, 1), at)
        odd.copy_(q)
        for _ in range(10):
            got = ops.kv_attention(c, odd, off, ints(keys), **kw)
            assert bool((got[0] == want[0]).all()) and bool((got[1] == want[1]).all())
