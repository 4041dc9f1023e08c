"""Log probabilities of finite logits far from 0: fills that exclude tokens (-1e9 .. -1e30), maxima of that
size, and rows whose values lie on both sides of the size where the kernel changes its arithmetic.  The
reference and the tolerances are those of test_gpu_operators.py (needs a B200)."""
import math

import pytest
import torch

from test_gpu_operators import check_logprobs, gen, ops  # noqa: F401

pytestmark = pytest.mark.gpu

DTYPES = [(torch.float32, 1e30), (torch.bfloat16, 1e30), (torch.float16, 6e4)]
IDS = ["f32", "bf16", "f16"]


@pytest.mark.parametrize("dtype,most", DTYPES, ids=IDS)
@pytest.mark.parametrize("fill", [-6e4, -1.5e6, -1e9, -3e9, -1e10, -1e20, -1e30])
@pytest.mark.parametrize("V", [9, 5003, 20000, 126464])
def test_fills(ops, dtype, most, fill, V):  # noqa: F811
    """Few tokens are left: at the row's end, in its middle, at its start; none is; every other one is."""
    if -fill > most:
        pytest.skip("the type has no such value")
    g = gen(V)
    x = torch.full((6, V), fill, device="cuda")
    live = torch.randn(V, generator=g, device="cuda")
    x[0, -3:] = live[-3:]
    x[1, V // 2 + 1] = live[0]
    x[2, :2] = live[:2]
    x[4, ::2] = live[::2] * 3
    x[5, V // 3 : V // 3 + 2] = live[:2] - 1000
    targets = [V - 2, V // 2 + 1, 1, 5, -1, 0]
    k = min(V, 9)
    check_logprobs(ops, x.to(dtype), targets, k)
    lp, ent, ids, top = check_logprobs(ops, x[3:4].to(dtype), [5], k)
    assert abs(float(lp[0]) + math.log(V)) <= 1e-3 and ids[0].tolist() == list(range(k))


@pytest.mark.parametrize("dtype,most", DTYPES, ids=IDS)
@pytest.mark.parametrize("big", [6e4, 1.5e6, 3e9, 1e10, 1e20, 1e30])
def test_large_maxima(ops, dtype, most, big):  # noqa: F811
    if big > most:
        pytest.skip("the type has no such value")
    V = 20000
    g = gen(3)
    x = torch.randn((5, V), generator=g, device="cuda")
    x[0] = big
    x[1, V - 1] = big           # behind the first batch
    x[2, 7::11] = big           # several
    x[3] = big
    x[3, 1::2] = -big
    x[4] = -math.inf
    x[4, 40:4000] = big
    check_logprobs(ops, x.to(dtype), [3, V - 1, 7, 0, 41], 12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("base", [2.0**18, 2.0**20, 2.0**21, 2.0**24, 2.0**31, 2.0**33, -(2.0**18), -(2.0**20), -(2.0**24), -(2.0**33)])
def test_small_steps_at_large_values(ops, dtype, base):  # noqa: F811
    """Rows of a base and a few steps of the type around it, rising, falling and mixed: the softmax is far from
    a single token's, and maxima cross powers of two on the way."""
    V = 30011
    g = gen(11)
    step = abs(base) * torch.finfo(dtype).eps
    i = torch.arange(V, device="cuda", dtype=torch.float64)
    rows = [base + step * torch.floor(i / V * 20 - 10), base - step * torch.floor(i / V * 20 - 10),
            base + step * torch.randint(-12, 13, (V,), generator=g, device="cuda"),
            torch.where(i < V - 5, base - 5 * step, base + 2 * step)]
    x = torch.stack(rows).float().to(dtype)
    check_logprobs(ops, x, [0, 1, 2, V - 1], 8)


def test_far_values_raise_no_flag(ops):  # noqa: F811
    """Rows of a fill and one token each: it is certain, and nothing is reported (check_logprobs looks at the status)."""
    x = torch.full((300, 6000), -1e10, device="cuda")
    x[:, 5990] = torch.arange(300, device="cuda").float()
    lp, ent, ids, top = check_logprobs(ops, x, [5990] * 300, 2)
    assert bool((ids[:, 0] == 5990).all()) and bool((ids[:, 1] == 0).all())
