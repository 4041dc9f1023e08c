"""Sizes that 32 bits do not hold are refused by the binding: the library would see them cut (no GPU needed; CPU
tensors stand for device ones, and no call may reach the library)."""
import pytest
import torch

N_KV, HD, PAGE = 2, 64, 16


@pytest.fixture
def cache(pkg, monkeypatch):
    ops = pkg.ops
    c = object.__new__(ops.PagedKV)
    c._index, c.n_kv, c.head_dim, c.n_pages, c.page, c._n_seq, c._ws, c._ref = -1, N_KV, HD, 4, PAGE, 1, {}, 0  # (-1: the CPU)

    def none(name):
        raise AssertionError(f"{name} called")

    monkeypatch.setattr(ops, "_fn", none)
    monkeypatch.setattr(ops, "_stream", lambda index, stream: 0)
    return c


def ints(n):
    return torch.zeros(n, dtype=torch.int32)


BIG = [2**31, 2**32, 2**32 + 5, 2**63]


@pytest.mark.parametrize("big", BIG)
def test_bounds(pkg, cache, big):
    ops = pkg.ops
    k = torch.zeros(3, N_KV, HD)
    q = torch.zeros(3, N_KV, HD, dtype=torch.float16)
    with pytest.raises(ValueError, match="32 bits"):
        ops.kv_append(cache, k, k, ints(2), ints(1), max_rows=big)
    for kw in (dict(max_rows=big, max_keys=5), dict(max_rows=3, max_keys=big)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.kv_attention(cache, q, ints(2), ints(1), workspace=ints(1), **kw)
        with pytest.raises(ValueError, match="32 bits"):
            ops.kv_attention_workspace(cache, n_q=2, n_rows=3, **kw)
    with pytest.raises(ValueError, match="32 bits"):
        ops.kv_attention_workspace(cache, n_q=2, n_rows=big, max_rows=3, max_keys=5)


def test_rows(pkg, cache):
    ops = pkg.ops
    n = 2**32 + 1  # (views of one element)
    with pytest.raises(ValueError, match="32 bits"):
        k = torch.zeros(1).expand(n, N_KV, HD)
        ops.kv_append(cache, k, k, ints(2), ints(1), max_rows=1)
    with pytest.raises(ValueError, match="32 bits"):
        ops.kv_attention(cache, torch.zeros(1, dtype=torch.float16).expand(n, N_KV, HD), ints(2), ints(1), max_rows=1, max_keys=1, workspace=ints(1))


def test_sizes_that_fit_go_on(pkg, cache):
    """... to the library."""
    ops = pkg.ops
    k = torch.zeros(3, N_KV, HD)
    with pytest.raises(AssertionError, match="dfb_kv_append"):
        ops.kv_append(cache, k, k, ints(2), ints(1), max_rows=2**31 - 1)
    with pytest.raises(AssertionError, match="dfb_kv_attention_workspace"):
        ops.kv_attention_workspace(cache, n_q=2, n_rows=3, max_rows=-1, max_keys=2**31 - 1)  # (the library refuses the negative one)


def test_a_decoding_loop_leaves_nothing_behind(pkg, cache, monkeypatch):
    """Each step's bound of the keys is another one: what a cache remembers of the calls stays small, and calls of
    the same sizes ask the library once."""
    ops = pkg.ops
    asked = []
    monkeypatch.setattr(ops, "_fn", lambda name: lambda *a: asked.append(name) or 0)
    q = torch.zeros(1, N_KV, HD, dtype=torch.float16)
    for keys in range(1, 3001):
        for _layer in range(2):
            ops.kv_attention(cache, q, ints(2), ints(1), max_rows=1, max_keys=keys)
    assert len(cache._ws) <= 100
    assert asked.count("dfb_kv_attention_workspace") == 3000 and asked.count("dfb_kv_attention") == 6000
