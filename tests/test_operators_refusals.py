"""What the operators on device tensors refuse on the host, before anything reaches a device: every
check of the C-ABI (no GPU needed; a call whose arguments all pass ends at the device lookup)."""
import ctypes as C

import pytest

ARG, UNSUPPORTED = -1, -6
P = 0x7000000000  # stands for a device address: never read by the checks


def cache(ops, **kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, pages=P, n_pages=8, n_kv=2, head_dim=128, page=64, n_seq=3, max_pages=4)
    d.update(kw)
    return ops._KvCache(**d)


def rows(ops, **kw):
    d = dict(k=P, v=P, type=1, n_rows=5, max_rows=5, k_tok=256, k_head=128, v_tok=256, v_head=128, row_off=P, len=P, pos=None,
             rope=P, n_rope=100, n_q=4, q=P, q_out=P, q_tok=512, q_head=128, q_out_tok=512, q_out_head=128)
    d.update(kw)
    return ops._KvRows(**d)


def attn(ops, **kw):
    d = dict(q=P, out=P, type=1, n_q=4, n_rows=5, max_rows=5, max_keys=100, scale=0.1, q_tok=512, q_head=128, out_tok=512,
             out_head=128, row_off=P, len=P, vis=None, lse=P)
    d.update(kw)
    return ops._KvAttn(**d)


def probs(ops, **kw):
    d = dict(logits=P, type=0, n_vocab=100, n_rows=4, n_logits=4, ld=100, rows=None, targets=P, logprob=P, entropy=P, top_k=3,
             top_ids=P, top_logprob=P)
    d.update(kw)
    return ops._Logprobs(**d)


BAD_CACHE = [(dict(k=None), ARG), (dict(v=None), ARG), (dict(k_scale=None), ARG), (dict(v_scale=None), ARG), (dict(pages=None), ARG),
             (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=16), UNSUPPORTED), (dict(page=48), UNSUPPORTED),
             (dict(page=256), UNSUPPORTED), (dict(n_pages=0), ARG), (dict(n_kv=0), ARG), (dict(n_seq=0), ARG), (dict(max_pages=0), ARG),
             (dict(k=P + 8), ARG), (dict(n_seq=70000), UNSUPPORTED), (dict(max_pages=1 << 26), UNSUPPORTED)]


@pytest.mark.parametrize("kw,rc", BAD_CACHE)
def test_cache_refusals(pkg, kw, rc):
    ops, c = pkg.ops, cache(pkg.ops, **kw)
    r, a = rows(ops), attn(ops)
    assert ops._fn("dfb_kv_append")(C.addressof(c), C.addressof(r), None, None) == rc
    assert ops._fn("dfb_kv_attention")(C.addressof(c), C.addressof(a), None, 0, None, None) == rc
    assert pkg.native()[0].dfb_last_error()


@pytest.mark.parametrize("kw,rc", [
    (dict(type=8), UNSUPPORTED), (dict(type=12), UNSUPPORTED), (dict(n_rows=-1), ARG), (dict(max_rows=-1), ARG), (dict(k=None), ARG),
    (dict(v=None), ARG), (dict(k=P + 1), ARG), (dict(k_tok=-1), ARG), (dict(v_head=-128), ARG), (dict(row_off=None), ARG),
    (dict(len=None), ARG), (dict(n_rope=0), ARG), (dict(rope=P + 4), ARG), (dict(q_out=None), ARG), (dict(n_q=0), ARG),
    (dict(q_tok=-5), ARG), (dict(q=P + 1), ARG)])
def test_append_refusals(pkg, kw, rc):
    c, r = cache(pkg.ops), rows(pkg.ops, **kw)
    assert pkg.ops._fn("dfb_kv_append")(C.addressof(c), C.addressof(r), None, None) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(type=0), UNSUPPORTED), (dict(type=8), UNSUPPORTED), (dict(n_q=3), ARG), (dict(n_q=0), ARG), (dict(n_rows=-1), ARG),
    (dict(max_rows=-2), ARG), (dict(max_keys=-1), ARG), (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG),
    (dict(q=None), ARG), (dict(out=None), ARG), (dict(q=P + 1), ARG), (dict(out_tok=-1), ARG), (dict(row_off=None), ARG),
    (dict(len=None), ARG)])
def test_attention_refusals(pkg, kw, rc):
    c, a = cache(pkg.ops), attn(pkg.ops, **kw)
    assert pkg.ops._fn("dfb_kv_attention")(C.addressof(c), C.addressof(a), None, 0, None, None) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(type=12), UNSUPPORTED), (dict(n_rows=-1), ARG), (dict(n_vocab=0), ARG), (dict(ld=99), ARG), (dict(top_k=-1), ARG),
    (dict(top_k=33), ARG), (dict(n_vocab=2, ld=2), ARG), (dict(top_ids=None), ARG), (dict(top_logprob=None), ARG),
    (dict(targets=None), ARG), (dict(logprob=None), ARG), (dict(n_rows=5), ARG), (dict(logits=None), ARG), (dict(logits=P + 2), ARG)])
def test_logprobs_refusals(pkg, kw, rc):
    a = probs(pkg.ops, **kw)
    assert pkg.ops._fn("dfb_token_logprobs")(C.addressof(a), None, None) == rc


def test_null_structs(pkg):
    ops = pkg.ops
    c, r, a = cache(ops), rows(ops), attn(ops)
    assert ops._fn("dfb_kv_append")(None, C.addressof(r), None, None) == ARG
    assert ops._fn("dfb_kv_append")(C.addressof(c), None, None, None) == ARG
    assert ops._fn("dfb_kv_attention")(C.addressof(c), None, None, 0, None, None) == ARG
    assert ops._fn("dfb_kv_attention_workspace")(C.addressof(c), C.addressof(a), None) == ARG
    assert ops._fn("dfb_token_logprobs")(None, None, None) == ARG


def test_nothing_to_do_is_no_error(pkg):
    ops = pkg.ops
    c = cache(ops)
    for kw in (dict(n_rows=0), dict(max_rows=0)):
        r, a = rows(ops, **kw), attn(ops, **kw)
        assert ops._fn("dfb_kv_append")(C.addressof(c), C.addressof(r), None, None) == 0
        assert ops._fn("dfb_kv_attention")(C.addressof(c), C.addressof(a), None, 0, None, None) == 0
    p = probs(ops, n_rows=0)
    assert ops._fn("dfb_token_logprobs")(C.addressof(p), None, None) == 0


def test_python_checks(pkg):
    """The binding's own checks, on CPU tensors: they are refused before any call."""
    import torch
    ops = pkg.ops
    codes = torch.zeros((4, 2, 16, 64), dtype=torch.uint8)
    scale = torch.ones((4, 2))
    pages = torch.zeros((1, 4), dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedKV(codes, codes.clone(), scale, scale.clone(), pages)
    with pytest.raises(ValueError, match="n_pages"):
        ops.PagedKV(codes[0], codes[0], scale, scale, pages)
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(3, 5))
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(3))
