"""The paged 8-bit K/V cache (append and attention) and the token log probabilities: cases and plain forms.

Where `own` is false, run() computes an operator with elementary torch operations; where it is true, it makes the
calls of this package that a user makes.

The cache holds E4M3 codes [page][kv head][position in the page][dimension] and one power-of-two scale for each
page and kv head; a value is code * scale.  Codes are returned as float8_e4m3fn numbers beside their scales.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

E4M3_MAX = 448.0
MIN_EXP = -64  # the smallest scale is 2^-64
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One token of one sequence after a 1000-position context, Dream-7B's heads: the smallest call.
        dict(name="append 1 token", op="append", n_q=28, n_kv=4, hd=128, page=64, n_seq=1, rows=1, ctx=1000, dtype="bf16"),
        # Odd row counts over odd contexts, small pages, 64-wide heads.
        dict(name="append ragged p16", op="append", n_q=8, n_kv=2, hd=64, page=16, n_seq=13, rows=37, ctx=301, dtype="f16"),
        # A 256-token denoising block of 16 sequences rewritten behind its prompts, LLaDA-8B's heads, f32 projections.
        dict(name="append 16x256 f32", op="append", n_q=32, n_kv=32, hd=128, page=64, n_seq=16, rows=256, ctx=512, dtype="f32"),
        # The prompts of a 64-sequence batch entering an empty cache, LLaDA-8B's heads.
        dict(name="append 64x512", op="append", n_q=32, n_kv=32, hd=128, page=64, n_seq=64, rows=512, ctx=0, dtype="bf16"),
        # One query token over a 4607-key cache, Dream-7B's heads: latency.
        dict(name="attention 1x4607", op="attention", n_q=28, n_kv=4, hd=128, page=64, n_seq=1, rows=1, keys=4607, vis="full", dtype="bf16"),
        # The headline block: 256 tokens over 320 positions, LLaDA-8B's heads.
        dict(name="attention 256x320", op="attention", n_q=32, n_kv=32, hd=128, page=64, n_seq=1, rows=256, keys=320, vis="full", dtype="f16"),
        # A 32-token block over Dream-7B's whole context.
        dict(name="attention 32x131072", op="attention", n_q=28, n_kv=4, hd=128, page=64, n_seq=1, rows=32, keys=131072, vis="full", dtype="bf16"),
        # Sixteen ragged sequences, each token seeing the keys up to the end of its own 32-token block.
        dict(name="attention 16x61 ragged", op="attention", n_q=28, n_kv=4, hd=128, page=32, n_seq=16, rows=61, keys=4100, vis="block", dtype="bf16"),
        # The 64-sequence batch: 256-token blocks over 768 positions, LLaDA-8B's heads: the largest.
        dict(name="attention 64x256x768", op="attention", n_q=32, n_kv=32, hd=128, page=64, n_seq=64, rows=256, keys=768, vis="full", dtype="bf16"),
        # One position's candidates.
        dict(name="logprobs 1 row", op="logprobs", n_rows=1, vocab=126464, k=5, masked=False, dtype="f32"),
        # A 256-token block's candidates, LLaDA-8B's vocabulary.
        dict(name="logprobs 256 rows", op="logprobs", n_rows=256, vocab=126464, k=8, masked=False, dtype="f32"),
        # Scored answers, Dream-7B's vocabulary, part of it excluded by -inf.
        dict(name="logprobs 2048 rows", op="logprobs", n_rows=2048, vocab=152064, k=20, masked=True, dtype="bf16"),
    ]


HEADS = [(28, 4, 128), (32, 32, 128), (14, 2, 128), (8, 8, 128), (8, 2, 64), (4, 1, 64), (12, 12, 64)]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "logprobs"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "logprobs":
        vocab = _log_int(rng, 17, 152064)
        n_rows = _log_int(rng, 1, min(2048, (150_000_000 if dtype == "f32" else 300_000_000) // vocab))
        return dict(op=op, n_rows=n_rows, vocab=vocab, k=rng.randint(0, min(32, vocab)), masked=rng.random() < 0.5, dtype=dtype)
    n_q, n_kv, hd = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    n_seq = _log_int(rng, 1, 64)
    if op == "append":
        most = 32768 * 128 * 128 // (n_seq * hd * (2 * n_q + 2 * n_kv) * (2 if dtype == "f32" else 1))
        rows = _log_int(rng, 1, max(1, min(8192, most)))
        return dict(op=op, n_q=n_q, n_kv=n_kv, hd=hd, page=page, n_seq=n_seq, rows=rows, ctx=_log_int(rng, 1, 4096) - 1, dtype=dtype)
    dtype = rng.choice(["f16", "bf16"])
    keys = _log_int(rng, 1, 32768 // max(1, n_seq * n_kv // 32))
    most = 64 * 256 * 768 * 32 * 128 // 2 // (n_seq * keys * n_q * hd)
    rows = _log_int(rng, 1, max(1, min(1024, keys, most)))
    return dict(op=op, n_q=n_q, n_kv=n_kv, hd=hd, page=page, n_seq=n_seq, rows=rows, keys=keys, vis=rng.choice(["full", "block", "causal"]), dtype=dtype)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _counts(case, most):
    """Rows or keys of each sequence, by the case alone: all alike where `most` is a multiple of 64, else ragged, one of them empty."""
    g = _generator(most)
    n = case["n_seq"]
    if n == 1 or most % 64 == 0:
        return torch.full((n,), most, dtype=torch.int64, device="cuda")
    c = torch.randint(max(1, most // 4), most + 1, (n,), generator=g, device="cuda")
    c[0] = most
    if n > 2:
        c[n // 2] = 0
    return c


def _offsets(c):
    return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), c.cumsum(0)]).to(torch.int32)


def _cache(case, g, lens):
    """A pool with a few pages to spare, handed out in a random order, filled with codes of N(0, 1)-like values."""
    page, n_kv, hd, n_seq = case["page"], case["n_kv"], case["hd"], case["n_seq"]
    max_pages = max(1, -(-int(lens.max()) // page))
    n_pages = n_seq * max_pages + 3
    pages = torch.randperm(n_pages, generator=g, device="cuda")[: n_seq * max_pages].reshape(n_seq, max_pages).to(torch.int32)
    shape = (n_pages, n_kv, page, hd)

    def pool():
        out = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
        flat = out.view(n_pages, -1)
        step = max(1, (1 << 26) // flat.shape[1])
        for i in range(0, n_pages, step):
            x = torch.randn((min(step, n_pages - i), flat.shape[1]), generator=g, device="cuda") * 100
            flat[i : i + step] = x.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        return out

    def scale():
        return torch.exp2(torch.randint(-8, -5, (n_pages, n_kv), generator=g, device="cuda").float())

    return dict(k_codes=pool(), v_codes=pool(), k_scale=scale(), v_scale=scale(), pages=pages)


def _rope_table(n, hd):
    """cos and sin of position * 500000^(-2 i / hd), rounded once from 64 bits."""
    inv = 500000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device="cuda") / hd)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        n, v = case["n_rows"], case["vocab"]
        logits = torch.empty((n, v), dtype=dt, device="cuda")
        step = max(1, (1 << 27) // v)
        for i in range(0, n, step):
            logits[i : i + step] = (torch.randn((min(step, n - i), v), generator=g, device="cuda") * 3).to(dt)
        # every third row is a confident one
        logits[::3, int(torch.randint(0, v, (1,), generator=g, device="cuda"))] = 20.0
        targets = torch.randint(0, v, (n,), generator=g, device="cuda")
        if case["masked"]:
            dead = torch.rand(v, generator=g, device="cuda") < 0.1
            logits.masked_fill_(dead[None], -math.inf)
            targets[1::5] = -1  # positions that are not scored
            if n > 3:
                logits[3] = -math.inf  # a row whose mask leaves nothing
        return dict(op="logprobs", k=case["k"], logits=logits, targets=targets.to(torch.int32))
    n_q, n_kv, hd, n_seq = case["n_q"], case["n_kv"], case["hd"], case["n_seq"]
    if case["op"] == "append":
        ctx = _counts(case, case["ctx"]) if case["ctx"] else torch.zeros(n_seq, dtype=torch.int64, device="cuda")
        rows = _counts(case, case["rows"])
        s = _cache(case, g, ctx + rows)
        total = int(rows.sum())
        qkv = torch.randn((total, (n_q + 2 * n_kv) * hd), generator=g, device="cuda").to(dt)
        s.update(op="append", qkv=qkv, n_q=n_q, row_off=_offsets(rows), lens=ctx.to(torch.int32), max_rows=case["rows"],
                 rope=_rope_table(int((ctx + rows).max()), hd), q_out=torch.zeros((total, n_q, hd), dtype=dt, device="cuda"))
        return s
    keys = _counts(case, case["keys"])
    rows = torch.minimum(_counts(case, case["rows"]), keys)
    if n_seq > 2 and case["rows"] % 64:
        rows[1] = max(1, int(rows[1]))
        keys[n_seq // 2] = 0  # queries without a key
        rows[n_seq // 2] = min(case["rows"], 3)
    s = _cache(case, g, keys)
    total = int(rows.sum())
    off = _offsets(rows)
    vis = None
    if case["vis"] != "full":
        # the block is the sequence's last tokens: token t sees the keys up to itself, or up to the end of its 32-token block
        seq = torch.repeat_interleave(torch.arange(n_seq, device="cuda"), rows)
        t = torch.arange(total, device="cuda") - off[:-1][seq]
        n = keys[seq] - rows[seq] + (t + 1 if case["vis"] == "causal" else (t // 32 + 1) * 32)
        vis = torch.minimum(n.clamp_min(0), keys[seq]).to(torch.int32)
        vis[total // 3] = 0  # a token that sees nothing
    s.update(op="attention", q=torch.randn((total, n_q, hd), generator=g, device="cuda").to(dt), row_off=off, lens=keys.to(torch.int32),
             max_rows=max(1, int(rows.max())), max_keys=case["keys"], vis=vis, scale=1.0 / math.sqrt(hd))
    return s


def _package():
    """This repository's package: its folder's name has a hyphen, so it is loaded by path."""
    name = "diffuse_b200"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join(os.getcwd(), "diffuse-cpp_b200", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _handle(s):
    """The cache handle that a program makes once over its pool."""
    if "handle" not in s:
        s["handle"] = _package().ops.PagedKV(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["pages"])
    return s["handle"]


def run(s):
    if own:
        ops = _package().ops
        if s["op"] == "logprobs":
            return ops.token_logprobs(s["logits"], s["targets"], top_k=s["k"])
        if s["op"] == "append":
            k, v, q = _qkv(s)
            ops.kv_append(_handle(s), k, v, s["row_off"], s["lens"], max_rows=s["max_rows"], rope=s["rope"], q=q, q_out=s["q_out"])
            return s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"], s["q_out"]
        return ops.kv_attention(_handle(s), s["q"], s["row_off"], s["lens"], max_rows=s["max_rows"], max_keys=s["max_keys"],
                                scale=s["scale"], vis=s["vis"], return_lse=True)
    if s["op"] == "logprobs":
        return _plain_logprobs(s["logits"], s["targets"], s["k"])
    if s["op"] == "append":
        return _plain_append(s)
    return _plain_attention(s)


def _qkv(s):
    """Views of the fused projection's rows."""
    n_kv, hd, n_q = s["k_codes"].shape[1], s["k_codes"].shape[3], s["n_q"]
    x = s["qkv"].view(s["qkv"].shape[0], n_q + 2 * n_kv, hd)
    return x[:, n_q : n_q + n_kv], x[:, n_q + n_kv :], x[:, :n_q]


# ── plain forms ──


def _rotate(x, cs):
    """NEOX pairs (i, i + hd/2) rotated, in 64 bits: a value next to a border of two codes has to fall on its own side."""
    a, b = x.double().chunk(2, -1)
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _need_exp(amax):
    """The smallest e >= MIN_EXP with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    e = e - torch.where(m <= 0.875, 9, 8)
    return torch.where(amax > 0, e.clamp_min(MIN_EXP), MIN_EXP)


def _to_code(x):
    """E4M3's nearest value, ties to even, of |x| <= 448."""
    e = (torch.frexp(x)[1] - 1).clamp_min(-6)
    step = torch.ldexp(torch.ones_like(x), e - 3)
    return (x / step).round() * step


def _plain_append(s):
    k, v, q = _qkv(s)
    page = s["k_codes"].shape[2]
    off, lens = s["row_off"].long(), s["lens"].long()
    n = off[1:] - off[:-1]
    r = torch.arange(k.shape[0], device="cuda")
    seq = torch.searchsorted(off[1:].contiguous(), r, right=True)
    pos = lens[seq] + r - off[seq]
    pid = s["pages"].long()[seq, pos // page]
    # surviving positions of the page that a sequence's first new row falls into
    first = s["pages"].long()[torch.arange(len(n), device="cuda"), (lens // page).clamp_max(s["pages"].shape[1] - 1)]
    left = torch.where(n > 0, lens % page, 0)
    kept = torch.zeros(s["k_codes"].shape[0], dtype=torch.int64, device="cuda").scatter_reduce_(0, first, left, "amax")
    touched = torch.zeros_like(kept, dtype=torch.bool).index_fill_(0, pid, True)
    cs = s["rope"][pos]
    for x, codes, scale in ((_rotate(k, cs), s["k_codes"], s["k_scale"]), (v.double(), s["v_codes"], s["v_scale"])):
        amax = torch.zeros(codes.shape[:2], dtype=torch.float64, device="cuda").index_reduce_(0, pid, x.abs().amax(-1), "amax")
        old = torch.frexp(scale)[1] - 1
        need = _need_exp(amax)
        e = torch.where((kept > 0)[:, None], torch.maximum(need, old), need)
        e = torch.where(touched[:, None], e, old)
        # survivors of pages whose scale grows
        grown = ((e > old) & (kept > 0)[:, None]).nonzero()
        pg, hd_ = grown[:, 0], grown[:, 1]
        keep = torch.arange(page, device="cuda")[None] < kept[pg][:, None]
        before = codes[pg, hd_].double()
        after = _to_code(torch.ldexp(before, (old - e)[pg, hd_][:, None, None]))
        codes[pg, hd_] = torch.where(keep[..., None], after, before).float().to(codes.dtype)
        scale.copy_(torch.ldexp(torch.ones_like(scale), e))
        codes[pid, :, pos % page] = _to_code(torch.ldexp(x, -e[pid][..., None])).float().to(codes.dtype)
    s["q_out"].copy_(_rotate(q, cs))
    return s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"], s["q_out"]


def _plain_attention(s):
    page, n_kv, hd = s["k_codes"].shape[2], s["k_codes"].shape[1], s["k_codes"].shape[3]
    q, off, lens = s["q"], s["row_off"].long(), s["lens"].long()
    total, n_q = q.shape[0], q.shape[1]
    n_seq, rep = len(lens), n_q // n_kv
    at = torch.arange(s["max_keys"], device="cuda")
    pid = s["pages"].long()[:, at // page]  # [sequence][key]
    # [sequence][kv head][key][dimension]
    k = (s["k_codes"][pid, :, at % page].float() * s["k_scale"][pid][..., None]).transpose(1, 2)
    v = (s["v_codes"][pid, :, at % page].float() * s["v_scale"][pid][..., None]).transpose(1, 2)
    live = at[None] < lens[:, None]
    v = torch.where(live[:, None, :, None], v, 0.0)
    r = torch.arange(total, device="cuda")
    seq = torch.searchsorted(off[1:].contiguous(), r, right=True)
    t = r - off[seq]
    qp = torch.zeros((n_seq, s["max_rows"], n_kv, rep, hd), device="cuda")
    qp[seq, t] = q.float().view(total, n_kv, rep, hd)
    see = torch.zeros((n_seq, s["max_rows"]), dtype=torch.int64, device="cuda")
    see[seq, t] = lens[seq] if s["vis"] is None else torch.minimum(s["vis"].long(), lens[seq])
    # [sequence][kv head][row, query head of the group][key]
    x = (qp.permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, -1, hd) @ k.transpose(2, 3)).mul_(s["scale"])
    dead = (at[None, None] >= see[..., None]).repeat_interleave(rep, 1)[:, None]
    x.masked_fill_(dead, -math.inf)
    m = x.amax(-1, keepdim=True)
    base = torch.where(m.isinf(), 0.0, m)
    p = x.sub_(base).exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.where(z > 0, (p @ v) / z, 0.0)
    lse = (z.log() + base)[..., 0]
    o = o.view(n_seq, n_kv, -1, rep, hd).transpose(1, 2)[seq, t].reshape(total, n_q, hd)
    lse = lse.view(n_seq, n_kv, -1, rep).transpose(1, 2)[seq, t].reshape(total, n_q)
    return o.to(q.dtype), lse


def _plain_logprobs(logits, targets, k):
    x = logits.float()
    n, v = x.shape
    m = x.amax(-1, keepdim=True)
    base = torch.where(m.isinf(), 0.0, m)
    d = x - base
    e = d.exp()
    z = e.sum(-1, keepdim=True)
    logz = z.log()
    lp = d - logz  # a row with nothing left: -inf - -inf, put right below
    none = m.isinf()
    # H = log Z - sum e d / Z; what has no probability adds nothing
    h = logz - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / z
    h = torch.where(none, 0.0, h)[:, 0]
    t = targets.long()
    got = torch.where(none[:, 0], -math.inf, lp.gather(1, t.clamp_min(0)[:, None])[:, 0])
    got = torch.where(t >= 0, got, 0.0)
    # values in their order, equal ones by the lower index, as whole numbers
    u = (x + 0.0).view(torch.int32).long()
    key = torch.where(u < 0, ~u & 0xFFFFFFFF, u | 0x80000000)
    del e, d
    key = (key - 0x80000000 << 32) + (v - 1 - torch.arange(v, device="cuda"))
    top = (v - 1 - (key.topk(k, -1).values & 0xFFFFFFFF)).to(torch.int32)
    top_lp = torch.where(none, -math.inf, lp.gather(1, top.long()))
    return got, h, top, top_lp


# ── work: each input read once, each output written once ──


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if case["op"] == "logprobs":
        n, v, k = case["n_rows"], case["vocab"], case["k"]
        return {"bytes": n * (v * size + 4 + 8 + 8 * k), "flops": 4 * n * v}
    n_q, n_kv, hd, page, n_seq = (case[x] for x in ("n_q", "n_kv", "hd", "page", "n_seq"))

    def mean(most):  # of _counts
        if n_seq == 1 or most % 64 == 0:
            return float(most)
        c = (most + max(1, most // 4)) / 2
        return (most + c * (n_seq - 1 - (n_seq > 2))) / n_seq

    rows = mean(case["rows"]) * n_seq
    if case["op"] == "append":
        ctx = mean(case["ctx"])
        table = (rows / n_seq if n_seq == 1 else ctx + rows / n_seq) * hd * 4
        return {"bytes": rows * hd * ((n_q + 2 * n_kv) * size + n_q * size + 2 * n_kv) + table + 8 * n_kv * (rows / page + n_seq), "flops": rows * hd * (3 * (n_q + n_kv) + 2 * 2 * n_kv)}
    keys = mean(case["keys"]) * n_seq
    seen = mean(case["keys"]) - (rows / n_seq / 2 if case["vis"] == "causal" else 0)
    return {"bytes": keys * n_kv * (2 * hd + 8 / page) + rows * n_q * (2 * hd * size + 4), "flops": 4 * rows * max(1.0, seen) * n_q * hd}


# ── the definitions in 64 bits ──


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "append":
        return _exact_append(s)
    return _exact_attention(s)


def _exact_logprobs(s):
    got, ent, ids, alt = [], [], [], []
    step = max(1, (1 << 26) // s["logits"].shape[1])
    for i in range(0, s["logits"].shape[0], step):
        x = s["logits"][i : i + step].double()
        t = s["targets"][i : i + step].long()
        lz = torch.logsumexp(x, -1, keepdim=True)
        lp = torch.where(lz.isinf(), -math.inf, x - lz)
        got.append(torch.where(t < 0, 0.0, lp.gather(1, t.clamp_min(0)[:, None])[:, 0]))
        ent.append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(-1))
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : s["k"]]
        ids.append(order.to(torch.int32))
        alt.append(lp.gather(1, order))
    return torch.cat(got), torch.cat(ent), torch.cat(ids), torch.cat(alt)


#: All of E4M3's finite values that are not negative, in order: their places are their codes.
def _e4m3_values():
    return torch.tensor([(m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127], dtype=torch.float64, device="cuda")


def _nearest_e4m3(x):
    """By search among the values: the nearer neighbour, on a tie the one with the even code."""
    t = _e4m3_values()
    a = x.abs().contiguous()
    hi = torch.searchsorted(t, a).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    dl, dh = a - t[lo], t[hi] - a
    c = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.where(x < 0, -t[c], t[c])


def _exact_append(s):
    page = s["k_codes"].shape[2]
    k, v, q = _qkv(s)
    off, lens = s["row_off"].tolist(), s["lens"].tolist()
    kc, vc, ks, vs = s["k_codes"].double(), s["v_codes"].double(), s["k_scale"].double(), s["v_scale"].double()
    q_out = torch.zeros(s["q_out"].shape, dtype=torch.float64, device="cuda")

    def turned(x, a, b, p0):
        z = torch.view_as_complex(s["rope"][p0 : p0 + b - a].double())[:, None]
        h = x.shape[-1] // 2
        w = torch.complex(x[a:b, :, :h].double(), x[a:b, :, h:].double()) * z
        return torch.cat([w.real, w.imag], -1)

    if len(off) - 1 + sum(off[-1:]) // page > 4000:
        return None
    for i, p0 in enumerate(lens):
        a, b = off[i], off[i + 1]
        if a == b:
            continue
        q_out[a:b] = turned(q, a, b, p0)
        for x, codes, scale in ((turned(k, a, b, p0), kc, ks), (v[a:b].double(), vc, vs)):
            p = p0
            while p < p0 + b - a:
                n = min(page - p % page, p0 + b - a - p)
                pid, at = int(s["pages"][i, p // page]), p % page
                new = x[p - p0 : p - p0 + n].transpose(0, 1)
                need = torch.exp2(torch.ceil(torch.log2((new.abs().amax((1, 2)) / E4M3_MAX).clamp_min(2.0**MIN_EXP))))
                to = torch.maximum(need, scale[pid]) if at else need
                codes[pid, :, :at] = _nearest_e4m3(codes[pid, :, :at] * (scale[pid] / to)[:, None, None])
                codes[pid, :, at : at + n] = _nearest_e4m3(new / to[:, None, None])
                scale[pid] = to
                p += n
    return kc, ks, vc, vs, q_out


def _exact_attention(s):
    page, n_kv = s["k_codes"].shape[2], s["k_codes"].shape[1]
    off, lens = s["row_off"].tolist(), s["lens"].tolist()
    q = s["q"]
    rep, hd = q.shape[1] // n_kv, q.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        a, b = off[i], off[i + 1]
        if a == b or n == 0:
            continue
        ids = s["pages"][i, : -(-n // page)].long()
        k, v = ((c[ids].double() * f[ids].double()[..., None, None]).transpose(0, 1).reshape(n_kv, -1, hd)[:, :n] for c, f in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])))
        qq = q[a:b].double().view(b - a, n_kv, rep, hd).permute(1, 0, 2, 3).reshape(n_kv, -1, hd)
        x = torch.matmul(qq, k.transpose(1, 2)) * s["scale"]
        if s["vis"] is not None:
            see = s["vis"][a:b].long().repeat_interleave(rep)
            x = torch.where(torch.arange(n, device="cuda")[None] < see[:, None], x, -math.inf)
        lz = torch.logsumexp(x, -1)
        p = torch.where(lz.isinf()[..., None], 0.0, torch.exp(x - lz[..., None]))
        out[a:b] = torch.matmul(p, v).view(n_kv, b - a, rep, hd).permute(1, 0, 2, 3).reshape(b - a, -1, hd)
        lse[a:b] = lz.view(n_kv, b - a, rep).permute(1, 0, 2).reshape(b - a, -1)
    return out, lse
