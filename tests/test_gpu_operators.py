"""The paged 8-bit K/V cache and the token log probabilities against their definitions in 64 bits
(needs a B200).

Tolerances, from the arithmetic (u = half a step relative to the value: f32 2^-24, bf16 2^-8, f16
2^-11, E4M3 2^-4):
* append: every code is the one rounding of the exact rotated value at a power-of-two scale, so the
  codes and scales are the reference's bit for bit; q_out is within half a step of its type.
* attention: out is one rounding to its type of sum p v with p rounded to f16 at most (u = 2^-11,
  f16's subnormals below 2^-24 of the largest), scores and sums in f32.  A score's error is at most
  ds = (hd + 4) 2^-24 scale sum |q k| (hd products and sums, the scale products), which changes p
  by 2 ds relative (its own and the sum's); the row sum adds at most n 2^-24.  So
  |out - ref| <= u |ref| + (2^-11 + 2 ds + n 2^-24 + 2^-20) S + n 2^-24 vmax, S = sum p |v|, where
  2^-20 covers the exponentials and the division, and |lse - ref| <= ds + n 2^-24 + 2^-20 (1 + |ref|).
* log probabilities: x - m is exact to f32's u, exponentials and the logarithm to a few u, sums of
  n terms in f32 by threads: |logprob - ref| <= (n / 128 + 16) 2^-24 (1 + |x - m| + log n), and the
  same for the entropy, whose terms are sums of probabilities times |x - m|: times (1 + max |x - m|).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

# half the step of a type's subnormals: the rounding error of a value below its smallest normal one is
# not relative to the value (f16's subnormals are multiples of 2^-24, so it is up to 2^-25)
SUB = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
E4M3 = torch.tensor([(m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rope_table(n, hd):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
    return torch.stack([a.cos(), a.sin()], -1).float().cuda()


def make_cache(ops, n_seq, n_kv, hd, page, max_pages, seed=0, spare=2):
    """A pool whose pages are handed out in random order and filled with random codes, NaN codes among them."""
    g = gen(seed)
    n_pages = n_seq * max_pages + spare
    pages = torch.randperm(n_pages, generator=g, device="cuda")[: n_seq * max_pages].reshape(n_seq, max_pages).to(torch.int32)
    shape = (n_pages, n_kv, page, hd)
    k, v = (torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.exp2(torch.randint(-9, -3, shape[:2], generator=g, device="cuda").float()) for _ in range(2))
    return ops.PagedKV(k, v, ks, vs, pages.contiguous())


def finite_codes(c):
    """No NaN codes: what a cache holds at its live positions."""
    for t in (c.k, c.v):
        t[(t & 127) == 127] = 5
    return c


def value(code):
    """E4M3 codes (uint8) as float64."""
    t = torch.cat([E4M3, torch.tensor([math.nan], dtype=torch.float64)]).to(code.device)
    x = t[(code & 127).long()]
    return torch.where(code >= 128, -x, x)


def nearest(x):
    """Code of the nearest E4M3 value, ties to the even code, of |x| <= 448."""
    t = E4M3.to(x.device)
    a = x.abs().contiguous()
    hi = torch.searchsorted(t, a).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    dl, dh = a - t[lo], t[hi] - a
    c = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (c + torch.where(torch.signbit(x), 128, 0)).to(torch.uint8)


def rotated(x, cs):
    h = x.shape[-1] // 2
    a, b = x[..., :h].double(), x[..., h:].double()
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def ref_append(c, k, v, off, lens, pos, rope):
    """Copies of the cache's tensors after the call, position by position of the definition."""
    kc, vc, ks, vs = c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone()
    P = c.page
    for s in range(len(lens)):
        a, b = off[s], off[s + 1]
        ps = [lens[s] + i for i in range(b - a)] if pos is None else pos[a:b]
        if not ps:
            continue
        at = torch.tensor(ps, device="cuda")
        kk = rotated(k[a:b], rope[at]) if rope is not None else k[a:b].double()
        for x, codes, scale in ((kk, kc, ks), (v[a:b].double(), vc, vs)):
            for pg in sorted({p // P for p in ps}):
                idx = [i for i, p in enumerate(ps) if p // P == pg]
                slots = [ps[i] % P for i in idx]
                pid = int(c.pages[s, pg])
                new = x[idx].transpose(0, 1)  # [n_kv][rows][hd]
                keep = [t for t in range(min(P, max(0, lens[s] - pg * P))) if t not in slots]
                for h in range(c.n_kv):
                    am = float(new[h].abs().max())
                    e = -64
                    while am > 448.0 * 2.0**e:
                        e += 1
                    if keep:
                        old = int(math.log2(float(scale[pid, h])))
                        if old < e:
                            codes[pid, h, keep] = nearest(value(codes[pid, h, keep]) * 2.0 ** (old - e))
                        e = max(e, old)
                    codes[pid, h, slots] = nearest(new[h] * 2.0**-e)
                    scale[pid, h] = 2.0**e
    return kc, vc, ks, vs


def check_append(c, want, q_out=None, q_want=None):
    for name, got, ref in zip(("k", "v", "k_scale", "v_scale"), (c.k, c.v, c.k_scale, c.v_scale), want):
        bad = (got != ref).nonzero()
        assert bad.numel() == 0, (name, len(bad), bad[:4].tolist())
    if q_out is not None:
        over = ((q_out.double() - q_want).abs() - U[q_out.dtype] * q_want.abs() - SUB[q_out.dtype]).max().item()
        assert over <= 0, over


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,n_q,hd,page,lens,counts", [
    (4, 28, 128, 64, [1000], [1]),
    (2, 8, 64, 16, [0, 15, 16, 17, 31], [1, 1, 1, 3, 0]),
    (3, 6, 128, 32, [5, 0, 100], [70, 129, 31]),
    (2, 2, 128, 128, [0, 200, 127], [128, 300, 2]),
    (1, 4, 64, 64, [63, 64], [1, 64]),
    (2, 4, 64, 128, [1], [260]),
], ids=["one-token", "p16", "p32", "p128", "p64-hd64", "p128-hd64"])
def test_append(ops, dtype, n_kv, n_q, hd, page, lens, counts):
    g = gen(3)
    n_seq, n = len(lens), sum(counts)
    most = max(1, max(-(-(a + b) // page) for a, b in zip(lens, counts)))
    c = finite_codes(make_cache(ops, n_seq, n_kv, hd, page, most))
    qkv = torch.randn((n, n_q + 2 * n_kv, hd), generator=g, device="cuda").to(dtype)
    if n > 2:
        qkv[n // 2] *= 64  # a row that makes its pages' scales grow
        qkv[1] = 0
    q, k, v = qkv[:, :n_q], qkv[:, n_q : n_q + n_kv], qkv[:, n_q + n_kv :]
    off = np.cumsum([0] + counts).tolist()
    rope = rope_table(most * page, hd)
    want = ref_append(c, k, v, off, lens, None, rope)
    at = torch.tensor([lens[s] + i for s in range(n_seq) for i in range(counts[s])], device="cuda")
    q_out, status = torch.zeros((n, n_q, hd), dtype=dtype, device="cuda"), ints([0])
    for _ in range(2):  # the second time the rows are rewritten: the same rows give the same cache
        ops.kv_append(c, k, v, ints(off), ints(lens), max_rows=max(counts), rope=rope, q=q, q_out=q_out, status=status)
        check_append(c, want, q_out, rotated(q, rope[at]))
    assert int(status) == 0


@pytest.mark.parametrize("lens,pos", [
    ([40], [[0, 1, 5, 15, 16, 33, 39]]),               # rewrites inside a filled sequence
    ([10, 0, 64], [[3, 9, 10, 11], [0, 40, 41], []]),  # rewrites and appends, a hole, nothing
    ([48], [list(range(16, 32))]),                     # a whole page: its scale may shrink
    ([47], [list(range(32, 47))]),                     # all that is filled of a page
])
def test_append_at_positions(ops, lens, pos):
    g = gen(5)
    n_kv, hd, page = 2, 64, 16
    counts = [len(p) for p in pos]
    n = sum(counts)
    flat = [p for x in pos for p in x]
    c = finite_codes(make_cache(ops, len(lens), n_kv, hd, page, 5))
    k, v = (torch.randn((n, n_kv, hd), generator=g, device="cuda", dtype=torch.float32) * s for s in (0.01, 50.0))
    off = np.cumsum([0] + counts).tolist()
    want = ref_append(c, k, v, off, lens, flat, None)
    status = ints([0])
    ops.kv_append(c, k, v, ints(off), ints(lens), max_rows=max(counts), pos=ints(flat), status=status)
    check_append(c, want)
    assert int(status) == 0


def test_append_layouts(ops):
    """Head-major rows, rows at odd element offsets and strides, in-place rotation of q, uint8 and float8 pools."""
    g = gen(6)
    n, n_kv, n_q, hd, page = 37, 2, 4, 64, 32
    rope = rope_table(64, hd)
    for dtype, shift in ((torch.bfloat16, 0), (torch.bfloat16, 1), (torch.float32, 3), (torch.float16, 8)):
        c = finite_codes(make_cache(ops, 1, n_kv, hd, page, 2))
        f = ops.PagedKV(c.k.clone().view(torch.float8_e4m3fn), c.v.clone().view(torch.float8_e4m3fn), c.k_scale.clone(), c.v_scale.clone(), c.pages)
        base = torch.randn(shift + 3 * n * (n_kv * (hd + 5)), generator=g, device="cuda").to(dtype)
        k = base[shift:].as_strided((n, n_kv, hd), (hd + 5, n * (hd + 5), 1), shift)  # [head][row][hd + 5]
        v = base.as_strided((n, n_kv, hd), (n_kv * (hd + 3), hd + 3, 1), n * n_kv * (hd + 5))
        q = torch.randn((n, n_q, hd), generator=g, device="cuda").to(dtype)
        want = ref_append(c, k, v, [0, n], [3], None, rope)
        q_want = rotated(q, rope[3 : 3 + n])
        ops.kv_append(c, k, v, ints([0, n]), ints([3]), max_rows=n, rope=rope, q=q, q_out=q)
        check_append(c, want, q, q_want)
        ops.kv_append(f, k, v, ints([0, n]), ints([3]), max_rows=n, rope=rope)
        check_append(ops.PagedKV(f.k.view(torch.uint8), f.v.view(torch.uint8), f.k_scale, f.v_scale, f.pages), want)


def test_append_borders(ops):
    """Rotated values on and next to the borders of two codes: the exact value decides."""
    hd, page = 128, 64
    g = gen(8)
    n = 64
    rope = rope_table(64, hd)
    # first halves that rotate onto borders m + 1/2 steps, solved in 64 bits and rounded to f32: the
    # exact product lies a few 2^-26 beside the border, either way
    target = (torch.randint(8, 16, (n, 1, hd // 2), generator=g, device="cuda").double() + 0.5) * 8
    b = torch.randn((n, 1, hd // 2), generator=g, device="cuda")
    a = ((target + b.double() * rope[:n, None, :, 1].double()) / rope[:n, None, :, 0].double()).float()
    k = torch.cat([a, b], -1).contiguous().clamp_(-400, 400)
    v = torch.randn((n, 1, hd), generator=g, device="cuda")
    c = finite_codes(make_cache(ops, 1, 1, hd, page, 1))
    want = ref_append(c, k, v, [0, n], [0], None, rope)
    ops.kv_append(c, k, v, ints([0, n]), ints([0]), max_rows=n, rope=rope)
    check_append(c, want)


def test_append_extremes(ops):
    """Zeros, the smallest and largest f32, amax exactly at 448 * 2^e, NaN and infinities."""
    hd, page = 64, 16
    rows = torch.zeros((6, 1, hd), device="cuda")
    rows[1, 0, 0] = 3.5          # 448 * 2^-7: e = -7 exactly
    rows[2, 0, 0] = 3.5000002    # just above: e = -6
    rows[3, 0, 3] = 1e-40
    rows[4, 0, 5] = -3.4e38
    rows[5, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 2.0])
    for i in range(6):
        c = finite_codes(make_cache(ops, 1, 1, hd, page, 1))
        x = rows[i : i + 1]
        clean = x.clone()
        clean[~clean.isfinite()] = 0
        want = ref_append(c, clean, clean, [0, 1], [0], None, None)
        if i == 5:
            for t in want[:2]:
                t[c.pages[0, 0].long(), 0, 0, :4] = torch.tensor([0, 0x7E, 0xFE, int(nearest(torch.tensor([448.0], dtype=torch.float64, device="cuda") * 0 + 2.0 * 2.0**7))], dtype=torch.uint8, device="cuda")
        status = ints([0])
        ops.kv_append(c, x, x, ints([0, 1]), ints([0]), max_rows=1, status=status)
        check_append(c, want)
        assert int(status) == (ops.STAT_NONFINITE if i == 5 else 0)


def test_append_bad_device_values(ops):
    """Values in device memory that cannot be used: reported, and nothing else is written."""
    n_kv, hd, page = 1, 64, 16
    k = torch.randn((8, n_kv, hd), generator=gen(1), device="cuda")

    def run(off, lens, pos=None, pages=None, rope=None, max_rows=8):
        c = finite_codes(make_cache(ops, len(lens), n_kv, hd, page, 2))
        if pages is not None:
            c.set_pages(ints(pages))
        before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
        status = ints([0])
        ops.kv_append(c, k, k, ints(off), ints(lens), max_rows=max_rows, pos=None if pos is None else ints(pos), rope=rope, status=status)
        return c, before, int(status)

    def same(c, before):
        return all(bool((a == b).all()) for a, b in zip((c.k, c.v, c.k_scale, c.v_scale), before))

    c, before, st = run([0, 8], [0], pages=[[99, 1]])
    assert st == ops.STAT_PAGE and same(c, before)
    c, before, st = run([0, 8], [0], pages=[[-1, 1]])
    assert st == ops.STAT_PAGE and same(c, before)
    for lens in ([-3], [33], [2**31 - 1], [-(2**31)]):
        c, before, st = run([0, 8], lens)
        assert st == ops.STAT_POSITION and same(c, before)
    c, before, st = run([0, 8], [28])  # four rows fit
    want = ref_append(c, k, k, [0, 4], [28], None, None)
    assert st == ops.STAT_POSITION and bool((c.k[c.pages[0, 1].long(), :, 12:] == want[0][c.pages[0, 1].long(), :, 12:]).all())
    c, before, st = run([5, 3], [0])
    assert st == ops.STAT_ROWS and same(c, before)
    c, before, st = run([0, 9], [0])
    assert st == ops.STAT_ROWS
    c, before, st = run([0, 8], [0], max_rows=3)
    assert st == ops.STAT_ROWS and bool((c.k[c.pages[0, 0].long(), :, 3:] == before[0][c.pages[0, 0].long(), :, 3:]).all())
    # positions that repeat, run backwards or leave the tables
    for pos in ([0, 1, 2, 2, 3, 4, 5, 6], [0, 5, 4, 6, 7, 8, 9, 10], [-2, 0, 1, 2, 3, 4, 5, 6], [0, 1, 2, 3, 4, 5, 6, 40], [2**31 - 1] * 8, [-(2**31)] * 8):
        c, before, st = run([0, 8], [0], pos=pos)
        assert st == ops.STAT_POSITION
    # the rotation table ends before the positions do
    c, before, st = run([0, 8], [0], rope=rope_table(5, hd))
    assert st == ops.STAT_POSITION and bool((c.k[c.pages[0, 0].long(), :, 5:] == before[0][c.pages[0, 0].long(), :, 5:]).all())


# ── attention ──


def ref_attention(c, q, off, lens, vis, scale):
    """(out, lse, bound on out, bound on lse) in 64 bits."""
    n, n_q, hd = q.shape
    rep = n_q // c.n_kv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((n, n_q), -math.inf, dtype=torch.float64, device="cuda")
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for s, m in enumerate(lens):
        a, b = off[s], off[s + 1]
        if a == b or m == 0:
            continue
        ids = c.pages[s, : -(-m // c.page)].long()
        k, v = ((value(x[ids].view(torch.uint8)) * f[ids].double()[..., None, None]).transpose(0, 1).reshape(c.n_kv, -1, hd)[:, :m].repeat_interleave(rep, 0)
                for x, f in ((c.k, c.k_scale), (c.v, c.v_scale)))
        qq = q[a:b].double().transpose(0, 1)  # [n_q][rows][hd]
        x = qq @ k.transpose(1, 2) * scale
        ds = (hd + 4) * 2.0**-24 * abs(scale) * (qq.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True)
        if vis is not None:
            see = torch.tensor(vis[a:b], device="cuda")
            x = torch.where(torch.arange(m, device="cuda")[None, None] < see[None, :, None], x, -math.inf)
        lz = torch.logsumexp(x, -1, keepdim=True)
        p = torch.where(lz.isinf(), 0.0, torch.exp(x - lz))
        o = p @ v
        S = p @ v.abs()
        t = U[q.dtype] * o.abs() + SUB[q.dtype] + (2.0**-11 + 2 * ds + m * 2.0**-24 + 2.0**-20) * S + m * 2.0**-24 * v.abs().amax((1, 2))[:, None, None] * p.amax(-1, keepdim=True)
        out[a:b], tol[a:b] = o.transpose(0, 1), t.transpose(0, 1)
        lse[a:b] = lz[..., 0].transpose(0, 1)
        ltol[a:b] = (ds + m * 2.0**-24 + 2.0**-20 * (1 + lz.abs().nan_to_num(0, 0, 0)))[..., 0].transpose(0, 1)
    return out, lse, tol, ltol


def check_attention(ops, c, q, off, lens, vis=None, scale=None, max_rows=None, max_keys=None, **kw):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    status = ints([0])
    out, lse = ops.kv_attention(c, q, ints(off), ints(lens), max_rows=max_rows or max(b - a for a, b in zip(off, off[1:])),
                                max_keys=max(lens) if max_keys is None else max_keys, scale=scale,
                                vis=None if vis is None else ints(vis), return_lse=True, status=status, **kw)
    assert int(status) == 0
    ref, rl, tol, ltol = ref_attention(c, q, off, lens, vis, scale)
    err = (out.double() - ref).abs()
    if q.dtype == torch.float16:  # from 65520 on (half a step above 65504) f16's nearest value is inf
        err = torch.where((out.double() == ref.sign() * math.inf) & (ref.abs() + tol >= 65520), 0.0, err)
    over = (err - tol).max().item()
    assert over <= 0, over
    none = rl.isinf()
    assert bool((lse[none] == -math.inf).all()) and bool((out[none] == 0).all())
    le = (lse.double() - rl).abs()[~none]
    assert bool((le <= ltol[~none]).all()), float((le - ltol[~none]).max())
    return out, lse


def kill_tail(c, lens):
    """Live positions hold numbers; positions behind a sequence's length NaN codes."""
    finite_codes(c)
    for s, m in enumerate(lens):
        for pg in range(c.pages.shape[1]):
            dead = max(0, min(c.page, m - pg * c.page))
            for t in (c.k, c.v):
                t[c.pages[s, pg].long(), :, dead:] = 0x7F
    return c


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("n_kv,n_q,hd,page,lens,counts", [
    (4, 28, 128, 64, [461], [1]),
    (2, 2, 64, 16, [1, 16, 17, 0, 33], [1, 2, 3, 4, 5]),
    (1, 7, 128, 32, [95, 31, 200], [9, 31, 100]),
    (3, 3, 128, 128, [129, 1, 384], [129, 1, 17]),
    (2, 16, 64, 64, [70, 300], [33, 16]),
    (1, 1, 128, 64, [640], [300]),
    (1, 1, 64, 16, [1], [1]),
    (4, 28, 128, 64, [5000, 1], [1, 1]),
    (1, 32, 64, 32, [1000], [130]),
    (5, 10, 128, 64, [1500, 3, 0, 900, 128, 129] * 7, [260, 3, 2, 70, 129, 40] * 7),
], ids=["decode", "tiny-p16", "gqa7-p32", "mha-p128", "gqa8-hd64", "long-rows", "one-one", "decode-2", "mqa32", "many-items"])
def test_attention(ops, dtype, n_kv, n_q, hd, page, lens, counts):
    most = max(1, max(-(-m // page) for m in lens))
    c = kill_tail(make_cache(ops, len(lens), n_kv, hd, page, most, seed=7), lens)
    q = torch.randn((sum(counts), n_q, hd), generator=gen(2), device="cuda").to(dtype)
    off = np.cumsum([0] + counts).tolist()
    out, lse = check_attention(ops, c, q, off, lens)
    # the same call again: the same bits
    again = ops.kv_attention(c, q, ints(off), ints(lens), max_rows=max(counts), max_keys=max(lens), return_lse=True)
    assert bool((again[0] == out).all()) and bool((again[1] == lse).all())


@pytest.mark.parametrize("rows,keys", [(1, 300), (40, 700), (150, 1000)])
def test_attention_visible_keys(ops, rows, keys):
    g = gen(4)
    c = kill_tail(make_cache(ops, 2, 2, 128, 64, -(-keys // 64), seed=1), [keys, keys - 5])
    q = torch.randn((2 * rows, 6, 128), generator=g, device="cuda").to(torch.bfloat16)
    off = [0, rows, 2 * rows]
    lens = [keys, keys - 5]
    causal = [m - rows + t + 1 for m in lens for t in range(rows)]
    check_attention(ops, c, q, off, lens, vis=causal)
    random = torch.randint(0, keys + 9, (2 * rows,), generator=g, device="cuda").tolist()  # beyond the length: all keys
    random[0] = 0
    random[-1] = 1
    check_attention(ops, c, q, off, lens, vis=random)
    none = [0] * (2 * rows)
    out, lse = ops.kv_attention(c, q, ints(off), ints(lens), max_rows=rows, max_keys=keys, vis=ints(none), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("rows", [1, 20, 140])
def test_attention_scales_apart(ops, rows):
    """Scales of different pages many powers of two apart, large scores, a large and a negative softmax scale."""
    g = gen(9)
    lens = [500]
    c = kill_tail(make_cache(ops, 1, 2, 128, 32, 16, seed=2), lens)
    c.v_scale.copy_(torch.exp2(torch.randint(-40, 20, c.v_scale.shape, generator=g, device="cuda").float()))
    c.k_scale.copy_(torch.exp2(torch.randint(-20, -4, c.k_scale.shape, generator=g, device="cuda").float()))
    q = torch.randn((rows, 4, 128), generator=g, device="cuda").half()
    check_attention(ops, c, q, [0, rows], lens)
    check_attention(ops, c, q, [0, rows], lens, scale=-0.3)
    check_attention(ops, c, (q * 2.0**-12), [0, rows], lens, scale=300.0)
    big = (torch.randn((rows, 4, 128), generator=g, device="cuda") * 2.0**30).bfloat16()
    check_attention(ops, c, big, [0, rows], lens, scale=2.0**-33)
    check_attention(ops, c, q, [0, rows], lens, scale=0.0)


def test_attention_layouts(ops):
    """Head-major q and out, rows at odd offsets, bounds larger than needed, a caller's workspace."""
    g = gen(10)
    n, n_q, hd = 21, 4, 128
    lens = [333]
    c = kill_tail(make_cache(ops, 1, 2, hd, 64, 6, seed=3), lens)
    base = torch.randn(n * n_q * (hd + 1) + 9, generator=g, device="cuda").half()
    q = base.as_strided((n, n_q, hd), (hd + 1, n * (hd + 1), 1), 3)
    out = torch.full((n_q, n + 2, hd + 3), 7.0, dtype=torch.float16, device="cuda")
    view = out[:, 1 : n + 1, 1 : hd + 1].transpose(0, 1)
    got, _ = check_attention(ops, c, q, [0, n], lens, out=view)
    edge = out.clone()
    edge[:, 1 : n + 1, 1 : hd + 1] = 7.0
    assert bool((edge == 7.0).all())
    need = ops.kv_attention_workspace(c, n_q=n_q, n_rows=n, max_rows=50, max_keys=384)
    ws = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    check_attention(ops, c, q, [0, n], lens, max_rows=50, max_keys=384, workspace=ws)
    assert bool((ws[need:] == 0xAB).all())


def test_attention_bad_device_values(ops):
    g = gen(11)
    n = 6
    c = kill_tail(make_cache(ops, 1, 2, 64, 16, 4, seed=4), [64])
    q = torch.randn((n, 4, 64), generator=g, device="cuda").half()

    def run(off, lens, max_rows=n, max_keys=64):
        st = ints([0])
        out, lse = ops.kv_attention(c, q, ints(off), ints(lens), max_rows=max_rows, max_keys=max_keys, return_lse=True, status=st,
                                    out=torch.full_like(q, 3.0))
        return out, lse, int(st)

    assert run([0, n], [65], max_keys=65)[2] == ops.STAT_POSITION   # beyond the table
    assert run([0, n], [64], max_keys=40)[2] == ops.STAT_POSITION   # beyond the bound
    out, lse, st = run([0, n], [-1])
    assert st == ops.STAT_POSITION and bool((out == 0).all())
    assert run([0, 7], [64])[2] == ops.STAT_ROWS
    out, _, st = run([4, 2], [64])
    assert st == ops.STAT_ROWS and bool((out == 3.0).all())
    out, _, st = run([0, n], [64], max_rows=2)
    assert st == ops.STAT_ROWS and bool((out[2:] == 3.0).all())
    # a bad page: its keys are left out
    pages = c.pages.clone()
    bad = pages.clone()
    bad[0, 1] = c.n_pages
    c.set_pages(bad)
    out, lse, st = run([0, n], [64])
    assert st == ops.STAT_PAGE
    kept = pages[:, [0, 2, 3]].contiguous()
    c.set_pages(kept)
    ref, rl, tol, ltol = ref_attention(c, q, [0, n], [48], None, 64**-0.5)
    assert bool(((out.double() - ref).abs() <= tol).all()) and bool(((lse.double() - rl).abs() <= ltol).all())


# Calls of many rows take large row tiles only where many sequences or a large bound of the keys make them
# pay: the same scenarios with them, the key axis split (a large max_keys) and whole (many sequences).
FAR = 200_000


@pytest.mark.parametrize("split", [True, False], ids=["split", "whole"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("n_kv,n_q,hd,page,lens,counts", [
    (1, 7, 128, 32, [95, 31, 200], [9, 31, 100]),
    (3, 3, 128, 128, [129, 1, 384], [129, 1, 17]),
    (2, 16, 64, 64, [70, 300, 0], [33, 16, 2]),
    (1, 1, 128, 64, [640], [300]),
    (1, 32, 64, 16, [1000, 17], [13, 40]),
    (2, 8, 128, 16, [1, 700], [70, 0]),
], ids=["gqa7-p32", "mha-p128", "gqa8-hd64", "long-rows", "mqa32-p16", "one-key"])
def test_attention_large_tiles(ops, split, dtype, n_kv, n_q, hd, page, lens, counts):
    times = 1 if split else -(-160 // (n_kv * len(lens)))
    lens, counts = lens * times, counts * times
    most = max(1, max(-(-m // page) for m in lens))
    c = kill_tail(make_cache(ops, len(lens), n_kv, hd, page, most, seed=17), lens)
    q = torch.randn((sum(counts), n_q, hd), generator=gen(12), device="cuda").to(dtype)
    off = np.cumsum([0] + counts).tolist()
    bound = FAR if split else max(lens)
    out, lse = check_attention(ops, c, q, off, lens, max_keys=bound)
    again = ops.kv_attention(c, q, ints(off), ints(lens), max_rows=max(counts), max_keys=bound, return_lse=True)
    assert bool((again[0] == out).all()) and bool((again[1] == lse).all())


@pytest.mark.parametrize("split", [True, False], ids=["split", "whole"])
def test_attention_large_tiles_visible_keys(ops, split):
    g = gen(14)
    n_seq, rows, keys, n_kv = (2, 150, 1000, 2) if split else (40, 40, 300, 2)
    lens = [keys - 5 * (i % 2) for i in range(n_seq)]
    c = kill_tail(make_cache(ops, n_seq, n_kv, 128, 64, -(-keys // 64), seed=11), lens)
    q = torch.randn((n_seq * rows, 3 * n_kv, 128), generator=g, device="cuda").to(torch.bfloat16)
    off = [rows * i for i in range(n_seq + 1)]
    bound = FAR if split else keys
    check_attention(ops, c, q, off, lens, vis=[m - rows + t + 1 for m in lens for t in range(rows)], max_keys=bound)
    random = torch.randint(0, keys + 9, (n_seq * rows,), generator=g, device="cuda").tolist()
    random[0], random[-1] = 0, 1
    check_attention(ops, c, q, off, lens, vis=random, max_keys=bound)
    out, lse = ops.kv_attention(c, q, ints(off), ints(lens), max_rows=rows, max_keys=bound, vis=ints([0] * (n_seq * rows)), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_attention_large_tiles_scales_apart(ops):
    g, rows, lens = gen(19), 140, [500]
    c = kill_tail(make_cache(ops, 1, 2, 128, 32, 16, seed=12), lens)
    c.v_scale.copy_(torch.exp2(torch.randint(-40, 20, c.v_scale.shape, generator=g, device="cuda").float()))
    c.k_scale.copy_(torch.exp2(torch.randint(-20, -4, c.k_scale.shape, generator=g, device="cuda").float()))
    q = torch.randn((rows, 4, 128), generator=g, device="cuda").half()
    for x, scale in ((q, None), (q, -0.3), (q * 2.0**-12, 300.0), (q, 0.0)):
        check_attention(ops, c, x, [0, rows], lens, scale=scale, max_keys=FAR)
    big = (torch.randn((rows, 4, 128), generator=g, device="cuda") * 2.0**30).bfloat16()
    check_attention(ops, c, big, [0, rows], lens, scale=2.0**-33, max_keys=FAR)


def test_attention_large_tiles_layouts_and_bad_values(ops):
    g, n, n_q, hd = gen(20), 70, 4, 128
    lens = [333]
    c = kill_tail(make_cache(ops, 1, 2, hd, 64, 6, seed=13), lens)
    base = torch.randn(n * n_q * (hd + 1) + 9, generator=g, device="cuda").half()
    q = base.as_strided((n, n_q, hd), (hd + 1, n * (hd + 1), 1), 3)
    out = torch.full((n_q, n + 2, hd + 3), 7.0, dtype=torch.float16, device="cuda")
    check_attention(ops, c, q, [0, n], lens, out=out[:, 1 : n + 1, 1 : hd + 1].transpose(0, 1), max_keys=FAR)
    edge = out.clone()
    edge[:, 1 : n + 1, 1 : hd + 1] = 7.0
    assert bool((edge == 7.0).all())
    q = q.contiguous()

    def run(off, lens, max_rows=n):
        st = ints([0])
        out, lse = ops.kv_attention(c, q, ints(off), ints(lens), max_rows=max_rows, max_keys=FAR, return_lse=True, status=st, out=torch.full_like(q, 3.0))
        return out, lse, int(st)

    assert run([0, n], [400])[2] == ops.STAT_POSITION
    out, lse, st = run([0, n], [-1])
    assert st == ops.STAT_POSITION and bool((out == 0).all()) and bool((lse == -math.inf).all())
    out, _, st = run([40, 20], [333])
    assert st == ops.STAT_ROWS and bool((out == 3.0).all())
    out, _, st = run([0, n], [333], max_rows=50)
    assert st == ops.STAT_ROWS and bool((out[50:] == 3.0).all())
    pages = c.pages.clone()
    bad = pages.clone()
    bad[0, 1] = -1
    c.set_pages(bad)
    out, lse, st = run([0, n], [320])
    assert st == ops.STAT_PAGE
    c.set_pages(pages[:, [0, 2, 3, 4]].contiguous())
    ref, rl, tol, ltol = ref_attention(c, q, [0, n], [256], None, hd**-0.5)
    assert bool(((out.double() - ref).abs() <= tol).all()) and bool(((lse.double() - rl).abs() <= ltol).all())


def test_attention_no_keys_at_all(ops):
    for rows, bound in ((3, 0), (90, 0), (90, FAR)):
        c = make_cache(ops, 2, 2, 64, 16, 2, seed=21)
        q = torch.randn((2 * rows, 4, 64), generator=gen(22), device="cuda").half()
        out, lse = ops.kv_attention(c, q, ints([0, rows, 2 * rows]), ints([0, 0]), max_rows=rows, max_keys=bound, return_lse=True)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_outputs_and_workspace_on_a_given_stream(ops):
    """Memory that a call allocates belongs to the stream it runs on: work on the current stream right after
    the call may not be given its workspace."""
    side = torch.cuda.Stream()
    lens, rows = [20000], 64
    c = kill_tail(make_cache(ops, 1, 2, 128, 64, 313, seed=23), lens)
    q = torch.randn((rows, 4, 128), generator=gen(24), device="cuda").half()
    off, ln = ints([0, rows]), ints(lens)
    x = torch.randn((40, 30000), generator=gen(25), device="cuda")
    want = ops.kv_attention(c, q, off, ln, max_rows=rows, max_keys=20000)
    ref = ops.token_logprobs(x, top_k=9)
    torch.cuda.synchronize()
    need = ops.kv_attention_workspace(c, n_q=4, n_rows=rows, max_rows=rows, max_keys=20000)
    for _ in range(20):
        got = ops.kv_attention(c, q, off, ln, max_rows=rows, max_keys=20000, stream=side.cuda_stream)
        lp = ops.token_logprobs(x, top_k=9, stream=side.cuda_stream)
        torch.empty(need, dtype=torch.uint8, device="cuda").fill_(0xFF)
        side.synchronize()
        assert bool((got == want).all()) and bool((lp[1] == ref[1]).all()) and bool((lp[2] == ref[2]).all())


# ── log probabilities ──


def check_logprobs(ops, logits, targets, k, rows=None):
    status = ints([0])
    lp, ent, ids, top = ops.token_logprobs(logits, None if targets is None else ints(targets), top_k=k, rows=None if rows is None else ints(rows), status=status)
    x = (logits if rows is None else logits[torch.tensor(rows, device="cuda")]).double()
    n, V = x.shape
    m = x.amax(-1, keepdim=True)
    # (x - m) - log sum exp(x - m): m + log(...) would lose the logarithm beside logits of 1e38
    p = torch.where(m.isinf(), -math.inf, (x - m) - (x - m).exp().sum(-1, keepdim=True).log())
    p = torch.where(p < -torch.finfo(torch.float32).max, -math.inf, p)  # f32 has no such value
    tol = lambda y: (V / 128 + 16) * 2.0**-24 * (1 + (m - y).abs().nan_to_num(0, 0, 0) + math.log(V))  # noqa: E731
    if targets is not None:
        t = torch.tensor(targets, device="cuda")
        want = torch.where(t < 0, 0.0, p.gather(1, t.clamp_min(0)[:, None])[:, 0])
        inf = want.isinf()
        assert bool((lp[inf] == -math.inf).all())
        assert bool(((lp.double() - want).abs() <= tol(x.gather(1, t.clamp_min(0)[:, None]))[:, 0])[~inf].all())
    h = -torch.special.xlogy(p.exp(), p.exp()).sum(-1)
    live = torch.where(p > -80, m - x, 0.0).amax(-1, keepdim=True).nan_to_num(0, 0, 0)
    assert bool(((ent.double() - h).abs() <= tol(x * 0 + m).nan_to_num(0, 0, 0).amax(-1) * (1 + live[:, 0])).all()), float((ent.double() - h).abs().max())
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
    assert bool((ids == order).all())
    want = p.gather(1, order)
    inf = want.isinf()
    assert bool((top[inf] == -math.inf).all()) and bool(((top.double() - want).abs() <= tol(x.gather(1, order)))[~inf].all())
    assert int(status) == 0
    return lp, ent, ids, top


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (3, 7, 7), (5, 32, 32), (2, 31, 0), (4, 1000, 20), (9, 4097, 5), (1, 126464, 32), (300, 5000, 8), (2, 152064, 1)])
def test_logprobs(ops, dtype, n, V, k):
    g = gen(V + n)
    x = (torch.randn((n, V), generator=g, device="cuda") * 4).to(dtype)
    t = torch.randint(-1, V, (n,), generator=g, device="cuda").tolist()
    check_logprobs(ops, x, t, k)
    check_logprobs(ops, x, None, k)


def test_logprobs_orders(ops):
    """Values in ascending and descending order, all equal, two values, a plateau across the row: ranks and ties."""
    V = 20000
    up = torch.arange(V, device="cuda", dtype=torch.float32) * 1e-3
    rows = torch.stack([up, up.flip(0), torch.zeros(V, device="cuda"), (torch.arange(V, device="cuda") % 2).float(), (up * 0.5).floor(),
                        -up, torch.where(torch.arange(V, device="cuda") % 777 == 5, 3.0, -2.0), torch.zeros(V, device="cuda")])
    rows[7, 1::2] = -0.0  # a zero is a zero
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        check_logprobs(ops, rows.to(dtype), [0, V - 1, 5, 7, 9, 1, 782, 3], 32)


def test_logprobs_masks(ops):
    """-inf logits, rows of -inf alone, a single live token, huge and tiny logits."""
    g = gen(3)
    V = 3001
    x = torch.randn((7, V), generator=g, device="cuda")
    x[0, torch.rand(V, generator=g, device="cuda") < 0.999] = -math.inf
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, 1234] = -5.0
    x[3] = -3.0e38
    x[3, 17] = 3.0e38
    x[4] = 1e-30
    x[5, 40] = 60.0
    x[6] = torch.finfo(torch.float32).min
    check_logprobs(ops, x, [3, 5, 1234, 17, -1, 41, 2], 9)


def test_logprobs_rows_and_strides(ops):
    g = gen(5)
    base = torch.randn((50, 1111 + 9), generator=g, device="cuda")
    for dtype, a in ((torch.float32, 1), (torch.float32, 4), (torch.float16, 3), (torch.bfloat16, 8)):
        x = base.to(dtype)[:, a : a + 1101]
        check_logprobs(ops, x, [1, 2, 3, 1100], 5, rows=[49, 0, 7, 7])
        check_logprobs(ops, x, list(range(50)), 3)


def test_logprobs_bad_rows(ops):
    x = torch.randn((6, 400), generator=gen(1), device="cuda")
    x[1, 77] = math.nan
    x[2, 3] = math.inf
    good = ops.token_logprobs(x[3:4].contiguous(), ints([9]), top_k=4)
    st = ints([0])
    lp, ent, ids, top = ops.token_logprobs(x, ints([0, 1, 2, 9, 1, 1]), top_k=4, status=st)
    assert int(st) == ops.STAT_LOGITS
    for r in (1, 2):
        assert bool(lp[r].isnan()) and bool(ent[r].isnan()) and bool((ids[r] == -1).all()) and bool(top[r].isnan().all())
    assert float(lp[3]) == float(good[0]) and bool((ids[3] == good[2][0]).all())
    st = ints([0])
    lp, ent, ids, top = ops.token_logprobs(x, ints([400, 9]), top_k=2, rows=ints([0, 3]), status=st)
    assert int(st) == ops.STAT_TARGET and bool(lp[0].isnan()) and float(lp[1]) == float(good[0]) and bool(ent[0].isfinite())
    st = ints([0])
    lp, ent, ids, top = ops.token_logprobs(x, ints([3, 9, 3]), top_k=2, rows=ints([6, 3, -1]), status=st)
    assert int(st) == ops.STAT_TARGET
    for r in (0, 2):
        assert bool(lp[r].isnan()) and bool(ent[r].isnan()) and bool((ids[r] == -1).all())
    assert float(lp[1]) == float(good[0])


# ── together ──


def test_block_step_graph_and_streams(ops):
    """A denoising block's step as a program runs it: rotate and store the block's rows behind its
    prompt, attend, score; eagerly, on another stream, and captured into a graph that is replayed on
    new inputs."""
    g = gen(12)
    n_kv, n_q, hd, page, V, n = 2, 4, 128, 64, 5000, 32
    lens0 = [100, 37]
    c = kill_tail(make_cache(ops, 2, n_kv, hd, page, 3, seed=6), lens0)
    rope = rope_table(192, hd)
    off, lens, total = ints([0, n, 2 * n]), ints(lens0), ints([m + n for m in lens0])
    qkv = torch.empty((2 * n, n_q + 2 * n_kv, hd), dtype=torch.bfloat16, device="cuda")
    w = torch.randn((n_q * hd, V), generator=g, device="cuda").bfloat16() * 0.05
    q_out = torch.empty((2 * n, n_q, hd), dtype=torch.bfloat16, device="cuda")
    att = torch.empty_like(q_out)
    targets = torch.randint(0, V, (2 * n,), generator=g, device="cuda").to(torch.int32)
    ws = torch.empty(max(1, ops.kv_attention_workspace(c, n_q=n_q, n_rows=2 * n, max_rows=n, max_keys=192)), dtype=torch.uint8, device="cuda")
    status = ints([0])

    def step():
        q, k, v = qkv[:, :n_q], qkv[:, n_q : n_q + n_kv], qkv[:, n_q + n_kv :]
        ops.kv_append(c, k, v, off, lens, max_rows=n, rope=rope, q=q, q_out=q_out, status=status)
        ops.kv_attention(c, q_out, off, total, max_rows=n, max_keys=192, out=att, workspace=ws, status=status)
        return ops.token_logprobs(att.view(2 * n, -1) @ w, targets, top_k=4, status=status)

    def inputs(seed):
        qkv.copy_(torch.randn(qkv.shape, generator=gen(seed), device="cuda").to(qkv.dtype))

    def keep(r):
        return [t.clone() for t in r] + [c.k.clone(), c.v.clone(), c.k_scale.clone(), att.clone()]

    start = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]

    def rewind():
        for t, s in zip((c.k, c.v, c.k_scale, c.v_scale), start):
            t.copy_(s)

    eager = []
    for seed in (1, 2):
        rewind()
        inputs(seed)
        eager.append(keep(step()))
    check_attention(ops, c, q_out, [0, n, 2 * n], [m + n for m in lens0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rewind()
        inputs(1)
        got = keep(step())
    torch.cuda.current_stream().wait_stream(side)
    assert all(bool((a == b).all()) for a, b in zip(got, eager[0]))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        res = step()
    for seed in (2, 1):
        rewind()
        inputs(seed)
        graph.replay()
        assert all(bool((a == b).all()) for a, b in zip(keep(res), eager[seed - 1]))
    assert int(status) == 0
