"""Operators on device tensors (include/diffuse_b200.h): the paged 8-bit K/V cache and the
token log probabilities.

Tensors are torch CUDA tensors of one GPU.  A call launches on the current stream of that GPU (or
on `stream`, a raw cudaStream_t) and does not wait for it; it can be captured into a CUDA graph.
Shapes, types and host values are checked here and in the library (DiffuseError / ValueError);
values in device memory are checked by the kernels, which skip what they cannot use and OR
`STAT_*` bits into `status` (an int32 tensor of one element, zeroed by the caller), if given.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import BF16, F16, F32, DiffuseError, native

(STAT_PAGE, STAT_POSITION, STAT_ROWS, STAT_NONFINITE, STAT_TARGET, STAT_LOGITS, STAT_TIMEOUT) = (1, 2, 4, 8, 16, 32, 64)

_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_P, _I32, _I64 = C.c_void_p, C.c_int32, C.c_int64
_MAX_WS = 64  # workspace sizes a cache remembers: a decoding loop's bound of the keys is another one at each step


class _KvCache(C.Structure):
    _fields_ = [("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("pages", _P), ("n_pages", _I32), ("n_kv", _I32),
                ("head_dim", _I32), ("page", _I32), ("n_seq", _I32), ("max_pages", _I32)]


class _KvRows(C.Structure):
    _fields_ = [("k", _P), ("v", _P), ("type", _I32), ("n_rows", _I32), ("max_rows", _I32), ("k_tok", _I64), ("k_head", _I64),
                ("v_tok", _I64), ("v_head", _I64), ("row_off", _P), ("len", _P), ("pos", _P), ("rope", _P), ("n_rope", _I32),
                ("n_q", _I32), ("q", _P), ("q_out", _P), ("q_tok", _I64), ("q_head", _I64), ("q_out_tok", _I64),
                ("q_out_head", _I64)]


class _KvAttn(C.Structure):
    _fields_ = [("q", _P), ("out", _P), ("type", _I32), ("n_q", _I32), ("n_rows", _I32), ("max_rows", _I32),
                ("max_keys", _I32), ("scale", C.c_float), ("q_tok", _I64), ("q_head", _I64), ("out_tok", _I64),
                ("out_head", _I64), ("row_off", _P), ("len", _P), ("vis", _P), ("lse", _P)]


class _Logprobs(C.Structure):
    _fields_ = [("logits", _P), ("type", _I32), ("n_vocab", _I32), ("n_rows", _I32), ("n_logits", _I32), ("ld", _I64),
                ("rows", _P), ("targets", _P), ("logprob", _P), ("entropy", _P), ("top_k", _I32), ("top_ids", _P),
                ("top_logprob", _P)]


_fns = {}


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = getattr(native()[0], name)
        f.restype = C.c_int
        f.argtypes = {"dfb_kv_append": [_P, _P, _P, _P], "dfb_kv_attention_workspace": [_P, _P, _P],
                      "dfb_kv_attention": [_P, _P, _P, C.c_size_t, _P, _P], "dfb_token_logprobs": [_P, _P, _P]}[name]
        _fns[name] = f
    return f


def _ck(rc):
    if rc != 0:
        raise DiffuseError(native()[0].dfb_last_error().decode())


def _stream(index, stream):
    return torch._C._cuda_getCurrentRawStream(index) if stream is None else stream


def _empty(like, shape, dtype, index, stream):
    """A new tensor whose memory goes back to the stream that the call runs on."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=index)):
        return like.new_empty(shape, dtype=dtype)


def _fits(sizes):
    """Sizes (all of them or-ed together) go to the library as int32: a larger one would arrive as another
    number.  (Negative ones are for the library to refuse.)"""
    if sizes >> 31 not in (0, -1):
        raise ValueError("a size does not fit 32 bits")


# (device indices are compared as integers: a call's checks take a few microseconds, and its kernel may not
# take more)
def _ints(name, t, index, n=None):
    """Data pointer of an int32 tensor of the call's GPU (None: a null pointer)."""
    if t is None:
        return None
    if t.dtype is not torch.int32 or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{name} must be a contiguous int32 tensor on cuda:{index}")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} elements, expected {n}")
    return t.data_ptr()


def _rows(name, t, dtype, index, shape):
    """(tensor's strides) of rows [n_rows, heads, head_dim]."""
    if t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{name} must be {dtype} on cuda:{index}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    st = t.stride()
    if st[2] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return st


class PagedKV:
    """A paged K/V cache in 8 bits: E4M3 codes [n_pages, n_kv, page, head_dim], one f32 scale for
    each page and KV head, and the page table [n_seq, max_pages] (int32) of the sequences.  The
    tensors stay the caller's; `pages` may be replaced (set_pages) as sequences come and go."""

    def __init__(self, k, v, k_scale, v_scale, pages):
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError(f"codes are [n_pages, n_kv, page, head_dim], got {tuple(k.shape)} and {tuple(v.shape)}")
        for t in (k, v):
            if t.dtype not in (torch.float8_e4m3fn, torch.uint8) or not t.is_contiguous() or not t.is_cuda or t.device != k.device:
                raise ValueError("codes must be contiguous float8_e4m3fn (or uint8) CUDA tensors of one device")
        for t in (k_scale, v_scale):
            if t.dtype != torch.float32 or tuple(t.shape) != tuple(k.shape[:2]) or not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"scales must be contiguous float32 tensors {tuple(k.shape[:2])} on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self._index = k.device, k.get_device()
        self.n_pages, self.n_kv, self.page, self.head_dim = k.shape
        self.set_pages(pages)

    @classmethod
    def empty(cls, n_pages: int, n_kv: int, head_dim: int, pages, page: int = 64):
        """A new pool on the page table's device (codes 0, scales 2^-64: nothing stored yet)."""
        codes = [torch.zeros((n_pages, n_kv, page, head_dim), dtype=torch.uint8, device=pages.device).view(torch.float8_e4m3fn)
                 for _ in range(2)]
        scales = [torch.full((n_pages, n_kv), 2.0**-64, dtype=torch.float32, device=pages.device) for _ in range(2)]
        return cls(*codes, *scales, pages)

    def set_pages(self, pages):
        if pages.dim() != 2:
            raise ValueError("pages is [n_seq, max_pages]")
        _fits(pages.shape[0] | pages.shape[1] | self.n_pages | self.n_kv)
        ptr = _ints("pages", pages, self._index)
        self.pages, self._n_seq = pages, pages.shape[0]
        self._ws = {}  # workspace sizes by the sizes of a call
        self._c = _KvCache(self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(), ptr,
                           self.n_pages, self.n_kv, self.head_dim, self.page, pages.shape[0], pages.shape[1])
        self._ref = C.addressof(self._c)


def kv_append(cache: PagedKV, k, v, row_off, lens, *, max_rows: int, pos=None, rope=None, q=None, q_out=None, status=None,
              stream=None):
    """Store rows k, v [n_rows, n_kv, head_dim] (f32 / f16 / bf16, any strides but a contiguous last
    dimension): sequence s's are row_off[s] .. row_off[s + 1] (int32 [n_seq + 1]) and go to the
    positions from lens[s] on, or to pos[row] (ascending within a sequence; lens[s] then says how
    many positions are filled).  max_rows: the most rows of any one sequence.  rope
    [n_positions, head_dim / 2, 2] (f32 cos, sin) rotates k, and q [n_rows, n_q, head_dim] into
    q_out.  See dfb_kv_append for the scales."""
    d, hd = cache._index, cache.head_dim
    typ = _TYPES.get(k.dtype)
    if k.dim() != 3 or typ is None:
        raise ValueError("k is [n_rows, n_kv, head_dim] in f32, f16 or bf16")
    n = k.shape[0]
    _fits(n | max_rows)
    sk = _rows("k", k, k.dtype, d, (n, cache.n_kv, hd))
    sv = _rows("v", v, k.dtype, d, (n, cache.n_kv, hd))
    r = _KvRows(k.data_ptr(), v.data_ptr(), typ, n, max_rows, sk[0], sk[1], sv[0], sv[1], _ints("row_off", row_off, d, cache._n_seq + 1),
                _ints("lens", lens, d, cache._n_seq), _ints("pos", pos, d, n))
    if rope is not None:
        if rope.dtype is not torch.float32 or not rope.is_contiguous() or rope.get_device() != d or rope.shape[1:] != (hd // 2, 2):
            raise ValueError(f"rope must be a contiguous float32 tensor [n_positions, {hd // 2}, 2] on {cache.device}")
        _fits(rope.shape[0])
        r.rope, r.n_rope = rope.data_ptr(), rope.shape[0]
    if (q is None) != (q_out is None):
        raise ValueError("q and q_out go together")
    if q is not None:
        if q.dim() != 3:
            raise ValueError("q is [n_rows, n_q, head_dim]")
        n_q = q.shape[1]
        _fits(n_q)
        sq = _rows("q", q, k.dtype, d, (n, n_q, hd))
        so = _rows("q_out", q_out, k.dtype, d, (n, n_q, hd))
        r.n_q, r.q, r.q_out = n_q, q.data_ptr(), q_out.data_ptr()
        r.q_tok, r.q_head, r.q_out_tok, r.q_out_head = sq[0], sq[1], so[0], so[1]
    _ck(_fn("dfb_kv_append")(cache._ref, C.addressof(r), _ints("status", status, d, 1), _stream(d, stream)))


def kv_attention(cache: PagedKV, q, row_off, lens, *, max_rows: int, max_keys: int, scale: float | None = None, vis=None,
                 out=None, return_lse: bool = False, workspace=None, status=None, stream=None):
    """softmax(scale q K^T) V of query rows q [n_rows, n_q, head_dim] (f16 / bf16; row_off as in
    kv_append) over the first min(vis[row], lens[s]) keys of their sequence (vis None: lens[s]).
    max_rows, max_keys: bounds of any one sequence's rows and keys.  scale None: 1 / sqrt(head_dim).
    workspace: a uint8 tensor of at least kv_attention_workspace(...) bytes (None: allocated here).
    Returns out (and lse [n_rows, n_q], the natural log of the softmax denominator)."""
    d = cache._index
    typ = _TYPES.get(q.dtype)
    if q.dim() != 3 or typ is None or typ == F32:
        raise ValueError("q is [n_rows, n_q, head_dim] in f16 or bf16")
    n, n_q, hd = q.shape
    _fits(n | n_q | max_rows | max_keys)
    sq = _rows("q", q, q.dtype, d, (n, n_q, cache.head_dim))
    if out is None:
        out = _empty(q, (n, n_q, hd), q.dtype, d, stream)
        so = (n_q * hd, hd)
    else:
        so = _rows("out", out, q.dtype, d, (n, n_q, hd))
    lse = _empty(q, (n, n_q), torch.float32, d, stream) if return_lse else None
    a = _KvAttn(q.data_ptr(), out.data_ptr(), typ, n_q, n, max_rows, max_keys, hd**-0.5 if scale is None else scale, sq[0], sq[1],
                so[0], so[1], _ints("row_off", row_off, d, cache._n_seq + 1), _ints("lens", lens, d, cache._n_seq),
                _ints("vis", vis, d, n), None if lse is None else lse.data_ptr())
    if workspace is None:
        sizes = (n_q, n, max_rows, max_keys)
        need = cache._ws.get(sizes)
        if need is None:
            if len(cache._ws) >= _MAX_WS:
                cache._ws.clear()
            need = cache._ws[sizes] = kv_attention_workspace(cache, n_q=n_q, n_rows=n, max_rows=max_rows, max_keys=max_keys)
        if need:
            workspace = _empty(q, (need,), torch.uint8, d, stream)
    elif workspace.get_device() != d or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on {cache.device}")
    _ck(_fn("dfb_kv_attention")(cache._ref, C.addressof(a), None if workspace is None else workspace.data_ptr(),
                                0 if workspace is None else workspace.numel() * workspace.element_size(),
                                _ints("status", status, d, 1), _stream(d, stream)))
    return (out, lse) if return_lse else out


def kv_attention_workspace(cache: PagedKV, *, n_q: int, n_rows: int, max_rows: int, max_keys: int) -> int:
    """Bytes of workspace a kv_attention call of these sizes needs (0: none)."""
    _fits(n_q | n_rows | max_rows | max_keys)
    a = _KvAttn(type=F16, n_q=n_q, n_rows=n_rows, max_rows=max_rows, max_keys=max_keys, scale=1.0)
    need = C.c_size_t()
    _ck(_fn("dfb_kv_attention_workspace")(cache._ref, C.addressof(a), C.addressof(need)))
    return need.value


def token_logprobs(logits, targets=None, *, top_k: int = 0, rows=None, status=None, stream=None):
    """Of rows of logits [n_logits, n_vocab] (f32 / f16 / bf16; rows: int32 row ids, None: all): the
    log probability of targets[i] (int32; negative: 0), the entropy in nats, and the top_k tokens
    with their log probabilities, equal logits by the lower id.
    Returns (logprob or None, entropy, top_ids [n, top_k], top_logprob [n, top_k])."""
    if logits.dim() != 2 or logits.dtype not in _TYPES or not logits.is_cuda:
        raise ValueError("logits is a CUDA tensor [n_logits, n_vocab] in f32, f16 or bf16")
    if logits.shape[1] > 1 and logits.stride(1) != 1:
        raise ValueError("logits: the last dimension must be contiguous")
    d, v = logits.get_device(), logits.shape[1]
    n = logits.shape[0] if rows is None else rows.numel()
    _fits(n | v | logits.shape[0] | top_k)
    k = max(top_k, 0)
    tp = _ints("targets", targets, d, n)
    # one allocation: logprob, entropy, top_logprob, then the ids
    lp, ent, top, ids = _empty(logits, (n * (2 + 2 * k),), torch.float32, d, stream).split((n, n, n * k, n * k))
    top, ids = top.view(n, k), ids.view(torch.int32).view(n, k)
    a = _Logprobs(logits.data_ptr(), _TYPES[logits.dtype], v, n, logits.shape[0], logits.stride(0), _ints("rows", rows, d), tp,
                  lp.data_ptr() if tp else None, ent.data_ptr(), top_k, ids.data_ptr() if k else None, top.data_ptr() if k else None)
    _ck(_fn("dfb_token_logprobs")(C.addressof(a), _ints("status", status, d, 1), _stream(d, stream)))
    return lp if tp else None, ent, ids, top
