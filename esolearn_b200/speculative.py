"""Speculative decoding over a (quantised) paged K/V cache, on torch CUDA tensors.

One step of B sequences with N tokens each: node 0 is the sequence's last
token, nodes 1..N-1 are drafted, node i under node parents[i] < i.

    q = kv_append(cache, k, v, ctx_len, q=q, rope=(cos, sin), depth=depth, q_scale=hd ** -0.5)
    x = tree_attention(q, cache, ctx_len, max_ctx, mask=mask)         # ... and the rest of the layers
    path, n_accept, token = verify_drafts(logits, tokens, parents, u, noise, temperature=0.8)
    kv_commit(cache, ctx_len, path, n_accept)
    ctx_len += n_accept                                               # `token` is the next step's node 0

N = 1 is plain decoding.  The calls run on torch's current stream and wait for
nothing; their tensors lie on the thread's current device.  A kernel whose wait
gave up makes a later call raise SbError (SB_ERR_TIMEOUT).  Every call goes to
libscryb200.so (declarations and the exact rules in include/sb_api.h).  The
reference decodes one token per step from an f32 cache and has no counterpart.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np

from . import _native as N

_SHAPE, _ARG = 4, 6


def _need(ok: bool, message: str, code: int = _SHAPE) -> None:
    if not ok:
        raise N.SbError(code, message)


_raw_stream = _raw_device = None


def _stream(t) -> int:
    """The current stream of t's device, which has to be the thread's current device: the library launches there (raw
    handle and number: torch.cuda.current_stream builds an object, 2 us a call)."""
    global _raw_stream, _raw_device
    if _raw_stream is None:
        import torch

        _raw_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    i, here = t.get_device(), _raw_device()
    if i != here:
        raise N.SbError(_ARG, f"tensors on cuda:{i}, but the current device is cuda:{here} (torch.cuda.device({i}) makes theirs current)")
    return _raw_stream(i)


def _dtype(t, who: str) -> int:
    import torch

    if t.dtype is torch.float32:
        return N.SB_DTYPE_F32
    _need(t.dtype is torch.bfloat16, f"{who}: dtype {t.dtype} is neither float32 nor bfloat16", _ARG)
    return N.SB_DTYPE_BF16


def _ints(t, shape, name: str, device) -> int:
    """Address of a contiguous int32 CUDA tensor of the given shape (None: NULL)."""
    if t is None:
        return 0
    import torch

    if t.dtype is torch.int32 and t.shape == shape and t.is_contiguous() and t.device == device:
        return t.data_ptr()
    _need(t.dtype is torch.int32 and t.device == device, f"{name}: int32 tensor on {device} expected", _ARG)
    raise N.SbError(_SHAPE, f"{name}: contiguous {tuple(shape)} expected, got {tuple(t.shape)}")


def _rows(t, name: str):
    """(tensor, row stride) of a [B, T, heads, head_dim] tensor whose (b, t) rows are equally far apart and 16-byte
    aligned and whose heads are contiguous; a copy where it is not."""
    b, n, h, d = t.shape
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, h * d
    sb, sn, sh, sd = t.stride()
    lanes = 4 if t.element_size() == 4 else 8
    ok = (sd == 1 or d == 1) and (sh == d or h == 1) and t.data_ptr() % 16 == 0
    if n > 1:
        ok = ok and (b == 1 or sb == n * sn)
        row = sn
    else:
        row = sb if b > 1 else h * d
    if ok and row >= h * d and row % lanes == 0:
        return t, row
    t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone()
    return t, h * d


def _matrix_rows(x):
    """(tensor, row stride) of a [B, V] tensor with contiguous rows; a copy where rows overlap, such as one row expanded
    over the batch."""
    b, v = x.shape
    if b <= 1:
        return x, v
    return (x, x.stride(0)) if x.stride(0) >= v else (x.contiguous(), v)


class KvCache:
    """A paged K/V cache: k and v [pages, n_kv, page_size, head_dim] of bfloat16, float32 or int8 (int8: codes with
    one float32 scale per row in k_scale, v_scale [pages, n_kv, page_size]) and the page table [B, max_pages] int32.
    The tensors stay the caller's; the handle keeps them alive."""

    def __init__(self, k, v, page_table, k_scale=None, v_scale=None):
        import torch

        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype, "KvCache: k and v must be [pages, n_kv, page_size, head_dim] alike")
        _need(k.is_cuda and v.device == k.device and k.is_contiguous() and v.is_contiguous(), "KvCache: contiguous CUDA tensors expected", _ARG)
        kinds = {torch.bfloat16: N.SB_KV_BF16, torch.float32: N.SB_KV_F32, torch.int8: N.SB_KV_I8}
        _need(k.dtype in kinds, f"KvCache: dtype {k.dtype} not in bfloat16, float32, int8", _ARG)
        if k.dtype == torch.int8:
            for s in (k_scale, v_scale):
                _need(s is not None and s.dtype == torch.float32 and s.device == k.device and s.is_contiguous()
                      and s.shape == k.shape[:3], "KvCache: int8 rows need float32 scales [pages, n_kv, page_size]", _ARG)
        else:
            _need(k_scale is None and v_scale is None, "KvCache: only int8 rows have scales", _ARG)
        _need(page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.device == k.device and page_table.is_contiguous(),
              "KvCache: page_table must be a contiguous int32 [B, max_pages] tensor beside the cache", _ARG)
        self.k, self.v, self.k_scale, self.v_scale, self.page_table = k, v, k_scale, v_scale, page_table
        self.n_pages, self.n_kv, self.page_size, self.head_dim = k.shape
        self.batch, self.max_pages = page_table.shape
        self.device = k.device
        c = N.KvCacheC()
        c.k, c.v, c.page_table = k.data_ptr(), v.data_ptr(), page_table.data_ptr()
        if k_scale is not None:
            c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        c.max_pages, c.n_pages, c.n_kv, c.page_size, c.head_dim, c.kv_dtype = (
            self.max_pages, self.n_pages, self.n_kv, self.page_size, self.head_dim, kinds[k.dtype])
        self._c = c
        self._ref = C.addressof(c)

    @classmethod
    def zeros(cls, batch: int, max_seq: int, n_kv: int, head_dim: int, page_size: int = 64, dtype: str = "int8", device="cuda"):
        """A cache for `batch` sequences of up to max_seq positions, sequence b on pages b*P .. b*P+P-1."""
        import torch

        kind = {"int8": torch.int8, "bf16": torch.bfloat16, "f32": torch.float32}
        _need(dtype in kind, f"KvCache.zeros: dtype {dtype!r} not in {sorted(kind)}", _ARG)
        per = -(-max_seq // page_size)
        shape = (batch * per, n_kv, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=kind[dtype], device=device) for _ in range(2))
        table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per)
        s = [torch.zeros(shape[:3], device=device) for _ in range(2)] if dtype == "int8" else [None, None]
        return cls(k, v, table, *s)


def kv_append(cache: KvCache, k, v, ctx_len, q=None, rope=None, depth=None, n_new=None, q_scale: float = 1.0, q_out=None):
    """Write the rows of k, v [B, T, n_kv, head_dim] (float32 or bfloat16, views of one fused projection allowed) to
    positions ctx_len[b] + t, rotated and quantised; returns q [B, T, n_heads, head_dim] rotated and scaled, or None
    (sb_kv_append).  rope: (cos, sin) [positions, head_dim/2] float32; depth: int32 [T] or [B, T], the rows' places
    behind ctx_len for the rotation (default t); n_new: int32 [B], rows t >= n_new[b] are skipped."""
    import torch

    dev = cache.device
    _need(k.dim() == 4 and v.shape == k.shape and k.dtype is v.dtype, "kv_append: k and v must be [B, T, n_kv, head_dim] alike")
    b, t, nkv, hd = k.shape
    if nkv != cache.n_kv or hd != cache.head_dim or b != cache.batch:
        raise N.SbError(_SHAPE, f"kv_append: k is {tuple(k.shape)}, the cache has {cache.batch} sequences of {cache.n_kv} heads of {cache.head_dim}")
    _need(k.device == dev and v.device == dev, "kv_append: k and v must lie beside the cache", _ARG)
    dt = _dtype(k, "kv_append")
    k, ks = _rows(k, "k")
    v, vs = _rows(v, "v")
    nh, qs, qp, op = 0, 0, 0, 0
    if q is not None:
        if q.dim() != 4 or q.dtype is not k.dtype or q.device != dev or (qsh := q.shape)[0] != b or qsh[1] != t or qsh[3] != hd:
            raise N.SbError(_SHAPE, f"kv_append: q must be [{b}, {t}, n_heads, {hd}] of k's dtype")
        nh = qsh[2]
        q, qs = _rows(q, "q")
        if q_out is None:
            q_out = q.new_empty((b, t, nh, hd))
        else:
            _need(q_out.shape == q.shape and q_out.dtype == q.dtype and q_out.device == q.device and q_out.is_contiguous(),
                  "kv_append: q_out must be contiguous and like q")
        qp, op = q.data_ptr(), q_out.data_ptr()
    cos = sin = rl = 0
    if rope is not None:
        x, y = rope
        if not (x.dim() == 2 and x.shape == y.shape and x.shape[1] * 2 == hd and x.dtype is torch.float32 and y.dtype is torch.float32
                and x.device == dev and y.device == dev and x.is_contiguous() and y.is_contiguous()):
            raise N.SbError(_SHAPE, f"kv_append: rope must be two contiguous float32 [positions, {hd // 2}] tables")
        cos, sin, rl = x.data_ptr(), y.data_ptr(), x.shape[0]
    dld = 0
    if depth is not None and depth.dim() == 2:
        dld = t
    dp = _ints(depth, (b, t) if dld else (t,), "kv_append: depth", cache.device)
    N.check(N.lib().sb_kv_append(cache._ref, qp, k.data_ptr(), v.data_ptr(), dt, qs, ks, vs, b, t, nh,
                                 _ints(ctx_len, (b,), "kv_append: ctx_len", cache.device), _ints(n_new, (b,), "kv_append: n_new", cache.device),
                                 dp, dld, cos, sin, rl, q_scale, op, _stream(k)))
    return q_out


def kv_commit(cache: KvCache, ctx_len, path, n_accept) -> None:
    """Keep a tree's accepted path: the row at ctx_len[b] + path[b, i] moves to ctx_len[b] + i for i < n_accept[b]
    (sb_kv_commit).  path: int32 [B, P] ascending, n_accept: int32 [B], as verify_drafts returns them."""
    _need(path.dim() == 2, "kv_commit: path must be [B, P]")
    b = cache.batch
    N.check(N.lib().sb_kv_commit(cache._ref, b, _ints(ctx_len, (b,), "kv_commit: ctx_len", cache.device),
                                 _ints(path, (b, path.shape[1]), "kv_commit: path", cache.device), path.shape[1],
                                 _ints(n_accept, (b,), "kv_commit: n_accept", cache.device), _stream(path)))


def kv_read(cache: KvCache, n: int, start=None, dtype=None):
    """(k, v) [B, n, n_kv, head_dim] of positions start[b] .. start[b]+n-1 (start None: from 0) as float32 or
    bfloat16 values (sb_kv_read); positions outside the cache read as zeros."""
    import torch

    _need(n >= 0, "kv_read: n < 0")
    dtype = torch.float32 if dtype is None else dtype
    k = cache.k.new_empty((cache.batch, n, cache.n_kv, cache.head_dim), dtype=dtype)
    v = torch.empty_like(k)
    N.check(N.lib().sb_kv_read(cache._ref, cache.batch, _ints(start, (cache.batch,), "kv_read: start", cache.device), n,
                               _dtype(k, "kv_read"), k.data_ptr(), v.data_ptr(), _stream(k)))
    return k, v


def tree_attention(q, cache: KvCache, ctx_len, max_ctx: int, mask=None, n_new=None, out=None):
    """Attention of q [B, T, n_heads, head_dim] (rotated and scaled, float32 or bfloat16) over each sequence's cached
    context and, among the T rows behind it, those that the token's mask row names (sb_tree_attention).  mask: int64
    words [T, ceil(T/64)] or [B, T, ceil(T/64)] from tree_mask (None: each token sees itself and those before it);
    max_ctx: an upper bound of ctx_len[b] + T; n_new: int32 [B], tokens t >= n_new[b] do not exist (their output is 0)."""
    import torch

    _need(q.dim() == 4 and q.device == cache.device, "tree_attention: q must be [B, T, n_heads, head_dim] beside the cache")
    b, t, nh, hd = q.shape
    if b != cache.batch or hd != cache.head_dim or nh < cache.n_kv or nh % cache.n_kv:
        raise N.SbError(_SHAPE, f"tree_attention: q is {tuple(q.shape)}, the cache has {cache.batch} sequences of {cache.n_kv} heads of {cache.head_dim}")
    dt = _dtype(q, "tree_attention")
    q, qs = _rows(q, "q")
    mp = mld = 0
    if mask is not None:
        w = (t + 63) // 64
        ms = mask.shape
        if not (mask.dtype is torch.int64 and mask.device == cache.device and mask.is_contiguous() and (ms == (t, w) or ms == (b, t, w))):
            raise N.SbError(_SHAPE, f"tree_attention: mask must be contiguous int64 [{t}, {w}] or [{b}, {t}, {w}]")
        mp, mld = mask.data_ptr(), t * w if len(ms) == 3 else 0
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((b, t, nh, hd))
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device and out.is_contiguous(),
              "tree_attention: out must be contiguous and like q")
    N.check(N.lib().sb_tree_attention(cache._ref, q.data_ptr(), dt, qs, b, t, nh, _ints(ctx_len, (b,), "tree_attention: ctx_len", cache.device),
                                      _ints(n_new, (b,), "tree_attention: n_new", cache.device), mp, mld, max_ctx, out.data_ptr(), _stream(q)))
    return out


def verify_drafts(logits, tokens, parents, u=None, noise=None, temperature: float = 1.0, draft_probs=None):
    """(path [B, N], n_accept [B], next_token [B]) int32: the drafted tokens accepted against the target's
    probabilities softmax(logits / temperature), and the next token (sb_verify_drafts).  logits [B, N, V] float32, row
    i after node i; tokens int32 [B, N]; parents int32 [N] or [B, N]; u [B, N] uniform in [0, 1) and noise [B, V]
    exponential(1) > 0, float32 (not needed at temperature 0); draft_probs [B, N, V] float32, row i the distribution
    the children of node i were drawn from, or None for given tokens."""
    import torch

    _need(logits.dim() == 3 and logits.is_cuda and logits.dtype == torch.float32, "verify_drafts: logits must be a float32 CUDA [B, N, V]", _ARG)
    b, n, v = logits.shape
    dev = logits.device

    def rows(x, name):
        if x.dtype is not torch.float32 or x.device != dev or x.shape != logits.shape:
            raise N.SbError(_SHAPE, f"verify_drafts: {name} must be float32 {tuple(logits.shape)}")
        if x.is_contiguous():
            return x, v
        if (x.stride(2) == 1 or v == 1) and (b == 1 or x.stride(0) == n * x.stride(1)) and x.stride(1) >= v:
            return x, x.stride(1)
        return x.contiguous(), v

    lg, ld = rows(logits, "logits")
    dp = dl = 0
    if draft_probs is not None:
        draft_probs, dl = rows(draft_probs, "draft_probs")
        dp = draft_probs.data_ptr()
    up = np_ = nl = 0
    if u is not None:
        if u.dtype is not torch.float32 or u.device != dev or u.shape != (b, n) or not u.is_contiguous():
            raise N.SbError(_SHAPE, f"verify_drafts: u must be contiguous float32 ({b}, {n})")
        up = u.data_ptr()
    if noise is not None:
        if noise.dtype is not torch.float32 or noise.device != dev or noise.shape != (b, v) or not (noise.stride(1) == 1 or v == 1):
            raise N.SbError(_SHAPE, f"verify_drafts: noise must be float32 ({b}, {v})")
        noise, nl = _matrix_rows(noise)
        np_ = noise.data_ptr()
    pld = n if parents.dim() == 2 else 0
    tp = _ints(tokens, (b, n), "verify_drafts: tokens", dev)
    path, n_accept = torch.empty_like(tokens), tokens.new_empty((b,))
    nxt = torch.empty_like(n_accept)
    N.check(N.lib().sb_verify_drafts(lg.data_ptr(), ld, tp,
                                     _ints(parents, (b, n) if pld else (n,), "verify_drafts: parents", dev), pld, dp, dl, up, np_, nl,
                                     b, n, v, temperature, path.data_ptr(), n_accept.data_ptr(), nxt.data_ptr(), _stream(lg)))
    return path, n_accept, nxt


def _check_parents(parents: Sequence[int]) -> list:
    p = [int(x) for x in parents]
    _need(len(p) >= 1 and all(0 <= p[i] < i for i in range(1, len(p))), "a tree's node i > 0 hangs under a node parents[i] < i", _ARG)
    return p


def tree_depth(parents: Sequence[int]) -> np.ndarray:
    """int32 [N]: steps from node 0, the rows' places behind ctx_len for kv_append's rotation."""
    p = _check_parents(parents)
    d = np.zeros(len(p), np.int32)
    for i in range(1, len(p)):
        d[i] = d[p[i]] + 1
    return d


def tree_mask(parents: Sequence[int]) -> np.ndarray:
    """int64 words [N, ceil(N/64)] for tree_attention: bit j of row i is set when node j is i or one of its ancestors."""
    p = _check_parents(parents)
    n = len(p)
    m = np.zeros((n, (n + 63) // 64), np.uint64)
    for i in range(n):
        if i:
            m[i] = m[p[i]]
        m[i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return m.view(np.int64)
