"""Paged key-value cache: device-tensor entry points and the cache of a model.

The reference crate attends whole sequences only; this is the serving side of
its operator: new rows are written to pages (paged_append), one new token per
sequence attends over them (paged_attention), and a cache is brought back to a
budget by the attention weight its keys have drawn (attention_key_weights for a
prompt, paged_attention's own sums while decoding, paged_evict).

Pools are [num_pages, kv_heads, page_size, head_dim] tensors (strided views
allowed, the head_dim contiguous); a page table is int32 [batch, max_pages] and
position t of sequence b is slot t % page_size of page table[b, t // page_size].
An entry outside [0, num_pages) holds no keys.

Every function runs on `stream` (default: the current stream of the tensors'
device), allocates what it returns and its workspace there, never synchronises
and may be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct

from . import GAEError, _check, _torch, lib

_I64_2, _I64_3 = C.c_int64 * 2, C.c_int64 * 3

# Small calls take as long as their host side: argument blocks are packed in one
# call, and tensors made by empty_strided, the quickest of torch's constructors.


class KvPool(C.Structure):
    """Mirror of gae_kv_pool (include/gae.h)."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_stride", _I64_3), ("v_stride", _I64_3),
                ("num_pages", C.c_int64), ("kv_heads", C.c_int64), ("page_size", C.c_int64),
                ("head_dim", C.c_int64), ("dtype", C.c_int)]


class PagedAppendArgs(C.Structure):
    """Mirror of gae_paged_append_args (include/gae.h)."""
    _fields_ = [("k_new", C.c_void_p), ("v_new", C.c_void_p), ("k_new_stride", _I64_3),
                ("v_new_stride", _I64_3), ("batch", C.c_int64), ("tokens", C.c_int64),
                ("page_table", C.c_void_p), ("table_stride", C.c_int64), ("max_pages", C.c_int64),
                ("start", C.c_void_p), ("counts", C.c_void_p)]


class PagedAttnArgs(C.Structure):
    """Mirror of gae_paged_attn_args (include/gae.h)."""
    _fields_ = [("q", C.c_void_p), ("o", C.c_void_p), ("lse", C.c_void_p), ("q_stride", _I64_2),
                ("o_stride", _I64_2), ("batch", C.c_int64), ("heads", C.c_int64),
                ("page_table", C.c_void_p), ("table_stride", C.c_int64), ("max_pages", C.c_int64),
                ("seq_lens", C.c_void_p), ("scale", C.c_float), ("weights", C.c_void_p),
                ("weights_out", C.c_void_p), ("w_stride", _I64_2), ("w_out_stride", _I64_2),
                ("weights_len", C.c_int64), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class KeyWeightsArgs(C.Structure):
    """Mirror of gae_key_weights_args (include/gae.h)."""
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("lse", C.c_void_p), ("out", C.c_void_p),
                ("batch", C.c_int64), ("heads", C.c_int64), ("kv_heads", C.c_int64),
                ("seq_q", C.c_int64), ("seq_kv", C.c_int64), ("head_dim", C.c_int64),
                ("q_stride", _I64_3), ("k_stride", _I64_3), ("lse_stride", _I64_2),
                ("out_stride", _I64_2), ("dtype", C.c_int), ("causal", C.c_int),
                ("accumulate", C.c_int), ("scale", C.c_float), ("q_offset", C.c_int64),
                ("kv_offset", C.c_int64), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class PagedEvictArgs(C.Structure):
    """Mirror of gae_paged_evict_args (include/gae.h)."""
    _fields_ = [("batch", C.c_int64), ("page_table", C.c_void_p), ("table_stride", C.c_int64),
                ("max_pages", C.c_int64), ("seq_lens", C.c_void_p), ("weights", C.c_void_p),
                ("w_stride", _I64_2), ("weights_len", C.c_int64), ("dst_table", C.c_void_p), ("dst_stride", C.c_int64),
                ("dst_max_pages", C.c_int64), ("keep", C.c_int64), ("recent", C.c_int64),
                ("new_lens", C.c_void_p), ("kept", C.c_void_p), ("kept_weights", C.c_void_p)]


def _packer(mirror):
    """struct packer of a mirror's fields in their C layout: one call fills a
    whole argument block, in a fifth of the time a ctypes structure takes."""
    code = {C.c_void_p: "P", C.c_int64: "q", C.c_size_t: "N", C.c_int: "i", C.c_float: "f", _I64_2: "2q", _I64_3: "3q"}
    s = struct.Struct("@" + "".join(code[t] for _, t in mirror._fields_) + "0q")
    assert s.size == C.sizeof(mirror)
    return s.pack


_pack_pool, _pack_append, _pack_attn, _pack_keys, _pack_evict = map(
    _packer, (KvPool, PagedAppendArgs, PagedAttnArgs, KeyWeightsArgs, PagedEvictArgs))


def _bind(L):
    vp, i64, sz = C.c_void_p, C.c_int64, C.c_size_t
    for name in ("gae_paged_append", "gae_paged_attn_fwd", "gae_paged_evict"):
        getattr(L, name).argtypes = [vp, vp, vp]
    L.gae_paged_attn_workspace_bytes.restype = sz
    L.gae_paged_attn_workspace_bytes.argtypes = [i64, i64, i64, i64, i64, C.c_int]
    L.gae_key_weights_workspace_bytes.restype = sz
    L.gae_key_weights_workspace_bytes.argtypes = [i64] * 5
    L.gae_key_weights.argtypes = [vp, vp]


@functools.lru_cache(maxsize=None)
def _load():
    """torch, imported by the first call; the dtypes' codes; int32; float32."""
    torch = _torch()
    return torch, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}, torch.int32, torch.float32


# The workspaces' sizes, by the calls' sizes alone.
@functools.lru_cache(maxsize=1024)
def _attn_workspace(*sizes):
    return lib().gae_paged_attn_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=1024)
def _keys_workspace(*sizes):
    return lib().gae_key_weights_workspace_bytes(*sizes)


def _run(what, names, tensors, stream, body):
    """body(stream pointer) with the tensors' device and `stream` current, so that
    what it allocates belongs to the stream it runs on; on a stream other than
    the current one the inputs are marked as used there.  The first tensor's
    device is everyone's; names is for the error that says whose is not."""
    torch = _load()[0]
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev or dev < 0:
            name = names.split()[next(i for i, x in enumerate(tensors) if x is t)]
            raise GAEError(1, f"{what}: tensors must be on one CUDA device, {name} is on {t.device}")
    if stream is None and torch._C._cuda_getDevice() == dev:
        return body(torch._C._cuda_getCurrentRawStream(dev))
    with torch.cuda.device(dev):
        if stream is None:
            return body(torch._C._cuda_getCurrentRawStream(dev))
        if stream.device.index != dev:
            raise GAEError(1, f"{what}: stream on {stream.device}, tensors on device {dev}")
        with torch.cuda.stream(stream):
            for t in tensors:
                if t is not None:
                    t.record_stream(stream)
            return body(stream.cuda_stream)


def _code(t):
    c = _load()[1].get(t.dtype)
    if c is None:
        raise GAEError(1, f"unsupported dtype {t.dtype}")
    return c


def _pool(what, k_pages, v_pages):
    """(packed gae_kv_pool, shape)"""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise GAEError(1, f"{what}: k_pages and v_pages must be [num_pages, kv_heads, page_size, head_dim]")
    if v_pages.dtype != k_pages.dtype:
        raise GAEError(1, f"{what}: k_pages and v_pages must share a dtype")
    kp, kh, ks, kd = k_pages.stride()
    vp, vh, vs, vd = v_pages.stride()
    if kd != 1 or vd != 1:
        raise GAEError(1, f"{what}: pages must have a contiguous head_dim")
    return _pack_pool(k_pages.data_ptr(), v_pages.data_ptr(), kp, kh, ks, vp, vh, vs, *shape, _code(k_pages)), shape


def _table(what, table, batch, name="page_table"):
    shape = table.shape
    if len(shape) != 2 or shape[0] != batch or table.dtype != _load()[2]:
        raise GAEError(1, f"{what}: {name} must be int32 [batch, max_pages]")
    row, one = table.stride()
    if one != 1 and shape[1] > 1:
        raise GAEError(1, f"{what}: {name} must have contiguous rows")
    return table.data_ptr(), row, shape[1]


def _ints(what, t, batch, name):
    if t.dtype != _load()[2] or t.shape != (batch,) or not t.is_contiguous():
        raise GAEError(1, f"{what}: {name} must be contiguous int32 [batch]")
    return t.data_ptr()


def _weights(what, t, batch, heads, n, name):
    """(address, batch stride, head stride)"""
    shape = t.shape
    if len(shape) != 3 or shape[0] != batch or shape[1] != heads or shape[2] < n or t.dtype != _load()[3]:
        raise GAEError(1, f"{what}: {name} must be fp32 [{batch}, {heads}, >= {n}]")
    sb, sh, one = t.stride()
    if one != 1 and shape[2] > 1:
        raise GAEError(1, f"{what}: {name} must have contiguous rows")
    return t.data_ptr(), sb, sh


def paged_append(k_new, v_new, k_pages, v_pages, page_table, start, *, counts=None, stream=None):
    """Writes new rows into the cache: k_new/v_new [B, Hkv, T, D] (strided views
    allowed); token t < counts[b] of sequence b (counts int32 [B], default T)
    becomes position start[b] + t.  Tokens beyond the page table, or whose entry
    names no page, are dropped."""
    what = "paged_append"
    shape = k_new.shape
    if len(shape) != 4 or v_new.shape != shape:
        raise GAEError(1, f"{what}: k_new and v_new must be [batch, kv_heads, tokens, head_dim]")
    B, H, T, D = shape
    pool, ps = _pool(what, k_pages, v_pages)
    if ps[1] != H or ps[3] != D:
        raise GAEError(1, f"{what}: k_new and k_pages differ in heads or head_dim")
    if k_new.dtype != k_pages.dtype or v_new.dtype != k_pages.dtype:
        raise GAEError(1, f"{what}: new rows and pages must share a dtype")
    kb, kh, kt, kd = k_new.stride()
    vb, vh, vt, vd = v_new.stride()
    if kd != 1 or vd != 1:
        raise GAEError(1, f"{what}: new rows must have a contiguous head_dim")
    a = _pack_append(k_new.data_ptr(), v_new.data_ptr(), kb, kh, kt, vb, vh, vt, B, T,
                     *_table(what, page_table, B), _ints(what, start, B, "start"),
                     0 if counts is None else _ints(what, counts, B, "counts"))
    _run(what, "k_pages v_pages k_new v_new page_table start counts",
         (k_pages, v_pages, k_new, v_new, page_table, start, counts), stream,
         lambda st: _check(lib().gae_paged_append(pool, a, st)))


def paged_attention(q, k_pages, v_pages, page_table, seq_lens, *, scale=None, out=None, lse=None,
                    return_lse=False, weights=None, weights_out=None, stream=None):
    """Attention of one new token per sequence: q [B, H, D] over the first
    seq_lens[b] cached positions (int32 [B]); H a multiple of the pages' heads.
    bf16/f16/f32, any head_dim <= 256 in 16-byte multiples.  An empty sequence
    gives 0 and lse -inf; an infinite value among a sequence's own gives NaN in
    16 bits (probabilities are held as the sum of two numbers).

    weights (fp32 [B, Hkv, >= the page table's positions]) asks for the keys'
    attention weight: weights_out = weights + the softmax summed over each key
    head's query heads; weights_out defaults to weights (in place).  Positions
    without a key are left as they are."""
    what = "paged_attention"
    torch = _load()[0]
    shape = q.shape
    if len(shape) != 3:
        raise GAEError(1, f"{what}: q must be [batch, heads, head_dim]")
    B, H, D = shape
    pool, (_, Hkv, page, pd) = _pool(what, k_pages, v_pages)
    if pd != D or k_pages.dtype != q.dtype:
        raise GAEError(1, f"{what}: q and the pages differ in head_dim or dtype")
    table = _table(what, page_table, B)
    lens = _ints(what, seq_lens, B, "seq_lens")
    qb, qh, qd = q.stride()
    if qd != 1:
        raise GAEError(1, f"{what}: q must have a contiguous head_dim")
    if out is not None and (out.shape != shape or out.dtype != q.dtype or out.stride(2) != 1):
        raise GAEError(1, f"{what}: out must be like q, with a contiguous head_dim")
    if lse is not None and (lse.shape != (B, H) or lse.dtype != torch.float32 or not lse.is_contiguous()):
        raise GAEError(1, f"{what}: lse must be contiguous fp32 [batch, heads]")
    cap = table[2] * page
    w = wo = (0, 0, 0)
    if weights is not None:
        weights_out = weights if weights_out is None else weights_out
        w = _weights(what, weights, B, Hkv, cap, "weights")
        wo = _weights(what, weights_out, B, Hkv, cap, "weights_out")
    elif weights_out is not None:
        raise GAEError(1, f"{what}: weights_out without weights")
    L = lib()

    def body(st):
        o, l = out, lse
        if o is None:
            o = torch.empty_like(q)
        if return_lse and l is None:
            l = torch.empty_strided((B, H), (H, 1), dtype=torch.float32, device=q.device)
        n = _attn_workspace(B, H, Hkv, D, cap, weights is not None)
        ws = torch.empty_strided((n,), (1,), dtype=torch.uint8, device=q.device)
        ob, oh, _ = o.stride()
        a = _pack_attn(q.data_ptr(), o.data_ptr(), 0 if l is None else l.data_ptr(), qb, qh, ob, oh, B, H, *table,
                       lens, 1.0 / math.sqrt(D) if scale is None else float(scale), w[0], wo[0], *w[1:], *wo[1:], cap,
                       ws.data_ptr(), n)
        _check(L.gae_paged_attn_fwd(pool, a, st))
        return (o, l) if return_lse else o

    return _run(what, "q k_pages v_pages page_table seq_lens out lse weights weights_out",
                (q, k_pages, v_pages, page_table, seq_lens, out, lse, weights, weights_out), stream, body)


def attention_key_weights(q, k, lse, *, causal=False, scale=None, q_offset=0, kv_offset=0, out=None,
                          accumulate=False, stream=None):
    """The attention weight that the queries put on each key: fp32 [B, Hkv, Nkv],
    sum over the queries that see the key (and the query heads of its key head)
    of exp(scale * <q, k> - lse).  q [B, H, Nq, D], k [B, Hkv, Nkv, D] (bf16/f16,
    head_dim 64/128, strided views allowed), lse [B, H, Nq] as attention(...,
    return_lse=True) gives it (contiguous rows; a query whose lse is -inf adds
    nothing, whatever it holds).  A window of a prompt's last
    queries is q[:, :, -n:], lse[:, :, -n:] with q_offset = N - n.  out may be a
    view of a cache's weights; accumulate=True adds to it."""
    what = "attention_key_weights"
    torch = _load()[0]
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4:
        raise GAEError(1, f"{what}: q and k must be [batch, heads, seq, head_dim]")
    B, H, Nq, D = qs
    Hkv, Nkv = ks[1], ks[2]
    if ks[0] != B or ks[3] != D or k.dtype != q.dtype:
        raise GAEError(1, f"{what}: q and k differ in batch, head_dim or dtype")
    qb, qh, qn, qd = q.stride()
    kb, kh, kn, kd = k.stride()
    if qd != 1 or kd != 1:
        raise GAEError(1, f"{what}: q and k must have a contiguous head_dim")
    l = _weights(what, lse, B, H, Nq, "lse")
    if lse.shape[2] != Nq:
        raise GAEError(1, f"{what}: lse must be [batch, heads, seq_q]")
    if accumulate and out is None:
        raise GAEError(1, f"{what}: accumulate needs out")
    if out is not None and out.shape != (B, Hkv, Nkv):
        raise GAEError(1, f"{what}: out must be [{B}, {Hkv}, {Nkv}]")
    L = lib()

    def body(st):
        w = out
        if w is None:
            w = torch.empty_strided((B, Hkv, Nkv), (Hkv * Nkv, Nkv, 1), dtype=torch.float32, device=q.device)
        n = _keys_workspace(B, H, Hkv, Nq, Nkv)
        ws = torch.empty_strided((n,), (1,), dtype=torch.uint8, device=q.device) if n else None
        wp, wb, wh = _weights(what, w, B, Hkv, Nkv, "out")
        a = _pack_keys(q.data_ptr(), k.data_ptr(), l[0], wp, B, H, Hkv, Nq, Nkv, D, qb, qh, qn, kb, kh, kn,
                       *l[1:], wb, wh, _code(q), 1 if causal else 0, 1 if accumulate else 0,
                       1.0 / math.sqrt(D) if scale is None else float(scale), q_offset, kv_offset,
                       ws.data_ptr() if n else 0, n)
        _check(L.gae_key_weights(a, st))
        return w

    return _run(what, "q k lse out", (q, k, lse, out), stream, body)


def paged_evict(k_pages, v_pages, page_table, seq_lens, weights, dst_table, *, keep, recent=0, stream=None):
    """Brings every sequence to at most `keep` cached positions: per key head the
    `recent` last positions and those of the largest weights (fp32 [B, Hkv, n];
    a sequence is cut to n; equal weights: the lower position, NaN largest).  The
    kept rows are copied in order to positions 0, 1, ... of dst_table, whose pages
    must not be among those read.  Returns (new lengths int32 [B], kept
    positions int32 [B, Hkv, keep], -1 beyond the length, their weights fp32,
    0 beyond)."""
    what = "paged_evict"
    torch = _load()[0]
    pool, (_, Hkv, _, _) = _pool(what, k_pages, v_pages)
    B = page_table.shape[0]
    table = _table(what, page_table, B)
    dst = _table(what, dst_table, B, "dst_table")
    lens = _ints(what, seq_lens, B, "seq_lens")
    w = _weights(what, weights, B, Hkv, 0, "weights")
    if keep < 1:
        raise GAEError(1, f"{what}: keep must be positive")

    def body(st):
        dev = k_pages.device
        new_lens = torch.empty_like(seq_lens)
        shape, strides = (B, Hkv, keep), (Hkv * keep, keep, 1)
        kept = torch.empty_strided(shape, strides, dtype=torch.int32, device=dev)
        kept_w = torch.empty_strided(shape, strides, dtype=torch.float32, device=dev)
        a = _pack_evict(B, *table, lens, *w, weights.shape[2], *dst, keep, recent, new_lens.data_ptr(),
                        kept.data_ptr(), kept_w.data_ptr())
        _check(lib().gae_paged_evict(pool, a, st))
        return new_lens, kept, kept_w

    return _run(what, "k_pages v_pages page_table seq_lens weights dst_table",
                (k_pages, v_pages, page_table, seq_lens, weights, dst_table), stream, body)


class PagedKVCache:
    """The keys and values of a batch of sequences for a model's layers.

    Every sequence owns max_len positions' worth of pages; the layers share one
    page table and one set of lengths.  A step over n new tokens is reserve(n),
    then per layer append() and attend() (or, for a prompt, the whole-sequence
    attention and add_prompt_weights()), then commit().  With a budget the cache
    also keeps the weight that each key has drawn, and evict() brings sequences
    longer than the budget back to it: the `recent` last positions and the
    heaviest others, per layer and key head (spare pages of a budget's size are
    held for that).

    reserve, append, attend and commit launch on the current stream and may be
    captured into a CUDA graph (a replay takes the counts of the capture);
    `lengths`, the host's count that the capacity check and evict() go by, moves
    once for the capture and not on a replay: refresh() reads it back from the
    device."""

    def __init__(self, n_layers, batch, kv_heads, head_dim, max_len, *, page_size=16, dtype=None, device="cuda",
                 budget=None, recent=0):
        torch = _torch()
        if min(n_layers, batch, kv_heads, head_dim, max_len, page_size) < 1:
            raise GAEError(1, "PagedKVCache: sizes must be positive")
        if budget is not None and not 0 < budget <= max_len:
            raise GAEError(1, f"PagedKVCache: budget must be in [1, {max_len}]")
        if budget is not None and not 0 <= recent <= budget:
            raise GAEError(1, "PagedKVCache: recent must be in [0, budget]")
        dtype = torch.bfloat16 if dtype is None else dtype
        self.batch, self.page_size, self.max_len, self.budget, self.recent = batch, page_size, max_len, budget, recent
        per = -(-max_len // page_size)
        spare = 0 if budget is None else -(-budget // page_size)
        pages = batch * (per + spare)
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        ids = torch.arange(pages, dtype=torch.int32, device=device).view(batch, per + spare)
        self.table = ids[:, :per].contiguous()
        self.spare = ids[:, per:].contiguous() if spare else None
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.next_lens = torch.zeros_like(self.lens)
        self.weights = None if budget is None else [
            torch.zeros((batch, kv_heads, per * page_size), dtype=torch.float32, device=device)
            for _ in range(n_layers)]
        self.lengths = [0] * batch
        self._reserved = None  # new tokens per sequence between reserve and commit
        self._tokens = 0       # their number in the padded batch

    def reserve(self, tokens, counts=None):
        """Makes room for `tokens` new tokens of every sequence (counts: a list
        of how many of them each sequence really has)."""
        if tokens < 0:
            raise GAEError(1, f"PagedKVCache: {tokens} tokens")
        n = [tokens] * self.batch if counts is None else [int(c) for c in counts]
        if len(n) != self.batch or any(not 0 <= c <= tokens for c in n):
            raise GAEError(1, f"PagedKVCache: counts must be {self.batch} numbers of [0, {tokens}]")
        longest = max(a + b for a, b in zip(self.lengths, n))
        if longest > self.max_len:
            raise GAEError(1, f"PagedKVCache: {longest} positions, room for {self.max_len}")
        torch = _torch()
        self._reserved, self._tokens = n, tokens
        if counts is None:
            torch.add(self.lens, tokens, out=self.next_lens)
        elif self.lens.is_cuda and torch.cuda.is_current_stream_capturing():  # which takes no copy from the host
            for b, c in enumerate(n):
                torch.add(self.lens[b: b + 1], c, out=self.next_lens[b: b + 1])
        else:
            torch.add(self.lens, torch.tensor(n, dtype=torch.int32, device=self.lens.device), out=self.next_lens)

    def append(self, layer, k_new, v_new):
        """Writes k_new/v_new [B, Hkv, T, D] behind the sequences of `layer`
        (T as reserved; a sequence's tokens beyond its count are dropped)."""
        if self._reserved is None:
            raise GAEError(1, "PagedKVCache: append without reserve")
        if k_new.shape[2] != self._tokens:
            raise GAEError(1, f"PagedKVCache: append of {k_new.shape[2]} tokens, {self._tokens} reserved")
        counts = None
        if any(c != k_new.shape[2] for c in self._reserved):
            counts = self.next_lens - self.lens
        paged_append(k_new, v_new, self.k[layer], self.v[layer], self.table, self.lens, counts=counts)

    def attend(self, layer, q, scale=None, out=None):
        """Attention of one new token per sequence, q [B, H, D], over everything
        appended so far; adds up the keys' weights where there is a budget (a
        sequence that reserve() counts no token of has no query: its keys' weights stay)."""
        w = None if self.weights is None else self.weights[layer]
        idle = [] if w is None else [(w[b], w[b].clone()) for b, c in enumerate(self._reserved or ()) if c == 0]
        o = paged_attention(q, self.k[layer], self.v[layer], self.table, self.next_lens, scale=scale, out=out, weights=w)
        for now, was in idle:
            now.copy_(was)
        return o

    def add_prompt_weights(self, layer, q, k, lse, scale=None):
        """Adds the weight that a prompt's queries put on its keys (an empty
        cache's first tokens): q [B, H, T, D], k [B, Hkv, T, D] and the lse of
        attention(q, k, v, causal=True, return_lse=True)."""
        if self.weights is None:
            return
        if self._reserved is None:
            raise GAEError(1, "PagedKVCache: prompt weights without reserve")
        if any(self.lengths):
            raise GAEError(1, "PagedKVCache: prompt weights need an empty cache")
        T = q.shape[2]
        if T != self._tokens or k.shape[2] != T:
            raise GAEError(1, f"PagedKVCache: weights of {T} queries and {k.shape[2]} keys, {self._tokens} tokens reserved")
        torch = _torch()
        if any(c != T for c in self._reserved):  # queries beyond a sequence's own tokens weigh nothing
            pad = torch.arange(T, device=lse.device)[None] >= self.next_lens[:, None]
            lse = lse.masked_fill(pad[:, None], -math.inf)
        w = self.weights[layer][:, :, :T]
        n = w.shape[2]  # beyond the pages lies padding only
        attention_key_weights(q[:, :, :n], k[:, :, :n], lse[:, :, :n], causal=True, scale=scale, out=w, accumulate=True)

    def commit(self):
        """The reserved tokens become part of the sequences."""
        if self._reserved is None:
            raise GAEError(1, "PagedKVCache: commit without reserve")
        self.lens.copy_(self.next_lens)
        self.lengths = [a + b for a, b in zip(self.lengths, self._reserved)]
        self._reserved = None

    def refresh(self):
        """Takes the host's lengths from the device (after replays; synchronises).
        Raises where replays went past max_len: tokens beyond the pages are lost."""
        self.lengths = self.lens.tolist()
        if max(self.lengths) > self.max_len:
            raise GAEError(1, f"PagedKVCache: {max(self.lengths)} positions, room for {self.max_len}")

    def evict(self):
        """Brings every sequence back to the budget, if any is longer.  Returns
        the kept positions per layer (int32 [B, Hkv, budget], -1 beyond the new
        length), or None where there was nothing to do."""
        if self.budget is None:
            raise GAEError(1, "PagedKVCache: evict without a budget")
        if self._reserved is not None:
            raise GAEError(1, "PagedKVCache: evict between reserve and commit")
        if max(self.lengths) <= self.budget:
            return None
        kept = []
        for k, v, w in zip(self.k, self.v, self.weights):
            lens, pos, left = paged_evict(k, v, self.table, self.lens, w, self.spare, keep=self.budget,
                                          recent=self.recent)
            w[:, :, : self.budget].copy_(left)
            w[:, :, self.budget:].zero_()
            kept.append(pos)
        # The kept rows lie in the spare pages: they change places with the first ones.
        n = self.spare.shape[1]
        first = self.table[:, :n].clone()
        self.table[:, :n].copy_(self.spare)
        self.spare.copy_(first)
        self.lens.copy_(lens)
        self.next_lens.copy_(lens)
        self.lengths = [min(a, self.budget) for a in self.lengths]
        return kept
