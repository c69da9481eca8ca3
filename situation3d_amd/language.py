"""Operators of the language head behind the point branch (Blip2T5.forward, blip2_t5.py:102-183), for training it and for
answering with it: attention with a learned relative position bias, the key / value cache, and attention of new tokens over
that cache for many questions about one scene.

The reference hands `inputs_t5` to a vendored T5 (modeling_t5.py), whose attention materialises the (b, heads, nq, nk) bias,
scores and probabilities; blip2.Blip2PointQFormer takes a `language_head` callable in its place.  These are the operators such
a head is built from, as hand-written HIP kernels (csrc/rel_attention.hip, kv_cache.hip, decode_attention.hip):

    relative_attention(q, k, v, table, ...)      prompts and training, forward and backward
    KVCache(...).append(k, v) / .read()          tokens into the cache (8 bits or the model's type) and back
    decode_attention(q, cache, shared, table)    the next tokens of a batch, over a scene prefix that the batch shares

Types: float32 (exact-f32 matrix instructions), bfloat16, float16; head sizes 64, 96, 128; grouped key heads (h a multiple of
hkv).  Statistics, sums and gradients' accumulators are float32; results are rounded once.  All calls run on the current
stream of their tensors' device, allocate their outputs and workspaces from torch, never synchronise, and may be captured into
a hipGraph.  GPU tensors only, like the rest of the HIP path.
"""
import ctypes
import functools
import math

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HEAD_SIZES = (64, 96, 128)


@functools.lru_cache(maxsize=64)
def relative_borders(buckets, max_distance, bidirectional):
    """(smallest distance of each bucket of one direction), from whole numbers alone.

    One direction has n = buckets // 2 (bidirectional) or buckets; the first e = n // 2 distances have a bucket each, beyond
    them distance a has bucket e + floor((n - e) log(a / e) / log(max_distance / e)), at most n - 1 (modeling_t5.py's
    _relative_position_bucket).  Bucket e + i therefore starts at the smallest a with a^(n-e) e^i >= e^(n-e) max_distance^i:
    no logarithm decides a border."""
    n = buckets // 2 if bidirectional else buckets
    e = n // 2
    if buckets < 1 or e < 1 or max_distance <= e:
        raise RuntimeError("relative position buckets need at least 2 buckets a direction and max_distance beyond half of "
                           "them: got %d buckets, max_distance %d" % (buckets, max_distance))
    if n > _lib.REL_MAX_BUCKETS:
        raise RuntimeError("at most %d relative position buckets a direction" % _lib.REL_MAX_BUCKETS)
    found = list(range(e + 1))
    for i in range(1, n - e):
        a = found[-1]
        while a ** (n - e) * e ** i < max_distance ** i * e ** (n - e):
            a += 1
        found.append(a)
    if found[n - 1] > _lib.REL_MAX_REACH:
        raise RuntimeError("the last relative position bucket must start at a distance of at most %d" % _lib.REL_MAX_REACH)
    return tuple(found[:n])


@functools.lru_cache(maxsize=64)
def _bucket_struct(buckets, max_distance, bidirectional):
    s = _lib.RelBuckets()
    if buckets:
        border = relative_borders(buckets, max_distance, bidirectional)
        s.n, s.both = len(border), int(bool(bidirectional))
        s.border[:len(border)] = border
    return s


def _dense_rows(t):
    """(tensor, its strides but the innermost) with rows as the kernels read them: dense, 16-byte aligned; copied if not."""
    for _ in range(2):
        e = t.element_size()
        strides = [0 if n == 1 else s for n, s in zip(t.shape[:-1], t.stride()[:-1])]
        if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * e % 16 == 0 for s in strides) and strides[1] * e < 1 << 24:
            return t, strides
        t = t.clone(memory_format=torch.contiguous_format)
    raise RuntimeError("could not lay out a tensor of shape %s" % (tuple(t.shape),))


def _check_heads(q, k, v, what):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise RuntimeError("%s takes (batch, tokens, heads, head size) tensors" % what)
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError("%s: q, k, v must share one of float32, bfloat16, float16" % what)
    if q.shape[3] not in _HEAD_SIZES:
        raise RuntimeError("%s: head size %d, the HIP kernels are built for 64, 96 and 128" % (what, q.shape[3]))
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise RuntimeError("%s: q %s, k %s, v %s do not belong together" % (what, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise RuntimeError("%s: %d heads over %d key heads" % (what, q.shape[2], k.shape[2]))


def _check_table(table, q, what):
    if table is not None and (table.dim() != 2 or table.shape[1] != q.shape[2] or table.dtype != q.dtype):
        raise RuntimeError("%s: the bias table is (buckets, heads) = (., %d) in q's type" % (what, q.shape[2]))


def _int_array(t, shape, device, name):
    if t is None:
        return None
    if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != device:
        raise RuntimeError("%s must be an int32 tensor of shape %s on %s" % (name, shape, device))
    return t.contiguous()


def document_ranges(documents):
    """documents (b, n): ids of packed documents, the tokens of one side by side -> key_ranges (b, n, 2) int32 for
    relative_attention: a token sees its own document alone.  Computed once a batch, for all layers."""
    n = documents.shape[1]
    at = torch.arange(n, device=documents.device).expand(documents.shape)
    new = torch.ones_like(documents, dtype=torch.bool)
    new[:, 1:] = documents[:, 1:] != documents[:, :-1]
    start = torch.where(new, at, 0).cummax(1).values
    last = torch.ones_like(new)
    last[:, :-1] = new[:, 1:]
    end = torch.where(last, at + 1, n).flip(1).cummin(1).values.flip(1)
    return torch.stack([start, end], -1).to(torch.int32)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rel_args(q, k, v, table, cfg, arrays, out, out32, lse, grad=None, grads=(None,) * 4, work=None):
    scale, bidirectional, max_distance, causal, offset = cfg
    q, qs = _dense_rows(q)
    k, ks = _dense_rows(k)
    v, vs = _dense_rows(v)
    gs = [0, 0, 0]
    if grad is not None:
        grad, gs = _dense_rows(grad)
    b, nq, h, d = q.shape
    rows = 0 if table is None else table.shape[0]
    a = _lib.RelAttentionArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(table), *[_ptr(x) for x in arrays], _ptr(out), _ptr(out32), _ptr(lse),
        _ptr(grad), *[_ptr(x) for x in grads], _ptr(work), *qs, *ks, *vs, *gs, _DTYPES[q.dtype], b, nq, k.shape[1], h, k.shape[2], d,
        int(causal), offset, rows, scale, _bucket_struct(rows, max_distance, bidirectional))
    return a, (q, k, v, grad)                  # copies that the strides belong to live until the launch


def _rel_forward(q, k, v, table, cfg, arrays, keep):
    dev = q.device
    b, nq, h, d = q.shape
    out = torch.empty((b, nq, h, d), dtype=q.dtype, device=dev)
    # the unrounded output: delta = dO.O decides dS where one key has almost all of a row, and O rounded to 8 bits would not do
    out32 = torch.empty((b, nq, h, d), dtype=torch.float32, device=dev) if keep else None
    lse = torch.empty((b, h, nq), dtype=torch.float32, device=dev) if keep else None
    if out.numel() == 0:
        return out, out32, lse
    if k.shape[1] == 0:
        return out.zero_(), out32.zero_() if keep else None, lse
    a, held = _rel_args(q, k, v, table, cfg, arrays, out, out32, lse)
    with torch.cuda.device(dev):
        _lib.call("sig3d_rel_attention_fwd", ctypes.byref(a), _lib.stream_ptr(dev))
    del held
    return out, out32, lse


class _RelativeAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, cfg, arrays):
        out, out32, lse = _rel_forward(q, k, v, table, cfg, arrays, True)
        ctx.save_for_backward(q, k, v, table, out, out32, lse, *arrays)
        ctx.cfg = cfg
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, table, out, out32, lse, *arrays = ctx.saved_tensors
        dev = q.device
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        dk, dv = torch.empty(k.shape, dtype=k.dtype, device=dev), torch.empty(v.shape, dtype=v.dtype, device=dev)
        dtable = None if table is None else torch.empty_like(table, memory_format=torch.contiguous_format)
        if q.numel() == 0 or k.numel() == 0:
            for t in (dq, dk, dv, dtable):
                if t is not None:
                    t.zero_()
            return dq, dk, dv, dtable, None, None
        # the query layout of `out` is dense: it names the strides, the kernels read out32
        a, held = _rel_args(q, k, v, table, ctx.cfg, arrays, out, out32, lse, grad, (dq, dk, dv, dtable))
        work = torch.empty(_lib.load().sig3d_rel_attention_bwd_work_floats(ctypes.byref(a)), dtype=torch.float32, device=dev)
        a.work = work.data_ptr()
        with torch.cuda.device(dev):
            _lib.call("sig3d_rel_attention_bwd", ctypes.byref(a), _lib.stream_ptr(dev))
        del held
        return dq, dk, dv, dtable, None, None


def relative_attention(q, k, v, table=None, *, scale=None, bidirectional=True, max_distance=128, causal=False, query_offset=0,
                       key_lengths=None, prefix_lengths=None, key_ranges=None):
    """softmax(scale q k^T + bias) v over the keys that each query sees; gradients for q, k, v and table.

    q (b, nq, h, d), k / v (b, nk, hkv, d), hkv dividing h: head i reads key head i // (h / hkv).  Query i stands at position
    p = i + query_offset, key j at j.
    table (buckets, h) in q's type, or None: the learned bias, table[bucket(j - p), head] (relative_borders has the buckets;
      T5's `relative_attention_bias.weight`).  bidirectional: keys ahead of the query have half of the buckets, else they share
      bucket 0.  T5 does not scale: pass scale=1.0 there; None is d ** -0.5.
    What a query sees: j < key_lengths[b] (b,), and with causal j <= p or j < prefix_lengths[b] (b,), and
      key_ranges[b, i, 0] <= j < key_ranges[b, i, 1] (b, nq, 2), all int32 on q's device; None does not restrict.  A query that
      sees nothing yields 0 and passes no gradient.  Keys that no query sees may hold anything; a key that some query sees
      must be finite for the others.
    -> (b, nq, h, d) in q's type."""
    dev = _lib.require_device(q, k, v, table, key_lengths, prefix_lengths, key_ranges)
    _check_heads(q, k, v, "relative_attention")
    _check_table(table, q, "relative_attention")
    if prefix_lengths is not None and not causal:
        raise RuntimeError("relative_attention: prefix_lengths only means something with causal=True")
    b, nq = q.shape[:2]
    arrays = (_int_array(key_lengths, (b,), dev, "key_lengths"), _int_array(prefix_lengths, (b,), dev, "prefix_lengths"),
              _int_array(key_ranges, (b, nq, 2), dev, "key_ranges"))
    cfg = (float(q.shape[3] ** -0.5 if scale is None else scale), bool(bidirectional), int(max_distance), bool(causal),
           int(query_offset))
    if not math.isfinite(cfg[0]):
        raise RuntimeError("relative_attention: scale must be finite")
    if table is not None:
        _bucket_struct(table.shape[0], cfg[2], cfg[1])         # refuses here, not inside backward
        table = table.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or table is not None and table.requires_grad):
        return _RelativeAttentionFn.apply(q, k, v, table, cfg, arrays)
    return _rel_forward(q, k, v, table, cfg, arrays, False)[0]


class KVCache:
    """Keys and values of `batch` sequences, `capacity` tokens each.

    quantized: held as float8_e4m3fn with one float32 scale per (token, head), the smallest power of two with
    max |x| <= 448 scale -- half the bytes of bfloat16; one rounding to 4 significant bits, at most 2^-4 of a value.  Else held
    in `dtype`.  Attributes: k, v (batch, capacity, kv_heads, head_dim), k_scale, v_scale (batch, capacity, kv_heads) or
    None, lengths (batch,) int32 -- tensors of fixed address that the program may read and write (scales must stay powers of
    two), and that captured graphs may keep using.  They are views of head-major storage."""

    def __init__(self, batch, capacity, kv_heads, head_dim, dtype=torch.bfloat16, quantized=False, device="cuda"):
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("CPU not supported")
        if dtype not in _DTYPES or head_dim not in _HEAD_SIZES:
            raise RuntimeError("KVCache: float32, bfloat16 or float16 and head sizes 64, 96, 128")
        if not (1 <= batch <= 65535 and 1 <= kv_heads <= 65535 and 1 <= capacity <= 1 << 29):
            raise RuntimeError("KVCache: sizes out of range: %d sequences of %d tokens, %d heads" % (batch, capacity, kv_heads))
        self.batch, self.capacity, self.kv_heads, self.head_dim, self.dtype, self.quantized = \
            batch, capacity, kv_heads, head_dim, dtype, bool(quantized)
        held = torch.float8_e4m3fn if quantized else dtype
        self._k, self._v = (torch.empty((batch, kv_heads, capacity, head_dim), dtype=held, device=device) for _ in range(2))
        self._ks = self._vs = None
        if quantized:
            self._ks, self._vs = (torch.ones((batch, kv_heads, capacity), dtype=torch.float32, device=device) for _ in range(2))
        self.k, self.v = self._k.transpose(1, 2), self._v.transpose(1, 2)
        self.k_scale = self._ks.transpose(1, 2) if quantized else None
        self.v_scale = self._vs.transpose(1, 2) if quantized else None
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.device = self.lengths.device

    def append(self, k, v, start=None, counts=None):
        """Tokens k, v (batch, t, kv_heads, head_dim) in the cache's type: the first counts[b] (None: t) go to rows
        start[b] + i (None: behind what is there), and lengths[b] becomes start[b] + counts[b]; both int32 (batch,).  Tokens
        beyond the capacity are dropped and lengths stops there; other rows stay as they are."""
        dev = _lib.require_device(k, v, self.lengths, start, counts)
        if k.dim() != 4 or k.shape != v.shape or k.shape[0] != self.batch or tuple(k.shape[2:]) != (self.kv_heads, self.head_dim):
            raise RuntimeError("KVCache.append: k and v must be (%d, t, %d, %d)" % (self.batch, self.kv_heads, self.head_dim))
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise RuntimeError("KVCache.append: the cache takes %s" % self.dtype)
        start, counts = _int_array(start, (self.batch,), dev, "start"), _int_array(counts, (self.batch,), dev, "counts")
        t = k.shape[1]
        if t == 0:
            if start is not None:
                self.lengths.copy_(start.clamp(0, self.capacity))
            return
        k, ks = _dense_rows(k.detach())
        v, vs = _dense_rows(v.detach())
        a = _lib.CacheAppendArgs(k.data_ptr(), v.data_ptr(), self._k.data_ptr(), self._v.data_ptr(), _ptr(self._ks), _ptr(self._vs),
                                 _ptr(start), _ptr(counts), self.lengths.data_ptr(), *ks, *vs, _DTYPES[self.dtype], self.batch, t,
                                 self.capacity, self.kv_heads, self.head_dim)
        with torch.cuda.device(dev):
            _lib.call("sig3d_cache_append", ctypes.byref(a), _lib.stream_ptr(dev))

    def read(self, tokens=None):
        """(k, v) (batch, tokens, kv_heads, head_dim) in the cache's type: the values that the first `tokens` rows (None: all)
        stand for, zeros from lengths on."""
        n = self.capacity if tokens is None else int(tokens)
        if not 0 <= n <= self.capacity:
            raise RuntimeError("KVCache.read: %d of %d rows" % (n, self.capacity))
        k, v = (torch.empty((self.batch, n, self.kv_heads, self.head_dim), dtype=self.dtype, device=self.device) for _ in range(2))
        if n:
            with torch.cuda.device(self.device):
                _lib.call("sig3d_cache_read", _DTYPES[self.dtype], self.batch, n, self.capacity, self.kv_heads, self.head_dim,
                          self._k.data_ptr(), self._v.data_ptr(), _ptr(self._ks), _ptr(self._vs), self.lengths.data_ptr(),
                          k.data_ptr(), v.data_ptr(), _lib.stream_ptr(self.device))
        return k, v


def decode_attention(q, cache, shared=None, table=None, *, scale=None, bidirectional=False, max_distance=128, counts=None):
    """Attention of the newest tokens of every sequence; inference only.

    q (b, t, h, d): queries of the t tokens that were last appended to `cache` (KVCache of b sequences, of q's type).  With
      counts (b,) int32, sequence i has counts[i] <= t of them, in the first rows of q; the other rows of the result are 0.
    shared: KVCache of g sequences held like `cache`, g dividing b: sequence i also sees shared sequence i // (b / g), wholly
      and before its own tokens -- b / g questions about one scene, read from memory once for all of them.
    table as in relative_attention (keys are never ahead of the query, so bidirectional only says which half of the table
      counts); positions count the shared tokens first.
    -> (b, t, h, d) in q's type."""
    dev = _lib.require_device(q, cache.lengths, None if shared is None else shared.lengths, table, counts)
    what = "decode_attention"
    if q.dim() != 4 or q.dtype != cache.dtype:
        raise RuntimeError("%s: q is (batch, new tokens, heads, head size) in the cache's type" % what)
    b, t, h, d = q.shape
    if b != cache.batch or d != cache.head_dim or h == 0 or h % cache.kv_heads:
        raise RuntimeError("%s: q %s does not belong to a cache of %d sequences, %d heads of %d" % (
            what, tuple(q.shape), cache.batch, cache.kv_heads, cache.head_dim))
    if shared is not None and (shared.dtype != cache.dtype or shared.quantized != cache.quantized or shared.kv_heads != cache.kv_heads
                               or shared.head_dim != d or b % shared.batch):
        raise RuntimeError("%s: the shared sequences must be held like the cache's, their number dividing %d" % (what, b))
    _check_table(table, q, what)
    counts = _int_array(counts, (b,), dev, "counts")
    q, qs = _dense_rows(q.detach())
    out = torch.empty((b, t, h, d), dtype=q.dtype, device=dev)
    if t == 0:
        return out
    rows = 0
    if table is not None:
        table, rows = table.detach().contiguous(), table.shape[0]
    s = shared
    a = _lib.DecodeAttentionArgs(
        q.data_ptr(), _ptr(table), cache._k.data_ptr(), cache._v.data_ptr(), _ptr(s and s._k), _ptr(s and s._v), _ptr(cache._ks),
        _ptr(cache._vs), _ptr(s and s._ks), _ptr(s and s._vs), cache.lengths.data_ptr(), _ptr(s and s.lengths), _ptr(counts),
        out.data_ptr(), None, *qs, _DTYPES[q.dtype], b, t, h, cache.kv_heads, d, cache.capacity, s.batch if s else 0,
        s.capacity if s else 0, rows, float(d ** -0.5 if scale is None else scale), _bucket_struct(rows, max_distance, bool(bidirectional)))
    need = _lib.load().sig3d_decode_attention_work_floats(ctypes.byref(a))
    if need:
        work = torch.empty(need, dtype=torch.float32, device=dev)
        a.work = work.data_ptr()
    with torch.cuda.device(dev):
        _lib.call("sig3d_decode_attention", ctypes.byref(a), _lib.stream_ptr(dev))
    return out
