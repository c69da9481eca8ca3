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
a hipGraph (a backward pass like any other of torch's: no eager graph of the same leaves may be alive meanwhile, so make the leaves
inside the capture).  The same call gives the same bits; how a sum is cut, and in 16 bits how P is rounded (relative_attention),
follows from the launch's size, so the last bit of a sequence's result may depend on the batch around it.  GPU tensors only, like
the rest of the HIP path.
"""
import functools

import torch
from torch.autograd import forward_ad

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
            if a > _lib.REL_MAX_REACH:
                raise RuntimeError("the last relative position bucket must start at a distance of at most %d" % _lib.REL_MAX_REACH)
        found.append(a)
    return tuple(found[:n])


@functools.lru_cache(maxsize=64)
def _bucket_struct(buckets, max_distance, bidirectional):
    s = _lib.RelBuckets()
    if buckets:
        border = relative_borders(buckets, max_distance, bidirectional)
        s.n, s.both = len(border), int(bool(bidirectional))
        s.border[:len(border)] = border
    return s


def _readable(shape, stride, itemsize):
    """Rows as the kernels read them: dense, strides multiples of 16 bytes, a token's below 16 MB; strides of dimensions of one do
    not matter."""
    return (stride[-1] == 1 or shape[-1] == 1) and all(n == 1 or s >= 0 and s * itemsize % 16 == 0 for n, s in
                                                      zip(shape[:-1], stride[:-1])) and (shape[1] == 1 or stride[1] * itemsize < 1 << 24)


def _strides(shape, stride):
    b, n, h, _ = shape
    return 0 if b == 1 else stride[0], 0 if n == 1 else stride[1], 0 if h == 1 else stride[2]


def _rows(t):
    """`t`, or a dense copy where the kernels cannot read its rows (differentiable)."""
    if t.data_ptr() % 16 == 0 and (t.is_contiguous() and t.numel() or _readable(t.shape, t.stride(), t.element_size())):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _new(like, dtype=None):
    return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)


def _launch(name, args, device):
    """One library call on the current stream of `device`."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        _lib.call(name, args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            _lib.call(name, args, torch._C._cuda_getCurrentRawStream(index))


def _check_numbers(what, scale, *integers):
    """An argument struct takes what does not fit modulo 2^32, and a scale beyond float32 (in log2 units) as infinity."""
    if not all(-1 << 31 <= n < 1 << 31 for n in integers):
        raise RuntimeError("%s: sizes and positions must be below 2^31" % what)
    if not abs(scale) < 2.0 ** 127:
        raise RuntimeError("%s: scale must be finite" % what)


def _check_heads(q, k, v, dtypes, what):
    if len(q) != 4 or len(k) != 4 or len(v) != 4:
        raise RuntimeError("%s takes (batch, tokens, heads, head size) tensors" % what)
    if dtypes[0] not in _DTYPES or len(set(dtypes)) != 1:
        raise RuntimeError("%s: q, k, v must share one of float32, bfloat16, float16" % what)
    if q[3] not in _HEAD_SIZES:
        raise RuntimeError("%s: head size %d, the HIP kernels are built for 64, 96 and 128" % (what, q[3]))
    if k != v or k[0] != q[0] or k[3] != q[3]:
        raise RuntimeError("%s: q %s, k %s, v %s do not belong together" % (what, tuple(q), tuple(k), tuple(v)))
    if k[2] == 0 or q[2] % k[2]:
        raise RuntimeError("%s: %d heads over %d key heads" % (what, q[2], k[2]))


def _check_table(shape, dtype, heads, q_dtype, what):
    if shape is not None and (len(shape) != 2 or shape[1] != heads or dtype != q_dtype):
        raise RuntimeError("%s: the bias table is (buckets, heads) = (., %d) in q's type" % (what, heads))


def _no_gradient(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("%s has no gradient: call it under torch.no_grad()" % what)


def _no_tangent(what, *tensors):
    """A dual tensor does not show in requires_grad: its tangent would be dropped."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("%s has no forward-mode derivative" % what)


def _int_array(t, shape, device, name):
    if t is None:
        return None
    if t.dtype != torch.int32 or t.shape != shape or t.device != device:
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


@functools.lru_cache(maxsize=1024)
def _rel_template(q, qs, k, ks, v, vs, dtypes, table, table_dtype, cfg):
    """Everything about a call that shapes, strides and types decide, checked once: the argument struct without its addresses,
    whether q, k, v can be read as they are, and the floats of workspace forward and backward."""
    _check_heads(q, k, v, dtypes, "relative_attention")
    _check_table(table, table_dtype, q[2], dtypes[0], "relative_attention")
    scale, bidirectional, max_distance, causal, offset = cfg
    _check_numbers("relative_attention", scale, offset, *q, *k)
    rows = 0 if table is None else table[0]
    e = dtypes[0].itemsize
    a = _lib.RelAttentionArgs(dtype=_DTYPES[dtypes[0]], b=q[0], nq=q[1], nk=k[1], h=q[2], hkv=k[2], d=q[3], causal=int(causal),
                              query_offset=offset, table_rows=rows, scale=scale,
                              buckets=_bucket_struct(rows, max_distance, bidirectional))
    for name, shape, stride in (("q", q, qs), ("k", k, ks), ("v", v, vs)):
        for dim, s in zip("bnh", _strides(shape, stride)):
            setattr(a, "%s_%s" % (name, dim), s)
    ok = all(_readable(*x, e) for x in ((q, qs), (k, ks), (v, vs)))
    work = (0, 0)
    if ok and q[0] and q[1] and k[1]:
        a.q = a.k = a.v = a.out = a.table = 16           # the sizes do not depend on addresses, only on there being some
        work = tuple(f(a) for f in (_lib.load().sig3d_rel_attention_fwd_work_floats, _lib.load().sig3d_rel_attention_bwd_work_floats))
        if min(work) < 0:
            raise RuntimeError("relative_attention: " + _lib.load().sig3d_last_error().decode())
        a.q = a.k = a.v = a.out = a.table = None
    return a, ok, work


def _rel_args(q, k, v, table, cfg, arrays):
    """(argument struct, readable, workspaces): see _rel_template."""
    a, ok, work = _rel_template(q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), (q.dtype, k.dtype, v.dtype),
                          None if table is None else table.shape, None if table is None else table.dtype, cfg)
    a = _lib.RelAttentionArgs.from_buffer_copy(a)
    a.q, a.k, a.v = qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if table is not None:
        a.table = table.data_ptr()
    lengths, prefix, ranges = arrays
    if lengths is not None:
        a.key_lengths = lengths.data_ptr()
    if prefix is not None:
        a.prefix_lengths = prefix.data_ptr()
    if ranges is not None:
        a.key_ranges = ranges.data_ptr()
    return a, ok and not (qp | kp | vp) & 15, work


def _rel_forward(a, q, k, keep, need):
    b, nq, h, _ = q.shape
    dev = q.device
    out = _new(q)
    # the unrounded output: delta = dO.O decides dS where one key has almost all of a row, and O rounded to 8 bits would not do
    out32 = _new(q, torch.float32) if keep else None
    lse = torch.empty((b, h, nq), dtype=torch.float32, device=dev) if keep else None
    if out.numel() == 0:
        return out, out32, lse
    if k.shape[1] == 0:
        return out.zero_(), out32.zero_() if keep else None, lse
    a.out = out.data_ptr()
    if need:
        work = torch.empty(need, dtype=torch.float32, device=dev)
        a.work = work.data_ptr()
    if keep:
        a.out32, a.lse = out32.data_ptr(), lse.data_ptr()
    _launch("sig3d_rel_attention_fwd", a, dev)
    return out, out32, lse


class _RelativeAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, cfg, arrays, a, work):
        out, out32, lse = _rel_forward(a, q, k, True, work[0])
        ctx.save_for_backward(q, k, v, table, out32, lse, *arrays)
        ctx.call = cfg, a, work, (q.stride(), k.stride(), v.stride())
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_tangent("relative_attention's backward pass", grad)
        q, k, v, table, out32, lse, *arrays = ctx.saved_tensors
        cfg, a, work, strides = ctx.call
        dev = q.device
        dq, dk, dv, dtable = _new(q), _new(k), _new(v), None if table is None else _new(table)
        if q.numel() == 0 or k.numel() == 0:
            for t in (dq, dk, dv, dtable):
                if t is not None:
                    t.zero_()
            return dq, dk, dv, dtable, None, None, None, None
        if (q.data_ptr(), k.data_ptr(), v.data_ptr()) == (a.q, a.k, a.v) and (q.stride(), k.stride(), v.stride()) == strides:
            a = _lib.RelAttentionArgs.from_buffer_copy(a)
        else:                                    # saved tensors came back from elsewhere (hooks)
            a, ok, work = _rel_args(q, k, v, table, cfg, arrays)
            if not ok:
                q, k, v = _rows(q), _rows(k), _rows(v)
                a, _, work = _rel_args(q, k, v, table, cfg, arrays)
        grad = _rows(grad)
        a.grad_b, a.grad_n, a.grad_h = _strides(grad.shape, grad.stride())
        # (out is not read again: the kernels take the unrounded copy; its address only has to be one)
        a.out = a.out32 = out32.data_ptr()
        a.lse, a.grad, a.dq, a.dk, a.dv = lse.data_ptr(), grad.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        if dtable is not None:
            a.table, a.dtable = table.data_ptr(), dtable.data_ptr()
        for name, x in zip(("key_lengths", "prefix_lengths", "key_ranges"), arrays):
            if x is not None:
                setattr(a, name, x.data_ptr())
        work = torch.empty(work[1], dtype=torch.float32, device=dev)
        a.work = work.data_ptr()
        _launch("sig3d_rel_attention_bwd", a, dev)
        return dq, dk, dv, dtable, None, None, None, None


def relative_attention(q, k, v, table=None, *, scale=None, bidirectional=True, max_distance=128, causal=False, query_offset=0,
                       key_lengths=None, prefix_lengths=None, key_ranges=None):
    """softmax(scale q k^T + bias) v over the keys that each query sees; gradients for q, k, v and table (first derivatives in
    reverse mode: a second one and forward mode are refused).

    q (b, nq, h, d), k / v (b, nk, hkv, d), hkv dividing h: head i reads key head i // (h / hkv).  Query i stands at position
    p = i + query_offset, key j at j.
    table (buckets, h) in q's type, or None: the learned bias, table[bucket(j - p), head] (relative_borders has the buckets;
      T5's `relative_attention_bias.weight`).  bidirectional: keys ahead of the query have half of the buckets, else they share
      bucket 0.  T5 does not scale: pass scale=1.0 there; None is d ** -0.5.
    What a query sees: j < key_lengths[b] (b,), and with causal j <= p or j < prefix_lengths[b] (b,), and
      key_ranges[b, i, 0] <= j < key_ranges[b, i, 1] (b, nq, 2), all int32 on q's device; None does not restrict.  A query that
      sees nothing yields 0 and passes no gradient.  Keys before the first and behind the last that any query of the sequence
      sees may hold anything; those between are finite, also for queries that do not see them.
    A bias of -inf weighs nothing, and neither do float32's and bfloat16's lowest values; a query that sees only such keys
      yields 0 as well.
    Rounding in 16 bits: P meets V with 16 bits of its own, and once more with what that left, where a backward pass follows or the
      launch is small; in large launches without one it is rounded once (the result's error 1.4 of one rounding instead of 1.0, so
      a checkpointed layer's two forward passes differ by that).  There is no dropout of probabilities.
    -> (b, nq, h, d) in q's type."""
    dev = q.device
    if not q.is_cuda:
        raise RuntimeError("CPU not supported")
    if k.device != dev or v.device != dev or table is not None and table.device != dev:
        raise RuntimeError("all tensors must be on the same device")
    _no_tangent("relative_attention", q, k, v, table)
    if prefix_lengths is not None and not causal:
        raise RuntimeError("relative_attention: prefix_lengths only means something with causal=True")
    if q.dim() != 4 or q.shape[3] not in _HEAD_SIZES:
        raise RuntimeError("relative_attention: q must be (batch, tokens, heads, head size), the head size 64, 96 or 128")
    cfg = (float(q.shape[3] ** -0.5 if scale is None else scale), bool(bidirectional), int(max_distance), bool(causal),
           int(query_offset))
    if table is not None:
        table = table.contiguous()
    none = (None, None, None)
    a, ok, work = _rel_args(q, k, v, table, cfg, none)
    b, nq = q.shape[:2]
    arrays = none
    if key_lengths is not None or prefix_lengths is not None or key_ranges is not None:
        arrays = (_int_array(key_lengths, (b,), dev, "key_lengths"), _int_array(prefix_lengths, (b,), dev, "prefix_lengths"),
                  _int_array(key_ranges, (b, nq, 2), dev, "key_ranges"))
        a.key_lengths, a.prefix_lengths, a.key_ranges = (None if x is None else x.data_ptr() for x in arrays)
    if not ok:
        q, k, v = _rows(q), _rows(k), _rows(v)
        a, ok, work = _rel_args(q, k, v, table, cfg, arrays)
        if not ok:
            raise RuntimeError("relative_attention: a token's heads must be below 16 MB")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or table is not None and table.requires_grad):
        return _RelativeAttentionFn.apply(q, k, v, table, cfg, arrays, a, work)
    return _rel_forward(a, q, k, False, work[0])[0]


class KVCache:
    """Keys and values of `batch` sequences, `capacity` tokens each.

    quantized: held as float8_e4m3fn with one float32 scale per (token, head), the smallest power of two with
    max |x| <= 448 scale -- half the bytes of bfloat16; one rounding to 4 significant bits, at most 2^-4 of a value.  Else held
    in `dtype`.  Attributes: k, v (batch, capacity, kv_heads, head_dim), k_scale, v_scale (batch, capacity, kv_heads) or
    None, lengths (batch,) int32 -- tensors of fixed address that the program may read and write (scales must stay powers of
    two), and that captured graphs may keep using.  They are views of head-major storage.  Inference only: no gradients."""

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
        self._lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.device = self._lengths.device
        # where the storage lies (what an append writes is not read beside it), and the calls' arguments without the tokens'
        self._spans = [(x.data_ptr(), x.data_ptr() + x.numel() * x.element_size()) for x in (self._k, self._v, self._lengths)]
        self._append = _lib.CacheAppendArgs(
            k_cache=self._k.data_ptr(), v_cache=self._v.data_ptr(), k_scale=_ptr(self._ks), v_scale=_ptr(self._vs),
            lengths=self._lengths.data_ptr(), dtype=_DTYPES[dtype], b=batch, capacity=capacity, hkv=kv_heads, d=head_dim)
        self._read = _lib.CacheReadArgs(
            k_cache=self._k.data_ptr(), v_cache=self._v.data_ptr(), k_scale=_ptr(self._ks), v_scale=_ptr(self._vs),
            lengths=self._lengths.data_ptr(), dtype=_DTYPES[dtype], b=batch, capacity=capacity, hkv=kv_heads, d=head_dim)

    def _apart(self, t):
        p = t.data_ptr()
        return t.clone() if any(lo <= p < hi for lo, hi in self._spans) else t

    # (nothing to assign to: the kernels use the storage)
    k = property(lambda self: self._k.transpose(1, 2))
    v = property(lambda self: self._v.transpose(1, 2))
    k_scale = property(lambda self: None if self._ks is None else self._ks.transpose(1, 2))
    v_scale = property(lambda self: None if self._vs is None else self._vs.transpose(1, 2))
    lengths = property(lambda self: self._lengths)

    def append(self, k, v, start=None, counts=None):
        """Tokens k, v (batch, t, kv_heads, head_dim) in the cache's type: the first counts[b] (None: t) go to rows
        start[b] + i (None: behind what is there), and lengths[b] becomes start[b] + counts[b]; both int32 (batch,).  Tokens
        beyond the capacity are dropped and lengths stops there; other rows stay as they are."""
        dev = self.device
        if not k.is_cuda or not v.is_cuda:
            raise RuntimeError("CPU not supported")
        if k.device != dev or v.device != dev:
            raise RuntimeError("all tensors must be on the same device")
        if k.requires_grad or v.requires_grad:
            _no_gradient("KVCache.append", k, v)
        _no_tangent("KVCache.append", k, v)
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or shape[0] != self.batch or shape[2:] != (self.kv_heads, self.head_dim):
            raise RuntimeError("KVCache.append: k and v must be (%d, t, %d, %d)" % (self.batch, self.kv_heads, self.head_dim))
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise RuntimeError("KVCache.append: the cache takes %s" % self.dtype)
        start, counts = _int_array(start, (self.batch,), dev, "start"), _int_array(counts, (self.batch,), dev, "counts")
        if shape[1] >= 1 << 31:                          # (broadcast: the struct would take them modulo 2^32)
            raise RuntimeError("KVCache.append: %d tokens" % shape[1])
        if shape[1] == 0:
            if start is not None:
                self._lengths.copy_(start.clamp(0, self.capacity))
            return
        k, v = _rows(self._apart(k)), _rows(self._apart(v))
        a = _lib.CacheAppendArgs.from_buffer_copy(self._append)
        a.t, a.k, a.v = shape[1], k.data_ptr(), v.data_ptr()
        a.k_b, a.k_n, a.k_h = _strides(shape, k.stride())
        a.v_b, a.v_n, a.v_h = _strides(shape, v.stride())
        if start is not None:
            start = self._apart(start)
            a.start = start.data_ptr()
        if counts is not None:
            counts = self._apart(counts)
            a.counts = counts.data_ptr()
        _launch("sig3d_cache_append", a, dev)

    def read(self, tokens=None):
        """(k, v) (batch, tokens, kv_heads, head_dim) in the cache's type: the values that the first `tokens` rows (None: all)
        stand for, zeros from lengths on."""
        n = self.capacity if tokens is None else int(tokens)
        if not 0 <= n <= self.capacity:
            raise RuntimeError("KVCache.read: %d of %d rows" % (n, self.capacity))
        k = torch.empty((self.batch, n, self.kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        if n:
            a = _lib.CacheReadArgs.from_buffer_copy(self._read)
            a.k_out, a.v_out, a.n = k.data_ptr(), v.data_ptr(), n
            _launch("sig3d_cache_read", a, self.device)
        return k, v


def decode_attention(q, cache, shared=None, table=None, *, scale=None, bidirectional=False, max_distance=128, counts=None):
    """Attention of the newest tokens of every sequence; inference only.

    q (b, t, h, d): queries of the t tokens that were last appended to `cache` (KVCache of b sequences, of q's type).  With
      counts (b,) int32, sequence i has counts[i] <= t of them, in the first rows of q; the other rows of the result are 0.
    shared: KVCache of g sequences held like `cache`, g dividing b: sequence i also sees shared sequence i // (b / g), wholly
      and before its own tokens -- b / g questions about one scene, read from memory once for all of them.
    table as in relative_attention (keys are never ahead of the query, so bidirectional only says which half of the table
      counts); positions count the shared tokens first.
    Rows of a cache from its length on may hold anything; those before it are finite, also the newest ones for the queries before
      them.  The queries are those of the last rows held: tokens that append dropped beyond the capacity have none.
    Cross-attention of one token is decode_attention(q, cache of the encoder's keys), without a table.
    -> (b, t, h, d) in q's type."""
    dev, what = cache.device, "decode_attention"
    if not q.is_cuda or table is not None and not table.is_cuda:
        raise RuntimeError("CPU not supported")
    if q.device != dev or shared is not None and shared.device != dev or table is not None and table.device != dev:
        raise RuntimeError("all tensors must be on the same device")
    if q.requires_grad or table is not None and table.requires_grad:
        _no_gradient(what, q, table)
    _no_tangent(what, q, table)
    if q.dim() != 4 or q.dtype != cache.dtype:
        raise RuntimeError("%s: q is (batch, new tokens, heads, head size) in the cache's type" % what)
    b, t, h, d = shape = q.shape
    if b != cache.batch or d != cache.head_dim or h == 0 or h % cache.kv_heads:
        raise RuntimeError("%s: q %s does not belong to a cache of %d sequences, %d heads of %d" % (
            what, tuple(shape), cache.batch, cache.kv_heads, cache.head_dim))
    if shared is not None and (shared.dtype != cache.dtype or shared.quantized != cache.quantized or shared.kv_heads != cache.kv_heads
                               or shared.head_dim != d or b % shared.batch):
        raise RuntimeError("%s: the shared sequences must be held like the cache's, their number dividing %d" % (what, b))
    rows = 0
    if table is not None:
        _check_table(table.shape, table.dtype, h, q.dtype, what)
        table, rows = table.contiguous(), table.shape[0]
    if counts is not None:
        counts = _int_array(counts, (b,), dev, "counts")
    out = _new(q)
    if t == 0:
        return out
    q = _rows(q)
    a, need = _decode_template(shape, q.stride(), _DTYPES[q.dtype], cache.kv_heads, cache.capacity, cache.quantized,
                               shared.batch if shared is not None else 0, shared.capacity if shared is not None else 0, rows,
                               float(d ** -0.5 if scale is None else scale), int(max_distance), bool(bidirectional))
    a = _lib.DecodeAttentionArgs.from_buffer_copy(a)
    a.q, a.out, a.k_cache, a.v_cache = q.data_ptr(), out.data_ptr(), cache._k.data_ptr(), cache._v.data_ptr()
    a.lengths = cache._lengths.data_ptr()
    if cache.quantized:
        a.k_scale, a.v_scale = cache._ks.data_ptr(), cache._vs.data_ptr()
    if shared is not None:
        a.shared_k, a.shared_v, a.shared_lengths = shared._k.data_ptr(), shared._v.data_ptr(), shared._lengths.data_ptr()
        if cache.quantized:
            a.shared_k_scale, a.shared_v_scale = shared._ks.data_ptr(), shared._vs.data_ptr()
    if rows:
        a.table = table.data_ptr()
    if counts is not None:
        a.counts = counts.data_ptr()
    if need:
        work = torch.empty(need, dtype=torch.float32, device=dev)
        a.work = work.data_ptr()
    _launch("sig3d_decode_attention", a, dev)
    return out


@functools.lru_cache(maxsize=1024)
def _decode_template(q, qs, dtype, hkv, capacity, quantized, groups, shared_capacity, rows, scale, max_distance, bidirectional):
    """What shapes and types decide of a decode_attention call: its argument struct without addresses, its workspace."""
    _check_numbers("decode_attention", scale, *q)
    b, t, h, d = q
    a = _lib.DecodeAttentionArgs(dtype=dtype, b=b, t=t, h=h, hkv=hkv, d=d, capacity=capacity, groups=groups,
                                 shared_capacity=shared_capacity, table_rows=rows, scale=scale,
                                 buckets=_bucket_struct(rows, max_distance, bidirectional))
    a.q_b, a.q_n, a.q_h = _strides(q, qs)
    a.table = 16 if rows else None                    # the size does not depend on the address, only on there being one
    need = _lib.load().sig3d_decode_attention_work_floats(a)
    if need < 0:
        raise RuntimeError("decode_attention: " + _lib.load().sig3d_last_error().decode())
    a.table = None
    return a, need
