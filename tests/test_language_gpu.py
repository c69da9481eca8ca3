"""Language-side operators on the GPU against their definitions in float64 (tests/language_ref.py derives every bound)."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import language_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def _lang():
    from situation3d_amd import language
    return language


# b, nq, nk, h, hkv, d, options
ATTENTION = [
    (1, 1, 1, 1, 1, 64, {}),
    (2, 5, 3, 2, 1, 64, dict(causal=True)),
    (1, 52, 52, 12, 12, 64, {}),
    (3, 33, 70, 4, 2, 96, dict(key_lengths=(70, 0, 17))),
    (2, 130, 257, 2, 2, 128, dict(key_lengths=(257, 63), bidirectional=False)),
    (1, 300, 300, 2, 1, 64, dict(causal=True, bidirectional=False)),
    (2, 64, 192, 2, 2, 64, dict(causal=True, query_offset=128, bidirectional=False)),
    (2, 40, 20, 2, 2, 96, dict(causal=True, query_offset=-25)),          # the first rows see nothing
    (2, 200, 200, 4, 1, 128, dict(causal=True, prefix_lengths=(150, 1))),
    (2, 260, 260, 2, 2, 64, dict(documents=True, causal=True, bidirectional=False)),
    (1, 321, 321, 2, 1, 96, dict(documents=True)),
    (1, 1, 777, 2, 1, 128, dict(query_offset=776, causal=True, bidirectional=False)),
    (1, 513, 1, 2, 2, 64, {}),
    (1, 160, 160, 3, 3, 64, dict(buckets=0)),
    (1, 150, 150, 2, 2, 64, dict(buckets=7, max_distance=9)),            # an odd count: the last row has no use
    (1, 90, 400, 2, 2, 64, dict(buckets=48, max_distance=300)),
    (1, 70, 70, 2, 2, 64, dict(buckets=2, max_distance=5, bidirectional=False)),
    (1, 600, 640, 1, 1, 64, dict(buckets=64, max_distance=1000, scale=1.0)),
    (2, 100, 100, 2, 2, 64, dict(key_ranges=True)),
    (2, 150, 2100, 4, 2, 96, dict(key_lengths=(2100, 300), causal=True, query_offset=1950, bidirectional=False)),     # runs of keys
    (2, 1100, 200, 8, 2, 128, dict(key_lengths=(200, 130))),                                       # runs of queries, heads apart
]


def _attention_case(case, dtype, seed=0):
    b, nq, nk, h, hkv, d, opts = case
    opts = dict(opts)
    g = torch.Generator().manual_seed(seed)
    buckets, distance = opts.pop("buckets", 32), opts.pop("max_distance", 128)
    documents, ranges = opts.pop("documents", False), opts.pop("key_ranges", False)
    q, k, v = _randn(g, b, nq, h, d, dtype=dtype), _randn(g, b, nk, hkv, d, dtype=dtype), _randn(g, b, nk, hkv, d, dtype=dtype)
    if opts.get("scale") == 1.0:
        q = q * 0.125
    table = _randn(g, buckets, h, dtype=dtype) if buckets else None
    grad = _randn(g, b, nq, h, d, dtype=dtype)
    for name in ("key_lengths", "prefix_lengths"):
        if name in opts:
            opts[name] = _i32(*opts[name])
    if documents:
        ids = (torch.rand(b, nq, generator=g) < 0.02).int().cumsum(1).to(DEV)
        opts["key_ranges"] = _lang().document_ranges(ids)
    if ranges:            # anything: empty, reversed, beyond the ends
        r = torch.randint(-20, nk + 20, (b, nq, 2), generator=g).int()
        opts["key_ranges"] = r.to(DEV)
    ok = ref.seen(b, nq, nk, opts.get("causal", False), opts.get("query_offset", 0), opts.get("key_lengths"),
                  opts.get("prefix_lengths"), opts.get("key_ranges"))
    index = ref.bucket_matrix(nq, nk, opts.get("query_offset", 0), buckets, distance, opts.get("bidirectional", True)) if buckets else None
    opts["max_distance"] = distance
    return q, k, v, table, grad, ok, index, opts


def _check_attention(q, k, v, table, grad, ok, index, opts):
    scale = opts.get("scale") or q.shape[3] ** -0.5
    want = ref.attention(q, k, v, table, ok, scale, index, grad)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([table.detach().requires_grad_()] if table is not None else [])
    with torch.no_grad():
        ref.check("out (no grad)", _lang().relative_attention(q, k, v, table, **opts), want["out"])
    out = _lang().relative_attention(*leaves[:3], leaves[3] if table is not None else None, **opts)
    ref.check("out", out, want["out"])
    grads = torch.autograd.grad(out, leaves, grad)
    for name, x in zip(("dq", "dk", "dv", "dtable"), grads):
        ref.check(name, x, want[name])


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("n", range(len(ATTENTION)))
def test_relative_attention(n, dtype):
    _check_attention(*_attention_case(ATTENTION[n], dtype, n))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_relative_attention_longer(dtype):
    """Several workgroups a head, several tiles a wave, every tile kind."""
    _check_attention(*_attention_case((1, 1030, 1100, 2, 1, 64, dict(causal=True, query_offset=70, bidirectional=False)), dtype, 5))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_relative_attention_reads_strided_and_broadcast_inputs(dtype):
    g = torch.Generator().manual_seed(3)
    stacked = _randn(g, 2, 75, 3, 4, 64, dtype=dtype)                 # one projection's q, k, v
    table, grad = _randn(g, 32, 4, dtype=dtype), _randn(g, 2, 4, 75, 64, dtype=dtype).transpose(1, 2)
    index = ref.bucket_matrix(75, 75, 0, 32, 128, True)
    _check_attention(stacked[:, :, 0], stacked[:, :, 1], stacked[:, :, 2], table, grad, ref.seen(2, 75, 75), index, {})
    # a head slice whose rows start off 16 bytes, and keys that one row stands for in the whole batch
    odd = _randn(g, 2, 75, 4, 68, dtype=dtype)[..., 3:67]
    one = _randn(g, 1, 75, 4, 64, dtype=dtype)
    want = ref.attention(odd, one.expand(2, -1, -1, -1), one.expand(2, -1, -1, -1), table, ref.seen(2, 75, 75), 0.125, index, grad)
    leaves = [odd.detach().requires_grad_(), one.detach().requires_grad_()]
    out = _lang().relative_attention(leaves[0], leaves[1].expand(2, -1, -1, -1), leaves[1].expand(2, -1, -1, -1), table)
    ref.check("out", out, want["out"])
    dq, dkv = torch.autograd.grad(out, leaves, grad)
    ref.check("dq", dq, want["dq"])
    # the broadcast's gradient: k's and v's, summed over the batch by torch in the type: two roundings of partial sums more
    value = (want["dk"][0] + want["dv"][0]).sum(0, keepdim=True)
    bound = (want["dk"][1] + want["dv"][1]).sum(0, keepdim=True)
    parts = (want["dk"][0].abs() + want["dv"][0].abs() + want["dk"][1] + want["dv"][1]).sum(0, keepdim=True)
    ref.check("dk + dv", dkv, (value, bound + 3 * ref.half_step(dtype) * parts))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("rubbish", [math.nan, math.inf, -math.inf], ids=str)
def test_padding_may_hold_anything(dtype, rubbish):
    case = (2, 70, 150, 2, 1, 64, dict(key_lengths=(150, 41)))
    q, k, v, table, grad, ok, index, opts = _attention_case(case, dtype)
    k[1, 41:] = rubbish
    v[1, 41:] = rubbish
    _check_attention(q, k, v, table, grad, ok, index, opts)
    q, k, v, table, grad, ok, index, opts = _attention_case((1, 70, 150, 2, 1, 64, dict(causal=True)), dtype)
    k[:, 70:] = rubbish
    v[:, 70:] = rubbish
    _check_attention(q, k, v, table, grad, ok, index, opts)


def test_large_scores_do_not_overflow():
    g = torch.Generator().manual_seed(0)
    q, k, v = (_randn(g, 1, 40, 2, 64, dtype=torch.float16) for _ in range(3))
    out = _lang().relative_attention(q * 100, k * 100, v)
    assert torch.isfinite(out).all()
    best = (q.double()[0, :, 0] @ k.double()[0, :, 0].t()).argmax(1)
    top2 = (q.double()[0, :, 0] @ k.double()[0, :, 0].t()).topk(2, 1).values
    sure = (top2[:, 0] - top2[:, 1]) * 1e4 / 8 > 40
    assert torch.equal(out[0, sure, 0], v[0, best[sure], 0])


def test_gradients_against_differences():
    """The f32 kernels' gradients against differences of their own forward pass along random directions.

    A central difference over step e: truncation e^2/6 |f'''|, rounding of f over e.  With e = 2^-6 and f of order 1 built from
    f32 outputs (relative error 2^-20 at these sizes) the rounding part is 2^-14 of the summed magnitudes; e^2/6 = 4e-5 times
    third derivatives of order 1 in directions of unit length.  Both stay under 1e-3 of |grad| |direction|."""
    q, k, v, table, grad, ok, index, opts = _attention_case((1, 48, 60, 2, 1, 64, dict(causal=True, query_offset=12)), torch.float32)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, table)]
    out = _lang().relative_attention(*leaves, **opts)
    grads = torch.autograd.grad(out, leaves, grad)
    g = torch.Generator().manual_seed(9)
    for n, (x, dx) in enumerate(zip((q, k, v, table), grads)):
        way = _randn(g, *x.shape)
        way /= way.norm()

        def loss(step):
            moved = [y + step * way if i == n else y for i, y in enumerate((q, k, v, table))]
            return float((_lang().relative_attention(*moved, **opts).double() * grad.double()).sum())

        e = 2.0 ** -6
        slope = (loss(e) - loss(-e)) / (2 * e)
        assert abs(slope - float((dx.double() * way.double()).sum())) <= 1e-3 * float(dx.double().norm()), n


def test_repeated_calls_give_the_same_bits():
    q, k, v, table, grad, ok, index, opts = _attention_case((2, 300, 300, 4, 2, 64, dict(causal=True)), torch.bfloat16)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, table)]
    runs = []
    for _ in range(3):
        out = _lang().relative_attention(*leaves, **opts)
        runs.append([out.detach()] + list(torch.autograd.grad(out, leaves, grad)))
    for a in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], a))


def test_a_captured_training_step_replays():
    lang = _lang()
    q, k, v, table, grad, ok, index, opts = _attention_case((2, 140, 140, 4, 2, 64, dict(key_lengths=(140, 77))), torch.bfloat16)
    static = [x.clone() for x in (q, k, v, table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        leaves = [x.detach().requires_grad_() for x in static]
        out = lang.relative_attention(*leaves, **opts)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, grad))

    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.Generator().manual_seed(1)
    for _ in range(4):
        for s in static:
            s.copy_(_randn(g, *s.shape, dtype=s.dtype))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_calls_on_another_stream():
    lang = _lang()
    q, k, v, table, grad, ok, index, opts = _attention_case((1, 200, 200, 2, 2, 64, {}), torch.bfloat16)
    want = lang.relative_attention(q, k, v, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lang.relative_attention(q, k, v, table)
    side.synchronize()
    assert torch.equal(want, got)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_no_tokens(dtype):
    lang = _lang()
    q = torch.randn(2, 3, 2, 64, device=DEV, dtype=dtype, requires_grad=True)
    none = torch.randn(2, 0, 2, 64, device=DEV, dtype=dtype, requires_grad=True)
    out = lang.relative_attention(q, none, none)
    assert not out.any()
    dq, = torch.autograd.grad(out.sum(), [q])
    assert not dq.any()
    assert lang.relative_attention(none, q, q).shape == (2, 0, 2, 64)


# ---- cache ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("quantized", [False, True], ids=["plain", "e4m3"])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_cache_holds_what_was_written(dtype, quantized, d):
    g = torch.Generator().manual_seed(d)
    b, capacity, hkv = 3, 50, 5
    cache = _lang().KVCache(b, capacity, hkv, d, dtype, quantized, DEV)
    want = [torch.zeros(b, capacity, hkv, d, dtype=dtype, device=DEV) for _ in range(2)]
    lengths = [0] * b

    def stands_for(x):
        if not quantized:
            return x
        y, s = ref.quantized(x)
        return (y.float() * s).to(dtype)

    for t, counts, start in ((7, None, None), (1, None, None), (4, (0, 4, 2), None), (1, (1, 0, 1), None), (9, (9, 3, 9), (5, 2, 11)),
                             (33, None, None)):
        # values of very different size, zeros, an all-zero row, the largest values that a scale holds
        k = _randn(g, b, t, hkv, d) * torch.exp2(_randn(g, b, t, hkv, 1) * 3)
        v = _randn(g, b, t, hkv, d)
        k[:, :, 0] = 0
        v[0, 0, 1, :] = 448.0
        v[0, 0, 2, 0] = 449.0
        k, v = k.to(dtype), v.to(dtype)
        cache.append(k, v, start=None if start is None else _i32(*start), counts=None if counts is None else _i32(*counts))
        for i in range(b):
            at, n = (lengths[i] if start is None else start[i]), (t if counts is None else counts[i])
            for x, w in ((k, want[0]), (v, want[1])):
                m = max(0, min(n, capacity - at))
                w[i, at:at + m] = stands_for(x[i, :m])
                w[i, min(at + n, capacity):] = 0
            lengths[i] = min(capacity, at + n)
        assert cache.lengths.tolist() == lengths
        for x, w in zip(cache.read(), want):
            assert torch.equal(x, w), (t, counts, start)
        for x, w in zip(cache.read(13), want):
            assert torch.equal(x, w[:, :13])


def test_cache_leaves_other_rows_alone():
    cache = _lang().KVCache(2, 20, 2, 64, torch.bfloat16, True, DEV)
    cache._k.view(torch.uint8).fill_(0x55)
    cache._ks.fill_(3.0)
    before, scales = cache._k.view(torch.uint8).clone(), cache._ks.clone()
    x = torch.randn(2, 3, 2, 64, device=DEV, dtype=torch.bfloat16)
    cache.append(x, x, start=_i32(18, -1), counts=_i32(3, 2))       # 18, 19 and (dropped) 20; (dropped) -1 and 0
    after = cache._k.view(torch.uint8)
    keep = torch.ones(2, 20, dtype=torch.bool)
    keep[0, 18:] = False
    keep[1, 0] = False
    for h in range(2):
        assert torch.equal(after[:, h][keep], before[:, h][keep]) and torch.equal(cache._ks[:, h][keep], scales[:, h][keep])
        assert not torch.equal(after[0, h, 18:], before[0, h, 18:])
    assert cache.lengths.tolist() == [20, 1]


def test_cache_special_values():
    cache = _lang().KVCache(1, 4, 1, 64, torch.float32, True, DEV)
    k = torch.zeros(1, 4, 1, 64, device=DEV)
    k[0, 0, 0, :3] = torch.tensor([math.inf, -math.inf, 1.0])      # scale from the 1: 2^-8, infinities at 448 of it
    k[0, 1, 0, :2] = torch.tensor([math.nan, 2.0])
    k[0, 2, 0, 0] = 1e-42                                          # scales stay normal numbers
    k[0, 3, 0, 0] = 3.0e38
    cache.append(k, k)
    got = cache.read()[0][0, :, 0]
    assert got[0, :3].tolist() == [448 * 2.0 ** -8, -448 * 2.0 ** -8, 1.0]
    assert math.isnan(got[1, 0]) and got[1, 1] == 2.0
    assert got[2, 0] == 0 and abs(got[3, 0].item() / 3.0e38 - 1) <= 2.0 ** -4
    assert not got[:, 4:].any()


def test_reading_and_writing_back_changes_nothing():
    g = torch.Generator().manual_seed(2)
    a, b = (_lang().KVCache(2, 33, 3, 96, torch.bfloat16, True, DEV) for _ in range(2))
    a.append(_randn(g, 2, 33, 3, 96, dtype=torch.bfloat16), _randn(g, 2, 33, 3, 96, dtype=torch.bfloat16))
    b.append(*a.read())
    assert all(torch.equal(x, y) for x, y in zip(a.read(), b.read()))


def test_append_reads_what_it_moves():
    """`start` and `counts` may be the lengths that the call moves, k and v rows of the cache itself."""
    lang = _lang()
    g = torch.Generator().manual_seed(8)
    cache = lang.KVCache(2, 700, 4, 64, torch.bfloat16, False, DEV)
    x, y = (_randn(g, 2, 300, 4, 64, dtype=torch.bfloat16) for _ in range(2))
    cache.append(x, y, counts=_i32(300, 40))
    cache.append(x, y, start=cache.lengths, counts=cache.lengths)          # as many once more
    assert cache.lengths.tolist() == [600, 80]
    for i, n in enumerate((300, 40)):
        assert torch.equal(cache.k[i, :2 * n], torch.cat([x[i, :n]] * 2)) and torch.equal(cache.v[i, :2 * n], torch.cat([y[i, :n]] * 2))
    before = cache.k.clone(), cache.v.clone()
    cache.append(cache.k[:, :500], cache.v[:, :500], start=_i32(1, 1))     # every row one further
    assert cache.lengths.tolist() == [501, 501]
    for now, was in zip((cache.k, cache.v), before):                       # as bits: some rows were never written
        assert torch.equal(now[:, 1:501].view(torch.int16), was[:, :500].view(torch.int16))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_cache_values_near_the_largest(dtype):
    """What a type holds comes back finite and within 2^-4 of itself; an infinity as the largest value there is."""
    top = torch.finfo(dtype).max
    cache = _lang().KVCache(1, 3, 1, 96, dtype, True, DEV)
    k = torch.zeros(1, 3, 1, 96, dtype=dtype)
    k[0, 0, 0, :5] = torch.tensor([top, -top, top * 0.97, top * 0.9, top / 3], dtype=dtype)
    k[0, 1, 0, :3] = torch.tensor([math.inf, -math.inf, top], dtype=dtype)
    k[0, 2, 0, 17] = top * 0.94
    cache.append(k.to(DEV), k.to(DEV))
    for got in cache.read():
        got, want = got[0, :, 0].cpu().double(), k[0, :, 0].double()
        assert got.isfinite().all()
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs())[[0, 2]].all() and not got[1, 3:].any()
        assert got[1, 0] == got[1, 2] == -got[1, 1] and abs(got[1, 2] / top - 1) <= 2.0 ** -4


# ---- decoding ------------------------------------------------------------------------------------------------------------

def _filled(g, n, capacity, hkv, d, dtype, quantized, lengths, rubbish=True):
    cache = _lang().KVCache(n, capacity, hkv, d, dtype, quantized, DEV)
    if rubbish:            # rows behind the last token may hold anything
        cache._k.view(torch.uint8).fill_(0x7f if quantized else 0xff)
        cache._v.view(torch.uint8).fill_(0x7f if quantized else 0xff)
    longest = max(max(lengths), 1)
    cache.append(_randn(g, n, longest, hkv, d, dtype=dtype), _randn(g, n, longest, hkv, d, dtype=dtype), start=_i32(*[0] * n),
                 counts=_i32(*lengths))
    return cache


def _check_decode(g, b, t, h, hkv, d, capacity, lengths, dtype, quantized, groups=0, prefix=(), shared_capacity=0, buckets=32,
                  max_distance=128, counts=None):
    lang = _lang()
    cache = _filled(g, b, capacity, hkv, d, dtype, quantized, lengths)
    shared = _filled(g, groups, shared_capacity, hkv, d, dtype, quantized, prefix) if groups else None
    q = _randn(g, b, t, h, d, dtype=dtype)
    table = _randn(g, buckets, h, dtype=dtype) if buckets else None
    got = lang.decode_attention(q, cache, shared, table, max_distance=max_distance, counts=None if counts is None else _i32(*counts))
    k, v = cache.read()
    if shared is not None:
        sk, sv = shared.read()
    for i in range(b):
        n, m = lengths[i], t if counts is None else counts[i]
        keys, values = k[i:i + 1, :n], v[i:i + 1, :n]
        far = 0
        if shared is not None:
            s = i // (b // groups)
            far = prefix[s]
            keys, values = torch.cat([sk[s:s + 1, :far], keys], 1), torch.cat([sv[s:s + 1, :far], values], 1)
        first = max(0, m - n)                       # rows before the first token
        live = list(range(first, m))
        dead = [j for j in range(t) if j not in live]
        assert not got[i, dead].any(), (i, dead)
        if not live:
            continue
        offset = far + n - m + first
        nq, nk = len(live), keys.shape[1]
        index = ref.bucket_matrix(nq, nk, offset, buckets, max_distance, False) if buckets else None
        want = ref.attention(q[i:i + 1, live], keys, values, table, ref.seen(1, nq, nk, True, offset), d ** -0.5, index)
        ref.check("sequence %d" % i, got[i:i + 1, live], want["out"])


DECODE = [
    dict(b=1, t=1, h=1, hkv=1, d=64, capacity=1, lengths=(1,)),
    dict(b=1, t=1, h=12, hkv=12, d=64, capacity=40, lengths=(40,)),
    dict(b=3, t=1, h=4, hkv=2, d=96, capacity=500, lengths=(500, 0, 33)),
    dict(b=2, t=5, h=8, hkv=1, d=128, capacity=300, lengths=(299, 3), buckets=16, max_distance=64),      # fewer rows than queries
    dict(b=3, t=4, h=4, hkv=4, d=64, capacity=64, lengths=(64, 10, 7), counts=(4, 0, 2)),
    dict(b=4, t=1, h=4, hkv=4, d=64, capacity=70, lengths=(70, 1, 32, 64), groups=1, prefix=(1000,), shared_capacity=1100),
    dict(b=4, t=1, h=8, hkv=2, d=64, capacity=70, lengths=(70, 1, 0, 64), groups=2, prefix=(777, 0), shared_capacity=777),
    dict(b=6, t=3, h=8, hkv=2, d=128, capacity=90, lengths=(90, 3, 5, 33, 64, 2), groups=3, prefix=(300, 512, 1), shared_capacity=512,
         counts=(3, 3, 1, 0, 2, 3)),
    dict(b=2, t=1, h=4, hkv=4, d=96, capacity=30, lengths=(30, 4), groups=2, prefix=(400, 11), shared_capacity=400),
    dict(b=24, t=1, h=6, hkv=2, d=64, capacity=24, lengths=tuple(range(24)), groups=1, prefix=(290,), shared_capacity=300, buckets=0),
    dict(b=5, t=1, h=2, hkv=2, d=64, capacity=20, lengths=(20, 1, 2, 3, 4), groups=1, prefix=(100,), shared_capacity=100),
    dict(b=2, t=40, h=2, hkv=1, d=64, capacity=200, lengths=(200, 77)),
    dict(b=1, t=1, h=64, hkv=1, d=64, capacity=900, lengths=(900,), buckets=64, max_distance=1000),
    dict(b=1, t=2, h=2, hkv=2, d=128, capacity=5000, lengths=(4999,)),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("quantized", [False, True], ids=["plain", "e4m3"])
@pytest.mark.parametrize("n", range(len(DECODE)))
def test_decode_attention(n, dtype, quantized):
    _check_decode(torch.Generator().manual_seed(n), dtype=dtype, quantized=quantized, **DECODE[n])


def test_decode_with_two_sided_buckets():
    g = torch.Generator().manual_seed(0)
    cache = _filled(g, 1, 300, 2, 64, torch.float32, False, (300,))
    q, table = _randn(g, 1, 2, 4, 64), _randn(g, 32, 4)
    got = _lang().decode_attention(q, cache, None, table, bidirectional=True)
    k, v = cache.read()
    want = ref.attention(q, k, v, table, ref.seen(1, 2, 300, True, 298), 0.125, ref.bucket_matrix(2, 300, 298, 32, 128, True))
    ref.check("out", got, want["out"])


@pytest.mark.parametrize("quantized", [False, True], ids=["plain", "e4m3"])
def test_answering_token_by_token_equals_the_prompt_at_once(quantized):
    """Used together: a scene prefix and a prompt go into the caches, the prompt through relative_attention, then tokens one by
    one; every step's result is row n of the whole sequence at once -- computed from what the cache holds."""
    lang = _lang()
    g = torch.Generator().manual_seed(4)
    dtype, scene, b, h, hkv, d, prompt, steps = torch.bfloat16, 300, 4, 8, 2, 64, 20, 6
    shared = lang.KVCache(1, scene, hkv, d, dtype, quantized, DEV)
    shared.append(_randn(g, 1, scene, hkv, d, dtype=dtype), _randn(g, 1, scene, hkv, d, dtype=dtype))
    cache = lang.KVCache(b, prompt + steps, hkv, d, dtype, quantized, DEV)
    n = prompt + steps
    q, k, v = _randn(g, b, n, h, d, dtype=dtype), _randn(g, b, n, hkv, d, dtype=dtype), _randn(g, b, n, hkv, d, dtype=dtype)
    table = _randn(g, 32, h, dtype=dtype)
    counts = _i32(20, 11, 1, 7)
    cache.append(k[:, :prompt], v[:, :prompt], counts=counts)
    first = lang.decode_attention(q[:, :prompt], cache, shared, table, counts=counts)
    rows = [[first[i, :c] for i, c in enumerate(counts.tolist())]]
    used = [[q[i, :c] for i, c in enumerate(counts.tolist())]]
    for s in range(steps):
        at = prompt + s
        cache.append(k[:, at:at + 1], v[:, at:at + 1])
        out = lang.decode_attention(q[:, at:at + 1], cache, shared, table)
        rows.append([out[i] for i in range(b)])
        used.append([q[i, at:at + 1] for i in range(b)])
    assert cache.lengths.tolist() == [c + steps for c in counts.tolist()]
    sk, sv = shared.read()
    ck, cv = cache.read()
    for i in range(b):
        m = int(cache.lengths[i])
        keys, values = torch.cat([sk, ck[i:i + 1, :m]], 1), torch.cat([sv, cv[i:i + 1, :m]], 1)
        queries = torch.cat([u[i] for u in used])[None]
        got = torch.cat([r[i] for r in rows])[None]
        index = ref.bucket_matrix(m, scene + m, scene, 32, 128, False)
        want = ref.attention(queries, keys, values, table, ref.seen(1, m, scene + m, True, scene), d ** -0.5, index)
        ref.check("decoded", got, want["out"])
        whole = lang.relative_attention(queries, keys, values, table, bidirectional=False, causal=True, query_offset=scene)
        ref.check("at once", whole, want["out"])


def test_a_captured_decoding_step_replays():
    lang = _lang()
    g = torch.Generator().manual_seed(7)
    b, h, hkv, d, dtype = 3, 4, 2, 64, torch.bfloat16
    shared = _filled(g, 1, 700, hkv, d, dtype, True, (650,))
    caches = [lang.KVCache(b, 40, hkv, d, dtype, True, DEV) for _ in range(2)]
    q, k, v = (torch.empty(b, 1, n, d, device=DEV, dtype=dtype) for n in (h, hkv, hkv))
    table = _randn(g, 32, h, dtype=dtype)

    def step(cache):
        cache.append(k, v)
        return lang.decode_attention(q, cache, shared, table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(caches[0])
        caches[0].lengths.zero_()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(5):
        for x in (q, k, v):
            x.copy_(_randn(g, *x.shape, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        want = step(caches[1])
        assert torch.equal(got, want), i
        assert caches[0].lengths.tolist() == [i + 1] * b == caches[1].lengths.tolist()


@pytest.mark.parametrize("groups", [0, 1, 3])
def test_queries_that_are_none_may_hold_anything(groups):
    lang = _lang()
    g = torch.Generator().manual_seed(12)
    cache = _filled(g, 6, 400, 2, 64, torch.bfloat16, False, (400, 3, 17, 0, 1, 90))
    shared = _filled(g, groups, 500, 2, 64, torch.bfloat16, False, (500, 0, 33)[:groups]) if groups else None
    q, table, counts = _randn(g, 6, 3, 8, 64, dtype=torch.bfloat16), _randn(g, 32, 8, dtype=torch.bfloat16), _i32(3, 0, 2, 1, 3, 1)
    want = lang.decode_attention(q, cache, shared, table, counts=counts)
    for i, n in enumerate(counts.tolist()):
        q[i, n:] = math.nan
        assert not want[i, n:].any()
    assert want.isfinite().all()
    assert torch.equal(lang.decode_attention(q, cache, shared, table, counts=counts), want)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_many_heads_with_a_far_reach_over_shared_rows(dtype):
    """The biases of 32 query rows of as many heads would not fit into LDS."""
    _check_decode(torch.Generator().manual_seed(9), b=2, t=1, h=32, hkv=1, d=128, capacity=40, lengths=(33, 4), dtype=dtype,
                  quantized=False, groups=1, prefix=(560,), shared_capacity=600, buckets=64, max_distance=1024)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_biases_of_minus_infinity_weigh_nothing(dtype):
    """-inf (or a lowest value that becomes one): the key is as if masked, and a query with nothing else yields 0."""
    lowest = -math.inf if dtype == torch.float16 else torch.finfo(dtype).min
    for b, nq, nk, offset, buckets in ((2, 200, 200, 0, (0,)), (1, 70, 2000, 1930, (5, 31)), (1, 40, 40, 0, tuple(range(32)))):
        case = (b, nq, nk, 4, 2, 64, dict(causal=True, query_offset=offset, bidirectional=False))
        q, k, v, table, grad, ok, index, opts = _attention_case(case, dtype, nq)
        table[list(buckets)] = 0
        for bucket in buckets:
            ok = ok & (index != bucket)
        want = ref.attention(q, k, v, table, ok, 0.125, index, grad)
        for value in (-math.inf, lowest):
            table[list(buckets)] = value
            leaves = [x.detach().requires_grad_() for x in (q, k, v, table)]
            out = _lang().relative_attention(*leaves, **opts)
            ref.check("out", out, want["out"])
            for name, x in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, grad)):
                ref.check(name, x, want[name])


def test_saved_tensors_may_move():
    g = torch.Generator().manual_seed(10)
    q, k, v = (_randn(g, 2, 90, 4, 64, dtype=torch.bfloat16).requires_grad_() for _ in range(3))
    table, grad = _randn(g, 32, 4, dtype=torch.bfloat16).requires_grad_(), _randn(g, 2, 90, 4, 64, dtype=torch.bfloat16)
    call = lambda: _lang().relative_attention(q, k, v, table, causal=True, key_lengths=_i32(90, 31))          # noqa: E731
    want = torch.autograd.grad(call(), [q, k, v, table], grad)
    with torch.autograd.graph.save_on_cpu():
        out = call()
    filler = [torch.full((2, 90, 4, 64), math.nan, device=DEV) for _ in range(8)]      # where the saved ones were
    got = torch.autograd.grad(out, [q, k, v, table], grad)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and filler
    out = call()
    for _ in range(2):                                                                  # and are read as often as asked
        got = torch.autograd.grad(out, [q, k, v, table], grad, retain_graph=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_addresses_beyond_32_bits():
    """Token strides of 8 MB: the last rows of 600 lie 5 GB behind the first."""
    n, stride = 600, 1 << 22
    x = torch.zeros(n * stride + 1024, dtype=torch.bfloat16, device=DEV)
    q, k, v = (x.as_strided((1, n, 2, 64), (n * stride, stride, 64, 1), 128 * i) for i in range(3))
    g = torch.Generator().manual_seed(11)
    dense = [_randn(g, 1, n, 2, 64, dtype=torch.bfloat16) for _ in range(3)]
    for to, of in zip((q, k, v), dense):
        to.copy_(of)
    grad = _randn(g, 1, n, 2, 64, dtype=torch.bfloat16)
    leaves = [[t.detach().requires_grad_() for t in ts] for ts in ((q, k, v), dense)]
    outs = [_lang().relative_attention(*ts, causal=True) for ts in leaves]
    assert torch.equal(*outs)
    for a, b in zip(*(torch.autograd.grad(out, ts, grad) for out, ts in zip(outs, leaves))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("quantized", [False, True], ids=["plain", "e4m3"])
def test_long_caches(quantized):
    """Heads of 4 GB: one key of the last head's last rows has all the weight (60 against 0: the others' is e^-60 2^25)."""
    capacity = 1 << (25 if quantized else 24)
    cache = _lang().KVCache(1, capacity, 3, 128, torch.bfloat16, quantized, DEV)
    cache._k.view(torch.uint8).zero_()
    cache._v.view(torch.uint8).zero_()
    k, v = torch.zeros(1, 2, 3, 128, device=DEV, dtype=torch.bfloat16), torch.zeros(1, 2, 3, 128, device=DEV, dtype=torch.bfloat16)
    k[0, 0, :, 0] = 64
    v[0, 0] = torch.arange(3 * 128, device=DEV).reshape(3, 128) % 13 + 1
    cache.append(k, v, start=_i32(capacity - 2))
    q = torch.zeros(1, 1, 6, 128, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1
    got = _lang().decode_attention(q, cache, scale=60 / 64)
    assert torch.equal(got[0, 0], v[0, 0].repeat_interleave(2, 0))
    cache.append(k, v, start=_i32(0))
    assert torch.equal(_lang().decode_attention(q, cache, scale=60 / 64)[0, 0], v[0, 0].repeat_interleave(2, 0))
    assert torch.equal(cache.k[0, -2:].float(), k[0].float() / (cache.k_scale[0, -2:, :, None] if quantized else 1))


def test_gpu_refusals():
    lang = _lang()
    x = torch.zeros(2, 4, 4, 64, device=DEV, dtype=torch.bfloat16)
    cache = lang.KVCache(2, 8, 4, 64, torch.bfloat16, False, DEV)
    for bad in (lambda: lang.relative_attention(x, x.float(), x), lambda: lang.relative_attention(x[..., :32], x[..., :32], x[..., :32]),
                lambda: lang.relative_attention(x, x[:, :, :3], x[:, :, :3]), lambda: lang.relative_attention(x[0], x[0], x[0]),
                lambda: lang.relative_attention(x, x, x, torch.zeros(32, 3, device=DEV, dtype=torch.bfloat16)),
                lambda: lang.relative_attention(x, x, x, torch.zeros(32, 4, device=DEV)),
                lambda: lang.relative_attention(x, x, x, torch.zeros(2, 4, device=DEV, dtype=torch.bfloat16)),
                lambda: lang.relative_attention(x, x, x, prefix_lengths=_i32(1, 1)),
                lambda: lang.relative_attention(x, x, x, key_lengths=_i32(1, 1).long()),
                lambda: lang.relative_attention(x, x, x, key_lengths=_i32(1)),
                lambda: lang.relative_attention(x, x, x, key_ranges=_i32(1, 1)),
                lambda: lang.relative_attention(x, x, x, scale=math.inf),
                lambda: lang.relative_attention(x, x.cpu(), x), lambda: cache.append(x.float(), x.float()),
                lambda: cache.append(x[:1], x[:1]), lambda: cache.append(x, x, counts=_i32(1)), lambda: cache.read(9),
                lambda: lang.decode_attention(x.float(), cache), lambda: lang.decode_attention(x[:1], cache),
                lambda: lang.decode_attention(x, cache, lang.KVCache(2, 8, 4, 64, torch.bfloat16, True, DEV)),
                lambda: lang.decode_attention(x, cache, lang.KVCache(3, 8, 4, 64, torch.bfloat16, False, DEV)),
                lambda: lang.decode_attention(x, cache, None, torch.zeros(32, 4, device=DEV)),
                lambda: lang.decode_attention(x.clone().requires_grad_(), cache), lambda: cache.append(x, x.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(AttributeError):
        cache.lengths = _i32(1, 1)
