"""Language-side operators on the GPU: the kernels that only larger launches take, and errors as a whole (language_accuracy).

Which kernel a call takes follows from its sizes; the rules are repeated here as arithmetic, so that a case says which one it is for."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import language_accuracy as acc  # noqa: E402
import language_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
IDS = {F32: "f32", BF16: "bf16", F16: "f16"}


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _lang():
    from situation3d_amd import language
    return language


def _up(a, b):
    return -(-a // b)


def _fwd_groups(b, h, nq, nk, dtype):
    """Workgroups of the forward kernel: 128 queries each, keys split where there are few."""
    items = b * h * _up(nq, 128)
    tiles, least = (_up(nk, 32), 4) if dtype == F32 else (_up(nk, 64), 8)
    return items * max(1, min(16, _up(512, items), tiles // least))


def _masks(kind, b, nq, nk, g):
    opts = dict(bidirectional=True)
    if kind == "lengths":
        opts["key_lengths"] = _i32(*[nk, 1, nk // 2, 0, nk - 1][:b])
    if kind in ("causal", "prefix"):
        opts.update(causal=True, bidirectional=False)
    if kind == "prefix":
        opts["prefix_lengths"] = _i32(*[nk // 3, 0, nk, 65, 1][:b])
    if kind == "documents":
        ids = (torch.rand(b, nq, generator=g) < 4 / nq).int().cumsum(1).to(DEV)
        opts["key_ranges"] = _lang().document_ranges(ids)
    ok = ref.seen(b, nq, nk, opts.get("causal", False), 0, opts.get("key_lengths"), opts.get("prefix_lengths"), opts.get("key_ranges"))
    return opts, ok, ref.bucket_matrix(nq, nk, 0, 32, 128, opts["bidirectional"])


# ---- forward without a backward pass, more than 256 workgroups: P in one part ---------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("kind", ["none", "lengths", "causal", "prefix", "documents"])
def test_large_launches_without_a_backward_pass(kind, d, dtype):
    b, h, hkv, n = 4, 24, 8, 300
    assert _fwd_groups(b, h, n, n, dtype) > 256
    g = torch.Generator().manual_seed(d)
    q, k, v, table, _ = (x.to(DEV) for x in acc.inputs(g, b, n, n, h, hkv, d, dtype=dtype, swing=0.0))
    opts, ok, index = _masks(kind, b, n, n, g)
    with torch.no_grad():
        out = _lang().relative_attention(q, k, v, table, **opts)
    ref.check("out", out, ref.attention(q, k, v, table, ok, d ** -0.5, index)["out"])
    acc.check("out", out, acc.variances(q, k, v, table, ok, d ** -0.5, index, parts=1)["out"])


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_a_large_launch_with_many_key_tiles(dtype):
    """Tiles of every kind -- beyond the reach behind and ahead, near, cut -- in the one-part kernel, keys ahead of the queries too."""
    b, h, nq, nk, d = 2, 24, 700, 1500, 64
    assert _fwd_groups(b, h, nq, nk, dtype) > 256
    g = torch.Generator().manual_seed(1)
    q, k, v, table, _ = (x.to(DEV) for x in acc.inputs(g, b, nq, nk, h, h, d, dtype=dtype, swing=0.0))
    lengths = _i32(1500, 901)
    ok, index = ref.seen(b, nq, nk, key_lengths=lengths), ref.bucket_matrix(nq, nk, 400, 32, 128, True)
    with torch.no_grad():
        out = _lang().relative_attention(q, k, v, table, query_offset=400, key_lengths=lengths)
    ref.check("out", out, ref.attention(q, k, v, table, ok, d ** -0.5, index)["out"])
    acc.check("out", out, acc.variances(q, k, v, table, ok, d ** -0.5, index, parts=1)["out"])


# ---- dK / dV: more than 256 query tiles for a workgroup ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 64), (BF16, 96), (F16, 96), (BF16, 128), (F32, 64), (F32, 96)], ids=str)
def test_gradients_of_more_queries_than_one_list_holds(dtype, d):
    tile = 32 if dtype == F32 or d == 96 else 64
    nq, nk = 16 * 256 * tile + 700, 17
    splits = min(16, _up(1024, 1), _up(nq, tile) // 8)
    assert _up(_up(nq, tile), splits) > 256
    g = torch.Generator().manual_seed(d)
    q, k, v, table, grad = (x.to(DEV) for x in acc.inputs(g, 1, nq, nk, 1, 1, d, dtype=dtype))
    # some runs of queries see nothing, some a part, so that lists skip tiles and hold cut ones
    r = torch.tensor([0, nk]).repeat(1, nq, 1).int()
    at = torch.arange(nq) // 1000
    r[0, at % 3 == 1] = 0
    r[0, at % 5 == 2, 1] = 9
    ok, index = ref.seen(1, nq, nk, key_ranges=r), ref.bucket_matrix(nq, nk, 0, 32, 128, True)
    case = (q, k, v, table, ok, d ** -0.5, index, grad)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, table)]
    out = _lang().relative_attention(*leaves, key_ranges=r.to(DEV))
    want, worst = acc.variances(*case), ref.attention(*case)
    got = dict(zip(("out", "dq", "dk", "dv", "dtable"), (out, *torch.autograd.grad(out, leaves, grad))))
    for name, x in got.items():
        ref.check(name, x, worst[name])
        acc.check(name, x, want[name])


# ---- training: errors as a whole ----------------------------------------------------------------------------------------------------

# b, nq, nk, h, hkv, d, swing, options
TRAIN = [(2, 150, 150, 8, 4, 64, 3.0, {}),
         (1, 432, 432, 16, 16, 64, 0.0, dict(causal=True, bidirectional=False)),
         (1, 432, 432, 16, 16, 64, 3.0, dict(causal=True, bidirectional=False)),
         (2, 300, 300, 8, 2, 96, 3.0, dict(causal=True)),
         (2, 150, 2100, 4, 2, 96, 3.0, dict(key_lengths=(2100, 300), causal=True, query_offset=1950, bidirectional=False)),   # keys split
         (2, 1100, 200, 8, 2, 128, 3.0, dict(key_lengths=(200, 130))),                                 # queries and heads split
         (1, 1030, 1100, 4, 2, 128, 3.0, dict(causal=True, query_offset=70))]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("n", range(len(TRAIN)))
def test_training_errors_as_a_whole(n, dtype):
    b, nq, nk, h, hkv, d, swing, opts = TRAIN[n]
    opts = dict(opts)
    if "key_lengths" in opts:
        opts["key_lengths"] = _i32(*opts["key_lengths"])
    q, k, v, table, grad = (x.to(DEV) for x in acc.inputs(torch.Generator().manual_seed(n), b, nq, nk, h, hkv, d, dtype=dtype, swing=swing))
    offset = opts.get("query_offset", 0)
    ok, index = ref.seen(b, nq, nk, opts.get("causal", False), offset, opts.get("key_lengths")), ref.bucket_matrix(
        nq, nk, offset, 32, 128, opts.get("bidirectional", True))
    case = (q, k, v, table, ok, d ** -0.5, index)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, table)]
    out = _lang().relative_attention(*leaves, **opts)
    want = acc.variances(*case, grad)
    got = dict(zip(("out", "dq", "dk", "dv", "dtable"), (out, *torch.autograd.grad(out, leaves, grad))))
    for name, x in got.items():
        acc.check(name, x, want[name])
    acc.check_buckets(got["dtable"], want["dtable"], index, ok)
    with torch.no_grad():
        out = _lang().relative_attention(q, k, v, table, **opts)
    acc.check("out (no grad)", out, acc.variances(*case, parts=2 if _fwd_groups(b, h, nq, nk, dtype) <= 256 else 1)["out"])


# ---- decoding -------------------------------------------------------------------------------------------------------------------------

def _filled(g, n, capacity, hkv, d, dtype, quantized, lengths):
    cache = _lang().KVCache(n, capacity, hkv, d, dtype, quantized, DEV)
    for x in (cache._k, cache._v):                       # rows behind the last token may hold anything
        x.view(torch.uint8).fill_(0x7f if quantized else 0xff)
    longest = max(max(lengths), 1)
    k, v = (torch.randn(n, longest, hkv, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    cache.append(k, v, start=_i32(*[0] * n), counts=_i32(*lengths))
    return cache


def _check_decode(g, b, t, h, hkv, d, capacity, lengths, dtype, quantized, prefix=(), shared_capacity=0, counts=None, parts=2):
    lang = _lang()
    cache = _filled(g, b, capacity, hkv, d, dtype, quantized, lengths)
    groups = len(prefix)
    shared = _filled(g, groups, shared_capacity, hkv, d, dtype, quantized, prefix) if groups else None
    q, table = torch.randn(b, t, h, d, generator=g).to(dtype).to(DEV), torch.randn(32, h, generator=g).to(dtype).to(DEV)
    got = lang.decode_attention(q, cache, shared, table, counts=None if counts is None else _i32(*counts))
    k, v = (x.cpu() for x in cache.read())
    if groups:
        sk, sv = (x.cpu() for x in shared.read())
    kept, values, spread = [], [], []
    for i in range(b):
        n, m = lengths[i], t if counts is None else counts[i]
        keys, vals, far = k[i:i + 1, :n], v[i:i + 1, :n], 0
        if groups:
            s = i // (b // groups)
            far = prefix[s]
            keys, vals = torch.cat([sk[s:s + 1, :far], keys], 1), torch.cat([sv[s:s + 1, :far], vals], 1)
        first = max(0, m - n)
        live = list(range(first, m))
        assert not got[i, [j for j in range(t) if j not in live]].any(), i
        if not live:
            continue
        offset, nq, nk = far + n - m + first, len(live), keys.shape[1]
        case = (q[i:i + 1, live].cpu(), keys, vals, table, ref.seen(1, nq, nk, True, offset), d ** -0.5,
                ref.bucket_matrix(nq, nk, offset, 32, 128, False))
        ref.check("sequence %d" % i, got[i:i + 1, live], ref.attention(*case)["out"])
        value, var = acc.variances(*case, parts=parts)["out"]
        kept.append(got[i, live].flatten())
        values.append(value.flatten())
        spread.append(var.flatten())
    acc.check("all sequences", torch.cat(kept), (torch.cat(values), torch.cat(spread)))


# Short sequences of a large batch: one wave a sequence and key head, from 1024 of them on up to 512 rows (64 rows in any batch)
RAGGED = (0, 1, 31, 32, 33, 64, 65, 96, 97, 128, 129, 200, 250, 249, 225, 2)
ONE_WAVE = {
    "own": dict(capacity=250),
    "own, longest": dict(capacity=512, lengths=RAGGED[:13] + (512, 511, 480)),
    "joined": dict(capacity=250, prefix=(256, 0, 33, 100), shared_capacity=256),
    "joined, one": dict(capacity=250, prefix=(97,), shared_capacity=100),
    "shared": dict(capacity=250, prefix=(1000, 31), shared_capacity=1000),
}


@pytest.mark.parametrize("dtype,d,quantized", [(BF16, 64, False), (BF16, 64, True), (F16, 64, False), (F16, 128, True), (BF16, 128, False),
                                               (F32, 64, False), (F32, 96, True), (BF16, 96, False)], ids=str)
@pytest.mark.parametrize("kind", ONE_WAVE)
def test_one_wave_a_sequence(kind, dtype, d, quantized):
    """64 sequences of 16 key heads, ragged from 0 rows on: several tiles a wave, odd and even numbers of them."""
    opts = dict(ONE_WAVE[kind])
    lengths = opts.pop("lengths", RAGGED) * 4
    b, hkv = 64, 16
    rows = opts["capacity"] + (opts["shared_capacity"] if opts.get("shared_capacity", 0) <= 256 and "prefix" in opts else 0)
    assert b * hkv >= 1024 and 64 < rows <= 512
    _check_decode(torch.Generator().manual_seed(3), b, 1, hkv, hkv, d, lengths=lengths, dtype=dtype, quantized=quantized,
                  parts=1 if kind == "shared" else 2, **opts)


@pytest.mark.parametrize("dtype,quantized", [(BF16, False), (F16, True), (F32, False)], ids=str)
@pytest.mark.parametrize("kind", ["own", "joined", "shared"])
def test_one_wave_a_sequence_several_tokens(kind, dtype, quantized):
    """... for the three newest tokens of some sequences and fewer of others, two heads on a key head."""
    counts = tuple(min(3, n) if i % 3 else i % 4 for i, n in enumerate(RAGGED * 4))
    _check_decode(torch.Generator().manual_seed(5), 64, 3, 32, 16, 64, lengths=RAGGED * 4, dtype=dtype, quantized=quantized, counts=counts,
                  parts=1 if kind == "shared" else 2, **ONE_WAVE[kind])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("quantized", [False, True], ids=["plain", "e4m3"])
def test_decoding_errors_as_a_whole(dtype, quantized):
    """Long rows of their own in several pieces (P in two parts), and shared ones under two blocks of queries (in one)."""
    g = torch.Generator().manual_seed(7)
    _check_decode(g, 3, 2, 16, 4, 128, 2500, (2500, 1, 1300), dtype, quantized)
    _check_decode(g, 24, 1, 16, 4, 64, 100, tuple(range(0, 96, 4)), dtype, quantized, prefix=(1500, 700), shared_capacity=1500, parts=1)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=IDS.get)
@pytest.mark.parametrize("quantized", [False, True], ids=["plain", "e4m3"])
def test_cross_attention_token_by_token(dtype, quantized):
    """One answer token over a cache of the encoder's keys: no table, every row held is seen."""
    lang = _lang()
    g = torch.Generator().manual_seed(8)
    lengths = (432, 1, 0, 100)
    cache = _filled(g, 4, 432, 8, 64, dtype, quantized, lengths)
    q = torch.randn(4, 1, 8, 64, generator=g).to(dtype).to(DEV)
    got = lang.decode_attention(q, cache, None, None, scale=1.0)
    k, v = cache.read()
    ok = ref.seen(4, 1, 432, key_lengths=_i32(*lengths))
    want = ref.attention(q, k, v, None, ok, 1.0)
    ref.check("token", got, want["out"])
    ref.check("prompt", lang.relative_attention(q, k, v, None, scale=1.0, key_lengths=cache.lengths), want["out"])


@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_repeated_calls_give_the_same_bits(dtype):
    """Splits of keys, queries and heads, pieces of shared and own rows: joined in their order, whichever workgroup ends first."""
    lang = _lang()
    g = torch.Generator().manual_seed(9)
    leaves = [x.to(DEV).requires_grad_() for x in acc.inputs(g, 1, 600, 1500, 4, 1, 64, dtype=dtype)]
    grad = leaves.pop().detach()
    cache, shared = _filled(g, 6, 2000, 2, 128, dtype, True, (2000, 1, 900, 33, 1999, 0)), _filled(g, 2, 3000, 2, 128, dtype, True, (3000, 700))
    q, table = torch.randn(6, 2, 16, 128, generator=g).to(dtype).to(DEV), torch.randn(32, 16, generator=g).to(dtype).to(DEV)
    runs = []
    for _ in range(4):
        out = lang.relative_attention(*leaves, causal=True, query_offset=900)
        runs.append([out.detach(), *torch.autograd.grad(out, leaves, grad), lang.decode_attention(q, cache, shared, table)])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
