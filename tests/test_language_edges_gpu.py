"""Language-side operators on the GPU: f16 gradients of values of very different size, forward-mode derivatives,
odd strides."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import language_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = ("dq", "dk", "dv", "dtable")


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def _lang():
    from situation3d_amd import language
    return language


# ---- f16: dS beyond what f16 holds -----------------------------------------------------------------------------------------

def _ds_most(q, k, v, table, grad, ok, scale, index):
    """max |dS| over all pairs."""
    q, k, v, do = (x.detach().double().cpu().transpose(1, 2) for x in (q, k, v, grad))
    group = q.shape[1] // k.shape[1]
    k, v = (x.repeat_interleave(group, 1) for x in (k, v))
    s = scale * q @ k.transpose(2, 3)
    if table is not None:
        s = s + table.detach().double().cpu()[index].permute(2, 0, 1)
    s = s.masked_fill(~ok[:, None], -torch.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    dp = do @ v.transpose(2, 3)
    return float((p * (dp - (p * dp).sum(-1, keepdim=True))).abs().max())


def _check_large(q, k, v, table, grad, ok, index, opts, scale):
    """language_ref's bounds, and what lowering the exponent costs: dS is then held times a power of two that keeps the largest of
    a query (dQ) or key (dK) at 2^11 or more, so that half a subnormal step of f16, 2^-25, stands for at most 2^-36 max |dS|."""
    want = ref.attention(q, k, v, table, ok, scale, index, grad)
    group = q.shape[2] // k.shape[2]
    most = _ds_most(q, k, v, table, grad, ok, scale, index) * 2.0 ** -36
    seen = ok[:, None].double()
    kk = k.double().abs().cpu().transpose(1, 2).repeat_interleave(group, 1)
    more_q = (scale * most * seen @ kk).transpose(1, 2)
    more_k = scale * most * seen.transpose(2, 3) @ q.double().abs().cpu().transpose(1, 2)
    more_k = more_k.view(k.shape[0], k.shape[2], group, k.shape[1], k.shape[3]).sum(2).transpose(1, 2)
    want["dq"] = want["dq"][0], want["dq"][1] + more_q
    want["dk"] = want["dk"][0], want["dk"][1] + more_k
    leaves = [x.detach().requires_grad_() for x in (q, k, v, table) if x is not None]
    out = _lang().relative_attention(*leaves, **opts)
    ref.check("out", out, want["out"])
    for name, x in zip(NAMES, torch.autograd.grad(out, leaves, grad)):
        ref.check(name, x, want[name])


@pytest.mark.parametrize("d", [64, 96, 128])
def test_f16_gradients_of_two_large_opposite_values(d):
    """dS = +-dO d V / 2 = +-128 for d = 128: more than f16 holds once dO = 0.01 has been raised to 4."""
    q, k = torch.zeros(1, 1, 1, d, dtype=torch.float16, device=DEV), torch.ones(1, 2, 1, d, dtype=torch.float16, device=DEV)
    k[0, 1] = -1
    q[..., 0] = 1
    k[..., 0] = 0.5                                   # the scores are equal, dQ is not 0
    v = torch.full((1, 2, 1, d), 200.0, dtype=torch.float16, device=DEV)
    v[0, 1] = -200
    grad = torch.full((1, 1, 1, d), 0.01, dtype=torch.float16, device=DEV)
    _check_large(q, k, v, None, grad, ref.seen(1, 1, 2), None, {}, d ** -0.5)


# b, nq, nk, h, hkv, d, options: one tile; several, causal; runs of keys; runs of queries
LARGE = [(2, 40, 60, 2, 1, 64, dict(key_lengths=(60, 33))), (1, 200, 200, 4, 2, 128, dict(causal=True, bidirectional=False)),
         (1, 70, 1100, 2, 2, 96, {}), (1, 1100, 150, 4, 1, 64, {}), (2, 300, 300, 2, 2, 96, dict(causal=True))]


@pytest.mark.parametrize("n", range(len(LARGE)))
@pytest.mark.parametrize("where", ["all", "late", "one"])
def test_f16_gradients_where_v_is_large_and_grads_are_small(n, where):
    """V of many thousand: everywhere, in late keys alone (the exponent moves between tiles), in one row; dO of many sizes.  Raised to
    4 <= max |dO| < 8, dS reaches 70 000 to 340 000 for dQ in all of these but one, up to 175 000 for dK."""
    b, nq, nk, h, hkv, d, opts = LARGE[n]
    opts = dict(opts)
    g = torch.Generator().manual_seed(n)
    f16 = torch.float16
    q, k, table = _randn(g, b, nq, h, d, dtype=f16) * 4, _randn(g, b, nk, hkv, d, dtype=f16), _randn(g, 32, h, dtype=f16)
    v = _randn(g, b, nk, hkv, d)
    if where == "all":
        v *= 12000
    elif where == "late":
        v[:, nk * 2 // 3:] *= 12000
    else:
        v[:, nk // 2] *= 14000
    # sizes 2^-16 .. 2^-8 by query: dQ and dK stay below 65504
    grad = _randn(g, b, nq, h, d) * torch.exp2(-8 - 8 * torch.rand(b, nq, 1, 1, generator=g)).to(DEV)
    if "key_lengths" in opts:
        opts["key_lengths"] = _i32(*opts["key_lengths"])
    ok = ref.seen(b, nq, nk, opts.get("causal", False), 0, opts.get("key_lengths"))
    index = ref.bucket_matrix(nq, nk, 0, 32, 128, opts.get("bidirectional", True))
    _check_large(q, k, v.to(f16), table, grad.to(f16), ok, index, opts, d ** -0.5)


def test_f16_infinite_grads_stay_where_they_are():
    """An infinite dO makes its own query's dQ and what it touches infinite or NaN, and nothing else (dV^T = dO^T P: its own element of
    every key's dV, 0 times infinity for the keys that it does not see)."""
    g = torch.Generator().manual_seed(3)
    q, k, v = (_randn(g, 1, 100, 2, 64, dtype=torch.float16).requires_grad_() for _ in range(3))
    grad = _randn(g, 1, 100, 2, 64, dtype=torch.float16)
    grad[0, 50, 1, 7] = torch.inf
    dq, dk, dv = torch.autograd.grad(_lang().relative_attention(q, k, v, causal=True), (q, k, v), grad)
    assert dq[0, :, 0].isfinite().all() and dk[0, :, 0].isfinite().all() and dv[0, :, 0].isfinite().all()
    assert not dq[0, 50, 1].isfinite().any()
    others, rest = torch.arange(100, device=DEV) != 50, torch.arange(64, device=DEV) != 7
    assert dq[0, others, 1].isfinite().all() and dk[0, 51:, 1].isfinite().all() and dv[0, :, 1, rest].isfinite().all()


# ---- f16: grads of queries that see nothing -----------------------------------------------------------------------------------

@pytest.mark.parametrize("how", ["masked", "biased"])
def test_f16_grads_of_queries_that_see_nothing_decide_nothing(how):
    """Their dO passes no gradient, so neither does its size decide how dS of the others is held."""
    g = torch.Generator().manual_seed(4)
    f16 = torch.float16
    q, k, v = (_randn(g, 1, 90, 2, 64, dtype=f16) for _ in range(3))
    table = _randn(g, 32, 2, dtype=f16)
    grad = _randn(g, 1, 90, 2, 64, dtype=f16) * 2.0 ** -10
    index = ref.bucket_matrix(90, 90, 0, 32, 128, True)
    if how == "masked":
        r = torch.tensor([0, 90]).repeat(1, 90, 1).int()
        r[0, 30:60] = 0
        opts, ok = dict(key_ranges=r.to(DEV)), ref.seen(1, 90, 90, key_ranges=r)
    else:                                             # a query whose only keys have a bias of -inf
        r = torch.tensor([0, 90]).repeat(1, 90, 1).int()
        r[0, 30:60, 0], r[0, 30:60, 1] = torch.arange(30, 60).int(), torch.arange(31, 61).int()
        table[0] = -torch.inf                         # its own place
        opts, ok = dict(key_ranges=r.to(DEV)), ref.seen(1, 90, 90, key_ranges=r) & (index != 0)
    live = ok[0].any(1)
    assert not live[30:60].any() and live[:30].all() and live[60:].all()
    held = torch.where(live.to(DEV)[None, :, None, None], grad, 0.0)
    want = ref.attention(q, k, v, torch.where(table.isinf(), 0.0, table), ok, 0.125, index, held)
    grad[0, 30:60] = 30000
    leaves = [x.detach().requires_grad_() for x in (q, k, v, table)]
    out = _lang().relative_attention(*leaves, **opts)
    ref.check("out", out, want["out"])
    for name, x in zip(NAMES, torch.autograd.grad(out, leaves, grad)):
        ref.check(name, x, want[name])


# ---- forward-mode derivatives ---------------------------------------------------------------------------------------------------

def test_tangents_are_refused():
    """There are no forward-mode derivatives; a dual tensor's tangent is never dropped."""
    from torch.autograd import forward_ad as fwd
    lang = _lang()
    q, k, v = (torch.randn(2, 5, 2, 64, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    table = torch.randn(32, 2, device=DEV, dtype=torch.bfloat16)
    ranges = _i32(*[0, 5] * 10).view(2, 5, 2)
    cache = lang.KVCache(2, 8, 2, 64, torch.bfloat16, False, DEV)
    cache.append(k, v)
    calls = [(lambda q, k, v, t: lang.relative_attention(q, k, v, t), 4), (lambda q, k, v, t: cache.append(k, v, start=_i32(0, 0)), (1, 2)),
             (lambda q, k, v, t: lang.decode_attention(q, cache, None, t), (0, 3)),
             (lambda q, k, v, t: lang.relative_attention(q[:, :, :, :], k, v, t, key_ranges=ranges), 4)]
    with fwd.dual_level():
        for call, which in calls:
            args = [q, k, v, table]
            call(*args)                                # nothing dual: as ever
            for i in range(4) if which == 4 else which:
                dual = [fwd.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(args)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
        leaf = q.clone().requires_grad_()
        out = lang.relative_attention(leaf, k, v, table)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, leaf, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: lang.relative_attention(x, k, v, table), (q,), (torch.ones_like(q),))


# ---- strides -----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("nk", [5, 2000])
def test_the_stride_of_a_single_token_does_not_matter(nk):
    """One token out of a token-major buffer of 16 MB a token; with many keys the call needs a workspace."""
    g = torch.Generator().manual_seed(6)
    big = torch.zeros(2 * (1 << 23), dtype=torch.bfloat16, device=DEV)
    q = big.as_strided((1, 1, 4, 64), (256, 1 << 23, 64, 1))
    dense = _randn(g, 1, 1, 4, 64, dtype=torch.bfloat16)
    q.copy_(dense)
    k, v = _randn(g, 1, nk, 2, 64, dtype=torch.bfloat16), _randn(g, 1, nk, 2, 64, dtype=torch.bfloat16)
    grads = []
    for x in (q, dense):
        leaves = [x.detach().requires_grad_(), k.detach().requires_grad_(), v.detach().requires_grad_()]
        out = _lang().relative_attention(*leaves)
        grads.append([out.detach(), *torch.autograd.grad(out, leaves, dense)])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_tokens_of_16_mb_are_refused():
    q = torch.zeros(1, 2, 1 << 17, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="16 MB"):
        _lang().relative_attention(q, q, q)
    assert not _lang().relative_attention(q[:, :1], q[:, :1], q[:, :1]).any()      # a single one has no stride


def test_numbers_that_do_not_fit_are_refused():
    lang = _lang()
    x = torch.zeros(1, 4, 2, 64, device=DEV)
    cache = lang.KVCache(1, 8, 2, 64, torch.float32, False, DEV)
    cache.append(x, x)
    many = x[:, :1].expand(1, (1 << 32) + 3, 2, 64)
    for bad in (lambda: lang.relative_attention(x, x, x, causal=True, query_offset=1 << 32), lambda: lang.relative_attention(x, x, x, scale=1e39),
                lambda: lang.relative_attention(x, many, many), lambda: lang.decode_attention(x, cache, scale=-1e39),
                lambda: lang.decode_attention(x, cache, scale=float("nan")), lambda: cache.append(many, many)):
        with pytest.raises(RuntimeError):
            bad()
    assert cache.lengths.tolist() == [4]


@pytest.mark.parametrize("shape", [(), (64,), (2, 3, 4, 0), (2, 3, 4, 80), (2, 3, 4, 64, 1)], ids=str)
def test_shapes_without_heads_are_refused(shape):
    x = torch.zeros(shape, device=DEV)
    with pytest.raises(RuntimeError):
        _lang().relative_attention(x, x, x)
    cache = _lang().KVCache(2, 8, 4, 64, torch.float32, False, DEV)
    with pytest.raises(RuntimeError):
        cache.append(x, x)
    with pytest.raises(RuntimeError):
        _lang().decode_attention(x, cache)


def test_no_tokens_of_odd_strides():
    x, none = torch.randn(2, 3, 2, 64, device=DEV), torch.empty(2, 0, 2, 65, device=DEV)[..., :64]
    assert _lang().relative_attention(none, x, x).shape == (2, 0, 2, 64)
    x.requires_grad_()
    out = _lang().relative_attention(x, none, none)
    assert not out.any() and not torch.autograd.grad(out.sum(), x)[0].any()
