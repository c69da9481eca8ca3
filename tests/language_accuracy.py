"""How far the language-side operators' results may be off as a whole: the root mean square of independent roundings, in quadrature.

language_ref bounds every element by the worst that can happen, which for long sums is many times what does happen.  Here each rounding
counts with its variance instead, and the norm of a tensor's error is held to the root of the sum:
  * a rounding to a type with half step u is off by at most u |x|, uniformly: variance at most u^2 x^2 / 3;
  * a sum of n f32 terms is n roundings of partial sums, each at most the sum of absolute values A: variance at most n A^2 2^-48 / 3;
  * a score therefore has variance d size^2 2^-48 / 3, size = scale sum |q k|; its bias, its conversion to log2 units and the
    exponential's argument and value round three times more, each by at most (|s| + |bias| + 2) 2^-24;
  * the sum of a row and its logarithm are one error for all of the row: (sqrt(nk / 3) + 2 |lse| + 2) 2^-24 of p;
  * P is rounded to 16 bits before it meets dO (dV), and dS before it meets K and Q: u^2 / 3 of their squares.  `parts` says how P meets
    V: 1 rounded once; 2 as rounded value and rest, which leaves u^2 of it -- so the unrounded output, and with it delta = dO.O, is as
    good as f32.  An error of delta is one error for all of a row of dS: it adds up over a row's keys in dQ and in the table's bucket;
  * f16 below its normal numbers: half a subnormal step, 2^-25, of P relative to a row's maximum, and of dS as the kernels hold it
    (a power of two that brings max |dO| to 4 at least: 2^-27 max |dO|);
  * the result's own rounding is not estimated: it is the distance of the exact value to its nearest in the type.
Sampling: the norm of n independent errors scatters by 1 / sqrt(2 n) of itself; four times that is allowed for.  Where the errors before
the result's rounding are small beside its step, a better bound needs no sampling of that rounding: |round(x + e) - x| is at most
|round(x) - x| + 2 |e| (if the two round apart, x is within |e| of the middle between them)."""
import math

import torch

STEP2 = 2.0 ** -48


def variances(q, k, v, table, ok, scale, index=None, grad=None, parts=2):
    """language_ref.attention's arguments -> {name: (value, variance of every element before the result's rounding)}."""
    dtype = q.dtype
    f32 = dtype == torch.float32
    u2 = (torch.finfo(dtype).eps / 2) ** 2 / 3
    w2 = 0.0 if f32 else u2                                  # of a 16-bit operand
    p2 = 0.0 if f32 else (u2 if parts == 1 else u2 ** 2)     # of P where it meets V
    least2 = (2.0 ** -25) ** 2 / 3 if dtype == torch.float16 else 0.0
    b, nq, h, d = q.shape
    nk, hkv = k.shape[1], k.shape[2]
    group = h // hkv
    live = ok.any(1)
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    k, v = (torch.where(live[:, :, None, None], x, 0.0) for x in (k, v))
    q = q.transpose(1, 2)
    k, v = (x.transpose(1, 2).repeat_interleave(group, 1) for x in (k, v))
    size = abs(scale) * q.abs() @ k.abs().transpose(2, 3)
    s = scale * q @ k.transpose(2, 3)
    near = s.abs() + 2
    if table is not None:
        bias = table.detach().double().cpu()[index].permute(2, 0, 1)
        s, near = s + bias, near + bias.abs()
    seen = ok[:, None].expand(b, h, nq, nk)
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    lse = torch.where(lse.isinf(), 0.0, lse)
    p = torch.exp(s - lse)
    ep = STEP2 * (d / 3 * size ** 2 + 3 * near ** 2)                                 # of one p
    er = STEP2 * ((nk / 3) ** 0.5 + 2 * lse.abs() + 2) ** 2                          # of a row's
    pp = p * p
    o, reach = p @ v, p @ v.abs()
    top = p.amax(-1, keepdim=True)                                                   # P is held relative to a row's maximum, about
    held = least2 * top ** 2 * seen
    var_o = (pp * (ep + p2) + held) @ v ** 2 + er * o ** 2 + nk / 3 * STEP2 * reach ** 2
    got = {"out": (o.transpose(1, 2), var_o.transpose(1, 2))}
    if grad is None:
        return got
    do = grad.detach().double().cpu().transpose(1, 2)
    dp, dl = do @ v.transpose(2, 3), (do * o).sum(-1, keepdim=True)
    ds = p * (dp - dl)
    size_dp = do.abs() @ v.abs().transpose(2, 3)
    kappa = ((pp * (ep + p2) + held) * dp ** 2).sum(-1, keepdim=True) + er * dl ** 2 + STEP2 / 3 * (
        nk * (do ** 2 * reach ** 2).sum(-1, keepdim=True) + d * (do * o).abs().sum(-1, keepdim=True) ** 2)
    var_s = pp * (ep * (dp - dl) ** 2 + d / 3 * STEP2 * size_dp ** 2)
    small = least2 * (float(do.abs().max()) / 4) ** 2 * seen
    n = nq * group

    def fold(x):
        return x.view(b, hkv, group, nk, d).sum(2).transpose(1, 2)

    pt, st = p.transpose(2, 3), ds.transpose(2, 3)
    dq, dk, dv = scale * ds @ k, scale * st @ q, pt @ do
    var_q = scale ** 2 * ((var_s + w2 * ds ** 2 + small) @ k ** 2 + kappa * (p @ k) ** 2 + nk / 3 * STEP2 * (ds.abs() @ k.abs()) ** 2) + er * dq ** 2
    var_k = scale ** 2 * ((var_s + (w2 + er) * ds ** 2 + kappa * pp + small).transpose(2, 3) @ q ** 2 + n / 3 * STEP2 * (st.abs() @ q.abs()) ** 2)
    var_v = (pp * (ep + er + w2) + held).transpose(2, 3) @ do ** 2 + n / 3 * STEP2 * (pt @ do.abs()) ** 2
    got["dq"] = dq.transpose(1, 2), var_q.transpose(1, 2)
    got["dk"], got["dv"] = (fold(dk), fold(var_k)), (fold(dv), fold(var_v))
    if table is not None:

        def of_bucket(x):
            """x (b, h, nq, nk) summed over the keys of each bucket: (b, h, nq, buckets)."""
            return torch.zeros(b, h, nq, table.shape[0], dtype=torch.float64).scatter_add_(3, index.expand(b, h, nq, nk), x)

        each = of_bucket(ds)
        value = each.sum((0, 2)).t()
        var = (of_bucket(var_s) + kappa * of_bucket(p) ** 2 + er * each ** 2 + (nq + nk) / 3 * STEP2 * of_bucket(ds.abs()) ** 2).sum((0, 2)).t()
        got["dtable"] = value, var
    return got


def bound(value, var, dtype):
    """Norm of the error: the result's own rounding and `var`."""
    own, e = float((value.to(dtype).double() - value).norm()), float(var.sum()) ** 0.5
    slack = 1 + 4 / (2 * value.numel()) ** 0.5
    return min(own + 2 * slack * e, slack * (own ** 2 + e ** 2) ** 0.5)


def off(got, value):
    return float((got.detach().double().cpu() - value).norm())


def check(name, got, want, share=0.1):
    """... and the bound says something: it is below `share` of the value."""
    value, var = want
    most, norm, far = bound(value, var, got.dtype), float(value.norm()), off(got, value)
    assert most <= share * norm, "%s: a bound of %g on a value of %g says nothing" % (name, most, norm)
    assert far <= most, "%s: off by %g, bound %g, value %g" % (name, far, most, norm)


def check_buckets(got, want, index, ok):
    """... of each bucket that holds a twentieth of the pairs or more, over its heads."""
    value, var = want
    pairs = ok.sum(0).double()
    looked = 0
    for bucket in range(value.shape[0]):
        if float((pairs * (index == bucket)).sum()) < 0.05 * float(pairs.sum()):
            continue
        looked += 1
        check("bucket %d" % bucket, got[bucket], (value[bucket], var[bucket]))
    assert looked


def inputs(g, b, nq, nk, h, hkv, d, buckets=32, dtype=torch.float32, swing=3.0):
    """Standard normal q, k, v, table, grad, plus (swing > 0) what makes a table's gradient large: every head's dO leans one way, and V
    swings along it with the key's place, so that a query's near and far keys pull apart."""
    rand = lambda *s: torch.randn(s, generator=g)                                      # noqa: E731
    q, k, v, table, grad = rand(b, nq, h, d), rand(b, nk, hkv, d), rand(b, nk, hkv, d), rand(buckets, h), rand(b, nq, h, d)
    way = rand(hkv, d) / d ** 0.5
    v = v + swing * torch.linspace(-1, 1, nk)[None, :, None, None] * way
    grad = grad + swing * way.repeat_interleave(h // hkv, 0)
    return [x.to(dtype) for x in (q, k, v, table, grad)]
