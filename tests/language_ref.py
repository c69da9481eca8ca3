"""The language-side operators in float64, with bounds on what a kernel may differ by -- from the definitions, by arithmetic.

u is half a step of the result's type (torch.finfo(t).eps / 2).  What rounds in a kernel, and nothing else:
  * a score is a sum of d products in f32 plus the bias, its exponential is one more f32 rounding or two, the sum of the row
    nk more: p is off by a factor 1 +- delta, delta = ((2 d + 16) 1.5 S + nk + 16) 2^-24 with S = max(scale sum|q k| + |bias|);
  * in bf16 / f16 p is rounded to the type before it meets V (w = u; in f32 w = 0), and dS before it meets K and Q;
  * the output is unrounded before dO.O, so delta_i = dO.O is off by (w + delta) sum_d |dO_d| A_d, A = p |V|;
  * every result is rounded once: u |result|;
  * below the smallest normal number of f16 a rounding is off by half the subnormal step, `least` = 2^-25, whatever the value:
    once for a result, once for each p (which is at most 1, relative to the row's maximum or to its sum), and for each dS, which
    the kernels hold times a power of two that brings max |dO| to 4 or more: least max |dO| / 4 (f32 and bf16: nothing there).
Sums over n f32 terms of the later products: n 2^-24 relative to the sum of absolute values."""
import math

import torch

STEP = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bucket(relative, buckets, max_distance, bidirectional):
    """Bucket of one relative position, by whole numbers."""
    n = buckets // 2 if bidirectional else buckets
    e = n // 2
    a = abs(relative) if bidirectional else max(0, -relative)
    at = a
    if a >= e:
        i = 0
        while e + i + 1 < n and a ** (n - e) * e ** (i + 1) >= max_distance ** (i + 1) * e ** (n - e):
            i += 1
        at = e + i
    return at + (n if bidirectional and relative > 0 else 0)


def bucket_matrix(nq, nk, offset, buckets, max_distance, bidirectional):
    line = torch.tensor([bucket(r, buckets, max_distance, bidirectional) for r in range(-(nq - 1) - offset, nk - offset)])
    return line[torch.arange(nk)[None, :] - torch.arange(nq)[:, None] + nq - 1]


def seen(b, nq, nk, causal=False, offset=0, key_lengths=None, prefix_lengths=None, key_ranges=None):
    i, j = torch.arange(nq)[:, None] + offset, torch.arange(nk)[None, :]
    ok = torch.ones(b, nq, nk, dtype=torch.bool)
    if key_lengths is not None:
        ok &= j < key_lengths.cpu()[:, None, None]
    if causal:
        c = (j <= i).expand(b, nq, nk)
        if prefix_lengths is not None:
            c = c | (j < prefix_lengths.cpu()[:, None, None])
        ok &= c
    if key_ranges is not None:
        r = key_ranges.cpu()
        ok &= (j >= r[:, :, :1]) & (j < r[:, :, 1:])
    return ok


def attention(q, k, v, table, ok, scale, index=None, grad=None):
    """q (b, nq, h, d), k / v (b, nk, hkv, d) of any type, ok (b, nq, nk), index (nq, nk) buckets ->
    {name: (value, bound)} for out, and with grad for dq, dk, dv, dtable."""
    dtype = q.dtype
    u = half_step(dtype)
    w = 0.0 if dtype == torch.float32 else u
    least = torch.finfo(dtype).smallest_normal * u                # half a subnormal step: smallest_normal eps is a whole one
    least_p = 0.0 if dtype == torch.float32 else least
    b, nq, h, d = q.shape
    nk, hkv = k.shape[1], k.shape[2]
    group = h // hkv
    live = ok.any(1)                                            # keys that somebody sees; the others may hold anything
    q, k, v = q.detach().double().cpu(), k.detach().double().cpu(), v.detach().double().cpu()
    k, v = (torch.where(live[:, :, None, None], x, 0.0) for x in (k, v))
    q = q.transpose(1, 2)
    k, v = (x.transpose(1, 2).repeat_interleave(group, 1) for x in (k, v))
    s = scale * q @ k.transpose(2, 3)
    size = abs(scale) * q.abs() @ k.abs().transpose(2, 3)
    if table is not None:
        bias = table.detach().double().cpu()[index].permute(2, 0, 1)
        s, size = s + bias, size + bias.abs()
    ok = ok[:, None].expand(b, h, nq, nk)
    s = s.masked_fill(~ok, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    big = float(torch.where(ok, size, 0.0).max()) if size.numel() else 0.0
    delta = ((2 * d + 16) * 1.5 * big + nk + 16) * STEP
    o = p @ v
    reach = p @ v.abs()
    under = least + least_p * (ok.double() @ v.abs())
    got = {"out": (o.transpose(1, 2), (u * o.abs() + (w + delta + nk * STEP) * reach * 1.01 + under).transpose(1, 2))}
    if grad is None:
        return got
    do = grad.detach().double().cpu().transpose(1, 2)
    dp, dl = do @ v.transpose(2, 3), (do * o).sum(-1, keepdim=True)
    ds = p * (dp - dl)
    dp_size = do.abs() @ v.abs().transpose(2, 3)
    dl_off = (do.abs() * ((w + delta + (nk + d) * STEP) * reach + under)).sum(-1, keepdim=True)
    # dS off by: p's factor, dP's and delta's own errors, and its rounding to the type
    ds_off = p * (delta * (dp.abs() + dl.abs()) + (d + 2) * STEP * dp_size + dl_off) * 1.01
    fold = lambda x: x.view(b, hkv, group, nk, d).sum(2).transpose(1, 2)   # noqa: E731
    n = nq * group * STEP
    dv, dv_size = p.transpose(2, 3) @ do, p.transpose(2, 3) @ do.abs()
    dq, dk = scale * ds @ k, scale * ds.transpose(2, 3) @ q
    off = ds_off + w * ds.abs() + ok * least_p * float(do.abs().max()) / 4
    dq_off = abs(scale) * ((off + nk * STEP * ds.abs()) @ k.abs())
    dk_off = abs(scale) * ((off + n * ds.abs()).transpose(2, 3) @ q.abs())
    got["dq"] = (dq.transpose(1, 2), (least + u * dq.abs() + 1.01 * dq_off).transpose(1, 2))
    got["dk"] = (fold(dk), least + u * fold(dk).abs() + 1.01 * fold(dk_off))
    got["dv"] = (fold(dv), least + u * fold(dv).abs() + 1.01 * fold((w + delta + n) * dv_size + least_p * (ok.double().transpose(2, 3) @ do.abs())))
    if table is not None:
        per, per_off = ds.sum(0), (ds_off + (nq + nk + b) * STEP * ds.abs()).sum(0)
        one = torch.nn.functional.one_hot(index, table.shape[0]).double().view(-1, table.shape[0])
        dt, dt_off = one.t() @ per.view(h, -1).t(), one.t() @ per_off.view(h, -1).t()
        got["dtable"] = (dt, least + u * dt.abs() + 1.01 * dt_off)
    return got


def check(name, got, want):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), "%s: not finite" % name
    far = (got - value).abs() - bound
    worst = float(far.max()) if far.numel() else 0.0
    assert worst <= 1e-30, "%s: %d of %d values outside their bound, worst by %g (bound there %g, value %g)" % (
        name, int((far > 1e-30).sum()), far.numel(), worst, float(bound.flatten()[far.argmax()]),
        float(value.flatten()[far.argmax()]))


def quantized(x):
    """(e4m3 values, scales (..., 1)) as torch rounds them: scale the smallest power of two with amax <= 448 scale."""
    amax = x.float().abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - 9 + (m > 0.875).int()), torch.ones_like(amax))
    return (x.float() / scale).to(torch.float8_e4m3fn), scale
