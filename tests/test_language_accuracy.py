"""The quadrature bounds of language_accuracy on the CPU: what they accept and what they reject."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import language_accuracy as acc  # noqa: E402
import language_ref as ref  # noqa: E402


def _rounded(p, dtype, parts):
    """P as the kernels put it into a product: relative to the row's maximum, in one part or two."""
    top = p.amax(-1, keepdim=True).clamp(min=1e-300)
    x = p / top
    one = x.to(dtype).double()
    return (one + ((x - one).to(dtype).double() if parts == 2 else 0.0)) * top


def _emulated(q, k, v, table, ok, scale, index, grad, parts, lost=()):
    """The kernels' roundings to 16 bits in 64-bit arithmetic; `lost`: names of gradients that come out as zero."""
    dtype = q.dtype
    group = q.shape[2] // k.shape[2]
    x, y, z, do = (t.double().transpose(1, 2) for t in (q, k, v, grad))
    y, z = (t.repeat_interleave(group, 1) for t in (y, z))
    s = scale * x @ y.transpose(2, 3) + table.double()[index].permute(2, 0, 1)
    p = torch.softmax(s.masked_fill(~ok[:, None], -torch.inf), -1).nan_to_num(0.0)
    o = _rounded(p, dtype, parts) @ z
    ds = p * (do @ z.transpose(2, 3) - (do * o).sum(-1, keepdim=True))
    held = ds.to(dtype).double()

    def fold(t):
        return t.view(t.shape[0], k.shape[2], group, *t.shape[2:]).sum(2).transpose(1, 2)

    got = {"out": o.transpose(1, 2), "dq": (scale * held @ y).transpose(1, 2), "dk": fold(scale * held.transpose(2, 3) @ x),
           "dv": fold(_rounded(p, dtype, 1).transpose(2, 3) @ do),
           "dtable": torch.stack([(ds * (index == i)).sum((0, 2, 3)) for i in range(table.shape[0])])}
    return {n: (torch.zeros_like(t) if n in lost else t).to(dtype) for n, t in got.items()}


CASES = [(2, 150, 150, 8, 4, 64, False), (1, 200, 260, 4, 4, 64, True), (1, 432, 432, 16, 16, 64, True)]


def _case(n, dtype, swing=3.0):
    b, nq, nk, h, hkv, d, causal = CASES[n]
    x = acc.inputs(torch.Generator().manual_seed(n), b, nq, nk, h, hkv, d, dtype=dtype, swing=swing)
    ok, index = ref.seen(b, nq, nk, causal, nk - nq), ref.bucket_matrix(nq, nk, nk - nq, 32, 128, not causal)
    return x[:4], ok, d ** -0.5, index, x[4]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n", range(len(CASES)))
def test_two_parts_are_accepted_one_is_not(n, dtype):
    case = _case(n, dtype)
    want = acc.variances(*case[0], *case[1:])
    two, one = (_emulated(*case[0], *case[1:], parts) for parts in (2, 1))
    for name in want:
        acc.check(name, two[name], want[name])
    acc.check_buckets(two["dtable"], want["dtable"], case[3], case[1])
    with pytest.raises(AssertionError, match="off by"):
        acc.check("out", one["out"], want["out"])
    loose = acc.variances(*case[0], *case[1:], parts=1)
    for name in want:
        acc.check(name, one[name], loose[name])


def test_delta_of_rounded_p_is_rejected():
    """The bucket that holds most of a long row's weight is where an error of delta adds up."""
    case = _case(2, torch.bfloat16, 0.0)
    want = acc.variances(*case[0], *case[1:])["dtable"]
    two, one = (_emulated(*case[0], *case[1:], parts)["dtable"] for parts in (2, 1))
    acc.check_buckets(two, want, case[3], case[1])
    with pytest.raises(AssertionError, match="bucket 31: off by"):
        acc.check_buckets(one, want, case[3], case[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("lost", ["dq", "dk", "dv", "dtable"])
def test_a_gradient_that_is_zero_is_rejected(lost, dtype):
    case = _case(0, dtype)
    want, got = acc.variances(*case[0], *case[1:]), _emulated(*case[0], *case[1:], 2, (lost,))
    with pytest.raises(AssertionError, match="off by"):
        acc.check(lost, got[lost], want[lost])
    if lost == "dtable":
        got = _emulated(*case[0], *case[1:], 2)["dtable"]
        pairs = [(int((case[3] == i).sum()), i) for i in range(32)]
        got[max(pairs)[1]] = 0                        # the bucket that holds most
        with pytest.raises(AssertionError, match="off by"):
            acc.check_buckets(got, want["dtable"], case[3], case[1])


def test_the_values_are_language_refs():
    case = _case(1, torch.float32)
    want = ref.attention(*case[0], *case[1:])
    for name, (value, var) in acc.variances(*case[0], *case[1:]).items():
        assert (value - want[name][0]).abs().max() <= 1e-10 * want[name][0].abs().max() and (var >= 0).all(), name
        assert (var.sqrt() <= want[name][1] + 1e-30).all(), name                       # no element's deviation beyond its worst
