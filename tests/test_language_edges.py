"""Language-side operators without a GPU: strides of dimensions of one, far distances, numbers
that an argument struct does not hold."""
import pytest
import torch

CFG = (1.0, True, 128, False, 0)


def _template(q, k):
    from situation3d_amd import language
    return language._rel_template(q.shape, q.stride(), k.shape, k.stride(), k.shape, k.stride(), (q.dtype,) * 3, None, None, CFG)


def _one(shape, stride, dtype=torch.bfloat16):
    """`shape` over a storage of its elements: only the strides of dimensions of one are beyond it."""
    n = 1
    for x in shape:
        n *= x
    return torch.empty(n, dtype=dtype).as_strided(shape, stride)


@pytest.mark.parametrize("stride", [(256, 1 << 23, 64, 1), (7, 1 << 40, 64, 1), (256, 3, 64, 1)], ids=str)
@pytest.mark.parametrize("nk", [5, 2000])
def test_the_stride_of_a_single_token_does_not_matter(stride, nk):
    """One token sliced out of a token-major buffer: its stride is nobody's, and may be 16 MB and more."""
    from situation3d_amd import language
    k, dense = torch.empty(1, nk, 4, 64, dtype=torch.bfloat16), torch.empty(1, 1, 4, 64, dtype=torch.bfloat16)
    for q, keys in ((_one((1, 1, 4, 64), stride), k), (dense, _one((1, 1, 4, 64), stride))):
        other = torch.empty(q.shape if keys is not k else (1, 1, 4, 64), dtype=torch.bfloat16)
        a, ok, work = _template(q, keys)
        _, _, want = _template(other, keys if keys is k else other)
        assert ok and work == want and a.q_n == a.q_b == 0
    assert language._rows(_one((1, 1, 4, 64), stride)).shape == (1, 1, 4, 64)


def test_what_cannot_be_read_is_copied():
    from situation3d_amd import language
    for t in (torch.empty(2, 3, 4, 65)[..., 1:], torch.empty(1, 3, 4, 64).expand(2, 3, 4, 64), torch.empty(2, 3, 64, 4).transpose(2, 3),
              torch.empty(2, 1, 1, 64), torch.empty(3, 2, 4, 64).transpose(0, 1), torch.empty(2, 3, 4, 1).expand(2, 3, 4, 64)):
        r = language._rows(t)
        assert language._readable(r.shape, r.stride(), 4) and torch.equal(r.isnan(), t.isnan())


def test_tokens_of_16_mb_are_refused():
    """A dense tensor whose tokens are that long cannot be copied into a shape that the kernels read."""
    q = torch.empty(1, 2, 1 << 17, 64, dtype=torch.float16, device="meta")
    assert not _template(q, q)[1]


@pytest.mark.timeout(20)
@pytest.mark.parametrize("args", [(32, 10 ** 9, True), (32, 10 ** 30, False), (4, 10 ** 12, False), (256, 10 ** 15, True), (128, 1300, False)], ids=str)
def test_far_distances_are_refused_at_once(args):
    from situation3d_amd import language
    with pytest.raises(RuntimeError, match="at most 1024"):
        language.relative_borders(*args)


@pytest.mark.parametrize("args", [(4, 10 ** 6, True), (2, 10 ** 30, False), (3, 1025, False), (64, 1024, False)], ids=str)
def test_far_distances_that_no_border_stands_at(args):
    """The last bucket starts before max_distance: there may be but one bucket beyond the single distances, or the last border is near."""
    from situation3d_amd import language
    border = language.relative_borders(*args)
    n = len(border)
    e, far = n // 2, args[1]
    assert list(border[:e + 1]) == list(range(e + 1))[:n] and border[-1] <= 1024
    for i in range(1, n - e):
        a = border[e + i]
        assert a ** (n - e) * e ** i >= far ** i * e ** (n - e) > (a - 1) ** (n - e) * e ** i


@pytest.mark.parametrize("cfg", [(1e39, True, 128, False, 0), (-2e38, True, 128, False, 0), (float("nan"), True, 128, False, 0),
                                 (float("inf"), True, 128, False, 0), (1.0, True, 128, True, 1 << 32), (1.0, True, 128, True, 5 - (1 << 33))], ids=str)
def test_numbers_that_do_not_fit_are_refused(cfg):
    """2^32 + 5 would be taken as 5."""
    from situation3d_amd import language
    q = torch.empty(1, 4, 2, 64)
    with pytest.raises(RuntimeError):
        language._rel_template(q.shape, q.stride(), q.shape, q.stride(), q.shape, q.stride(), (q.dtype,) * 3, None, None, cfg)
    if cfg[4] == 0:
        with pytest.raises(RuntimeError):
            language._decode_template((1, 1, 2, 64), (128, 128, 64, 1), 0, 2, 8, False, 0, 0, 0, cfg[0], 128, False)


def test_broadcast_tokens_beyond_an_int_are_refused():
    q, k = torch.empty(1, 4, 2, 64), torch.empty(1, 1, 2, 64).expand(1, (1 << 32) + 5, 2, 64)
    with pytest.raises(RuntimeError):
        _template(q, k)
    with pytest.raises(RuntimeError):
        _template(q.expand((1 << 32) + 1, 4, 2, 64), k[:, :5].expand((1 << 32) + 1, 5, 2, 64))


def test_no_tokens_of_odd_strides():
    """Nothing is contiguous whatever its strides; the kernels' view of it is made all the same."""
    from situation3d_amd import language
    for t in (torch.empty(2, 0, 2, 65)[..., :64], torch.empty(0, 3, 2, 67)[..., 3:], torch.empty(2, 0, 64, 2).transpose(2, 3)):
        assert t.is_contiguous() or t.numel() == 0
        r = language._rows(t)
        assert r.shape == t.shape and _template(r, torch.empty(r.shape[0], 5, 2, 64))[1]
