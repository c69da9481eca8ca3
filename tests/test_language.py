"""Language-side operators without a GPU: bucket borders, key ranges of packed documents, struct layouts, every refusal of the C
entry points and of the Python ones that needs no device."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import language_ref as ref  # noqa: E402


@pytest.mark.parametrize("buckets,distance,both", [(32, 128, True), (32, 128, False), (16, 64, True), (48, 300, False), (7, 9, True),
                                                   (2, 5, False), (64, 1000, True), (4, 1024, True), (128, 1024, False)])
def test_bucket_borders(buckets, distance, both):
    from situation3d_amd import language
    border = language.relative_borders(buckets, distance, both)
    n = buckets // 2 if both else buckets
    e = n // 2
    assert len(border) == n and border[0] == 0 and list(border) == sorted(border)
    for a in range(0, distance + 50):
        mine = max(i for i in range(n) if border[i] <= a)
        assert mine == ref.bucket(-a, buckets, distance, both)
        # the logarithm's formula wherever it does not stand on a border
        if a >= e:
            x = (n - e) * math.log(a / e) / math.log(distance / e)
            if abs(x - round(x)) > 1e-9:
                assert mine == min(n - 1, e + math.floor(x))


@pytest.mark.parametrize("args", [(0, 128, False), (1, 128, True), (3, 128, True), (32, 8, True), (32, 16, False), (512, 1000, False),
                                  (32, 100000, False)])
def test_bucket_refusals(args):
    from situation3d_amd import language
    with pytest.raises(RuntimeError):
        language.relative_borders(*args)


def test_document_ranges():
    from situation3d_amd import language
    ids = torch.tensor([[4, 4, 4, 7, 1, 1], [0, 1, 2, 2, 2, 2]])
    got = language.document_ranges(ids)
    assert got.dtype == torch.int32 and got.tolist() == [
        [[0, 3], [0, 3], [0, 3], [3, 4], [4, 6], [4, 6]], [[0, 1], [1, 2], [2, 6], [2, 6], [2, 6], [2, 6]]]
    assert language.document_ranges(torch.zeros(2, 1, dtype=torch.int64)).tolist() == [[[0, 1]], [[0, 1]]]


def test_language_structs_match_the_c_header(tmp_path):
    from situation3d_amd import _lib
    structs = {"sig3d_rel_buckets": _lib.RelBuckets, "sig3d_rel_attention_args": _lib.RelAttentionArgs,
               "sig3d_cache_append_args": _lib.CacheAppendArgs, "sig3d_cache_read_args": _lib.CacheReadArgs, "sig3d_decode_attention_args": _lib.DecodeAttentionArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "sig3d_hip.h"', 'int main(void) {',
             'printf("max %d %d\\n", SIG3D_REL_MAX_BUCKETS, SIG3D_REL_MAX_REACH);']
    for name, cls in structs.items():
        lines.append('printf("%s size %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f) for f, _ in cls._fields_]
    (tmp_path / "p.c").write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "p.c"), "-o", str(tmp_path / "p")])
    for line in subprocess.check_output([str(tmp_path / "p")], text=True).splitlines():
        name, field, value = line.split()
        if name == "max":
            assert (int(field), int(value)) == (_lib.REL_MAX_BUCKETS, _lib.REL_MAX_REACH)
        elif field == "size":
            assert int(value) == ctypes.sizeof(structs[name]), name
        else:
            assert int(value) == getattr(structs[name], field).offset, (name, field)


def _buckets(n=16, border=None):
    from situation3d_amd import _lib
    b = _lib.RelBuckets(n=n, both=1)
    for i in range(min(n, _lib.REL_MAX_BUCKETS)):
        b.border[i] = i if border is None else border[i]
    return b


# An address that the host checks accept; every call below is refused before a launch (there is no GPU to launch on).
A = 1 << 20


def _rel_args(**kw):
    from situation3d_amd import _lib
    base = dict(q=A, k=A, v=A, table=A, out=A, out32=A, lse=A, grad=A, dq=A, dk=A, dv=A, dtable=A, work=A, q_b=64, q_n=64, q_h=64, k_b=64,
                k_n=64, k_h=64, v_b=64, v_n=64, v_h=64, grad_b=64, grad_n=64, grad_h=64, dtype=1, b=1, nq=4, nk=4, h=2, hkv=1, d=64,
                table_rows=32, scale=1.0, buckets=_buckets())
    return _lib.RelAttentionArgs(**{**base, **kw})


REL_BAD = [dict(dtype=3), dict(dtype=-1), dict(b=0), dict(nq=0), dict(nk=0), dict(h=0), dict(hkv=0), dict(h=3, hkv=2), dict(d=80), dict(d=0),
           dict(q_n=4), dict(k_h=-64), dict(v_b=1), dict(q=0), dict(k=A + 8), dict(v=A + 2), dict(out=A + 4), dict(lse=0), dict(out32=0),
           dict(table=0), dict(table_rows=31), dict(buckets="many"), dict(buckets="falling"), dict(buckets="late"), dict(buckets="far"),
           dict(nq=1 << 30), dict(nk=1 << 30), dict(query_offset=1 << 29), dict(b=1 << 20, h=1 << 10, nq=1 << 10)]


@pytest.mark.parametrize("n", range(len(REL_BAD)))
@pytest.mark.parametrize("name", ["sig3d_rel_attention_fwd", "sig3d_rel_attention_bwd"])
def test_rel_attention_refuses(n, name):
    from situation3d_amd import _lib
    made = {"many": lambda: _buckets(129), "falling": lambda: _buckets(3, (0, 5, 4)), "late": lambda: _buckets(2, (1, 2)),
            "far": lambda: _buckets(2, (0, 1025))}
    bad = {k: made[v]() if isinstance(v, str) else v for k, v in REL_BAD[n].items()}
    a = _rel_args(**bad)
    with pytest.raises(_lib.Sig3dError):
        _lib.call(name, ctypes.byref(a), None)
    assert _lib.load().sig3d_rel_attention_bwd_work_floats(ctypes.byref(a)) == -1
    assert _lib.load().sig3d_rel_attention_fwd_work_floats(ctypes.byref(a)) == -1


def test_rel_attention_fwd_wants_its_workspace():
    from situation3d_amd import _lib
    a = _rel_args(nq=32, nk=4096, work=0)
    assert _lib.load().sig3d_rel_attention_fwd_work_floats(ctypes.byref(a)) > 0
    with pytest.raises(_lib.Sig3dError):
        _lib.call("sig3d_rel_attention_fwd", ctypes.byref(a), None)
    assert _lib.load().sig3d_rel_attention_fwd_work_floats(ctypes.byref(_rel_args())) == 0


@pytest.mark.parametrize("bad", [dict(grad=0), dict(dq=0), dict(dk=0), dict(dv=0), dict(work=0), dict(dtable=0), dict(out32=0, lse=0),
                                 dict(grad_n=3), dict(dq=A + 8)], ids=str)
def test_rel_attention_bwd_refuses(bad):
    from situation3d_amd import _lib
    with pytest.raises(_lib.Sig3dError):
        _lib.call("sig3d_rel_attention_bwd", ctypes.byref(_rel_args(**bad)), None)


def test_null_arguments_are_refused():
    from situation3d_amd import _lib
    lib = _lib.load()
    for name in ("sig3d_rel_attention_fwd", "sig3d_rel_attention_bwd", "sig3d_cache_append", "sig3d_cache_read", "sig3d_decode_attention"):
        with pytest.raises(_lib.Sig3dError):
            _lib.call(name, None, None)
    assert lib.sig3d_rel_attention_bwd_work_floats(None) == -1 and lib.sig3d_decode_attention_work_floats(None) == -1


@pytest.mark.parametrize("bad", [dict(dtype=5), dict(b=0), dict(b=70000), dict(t=0), dict(capacity=0), dict(hkv=0), dict(d=72), dict(k=0),
                                 dict(v_cache=0), dict(lengths=0), dict(start=A), dict(counts=A), dict(k_scale=0), dict(k=A + 1), dict(k_n=7), dict(v_h=-8),
                                 dict(t=1 << 29, hkv=2)], ids=str)
def test_cache_append_refuses(bad):
    from situation3d_amd import _lib
    base = dict(k=A, v=A, k_cache=A, v_cache=A, k_scale=A, v_scale=A, lengths=A, k_b=64, k_n=64, k_h=64, v_b=64, v_n=64, v_h=64, dtype=1,
                b=1, t=1, capacity=4, hkv=1, d=64)
    with pytest.raises(_lib.Sig3dError):
        _lib.call("sig3d_cache_append", ctypes.byref(_lib.CacheAppendArgs(**{**base, **bad})), None)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(b=0), dict(n=0), dict(n=9), dict(capacity=0), dict(hkv=0), dict(d=65), dict(k_cache=0),
                                 dict(k_scale=0), dict(v_scale=0), dict(lengths=0), dict(k_out=0), dict(k_out=A + 4)], ids=str)
def test_cache_read_refuses(bad):
    from situation3d_amd import _lib
    base = dict(k_cache=A, v_cache=A, k_scale=A, v_scale=A, lengths=A, k_out=A, v_out=A, dtype=1, b=1, n=4, capacity=8, hkv=1, d=64)
    with pytest.raises(_lib.Sig3dError):
        _lib.call("sig3d_cache_read", ctypes.byref(_lib.CacheReadArgs(**{**base, **bad})), None)


DECODE_BAD = [dict(dtype=4), dict(b=0), dict(t=0), dict(h=3), dict(hkv=0), dict(d=32), dict(capacity=0), dict(groups=3), dict(groups=-1),
              dict(shared_capacity=0), dict(b=1 << 14, t=1 << 5, h=1 << 6, hkv=1 << 6), dict(table=0), dict(table_rows=3), dict(buckets="far")]


@pytest.mark.parametrize("n", range(len(DECODE_BAD)))
def test_decode_attention_refuses(n):
    from situation3d_amd import _lib
    bad = {k: _buckets(2, (0, 1025)) if isinstance(v, str) else v for k, v in DECODE_BAD[n].items()}
    a = _decode_args(**bad)
    with pytest.raises(_lib.Sig3dError):
        _lib.call("sig3d_decode_attention", ctypes.byref(a), None)
    assert _lib.load().sig3d_decode_attention_work_floats(ctypes.byref(a)) == -1


def _decode_args(**kw):
    from situation3d_amd import _lib
    base = dict(q=A, table=A, k_cache=A, v_cache=A, shared_k=A, shared_v=A, k_scale=A, v_scale=A, shared_k_scale=A, shared_v_scale=A,
                lengths=A, shared_lengths=A, out=A, work=A, q_b=64, q_n=64, q_h=64, dtype=1, b=4, t=1, h=4, hkv=2, d=64, capacity=4096,
                groups=2, shared_capacity=1024, table_rows=32, scale=1.0, buckets=_buckets())
    return _lib.DecodeAttentionArgs(**{**base, **kw})


@pytest.mark.parametrize("bad", [dict(q=0), dict(out=0), dict(k_cache=0), dict(lengths=0), dict(work=0), dict(shared_k=0),
                                 dict(shared_lengths=0), dict(k_scale=0), dict(shared_v_scale=0), dict(v_cache=A + 8), dict(q_n=2)], ids=str)
def test_decode_attention_refuses_arrays(bad):
    from situation3d_amd import _lib
    with pytest.raises(_lib.Sig3dError):
        _lib.call("sig3d_decode_attention", ctypes.byref(_decode_args(**bad)), None)


def test_cpu_tensors_are_refused():
    from situation3d_amd import language
    x = torch.zeros(1, 2, 2, 64)
    with pytest.raises(RuntimeError, match="CPU not supported"):
        language.relative_attention(x, x, x)
    with pytest.raises(RuntimeError, match="CPU not supported"):
        language.KVCache(1, 4, 2, 64, device="cpu")


def test_the_reference_in_64_bits_against_its_own_differences():
    """language_ref.attention's gradients, which the kernels are held to, are those of its forward pass."""
    g = torch.Generator().manual_seed(0)
    q, k, v, grad = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((2, 5, 4, 64), (2, 7, 2, 64), (2, 7, 2, 64), (2, 5, 4, 64)))
    table = torch.randn(32, 4, generator=g, dtype=torch.float64)
    ok, index = ref.seen(2, 5, 7, True, 1), ref.bucket_matrix(5, 7, 1, 32, 128, True)
    got = ref.attention(q, k, v, table, ok, 0.125, index, grad)
    for n, name in enumerate(("dq", "dk", "dv", "dtable")):
        way = torch.randn((q, k, v, table)[n].shape, generator=g, dtype=torch.float64)

        def loss(e):
            x = [y + e * way if i == n else y for i, y in enumerate((q, k, v, table))]
            return float((ref.attention(*x, ok, 0.125, index)["out"][0] * grad).sum())

        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        assert abs(slope - float((got[name][0] * way).sum())) <= 1e-6 * max(1.0, abs(slope)), name
