"""Refusals of the row operators over vocabulary logits that need no GPU: the wrappers take no CPU
tensors, and the entry points return their status for bad arguments before they touch the device."""

import ctypes

import pytest
import torch


def _lib():
    from orthrus_training_b200 import _lib

    return _lib


def test_wrappers_refuse_cpu_tensors():
    from orthrus_training_b200 import ops

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        ops.topk_rows(x, 2)
    with pytest.raises(ValueError):
        ops.sample_logits(x, torch.zeros(2))


def _topk(R=2, V=8, ld=8, k=2, temperature=1.0, dtype=1, p=64, ws=64, ws_bytes=1 << 50):
    return _lib().lib().orthrus_topk_rows(p, ld, R, V, k, ctypes.c_float(temperature), p, p, p, ws, ws_bytes, dtype,
                                          None)


@pytest.mark.parametrize("bad", [dict(R=-1), dict(V=0), dict(ld=-1), dict(k=0), dict(k=1025), dict(temperature=0.0),
                                 dict(temperature=float("nan")), dict(dtype=2), dict(p=None), dict(V=2 ** 20 + 1),
                                 dict(V=2 ** 31), dict(R=2 ** 40), dict(R=2 ** 28, V=2 ** 20), dict(p=66)])
def test_topk_rows_status(bad):
    assert _topk(**bad) == _lib().EINVAL


def test_row_workspace():
    lib, L = _lib().lib(), _lib()
    assert _topk(ws=None) == L.EWORKSPACE and _topk(ws_bytes=8) == L.EWORKSPACE
    for dtype in (L.F32, L.BF16):
        assert lib.orthrus_topk_rows_workspace_bytes(0, 100, dtype) == 0
        for R, V in ((1, 1), (3, 1000), (1024, 151936), (2, 2 ** 20)):
            # a maximum for 32 entries, and a record of 16 bytes for 2048 or 8192
            small = lib.orthrus_topk_rows_workspace_bytes(R, V, dtype)
            assert R * V / 8 <= small <= R * (V / 8 + V / 128 + 80) + 512
            assert lib.orthrus_sample_logits_workspace_bytes(R, V, 0, dtype) == small
            # and the lists of up to 2048 rows that keep much, an eighth of the row at 8 bytes
            more = lib.orthrus_sample_logits_workspace_bytes(R, V, 1, dtype) - small
            assert min(R, 2048) * V <= more <= min(R, 2048) * (V + 8192 + V / 64 + 8192) + 2048


def test_no_rows_are_no_work():
    assert _topk(R=0) == _lib().OK
    f = ctypes.c_float
    assert _lib().lib().orthrus_sample_logits(None, 8, 0, 8, None, None, f(1), None, 0, None, f(1), None, f(0), None,
                                              None, 0, 1, None) == _lib().OK


@pytest.mark.parametrize("bad,status", [
    (dict(R=-1), "EINVAL"), (dict(V=0), "EINVAL"), (dict(ld=-1), "EINVAL"), (dict(dtype=7), "EINVAL"),
    (dict(p=None), "EINVAL"), (dict(V=2 ** 20 + 1), "EINVAL"), (dict(R=2 ** 40), "EINVAL"),
    (dict(ws=None), "EWORKSPACE"), (dict(ws_bytes=8), "EWORKSPACE")])
def test_sample_logits_status(bad, status):
    a = dict(dict(R=2, V=8, ld=8, dtype=1, p=64, ws=64, ws_bytes=1 << 50), **bad)
    f = ctypes.c_float
    assert _lib().lib().orthrus_sample_logits(a["p"], a["ld"], a["R"], a["V"], a["p"], None, f(1), None, 0, None, f(1),
                                              None, f(0), a["p"], a["ws"], a["ws_bytes"], a["dtype"],
                                              None) == getattr(_lib(), status)


def test_distillation_refuses_cpu_tensors():
    from orthrus_training_b200 import ops

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        ops.lmhead_topk_kl(x, x, x.long(), None, x)


GOOD = dict(student=64, n=4, values=64, ids=64, m=4, k=2, index=64, lse=None, weight=64, V=10, d=8, T=1.0, total=64,
            kl=64, agree=64, grad=64, offsets=None, num=0, ws=64, ws_bytes=1 << 40, dtype=0)


@pytest.mark.parametrize("bad,status", [
    (dict(n=-1), "EINVAL"), (dict(V=0), "EINVAL"), (dict(d=0), "EINVAL"), (dict(d=12), "EINVAL"), (dict(k=0), "EINVAL"),
    (dict(k=1025), "EINVAL"), (dict(T=0.0), "EINVAL"), (dict(T=float("nan")), "EINVAL"), (dict(m=0), "EINVAL"),
    (dict(index=None, m=3), "EINVAL"), (dict(student=None), "EINVAL"), (dict(weight=None), "EINVAL"),
    (dict(values=None), "EINVAL"), (dict(student=72), "EINVAL"), (dict(offsets=64), "EINVAL"), (dict(dtype=3), "EINVAL"),
    (dict(n=2 ** 31), "EINVAL"), (dict(ws=None), "EWORKSPACE"), (dict(ws_bytes=16), "EWORKSPACE")])
def test_distillation_status(bad, status):
    a = dict(GOOD, **bad)
    got = _lib().lib().orthrus_lmhead_topk_kl_fwd(
        a["student"], a["n"], a["values"], a["ids"], a["m"], a["k"], a["index"], a["lse"], a["weight"], a["V"], a["d"],
        ctypes.c_float(a["T"]), None, a["offsets"], a["num"], a["total"], a["kl"], a["agree"], a["grad"], None, None,
        4096, a["ws"], a["ws_bytes"], a["dtype"], None)
    assert got == getattr(_lib(), status)


@pytest.mark.parametrize("t", [0.0, 1e-31, 1e31, float("inf"), float("nan"), -1.0])
def test_temperatures_out_of_range(t):
    lib, f = _lib().lib(), ctypes.c_float
    assert lib.orthrus_topk_rows(64, 8, 2, 8, 3, f(t), 64, 64, 64, 64, 1 << 50, 1, None) == _lib().EINVAL
    a = dict(GOOD, T=t)
    assert lib.orthrus_lmhead_topk_kl_fwd(
        a["student"], a["n"], a["values"], a["ids"], a["m"], a["k"], a["index"], a["lse"], a["weight"], a["V"], a["d"],
        f(t), None, a["offsets"], a["num"], a["total"], a["kl"], a["agree"], a["grad"], None, None, 4096, a["ws"],
        a["ws_bytes"], a["dtype"], None) == _lib().EINVAL
