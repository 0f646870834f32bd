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


def _topk(R=2, V=8, ld=8, k=2, temperature=1.0, dtype=1, p=64):
    return _lib().lib().orthrus_topk_rows(p, ld, R, V, k, ctypes.c_float(temperature), p, p, p, dtype, None)


@pytest.mark.parametrize("bad", [dict(R=-1), dict(V=0), dict(ld=-1), dict(k=0), dict(k=1025), dict(temperature=0.0),
                                 dict(temperature=float("nan")), dict(dtype=2), dict(p=None), dict(V=400_000),
                                 dict(V=2 ** 31), dict(R=2 ** 40)])
def test_topk_rows_status(bad):
    assert _topk(**bad) == _lib().EINVAL


def test_no_rows_are_no_work():
    assert _topk(R=0) == _lib().OK
    f = ctypes.c_float
    assert _lib().lib().orthrus_sample_logits(None, 8, 0, 8, None, None, f(1), None, 0, None, f(1), None, f(0), None,
                                              1, None) == _lib().OK


@pytest.mark.parametrize("bad", [dict(R=-1), dict(V=0), dict(ld=-1), dict(dtype=7), dict(p=None), dict(V=400_000),
                                 dict(R=2 ** 40)])
def test_sample_logits_status(bad):
    a = dict(dict(R=2, V=8, ld=8, dtype=1, p=64), **bad)
    f = ctypes.c_float
    assert _lib().lib().orthrus_sample_logits(a["p"], a["ld"], a["R"], a["V"], a["p"], None, f(1), None, 0, None, f(1),
                                              None, f(0), a["p"], a["dtype"], None) == _lib().EINVAL
