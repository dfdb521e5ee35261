"""Refusals of the 8-bit LM-head calls, on the host: nothing is enqueued for a bad argument."""
import ctypes
import math

import pytest
import torch

import loom_select as ls

FAKE = ctypes.c_void_p(1 << 20)  # never dereferenced: every call below fails its host-side checks
OTHER = ctypes.c_void_p(1 << 21)
ODD = ctypes.c_void_p((1 << 20) + 1)
BY4 = ctypes.c_void_p((1 << 20) + 4)


def _norm(**kw):
    a = dict(x=FAKE, dtype=0, rows=2, dim=8, stride=8, res=OTHER, res_stride=8, w=FAKE, wdtype=0, eps=1e-6, q=FAKE,
             scale=FAKE, out_sum=ctypes.c_void_p(1 << 22), sum_stride=8)
    assert set(kw) <= set(a)
    a.update(kw)
    return ls.lib().loom_rms_norm_i8(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), ls.EDTYPE), (dict(wdtype=9), ls.EDTYPE), (dict(x=None), ls.EINVAL), (dict(w=None), ls.EINVAL),
    (dict(q=None), ls.EINVAL), (dict(scale=None), ls.EINVAL), (dict(rows=0), ls.EINVAL), (dict(dim=0), ls.EINVAL),
    (dict(stride=7), ls.EINVAL), (dict(res_stride=7), ls.EINVAL), (dict(sum_stride=7), ls.EINVAL),
    (dict(res=None), ls.EINVAL), (dict(out_sum=FAKE, sum_stride=9), ls.EINVAL),
    (dict(out_sum=OTHER, sum_stride=9), ls.EINVAL), (dict(eps=0.0), ls.EPARAM), (dict(eps=-1.0), ls.EPARAM),
    (dict(eps=math.nan), ls.EPARAM), (dict(eps=math.inf), ls.EPARAM),
    (dict(dim=32769, stride=32769, res_stride=32769, sum_stride=32769), ls.ESHAPE), (dict(rows=1 << 31), ls.ESHAPE),
    (dict(x=ODD), ls.EINVAL), (dict(res=ODD), ls.EINVAL), (dict(out_sum=ODD), ls.EINVAL), (dict(w=ODD), ls.EINVAL),
    (dict(scale=ODD), ls.EINVAL), (dict(x=ODD, dtype=1), ls.EINVAL),
])
def test_norm_refusals(kw, status):
    assert _norm(**kw) == status


def _quantize(**kw):
    a = dict(x=FAKE, dtype=0, rows=2, dim=8, stride=8, q=FAKE, scale=FAKE)
    a.update(kw)
    return ls.lib().loom_quantize_rows_i8(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), ls.EDTYPE), (dict(x=None), ls.EINVAL), (dict(q=None), ls.EINVAL), (dict(scale=None), ls.EINVAL),
    (dict(rows=-1), ls.EINVAL), (dict(dim=0), ls.EINVAL), (dict(stride=7), ls.EINVAL),
    (dict(dim=40000, stride=40000), ls.ESHAPE), (dict(x=ODD), ls.EINVAL), (dict(scale=ODD), ls.EINVAL),
])
def test_quantize_refusals(kw, status):
    assert _quantize(**kw) == status


def _head(**kw):
    a = dict(h=FAKE, hs=FAKE, w=FAKE, ws=FAKE, rows=2, hidden=64, vocab=10, out=FAKE, dtype=0, stride=10, work=FAKE,
             bytes=256)
    assert set(kw) <= set(a)
    a.update(kw)
    return ls.lib().loom_lm_head_logits_i8(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), ls.EDTYPE), (dict(h=None), ls.EINVAL), (dict(hs=None), ls.EINVAL), (dict(w=None), ls.EINVAL),
    (dict(ws=None), ls.EINVAL), (dict(out=None), ls.EINVAL), (dict(rows=0), ls.EINVAL), (dict(vocab=0), ls.EINVAL),
    (dict(hidden=0), ls.EINVAL), (dict(stride=9), ls.EINVAL), (dict(hidden=24), ls.ESHAPE),
    (dict(hidden=65552), ls.ESHAPE), (dict(rows=1 << 31), ls.ESHAPE), (dict(vocab=1 << 31, stride=1 << 31), ls.ESHAPE),
    (dict(rows=1 << 30, vocab=1 << 30, stride=1 << 30), ls.ESHAPE), (dict(h=BY4), ls.EINVAL), (dict(w=BY4), ls.EINVAL),
    (dict(hs=ODD), ls.EINVAL), (dict(ws=ODD), ls.EINVAL), (dict(out=ODD), ls.EINVAL), (dict(out=ODD, dtype=1), ls.EINVAL),
    (dict(work=None), ls.EWORKSPACE), (dict(bytes=255), ls.EWORKSPACE), (dict(work=BY4), ls.EWORKSPACE),
])
def test_head_refusals(kw, status):
    assert _head(**kw) == status


def test_head_workspace_is_the_status_word():
    assert ls.lib().loom_lm_head_logits_i8_workspace_size(1024, 151936) == 256


def test_host_tensors_are_refused():
    x, w = torch.zeros(2, 16), torch.ones(16)
    q, s = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2)
    for call in (lambda: ls.rms_norm_i8_into(x, w, q, s), lambda: ls.quantize_rows_i8_into(x, q, s),
                 lambda: ls.lm_head_logits_i8_into(q, s, q, s, torch.zeros(2, 2))):
        with pytest.raises(ls.SelectError) as e:
            call()
        assert e.value.status == ls.EINVAL
