"""Refusals of token_logprobs and its gradient, on the host: nothing is enqueued for a bad argument."""
import ctypes
import math

import pytest
import torch

import loom_select as ls

FAKE = ctypes.c_void_p(1 << 20)  # never dereferenced: every call below fails its host-side checks
ODD = ctypes.c_void_p((1 << 20) + 1)


def _fwd(**kw):
    a = dict(logits=FAKE, dtype=0, rows=2, n=10, stride=10, ids=FAKE, T=1.0, n_top=2, logp=FAKE, ent=FAKE, lse=FAKE,
             rank=FAKE, top_ids=FAKE, top_logp=FAKE)
    assert set(kw) <= set(a)
    a.update(kw)
    return ls.lib().loom_token_logprobs(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=7), ls.EDTYPE), (dict(logits=None), ls.EINVAL), (dict(rows=0), ls.EINVAL), (dict(rows=-1), ls.EINVAL),
    (dict(n=0), ls.EINVAL), (dict(stride=9), ls.EINVAL), (dict(ids=None), ls.EINVAL),
    (dict(ids=None, logp=None), ls.EINVAL), (dict(ids=None, rank=None), ls.EINVAL),
    (dict(logp=None, ent=None, lse=None, rank=None, top_ids=None, top_logp=None, n_top=0), ls.EINVAL),
    (dict(n_top=0), ls.EINVAL), (dict(top_ids=None, top_logp=None), ls.EINVAL),
    (dict(n_top=-1), ls.EPARAM), (dict(n_top=11), ls.EPARAM), (dict(n_top=33, n=100, stride=100), ls.EPARAM),
    (dict(T=0.0), ls.EPARAM), (dict(T=-1.0), ls.EPARAM), (dict(T=math.nan), ls.EPARAM), (dict(T=math.inf), ls.EPARAM),
    (dict(T=1e-40), ls.EPARAM), (dict(rows=1 << 27), ls.ESHAPE), (dict(n=1 << 31, stride=1 << 31), ls.ESHAPE),
    (dict(logits=ODD), ls.EINVAL), (dict(logits=ODD, dtype=1), ls.EINVAL), (dict(ids=ODD), ls.EINVAL),
    (dict(logp=ODD), ls.EINVAL), (dict(ent=ODD), ls.EINVAL), (dict(lse=ODD), ls.EINVAL), (dict(rank=ODD), ls.EINVAL),
    (dict(top_ids=ODD), ls.EINVAL), (dict(top_logp=ODD), ls.EINVAL),
])
def test_forward_refusals(kw, status):
    assert _fwd(**kw) == status


def _bwd(**kw):
    a = dict(logits=FAKE, dtype=0, rows=2, n=10, stride=10, ids=FAKE, T=1.0, lse=FAKE, ent=FAKE, g=FAKE, h=FAKE,
             out=ctypes.c_void_p(1 << 21), out_stride=10)
    assert set(kw) <= set(a)
    a.update(kw)
    return ls.lib().loom_token_logprobs_grad(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=-1), ls.EDTYPE), (dict(logits=None), ls.EINVAL), (dict(lse=None), ls.EINVAL), (dict(out=None), ls.EINVAL),
    (dict(rows=0), ls.EINVAL), (dict(n=0), ls.EINVAL), (dict(stride=9), ls.EINVAL), (dict(out_stride=9), ls.EINVAL),
    (dict(g=None, h=None), ls.EINVAL), (dict(ids=None), ls.EINVAL), (dict(ent=None), ls.EINVAL),
    (dict(out=FAKE, out_stride=12), ls.EINVAL), (dict(T=0.0), ls.EPARAM), (dict(T=math.inf), ls.EPARAM),
    (dict(rows=1 << 27), ls.ESHAPE), (dict(n=1 << 31, stride=1 << 31, out_stride=1 << 31), ls.ESHAPE),
    (dict(out=ODD), ls.EINVAL), (dict(lse=ODD), ls.EINVAL), (dict(ent=ODD), ls.EINVAL), (dict(g=ODD), ls.EINVAL),
    (dict(h=ODD), ls.EINVAL), (dict(ids=ODD), ls.EINVAL),
])
def test_gradient_refusals(kw, status):
    assert _bwd(**kw) == status


def test_host_tensors_are_refused():
    x = torch.zeros(2, 5)
    ids = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ls.SelectError) as e:
        ls.token_logprobs_into(x, ids, torch.zeros(2))
    assert e.value.status == ls.EINVAL
    with pytest.raises(ls.SelectError) as e:
        ls.token_logprobs_into(x.half(), ids, torch.zeros(2))
    assert e.value.status == ls.EDTYPE
    with pytest.raises(ls.SelectError):
        ls.token_logprobs(x.t(), ids)
