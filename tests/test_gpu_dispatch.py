"""Shapes for each way in which the scores, their gradient and the 8-bit rows share out a row: the ranges between the
shapes of the other tests, with the same masks, ties, empty rows and odd offsets."""
import math

import pytest
import torch

import loom_select as ls
from test_gpu_lmhead_i8 import _norm, _quantise, _rows, _same
from test_gpu_logprobs import TOL, U, _close, _logits, _reference
from test_gpu_logprobs_likely import _rows_with, _state, _want

pytestmark = pytest.mark.gpu


def _patterns(x, ids):
    vocab = x.shape[1]
    x[0::7] = x[0::7].round().clamp(-2, 2)
    x[1::7, 40:] = -math.inf
    x[2::49, :] = -math.inf
    x[3::7, ::3] = -math.inf
    x[4::7, 3:] = -math.inf
    x[5::49, :] = torch.finfo(x.dtype).min
    ids[::5], ids[1::5], ids[2::25] = 0, vocab - 1, -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,offset", [
    (200, 900, 0), (200, 900, 1),        # a warp to a row: two or four vectors a step
    (700, 1500, 3), (2100, 3001, 1), (2100, 8000, 0),
    (600, 51865, 0), (600, 51864, 0),    # four warps to a row, several steps to a slot
    (600, 151936, 0), (160, 8190, 5),
    (300, 51865, 1),                     # two blocks of eight warps
])
def test_scores(rows, vocab, offset, dtype):
    x, ids = _logits(rows, vocab, seed=rows + vocab, dtype=dtype, offset=offset, stride=vocab + offset)
    _patterns(x, ids)
    for n_top in (0, 7, 32):
        r = ls.token_logprobs(x, ids, n_top=n_top, want_rank=True)
        for a in range(0, rows, 150):
            part = slice(a, min(a + 150, rows))
            w = _reference(x[part], ids[part], 1.0, n_top)
            # (the lowest values' log-sum-exp is within f32's range at T = 1)
            _close(r.lse[part], w["lse"], lambda v: TOL + 2 * U * v.abs(), "lse")
            _close(r.logp[part], w["logp"], lambda v: TOL + 4 * U * v.abs(), "logp")
            _close(r.entropy[part], w["entropy"], lambda v: 14 * TOL, "entropy")
            assert torch.equal(r.rank[part], w["rank"])
            if n_top:
                assert torch.equal(r.top_ids[part], w["top_ids"])
                _close(r.top_logp[part], w["top_logp"], lambda v: TOL + 4 * U * v.abs(), "top_logp")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,offset", [
    (5000, 1025, 0), (5000, 4000, 0), (5000, 4001, 1),   # a warp to a row, several steps
    (700, 4000, 2), (500, 8100, 0),                      # a block of four warps
    (460, 12007, 0), (500, 30011, 1), (300, 51865, 0),   # clusters of 1, 2, 4 (f32)
    (60, 51865, 3), (9, 151936, 0),                      # and of 8
    (4, 151936, 1), (3, 262147, 0), (2, 30011, 0),       # blocks of sixteen warps
    (9, 1025, 1), (140, 8100, 0),                        # and one to a row
])
def test_gradients(rows, vocab, offset, dtype):
    """Rows with a likely id and without one, padded and weightless rows between them; what lies between the rows stays."""
    x, ids = _rows_with(rows, vocab, 1e-3, 1.0, seed=vocab, dtype=dtype, offset=offset, extra=offset)
    flat = torch.arange(rows, device="cuda") % 3 == 1
    x[flat, ids.long()[flat]] = 0.0
    ids[::7] = -1
    g = torch.linspace(-2, 2, rows + 1, device="cuda")[1:]
    g[3::11] = 0
    h = 0.05 * g.abs()
    lse, ent, _ = _state(x, 1.0, False)
    buf = torch.full((rows * (vocab + offset) + offset + 64,), 77.0, dtype=dtype, device="cuda")
    out = buf[offset:offset + rows * (vocab + offset)].view(rows, vocab + offset)[:, :vocab]
    has = ids >= 0
    for weights in ((g, None), (g, h)):
        ls.token_logprobs_grad_into(x, ids, lse, out, weights[0], weights[1], ent if weights[1] is not None else None)
        for a in range(0, rows, 100):
            part = slice(a, min(a + 100, rows))
            gp = torch.where(has[part], g[part], 0.0)
            want, tol = _want(x[part], ids[part].clamp(min=0), 1.0, gp, None if weights[1] is None else h[part], 0.0, dtype)
            assert ((out[part].double() - want).abs() - tol).max().item() <= 0
        none = (torch.where(has, g, 0.0) == 0) & (True if weights[1] is None else h == 0)
        assert (out[none] == 0).all()
    out.fill_(77.0)
    assert (buf == 77.0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("rows,dim", [(5000, 100), (5000, 125), (5000, 128), (4800, 250), (40000, 33), (2500, 400)])
def test_rows_of_several_runs_to_a_thread(rows, dim, offset, dtype):
    x, res = _rows(rows, dim, dtype, 1, offset), _rows(rows, dim, dtype, 2, offset, dim + offset)
    w = _rows(1, dim, torch.float32, 3, offset)[0]
    wq, ws = _quantise(x.cpu().float())
    q, scale = ls.quantize_rows_i8(x)
    assert _same(q, wq) and _same(scale, ws)
    wq, ws, h = _norm(x, w, res, 1e-6)
    q, scale, total = ls.rms_norm_i8(x, w, res)
    assert torch.equal(total.cpu(), h)
    # (one row in 10^8 may have another rounding of its 1 / sqrt: none here)
    assert _same(q, wq) and _same(scale, ws)
