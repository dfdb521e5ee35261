"""token_logprobs where x / T leaves f32's range: masks of the lowest value under a very low temperature."""
import math

import pytest
import torch

import loom_select as ls

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1e-6, 1e-8, 3e-9, 1e-9, 7e-10, 2e-10, 1e-10, 1e-12, 3e-20, 1e-37])
@pytest.mark.parametrize("vocab", [300, 20011])
def test_masked_ids_under_a_low_temperature(vocab, T, dtype):
    """Every masked id has log-probability -infinity, (-3.4e38 - 1) / T, whichever way 1 / T is rounded; a row of masks alone
    is a uniform one whose log-sum-exp is -infinity."""
    lowest = torch.finfo(dtype).min
    x = torch.full((3, vocab), lowest, dtype=dtype, device="cuda")
    x[0, 7], x[0, 9] = 1.0, 1.0
    x[1, 5] = -2.0
    ids = torch.tensor([11, 5, 0], dtype=torch.int32, device="cuda")
    r = ls.token_logprobs(x, ids, temperature=T, n_top=6, want_rank=True)
    assert r.top_ids[0].tolist() == [7, 9, 0, 1, 2, 3] and r.top_ids[1].tolist() == [5, 0, 1, 2, 3, 4]
    assert r.logp[0].item() == -math.inf and (r.top_logp[0, 2:] == -math.inf).all()
    assert r.logp[1].item() == 0 and (r.top_logp[1, 1:] == -math.inf).all()
    assert (r.top_logp[0, :2] + math.log(2)).abs().max().item() <= 4 * 2.0 ** -24
    assert r.lse[2].item() == -math.inf
    n = math.log(vocab)
    assert abs(r.entropy[2].item() - n) <= 600 * 2.0 ** -24 and abs(r.logp[2].item() + n) <= 600 * 2.0 ** -24
    assert r.rank.tolist() == [2 + 9, 0, 0]  # (ids 0 .. 10 but 7 and 9 are ahead of 11, and those two)
