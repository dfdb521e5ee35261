"""Arguments that the calls which make their own outputs refuse before making them, on the host."""
import pytest
import torch

import loom_select as ls


def test_negative_number_of_alternatives():
    with pytest.raises(ls.SelectError) as e:
        ls.token_logprobs(torch.zeros(2, 5), n_top=-1)
    assert e.value.status == ls.EPARAM


@pytest.mark.parametrize("hidden,weight", [((), (5, 16)), ((2, 16), ()), ((2, 16), (16,)), ((1, 2, 16), (5, 16))])
def test_operands_of_another_rank(hidden, weight):
    q, w = torch.zeros(hidden, dtype=torch.int8), torch.zeros(weight, dtype=torch.int8)
    with pytest.raises(ls.SelectError) as e:
        ls.lm_head_logits_i8(q, torch.zeros(2), w, torch.zeros(5))
    assert e.value.status == ls.EINVAL
