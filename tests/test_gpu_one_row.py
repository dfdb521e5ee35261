"""One row of logits whose stride torch gives as anything (a transposed column, a slice): every call takes it as the row
that it is."""
import pytest
import torch

import loom_select as ls

pytestmark = pytest.mark.gpu


@pytest.fixture
def rows():
    x = torch.randn(5003, 1, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").t()
    assert x.shape == (1, 5003) and x.stride(0) < 5003
    return x, torch.randn(1, 5003, device="cuda").copy_(x)


def test_argmax(rows):
    odd, plain = rows
    assert ls.argmax_rows(odd) == ls.argmax_rows(plain) == [float(plain.argmax())]
    assert ls.argmax_row(odd) == ls.argmax_row(plain)
    windows = [(0, 100), (100, -1)]
    assert torch.equal(ls.argmax_windows(odd, windows), ls.argmax_windows(plain, windows))


def test_sampler(rows):
    u = torch.rand(1, device="cuda")
    history = torch.tensor([[5, 9]], dtype=torch.int32, device="cuda")
    got, want = (ls.sample_rows(x, u, 0.8, 1.1, top_k=20, top_p=0.9, history=history, want_logp=True, want_topk=True)
                 for x in rows)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_shards(rows):
    u, k = torch.rand(1, device="cuda"), 16
    results = []
    for x in rows:
        records = torch.empty(2, 1, ls.shard_record_bytes(k), dtype=torch.uint8, device="cuda")
        for i, (lo, hi) in enumerate(((0, 2500), (2500, 5003))):
            ls.shard_partial_into(x[:, lo:hi], records[i], lo, 5003, 0.8, top_k=k)
        ids = torch.empty(1, dtype=torch.int32, device="cuda")
        prob = torch.empty(1, device="cuda")
        ls.shard_merge_into(records, 2, 1, u, ids, prob, 0.8, top_k=k)
        results.append((ids, prob))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


def test_scores(rows):
    ids = torch.tensor([17], dtype=torch.int32, device="cuda")
    a, b = (ls.token_logprobs(x, ids, n_top=4, want_rank=True) for x in rows)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = torch.ones(1, device="cuda")
    d = [ls.token_logprobs_grad(x, ids, a.lse, g) for x in rows]
    assert torch.equal(d[0], d[1])
