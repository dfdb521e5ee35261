"""token_logprobs_grad where one id of a row has nearly all of the probability: a well predicted token's entry,
g (1 - p_t) / T, is then the row's largest and a small difference, and so is an entropy bonus's at the likeliest id.

Tolerances, in units u = 2^-24. With lse rounded once from 64 bits, a probability far from 1 is off by u |lse| from that
rounding, u |l| from each of the two roundings of x - lse T and u |l| from the product and from the constant, l = log2 p
(|l| <= 200 where p is not 0), and 4u from ex2: relative, (|lse| + 4 |l| + 4) u. An entry takes five more roundings.
The likeliest id's entry is minus the sum of the others: a thread adds at most 192 of them one after another, and 46
more additions join the sums of its halves, warps and blocks: 240 u of the sum of their magnitudes. A bf16 entry is
rounded once more, by 2^-8 of itself.
With the forward call's lse, the log-sum-exp's own 600 u (see test_gpu_logprobs.py) comes on top.
"""
import math

import pytest
import torch

import loom_select as ls

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LSE = 600 * U


def _rows_with(rows, vocab, rest, T, seed, dtype=torch.float32, keep=1.0, offset=0, extra=0, top=None):
    """Rows whose given id (`top`: another one) has probability 1 - rest, about, after rounding to the type."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device="cuda", dtype=torch.float64) * 3
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    top = ids if top is None else (ids + top) % vocab
    if keep < 1:
        off = torch.rand(rows, vocab, generator=g, device="cuda") >= keep
        off[torch.arange(rows), (top + 1) % vocab] = False
        x[off] = -math.inf
    x[torch.arange(rows), top] = -math.inf
    others = T * torch.logsumexp(x / T, dim=1)
    x[torch.arange(rows), top] = others + T * math.log((1 - rest) / rest)
    buf = torch.full((rows * (vocab + extra) + offset + 64,), 1e9, dtype=dtype, device="cuda")
    view = buf[offset:offset + rows * (vocab + extra)].view(rows, vocab + extra)[:, :vocab]
    view.copy_(x.to(dtype))
    return view, ids.int()


def _parts(x, T):
    """log p, p, 1 - p and the entropy of each row in 64 bits, the likeliest id's 1 - p without cancellation."""
    y = x.double() / T
    lp = torch.log_softmax(y, dim=1)
    p = lp.exp()
    top = y.argmax(dim=1, keepdim=True)
    rest = p.clone().scatter_(1, top, 0.0).sum(dim=1, keepdim=True)
    lp = lp.scatter(1, top, torch.log1p(-rest))
    p = p.scatter(1, top, 1 - rest)
    not_p = (1 - p).scatter(1, top, rest)
    ent = -torch.where(p > 0, p * lp, 0.0).sum(dim=1, keepdim=True)
    return lp, p, not_p, ent, top


def _want(x, ids, T, g, h, lse_err, dtype):
    """The gradient in 64 bits and how far each entry may be off."""
    lp, p, not_p, ent, top = _parts(x, T)
    at = ids.long()[:, None]
    g = torch.zeros_like(ent) if g is None else g.double()[:, None]
    h = torch.zeros_like(ent) if h is None else h.double()[:, None]
    d = -g * p
    d.scatter_(1, at, g * not_p.gather(1, at))
    d -= h * torch.where(p > 0, p * (lp + ent), 0.0)
    lse = torch.logsumexp(x.double() / T, dim=1, keepdim=True).abs()
    l = torch.where(p > 0, lp, 0.0).abs() / math.log(2)
    eps = lse_err + U * (lse + 4 * l + 9)
    # the entropy is rounded once from 64 bits, or off by as much again as the log-sum-exp's bound (times |A / S| + 1)
    ent_err = U * ent + (ent + 2) * lse_err
    tol = p * (g.abs() * eps + h.abs() * ((l + ent + 1) * eps + ent_err))
    tol = tol.scatter_add(1, at, U * 5 * g.abs() * not_p.gather(1, at))  # (of an unlikely given token)
    others = torch.ones_like(p, dtype=torch.bool).scatter_(1, top, False)
    likely = p.gather(1, top) > 0.78  # (below 0.758 by the formula, with the tolerance above)
    total = torch.where(others, tol + 240 * U * d.abs(), 0.0).sum(dim=1, keepdim=True)
    tol = tol.scatter(1, top, torch.where(likely, total, tol.gather(1, top)))
    return d / T, tol / T + (d / T).abs() * (torch.finfo(dtype).eps / 2 + 5 * U) + 1e-37


def _state(x, T, from_forward):
    if from_forward:
        f = ls.token_logprobs(x, temperature=T)
        return f.lse, f.entropy, LSE
    _, _, _, ent, _ = _parts(x, T)
    return torch.logsumexp(x.double() / T, dim=1).float(), ent[:, 0].float(), 0.0


def _check(x, ids, T, g, h, dtype=torch.float32, from_forward=False):
    lse, ent, lse_err = _state(x, T, from_forward)
    want, tol = _want(x, ids, T, g, h, lse_err, dtype)
    got = ls.token_logprobs_grad(x, None if g is None else ids, lse, g, h, ent if h is not None else None, temperature=T)
    off = (got.double() - want).abs() - tol
    assert off.max().item() <= 0, (off.max().item(), (got.double() - want).norm().item() / want.norm().item())
    if dtype == torch.float32 and not from_forward:
        assert (got.double() - want).norm().item() <= 2e-5 * want.norm().item()
    return got


@pytest.mark.parametrize("from_forward", [False, True])
@pytest.mark.parametrize("T", [0.7, 1.0, 1.3])
@pytest.mark.parametrize("rest", [0.2, 1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("rows,vocab,keep", [(1, 100, 1.0), (1, 1000, 0.01), (3, 4099, 1.0), (2, 51865, 0.5),
                                             (1, 151936, 1.0), (300, 3001, 0.1), (40, 20000, 0.01), (2000, 700, 1.0)])
def test_given_token_that_is_likely(rows, vocab, keep, rest, T, from_forward):
    x, ids = _rows_with(rows, vocab, rest, T, seed=vocab + rows, keep=keep)
    g = torch.randn(rows, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    _check(x, ids, T, g, None, from_forward=from_forward)


@pytest.mark.parametrize("rest", [0.2, 1e-2, 1e-5])
@pytest.mark.parametrize("given", ["likely", "another", "none"])
@pytest.mark.parametrize("rows,vocab", [(1, 300), (5, 5003), (2, 151936), (700, 1025)])
def test_entropy_of_a_row_with_a_likely_id(rows, vocab, given, rest):
    x, ids = _rows_with(rows, vocab, rest, 0.9, seed=vocab, top=0 if given == "likely" else 7)
    g = None if given == "none" else torch.linspace(0.5, 2, rows, device="cuda")
    h = torch.linspace(2, 0.3, rows, device="cuda")
    _check(x, ids, 0.9, g, h)


@pytest.mark.parametrize("rest", [1e-2, 1e-5])
@pytest.mark.parametrize("rows,vocab", [(1, 1000), (33, 51865), (400, 2050)])
def test_bf16(rows, vocab, rest):
    x, ids = _rows_with(rows, vocab, rest, 1.0, seed=rows, dtype=torch.bfloat16)
    g = torch.linspace(-2, 2, rows + 1, device="cuda")[1:]
    _check(x, ids, 1.0, g, None, dtype=torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [3, 600])
@pytest.mark.parametrize("vocab", [45, 1025, 4097, 12007])
def test_alignments_places_and_in_place(vocab, rows, dtype):
    """The likely id in every place that a row starts and ends with, rows between vectors, and over the logits."""
    for place in (0, 1, vocab // 2, vocab - 2, vocab - 1):
        for offset, extra in ((0, 0), (1, 2), (3, 5)):
            x, _ = _rows_with(rows, vocab, 1e-3, 1.0, seed=place, dtype=dtype, offset=offset, extra=extra)
            top = x.float().argmax(dim=1)
            last = x[:, place].clone()
            x[:, place] = x[torch.arange(rows), top]
            x[torch.arange(rows), top] = torch.where(top == place, x[:, place], last)
            ids = torch.full((rows,), place, dtype=torch.int32, device="cuda")
            g = torch.linspace(1, 2, rows, device="cuda")
            got = _check(x, ids, 1.0, g, 0.1 * g, dtype=dtype)
            lse, ent, _ = _state(x, 1.0, False)
            want, tol = _want(x, ids, 1.0, g, 0.1 * g, 0.0, dtype)
            ls.token_logprobs_grad_into(x, ids, lse, x, g, 0.1 * g, ent)
            if offset == 0 and extra == 0:
                assert torch.equal(x, got)
            else:
                # `got` went element by element: the likely id's sum, in which the two weights' parts cancel, has another
                # order there, so that the two differ by 240 u of the sum of magnitudes and not of the result
                assert ((x.double() - want).abs() <= tol).all()


def test_lse_of_a_larger_row():
    """Columns of a longer row with that row's lse and entropy: their entries do not add up to zero, and each is the
    formula's, with what lse's rounding leaves it."""
    rows, vocab = 6, 4001
    x, ids = _rows_with(rows, vocab, 1e-3, 1.0, seed=3)
    own = torch.logsumexp(x.double(), dim=1)
    elsewhere = torch.tensor([0.5, 0.1, 1e-2, 1e-3, 3e-4, 1e-4], dtype=torch.float64, device="cuda")
    lse = (own - torch.log1p(-elsewhere)).float()
    g = torch.ones(rows, device="cuda")
    got = ls.token_logprobs_grad(x, ids, lse, g)
    lp = x.double() - lse.double()[:, None]
    want = -lp.exp()
    want.scatter_add_(1, ids.long()[:, None], torch.ones(rows, 1, dtype=torch.float64, device="cuda"))
    assert ((got.double() - want).abs() <= lp.exp() * U * (4 * lp.abs() / math.log(2) + 9) + 4 * U * want.abs()).all()


def test_entropy_of_rows_without_its_weight_is_not_read():
    """Rows whose entropy weight is 0 may hold anything there."""
    x, ids = _rows_with(8, 3001, 1e-4, 1.0, seed=4)
    lse, ent, _ = _state(x, 1.0, False)
    g = torch.linspace(1, 2, 8, device="cuda")
    h = torch.zeros(8, device="cuda")
    h[::2] = 0.1
    ent[1::2] = math.nan
    got = ls.token_logprobs_grad(x, ids, lse, g, h, ent)
    want, tol = _want(x, ids, 1.0, g, h, 0.0, torch.float32)
    assert ((got.double() - want).abs() <= tol).all()


def test_captured_and_on_two_streams():
    x1, i1 = _rows_with(3, 151936, 1e-4, 1.0, seed=1)
    x2, i2 = _rows_with(500, 1500, 1e-4, 1.0, seed=2)
    calls = []
    for x, ids in ((x1, i1), (x2, i2)):
        lse, ent, _ = _state(x, 1.0, False)
        g = torch.ones(len(ids), device="cuda")
        want = _check(x, ids, 1.0, g, g)
        torch.cuda.synchronize()
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(x)
        with torch.cuda.graph(graph):
            ls.token_logprobs_grad_into(x, ids, lse, out, g, g, ent)
        calls.append((graph, out, want, torch.cuda.Stream(), (x, ids, lse, g, ent)))  # (a graph keeps no tensor alive)
    for _ in range(10):
        for graph, _, _, s, _ in calls:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _ in calls:
        assert torch.equal(out, want)  # the same bits every time


# ---- the forward call ----

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rest", [0.1, 1e-3, 1e-6, 1e-9])
@pytest.mark.parametrize("rows,vocab,offset,T", [
    (1, 1, 0, 1.0), (2, 9, 1, 1.0), (1, 300, 0, 0.7), (3, 900, 2, 1.0), (200, 900, 0, 1.0), (700, 1500, 3, 1.3),
    (2100, 3001, 1, 1.0), (40, 5003, 0, 0.7), (300, 20000, 1, 1.0), (700, 12007, 0, 1.0), (700, 30011, 5, 1.0),
    (2, 51865, 1, 1.0), (1, 151936, 0, 1.3), (20, 151936, 3, 1.0), (1, 262147, 7, 1.0),
])
def test_log_probability_of_a_likely_id(rows, vocab, offset, T, rest, dtype):
    """log p = -ln S of the largest element, S = 1 + the others' exponentials: off by what the others are, 600 u (see
    test_gpu_logprobs.py) and 3 u |d| + 4 u of each, d its distance in powers of 2, relative to themselves; and so the
    entropy ln S + sum e |d| ln 2 / S. Then four roundings of each."""
    x, ids = _rows_with(rows, vocab, rest, T, seed=rows + vocab, dtype=dtype, offset=offset, extra=offset)
    lp, p, _, ent, top = _parts(x, T)
    if vocab == 1:
        x.fill_(1.5)
        lp, p, _, ent, top = _parts(x, T)
    r = ls.token_logprobs(x, ids, temperature=T, n_top=1)
    assert torch.equal(r.top_ids, top.int()) and torch.equal(ids.long(), top[:, 0])
    e = torch.where(p > 0, p / p.gather(1, top), 0.0).scatter(1, top, 0.0)
    d = torch.where(e > 0, -torch.log2(e), 0.0)
    off = e * (600 + 3 * d + 4) * U
    want = lp.gather(1, top)[:, 0]
    tol = off.sum(dim=1) + 4 * U * want.abs()
    assert ((r.logp.double() - want).abs() <= tol).all() and torch.equal(r.top_logp[:, 0], r.logp)
    tol = (off * (2 + d * math.log(2))).sum(dim=1) + 8 * U * ent[:, 0]
    assert ((r.entropy.double() - ent[:, 0]).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [2, 700])
@pytest.mark.parametrize("vocab", [13, 257, 4099, 20011])
def test_the_likely_id_in_every_place(vocab, rows, dtype):
    """At the row's ends and in the vectors that the row only partly fills."""
    for place in (0, 1, 5, vocab // 2, vocab - 2, vocab - 1):
        for offset in (0, 1, 3, 5):
            g = torch.Generator(device="cuda").manual_seed(place + offset)
            buf = torch.randn(rows * (vocab + 3) + 16, generator=g, device="cuda").to(dtype)
            x = buf[offset:offset + rows * (vocab + 3)].view(rows, vocab + 3)[:, :vocab]
            x[:, place] = 20.0
            ids = torch.full((rows,), place, dtype=torch.int32, device="cuda")
            lp, p, _, _, top = _parts(x, 1.0)
            e = (p / p.gather(1, top)).scatter(1, top, 0.0)
            want = lp.gather(1, top)[:, 0]
            tol = (e * (604 - 3 * torch.log2(e.clamp(min=1e-30))) * U).sum(dim=1) + 4 * U * want.abs()
            got = ls.token_logprobs(x, ids, n_top=2).logp
            assert ((got.double() - want).abs() <= tol).all()
