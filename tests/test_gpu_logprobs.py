"""token_logprobs and its gradient against their definitions in 64 bits.

Tolerances, in units u = 2^-24 (half a step of f32, relative). A term 2^((x - m) c) carries 3u |d| from the
difference, the product and the constant c, and 4u from ex2; |d| weighted by the probabilities is the entropy in
bits, at most 18 here. A thread adds at most 64 partial sums of 16 elements (16 + 64 roundings), rescales them when
its maximum rises (at most 64 times, 6u each), and 13 merges follow (6u each): below
(54 + 4 + 80 + 384 + 78) u = 600 u = 3.6e-5 for log S. That bound is TOL; the entropy's second term A / S carries
the same relative error, |A / S| < 13.
"""
import math

import pytest
import torch

import loom_select as ls

pytestmark = pytest.mark.gpu

TOL = 600 * 2.0 ** -24
U = 2.0 ** -24


def _reference(x, ids, T, n_top):
    """All outputs in 64 bits, by the documented rules (rows without NaN or +inf)."""
    xd = x.double()
    y = xd / T
    lp = torch.log_softmax(y, dim=1)
    empty = torch.isinf(xd).all(dim=1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(dim=1)
    ent[empty] = math.nan
    V = x.shape[1]
    t = ids.long()
    has = (t >= 0) & (t < V)
    at = t.clamp(0, V - 1)[:, None]
    logp = torch.where(has, lp.gather(1, at)[:, 0], torch.where(t < 0, 0.0, math.nan))
    idx = torch.arange(V, device=x.device)
    xt = xd.gather(1, at)
    rank = torch.where(has, ((xd > xt) | ((xd == xt) & (idx < at))).sum(dim=1), -1).int()
    # stable sort, descending: equal values keep the lower id first
    order = torch.sort(xd, dim=1, descending=True, stable=True).indices[:, :n_top]
    return {"logp": logp, "entropy": ent, "lse": torch.logsumexp(y, dim=1), "rank": rank, "top_ids": order.int(),
            "top_logp": lp.gather(1, order)}


def _close(got, want, tol, name):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), name
    err = (got - want)[fin].abs() - tol(want[fin])
    assert err.numel() == 0 or err.max().item() <= 0, (name, err.max().item())


def _check(x, ids, T=1.0, n_top=0):
    r = ls.token_logprobs(x, ids, temperature=T, n_top=n_top, want_rank=True)
    torch.cuda.synchronize()
    w = _reference(x, ids, T, n_top)
    # an lse past f32's largest value, (2 - 2^-23) 2^127 (the lowest value over T = 0.9 is -3.78e38), is infinite in f32
    lse = torch.where(w["lse"].abs() >= 2.0 ** 128, w["lse"].float().double(), w["lse"])
    _close(r.lse, lse, lambda v: TOL + 2 * U * v.abs(), "lse")
    _close(r.logp, w["logp"], lambda v: TOL + 4 * U * v.abs(), "logp")
    _close(r.entropy, w["entropy"], lambda v: 14 * TOL, "entropy")
    assert torch.equal(r.rank, w["rank"])
    if n_top:
        assert torch.equal(r.top_ids, w["top_ids"])
        _close(r.top_logp, w["top_logp"], lambda v: TOL + 4 * U * v.abs(), "top_logp")
    return r


def _logits(rows, vocab, seed, dtype=torch.float32, offset=0, stride=None, scale=3.0):
    """N(0, scale^2) rows of any stride whose first element lies `offset` elements past an aligned address."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    stride = stride or vocab
    buf = torch.full((rows * stride + offset + 64,), 1e9, dtype=dtype, device="cuda")
    x = buf[offset:offset + rows * stride].view(rows, stride)[:, :vocab]
    x.copy_(torch.randn(rows, vocab, generator=g, device="cuda") * scale)
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return x, ids


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,n_top", [
    (1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 8, 8), (4, 9, 0), (3, 31, 31), (3, 33, 32), (2, 257, 5), (3, 1000, 20),
    (9, 4099, 32), (40, 30011, 1), (77, 51865, 3), (1, 151936, 20), (2, 151936, 32), (300, 151936, 5), (1, 262144, 32),
])
def test_against_64_bits(rows, vocab, n_top, dtype):
    x, ids = _logits(rows, vocab, seed=rows + vocab, dtype=dtype)
    _check(x, ids, n_top=n_top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,extra", [(1, 0), (3, 1), (0, 7), (5, 3), (7, 13)])
@pytest.mark.parametrize("vocab", [6, 13, 2049, 20000])
def test_any_alignment_and_stride(offset, extra, vocab, dtype):
    x, ids = _logits(6, vocab, seed=vocab + offset, dtype=dtype, offset=offset, stride=vocab + extra)
    _check(x, ids, T=0.7, n_top=min(vocab, 9))


@pytest.mark.parametrize("T", [0.05, 0.7, 1.0, 3.0, 1e4])
def test_temperatures(T):
    x, ids = _logits(7, 12345, seed=4)
    _check(x, ids, T=T, n_top=4)


@pytest.mark.parametrize("kind", ["ascending", "descending", "equal", "few values", "one peak", "huge"])
@pytest.mark.parametrize("vocab", [100, 40001])
def test_value_patterns(kind, vocab):
    x, ids = _logits(4, vocab, seed=8)
    if kind == "ascending":
        x.copy_(torch.linspace(-30, 30, vocab, device="cuda").expand(4, -1))
    elif kind == "descending":
        x.copy_(torch.linspace(30, -30, vocab, device="cuda").expand(4, -1))
    elif kind == "equal":
        x.fill_(2.5)
    elif kind == "few values":
        x.copy_(x.round().clamp(-2, 2))
        x[0, ::3] = -0.0
    elif kind == "one peak":
        x[:, vocab // 2] = 200.0
    else:
        x.mul_(1e4)
    _check(x, ids, n_top=20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks(dtype):
    vocab = 20011
    x, ids = _logits(8, vocab, seed=15, dtype=dtype)
    x[0, :] = -math.inf                       # empty row
    x[1, 5:] = -math.inf                      # fewer ids than alternatives
    x[2, :] = torch.finfo(dtype).min          # masks of the lowest value only: a uniform row
    x[3, 100:] = torch.finfo(dtype).min
    x[4, ids[4].item()] = -math.inf           # the given token itself is masked
    x[5, :vocab - 1] = -math.inf              # one id left, the last
    x[6, 1:] = -math.inf                      # one id left, the first
    r = _check(x, ids, n_top=20)
    assert r.lse[0].item() == -math.inf and math.isnan(r.logp[0].item()) and math.isnan(r.entropy[0].item())
    assert r.top_ids[0].tolist() == list(range(20)) and torch.isnan(r.top_logp[0]).all()
    assert r.logp[4].item() == -math.inf
    assert r.entropy[5].item() == 0.0 and r.top_ids[5, 0].item() == vocab - 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 3])
def test_few_long_rows(dtype, offset):
    """Long rows that have the device to themselves: masks, ties and edges there (each thread's sums are shorter than the
    bound's)."""
    vocab = 262147
    x, ids = _logits(7, vocab, seed=57, dtype=dtype, offset=offset, stride=vocab + 5)
    x[0, :] = -math.inf
    x[1, 5:] = -math.inf
    x[2, :] = torch.finfo(dtype).min
    x[3, :] = x[3].round().clamp(-2, 2)
    x[4, ::2] = -math.inf
    x[5, :vocab - 1] = -math.inf
    ids[3], ids[5] = vocab - 1, vocab - 1
    for n_top in (0, 5, 32):
        _check(x, ids, T=0.9, n_top=n_top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,offset", [(160, 3001, 1), (151, 8000, 0), (700, 8193, 0), (640, 12007, 3),
                                               (1201, 20000, 1)])
def test_many_rows(rows, vocab, offset, dtype):
    """Rows enough for every block of the device, some of them masked, tied, empty or with their token at the ends."""
    x, ids = _logits(rows, vocab, seed=rows, dtype=dtype, offset=offset, stride=vocab + offset)
    x[0::7] = x[0::7].round().clamp(-2, 2)
    x[1::7, 40:] = -math.inf
    x[2::49, :] = -math.inf
    x[3::7, ::3] = -math.inf
    x[4::7, 3:] = -math.inf
    x[5::49, :] = torch.finfo(dtype).min
    ids[::5], ids[1::5], ids[2::25] = 0, vocab - 1, -1
    for n_top in (0, 7, 32):
        _check(x, ids, T=1.0, n_top=n_top)


def test_ids_outside_the_vocabulary():
    x, ids = _logits(4, 1000, seed=2)
    ids[0], ids[1], ids[2] = -1, -100, 1000
    r = _check(x, ids, n_top=2)
    assert r.logp[0].item() == 0 and r.logp[1].item() == 0 and math.isnan(r.logp[2].item())
    assert r.rank[:3].tolist() == [-1, -1, -1]


def test_nan_and_inf_logits():
    x, ids = _logits(5, 5000, seed=3)
    x[0, 17] = math.nan
    x[1, 4000] = math.inf
    x[2, :] = math.nan
    x[3, 3:] = math.nan
    ids[2] = 5
    clean = x[4:5].clone()
    r = ls.token_logprobs(x, ids, n_top=5, want_rank=True)
    for row in (0, 1, 2, 3):
        assert math.isnan(r.lse[row].item()) and math.isnan(r.logp[row].item()) and math.isnan(r.entropy[row].item())
        assert torch.isnan(r.top_logp[row]).all()
    assert 17 not in r.top_ids[0].tolist() and r.top_ids[1, 0].item() == 4000
    assert r.top_ids[2].tolist() == [-1] * 5 and r.rank[2].item() == -1
    want = torch.sort(x[3, :3], descending=True).indices.tolist()
    assert r.top_ids[3].tolist() == want + [-1, -1]
    alone = ls.token_logprobs(clean, ids[4:5], n_top=5, want_rank=True)
    for a, b in zip(r, alone):
        assert torch.equal(a[4:5], b)  # a neighbour's NaN changes nothing


def test_every_subset_of_outputs_agrees():
    x, ids = _logits(6, 9001, seed=21)
    full = ls.token_logprobs(x, ids, n_top=6, want_rank=True)
    for k in range(4):
        outs = [torch.empty_like(full[k]) if j == k else None for j in range(4)]
        ls.token_logprobs_into(x, ids if k in (0, 3) else None, *outs)
        assert torch.equal(outs[k], full[k])
    only_ids, only_logp = torch.empty_like(full.top_ids), torch.empty_like(full.top_logp)
    ls.token_logprobs_into(x, None, out_top_ids=only_ids)
    ls.token_logprobs_into(x, None, out_top_logp=only_logp)
    assert torch.equal(only_ids, full.top_ids) and torch.equal(only_logp, full.top_logp)


def test_one_dimensional_row():
    x, _ = _logits(1, 777, seed=5)
    r = ls.token_logprobs(x[0], torch.tensor([9], dtype=torch.int32, device="cuda"), n_top=3, want_rank=True)
    two = ls.token_logprobs(x, torch.tensor([9], dtype=torch.int32, device="cuda"), n_top=3, want_rank=True)
    assert torch.equal(r.logp, two.logp) and torch.equal(r.top_ids, two.top_ids[0]) and torch.equal(r.rank, two.rank)


def test_agrees_with_the_sampler():
    """The sampled token's log-probability and the alternatives are those of loom_sample_rows."""
    x, _ = _logits(16, 151936, seed=33)
    u = torch.rand(16, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    ids, _, logp, topk = ls.sample_rows(x, u, 0.7, top_k=20, top_p=0.95, want_logp=True, want_topk=True)
    r = ls.token_logprobs(x, ids, temperature=0.7, n_top=20, want_rank=True)
    assert torch.equal(r.top_ids, topk)
    assert (r.rank < 20).all() and torch.equal(topk.gather(1, r.rank.long()[:, None])[:, 0], ids)
    _close(r.logp, logp, lambda v: TOL + 1e-5 * v.abs().clamp(min=1), "sampled logp")


def test_captured_graphs_replayed_side_by_side():
    x1, i1 = _logits(3, 151936, seed=41)
    x2, i2 = _logits(50, 20000, seed=42)
    w1, w2 = ls.token_logprobs(x1, i1, n_top=7), ls.token_logprobs(x2, i2, n_top=7)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1 = ls.token_logprobs(x1, i1, n_top=7)
    with torch.cuda.graph(g2):
        r2 = ls.token_logprobs(x2, i2, n_top=7)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
    torch.cuda.synchronize()
    for r, w in ((r1, w1), (r2, w2)):
        for a, b in zip(r, w):
            assert a is b is None or torch.equal(a, b)


def test_given_stream_owns_its_results():
    x, ids = _logits(4, 50000, seed=9)
    want = ls.token_logprobs(x, ids, n_top=3)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = ls.token_logprobs(x, ids, n_top=3, stream=s)
    s.synchronize()
    assert torch.equal(got.logp, want.logp) and torch.equal(got.top_ids, want.top_ids)


# ---- the gradient ----

def _grad_reference(x, ids, T, g, h):
    xd = x.double()
    lp = torch.log_softmax(xd / T, dim=1)
    p = lp.exp()
    V = x.shape[1]
    has = (ids >= 0) & (ids < V)
    gg = torch.where(has, g.double(), 0.0)
    d = -gg[:, None] * p
    if h is not None:
        ent = -torch.where(p > 0, p * lp, 0.0).sum(dim=1, keepdim=True)
        d -= h.double()[:, None] * torch.where(p > 0, p * (lp + ent), 0.0)
    d.scatter_add_(1, ids.long().clamp(0, V - 1)[:, None], gg[:, None])
    return d / T


def _grad_tol(x, T, g, h, want, dtype):
    """|p| is off by e^TOL from lse (rounded to f32 on top: u |lse|), u |l| from l = x / T - lse, 3u |l| from the
    exponent's product and 4u from ex2; l + H by as much again. Then five f32 roundings, and the type's own."""
    xd = x.double()
    lp = torch.log_softmax(xd / T, dim=1)
    p = lp.exp()
    lse = torch.logsumexp(xd / T, dim=1, keepdim=True).abs()
    l = torch.where(p > 0, lp, 0.0).abs()
    rel = TOL + U * (2 * lse + 4 * l + 16)
    w = g.abs().double()[:, None]
    if h is not None:
        w = w + h.abs().double()[:, None] * (l + 13 + 14 * TOL)
    tol = p * (w * rel + (h.abs().double()[:, None] * 15 * TOL if h is not None else 0.0)) / T
    return tol + want.abs() * (torch.finfo(dtype).eps / 2 + 4 * U) + 1e-38


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,T,entropy", [
    (1, 1, 1.0, True), (3, 5, 1.0, True), (2, 8, 0.7, False), (4, 1000, 1.0, True), (5, 1003, 0.7, True),
    (77, 51865, 1.0, False), (3, 151936, 1.3, True), (300, 4099, 0.7, True), (1, 262144, 1.0, True),
])
def test_grad_against_64_bits(rows, vocab, T, entropy, dtype):
    x, ids = _logits(rows, vocab, seed=rows * 3 + vocab, dtype=dtype)
    g = torch.randn(rows, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    h = 0.1 * g.flip(0) if entropy else None
    f = ls.token_logprobs(x, ids, temperature=T)
    got = ls.token_logprobs_grad(x, ids, f.lse, g, h, f.entropy if entropy else None, temperature=T)
    want = _grad_reference(x, ids, T, g, h)
    assert got.dtype == dtype and got.shape == x.shape
    off = (got.double() - want).abs() - _grad_tol(x, T, g, h, want, dtype)
    assert off.max().item() <= 0, off.max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off_in,extra_in,off_out,extra_out", [(0, 0, 1, 3), (3, 1, 3, 1), (1, 2, 0, 0), (5, 8, 5, 0)])
def test_grad_alignment_strides_and_untouched_gaps(off_in, extra_in, off_out, extra_out, dtype):
    rows, vocab = 5, 3001
    x, ids = _logits(rows, vocab, seed=1, dtype=dtype, offset=off_in, stride=vocab + extra_in)
    buf = torch.full((rows * (vocab + extra_out) + off_out + 16,), 77.0, dtype=dtype, device="cuda")
    out = buf[off_out:off_out + rows * (vocab + extra_out)].view(rows, vocab + extra_out)[:, :vocab]
    g = torch.ones(rows, device="cuda")
    f = ls.token_logprobs(x, ids)
    ls.token_logprobs_grad_into(x, ids, f.lse, out, g, g, f.entropy)
    assert torch.equal(out, ls.token_logprobs_grad(x.contiguous(), ids, f.lse, g, g, f.entropy))
    out.fill_(77.0)
    assert (buf == 77.0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_in_place(dtype):
    x, ids = _logits(6, 7001, seed=12, dtype=dtype, offset=1, stride=7003)
    g = torch.linspace(-1, 1, 6, device="cuda")
    f = ls.token_logprobs(x, ids)
    want = ls.token_logprobs_grad(x, ids, f.lse, g, g, f.entropy)
    ls.token_logprobs_grad_into(x, ids, f.lse, x, g, g, f.entropy)
    assert torch.equal(x, want)


def test_grad_masks_padding_and_bad_rows():
    V = 5003
    x, ids = _logits(7, V, seed=6)
    x[0, 10:] = -math.inf
    ids[0] = 3
    ids[1] = -1                    # padding: only the entropy's part
    x[2, :] = -math.inf            # an empty row without weight: zeros
    x[3, :] = -math.inf            # an empty row with weight: NaN
    ids[4] = V                     # an id past the vocabulary: NaN
    x[5, 7] = math.nan             # NaN without weight: zeros
    g = torch.ones(7, device="cuda")
    h = torch.ones(7, device="cuda")
    for r in (2, 5):
        g[r] = h[r] = 0
    f = ls.token_logprobs(x, ids)
    d = ls.token_logprobs_grad(x, ids, f.lse, g, h, f.entropy)
    assert (d[0, 10:] == 0).all() and torch.isfinite(d[0]).all()
    assert (d[2] == 0).all() and (d[5] == 0).all()
    assert torch.isnan(d[3]).all() and torch.isnan(d[4]).all()
    only_h = ls.token_logprobs_grad(x, None, f.lse, None, h, f.entropy)
    assert torch.equal(d[1], only_h[1])
    for r in (0, 1, 6):
        want = _grad_reference(x[r:r + 1], ids[r:r + 1], 1.0, g[r:r + 1], h[r:r + 1])
        tol = _grad_tol(x[r:r + 1], 1.0, g[r:r + 1], h[r:r + 1], want, torch.float32)
        assert ((d[r:r + 1].double() - want).abs() - tol).max().item() <= 0


def test_grad_against_differences():
    """Central differences of the 64-bit objective: the gradient formula itself, not only its arithmetic."""
    V, T, eps = 23, 0.8, 1e-5
    x, ids = _logits(2, V, seed=19)
    g, h = torch.tensor([1.5, -0.5], device="cuda"), torch.tensor([0.3, 0.7], device="cuda")

    def objective(xd):
        lp = torch.log_softmax(xd / T, dim=1)
        picked = lp.gather(1, ids.long()[:, None])[:, 0]
        return (g.double() * picked - h.double() * (lp.exp() * lp).sum(dim=1)).sum().item()

    f = ls.token_logprobs(x, ids, temperature=T)
    d = ls.token_logprobs_grad(x, ids, f.lse, g, h, f.entropy, temperature=T)
    for r in range(2):
        for j in range(V):
            e = torch.zeros(2, V, dtype=torch.float64, device="cuda")
            e[r, j] = eps
            diff = (objective(x.double() + e) - objective(x.double() - e)) / (2 * eps)
            # third derivatives below 10: 10 eps^2 / 6, 64-bit cancellation 1e-15 / eps, the kernel's f32
            assert abs(diff - d[r, j].item()) <= 1e-9 + 1e-9 + 20 * TOL


def test_grad_captured_into_a_graph():
    x, ids = _logits(9, 30000, seed=14)
    g = torch.ones(9, device="cuda")
    f = ls.token_logprobs(x, ids)
    want = ls.token_logprobs_grad(x, ids, f.lse, g, g, f.entropy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f2 = ls.token_logprobs(x, ids)
        d = ls.token_logprobs_grad(x, ids, f2.lse, g, g, f2.entropy)
    for _ in range(3):
        d.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 30011), (3, 151936), (200, 3001), (400, 20000)])
def test_fewer_finite_ids_than_alternatives(rows, vocab, dtype):
    """Constrained decoding: a handful of ids allowed, the alternatives run into the masked ones, lowest ids first."""
    x, ids = _logits(rows, vocab, seed=rows, dtype=dtype)
    keep = torch.rand(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") < 10.0 / vocab
    keep.scatter_(1, ids.long()[:, None], True)
    x.masked_fill_(~keep, -math.inf)
    _check(x, ids, n_top=32)


@pytest.mark.parametrize("rows,vocab", [(2, 151936), (300, 20000), (500, 2000)])
def test_many_ties_at_the_threshold(rows, vocab):
    """More equal values at the n_top-th place than the candidates' store holds: the lowest ids win."""
    x, ids = _logits(rows, vocab, seed=rows, dtype=torch.bfloat16)
    x.copy_((x / 4).round())
    x[:, vocab // 3:vocab // 3 + 7] = 50.0
    _check(x, ids, n_top=20)
