"""The 8-bit LM head: rms_norm_i8, quantize_rows_i8 and lm_head_logits_i8.

Their definitions fix every rounding (the sum of squares is held in 64 bits, the integer product is exact), so the
plain forms below, with the same roundings, have to be met bit for bit. The one place where an order of summation could
show is inv's rounding to f32: 64-bit sums differ by some 1e-15, so for about one row in 10^8. Against the
unrounded definition: inv, the two products, 1 / a, its product with 127 and q's own product are off by 2^-24 each, so
q is off by 1/2 + 127 * 6 * 2^-24.
"""
import math

import numpy as np
import pytest
import torch

import loom_select as ls

pytestmark = pytest.mark.gpu


def _quantise(y):
    """(q, scale) of f32 rows by the documented steps, on the host."""
    y = y.numpy().astype(np.float32)
    a = np.abs(y).max(axis=1)
    q = np.zeros(y.shape, dtype=np.int8)
    scale = np.zeros(len(y), dtype=np.float32)
    for r in range(len(y)):
        if not np.isfinite(a[r]):
            scale[r] = np.nan
        elif a[r] >= 2.0 ** -100:
            inv = (np.float32(1) / a[r]) * np.float32(127)
            q[r] = np.rint(y[r] * inv).astype(np.int8)
            scale[r] = a[r] / np.float32(127)
    return torch.from_numpy(q), torch.from_numpy(scale)


def _norm(x, weight, residual, eps):
    h = x.cpu() if residual is None else (x.cpu().float() + residual.cpu().float()).to(x.dtype)
    hf = h.float().numpy()
    ss = np.square(hf.astype(np.float64)).sum(axis=1)
    with np.errstate(all="ignore"):
        inv = (1.0 / np.sqrt(ss / x.shape[1] + eps)).astype(np.float32)
        y = (hf * inv[:, None]) * weight.cpu().float().numpy()
    return (*_quantise(torch.from_numpy(y)), h)


def _same(a, b):
    return torch.equal(a.cpu().view(torch.uint8 if a.dtype == torch.int8 else torch.int32),
                       b.cpu().view(torch.uint8 if b.dtype == torch.int8 else torch.int32))


def _rows(rows, dim, dtype, seed, offset=0, stride=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    stride = stride or dim
    buf = torch.full((rows * stride + offset + 64,), 7e4, dtype=dtype, device="cuda")
    x = buf[offset:offset + rows * stride].view(rows, stride)[:, :dim]
    v = torch.randn(rows, dim, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))
    x.copy_(v)
    return x


DIMS = [1, 5, 16, 31, 127, 128, 1000, 1024, 1025, 2048, 4096, 5000, 8192, 8193, 16384, 32768]


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", DIMS)
def test_norm(dim, dtype, wdtype):
    rows = 9
    x, res = _rows(rows, dim, dtype, dim), _rows(rows, dim, dtype, dim + 1)
    w = _rows(1, dim, wdtype, dim + 2)[0]
    for residual in (None, res):
        q, scale, total = ls.rms_norm_i8(x, w, residual, eps=1e-5)
        wq, ws, h = _norm(x, w, residual, 1e-5)
        assert _same(q, wq) and _same(scale, ws)
        assert total is None if residual is None else torch.equal(total.cpu(), h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", DIMS)
def test_quantize(dim, dtype):
    x = _rows(33, dim, dtype, dim)
    q, scale = ls.quantize_rows_i8(x)
    wq, ws = _quantise(x.cpu().float())
    assert _same(q, wq) and _same(scale, ws)
    # and against the definition without its f32 steps
    xd = x.double()
    a = xd.abs().amax(dim=1, keepdim=True)
    assert (q.double() - xd / a * 127).abs().max().item() <= 0.5 + 127 * 6 * 2.0 ** -24


@pytest.mark.parametrize("rows", [1, 2, 148, 1000])
def test_norm_row_counts(rows):
    x, res = _rows(rows, 2048, torch.bfloat16, rows), _rows(rows, 2048, torch.bfloat16, rows + 1)
    w = _rows(1, 2048, torch.float32, 3)[0]
    q, scale, total = ls.rms_norm_i8(x, w, res)
    wq, ws, h = _norm(x, w, res, 1e-6)
    assert _same(q, wq) and _same(scale, ws) and torch.equal(total.cpu(), h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,extra", [(1, 0), (0, 1), (4, 4), (3, 5), (8, 8)])
@pytest.mark.parametrize("dim", [40, 1001, 2048])
def test_norm_alignment_strides_and_untouched_gaps(offset, extra, dim, dtype):
    rows = 6
    x = _rows(rows, dim, dtype, 1, offset, dim + extra)
    res = _rows(rows, dim, dtype, 2, extra, dim + offset)
    w = _rows(1, dim, torch.float32, 3, offset)[0]
    buf = torch.full((rows * (dim + extra) + 64,), 55.0, dtype=dtype, device="cuda")
    total = buf[offset:offset + rows * (dim + extra)].view(rows, dim + extra)[:, :dim]
    qbuf = torch.full((rows * dim + 32,), 99, dtype=torch.int8, device="cuda")
    q = qbuf[offset:offset + rows * dim].view(rows, dim)
    scale = torch.empty(rows, device="cuda")
    ls.rms_norm_i8_into(x, w, q, scale, res, total)
    wq, ws, h = _norm(x, w, res, 1e-6)
    assert _same(q, wq) and _same(scale, ws) and torch.equal(total.cpu(), h)
    q.fill_(99)
    total.fill_(55.0)
    assert (qbuf == 99).all() and (buf == 55.0).all()
    q2, s2 = ls.quantize_rows_i8(x)
    assert _same(q2, _quantise(x.cpu().float())[0]) and _same(s2, _quantise(x.cpu().float())[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [*range(1, 50), 255, 257, 509, 1023, 4097])
def test_every_small_width_unaligned(dim, dtype):
    rows = 5
    for offset in (1, 6):
        x, res = _rows(rows, dim, dtype, 1, offset), _rows(rows, dim, dtype, 2, offset + 1, dim + 1)
        w = _rows(1, dim, torch.float32, 3, offset)[0]
        wq, ws, h = _norm(x, w, res, 1e-6)
        q, scale, total = ls.rms_norm_i8(x, w, res)
        assert _same(q, wq) and _same(scale, ws) and torch.equal(total.cpu(), h)
        wq, ws = _quantise(x.cpu().float())
        qbuf = torch.full((rows * dim + 40,), 99, dtype=torch.int8, device="cuda")
        q = qbuf[offset + 2:offset + 2 + rows * dim].view(rows, dim)
        ls.quantize_rows_i8_into(x, q, scale)
        assert _same(q, wq) and _same(scale, ws)
        q.fill_(99)
        assert (qbuf == 99).all()


@pytest.mark.parametrize("into", ["x", "residual"])
def test_norm_in_place(into):
    x, res = _rows(5, 4096, torch.bfloat16, 1), _rows(5, 4096, torch.bfloat16, 2)
    w = _rows(1, 4096, torch.float32, 3)[0]
    wq, ws, h = _norm(x, w, res, 1e-6)
    q, scale = torch.empty(5, 4096, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
    total = x if into == "x" else res
    ls.rms_norm_i8_into(x, w, q, scale, res, total)
    assert _same(q, wq) and _same(scale, ws) and torch.equal(total.cpu(), h)


@pytest.mark.parametrize("dim", [64, 3001])
def test_special_rows(dim):
    x = _rows(8, dim, torch.float32, 4)
    x[0] = 0
    x[1, 3] = math.nan
    x[2, dim - 1] = math.inf
    x[3, 0] = -math.inf
    x[4] = 1e-38
    x[5] = 3e38
    x[6] = -0.0
    for q, scale in (ls.quantize_rows_i8(x), ls.rms_norm_i8(x, torch.ones(dim, device="cuda"))[:2]):
        assert (q[0] == 0).all() and scale[0].item() == 0 and (q[6] == 0).all() and scale[6].item() == 0
        for r in (1, 2, 3):
            assert (q[r] == 0).all() and math.isnan(scale[r].item())
        assert (q[5] == 127).all() and math.isfinite(scale[5].item())
    q, scale = ls.quantize_rows_i8(x)
    assert (q[4] == 0).all() and scale[4].item() == 0
    wq, ws = _quantise(x.cpu())
    assert _same(q, wq) and torch.equal(torch.isnan(scale).cpu(), torch.isnan(ws))


# ---- the product ----

def _operands(rows, hidden, vocab, seed, lo=-127):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(lo, 128, (rows, hidden), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(lo, 128, (vocab, hidden), generator=g, device="cuda", dtype=torch.int8)
    return q, torch.rand(rows, generator=g, device="cuda") + 0.01, w, torch.rand(vocab, generator=g, device="cuda") + 0.01


def _product(q, qs, w, ws, dtype):
    acc = q.double() @ w.double().t()  # exact: below 2^53
    return (acc.float() * qs[:, None] * ws).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,hidden,vocab", [
    (1, 16, 1), (1, 128, 7), (2, 144, 208), (3, 48, 209), (16, 1024, 4099), (17, 1040, 4099), (127, 256, 256),
    (128, 128, 257), (129, 272, 513), (200, 512, 4099), (1, 2048, 151936), (300, 96, 51865), (16, 8192, 3001),
    (70, 65536, 300),
])
def test_product(rows, hidden, vocab, dtype):
    q, qs, w, ws = _operands(rows, hidden, vocab, rows + hidden + vocab, lo=-128)
    out = ls.lm_head_logits_i8(q, qs, w, ws, dtype=dtype)
    assert torch.equal(out, _product(q, qs, w, ws, dtype))


@pytest.mark.parametrize("rows,hidden,vocab", [(1024, 2048, 151936), (1024, 512, 30011)])
def test_product_many_rows(rows, hidden, vocab):
    q, qs, w, ws = _operands(rows, hidden, vocab, 5)
    out = ls.lm_head_logits_i8(q, qs, w, ws, dtype=torch.bfloat16)
    for v in range(0, vocab, 32768):
        assert torch.equal(out[:, v:v + 32768], _product(q, qs, w[v:v + 32768], ws[v:v + 32768], torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,hidden,vocab", [
    (150, 272, 20011), (185, 144, 20011), (220, 48, 20011), (256, 1040, 20011), (260, 128, 30000), (700, 400, 20011),
    (129, 8192, 130), (300, 1040, 500), (600, 400, 1900), (1000, 272, 1100), (1024, 2048, 100),
])
def test_product_tile_shapes(rows, hidden, vocab, dtype):
    """Every height of tile, of pairs and of single CTAs, with rows and ids left over."""
    q, qs, w, ws = _operands(rows, hidden, vocab, rows + vocab, lo=-128)
    out = ls.lm_head_logits_i8(q, qs, w, ws, dtype=dtype)
    assert torch.equal(out, _product(q, qs, w, ws, dtype))


@pytest.mark.parametrize("hidden", [2048, 65536])
def test_product_extremes(hidden):
    """The largest sums of either sign: 2^14 hidden, at most 2^30."""
    rows, vocab = 20, 300
    q = torch.full((rows, hidden), -128, dtype=torch.int8, device="cuda")
    w = torch.full((vocab, hidden), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    one_r, one_v = torch.ones(rows, device="cuda"), torch.ones(vocab, device="cuda")
    out = ls.lm_head_logits_i8(q, one_r, w, one_v)
    assert (out[:, ::2] == 16384.0 * hidden).all() and (out[:, 1::2] == -16256.0 * hidden).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,extra", [(0, 1), (1, 0), (1, 2), (3, 5), (8, 64)])
@pytest.mark.parametrize("rows", [5, 140])
def test_product_strided_output_and_untouched_gaps(rows, offset, extra, dtype):
    vocab = 777
    q, qs, w, ws = _operands(rows, 256, vocab, 11)
    buf = torch.full((rows * (vocab + extra) + offset + 64,), 55.0, dtype=dtype, device="cuda")
    out = buf[offset:offset + rows * (vocab + extra)].view(rows, vocab + extra)[:, :vocab]
    ls.lm_head_logits_i8_into(q, qs, w, ws, out)
    assert torch.equal(out, _product(q, qs, w, ws, dtype))
    out.fill_(55.0)
    assert (buf == 55.0).all()


def test_product_nan_scale_reaches_its_row_only():
    q, qs, w, ws = _operands(4, 64, 500, 3)
    q[2], qs[2] = 0, math.nan
    out = ls.lm_head_logits_i8(q, qs, w, ws)
    assert torch.isnan(out[2]).all() and torch.isfinite(out[[0, 1, 3]]).all()


def test_product_offsets_past_32_bits():
    """Output rows whose offset passes 2^31 elements (a view with a huge stride: only its first and last rows are kept)."""
    rows, vocab, stride = 3, 1000, (1 << 30) + 24
    q, qs, w, ws = _operands(rows, 64, vocab, 8)
    buf = torch.empty(2 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    out = torch.as_strided(buf, (rows, vocab), (stride, 1))
    ls.lm_head_logits_i8_into(q, qs, w, ws, out)
    assert torch.equal(out, _product(q, qs, w, ws, torch.bfloat16))
    r = ls.token_logprobs(out, torch.zeros(rows, dtype=torch.int32, device="cuda"), n_top=4)
    assert torch.equal(r.top_ids, ls.token_logprobs(out.contiguous(), None, n_top=4).top_ids)


@pytest.mark.parametrize("rows", [40, 300])
def test_wait_that_gives_up_is_reported(rows):
    """The bounded waits' give-up path, through the test hook (nothing faults), of single CTAs and of pairs; the next
    call is exact again."""
    q, qs, w, ws = _operands(rows, 512, 60000, 9)
    want = _product(q, qs, w, ws, torch.float32)
    mine = ls.Workspace(torch.device("cuda", torch.cuda.current_device()))
    buf = mine.get(256)
    out = torch.empty(rows, 60000, device="cuda")
    ls.check(ls.lib().loom_select_test_wait_fault(ls._ptr(buf), 50_000, 2, ls._stream_handle()), "hook")
    ls.lm_head_logits_i8_into(q, qs, w, ws, out, workspace=mine)
    assert mine.read_status() == ls.ETIMEOUT
    ls.check(ls.lib().loom_select_workspace_init(ls._ptr(buf), buf.numel(), ls._stream_handle()), "init")
    ls.lm_head_logits_i8_into(q, qs, w, ws, out, workspace=mine)
    assert mine.read_status() == ls.OK
    assert torch.equal(out, want)


def test_one_row_of_any_stride():
    """A row's own stride means nothing when there is one: views that torch gives an odd one are taken."""
    q, qs, w, ws = _operands(1, 256, 500, 4)
    out = torch.empty(500, 1, device="cuda").t()
    ls.lm_head_logits_i8_into(q, qs, w, ws, out)
    assert torch.equal(out, _product(q, qs, w, ws, torch.float32))
    x = torch.randn(64, 1, device="cuda").t()
    assert _same(ls.quantize_rows_i8(x)[0], ls.quantize_rows_i8(x.contiguous())[0])
    assert torch.equal(ls.token_logprobs(out).lse, ls.token_logprobs(out.contiguous()).lse)


def test_two_streams_and_two_graphs_at_once():
    a, b = _operands(1, 1024, 50000, 1), _operands(200, 256, 20000, 2)
    wa, wb = _product(*a, torch.float32), _product(*b, torch.float32)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        ra = ls.lm_head_logits_i8(*a, stream=s1)
        rb = ls.lm_head_logits_i8(*b, stream=s2)
        torch.cuda.synchronize()
        assert torch.equal(ra, wa) and torch.equal(rb, wb)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        ra = ls.lm_head_logits_i8(*a)
    with torch.cuda.graph(g2):
        rb = ls.lm_head_logits_i8(*b)
    for _ in range(5):
        ra.zero_(), rb.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(ra, wa) and torch.equal(rb, wb)


# ---- the chain ----

@pytest.mark.parametrize("rows", [1, 33])
def test_chain_from_hidden_states_to_scored_tokens(rows):
    """Final norm, 8-bit LM head, greedy and sampled tokens, their log-probabilities, and the gradient back."""
    hidden, vocab, T = 1024, 30011, 0.8
    x, res = _rows(rows, hidden, torch.bfloat16, 1), _rows(rows, hidden, torch.bfloat16, 2)
    norm_w = 1 + 0.1 * _rows(1, hidden, torch.float32, 3)[0].tanh()
    g = torch.Generator(device="cuda").manual_seed(4)
    head = torch.randn(vocab, hidden, generator=g, device="cuda").to(torch.bfloat16) / 10
    w8, w_scale = ls.quantize_rows_i8(head)
    q, scale, total = ls.rms_norm_i8(x, norm_w, res)
    logits = ls.lm_head_logits_i8(q, scale, w8, w_scale)
    u = torch.rand(rows, generator=g, device="cuda")
    ids, _, logp, topk = ls.sample_rows(logits, u, T, top_k=8, want_logp=True, want_topk=True)
    r = ls.token_logprobs(logits, ids, temperature=T, n_top=8, want_rank=True)
    d = ls.token_logprobs_grad(logits, ids, r.lse, torch.ones(rows, device="cuda"), temperature=T)

    want_q, want_scale, h = _norm(x, norm_w, res, 1e-6)
    assert _same(q, want_q) and torch.equal(total.cpu(), h)
    want = _product(q, scale, w8, w_scale, torch.float32)
    assert torch.equal(logits, want)
    assert [int(v) for v in ls.argmax_rows(logits)] == r.top_ids[:, 0].tolist()
    assert torch.equal(r.top_ids, topk)
    lp = torch.log_softmax(want.double() / T, dim=1)
    picked = lp.gather(1, ids.long()[:, None])[:, 0]
    assert ((r.logp - picked).abs() <= 4e-5 + 1e-6 * picked.abs()).all()  # (the bounds of the two calls: see their tests)
    assert ((r.logp - logp).abs() <= 5e-5 + 1e-5 * logp.abs()).all()
    back = -lp.exp()
    back.scatter_add_(1, ids.long()[:, None], torch.ones_like(picked)[:, None])
    assert ((d.double() - back / T).abs().max() <= 1e-4)
    # 8 bits per hidden state and weight: each is off by at most half a step, 1 / 254 of its row's largest
    y = h.double().cuda() * torch.rsqrt(h.double().cuda().square().mean(dim=1, keepdim=True) + 1e-6) * norm_w.double()
    full = y @ head.double().t()
    step_q = (scale.double() * (0.5 + 1e-4))[:, None]
    step_w = w_scale.double() * (0.5 + 1e-4)
    bound = step_q * head.double().abs().sum(dim=1) + y.abs().sum(dim=1, keepdim=True) * step_w + hidden * step_q * step_w
    assert ((logits.double() - full).abs() <= bound * (1 + 1e-5)).all()


@pytest.mark.parametrize("rows", [130, 160, 161, 193, 224, 225, 257, 321, 400, 449, 513, 700])
def test_product_row_tiles(rows):
    """Every height of a tile of rows, one tile and several, with a last tile that is not full."""
    q, qs, w, ws = _operands(rows, 160, 1500, rows)
    out = ls.lm_head_logits_i8(q, qs, w, ws)
    assert torch.equal(out, _product(q, qs, w, ws, torch.float32))


def test_captured_calls_use_the_status_word_that_is_there():
    """Two graphs and an eager call, which share the device's status word, side by side."""
    q, qs, w, ws = _operands(9, 512, 4099, 6)
    want = ls.lm_head_logits_i8(q, qs, w, ws)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
        with torch.cuda.graph(g):
            ls.lm_head_logits_i8_into(q, qs, w, ws, out)
        graphs.append((g, out, torch.cuda.Stream()))
    for _ in range(10):
        for g, out, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        eager = ls.lm_head_logits_i8(q, qs, w, ws)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, _ in graphs) and torch.equal(eager, want)
