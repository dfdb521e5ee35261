"""The measured cases of the scoring and 8-bit LM-head operators.

Operators: token_logprobs (log-probabilities of given tokens with entropy, rank and top alternatives),
token_logprobs_grad (its gradient), rms_norm_i8 (residual addition, RMS norm, 8-bit output with a scale
per row), quantize_rows_i8 (the same quantisation of plain rows: an LM-head weight) and
lm_head_logits_i8 (the 8-bit integer LM-head product with scales per row and per vocabulary id).

run() computes them in elementary torch operations, or, where `own` is true, through the framework's
calls. exact() computes them from their definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "loom.cpp_b200")
_ls = None


def _framework():
    """The framework's Python binding (a directory name with a dot cannot be imported as a package)."""
    global _ls
    if _ls is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import loom_select

        _ls = loom_select
    return _ls


def listed():
    return [
        # One decode step of one sequence: the log-probability an API returns beside the sampled token,
        # with 20 alternatives. Latency.
        {"name": "logprobs decode", "op": "logprobs", "rows": 1, "vocab": 151936, "dtype": "f32", "n_top": 20,
         "temperature": 1.0, "masked": 0.0},
        # A scored prompt or a training batch's forward: every position of 1024, with entropy and 5 alternatives.
        {"name": "logprobs prompt", "op": "logprobs", "rows": 1024, "vocab": 151936, "dtype": "f32", "n_top": 5,
         "temperature": 1.0, "masked": 0.0},
        # A decode batch of the larger vocabulary in bf16, tempered, the most alternatives.
        {"name": "logprobs batch bf16", "op": "logprobs", "rows": 256, "vocab": 262144, "dtype": "bf16", "n_top": 32,
         "temperature": 0.7, "masked": 0.0},
        # A ragged batch of a speech decoder: odd vocabulary, half of the ids masked off, padded positions.
        {"name": "logprobs ragged", "op": "logprobs", "rows": 77, "vocab": 51865, "dtype": "bf16", "n_top": 3,
         "temperature": 1.0, "masked": 0.5},
        # The backward pass of the 1024-position batch: policy-gradient weights and an entropy bonus.
        {"name": "grad prompt", "op": "grad", "rows": 1024, "vocab": 151936, "dtype": "f32", "temperature": 1.0,
         "masked": 0.0, "entropy": True},
        # The backward pass of a small odd batch in bf16, without the entropy term.
        {"name": "grad ragged bf16", "op": "grad", "rows": 77, "vocab": 51865, "dtype": "bf16", "temperature": 0.7,
         "masked": 0.5, "entropy": False},
        # The final norm of one decode step. Latency.
        {"name": "norm decode", "op": "norm", "rows": 1, "dim": 2048, "dtype": "bf16", "residual": True},
        # The final norm of a prefill of 16384 positions, wide hidden state, in f32.
        {"name": "norm prefill", "op": "norm", "rows": 16384, "dim": 4096, "dtype": "f32", "residual": True},
        # An LM-head weight made 8-bit at load time.
        {"name": "quantize weight", "op": "quantize", "rows": 151936, "dim": 2048, "dtype": "bf16"},
        # Hidden states quantised without a norm, odd width.
        {"name": "quantize hidden", "op": "quantize", "rows": 1024, "dim": 1025, "dtype": "f32"},
        # The 8-bit LM head of one decode step: the weight is read once.
        {"name": "lm head decode", "op": "lm_head", "rows": 1, "hidden": 2048, "vocab": 151936, "out": "f32"},
        # The 8-bit LM head over 1024 positions, bf16 logits.
        {"name": "lm head prompt", "op": "lm_head", "rows": 1024, "hidden": 2048, "vocab": 151936, "out": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "grad", "norm", "quantize", "lm_head", "lm_head"])
    if op in ("logprobs", "grad"):
        vocab = _log_uniform(rng, 100, 262144)
        rows = _log_uniform(rng, 1, max(1, min(16384, 1024 * 151936 // vocab)))
        case = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "bf16"]),
                "temperature": rng.choice([1.0, 1.0, 0.7, 1.3]), "masked": rng.choice([0.0, 0.0, 0.5, 0.99])}
        if op == "logprobs":
            case["n_top"] = rng.randint(0, 32)
        else:
            case["entropy"] = rng.random() < 0.5
        return case
    if op == "norm":
        dim = _log_uniform(rng, 64, 16384)
        return {"op": op, "rows": _log_uniform(rng, 1, 16384 * 4096 // dim // 2), "dim": dim,
                "dtype": rng.choice(["f32", "bf16"]), "residual": rng.random() < 0.7}
    if op == "quantize":
        dim = _log_uniform(rng, 64, 16384)
        return {"op": op, "rows": _log_uniform(rng, 1, 151936 * 2048 // dim // 2), "dim": dim,
                "dtype": rng.choice(["f32", "bf16"])}
    hidden = 16 * _log_uniform(rng, 4, 512)
    vocab = _log_uniform(rng, 100, max(101, min(262144, 151936 * 2048 // hidden)))
    return {"op": op, "rows": _log_uniform(rng, 1, 1024), "hidden": hidden, "vocab": vocab,
            "out": rng.choice(["f32", "bf16"])}


_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}


def _logits(case, g):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 3.0
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    if case["masked"]:
        # grammar or language masks: ids switched off with -inf, never the given one
        off = torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"]
        off.scatter_(1, ids.long()[:, None], False)
        x.masked_fill_(off, -math.inf)
        del off
    # half of the given tokens are likely ones (a sampled token, a well predicted prompt token)
    likely = torch.rand(rows, generator=g, device="cuda") < 0.5
    bump = torch.where(likely, 10.0, 0.0)[:, None]
    x.scatter_add_(1, ids.long()[:, None], bump)
    # padded positions carry no token
    if rows > 8:
        pad = torch.rand(rows, generator=g, device="cuda") < 0.05
        ids = torch.where(pad, torch.full_like(ids, -1), ids)
    return x.to(_TORCH[case["dtype"]]), ids


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    st = {"case": case}
    if op in ("logprobs", "grad"):
        x, ids = _logits(case, g)
        st.update(logits=x, ids=ids)
        rows, dev = case["rows"], x.device
        if op == "logprobs":
            n = case["n_top"]
            st.update(logp=torch.empty(rows, device=dev), entropy=torch.empty(rows, device=dev),
                      lse=torch.empty(rows, device=dev), rank=torch.empty(rows, dtype=torch.int32, device=dev),
                      top_ids=torch.empty(rows, n, dtype=torch.int32, device=dev) if n else None,
                      top_logp=torch.empty(rows, n, device=dev) if n else None)
        else:
            st["g_logp"] = torch.randn(rows, generator=g, device=dev)
            st["g_entropy"] = 0.01 * torch.rand(rows, generator=g, device=dev) if case["entropy"] else None
            # what the forward pass has left
            y = x.double() / case["temperature"]
            m = y.max(dim=1, keepdim=True).values
            e = torch.exp(y - m)
            s = e.sum(dim=1)
            a = torch.where(e > 0, e * (y - m), 0.0).sum(dim=1)
            st["lse"] = (m[:, 0] + torch.log(s)).float()
            st["entropy"] = (torch.log(s) - a / s).float()
            st["grad"] = torch.empty_like(x)
        return st
    if op in ("norm", "quantize"):
        rows, dim, dt = case["rows"], case["dim"], _TORCH[case["dtype"]]
        x = torch.randn(rows, dim, generator=g, device="cuda")
        # a few channels are far larger than the rest, as hidden states have them
        if op == "norm":
            x *= torch.where(torch.rand(dim, generator=g, device="cuda") < 0.01, 20.0, 1.0)
            if case["residual"]:
                st["residual"] = (4.0 * torch.randn(rows, dim, generator=g, device="cuda")).to(dt)
                st["sum"] = torch.empty(rows, dim, dtype=dt, device="cuda")
            st["weight"] = 1.0 + 0.1 * torch.randn(dim, generator=g, device="cuda")
        st["x"] = x.to(dt)
        st["q"] = torch.empty(rows, dim, dtype=torch.int8, device="cuda")
        st["scale"] = torch.empty(rows, device="cuda")
        return st
    rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
    st["q"] = torch.randint(-127, 128, (rows, hidden), generator=g, device="cuda", dtype=torch.int8)
    st["w"] = torch.randint(-127, 128, (vocab, hidden), generator=g, device="cuda", dtype=torch.int8)
    st["scale"] = 0.01 + 0.02 * torch.rand(rows, generator=g, device="cuda")
    st["w_scale"] = (0.5 + torch.rand(vocab, generator=g, device="cuda")) / (127.0 * math.sqrt(hidden))
    st["out"] = torch.empty(rows, vocab, dtype=_TORCH[case["out"]], device="cuda")
    return st


EPS = 1e-6


def _dequantised(q, scale):
    return q.float() * scale[:, None]


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    ls, case = _framework(), st["case"]
    op = case["op"]
    if op == "logprobs":
        ls.token_logprobs_into(st["logits"], st["ids"], st["logp"], out_entropy=st["entropy"], out_lse=st["lse"],
                               out_rank=st["rank"], out_top_ids=st["top_ids"], out_top_logp=st["top_logp"],
                               temperature=case["temperature"])
        return {k: st[k] for k in ("logp", "entropy", "lse", "rank", "top_ids", "top_logp")}
    if op == "grad":
        ls.token_logprobs_grad_into(st["logits"], st["ids"], st["lse"], st["grad"], grad_logp=st["g_logp"],
                                    grad_entropy=st["g_entropy"], entropy=st["entropy"],
                                    temperature=case["temperature"])
        return st["grad"]
    if op == "norm":
        ls.rms_norm_i8_into(st["x"], st["weight"], st["q"], st["scale"], residual=st.get("residual"),
                            out_sum=st.get("sum"), eps=EPS)
        return {"q": st["q"], "scale": st["scale"], "sum": st.get("sum")}
    if op == "quantize":
        ls.quantize_rows_i8_into(st["x"], st["q"], st["scale"])
        return {"q": st["q"], "scale": st["scale"]}
    ls.lm_head_logits_i8_into(st["q"], st["scale"], st["w"], st["w_scale"], st["out"])
    return st["out"]


def _order_keys(x):
    """One int64 per logit: larger logits first, then lower ids (-0 == +0)."""
    bits = (x.float() + 0.0).view(torch.int32)
    o = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    idx = torch.arange(x.shape[1], device=x.device)
    return o * (1 << 31) - idx


def _quantise_plain(y):
    a = y.abs().amax(dim=1)
    scale = a / 127.0
    inv = torch.where(a > 0, 127.0 / a, 0.0)
    return torch.round(y * inv[:, None]).to(torch.int8), scale


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "logprobs":
        x, ids, T = st["logits"], st["ids"].long(), case["temperature"]
        y = x.float() / T
        m = y.amax(dim=1)
        d = y - m[:, None]
        e = torch.exp(d)
        s = e.sum(dim=1)
        ent = torch.log(s) - torch.where(e > 0, e * d, 0.0).sum(dim=1) / s
        lse = m + torch.log(s)
        at = ids.clamp(min=0)[:, None]
        none = ids < 0
        logp = torch.where(none, 0.0, d.gather(1, at)[:, 0] - torch.log(s))
        xt = x.gather(1, at)
        idx = torch.arange(x.shape[1], device=x.device)
        rank = ((x > xt) | ((x == xt) & (idx < at))).sum(dim=1).int()
        rank = torch.where(none, -1, rank)
        out = {"logp": logp, "entropy": ent, "lse": lse, "rank": rank.int(), "top_ids": None, "top_logp": None}
        if case["n_top"]:
            top = torch.topk(_order_keys(x), case["n_top"], dim=1).indices
            out["top_ids"] = top.int()
            out["top_logp"] = d.gather(1, top) - torch.log(s)[:, None]
        return out
    if op == "grad":
        x, ids, T = st["logits"], st["ids"].long(), case["temperature"]
        ly = x.float() / T - st["lse"][:, None]
        p = torch.exp(ly)
        none = ids < 0
        g = torch.where(none, 0.0, st["g_logp"])
        d = -g[:, None] * p
        if st["g_entropy"] is not None:
            d -= st["g_entropy"][:, None] * torch.where(p > 0, p * (ly + st["entropy"][:, None]), 0.0)
        d.scatter_add_(1, ids.clamp(min=0)[:, None], g[:, None])
        return (d / T).to(x.dtype)
    if op == "norm":
        x = st["x"]
        h = (x.float() + st["residual"].float()).to(x.dtype) if "residual" in st else x
        # 64 bits: values next to a rounding border of the 8-bit output
        ss = h.double().square().sum(dim=1)
        inv = (1.0 / torch.sqrt(ss / x.shape[1] + EPS)).float()
        q, scale = _quantise_plain(h.float() * inv[:, None] * st["weight"])
        return {"q": q, "scale": scale, "sum": h if "residual" in st else None}
    if op == "quantize":
        q, scale = _quantise_plain(st["x"].float())
        return {"q": q, "scale": scale}
    acc = torch.matmul(st["q"].float(), st["w"].float().t())
    return (acc * st["scale"][:, None] * st["w_scale"]).to(st["out"].dtype)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("logprobs", "grad"):
        lp = torch.log_softmax(st["logits"].double() / case["temperature"], dim=1)
        ids = st["ids"].long()
        has = ids >= 0
        p = lp.exp()
        ent = -(p * lp).nan_to_num(nan=0.0).sum(dim=1)
        if op == "logprobs":
            picked = lp[torch.arange(len(ids), device=ids.device), ids.clamp(min=0)]
            logp = torch.where(has, picked, torch.zeros_like(picked))
            lse = torch.logsumexp(st["logits"].double() / case["temperature"], dim=1)
            n = case["n_top"]
            return {"logp": logp, "entropy": ent, "lse": lse, "rank": None, "top_ids": None,
                    "top_logp": lp.topk(n, dim=1).values if n else None}
        g = torch.where(has, st["g_logp"].double(), 0.0)
        grad = -g[:, None] * p
        grad[torch.arange(len(ids), device=ids.device), ids.clamp(min=0)] += g
        if st["g_entropy"] is not None:
            grad -= st["g_entropy"].double()[:, None] * (p * (lp + ent[:, None])).nan_to_num(nan=0.0)
        return grad / case["temperature"]
    if op == "norm":
        h = st["x"].double()
        if "residual" in st:
            h = (h + st["residual"].double()).to(st["x"].dtype).double()
        y = h / torch.sqrt(h.pow(2).mean(dim=1, keepdim=True) + EPS) * st["weight"].double()
        # which side of a rounding border a value falls on is the definition's own f32 arithmetic: no 64-bit q
        return {"q": None, "scale": y.abs().amax(dim=1) / 127.0, "sum": h if "residual" in st else None}
    if op == "quantize":
        return {"q": None, "scale": st["x"].double().abs().amax(dim=1) / 127.0}
    acc = torch.mm(st["q"].double(), st["w"].double().t())
    acc.mul_(st["scale"].double()[:, None]).mul_(st["w_scale"].double())
    return acc


def work(case):
    op = case["op"]
    if op in ("logprobs", "grad"):
        rows, vocab = case["rows"], case["vocab"]
        logits = rows * vocab * (4 if case["dtype"] == "f32" else 2)
        if op == "logprobs":
            return {"bytes": logits + rows * (4 + 16 + 8 * case["n_top"]), "flops": 5 * rows * vocab}
        return {"bytes": 2 * logits + rows * (4 * 3 + (8 if case["entropy"] else 0)),
                "flops": (6 if case["entropy"] else 4) * rows * vocab}
    if op in ("norm", "quantize"):
        rows, dim = case["rows"], case["dim"]
        n, esz = rows * dim, 4 if case["dtype"] == "f32" else 2
        if op == "quantize":
            return {"bytes": n * (esz + 1) + 4 * rows, "flops": 3 * n}
        return {"bytes": n * (esz * (3 if case["residual"] else 1) + 1) + 4 * rows + 4 * dim, "flops": 8 * n}
    rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
    return {"bytes": (rows + vocab) * (hidden + 4) + rows * vocab * (4 if case["out"] == "f32" else 2),
            "flops": 2 * rows * hidden * vocab}
