"""The status of calls without a workspace of their own: lm_head_logits_i8's words, and the default workspace."""
import threading

import pytest
import torch

import loom_select as ls

pytestmark = pytest.mark.gpu


def _operands(rows=40, hidden=512, vocab=60000):
    g = torch.Generator(device="cuda").manual_seed(9)
    q = torch.randint(-128, 128, (rows, hidden), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (vocab, hidden), generator=g, device="cuda", dtype=torch.int8)
    qs, ws = torch.rand(rows, generator=g, device="cuda") + 0.01, torch.rand(vocab, generator=g, device="cuda") + 0.01
    return (q, qs, w, ws), (q.double() @ w.double().t()).float() * qs[:, None] * ws


def _hook(ws):
    """The next calls with this workspace leave a slice out and give up their waits after 50 us (nothing faults)."""
    ls.check(ls.lib().loom_select_test_wait_fault(ls._ptr(ws.buf), 50_000, 2, ls._stream_handle()), "hook")


def test_wait_that_gives_up_without_a_workspace():
    args, want = _operands()
    ls.lm_head_logits_i8(*args)
    assert ls.read_status() == ls.OK
    _hook(ls._STATUS_WS[torch.cuda.current_device()])
    ls.lm_head_logits_i8(*args)
    assert ls.read_status() == ls.ETIMEOUT and ls.read_status() == ls.OK
    assert torch.equal(ls.lm_head_logits_i8(*args), want) and ls.read_status() == ls.OK


def test_wait_that_gives_up_in_a_graph():
    args, want = _operands()
    ls.lm_head_logits_i8(*args)
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        ls.lm_head_logits_i8_into(*args, out)
    _hook(ls._STATUS_WS[torch.cuda.current_device()])
    graph.replay()
    assert ls.read_status() == ls.ETIMEOUT
    graph.replay()
    assert ls.read_status() == ls.OK and torch.equal(out, want)


def test_call_captured_before_any_other(monkeypatch):
    """Its own status word is not memory that the graph gives to another tensor, and is read like the device's."""
    args, want = _operands()
    monkeypatch.setattr(ls, "_STATUS_WS", {})
    monkeypatch.setattr(ls, "_CAPTURED_WS", {})
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        ls.lm_head_logits_i8_into(*args, out)
        later = [torch.full((128,), 7, dtype=torch.int32, device="cuda") for _ in range(8)]
    (ws,) = ls._CAPTURED_WS[torch.cuda.current_device()]
    graph.replay()
    assert ls.read_status() == ls.OK and torch.equal(out, want)
    assert not (ws.buf.view(torch.int32) == 7).any() and all((t == 7).all() for t in later)
    ws.buf.view(torch.int32)[0] = ls.ETIMEOUT  # (a kernel's own record; the hook's header is zeroed with every replay)
    assert ls.read_status() == ls.ETIMEOUT
    graph.replay()
    assert ls.read_status() == ls.OK and torch.equal(out, want)


def test_first_calls_of_several_host_threads_share_one_word(monkeypatch):
    monkeypatch.setattr(ls, "_STATUS_WS", {})
    torch.cuda.synchronize()
    n, got = 8, []
    start = threading.Barrier(n)

    def first():
        start.wait()
        got.append(ls._status_buffer(None))

    threads = [threading.Thread(target=first) for _ in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len({b.data_ptr() for b in got}) == 1 and got[0] is ls._STATUS_WS[torch.cuda.current_device()].buf


def test_default_workspace_is_read_too():
    """A history id outside the vocabulary, recorded by a call with the default workspace."""
    logits, u = torch.randn(3, 1000, device="cuda"), torch.rand(3, device="cuda")
    history = torch.tensor([[1], [1000], [2]], dtype=torch.int32, device="cuda")
    ls.read_status()
    ls.sample_rows(logits, u, 1.0, repetition_penalty=1.2, top_k=5, history=history)
    assert ls.read_status() == ls.EHISTORY and ls.read_status() == ls.OK
