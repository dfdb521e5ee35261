"""Python mirror of loom.cpp's logits->token selection, running on the B200 kernels.

This module binds the C-ABI of include/loom_select.h (libloom_select.so, built in place by
build.py next to this file) with ctypes, and offers the selection calls of loom.cpp under their
loom.cpp names on CUDA tensors:

    argmax_row(logits, row=-1)               loom.argmax_row(module, row)     src/core/lua_bridge.cpp:729-743
    argmax_row_range(logits, row, lo, hi)    loom.argmax_row_range(...)       src/core/lua_bridge.cpp:779-797
    argmax_rows(logits)                      loom.argmax_rows(module)         src/core/lua_bridge.cpp:808-822
    ctc_greedy_decode(logits, blank_id)      loom::ctc_greedy_decode          src/core/ctc_decode.cpp:7-31
    sample_rows(logits, ...)                 the sampling chain (no loom.cpp counterpart)
    shard_partial / shard_merge              the vocabulary-sharded chain (no loom.cpp counterpart)
    token_logprobs / token_logprobs_grad     log-probabilities of given tokens, and their gradient (none)
    rms_norm_i8, quantize_rows_i8, lm_head_logits_i8
                                             the final norm and the LM head in 8-bit integers (none)

Errors raise SelectError, as loom.cpp raises loom::Error (include/loom/loom_errors.h:10) and its
Lua bindings turn that into a Lua error (lua_bridge.cpp:26-32). The library must be present: there
is no fallback of any kind, and importing this module on a machine without it fails.

torch is used for device memory, streams and host<->device copies only.
"""
import collections
import contextlib
import ctypes
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libloom_select.so")

F32 = 0
BF16 = 1
MAX_TOP_K = 1024
MAX_WINDOWS = 8
MAX_TOP_LOGPROBS = 32

OK = 0
EINVAL = 1
EDTYPE = 2
EWINDOW = 3
EWORKSPACE = 4
ECUDA = 5
ETIMEOUT = 6
EHISTORY = 7
EPARAM = 8
ESHAPE = 9

# Every entry point include/loom_select.h declares.
EXPORTS = (
    "loom_select_strerror",
    "loom_select_abi_version",
    "loom_argmax_workspace_size",
    "loom_sample_workspace_size",
    "loom_ctc_workspace_size",
    "loom_select_workspace_init",
    "loom_select_read_status",
    "loom_select_test_wait_fault",
    "loom_argmax_rows",
    "loom_argmax_windows_workspace_size",
    "loom_argmax_windows",
    "loom_sample_rows",
    "loom_sample_rows_noalloc",
    "loom_shard_record_bytes",
    "loom_sample_shard_partial",
    "loom_sample_shard_merge",
    "loom_ctc_greedy",
    "loom_lm_head_workspace_size",
    "loom_lm_head_argmax",
    "loom_token_logprobs",
    "loom_token_logprobs_grad",
    "loom_rms_norm_i8",
    "loom_quantize_rows_i8",
    "loom_lm_head_logits_i8_workspace_size",
    "loom_lm_head_logits_i8",
)


class SampleParams(ctypes.Structure):
    _fields_ = [
        ("temperature", ctypes.c_float),
        ("repetition_penalty", ctypes.c_float),
        ("top_k", ctypes.c_int32),
        ("top_p", ctypes.c_float),
    ]


class SelectError(RuntimeError):
    def __init__(self, status, what=""):
        self.status = status
        msg = _lib().loom_select_strerror(status).decode()
        super().__init__(f"{what}: {msg} (status {status})" if what else f"{msg} (status {status})")


_LIB = None


def _lib():
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python {os.path.join(_HERE, 'build.py')}`")
        lib = ctypes.CDLL(LIB_PATH)
        vp, i32, i64, sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t
        f32 = ctypes.c_float
        sig = {
            "loom_select_strerror": (ctypes.c_char_p, [ctypes.c_int]),
            "loom_select_abi_version": (ctypes.c_int, []),
            "loom_argmax_workspace_size": (sz, [i64, i64]),
            "loom_sample_workspace_size": (sz, [i64, i64, i32]),
            "loom_ctc_workspace_size": (sz, [i64, i64]),
            "loom_select_workspace_init": (ctypes.c_int, [vp, sz, vp]),
            "loom_select_read_status": (ctypes.c_int, [vp, vp]),
            "loom_select_test_wait_fault": (ctypes.c_int, [vp, i64, i32, vp]),
            "loom_argmax_rows": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, i64, i64, vp, vp, sz, vp]),
            "loom_argmax_windows_workspace_size": (sz, [i64, i32]),
            "loom_argmax_windows": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, vp, vp, i32, vp, vp, sz, vp]),
            "loom_sample_rows": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, vp, i32, vp,
                                                ctypes.POINTER(SampleParams), vp, vp, vp, vp, vp, sz, vp]),
            "loom_sample_rows_noalloc": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, vp, i32, vp,
                                                        ctypes.POINTER(SampleParams), vp, vp, vp, vp, vp, vp]),
            "loom_shard_record_bytes": (sz, [i32]),
            "loom_sample_shard_partial": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, i64, i64, vp, i32,
                                                         ctypes.POINTER(SampleParams), vp, vp, sz, vp]),
            "loom_sample_shard_merge": (ctypes.c_int, [vp, i32, i64, vp, ctypes.POINTER(SampleParams),
                                                       vp, vp, vp, vp, vp]),
            "loom_ctc_greedy": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, i32, vp, vp, vp, vp, vp, vp, sz, vp]),
            "loom_lm_head_workspace_size": (sz, [i64, i64]),
            "loom_lm_head_argmax": (ctypes.c_int, [vp, vp, i64, i64, i64, vp, vp, vp, vp, sz, vp]),
            "loom_token_logprobs": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, vp, f32, i32, vp, vp, vp, vp, vp,
                                                   vp, vp]),
            "loom_token_logprobs_grad": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, vp, f32, vp, vp, vp, vp, vp,
                                                        i64, vp]),
            "loom_rms_norm_i8": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, vp, i64, vp, ctypes.c_int,
                                                ctypes.c_double, vp, vp, vp, i64, vp]),
            "loom_quantize_rows_i8": (ctypes.c_int, [vp, ctypes.c_int, i64, i64, i64, vp, vp, vp]),
            "loom_lm_head_logits_i8_workspace_size": (sz, [i64, i64]),
            "loom_lm_head_logits_i8": (ctypes.c_int, [vp, vp, vp, vp, i64, i64, i64, vp, ctypes.c_int, i64, vp, sz,
                                                      vp]),
        }
        for name, (res, args) in sig.items():
            f = getattr(lib, name)
            f.restype = res
            f.argtypes = args
        _LIB = lib
    return _LIB


def lib():
    """The loaded libloom_select.so (ctypes.CDLL)."""
    return _lib()


def check(status, what=""):
    if status != OK:
        raise SelectError(status, what)


# ----------------------------------------------------------------------------------------------
# torch plumbing

def _torch():
    import torch
    return torch


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream_handle(stream=None):
    torch = _torch()
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _dtype_code(t):
    torch = _torch()
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    raise SelectError(EDTYPE, f"logits dtype {t.dtype}")


def _rows_view(logits):
    """(rows, n_vocab, row_stride) of a 1-D or 2-D CUDA tensor with unit column stride."""
    if logits.dim() == 1:
        return 1, logits.shape[0], logits.shape[0]
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise SelectError(EINVAL, "logits must be [rows, n_vocab] with contiguous rows")
    # (one row's stride may be anything)
    return logits.shape[0], logits.shape[1], logits.shape[1] if logits.shape[0] == 1 else logits.stride(0)


class Workspace:
    """A caller-owned workspace (a CUDA uint8 tensor), zeroed once, grown on demand."""

    def __init__(self, device=None):
        self.device = device
        self.buf = None

    def get(self, nbytes, stream=None):
        torch = _torch()
        nbytes = max(int(nbytes), 256)
        if self.buf is None or self.buf.numel() < nbytes:
            dev = self.device if self.device is not None else torch.device("cuda", torch.cuda.current_device())
            self.buf = torch.empty(nbytes + 256, dtype=torch.uint8, device=dev)
            check(_lib().loom_select_workspace_init(_ptr(self.buf), self.buf.numel(), _stream_handle(stream)),
                  "loom_select_workspace_init")
        return self.buf

    def read_status(self, stream=None):
        if self.buf is None:
            return OK
        return _lib().loom_select_read_status(_ptr(self.buf), _stream_handle(stream))


_DEFAULT_WS = {}


def default_workspace():
    torch = _torch()
    dev = torch.cuda.current_device()
    if dev not in _DEFAULT_WS:
        _DEFAULT_WS[dev] = Workspace(torch.device("cuda", dev))
    return _DEFAULT_WS[dev]


# ----------------------------------------------------------------------------------------------
# greedy argmax

def argmax_rows_into(logits, out, lo=0, hi=-1, workspace=None, stream=None):
    """One absolute id per row over [lo, hi) into the int32 CUDA tensor `out` (asynchronous)."""
    rows, n_vocab, stride = _rows_view(logits)
    ws = workspace or default_workspace()
    need = _lib().loom_argmax_workspace_size(rows, n_vocab)
    buf = ws.get(need, stream)
    check(_lib().loom_argmax_rows(_ptr(logits), _dtype_code(logits), rows, n_vocab, stride, lo, hi, _ptr(out),
                                  _ptr(buf), buf.numel(), _stream_handle(stream)), "loom_argmax_rows")
    return out


def argmax_rows(logits, lo=0, hi=-1, workspace=None, stream=None):
    """loom.argmax_rows: one id per row, as a list of floats like the Lua binding returns."""
    torch = _torch()
    rows, _, _ = _rows_view(logits)
    out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    argmax_rows_into(logits, out, lo, hi, workspace, stream)
    return [float(v) for v in out.cpu().tolist()]


def argmax_row_range(logits, row, lo, hi, workspace=None, stream=None):
    """loom.argmax_row_range / argmax_tensor_row (lua_bridge.cpp:302-330): row < 0 means the last row,
    hi < 0 means n_vocab, the id is absolute; an empty or out-of-range window or row raises."""
    torch = _torch()
    rows, n_vocab, _ = _rows_view(logits)
    r = rows - 1 if row < 0 else row
    if n_vocab <= 0 or r < 0 or r >= rows:
        raise SelectError(EWINDOW, f"row {row} out of range for an output with {rows} row(s) of width {n_vocab}")
    view = logits if logits.dim() == 1 else logits[r:r + 1]
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    argmax_rows_into(view, out, lo, hi, workspace, stream)
    return float(out.item())


def argmax_windows_into(logits, windows, out, workspace=None, stream=None):
    """Every row's absolute argmax over each [lo, hi) of `windows` (a list of (lo, hi), hi < 0 meaning
    n_vocab) into the int32 CUDA tensor `out` of shape [rows, len(windows)], in one launch."""
    rows, n_vocab, stride = _rows_view(logits)
    n = len(windows)
    lo = (ctypes.c_int64 * max(n, 1))(*[int(w[0]) for w in windows])
    hi = (ctypes.c_int64 * max(n, 1))(*[int(w[1]) for w in windows])
    ws = workspace or default_workspace()
    buf = ws.get(_lib().loom_argmax_windows_workspace_size(rows, max(n, 1)), stream)
    check(_lib().loom_argmax_windows(_ptr(logits), _dtype_code(logits), rows, n_vocab, stride, lo, hi, n, _ptr(out),
                                     _ptr(buf), buf.numel(), _stream_handle(stream)), "loom_argmax_windows")
    return out


def argmax_windows(logits, windows, workspace=None, stream=None):
    """loom.argmax_row_range over several windows of every row at once: an int32 CUDA tensor
    [rows, len(windows)] of absolute ids (lua_bridge.cpp:779-797, batched)."""
    torch = _torch()
    rows, _, _ = _rows_view(logits)
    out = torch.empty(rows, len(windows), dtype=torch.int32, device=logits.device)
    return argmax_windows_into(logits, windows, out, workspace, stream)


def argmax_row(logits, row=-1, workspace=None, stream=None):
    """loom.argmax_row (module form) / Generator::argmax on one row."""
    return argmax_row_range(logits, row, 0, -1, workspace, stream)


# ----------------------------------------------------------------------------------------------
# sampling chain

def sample_rows_into(logits, u, out_ids, out_prob, temperature, repetition_penalty=1.0, top_k=40, top_p=1.0,
                     history=None, out_logp=None, out_topk=None, workspace=None, stream=None):
    """The fused sampling chain on device tensors (asynchronous). history: int32 [rows, H] or None."""
    rows, n_vocab, stride = _rows_view(logits)
    hl = 0 if history is None else int(history.shape[-1])
    p = SampleParams(temperature, repetition_penalty, top_k, top_p)
    ws = workspace or default_workspace()
    buf = ws.get(_lib().loom_sample_workspace_size(rows, n_vocab, top_k), stream)
    check(_lib().loom_sample_rows(_ptr(logits), _dtype_code(logits), rows, n_vocab, stride, _ptr(history), hl,
                                  _ptr(u), ctypes.byref(p), _ptr(out_ids), _ptr(out_prob), _ptr(out_logp),
                                  _ptr(out_topk), _ptr(buf), buf.numel(), _stream_handle(stream)),
          "loom_sample_rows")


def sample_rows_noalloc_into(logits, u, out_ids, out_prob, temperature, repetition_penalty=1.0, top_k=40,
                             top_p=1.0, history=None, out_logp=None, out_topk=None, out_status=None, stream=None):
    """sample_rows_into without a workspace: the library's own fixed scratch (top_k <= 64; calls must
    not overlap on the GPU). out_status: an int32 device tensor of one element, or None."""
    rows, n_vocab, stride = _rows_view(logits)
    hl = 0 if history is None else int(history.shape[-1])
    p = SampleParams(temperature, repetition_penalty, top_k, top_p)
    check(_lib().loom_sample_rows_noalloc(_ptr(logits), _dtype_code(logits), rows, n_vocab, stride, _ptr(history),
                                          hl, _ptr(u), ctypes.byref(p), _ptr(out_ids), _ptr(out_prob),
                                          _ptr(out_logp), _ptr(out_topk), _ptr(out_status),
                                          _stream_handle(stream)),
          "loom_sample_rows_noalloc")


def sample_rows(logits, u, temperature, repetition_penalty=1.0, top_k=40, top_p=1.0, history=None,
                want_logp=False, want_topk=False, workspace=None, stream=None):
    """Returns (ids int32, probs f32[, logp f32][, topk int32 [rows, k]]) as CUDA tensors."""
    torch = _torch()
    rows, _, _ = _rows_view(logits)
    dev = logits.device
    ids = torch.empty(rows, dtype=torch.int32, device=dev)
    prob = torch.empty(rows, dtype=torch.float32, device=dev)
    logp = torch.empty(rows, dtype=torch.float32, device=dev) if want_logp else None
    topk = torch.empty(rows, top_k, dtype=torch.int32, device=dev) if want_topk else None
    sample_rows_into(logits, u, ids, prob, temperature, repetition_penalty, top_k, top_p, history, logp, topk,
                     workspace, stream)
    out = [ids, prob]
    if want_logp:
        out.append(logp)
    if want_topk:
        out.append(topk)
    return tuple(out)


def shard_record_bytes(top_k):
    return int(_lib().loom_shard_record_bytes(top_k))


def shard_partial_into(logits, out_records, vocab_offset, vocab_total, temperature, repetition_penalty=1.0,
                       top_k=64, top_p=1.0, history=None, workspace=None, stream=None):
    """This GPU's shard [rows, shard_vocab] -> rows records of shard_record_bytes(top_k) (uint8 tensor)."""
    rows, n_vocab, stride = _rows_view(logits)
    hl = 0 if history is None else int(history.shape[-1])
    p = SampleParams(temperature, repetition_penalty, top_k, top_p)
    ws = workspace or default_workspace()
    buf = ws.get(_lib().loom_sample_workspace_size(rows, n_vocab, top_k), stream)
    check(_lib().loom_sample_shard_partial(_ptr(logits), _dtype_code(logits), rows, n_vocab, stride, vocab_offset,
                                           vocab_total, _ptr(history), hl, ctypes.byref(p), _ptr(out_records),
                                           _ptr(buf), buf.numel(), _stream_handle(stream)),
          "loom_sample_shard_partial")


def shard_merge_into(records, n_shards, rows, u, out_ids, out_prob, temperature, top_k=64, top_p=1.0,
                     out_logp=None, out_topk=None, stream=None):
    """Gathered records [n_shards][rows] -> the same outputs as sample_rows over the whole vocabulary."""
    p = SampleParams(temperature, 1.0, top_k, top_p)
    check(_lib().loom_sample_shard_merge(_ptr(records), n_shards, rows, _ptr(u), ctypes.byref(p), _ptr(out_ids),
                                         _ptr(out_prob), _ptr(out_logp), _ptr(out_topk), _stream_handle(stream)),
          "loom_sample_shard_merge")


# ----------------------------------------------------------------------------------------------
# CTC

def ctc_greedy_into(logits, blank, out_ids, out_frames, out_len, out_frame_ids=None, out_frame_logp=None,
                    workspace=None, stream=None):
    """logits: [n_utt, n_frames, n_classes] (or [n_frames, n_classes]) contiguous CUDA tensor."""
    if logits.dim() == 2:
        n_utt, (n_frames, n_classes) = 1, logits.shape
    else:
        n_utt, n_frames, n_classes = logits.shape
    if not logits.is_contiguous():
        raise SelectError(EINVAL, "CTC logits must be contiguous")
    ws = workspace or default_workspace()
    buf = ws.get(_lib().loom_ctc_workspace_size(n_utt, n_frames), stream)
    check(_lib().loom_ctc_greedy(_ptr(logits), _dtype_code(logits), n_utt, n_frames, n_classes, blank, _ptr(out_ids),
                                 _ptr(out_frames), _ptr(out_len), _ptr(out_frame_ids), _ptr(out_frame_logp),
                                 _ptr(buf), buf.numel(), _stream_handle(stream)), "loom_ctc_greedy")


def ctc_greedy(logits, blank, want_frame_ids=False, want_frame_logp=False, workspace=None, stream=None):
    """Returns (ids [n_utt, n_frames], frames [n_utt, n_frames], lens [n_utt][, frame_ids][, frame_logp])."""
    torch = _torch()
    n_utt, n_frames = (1, logits.shape[0]) if logits.dim() == 2 else (logits.shape[0], logits.shape[1])
    dev = logits.device
    ids = torch.empty(n_utt, n_frames, dtype=torch.int32, device=dev)
    frames = torch.empty(n_utt, n_frames, dtype=torch.int32, device=dev)
    lens = torch.empty(n_utt, dtype=torch.int32, device=dev)
    fid = torch.empty(n_utt, n_frames, dtype=torch.int32, device=dev) if want_frame_ids else None
    flp = torch.empty(n_utt, n_frames, dtype=torch.float32, device=dev) if want_frame_logp else None
    ctc_greedy_into(logits, blank, ids, frames, lens, fid, flp, workspace, stream)
    out = [ids, frames, lens]
    if want_frame_ids:
        out.append(fid)
    if want_frame_logp:
        out.append(flp)
    return tuple(out)


def ctc_greedy_decode(logits, blank_id, workspace=None, stream=None):
    """loom::ctc_greedy_decode(logits, n_frames, n_classes, blank_id) on a [n_frames, n_classes] CUDA
    tensor: the collapsed token ids as a list."""
    ids, _, lens = ctc_greedy(logits, blank_id, workspace=workspace, stream=stream)
    n = int(lens[0].item())
    return ids[0, :n].cpu().tolist()


# ----------------------------------------------------------------------------------------------
# greedy selection fused into the LM-head GEMM

def lm_head_argmax_into(hidden, weight, out_ids, out_logit=None, out_lse=None, workspace=None, stream=None):
    """Greedy ids of logits = hidden @ weight.T without materialising the logits (asynchronous).

    hidden [rows, hidden_dim] and weight [n_vocab, hidden_dim] are contiguous bf16 CUDA tensors (the
    weight in ggml's lm_head layout); out_ids int32 [rows]; out_logit / out_lse f32 [rows] or None."""
    torch = _torch()
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise SelectError(EDTYPE, "lm_head_argmax takes bf16 hidden states and weight")
    if hidden.dim() == 1:
        hidden = hidden.view(1, -1)
    if hidden.dim() != 2 or weight.dim() != 2 or not hidden.is_contiguous() or not weight.is_contiguous():
        raise SelectError(EINVAL, "hidden [rows, hidden_dim] and weight [n_vocab, hidden_dim] must be contiguous")
    if hidden.shape[1] != weight.shape[1]:
        raise SelectError(EINVAL, "hidden and weight disagree on hidden_dim")
    rows, hdim = hidden.shape
    n_vocab = weight.shape[0]
    ws = workspace or default_workspace()
    need = _lib().loom_lm_head_workspace_size(rows, n_vocab)
    buf = ws.get(need, stream)
    check(_lib().loom_lm_head_argmax(_ptr(hidden), _ptr(weight), rows, hdim, n_vocab, _ptr(out_ids),
                                     _ptr(out_logit), _ptr(out_lse), _ptr(buf), buf.numel(), _stream_handle(stream)),
          "loom_lm_head_argmax")
    return out_ids


def lm_head_argmax(hidden, weight, want_logit=True, want_lse=True, workspace=None, stream=None):
    """(ids, logit or None, log-sum-exp or None) per row of hidden @ weight.T."""
    torch = _torch()
    rows = 1 if hidden.dim() == 1 else hidden.shape[0]
    dev = hidden.device
    ids = torch.empty(rows, dtype=torch.int32, device=dev)
    logit = torch.empty(rows, dtype=torch.float32, device=dev) if want_logit else None
    lse = torch.empty(rows, dtype=torch.float32, device=dev) if want_lse else None
    lm_head_argmax_into(hidden, weight, ids, logit, lse, workspace, stream)
    return ids, logit, lse


# ----------------------------------------------------------------------------------------------
# log-probabilities of given tokens

def _check_tensor(t, name, dtype, shape, dev):
    """A contiguous tensor of this type and shape (a tuple) on CUDA device number `dev`, or None."""
    if t is None or (t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous()):
        return
    if t.dtype != dtype:
        raise SelectError(EDTYPE, f"{name} is {t.dtype}, expected {dtype}")
    if t.get_device() != dev:
        raise SelectError(EINVAL, f"{name} is on {t.device}, expected cuda:{dev}")
    raise SelectError(EINVAL, f"{name} must be contiguous, of shape {tuple(shape)}")


def _current_device(t, name):
    """The number of the current CUDA device, where the kernels run: a tensor elsewhere is an error, not a fault."""
    dev = t.get_device()
    if dev < 0 or dev != _torch().cuda.current_device():
        raise SelectError(EINVAL, f"{name} is on {t.device}, not on the current CUDA device")
    return dev


def _addr(t):
    """A tensor's address as ctypes takes it for a void pointer."""
    return None if t is None else t.data_ptr()


def _raw_stream(stream, dev):
    """The handle of `stream`, or of the device's current one (without making a Stream object for it)."""
    if stream is None:
        return _torch()._C._cuda_getCurrentRawStream(dev)
    if stream.device_index != dev:
        raise SelectError(EINVAL, f"the stream is of device {stream.device_index}, the tensors of {dev}")
    return stream.cuda_stream


def _on(stream):
    """New tensors belong to the stream that fills them."""
    return contextlib.nullcontext() if stream is None else _torch().cuda.stream(stream)


def token_logprobs_into(logits, ids, out_logp=None, out_entropy=None, out_lse=None, out_rank=None, out_top_ids=None,
                        out_top_logp=None, temperature=1.0, stream=None):
    """Log-probabilities of ids [rows] (int32; negative: no token) under logits [rows, n_vocab] (asynchronous).

    out_logp, out_entropy, out_lse f32 [rows], out_rank int32 [rows], out_top_ids int32 and out_top_logp f32
    [rows, n] (n alternatives, at most MAX_TOP_LOGPROBS), each of them or None. See loom_token_logprobs."""
    torch = _torch()
    rows, n_vocab, stride = _rows_view(logits)
    code, dev = _dtype_code(logits), _current_device(logits, "logits")
    n_top = 0
    for t in (out_top_ids, out_top_logp):
        if t is not None:
            if t.dim() == 0:
                raise SelectError(EINVAL, "alternatives must be [rows, n]")
            n_top = t.shape[-1]
    top = (rows, n_top) if logits.dim() == 2 else (n_top,)
    per_row = (rows,)
    for t, name, dtype, shape in ((ids, "ids", torch.int32, per_row), (out_logp, "out_logp", torch.float32, per_row),
                                  (out_entropy, "out_entropy", torch.float32, per_row),
                                  (out_lse, "out_lse", torch.float32, per_row),
                                  (out_rank, "out_rank", torch.int32, per_row),
                                  (out_top_ids, "out_top_ids", torch.int32, top),
                                  (out_top_logp, "out_top_logp", torch.float32, top)):
        _check_tensor(t, name, dtype, shape, dev)
    check(_lib().loom_token_logprobs(logits.data_ptr(), code, rows, n_vocab, stride, _addr(ids), temperature, n_top,
                                     _addr(out_logp), _addr(out_entropy), _addr(out_lse), _addr(out_rank),
                                     _addr(out_top_ids), _addr(out_top_logp), _raw_stream(stream, dev)),
          "loom_token_logprobs")


TokenLogprobs = collections.namedtuple("TokenLogprobs", "logp entropy lse rank top_ids top_logp")


def token_logprobs(logits, ids=None, temperature=1.0, n_top=0, want_entropy=True, want_rank=False, stream=None):
    """TokenLogprobs(logp, entropy, lse, rank, top_ids, top_logp) as CUDA tensors, None for what is not asked for
    (logp and rank without ids, alternatives with n_top == 0)."""
    torch = _torch()
    rows, _, _ = _rows_view(logits)
    dev = logits.device
    if want_rank and ids is None:
        raise SelectError(EINVAL, "a rank needs ids")
    if n_top < 0:
        raise SelectError(EPARAM, f"{n_top} alternatives")
    with _on(stream):
        f32 = [torch.empty(rows, dtype=torch.float32, device=dev) if w else None
               for w in (ids is not None, want_entropy, True)]
        rank = torch.empty(rows, dtype=torch.int32, device=dev) if want_rank else None
        top = (rows, n_top) if logits.dim() == 2 else (n_top,)
        top_ids = torch.empty(top, dtype=torch.int32, device=dev) if n_top else None
        top_logp = torch.empty(top, dtype=torch.float32, device=dev) if n_top else None
    token_logprobs_into(logits, ids, f32[0], f32[1], f32[2], rank, top_ids, top_logp, temperature, stream)
    return TokenLogprobs(f32[0], f32[1], f32[2], rank, top_ids, top_logp)


def token_logprobs_grad_into(logits, ids, lse, out_grad, grad_logp=None, grad_entropy=None, entropy=None,
                             temperature=1.0, stream=None):
    """d/dlogits of sum(grad_logp * logp + grad_entropy * entropy) into out_grad, of the logits' shape and type
    (rows may be strided; out_grad may be the logits themselves). lse and entropy are the forward call's."""
    torch = _torch()
    rows, n_vocab, stride = _rows_view(logits)
    code, dev = _dtype_code(logits), _current_device(logits, "logits")
    if out_grad.dtype != logits.dtype:
        raise SelectError(EDTYPE, f"out_grad is {out_grad.dtype}, expected {logits.dtype}")
    if out_grad.shape != logits.shape or out_grad.get_device() != dev:
        raise SelectError(EINVAL, "out_grad must have the logits' shape and device")
    _, _, grad_stride = _rows_view(out_grad)
    for t, name, dtype in ((ids, "ids", torch.int32), (lse, "lse", torch.float32), (entropy, "entropy", torch.float32),
                           (grad_logp, "grad_logp", torch.float32), (grad_entropy, "grad_entropy", torch.float32)):
        _check_tensor(t, name, dtype, (rows,), dev)
    check(_lib().loom_token_logprobs_grad(logits.data_ptr(), code, rows, n_vocab, stride, _addr(ids), temperature,
                                          _addr(lse), _addr(entropy), _addr(grad_logp), _addr(grad_entropy),
                                          out_grad.data_ptr(), grad_stride, _raw_stream(stream, dev)),
          "loom_token_logprobs_grad")
    return out_grad


def token_logprobs_grad(logits, ids, lse, grad_logp=None, grad_entropy=None, entropy=None, temperature=1.0,
                        stream=None):
    """token_logprobs_grad_into a new tensor."""
    with _on(stream):
        out = _torch().empty(logits.shape, dtype=logits.dtype, device=logits.device)
    return token_logprobs_grad_into(logits, ids, lse, out, grad_logp, grad_entropy, entropy, temperature, stream)


# ----------------------------------------------------------------------------------------------
# the LM head in 8-bit integers

def _matrix_view(t, name):
    """(rows, dim, row_stride) of a 1-D or 2-D tensor with unit column stride."""
    if t.dim() == 1:
        return 1, t.shape[0], t.shape[0]
    if t.dim() != 2 or t.stride(1) != 1:
        raise SelectError(EINVAL, f"{name} must be [rows, dim] with contiguous rows")
    return t.shape[0], t.shape[1], t.shape[1] if t.shape[0] == 1 else t.stride(0)


def rms_norm_i8_into(x, weight, out_q, out_scale, residual=None, out_sum=None, eps=1e-6, stream=None):
    """RMS norm of x (+ residual) [rows, dim] with weight [dim], as 8-bit integers with a scale per row (asynchronous).

    out_q int8 [rows, dim], out_scale f32 [rows]; residual and out_sum (x + residual, which may be x or residual
    itself) are like x or None. out_q * out_scale stands for the normed rows. See loom_rms_norm_i8."""
    torch = _torch()
    rows, dim, stride = _matrix_view(x, "x")
    code, dev = _dtype_code(x), _current_device(x, "x")
    wcode = _dtype_code(weight)
    _check_tensor(weight, "weight", weight.dtype, (dim,), dev)
    strides = []
    for t, name in ((residual, "residual"), (out_sum, "out_sum")):
        if t is not None:
            if t.dtype != x.dtype:
                raise SelectError(EDTYPE, f"{name} is {t.dtype}, expected {x.dtype}")
            if t.shape != x.shape or t.get_device() != dev:
                raise SelectError(EINVAL, f"{name} must have x's shape and device")
        strides.append(0 if t is None else _matrix_view(t, name)[2])
    _check_tensor(out_q, "out_q", torch.int8, x.shape, dev)
    _check_tensor(out_scale, "out_scale", torch.float32, (rows,), dev)
    check(_lib().loom_rms_norm_i8(x.data_ptr(), code, rows, dim, stride, _addr(residual), strides[0], weight.data_ptr(),
                                  wcode, eps, out_q.data_ptr(), out_scale.data_ptr(), _addr(out_sum), strides[1],
                                  _raw_stream(stream, dev)), "loom_rms_norm_i8")
    return out_q, out_scale


def rms_norm_i8(x, weight, residual=None, eps=1e-6, stream=None):
    """(q int8, scale f32, x + residual or None) in new tensors."""
    torch = _torch()
    rows, _, _ = _matrix_view(x, "x")
    with _on(stream):
        q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        scale = torch.empty(rows, dtype=torch.float32, device=x.device)
        total = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rms_norm_i8_into(x, weight, q, scale, residual, total, eps, stream)
    return q, scale, total


def quantize_rows_i8_into(x, out_q, out_scale, stream=None):
    """Rows of x [rows, dim] as 8-bit integers with a scale per row (asynchronous): q * scale stands for x."""
    torch = _torch()
    rows, dim, stride = _matrix_view(x, "x")
    code, dev = _dtype_code(x), _current_device(x, "x")
    _check_tensor(out_q, "out_q", torch.int8, x.shape, dev)
    _check_tensor(out_scale, "out_scale", torch.float32, (rows,), dev)
    check(_lib().loom_quantize_rows_i8(x.data_ptr(), code, rows, dim, stride, out_q.data_ptr(), out_scale.data_ptr(),
                                       _raw_stream(stream, dev)), "loom_quantize_rows_i8")
    return out_q, out_scale


def quantize_rows_i8(x, stream=None):
    """(q int8, scale f32) in new tensors: an LM-head weight [n_vocab, hidden_dim] for lm_head_logits_i8, say."""
    torch = _torch()
    rows, _, _ = _matrix_view(x, "x")
    with _on(stream):
        q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    return quantize_rows_i8_into(x, q, scale, stream)


_STATUS_WS = {}
_STATUS_LOCK = threading.Lock()
_CAPTURED_WS = {}


def _status_buffer(stream):
    """The workspace of a call that needs only the status word: one per device, never replaced, which captured calls
    use too. A call captured before there is one gets one of its own (zeroed by the graph: a node of 2 us each time
    it is replayed). read_status() reads them all, so they stay."""
    torch = _torch()
    with _on(stream):
        dev = torch.cuda.current_device()
        if dev in _STATUS_WS:
            return _STATUS_WS[dev].buf
        ws = Workspace(torch.device("cuda", dev))
        if torch.cuda.is_current_stream_capturing():
            ws.get(256, stream)
            _CAPTURED_WS.setdefault(dev, []).append(ws)
            return ws.buf
        with _STATUS_LOCK:  # (the first of several host threads: the others, and what they capture, use its word)
            if dev not in _STATUS_WS:
                ws.get(256, stream)
                torch.cuda.current_stream().synchronize()  # zeroed before another stream's call reads it
                _STATUS_WS[dev] = ws
            return _STATUS_WS[dev].buf


def read_status(stream=None):
    """The first device-side error (EHISTORY, ETIMEOUT) that calls without a workspace of their own have recorded on the
    current device since this was last asked, or OK. Waits for `stream`: ask on the one that the calls, or the replayed
    graphs, ran on. After ETIMEOUT the outputs of such calls are invalid; the calls that follow are not affected."""
    dev = _torch().cuda.current_device()
    status = OK
    for ws in (_DEFAULT_WS.get(dev), _STATUS_WS.get(dev), *_CAPTURED_WS.get(dev, ())):
        found = OK if ws is None else ws.read_status(stream)
        if found == ETIMEOUT:
            check(_lib().loom_select_workspace_init(_ptr(ws.buf), ws.buf.numel(), _stream_handle(stream)),
                  "loom_select_workspace_init")
        status = status or found
    return status


def lm_head_logits_i8_into(hidden, hidden_scale, weight, weight_scale, out, workspace=None, stream=None):
    """out[r, v] = (hidden[r] . weight[v]) * hidden_scale[r] * weight_scale[v] (asynchronous).

    hidden int8 [rows, hidden_dim] with hidden_scale f32 [rows], weight int8 [n_vocab, hidden_dim] with weight_scale
    f32 [n_vocab], all contiguous; out f32 or bf16 [rows, n_vocab], rows of any stride. See loom_lm_head_logits_i8.
    Without a workspace, read_status() tells whether a wait gave up."""
    torch = _torch()
    if hidden.dim() not in (1, 2) or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise SelectError(EINVAL, "hidden must be [rows, hidden_dim] and weight [n_vocab, hidden_dim]")
    rows = 1 if hidden.dim() == 1 else hidden.shape[0]
    n_vocab, hdim = weight.shape
    dev = _current_device(hidden, "hidden")
    _check_tensor(hidden, "hidden", torch.int8, hidden.shape, dev)
    _check_tensor(hidden_scale, "hidden_scale", torch.float32, (rows,), dev)
    _check_tensor(weight, "weight", torch.int8, weight.shape, dev)
    _check_tensor(weight_scale, "weight_scale", torch.float32, (n_vocab,), dev)
    code = _dtype_code(out)
    if tuple(out.shape) != ((n_vocab,) if hidden.dim() == 1 else (rows, n_vocab)) or out.get_device() != dev:
        raise SelectError(EINVAL, "out must be [rows, n_vocab] on the hidden states' device")
    _, _, stride = _rows_view(out)
    buf = workspace.get(256, stream) if workspace is not None else _status_buffer(stream)
    check(_lib().loom_lm_head_logits_i8(hidden.data_ptr(), hidden_scale.data_ptr(), weight.data_ptr(),
                                        weight_scale.data_ptr(), rows, hdim, n_vocab, out.data_ptr(), code, stride,
                                        buf.data_ptr(), buf.numel(), _raw_stream(stream, dev)),
          "loom_lm_head_logits_i8")
    return out


def lm_head_logits_i8(hidden, hidden_scale, weight, weight_scale, dtype=None, workspace=None, stream=None):
    """lm_head_logits_i8_into a new tensor of `dtype` (f32 by default, or bf16)."""
    torch = _torch()
    if hidden.dim() not in (1, 2) or weight.dim() != 2:
        raise SelectError(EINVAL, "hidden must be [rows, hidden_dim] and weight [n_vocab, hidden_dim]")
    shape = (weight.shape[0],) if hidden.dim() == 1 else (hidden.shape[0], weight.shape[0])
    with _on(stream):
        out = torch.empty(shape, dtype=dtype or torch.float32, device=hidden.device)
    return lm_head_logits_i8_into(hidden, hidden_scale, weight, weight_scale, out, workspace, stream)
