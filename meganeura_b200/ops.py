"""Array-level entry points over the C ABI (numpy for host data, torch for device data).

These are thin argument marshallers: every computation happens in libmgq.
"""
from __future__ import annotations

import contextlib
import functools
from typing import NamedTuple

import numpy as np

from . import _lib
from ._lib import A_BF16, A_F32, FMT_BF16, FMT_F16, FMT_F32, FMT_Q4, FMT_Q8, check, lib


def set_option(name: str, value: int) -> None:
    """Runtime option of the library (mgq_set_option), e.g. "gemv.serial_dispatch"."""
    check(lib.mgq_set_option(name.encode(), int(value)))


def device_status() -> None:
    """Raises MgqError(MGQ_ERR_TIMEOUT) if a bounded device-side wait ran out (mgq_device_status)."""
    check(lib.mgq_device_status())


def packed_bytes(fmt: int, k: int, n: int) -> int:
    return int(lib.mgq_packed_bytes(fmt, k, n))


def quantize(fmt: int, w: np.ndarray) -> np.ndarray:
    """Host quantizer: row-major [K,N] f32 -> packed bytes (quantize_q4_0 / quantize_q8_0)."""
    w = np.ascontiguousarray(w, dtype=np.float32)
    if w.ndim != 2:
        raise ValueError("weights must be 2-D [K, N]")
    k, n = w.shape
    out = np.empty(packed_bytes(fmt, k, n) if k % 32 == 0 else 1, dtype=np.uint8)
    fn = lib.mgq_quantize_q4 if fmt == FMT_Q4 else lib.mgq_quantize_q8
    check(fn(w.ctypes.data, k, n, out.ctypes.data))
    return out


def dequantize(fmt: int, packed: np.ndarray, k: int, n: int) -> np.ndarray:
    packed = np.ascontiguousarray(packed, dtype=np.uint8)
    out = np.empty((k, n), dtype=np.float32)
    fn = lib.mgq_dequantize_q4 if fmt == FMT_Q4 else lib.mgq_dequantize_q8
    check(fn(packed.ctypes.data, k, n, out.ctypes.data))
    return out


def shard_columns(fmt: int, packed: np.ndarray, k: int, n: int, n0: int, n1: int) -> np.ndarray:
    packed = np.ascontiguousarray(packed, dtype=np.uint8)
    out = np.empty(packed_bytes(fmt, k, max(n1 - n0, 0)) or 1, dtype=np.uint8)
    check(lib.mgq_shard_columns(fmt, packed.ctypes.data, k, n, n0, n1, out.ctypes.data))
    return out


def _stream_ptr(stream=None):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def matmul(fmt: int, a, w, k: int, n: int, addend=None, out=None, stream=None, route: str = "auto"):
    """c = a . dequant(w) (+ addend) on torch CUDA tensors.

    a: [m,k] float32 or bfloat16; w: uint8 tensor holding the packed weight; returns float32 [m,n].
    route: "auto" (mgq_matmul), "gemv" (mgq_gemv) or "gemm" (mgq_gemm).
    """
    import torch
    if not (a.is_cuda and w.is_cuda):
        raise ValueError("matmul takes CUDA tensors; the library has no CPU path")
    a2 = a.reshape(-1, k)
    if not a2.is_contiguous():
        a2 = a2.contiguous()
    m = a2.shape[0]
    if out is None:
        out = torch.empty((m, n), dtype=torch.float32, device=a.device)
    a_dtype = A_BF16 if a2.dtype == torch.bfloat16 else A_F32
    if a2.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("activations must be float32 or bfloat16")
    add_p = addend.data_ptr() if addend is not None else None
    sp = _stream_ptr(stream)
    if route == "gemv":
        check(lib.mgq_gemv(fmt, a2.data_ptr(), w.data_ptr(), add_p, out.data_ptr(), m, k, n, sp))
    elif route == "gemm":
        check(lib.mgq_gemm(fmt, a2.data_ptr(), a_dtype, w.data_ptr(), add_p, out.data_ptr(), m, k, n, sp))
    else:
        check(lib.mgq_matmul(fmt, a2.data_ptr(), a_dtype, w.data_ptr(), add_p, out.data_ptr(), m, k, n, sp))
    return out


class Plan:
    """A static list of single-row GEMVs executed by one persistent kernel (mgq_plan_*).

    ops: iterable of (fmt, x, w, addend_or_None, y, k, n, wait_for) with torch CUDA tensors; the
    tensors are kept alive by the plan.  With `links` (one (push_ptr, wait_ptr) pair of device
    addresses or None per op) the plan uses caller-owned gathered vectors (mgq_plan_create_linked):
    `epoch_ptr` / `error_ptr` are the token index and timeout flag in local device memory and
    `final` = (vector address, length) is the gathered vector that must be complete when a launch ends.
    """

    def __init__(self, ops_list, links=None, epoch_ptr=None, error_ptr=None, final=None, keep=None):
        import ctypes
        self._keep = [keep]
        arr = (_lib.PlanOp * len(ops_list))()
        for i, (fmt, x, w, addend, y, k, n, wait_for) in enumerate(ops_list):
            self._keep.append((x, w, addend, y))
            arr[i] = _lib.PlanOp(fmt, x.data_ptr() if x is not None else None, w.data_ptr(),
                                 addend.data_ptr() if addend is not None else None, y.data_ptr(), 1, k, n, wait_for)
        handle = ctypes.c_void_p()
        if links is None:
            check(lib.mgq_plan_create(arr, len(ops_list), ctypes.byref(handle)))
        else:
            larr = (_lib.PlanLink * len(ops_list))()
            for i, (push_ptr, wait_ptr) in enumerate(links):
                larr[i] = _lib.PlanLink(push_ptr, wait_ptr)
            fvec, flen = final if final is not None else (None, 0)
            check(lib.mgq_plan_create_linked(arr, larr, len(ops_list), epoch_ptr, error_ptr, fvec, flen, ctypes.byref(handle)))
        self._h = handle
        self.count = len(ops_list)

    def launch(self, stream=None) -> None:
        check(lib.mgq_plan_launch(self._h, _stream_ptr(stream)))

    def check(self, stream=None) -> None:
        check(lib.mgq_plan_check(self._h, _stream_ptr(stream)))

    def info(self) -> dict:
        import ctypes
        g, t, c, s = ctypes.c_uint32(), ctypes.c_uint32(), ctypes.c_uint32(), ctypes.c_size_t()
        check(lib.mgq_plan_info(self._h, ctypes.byref(g), ctypes.byref(t), ctypes.byref(c), ctypes.byref(s)))
        return {"grid": g.value, "threads": t.value, "ring_slots": c.value, "smem_bytes": s.value}

    def __del__(self):
        if getattr(self, "_h", None) and lib is not None:
            lib.mgq_plan_destroy(self._h)
            self._h = None


def matmul_host(fmt: int, a: np.ndarray, w_dev_ptr: int, k: int, n: int, addend: np.ndarray | None = None) -> np.ndarray:
    """Host activations in, host result out, device-resident weight (mgq_matmul_host)."""
    a = np.ascontiguousarray(a, dtype=np.float32).reshape(-1, k)
    m = a.shape[0]
    out = np.empty((m, n), dtype=np.float32)
    add_p = None
    if addend is not None:
        addend = np.ascontiguousarray(addend, dtype=np.float32)
        add_p = addend.ctypes.data
    check(lib.mgq_matmul_host(fmt, a.ctypes.data, A_F32, w_dev_ptr, add_p, out.ctypes.data, m, k, n))
    return out


# ---------------------------------------------------------------------------------------------- many sequences over one paged cache

NO_SLOT = NO_PAGE = NO_TOKEN = -1           # MGQ_NO_SLOT and its like as they read in an int32 tensor


class PagedStep(NamedTuple):
    """Where a step's rows belong (int32 CUDA tensors): what paged_plan writes, paged_append and paged_attention read."""
    starts: "object"                        # [sequences + 1] first row of each sequence, then the end
    lengths: "object"                       # [sequences] tokens of each sequence, new ones included
    positions: "object"                     # [rows]
    slots: "object"                         # [rows]
    lacking: "object"                       # [1] pages that the pool was short of

    @staticmethod
    def empty(sequences: int, rows: int, device="cuda") -> "PagedStep":
        import torch
        return PagedStep(*(torch.empty(n, dtype=torch.int32, device=device) for n in (sequences + 1, sequences, rows, rows, 1)))


@functools.lru_cache(maxsize=None)
def _formats() -> dict:
    import torch
    return {torch.float32: FMT_F32, torch.float16: FMT_F16, torch.bfloat16: FMT_BF16}


@functools.lru_cache(maxsize=None)
def _attention_workspace(heads: int, kv_heads: int, head_dim: int, max_fresh: int, dtype: int) -> int:
    return int(lib.mgq_paged_attention_workspace(heads, kv_heads, head_dim, max_fresh, dtype))


def _words(name: str, t, device, *shape):
    """Address of a contiguous int32 tensor on `device`; `shape`: its sizes, None for any."""
    import torch
    if t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor on {device}")
    if len(t.shape) != len(shape) or any(want is not None and have != want for have, want in zip(t.shape, shape)):
        raise ValueError(f"{name} has the shape {tuple(t.shape)}, not {shape}")
    return t.data_ptr()


def _floats(name: str, t, device, count: int):
    import torch
    if t.dtype is not torch.float32 or t.device != device or not t.is_contiguous() or t.numel() != count:
        raise ValueError(f"{name} must be {count} contiguous float32 values on {device}")
    return t.data_ptr()


def _rows(name: str, t, device, *tail):
    """(address, elements from row to row) of a tensor [rows, *tail] whose rows are contiguous."""
    if t.device != device or tuple(t.shape[1:]) != tail:
        raise ValueError(f"{name} must be a [rows, {', '.join(map(str, tail))}] tensor on {device}, got {tuple(t.shape)} on {t.device}")
    inner = 1
    for size, stride in zip(reversed(tail), reversed(t.stride()[1:])):
        if size > 1 and stride != inner:
            raise ValueError(f"the rows of {name} must be contiguous")
        inner *= size
    pitch = t.stride(0) if t.shape[0] > 1 else inner
    if not inner <= pitch < 1 << 32:
        raise ValueError(f"the rows of {name} are {pitch} elements apart")
    return t.data_ptr(), pitch


def _cache(k_cache, v_cache):
    if not k_cache.is_cuda:
        raise ValueError("a paged cache lives on the GPU; the library has no CPU path")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype is not v_cache.dtype or k_cache.device != v_cache.device:
        raise ValueError("k_cache and v_cache must be alike: [pages, page_size, kv_heads, head_dim]")
    if k_cache.dtype not in _formats():
        raise ValueError("a paged cache is float32, float16 or bfloat16")
    if not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError("k_cache and v_cache must be contiguous")
    return k_cache.shape


@contextlib.contextmanager
def _elsewhere(device, stream):
    import torch
    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield


def _at(device, stream):
    """Whether calls on `device` and `stream` (None: its current one) go there as things stand; else the context that sees to it."""
    import torch
    if stream is None:
        return None if device.index == torch.cuda.current_device() else torch.cuda.device(device)
    if stream.device != device:
        raise ValueError(f"the stream belongs to {stream.device}, the tensors to {device}")
    return _elsewhere(device, stream)


def _launch(device, stream, call):
    """call(stream address) with the tensors' device current and, where a stream is given, tensors allocated for it."""
    import torch
    at = _at(device, stream)
    if at is None:
        return call(torch.cuda.current_stream(device).cuda_stream)
    with at:
        return call(torch.cuda.current_stream(device).cuda_stream)


def paged_plan(cached, fresh, table, held, free_pages, free_count, page_size: int, rows: int, step: PagedStep | None = None, stream=None) -> PagedStep:
    """Rows, positions and slots of a step, and the pages that it needs (mgq_paged_plan).

    cached, fresh, held: [sequences]; table: [sequences, width]; free_pages: [pages]; free_count: [1]; all int32 on the GPU.  table, held
    and free_count are updated.  `rows` bounds the new tokens of the step; rows behind the last sequence get slot NO_SLOT.
    """
    if not table.is_cuda or table.dim() != 2:
        raise ValueError("table must be a [sequences, width] CUDA tensor; the library has no CPU path")
    device, (sequences, width) = table.device, table.shape
    args = [_words("cached", cached, device, sequences), _words("fresh", fresh, device, sequences), sequences, page_size, _words("table", table, device, None, None), width,
            _words("held", held, device, sequences), _words("free_pages", free_pages, device, None), free_pages.shape[0], _words("free_count", free_count, device, 1), rows]

    def call(sp):
        out = PagedStep.empty(sequences, rows, device) if step is None else step
        check(lib.mgq_paged_plan(*args, _words("starts", out.starts, device, sequences + 1), _words("lengths", out.lengths, device, sequences),
                                 _words("positions", out.positions, device, rows), _words("slots", out.slots, device, rows), _words("lacking", out.lacking, device, 1), sp))
        return out
    return _launch(device, stream, call)


def paged_trim(lengths, table, held, free_pages, free_count, page_size: int, stream=None) -> None:
    """Returns the pages behind the first lengths[s] tokens of each sequence to the pool (mgq_paged_trim)."""
    if not table.is_cuda or table.dim() != 2:
        raise ValueError("table must be a [sequences, width] CUDA tensor; the library has no CPU path")
    device, (sequences, width) = table.device, table.shape
    args = [_words("lengths", lengths, device, sequences), sequences, page_size, _words("table", table, device, None, None), width, _words("held", held, device, sequences),
            _words("free_pages", free_pages, device, None), free_pages.shape[0], _words("free_count", free_count, device, 1)]
    _launch(device, stream, lambda sp: check(lib.mgq_paged_trim(*args, sp)))


def paged_append(q, k, v, positions, slots, k_cache, v_cache, theta: float = 0.0, q_out=None, stream=None):
    """Rows of keys (rotated where theta > 0) and values into the cache, and the rotated queries (mgq_paged_append).

    q: [rows, heads, head_dim] or None; k, v: [rows, kv_heads, head_dim], float32 or of the cache's type, rows any distance apart;
    positions, slots: [rows] as in a PagedStep; caches: [pages, page_size, kv_heads, head_dim].  Returns q_out [rows, heads, head_dim] in the cache's type.
    """
    import torch
    pages, page_size, kv_heads, d = _cache(k_cache, v_cache)
    device, rows, formats = k_cache.device, k.shape[0], _formats()
    if v.dtype is not k.dtype or (q is not None and q.dtype is not k.dtype) or k.dtype not in (torch.float32, k_cache.dtype):
        raise ValueError("q, k and v must have one type: float32 or the cache's")
    (kp, k_pitch), (vp, v_pitch) = _rows("k", k, device, kv_heads, d), _rows("v", v, device, kv_heads, d)
    if v.shape[0] != rows or (q is not None and q.shape[0] != rows):
        raise ValueError("q, k and v must have the same rows")
    heads = 0 if q is None else q.shape[1]
    qp, q_pitch = (None, 0) if q is None else _rows("q", q, device, heads, d)
    pp, sl = _words("positions", positions, device, rows), _words("slots", slots, device, rows)

    def call(sp):
        out = q_out
        if q is not None:
            if out is None:
                out = torch.empty((rows, heads, d), dtype=k_cache.dtype, device=device)
            elif out.dtype is not k_cache.dtype or out.device != device or not out.is_contiguous() or out.numel() != rows * heads * d:
                raise ValueError("q_out must be a contiguous [rows, heads, head_dim] tensor of the cache's type")
        check(lib.mgq_paged_append(qp, kp, vp, formats[k.dtype], pp, sl, out.data_ptr() if q is not None else None, k_cache.data_ptr(), v_cache.data_ptr(),
                                   formats[k_cache.dtype], rows, heads, kv_heads, d, q_pitch, k_pitch, v_pitch, page_size, pages, theta, sp))
        return out if q is not None else None
    return _launch(device, stream, call)


def paged_attention(q, k_cache, v_cache, table, starts, lengths, max_fresh: int, scale: float | None = None, window: int = 0, out=None, stream=None):
    """Attention of a step's new tokens over their sequences' pages (mgq_paged_attention).

    q: [rows, heads, head_dim] in the cache's type, rows any distance apart; table: [sequences, width]; starts, lengths as in a
    PagedStep; max_fresh: the most new tokens that a sequence has in this step; scale: 1 / sqrt(head_dim) where None; window: tokens that a token sees, itself
    included (0: all).  Returns `out` [rows, heads, head_dim]; rows behind the last sequence keep what they hold (zeros where out is None).
    """
    import torch
    pages, page_size, kv_heads, d = _cache(k_cache, v_cache)
    device, rows, heads = k_cache.device, q.shape[0], q.shape[1]
    if q.dtype is not k_cache.dtype:
        raise ValueError("q must have the cache's type")
    qp, q_pitch = _rows("q", q, device, heads, d)
    if table.dim() != 2 or window < 0 or max_fresh < 1:
        raise ValueError("table must be [sequences, width], window not negative and max_fresh positive")
    sequences, width = table.shape
    tp, sp_, lp = _words("table", table, device, None, None), _words("starts", starts, device, sequences + 1), _words("lengths", lengths, device, sequences)
    fmt = _formats()[q.dtype]
    if scale is None:
        scale = d ** -0.5

    def call(sp):
        o = torch.zeros((rows, heads, d), dtype=q.dtype, device=device) if out is None else out
        if o.dtype is not q.dtype or o.shape[0] != rows:
            raise ValueError("out must have the rows and the type of q")
        op, out_pitch = _rows("out", o, device, heads, d)
        room = torch.empty(max(_attention_workspace(heads, kv_heads, d, max_fresh, fmt), 16), dtype=torch.uint8, device=device)
        check(lib.mgq_paged_attention(qp, k_cache.data_ptr(), v_cache.data_ptr(), fmt, tp, sp_, lp, op, sequences, rows, max_fresh, heads, kv_heads, d, page_size, pages,
                                      width, q_pitch, out_pitch, scale, window, room.data_ptr(), sp))
        return o
    return _launch(device, stream, call)


def token_probs(logits, temperature=None, out=None, stream=None):
    """Probabilities of rows of logits [rows, vocab] float32 (mgq_token_probs); temperature: [rows] float32, 0 for the greedy choice."""
    import torch
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype is not torch.float32:
        raise ValueError("logits must be a [rows, vocab] float32 CUDA tensor; the library has no CPU path")
    device, (rows, vocab) = logits.device, logits.shape
    lp, pitch = _rows("logits", logits, device, vocab)
    tp = None if temperature is None else _floats("temperature", temperature, device, rows)

    def call(sp):
        o = torch.empty((rows, vocab), dtype=torch.float32, device=device) if out is None else out
        if o.dtype is not torch.float32 or o.shape[0] != rows:
            raise ValueError("out must be float32 and have the rows of logits")
        op, out_pitch = _rows("out", o, device, vocab)
        check(lib.mgq_token_probs(lp, pitch, tp, op, out_pitch, rows, vocab, sp))
        return o
    return _launch(device, stream, call)


def verify_drafts(target, draft, tokens, starts, accept, sample, out=None, stream=None):
    """Which drafted tokens stay, and the token behind them (mgq_verify_drafts).

    target, draft: [rows, vocab] float32 probabilities (draft None: chosen outright); tokens: [rows] int32, each sequence's last token and its drafts; starts:
    [sequences + 1] int32; accept: [rows], sample: [sequences] float32 in [0, 1).  Returns (accepted [sequences], next [sequences],
    tokens [rows]: kept drafts, next, then NO_TOKEN), into the three tensors of `out` where given.
    """
    import torch
    if not target.is_cuda or target.dim() != 2 or target.dtype is not torch.float32:
        raise ValueError("target must be a [rows, vocab] float32 CUDA tensor; the library has no CPU path")
    device, (rows, vocab), sequences = target.device, target.shape, starts.shape[0] - 1
    tp, t_pitch = _rows("target", target, device, vocab)
    dp, d_pitch = None, 0
    if draft is not None:
        if draft.dtype is not torch.float32 or draft.shape != target.shape:
            raise ValueError("draft must be like target")
        dp, d_pitch = _rows("draft", draft, device, vocab)
    args = [tp, t_pitch, dp, d_pitch, _words("tokens", tokens, device, rows), _words("starts", starts, device, None), _floats("accept", accept, device, rows),
            _floats("sample", sample, device, sequences)]

    def call(sp):
        o = tuple(torch.empty(n, dtype=torch.int32, device=device) for n in (sequences, sequences, rows)) if out is None else tuple(out)
        check(lib.mgq_verify_drafts(*args, _words("accepted", o[0], device, sequences), _words("next", o[1], device, sequences), _words("out", o[2], device, rows), sequences,
                                    rows, vocab, sp))
        return o
    return _launch(device, stream, call)


__all__ = ["PagedStep", "paged_plan", "paged_trim", "paged_append", "paged_attention", "token_probs", "verify_drafts", "NO_SLOT", "NO_PAGE", "NO_TOKEN", "Plan", "set_option", "device_status", "packed_bytes", "quantize", "dequantize", "shard_columns", "matmul", "matmul_host",
           "FMT_Q4", "FMT_Q8", "A_F32", "A_BF16"]
_ = _lib
