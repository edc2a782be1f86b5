"""Serving many sequences over one paged cache: torch-level entry points over the C ABI (mgq_paged_*, mgq_token_probs,
mgq_verify_drafts), reached as functions of `ops`.

These are thin argument marshallers: every computation happens in libmgq.  A call's checks cost as much as a small kernel, so each
function asks once whether everything is as it should be and looks for what is wrong only if not.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from ._lib import FMT_BF16, FMT_F16, FMT_F32, check, lib

NO_SLOT = NO_PAGE = NO_TOKEN = -1           # MGQ_NO_SLOT and its like as they read in an int32 tensor

_FORMATS = {torch.float32: FMT_F32, torch.float16: FMT_F16, torch.bfloat16: FMT_BF16}
_i32, _f32 = torch.int32, torch.float32
# what torch.cuda.current_device and current_stream ask, without their checks (2 us of a call); a torch without CUDA has neither
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: torch.cuda.current_stream(device).cuda_stream)


class PagedStep(NamedTuple):
    """Where a step's rows belong (int32 CUDA tensors): what paged_plan writes, paged_append and paged_attention read."""
    starts: torch.Tensor                    # [sequences + 1] first row of each sequence, then the end
    lengths: torch.Tensor                   # [sequences] tokens of each sequence, new ones included
    positions: torch.Tensor                 # [rows]
    slots: torch.Tensor                     # [rows]
    lacking: torch.Tensor                   # [1] pages that the pool was short of

    @staticmethod
    def empty(sequences: int, rows: int, device="cuda") -> "PagedStep":
        return PagedStep(*(torch.empty(n, dtype=_i32, device=device) for n in (sequences + 1, sequences, rows, rows, 1)))


@functools.lru_cache(maxsize=4096)
def _attention_workspace(heads: int, kv_heads: int, head_dim: int, max_fresh: int, dtype: int) -> int:
    return max(int(lib.mgq_paged_attention_workspace(heads, kv_heads, head_dim, max_fresh, dtype)), 16)


def _is(t, dtype, device: int, shape) -> bool:
    return t.dtype is dtype and t.get_device() == device and t.shape == shape and t.is_contiguous()


def _refuse(device: int, **wanted):
    """Names the first tensor that is not a contiguous tensor of its (type, shape) on the device; a size of None is any."""
    if device < 0:
        raise ValueError("the operators take CUDA tensors; the library has no CPU path")
    for name, (t, dtype, shape) in wanted.items():
        fits = len(t.shape) == len(shape) and all(want is None or have == want for have, want in zip(t.shape, shape))
        if not (t.dtype is dtype and t.get_device() == device and fits and t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on cuda:{device}, not {tuple(t.shape)} {t.dtype} on {t.device}")
    raise AssertionError("nothing to refuse")


def _words(**values):
    """Refuses whole numbers that a 32-bit word of the C entries would cut."""
    for name, value in values.items():
        if not 0 <= value < 1 << 32:
            raise ValueError(f"{name} {value} is not from 0 to 2^32 - 1")


def _pitch(name: str, t, device: int, inner: int) -> int:
    """Elements from row to row of a tensor whose rows of `inner` elements are contiguous."""
    if t.is_contiguous() and t.get_device() == device:
        return inner
    if t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device}, not {t.device}")
    shape, strides = t.shape, t.stride()
    if shape[0] > 1 and strides[-1] == 1 and (len(shape) == 2 or len(shape) == 3 and strides[1] == shape[2]):       # what a slice of wider rows has
        pitch = strides[0]
    else:
        run = 1
        for size, stride in zip(reversed(shape[1:]), reversed(strides[1:])):
            if size > 1 and stride != run:
                raise ValueError(f"the rows of {name} must be contiguous")
            run *= size
        pitch = strides[0] if shape[0] > 1 else inner
    if not inner <= pitch < 1 << 32:
        raise ValueError(f"the rows of {name} are {pitch} elements apart")
    return pitch


def _on(device: int, stream, call):
    """call(stream address) with the tensors' device current and, where a stream is given, tensors allocated for it."""
    if stream is None:
        if device == _current_device():
            return call(_current_stream(device))
        with torch.cuda.device(device):
            return call(_current_stream(device))
    if stream.device.index != device:
        raise ValueError(f"the stream belongs to {stream.device}, the tensors to cuda:{device}")
    with torch.cuda.device(device), torch.cuda.stream(stream):
        return call(stream.cuda_stream)


def _table(table):
    device = table.get_device()
    if device < 0 or table.dim() != 2 or table.dtype is not _i32 or not table.is_contiguous():
        raise ValueError("table must be a contiguous int32 CUDA tensor [sequences, width]; the library has no CPU path")
    return device, *table.shape


def paged_plan(cached, fresh, table, held, free_pages, free_count, page_size: int, rows: int, step: PagedStep | None = None, stream=None) -> PagedStep:
    """Rows, positions and slots of a step, and the pages that it needs (mgq_paged_plan).

    cached, fresh, held: [sequences]; table: [sequences, width]; free_pages: [pages]; free_count: [1]; all int32 on the GPU.  table, held
    and free_count are updated.  `rows` bounds the new tokens of the step; rows behind the last sequence get slot NO_SLOT.
    """
    device, sequences, width = _table(table)
    each, one = (sequences,), (1,)
    if not (0 <= page_size < 1 << 32 and 0 <= rows < 1 << 32):
        _words(page_size=page_size, rows=rows)
    if not (_is(cached, _i32, device, each) and _is(fresh, _i32, device, each) and _is(held, _i32, device, each) and _is(free_count, _i32, device, one)
            and free_pages.dim() == 1 and _is(free_pages, _i32, device, free_pages.shape)):
        _refuse(device, cached=(cached, _i32, each), fresh=(fresh, _i32, each), held=(held, _i32, each), free_count=(free_count, _i32, one), free_pages=(free_pages, _i32, (None,)))
    if step is not None:
        row = (rows,)
        if not (_is(step[0], _i32, device, (sequences + 1,)) and _is(step[1], _i32, device, each) and _is(step[2], _i32, device, row) and _is(step[3], _i32, device, row)
                and _is(step[4], _i32, device, one)):
            _refuse(device, starts=(step[0], _i32, (sequences + 1,)), lengths=(step[1], _i32, each), positions=(step[2], _i32, row), slots=(step[3], _i32, row),
                    lacking=(step[4], _i32, one))

    def call(sp):
        out = PagedStep.empty(sequences, rows, table.device) if step is None else step
        check(lib.mgq_paged_plan(cached.data_ptr(), fresh.data_ptr(), sequences, page_size, table.data_ptr(), width, held.data_ptr(), free_pages.data_ptr(),
                                 free_pages.shape[0], free_count.data_ptr(), rows, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(),
                                 out[4].data_ptr(), sp))
        return out
    return _on(device, stream, call)


def paged_trim(lengths, table, held, free_pages, free_count, page_size: int, stream=None) -> None:
    """Returns the pages behind the first lengths[s] tokens of each sequence to the pool (mgq_paged_trim)."""
    device, sequences, width = _table(table)
    each, one = (sequences,), (1,)
    if not 0 <= page_size < 1 << 32:
        _words(page_size=page_size)
    if not (_is(lengths, _i32, device, each) and _is(held, _i32, device, each) and _is(free_count, _i32, device, one) and free_pages.dim() == 1
            and _is(free_pages, _i32, device, free_pages.shape)):
        _refuse(device, lengths=(lengths, _i32, each), held=(held, _i32, each), free_count=(free_count, _i32, one), free_pages=(free_pages, _i32, (None,)))
    _on(device, stream, lambda sp: check(lib.mgq_paged_trim(lengths.data_ptr(), sequences, page_size, table.data_ptr(), width, held.data_ptr(), free_pages.data_ptr(),
                                                            free_pages.shape[0], free_count.data_ptr(), sp)))


def _caches(k_cache, v_cache):
    device, shape = k_cache.get_device(), k_cache.shape
    if device < 0:
        raise ValueError("a paged cache lives on the GPU; the library has no CPU path")
    if len(shape) != 4 or not _is(v_cache, k_cache.dtype, device, shape) or not k_cache.is_contiguous() or k_cache.dtype not in _FORMATS:
        raise ValueError("k_cache and v_cache must be alike: contiguous [pages, page_size, kv_heads, head_dim] of float32, float16 or bfloat16 on one device")
    return device, *shape


def paged_append(q, k, v, positions, slots, k_cache, v_cache, theta: float = 0.0, q_out=None, stream=None):
    """Rows of keys (rotated where theta > 0) and values into the cache, and the rotated queries (mgq_paged_append).

    q: [rows, heads, head_dim] or None; k, v: [rows, kv_heads, head_dim], float32 or of the cache's type, rows any distance apart;
    positions, slots: [rows] as in a PagedStep; caches: [pages, page_size, kv_heads, head_dim].  Returns q_out [rows, heads, head_dim] in the cache's type.
    """
    device, pages, page_size, kv_heads, d = _caches(k_cache, v_cache)
    rows, src, dst = k.shape[0], k.dtype, k_cache.dtype
    if src is not _f32 and src is not dst or v.dtype is not src or q is not None and q.dtype is not src:
        raise ValueError("q, k and v must have one type: float32 or the cache's")
    if k.shape != (rows, kv_heads, d) or v.shape != k.shape or q is not None and (q.dim() != 3 or q.shape[0] != rows or q.shape[2] != d):
        raise ValueError(f"k and v must be [rows, {kv_heads}, {d}] and q [rows, heads, {d}], not {tuple(k.shape)}, {tuple(v.shape)}, {None if q is None else tuple(q.shape)}")
    if not (_is(positions, _i32, device, (rows,)) and _is(slots, _i32, device, (rows,))):
        _refuse(device, positions=(positions, _i32, (rows,)), slots=(slots, _i32, (rows,)))
    heads = 0 if q is None else q.shape[1]
    q_pitch, k_pitch, v_pitch = 0 if q is None else _pitch("q", q, device, heads * d), _pitch("k", k, device, kv_heads * d), _pitch("v", v, device, kv_heads * d)
    if q is not None and q_out is not None and not (_is(q_out, dst, device, q_out.shape) and q_out.numel() == rows * heads * d):
        _refuse(device, q_out=(q_out, dst, (rows, heads, d)))

    def call(sp):
        out = q_out
        if q is None:
            out = None
        elif out is None:
            out = torch.empty((rows, heads, d), dtype=dst, device=k_cache.device)
        check(lib.mgq_paged_append(None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), _FORMATS[src], positions.data_ptr(), slots.data_ptr(),
                                   None if out is None else out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _FORMATS[dst], rows, heads, kv_heads, d, q_pitch,
                                   k_pitch, v_pitch, page_size, pages, theta, sp))
        return out
    return _on(device, stream, call)


def paged_attention(q, k_cache, v_cache, table, starts, lengths, max_fresh: int, scale: float | None = None, window: int = 0, out=None, stream=None):
    """Attention of a step's new tokens over their sequences' pages (mgq_paged_attention).

    q: [rows, heads, head_dim] in the cache's type, rows any distance apart; table: [sequences, width]; starts, lengths as in a
    PagedStep; max_fresh: the most new tokens that a sequence has in this step; scale: 1 / sqrt(head_dim) where None; window: tokens that a token sees, itself
    included (0: all).  Returns `out` [rows, heads, head_dim]; rows behind the last sequence keep what they hold (zeros where out is None).
    """
    device, pages, page_size, kv_heads, d = _caches(k_cache, v_cache)
    dtype = q.dtype
    if dtype is not k_cache.dtype or q.dim() != 3 or q.shape[2] != d:
        raise ValueError(f"q must be [rows, heads, {d}] in the cache's type, not {tuple(q.shape)} {dtype}")
    rows, heads, _ = q.shape
    _, sequences, width = _table(table)
    if table.get_device() != device or not (_is(starts, _i32, device, (sequences + 1,)) and _is(lengths, _i32, device, (sequences,))):
        _refuse(device, table=(table, _i32, (None, None)), starts=(starts, _i32, (sequences + 1,)), lengths=(lengths, _i32, (sequences,)))
    if window < 0 or max_fresh < 1:
        raise ValueError(f"window {window} is negative or max_fresh {max_fresh} not positive")
    if window >> 31:                                    # no sequence is that long
        window = 0
    most = min(max_fresh, 0xFFFFFFFF)
    q_pitch = _pitch("q", q, device, heads * d)
    if out is not None and (out.dtype is not dtype or out.shape != q.shape):
        raise ValueError("out must have the shape and the type of q")
    fmt = _FORMATS[dtype]

    def call(sp):
        o = torch.zeros((rows, heads, d), dtype=dtype, device=q.device) if out is None else out
        room = torch.empty(_attention_workspace(heads, kv_heads, d, most, fmt), dtype=torch.uint8, device=q.device)
        check(lib.mgq_paged_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), fmt, table.data_ptr(), starts.data_ptr(), lengths.data_ptr(), o.data_ptr(),
                                      sequences, rows, most, heads, kv_heads, d, page_size, pages, width, q_pitch, _pitch("out", o, device, heads * d),
                                      d ** -0.5 if scale is None else scale, window, room.data_ptr(), sp))
        return o
    return _on(device, stream, call)


def _logits(name, t):
    device = t.get_device()
    if device < 0 or t.dim() != 2 or t.dtype is not _f32:
        raise ValueError(f"{name} must be a [rows, vocab] float32 CUDA tensor; the library has no CPU path")
    rows, vocab = t.shape
    return device, rows, vocab, _pitch(name, t, device, vocab)


def token_probs(logits, temperature=None, out=None, stream=None):
    """Probabilities of rows of logits [rows, vocab] float32 (mgq_token_probs); temperature: [rows] float32, 0 for the greedy choice."""
    device, rows, vocab, pitch = _logits("logits", logits)
    if temperature is not None and not _is(temperature, _f32, device, (rows,)):
        _refuse(device, temperature=(temperature, _f32, (rows,)))
    if out is not None and (out.dtype is not _f32 or out.shape != logits.shape):
        raise ValueError("out must be float32 and have the shape of logits")

    def call(sp):
        o = torch.empty((rows, vocab), dtype=_f32, device=logits.device) if out is None else out
        check(lib.mgq_token_probs(logits.data_ptr(), pitch, None if temperature is None else temperature.data_ptr(), o.data_ptr(), _pitch("out", o, device, vocab), rows,
                                  vocab, sp))
        return o
    return _on(device, stream, call)


def verify_drafts(target, draft, tokens, starts, accept, sample, out=None, stream=None):
    """Which drafted tokens stay, and the token behind them (mgq_verify_drafts).

    target, draft: [rows, vocab] float32 probabilities (draft None: chosen outright); tokens: [rows] int32, each sequence's last token and its drafts; starts:
    [sequences + 1] int32; accept: [rows], sample: [sequences] float32 in [0, 1).  Returns (accepted [sequences], next [sequences],
    tokens [rows]: kept drafts, next, then NO_TOKEN), into the three tensors of `out` where given; rows behind the last sequence keep what they hold (NO_TOKEN
    where out is None).
    """
    device, rows, vocab, t_pitch = _logits("target", target)
    sequences = starts.shape[0] - 1
    d_pitch = 0
    if draft is not None:
        if draft.dtype is not _f32 or draft.shape != target.shape:
            raise ValueError("draft must be like target")
        d_pitch = _pitch("draft", draft, device, vocab)
    row, each = (rows,), (sequences,)
    if not (_is(tokens, _i32, device, row) and _is(starts, _i32, device, (sequences + 1,)) and _is(accept, _f32, device, row) and _is(sample, _f32, device, each)):
        _refuse(device, tokens=(tokens, _i32, row), starts=(starts, _i32, (sequences + 1,)), accept=(accept, _f32, row), sample=(sample, _f32, each))
    if out is not None and not (_is(out[0], _i32, device, each) and _is(out[1], _i32, device, each) and _is(out[2], _i32, device, row)):
        _refuse(device, accepted=(out[0], _i32, each), next=(out[1], _i32, each), out=(out[2], _i32, row))

    def call(sp):
        if out is None:
            o = (*torch.empty((2, sequences), dtype=_i32, device=target.device), torch.full((rows,), NO_TOKEN, dtype=_i32, device=target.device))
        else:
            o = tuple(out)
        check(lib.mgq_verify_drafts(target.data_ptr(), t_pitch, None if draft is None else draft.data_ptr(), d_pitch, tokens.data_ptr(), starts.data_ptr(), accept.data_ptr(),
                                    sample.data_ptr(), o[0].data_ptr(), o[1].data_ptr(), o[2].data_ptr(), sequences, rows, vocab, sp))
        return o
    return _on(device, stream, call)
