"""Decoder attention for a serving loop: rotary positions, a paged key/value cache and the attention that reads it.

What a decoder layer does between its query/key/value projection and its output projection:

    q = kv_append(k, v, k_cache, v_cache, page_table, q_start, kv_len, q=q, inv_freq=inv_freq)   # turn q and k, store k and v
    out = paged_attention(q, k_cache, v_cache, page_table, q_start, kv_len, max_q=longest)

A cache is a pool of pages, ``k_cache`` and ``v_cache`` of shape ``[num_pages, page_size, kv_heads, head_dim]`` (a pool stored
``[num_pages, kv_heads, page_size, head_dim]`` is passed as ``pool.transpose(1, 2)``).  A batch of sequences is three int32
tensors on the device: ``page_table [batch, width]``, ``q_start [batch + 1]`` (rows of ``q``/``k``/``v`` of each sequence) and
``kv_len [batch]`` (tokens in the cache, the new ones included).  The calls read them on the device and enqueue work on
the current stream of the tensors' device, so a step can be captured into a CUDA graph and replayed with other lengths.
Rows behind ``q_start[batch]`` are left as they are.  Inference only: a tensor that requires a gradient is refused.

The reference has no counterpart (its attention is the decomposed chain of llcompiler/compiler/torch_compile_config.py:24
over dense tensors); the entry points are llc_cuda_rotary, llc_cuda_kv_append and llc_cuda_paged_attention of the C ABI.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

try:
    from llcompiler_ import ops as _ops
except ImportError as e:  # the CUDA path is the only path: fail loudly
    raise ImportError("the llcompiler_ extension module is not built; run `python -m llcompiler_b200.build`") from e

_DTYPE = {torch.float32: 4, torch.float16: 7, torch.bfloat16: 8}
_INDEX = {torch.int32: 2, torch.int64: 3}


def _tensor(name: str, t, rank: int, device: torch.device, dtype=None) -> None:
    """Checks one operand: a tensor of `rank` dims on `device`, of `dtype`, that wants no gradient."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t).__name__}")
    if t.dim() != rank:
        raise ValueError(f"{name}: expected {rank} dims, got shape {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, expected {device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: inference only, it requires a gradient")


def _rows(name: str, t, device: torch.device, dtype) -> None:
    _tensor(name, t, 3, device, dtype)
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: the head dim must have unit stride")


def _first(name: str, t) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor; there is no CPU fallback")
    if t.dtype not in _DTYPE:
        raise ValueError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return t.device


def _output(name: str, out, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _rows(name, out, like.device, like.dtype)
    if out.shape != like.shape:
        raise ValueError(f"{name}: expected shape {tuple(like.shape)}, got {tuple(out.shape)}")
    for n, s in zip(out.shape, out.stride()):
        if n > 1 and s == 0:
            raise ValueError(f"{name}: an output may not repeat its elements (stride 0)")
    return out


def _turns(positions, inv_freq, sections, tokens: int, head_dim: int, device: torch.device):
    """(positions' address, their type code, axis stride, pairs, axes, sections padded to four) of the rotary arguments."""
    _tensor("inv_freq", inv_freq, 1, device, torch.float64)
    pairs = inv_freq.shape[0]
    if pairs > 1 and inv_freq.stride(0) != 1:
        raise ValueError("inv_freq: must be contiguous")
    if not 1 <= pairs <= head_dim // 2:
        raise ValueError(f"inv_freq: {pairs} pairs do not fit a head of {head_dim}")
    sections = [pairs] if sections is None else [int(n) for n in sections]
    if not 1 <= len(sections) <= 4 or sum(sections) != pairs or min(sections) < 0:
        raise ValueError(f"sections: 1 to 4 numbers that add up to {pairs} pairs, got {sections}")
    axes = len(sections)
    sections = sections + [0] * (4 - axes)
    if positions is None:
        return 0, 3, 0, pairs, axes, sections
    if isinstance(positions, torch.Tensor) and positions.dim() == 1:
        positions = positions[None]
    _tensor("positions", positions, 2, device)
    if positions.dtype not in _INDEX:
        raise ValueError(f"positions: expected int32 or int64, got {positions.dtype}")
    if positions.shape != (axes, tokens):
        raise ValueError(f"positions: expected shape ({axes}, {tokens}), got {tuple(positions.shape)}")
    if tokens > 1 and positions.stride(1) != 1:
        raise ValueError("positions: must have unit stride along the tokens")
    return positions.data_ptr(), _INDEX[positions.dtype], positions.stride(0), pairs, axes, sections


def _batch(page_table, q_start, kv_len, bad_pages, device: torch.device):
    _tensor("page_table", page_table, 2, device, torch.int32)
    _tensor("q_start", q_start, 1, device, torch.int32)
    _tensor("kv_len", kv_len, 1, device, torch.int32)
    batch, width = page_table.shape
    if width > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table: must have unit stride along a sequence's pages")
    if q_start.shape[0] != batch + 1 or kv_len.shape[0] != batch:
        raise ValueError(f"q_start and kv_len: expected {batch + 1} and {batch} entries, got {q_start.shape[0]} and {kv_len.shape[0]}")
    if (q_start.stride(0) != 1) or (batch > 1 and kv_len.stride(0) != 1):
        raise ValueError("q_start and kv_len: must be contiguous")
    if bad_pages is not None:
        _tensor("bad_pages", bad_pages, 1, device, torch.int32)
        if bad_pages.shape[0] != 1:
            raise ValueError("bad_pages: one counter")
    return batch, width


def _caches(k_cache, v_cache, device: torch.device, dtype):
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _tensor(name, t, 4, device, dtype)
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError(f"{name}: the head dim must have unit stride")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"v_cache: expected shape {tuple(k_cache.shape)}, got {tuple(v_cache.shape)}")
    if k_cache.shape[1] < 1 or k_cache.shape[2] < 1:
        raise ValueError(f"k_cache: empty pages, shape {tuple(k_cache.shape)}")
    return k_cache.shape


def _on_device(device: torch.device):
    """A context that makes `device` current, or None when it is already."""
    return None if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _call(device: torch.device, f, *args):
    ctx = _on_device(device)
    if ctx is None:
        return f(*args, torch.cuda.current_stream(device).cuda_stream)
    with ctx:
        return f(*args, torch.cuda.current_stream(device).cuda_stream)


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections: Optional[Sequence[int]] = None,
           interleaved: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns ``x [tokens, heads, head_dim]`` by its rotary positions and returns the result (``out``, or a new tensor).

    ``positions`` is ``[tokens]`` or ``[axes, tokens]`` (int32 or int64); ``inv_freq`` holds one float64 frequency per pair, and
    ``sections`` says how many pairs belong to each axis, in order (time, height, width of a video, say; default: one axis).
    Pair i is elements ``(i, i + pairs)``, or ``(2i, 2i + 1)`` when ``interleaved``; elements past the pairs are copied.
    ``out`` may be ``x`` itself."""
    device = _first("x", x)
    _rows("x", x, device, x.dtype)
    tokens, heads, d = x.shape
    if positions is None:
        raise ValueError("positions: required")
    pos, pos_type, pos_sa, pairs, axes, sections = _turns(positions, inv_freq, sections, tokens, d, device)
    out = _output("out", out, x)
    _call(device, _ops.rotary, (x.data_ptr(), out.data_ptr(), pos, inv_freq.data_ptr()), _DTYPE[x.dtype], pos_type, (tokens, heads, d, pairs),
          (x.stride(0), x.stride(1), out.stride(0), out.stride(1), pos_sa), axes, sections, interleaved)
    return out


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, q_start: torch.Tensor,
              kv_len: torch.Tensor, q: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
              sections: Optional[Sequence[int]] = None, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
              bad_pages: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the new tokens' ``k`` and ``v`` (``[tokens, kv_heads, head_dim]``) into their slots of the cache.

    With ``inv_freq`` the keys are turned on the way (see ``rotary``; ``positions`` default to the tokens' places in their
    sequences), and so are the queries ``q [tokens, heads, head_dim]``, which are returned (``q_out``, or a new tensor; rows
    of no sequence are not written).  A token whose page number is no page of the pool, or whose place lies outside the
    table, is not stored and is counted in ``bad_pages`` (one int32) if that is given.  Two tokens must not share a slot."""
    device = _first("k", k)
    dtype = k.dtype
    _rows("k", k, device, dtype)
    _rows("v", v, device, dtype)
    pages, page, kv_heads, d = _caches(k_cache, v_cache, device, dtype)
    tokens = k.shape[0]
    if k.shape != v.shape or k.shape[1:] != (kv_heads, d):
        raise ValueError(f"k and v: expected [tokens, {kv_heads}, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    batch, width = _batch(page_table, q_start, kv_len, bad_pages, device)
    heads, q_strides, ptr_q, ptr_out = 0, (0, 0, 0, 0), 0, 0
    if q is not None:
        _rows("q", q, device, dtype)
        if q.shape[0] != tokens or q.shape[2] != d:
            raise ValueError(f"q: expected [{tokens}, heads, {d}], got {tuple(q.shape)}")
        q_out = _output("q_out", q_out, q)
        heads, q_strides = q.shape[1], (q.stride(0), q.stride(1), q_out.stride(0), q_out.stride(1))
        ptr_q, ptr_out = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out: no queries were given")
    if inv_freq is None:
        if positions is not None or sections is not None:
            raise ValueError("positions and sections: no inv_freq was given")
        pos, pos_type, pos_sa, pairs, axes, sections, freq = 0, 3, 0, 0, 0, (0, 0, 0, 0), 0
    else:
        pos, pos_type, pos_sa, pairs, axes, sections = _turns(positions, inv_freq, sections, tokens, d, device)
        freq = inv_freq.data_ptr()
    _call(device, _ops.kv_append,
          (k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), ptr_q, ptr_out, page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), pos, freq,
           0 if bad_pages is None else bad_pages.data_ptr()), _DTYPE[dtype], pos_type,
          (tokens, batch, heads, kv_heads, d, pairs, pages, page, width, page_table.stride(0)),
          (*q_strides, k.stride(0), k.stride(1), v.stride(0), v.stride(1), *k_cache.stride()[:3], *v_cache.stride()[:3], pos_sa), axes, sections, interleaved)
    return q_out


def _run_attention(args, device: torch.device) -> None:
    bytes_ = _ops.paged_attention_workspace(*args)
    # from the caching allocator at every call: ordered with the stream, and a captured graph gets memory of its own
    workspace = torch.empty(bytes_, dtype=torch.uint8, device=device) if bytes_ else None
    _ops.paged_attention(*args, 0 if workspace is None else workspace.data_ptr(), bytes_, torch.cuda.current_stream(device).cuda_stream)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                    scale: Optional[float] = None, window: int = 0, sinks: int = 0, max_q: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    bad_pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens ``q [tokens, heads, head_dim]`` over the cache, which holds their keys and values already.

    A token at place p of its sequence sees the keys at places j <= p; with ``window`` > 0 those with ``p - j < window`` and the
    first ``sinks`` of the sequence.  Query head h reads key head ``h // (heads // kv_heads)``.  ``scale`` defaults to
    ``1 / sqrt(head_dim)``.  ``max_q`` bounds the new tokens of one sequence (default: all of them); a decoding step says 1,
    which lets the call choose the kernel for few rows; a sequence that has more is left out.  A token that sees nothing gets
    zeros; rows of no sequence are not written.  Pages that are none of the pool's read as zeros and are counted in
    ``bad_pages`` (one int32) if that is given."""
    device = _first("q", q)
    dtype = q.dtype
    _rows("q", q, device, dtype)
    pages, page, kv_heads, d = _caches(k_cache, v_cache, device, dtype)
    tokens, heads = q.shape[0], q.shape[1]
    if q.shape[2] != d or heads == 0 or heads % kv_heads:
        raise ValueError(f"q: expected [tokens, a multiple of {kv_heads}, {d}], got {tuple(q.shape)}")
    batch, width = _batch(page_table, q_start, kv_len, bad_pages, device)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks: must not be negative")
    if max_q is None:
        max_q = tokens
    elif max_q < 0:
        raise ValueError("max_q: must not be negative")
    out = _output("out", out, q)
    args = ((q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(),
             0 if bad_pages is None else bad_pages.data_ptr()), _DTYPE[dtype], 1.0 / math.sqrt(d) if scale is None else scale,
            (tokens, batch, heads, kv_heads, d, max_q, pages, page, width, page_table.stride(0), window, sinks),
            (q.stride(0), q.stride(1), out.stride(0), out.stride(1), *k_cache.stride()[:3], *v_cache.stride()[:3]))
    ctx = _on_device(device)
    if ctx is None:
        _run_attention(args, device)
    else:
        with ctx:
            _run_attention(args, device)
    return out
