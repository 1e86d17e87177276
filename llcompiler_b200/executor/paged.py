"""Decoder attention for a serving loop: rotary positions, a paged key/value cache and the attention that reads it.

What a decoder layer does between its query/key/value projection and its output projection:

    q = kv_append(k, v, k_cache, v_cache, page_table, q_start, kv_len, q=q, inv_freq=inv_freq)   # turn q and k, store k and v
    out = paged_attention(q, k_cache, v_cache, page_table, q_start, kv_len, max_q=longest)

A cache is a pool of pages, ``k_cache`` and ``v_cache`` of shape ``[num_pages, page_size, kv_heads, head_dim]`` (a pool stored
``[num_pages, kv_heads, page_size, head_dim]`` is passed as ``pool.transpose(1, 2)``).  A batch of sequences is three int32
tensors on the device: ``page_table [batch, width]``, ``q_start [batch + 1]`` (rows of ``q``/``k``/``v`` of each sequence) and
``kv_len [batch]`` (tokens in the cache, the new ones included).  The calls read them on the device and enqueue work on
the current stream of the tensors' device, so a step can be captured into a CUDA graph and replayed with other lengths.
Rows behind ``q_start[batch]`` are left as they are.  Inference only: a tensor that requires a gradient
or carries a forward-mode tangent is refused; tensors of the caller's that a call writes count as changed in place.

The reference has no counterpart (its attention is the decomposed chain of llcompiler/compiler/torch_compile_config.py:24
over dense tensors); the entry points are llc_cuda_rotary, llc_cuda_kv_append and llc_cuda_paged_attention of the C ABI.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

try:
    from llcompiler_ import ops as _ops
except ImportError as e:  # the CUDA path is the only path: fail loudly
    raise ImportError("the llcompiler_ extension module is not built; run `python -m llcompiler_b200.build`") from e

_current = torch._C._cuda_getDevice


def _elsewhere(f, first, *args):
    """Runs `f`, which makes the checks and launches, with the first operand's device current."""
    index = first.get_device() if isinstance(first, torch.Tensor) else -1
    if index < 0:
        return f(first, *args)      # which refuses it
    with torch.cuda.device(index):
        return f(first, *args)


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections: Optional[Sequence[int]] = None,
           interleaved: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns ``x [tokens, heads, head_dim]`` by its rotary positions and returns the result (``out``, or a new tensor).

    ``positions`` is ``[tokens]`` or ``[axes, tokens]`` (int32 or int64); ``inv_freq`` holds one float64 frequency per pair, and
    ``sections`` says how many pairs belong to each axis, in order (time, height, width of a video, say; default: one axis).
    Pair i is elements ``(i, i + pairs)``, or ``(2i, 2i + 1)`` when ``interleaved``; elements past the pairs are copied.
    ``out`` may be ``x`` itself, and shares no memory with it otherwise."""
    if isinstance(x, torch.Tensor) and x.is_cuda and x.get_device() == _current():
        return _ops.rotary(x, positions, inv_freq, sections, interleaved, out)
    return _elsewhere(_ops.rotary, x, positions, inv_freq, sections, interleaved, out)


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, q_start: torch.Tensor,
              kv_len: torch.Tensor, q: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
              sections: Optional[Sequence[int]] = None, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
              bad_pages: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the new tokens' ``k`` and ``v`` (``[tokens, kv_heads, head_dim]``) into their slots of the cache.

    With ``inv_freq`` the keys are turned on the way (see ``rotary``; ``positions`` default to the tokens' places in their
    sequences), and so are the queries ``q [tokens, heads, head_dim]``, which are returned (``q_out``, or a new tensor; rows
    of no sequence are not written).  A token whose page number is no page of the pool, or whose place lies outside the
    table, is not stored and is counted in ``bad_pages`` (one int32) if that is given.  Two tokens must not share a slot.
    ``q_out`` may be ``q`` itself; nothing else that the call writes may lie in memory that it reads or writes otherwise."""
    if isinstance(k, torch.Tensor) and k.is_cuda and k.get_device() == _current():
        return _ops.kv_append(k, v, k_cache, v_cache, page_table, q_start, kv_len, q, positions, inv_freq, sections, interleaved, q_out, bad_pages)
    return _elsewhere(_ops.kv_append, k, v, k_cache, v_cache, page_table, q_start, kv_len, q, positions, inv_freq, sections, interleaved, q_out, bad_pages)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                    scale: Optional[float] = None, window: int = 0, sinks: int = 0, max_q: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    bad_pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens ``q [tokens, heads, head_dim]`` over the cache, which holds their keys and values already.

    A token at place p of its sequence sees the keys at places j <= p; with ``window`` > 0 those with ``p - j < window`` and the
    first ``sinks`` of the sequence.  Query head h reads key head ``h // (heads // kv_heads)``.  ``scale`` defaults to
    ``1 / sqrt(head_dim)``.  ``max_q`` bounds the new tokens of one sequence (default: all of them); a decoding step says 1,
    which lets the call choose the kernel for few rows alone (without it, 64 sequences of 1000 keys: 67 us instead of 55); a
    sequence that has more is left out.  A token that sees nothing gets
    zeros, one whose visible scores are all -inf NaN (0 / 0); rows of no sequence are not written.  Pages that are none of the pool's
    read as zeros and are counted in ``bad_pages`` (one int32) if that is given.  ``out`` may be ``q`` itself, and shares no memory with
    the operands otherwise."""
    if isinstance(q, torch.Tensor) and q.is_cuda and q.get_device() == _current():
        return _ops.paged_attention(q, k_cache, v_cache, page_table, q_start, kv_len, scale, window, sinks, max_q, out, bad_pages)
    return _elsewhere(_ops.paged_attention, q, k_cache, v_cache, page_table, q_start, kv_len, scale, window, sinks, max_q, out, bad_pages)


def device_status(device: Optional[int] = None) -> int:
    """Waits for the device (default: the current one) and raises if a kernel of an earlier call recorded a failure, which it cannot
    raise itself: a wait of a tensor-core kernel that gave up, so that its output is wrong.  Returns 0 otherwise.  Reading clears
    what was recorded.  The calls above return before their kernels have run; a caller asks here after its own synchronisation, as
    ``Torch_ExecutionEngine.status`` does for compiled plans.  Not to be called while a stream is being captured."""
    if device is None:
        code = _ops.status()
    else:
        with torch.cuda.device(device):
            code = _ops.status()
    if code < 0:
        raise RuntimeError("device_status: the device cannot be read")
    if code:
        who = "attention over the paged cache" if code >= 8 else "attention" if code >= 6 else "a matrix product or convolution"
        raise RuntimeError(f"device_status: a kernel of {who} gave up (code {code}); its output is wrong")
    return code
