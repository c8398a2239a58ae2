"""The rules a server puts on a step's logits before a token is drawn: penalties for tokens that were there, a bias, a grammar's mask.

:class:`Penalties` says what they are and :func:`penalize` applies them in one pass over the logits (``dash_sample_penalize``);
``dashmag_b200.sample.sample`` takes them too.
"""
from __future__ import annotations

import ctypes
import dataclasses
from typing import Any, Optional

import torch

from . import _lib
from .attention import AttentionError, _check_device, _DTYPES, _index_bytes, _on, _ptr, _raise, _result, _stream


@dataclasses.dataclass(frozen=True)
class Penalties:
    """What is done to the logits ``[B, V]`` of a step, per row, in this order:

    - ``repetition``: a token anywhere in the history has its logit divided by it where positive, multiplied where not;
    - ``frequency``, ``presence``: subtracted for a token among the answer's ids, ``frequency`` as often as it is there;
    - ``bias``: added, ``[V]`` for every row or ``[B, V]``, f32 or the logits' dtype;
    - ``allowed``: a grammar's mask, ``[B, ceil(V / 32)]`` (or ``[ceil(V / 32)]`` for every row) of int32 words, bit ``v % 32`` of word
      ``v // 32`` set where token ``v`` may come; every other token's logit becomes ``-inf``.

    ``tokens [B, T]`` is the history, int32 or int64: the prompt's ids and behind them the answer's, ``lengths [B]`` of them there
    (``None``: all ``T``) and the first ``prompt_lengths [B]`` of those the prompt's (``None``: none).  Ids outside the vocabulary count
    for nothing.  The three penalties are numbers, or f32 tensors ``[B]``."""
    tokens: Optional[torch.Tensor] = None
    lengths: Optional[torch.Tensor] = None
    prompt_lengths: Optional[torch.Tensor] = None
    repetition: Any = 1.0
    frequency: Any = 0.0
    presence: Any = 0.0
    bias: Optional[torch.Tensor] = None
    allowed: Optional[torch.Tensor] = None


def penalize(logits: torch.Tensor, penalties: Penalties, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``logits [B, V]`` (f32, bf16 or f16) under ``penalties``, f32 arithmetic rounded once; into ``out`` (which may be the logits, but
    not other memory of theirs) where given.  Not differentiable (as ``sample`` itself)."""
    if out is None:
        done = _lib.binding().penalize(logits, penalties)
        if done is not None:
            return _result(done)
    op = "penalize"
    if logits.dim() != 2:
        raise AttentionError(f"{op}: logits must be [B, V], got {list(logits.shape)}")
    if logits.dtype not in _DTYPES:
        raise AttentionError(f"{op}: logits must be f32, bf16 or f16, got {logits.dtype}")
    b, v = logits.shape
    p = _lib.PenalizeParams()
    keep = []

    def rows(t: torch.Tensor) -> int:
        return t.stride(0) if t.shape[0] > 1 else t.shape[1]

    def index(name: str, t: Optional[torch.Tensor]):
        if t is None:
            return None, 0
        if tuple(t.shape) != (b,):
            raise AttentionError(f"{op}: the {name} are [B] = [{b}], got {list(t.shape)}")
        keep.append(t.contiguous())
        return _ptr(keep[-1]), _index_bytes(t, f"{op}: the {name}")

    p.dtype, p.b, p.v = int(_DTYPES[logits.dtype]), b, v
    tokens = penalties.tokens
    if tokens is not None:
        if tokens.dim() != 2 or tokens.shape[0] != b:
            raise AttentionError(f"{op}: the tokens are [B, T], B = {b}, got {list(tokens.shape)}")
        p.ids_elem_bytes = _index_bytes(tokens, f"{op}: the tokens")
        tokens = tokens if tokens.stride(1) == 1 else tokens.contiguous()
        keep.append(tokens)
        p.ids, p.ids_len, p.ids_stride = _ptr(tokens), tokens.shape[1], rows(tokens)
    elif penalties.lengths is not None or penalties.prompt_lengths is not None:
        raise AttentionError(f"{op}: lengths without tokens")
    p.lengths, p.lengths_elem_bytes = index("lengths", penalties.lengths)
    p.prompt_lengths, p.prompt_lengths_elem_bytes = index("prompt lengths", penalties.prompt_lengths)
    for name, nothing in (("repetition", 1.0), ("frequency", 0.0), ("presence", 0.0)):
        x = getattr(penalties, name)
        if isinstance(x, torch.Tensor):
            if tuple(x.shape) != (b,) or x.dtype != torch.float32:
                raise AttentionError(f"{op}: the {name} penalty is a number or f32 [B] = [{b}], got {x.dtype} {list(x.shape)}")
            if tokens is None:
                raise AttentionError(f"{op}: a {name} penalty needs the tokens")
            keep.append(x.contiguous())
            setattr(p, name, _ptr(keep[-1]))
            x = nothing
        elif x != nothing and tokens is None:
            raise AttentionError(f"{op}: a {name} penalty needs the tokens")
        setattr(p, name + "_all", float(x))
    bias = penalties.bias
    if bias is not None:
        if tuple(bias.shape) not in ((v,), (b, v)):
            raise AttentionError(f"{op}: the bias is [V] = [{v}] or [B, V] = [{b}, {v}], got {list(bias.shape)}")
        if bias.dtype not in (logits.dtype, torch.float32):
            raise AttentionError(f"{op}: the bias is {logits.dtype} or torch.float32, got {bias.dtype}")
        bias = bias if bias.stride(-1) == 1 else bias.contiguous()
        keep.append(bias)
        p.bias, p.bias_dtype, p.bias_stride = _ptr(bias), int(_DTYPES[bias.dtype]), 0 if bias.dim() == 1 else rows(bias)
    allowed = penalties.allowed
    if allowed is not None:
        words = (v + 31) // 32
        if tuple(allowed.shape) not in ((words,), (b, words)) or allowed.dtype != torch.int32:
            raise AttentionError(f"{op}: the allowed tokens are int32 words [{words}] or [{b}, {words}], got {allowed.dtype} {list(allowed.shape)}")
        allowed = allowed if allowed.stride(-1) == 1 else allowed.contiguous()
        keep.append(allowed)
        p.allowed, p.allowed_stride = _ptr(allowed), 0 if allowed.dim() == 1 else rows(allowed)
    if out is None:
        out = torch.empty((b, v), dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype or (v > 1 and out.stride(1) != 1):
        raise AttentionError(f"{op}: out must be {list(logits.shape)} of {logits.dtype} with a contiguous vocabulary, got {list(out.shape)} of {out.dtype}")
    elif b > 1 and out.stride(0) < v:
        raise AttentionError(f"{op}: out's rows overlap")
    logits = logits if logits.stride(1) == 1 or v == 1 else logits.contiguous()
    _check_device(op, logits, out, *keep)
    for t in (out, *keep):
        if t.device != logits.device:
            raise AttentionError(f"{op}: tensors of {logits.device} and of {t.device}")
    p.row_stride, p.out_stride = rows(logits), rows(out)
    with _on(logits.device):
        rc = _lib.lib().dash_sample_penalize(ctypes.byref(p), _ptr(logits), _ptr(out), _stream(logits.device))
    if rc != _lib.OK:
        _raise(rc)
    return out
