"""The decoding step of a batch whose sequences share prompts.

Several answers to one prompt, many users behind one instruction: the keys and values of a prompt are held once, ``[N,P,Hkv,D]`` for
``N`` prompts, beside the sequences' own caches ``[B,S,Hkv,D]``, and one step reads each prompt once for many of its sequences
(``dash_attn_decode_shared``: once for each tile of their heads' rows).  The result is that of ``attention_decode`` over caches that hold the prompt's rows and then the
sequence's own, as finely rounded and with its sums in another order.  Where a prompt's sequences are few, ``attention_decode`` over joined
caches is the faster (up to eight behind 1000 keys, one behind 8192).  Not differentiable (as ``attention.attention_decode`` itself).
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .attention import AttentionError, _check_device, _index_bytes, _on, _ptr, _raise, _result, _stream, _workspace, make_decode_params
from .contract import AttentionOptions


def _prefix_params(op, key, value, prefix_key, prefix_value, prefix_lengths):
    for t in (prefix_key, prefix_value):
        if t.dim() != 4:
            raise AttentionError(f"{op}: the prompts are [N, P, Hkv, D], got {list(t.shape)}")
        if t.dtype != key.dtype:
            raise AttentionError(f"{op}: the prompts and the caches share one dtype, got {t.dtype} and {key.dtype}")
    x = _lib.PrefixParams()
    x.n, x.p, x.hkv, x.d = prefix_key.shape
    x.v_n, x.v_p, x.v_hkv, x.v_d = prefix_value.shape
    x.k_stride = (ctypes.c_int64 * 4)(*prefix_key.stride())
    x.v_stride = (ctypes.c_int64 * 4)(*prefix_value.stride())
    if prefix_lengths is not None:
        if prefix_lengths.dim() != 1:
            raise AttentionError(f"{op}: the prompts' lengths are [N] = [{x.n}]")
        prefix_lengths = prefix_lengths.contiguous()
        x.lengths_elem_bytes = _index_bytes(prefix_lengths, f"{op}: the prompts' lengths")
        x.lengths, x.lengths_len = prefix_lengths.data_ptr(), prefix_lengths.shape[0]
    return x, prefix_lengths


def _step(op, query, new_key, new_value, prefix_key, prefix_value, key, value, cache_lengths, prefix_lengths, options):
    p, keep = make_decode_params(query, key, value, cache_lengths, options)
    x, prefix_lengths = _prefix_params(op, key, value, prefix_key, prefix_value, prefix_lengths)
    tensors = (query, prefix_key, prefix_value, key, value, new_key, new_value, prefix_lengths, *keep)
    _check_device(op, *tensors)
    for t in tensors:
        if t is not None and t.device != query.device:
            raise AttentionError(f"{op}: tensors of {query.device} and of {t.device}")
    if new_key is not None:
        want = (key.shape[0], key.shape[2], key.shape[3])
        for name, t in (("new_key", new_key), ("new_value", new_value)):
            if tuple(t.shape) != want or t.dtype != key.dtype:
                raise AttentionError(f"{op}: {name} must be {list(want)} of the cache's dtype, got {list(t.shape)} {t.dtype}")
        new_key, new_value = new_key.contiguous(), new_value.contiguous()
    lib = _lib.lib()
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    ws = _workspace(lib.dash_attn_decode_shared_workspace(ctypes.byref(p), ctypes.byref(x)), query.device)
    with _on(query.device):
        rc = lib.dash_attn_decode_shared(ctypes.byref(p), ctypes.byref(x), _ptr(query), _ptr(prefix_key), _ptr(prefix_value), _ptr(new_key), _ptr(new_value),
                                         _ptr(key), _ptr(value), _ptr(out), _ptr(ws), 0 if ws is None else ws.numel(), _stream(query.device))
    if rc != _lib.OK:
        _raise(rc)
    return out


def attention_decode_shared(query, prefix_key, prefix_value, key, value, cache_lengths: Optional[torch.Tensor] = None,
                            prefix_lengths: Optional[torch.Tensor] = None, options: AttentionOptions = AttentionOptions()):
    """``query [B,Hq,D]`` against its prompt's keys and, behind them, its own cache.

    ``prefix_key`` / ``prefix_value`` ``[N,P,Hkv,D]``: the prompts, of which ``prefix_lengths [N]`` rows are there (``None``: all ``P``);
    ``N`` divides ``B`` and sequence ``b`` continues prompt ``b // (B // N)``.  ``key`` / ``value`` ``[B,S,Hkv,D]`` and ``cache_lengths [B]``
    as for ``attention_decode``.  Of the options the scale and the window's ``left`` apply, which counts over both.  What lies
    past the lengths may be anything, NaN included; but under a window, rows of a prompt that some of its sequences see and others do not
    must be finite: a NaN or an infinity there may reach the others too."""
    done = _lib.binding().decode_shared(query, None, None, prefix_key, prefix_value, key, value, cache_lengths, prefix_lengths, options)
    if done is not None:
        return _result(done)
    return _step("attention_decode_shared", query, None, None, prefix_key, prefix_value, key, value, cache_lengths, prefix_lengths, options)


def attention_decode_shared_append(query, new_key, new_value, prefix_key, prefix_value, key, value, cache_lengths: torch.Tensor,
                                   prefix_lengths: Optional[torch.Tensor] = None, options: AttentionOptions = AttentionOptions()):
    """The same step with the new rows ``[B,Hkv,D]`` written into the sequences' own caches first, at ``cache_lengths`` (the lengths
    before the step; a full cache gets no row), as ``attention_decode_append`` does."""
    op = "attention_decode_shared_append"
    if new_key is not None and new_value is not None:
        done = _lib.binding().decode_shared(query, new_key, new_value, prefix_key, prefix_value, key, value, cache_lengths, prefix_lengths, options)
        if done is not None:
            return _result(done)
    if cache_lengths is None:
        raise AttentionError(f"{op}: the lengths are needed: they say where each sequence's new row goes")
    if new_key is None or new_value is None:
        raise AttentionError(f"{op}: a new row is null")
    return _step(op, query, new_key, new_value, prefix_key, prefix_value, key, value, cache_lengths, prefix_lengths, options)
