"""The norm of every query and key head with the position rotation in the same pass.

A layer that norms its heads (root mean square over a head's features, one weight per feature for the queries and one for the keys)
does so right in front of the rotation: :class:`QkNorm` makes both one pass over the projection's output, forward and backward, through
the C ABI (``dash_rope_norm_apply``, ``dash_rope_norm_backward``).  It stands beside :class:`~dashmag_b200.rope.Rope` and takes the same
positions: a range, one position per sequence, sequences packed back to back.  Arithmetic is f32 and a result rounds once.
``dashmag_b200.autodiff`` has the same calls for tensors that may be tracked.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .attention import AttentionError, _check_device, _DTYPES, _index_bytes, _on, _ptr, _raise, _result, _stream, _workspace
from .rope import Rope


# Where a call's tokens are, as the native host side takes it.
_RANGE, _AT, _PACKED = 0, 1, 2


class QkNormGradients(NamedTuple):
    """The gradients of a call's query, key and weights (``None`` for a weight that is not there)."""
    query: torch.Tensor
    key: torch.Tensor
    query_weight: Optional[torch.Tensor]
    key_weight: Optional[torch.Tensor]


class QkNorm:
    """``rotate(x / sqrt(mean(x^2) + eps) * weight)`` of every head of a layer's query and key.

    ``rope`` rotates (its dtype is the tensors'); ``query_weight`` and ``key_weight`` are ``[D]``, in the tensors' dtype or f32, or
    ``None`` for ones.  Queries and keys may be slices of one projection's output: any strides are read in place as long as a
    head's features are contiguous."""

    def __init__(self, rope: Rope, query_weight: Optional[torch.Tensor] = None, key_weight: Optional[torch.Tensor] = None, eps: float = 1e-6):
        for name, w in (("query", query_weight), ("key", key_weight)):
            if w is not None and (w.dim() != 1 or w.dtype not in (rope.dtype, torch.float32)):
                raise AttentionError(f"qk_norm: the {name} weight is [D] in {rope.dtype} or torch.float32, got {w.dtype} {list(w.shape)}")
        if query_weight is not None and key_weight is not None and query_weight.dtype != key_weight.dtype:
            raise AttentionError(f"qk_norm: one dtype for both weights, got {query_weight.dtype} and {key_weight.dtype}")
        if not 0.0 <= eps < float("inf"):
            raise AttentionError(f"qk_norm: eps must be finite and >= 0, got {eps}")
        self.rope, self.query_weight, self.key_weight, self.eps = rope, query_weight, key_weight, eps

    # ------------------------------------------------------------------------------------------
    # Where the tokens are
    # ------------------------------------------------------------------------------------------
    def apply_range(self, query: torch.Tensor, key: torch.Tensor, positions: range):
        """``query [B,T,Hq,D]`` and ``key [B,T,Hkv,D]`` at the positions ``positions`` of every sequence, ``T`` of them."""
        if positions.step == 1:
            done = _lib.binding().norm(self.rope, query, key, self.query_weight, self.key_weight, self.eps, _RANGE, None, positions.start, positions.stop)
            if done is not None:
                return _result(done)
        return self._forward(query, key, self._range(query, key, positions))

    def apply_at(self, query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor):
        """``query [B,Hq,D]`` and ``key [B,Hkv,D]``, one token per sequence, at ``positions [B]``, integer.  One outside the tables
        gives NaN in the rotated features, as ``Rope.apply_at`` does."""
        done = _lib.binding().norm(self.rope, query, key, self.query_weight, self.key_weight, self.eps, _AT, positions, 0, 0)
        if done is not None:
            return _result(done)
        return self._forward(query, key, self._at(query, key, positions))

    def apply_packed(self, query: torch.Tensor, key: torch.Tensor, cu_seqlens: torch.Tensor, start: int = 0):
        """``[tokens,H,D]`` (or ``[1,tokens,H,D]``) of sequences packed back to back with the attention mask's offsets, every sequence
        from position ``start`` on; tokens of no sequence pass unchanged, neither normed nor rotated."""
        done = _lib.binding().norm(self.rope, query, key, self.query_weight, self.key_weight, self.eps, _PACKED, cu_seqlens, start, 0)
        if done is not None:
            return _result(done)
        return self._forward(query, key, self._packed(query, key, cu_seqlens, start))

    def backward_range(self, query, key, grad_query, grad_key, positions: range) -> QkNormGradients:
        """The gradients of ``apply_range``'s inputs from those of its outputs."""
        if positions.step == 1:
            done = _lib.binding().norm_backward(self.rope, query, key, grad_query, grad_key, self.query_weight, self.key_weight, self.eps, _RANGE, None,
                                                positions.start, positions.stop)
            if done is not None:
                return QkNormGradients(*_result(done))
        return self._backward(query, key, grad_query, grad_key, self._range(query, key, positions))

    def backward_at(self, query, key, grad_query, grad_key, positions: torch.Tensor) -> QkNormGradients:
        """The gradients of ``apply_at``'s inputs from those of its outputs."""
        done = _lib.binding().norm_backward(self.rope, query, key, grad_query, grad_key, self.query_weight, self.key_weight, self.eps, _AT, positions, 0, 0)
        if done is not None:
            return QkNormGradients(*_result(done))
        return self._backward(query, key, grad_query, grad_key, self._at(query, key, positions))

    def backward_packed(self, query, key, grad_query, grad_key, cu_seqlens: torch.Tensor, start: int = 0) -> QkNormGradients:
        """The gradients of ``apply_packed``'s inputs from those of its outputs."""
        done = _lib.binding().norm_backward(self.rope, query, key, grad_query, grad_key, self.query_weight, self.key_weight, self.eps, _PACKED, cu_seqlens,
                                            start, 0)
        if done is not None:
            return QkNormGradients(*_result(done))
        return self._backward(query, key, grad_query, grad_key, self._packed(query, key, cu_seqlens, start))

    # ------------------------------------------------------------------------------------------
    def _range(self, query, key, positions: range):
        if query.dim() != 4 or query.shape[1] != len(positions) or positions.step != 1 or positions.start < 0 or positions.stop > len(self.rope):
            raise AttentionError(f"Rope: positions {positions.start}..{positions.stop} of {len(self.rope)} for {list(query.shape)}")
        if key.dim() != 4 or key.shape[:2] != query.shape[:2]:
            raise AttentionError(f"Rope: {list(key.shape)} beside {list(query.shape)}")
        return {"start": positions.start, "stop": positions.stop}

    def _at(self, query, key, positions: torch.Tensor):
        if positions.dtype not in (torch.int32, torch.int64) or query.dim() != 3 or tuple(positions.shape) != (query.shape[0],):
            raise AttentionError(f"Rope: positions of {positions.dtype} {list(positions.shape)} for {list(query.shape)}")
        if key.dim() != 3 or key.shape[0] != query.shape[0]:
            raise AttentionError(f"Rope: {list(key.shape)} beside {list(query.shape)}")
        return {"positions": positions.contiguous()}

    def _packed(self, query, key, cu_seqlens: torch.Tensor, start: int):
        for x in (query, key):
            if x.dim() not in (3, 4) or x.dim() == 4 and x.shape[0] != 1:
                raise AttentionError(f"Rope: packed tokens are [tokens, H, D], got {list(x.shape)}")
        if query.shape[-3] != key.shape[-3]:
            raise AttentionError(f"Rope: {list(key.shape)} beside {list(query.shape)}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise AttentionError(f"Rope: the offsets are [S + 1], got {list(cu_seqlens.shape)}")
        _index_bytes(cu_seqlens, "Rope: the offsets")
        return {"cu_seqlens": cu_seqlens.contiguous(), "start": start}

    def _params(self, op, query, key, where, grads=()):
        """The parameters of a call and its tensors, the features of each contiguous."""
        rope = self.rope
        d = rope._check_features(query)
        if rope._check_features(key) != d:
            raise AttentionError(f"{op}: {list(query.shape)} and {list(key.shape)} must have one head dimension")
        for name, w in (("query", self.query_weight), ("key", self.key_weight)):
            if w is not None and w.shape[0] != d:
                raise AttentionError(f"{op}: the {name} weight is [D] = [{d}], got {list(w.shape)}")
        for name, g, x in zip(("query", "key"), grads, (query, key)):
            if g.shape != x.shape or g.dtype != x.dtype:
                raise AttentionError(f"{op}: the {name}'s gradient is {list(x.shape)} of {x.dtype}, got {list(g.shape)} of {g.dtype}")
        index = where.get("positions", where.get("cu_seqlens"))
        weights = [w if w is None else w.detach().contiguous() for w in (self.query_weight, self.key_weight)]
        _check_device(op, query, key, rope.cos, index, *weights, *grads)
        for t in (key, rope.cos, index, *weights, *grads):
            if t is not None and t.device != query.device:
                raise AttentionError(f"{op}: tensors of {query.device} and of {t.device}")
        tensors = [t if t.stride(-1) == 1 or d == 1 else t.contiguous() for t in (query, key, *grads)]
        p = _lib.QkNormParams()
        p.b, p.t = (query.shape[0], query.shape[1]) if query.dim() == 4 else (1, query.shape[0])
        p.d, p.heads_q, p.heads_k, p.eps = d, query.shape[-2], key.shape[-2], self.eps
        for name, t in zip(("q_stride", "k_stride", "grad_q_stride", "grad_k_stride"), tensors):
            setattr(p, name, (ctypes.c_int64 * 3)(t.stride(0) if t.dim() == 4 else 0, t.stride(-3), t.stride(-2)))
        given = [w for w in weights if w is not None]
        p.weight_dtype = int(_DTYPES[given[0].dtype if given else query.dtype])
        if "positions" in where:
            p.positions, p.positions_elem_bytes = _ptr(index), index.element_size()
        elif "cu_seqlens" in where:
            p.cu_seqlens, p.cu_seqlens_len, p.index_elem_bytes = _ptr(index), index.numel(), index.element_size()
        p.start = where.get("start", 0)
        return p, tensors, weights

    @staticmethod
    def _native(where):
        """``where`` as the native host side takes it."""
        form = _AT if "positions" in where else _PACKED if "cu_seqlens" in where else _RANGE
        return form, where.get("positions", where.get("cu_seqlens")), where.get("start", 0), where.get("stop", 0)

    def forward_of(self, query, key, where):
        """The forward of a call that has been checked (``autodiff``'s node)."""
        done = _lib.binding().norm(self.rope, query, key, self.query_weight, self.key_weight, self.eps, *self._native(where))
        return _result(done) if done is not None else self._forward(query, key, where)

    def backward_of(self, query, key, grad_query, grad_key, where):
        """Its gradients."""
        done = _lib.binding().norm_backward(self.rope, query, key, grad_query, grad_key, self.query_weight, self.key_weight, self.eps, *self._native(where))
        return QkNormGradients(*_result(done)) if done is not None else self._backward(query, key, grad_query, grad_key, where)

    def _forward(self, query, key, where):
        p, (query, key), (wq, wk) = self._params("qk_norm", query, key, where)
        out_q, out_k = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (query, key))
        tables = self.rope.tables()
        with _on(query.device):
            rc = _lib.lib().dash_rope_norm_apply(ctypes.byref(tables), ctypes.byref(p), _ptr(query), _ptr(key), _ptr(wq), _ptr(wk), _ptr(out_q), _ptr(out_k),
                                               _stream(query.device))
        if rc != _lib.OK:
            _raise(rc)
        return out_q, out_k

    def _backward(self, query, key, grad_query, grad_key, where) -> QkNormGradients:
        p, (query, key, grad_query, grad_key), (wq, wk) = self._params("qk_norm_backward", query, key, where, (grad_query, grad_key))
        dq, dk = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (query, key))
        dwq, dwk = (None if w is None else torch.empty_like(w) for w in (wq, wk))
        lib = _lib.lib()
        ws = _workspace(lib.dash_rope_norm_backward_workspace(ctypes.byref(p)), query.device)
        tables = self.rope.tables()
        with _on(query.device):
            rc = lib.dash_rope_norm_backward(ctypes.byref(tables), ctypes.byref(p), _ptr(query), _ptr(key), _ptr(wq), _ptr(wk), _ptr(grad_query),
                                           _ptr(grad_key), _ptr(dq), _ptr(dk), _ptr(dwq), _ptr(dwk), _ptr(ws), 0 if ws is None else ws.numel(),
                                           _stream(query.device))
        if rc != _lib.OK:
            _raise(rc)
        return QkNormGradients(dq, dk, dwq, dwk)
