"""Attention over a causal sliding window and a few first tokens that stay
visible (sinks): the window layers of a model whose other layers are elastic
(:class:`elastic_sparse_attention.ElasticSparseAttention`).  No counterpart in
the reference, whose only window is its layer 0.

The row at position p of a sequence whose first key is f sees key j when

    f <= j <= p  and  (p - j < window  or  j - f < num_sinks)

* :class:`SinkWindowAttention`, the module, with ElasticSparseAttention's
  calls: whole sequences (with gradients), chunks and decode rows against a
  cache (``cache_position``), grouped kv heads.
* :func:`sink_window_attention_fwd`, :func:`sink_window_attention_bwd`, the
  calls on tensors.

q is ``[B, H, Lq, D]``, k and v ``[B, Hkv, Lk, D]`` in bfloat16, float16 (D a
multiple of 8 up to 128) or float32 (of 4), any strides with a contiguous D.
Scores, softmax statistics and sums are float32; in 16-bit types the
probabilities enter the products rounded to the inputs' type.  Every call goes
through libesa.so's C ABI to hand-written gfx950 kernels; CPU tensors raise.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from elastic_sparse_attention import (_check_qkv, _dtype_code, _fwd_args, _prep, _require_gpu)
from esa_native import EsaBwdArgs, EsaWindow, check, load
from qk_norm_rope import _launch, _like, check_cache_position

__all__ = ["SinkWindowAttention", "sink_window_attention_fwd", "sink_window_attention_bwd"]


def _window(window: int, sinks: int, positions: Optional[torch.Tensor],
            first_key: Optional[torch.Tensor],
            residual: Optional[torch.Tensor] = None) -> EsaWindow:
    pos_ptr = pos_sb = 0
    if positions is not None:
        pos_ptr = positions.data_ptr()
        if positions.dim() == 2 and positions.shape[0] > 1:
            pos_sb = positions.stride(0)
    return EsaWindow(min(window, 0x7fffffff), min(sinks, 0x7fffffff), pos_ptr or None, pos_sb,
                     None if first_key is None else first_key.data_ptr(),
                     None if residual is None else residual.data_ptr())


def _check_window(window: int, sinks: int) -> None:
    if window < 1:
        raise ValueError(f"`window` ({window}) must be at least 1.")
    if sinks < 0:
        raise ValueError(f"`num_sinks` ({sinks}) must not be negative.")


def _first_keys(first_key, batch: int, device: torch.device) -> Optional[torch.Tensor]:
    """first_key as int64 ``[batch]`` on ``device``."""
    if first_key is None:
        return None
    f = first_key if isinstance(first_key, torch.Tensor) else torch.as_tensor(first_key)
    if f.dtype.is_floating_point or f.dtype.is_complex or f.dtype == torch.bool:
        raise ValueError(f"first_key must be integers, got {f.dtype}")
    if f.dim() != 1 or f.shape[0] != batch:
        raise ValueError(f"first_key must be [{batch}], got {list(f.shape)}")
    if f.dtype != torch.int64 or f.device != device:
        f = f.to(device=device, dtype=torch.int64)
    return f.contiguous()


def _checked(q, k, v, positions, first_key):
    """positions and first_key as the kernels take them (q, k, v having passed
    _check_qkv)."""
    if not (q.device == k.device == v.device):
        raise ValueError(f"q, k and v must share one device, got {q.device}, {k.device} and "
                         f"{v.device}")
    B, _, Lq, _ = q.shape
    kv_len = k.shape[2]
    if positions is None:
        if Lq > kv_len:
            raise ValueError(f"q_len ({Lq}) exceeds kv_len ({kv_len}) without positions")
    else:
        positions = check_cache_position(positions, B, Lq, kv_len, q.device)
    return positions, _first_keys(first_key, B, q.device)


def sink_window_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int,
                              num_sinks: int, scaling: float, positions=None, first_key=None,
                              return_lse: bool = True, return_residual: bool = False):
    """``o`` as ``[B, Lq, H, D]`` and, if asked, ``lse`` float32 ``[B, H, Lq]``
    (natural log).

    ``positions``: None (row r is position r) or the rows' places in the
    cache, ``[Lq]`` or ``[B, Lq]``, consecutive in each sequence (a host value
    is checked, a device tensor used as given: a row that breaks this, or lies
    outside the cache, gives NaN).  ``first_key``: None or int ``[B]``, the
    first key of each sequence (left padding); rows before it give 0 and
    lse -inf.  ``return_residual`` adds a third value for the backward: what
    rounding o to 16 bits lost (None for float32)."""
    _check_qkv(q, k, v)
    positions, first_key = _checked(q, k, v, positions, first_key)
    _check_window(window, num_sinks)
    got = _fwd(q, k, v, window, num_sinks, scaling, positions, first_key, return_lse,
               return_residual)
    return got if return_residual else got[:2]


# workspace bytes of the forward by its shape (a question to the library that
# a decode step need not ask again)
_WORKSPACE = {}


def _fwd(q, k, v, window, sinks, scaling, positions, first_key, return_lse, residual=False):
    """The forward after its checks (the module makes them itself): o, lse and,
    for a backward, what rounding o lost (None for float32)."""
    B, H, Lq, D = q.shape
    device = q.device
    align = 16 // q.element_size()
    o = torch.empty((B, Lq, H, D), dtype=q.dtype, device=device)
    lse = torch.empty((B, H, Lq), dtype=torch.float32, device=device) if return_lse else None
    res = torch.empty_like(o) if residual and o.dtype != torch.float32 else None
    if B == 0 or Lq == 0:
        return o, lse, res
    if k.shape[2] == 0:  # every row lies outside an empty cache
        o.fill_(float("nan"))
        return o, None if lse is None else lse.fill_(float("nan")), res
    q, k, v = _prep(q, align), _prep(k, align), _prep(v, align)
    a = _fwd_args(q, k, v, o, (Lq * H * D, D, H * D), lse, scaling)
    w = _window(window, sinks, positions, first_key, res)
    lib = load()
    key = (B, H, k.shape[1], Lq, k.shape[2], D, q.dtype, window, sinks, positions is None)
    n = _WORKSPACE.get(key)
    if n is None:
        ws = ctypes.c_size_t()
        check(lib.esa_sink_window_fwd_workspace_size(ctypes.byref(a), ctypes.byref(w),
                                                     ctypes.byref(ws)),
              "esa_sink_window_fwd_workspace_size")
        n = ws.value
        if len(_WORKSPACE) >= 4096:
            _WORKSPACE.clear()
        _WORKSPACE[key] = n
    work = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    _launch(device, "esa_sink_window_fwd", lib.esa_sink_window_fwd, ctypes.byref(a),
            ctypes.byref(w), work.data_ptr() if n else None, n)
    return o, lse, res


def sink_window_attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                              lse: torch.Tensor, dout: torch.Tensor, window: int, num_sinks: int,
                              scaling: float, positions=None, first_key=None,
                              o_residual: Optional[torch.Tensor] = None
                              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``dq``, ``dk``, ``dv`` in the inputs' shapes and dtype from the
    forward's ``o`` and ``dout`` ``[B, Lq, H, D]`` and ``lse``; sums in a fixed
    order, no atomics.  ``o_residual``: the forward's third value, with which
    dq and dk come out closer (rowsum(dout * o) from the o before its
    rounding); the module's backward has it."""
    _check_qkv(q, k, v)
    positions, first_key = _checked(q, k, v, positions, first_key)
    _check_window(window, num_sinks)
    B, H, Lq, D = q.shape
    if o.shape != (B, Lq, H, D) or dout.shape != (B, Lq, H, D) or lse.shape != (B, H, Lq):
        raise ValueError(f"o and dout must be [{B}, {Lq}, {H}, {D}] and lse [{B}, {H}, {Lq}]; got "
                         f"{list(o.shape)}, {list(dout.shape)} and {list(lse.shape)}")
    _require_gpu(o, lse, dout)
    if not (o.device == lse.device == dout.device == q.device):
        raise ValueError("o, lse and dout must be on q's device")
    if o.dtype != q.dtype or lse.dtype != torch.float32:
        raise ValueError("o must have q's dtype and lse float32, as the forward returns them")
    if o_residual is not None:
        if o_residual.shape != o.shape or o_residual.dtype != o.dtype or \
                o_residual.device != o.device:
            raise ValueError("o_residual must have o's shape, dtype and device")
        o, o_residual = _prep(o.contiguous(), 8), _prep(o_residual.contiguous(), 8)
    return _bwd(q, k, v, o, lse, dout, window, num_sinks, scaling, positions, first_key,
                o_residual)


def _rows_of(t: torch.Tensor, order=(0, 1, 2)):
    st = t.stride()
    return t.data_ptr(), st[order[0]], st[order[1]], st[order[2]]


def _bwd(q, k, v, o, lse, dout, window, sinks, scaling, positions, first_key, residual):
    """The backward after its checks (o contiguous where residual is given)."""
    B, H, Lq, D = q.shape
    dq, dk, dv = _like(q), _like(k), _like(v)
    if B == 0 or Lq == 0 or k.shape[2] == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()  # no query row reaches a key
    align = 16 // q.element_size()
    q, k, v, o = _prep(q, align), _prep(k, align), _prep(v, align), _prep(o, align)
    dout = _prep(dout if dout.dtype == q.dtype else dout.to(q.dtype), align)
    lse = lse.contiguous()
    bshd = (0, 2, 1)
    # in the order of esa_bwd_args' fields
    a = EsaBwdArgs(_dtype_code(q.dtype), B, H, k.shape[1], Lq, k.shape[2], D, *_rows_of(q),
                   *_rows_of(k), *_rows_of(v), *_rows_of(o, bshd), *_rows_of(dout, bshd),
                   *_rows_of(dq), *_rows_of(dk), *_rows_of(dv), lse.data_ptr(), lse.stride(0),
                   lse.stride(1), float(scaling))
    w = _window(window, sinks, positions, first_key, residual)
    lib = load()
    ws = ctypes.c_size_t()
    check(lib.esa_sink_window_bwd_workspace_size(ctypes.byref(a), ctypes.byref(w),
                                                 ctypes.byref(ws)),
          "esa_sink_window_bwd_workspace_size")
    n = ws.value
    work = torch.empty(n, dtype=torch.uint8, device=q.device)
    _launch(q.device, "esa_sink_window_bwd", lib.esa_sink_window_bwd, ctypes.byref(a),
            ctypes.byref(w), work.data_ptr(), n)
    return dq, dk, dv


class _SinkWindowFunction(torch.autograd.Function):
    """``apply(q, k, v, window, num_sinks, scaling, positions, first_key) ->
    o [B, Lq, H, D]``."""

    @staticmethod
    def forward(ctx, q, k, v, window, num_sinks, scaling, positions, first_key):
        o, lse, res = _fwd(q, k, v, window, num_sinks, scaling, positions, first_key, True, True)
        ctx.save_for_backward(q, k, v, o, lse, res, positions, first_key)
        ctx.window, ctx.num_sinks, ctx.scaling = window, num_sinks, scaling
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, res, positions, first_key = ctx.saved_tensors
        dq, dk, dv = _bwd(q, k, v, o, lse, do, ctx.window, ctx.num_sinks, ctx.scaling, positions,
                          first_key, res)
        return dq, dk, dv, None, None, None, None, None


class SinkWindowAttention(nn.Module):
    """A model's window layer.

    Args:
        num_attention_heads, head_dim, num_key_value_heads: as
            ElasticSparseAttention's; ``scaling = head_dim ** -0.5``, query
            head h reads kv head ``h // num_kv_groups``.
        window: keys a row sees, itself among them (one no shorter than the
            sequence makes the layer causal attention).
        num_sinks: first keys of a sequence that every later row sees too.
        rotary: a :class:`qk_norm_rope.QKNormRope` applied to queries and keys
            before the attention (see ``forward``).
    """

    def __init__(self, num_attention_heads: int, head_dim: int, window: int, num_sinks: int = 4,
                 num_key_value_heads: Optional[int] = None,
                 rotary: Optional[nn.Module] = None):
        super().__init__()
        _check_window(window, num_sinks)
        if head_dim < 4 or head_dim > 128 or head_dim % 4 != 0:
            raise ValueError(f"`head_dim` ({head_dim}) must be a multiple of 4 up to 128.")
        self.num_attention_heads = num_attention_heads
        self.head_dim = head_dim
        self.window = window
        self.num_sinks = num_sinks
        self.num_key_value_heads = (num_key_value_heads if num_key_value_heads is not None
                                    else num_attention_heads)
        if self.num_attention_heads % self.num_key_value_heads != 0:
            raise ValueError(
                f"`num_attention_heads` ({self.num_attention_heads}) must be divisible by "
                f"`num_key_value_heads` ({self.num_key_value_heads}) for GQA.")
        self.num_kv_groups = self.num_attention_heads // self.num_key_value_heads
        self.scaling = self.head_dim ** -0.5
        self.rotary = rotary

    def _check_heads(self, q: torch.Tensor, k: torch.Tensor) -> None:
        if q.shape[1] != self.num_attention_heads or k.shape[1] != self.num_key_value_heads \
                or q.shape[3] != self.head_dim:
            raise ValueError(
                f"expected {self.num_attention_heads} query heads and "
                f"{self.num_key_value_heads} key/value heads of {self.head_dim}; got "
                f"{q.shape[1]} and {k.shape[1]} of {q.shape[3]}")

    def forward(self, query_states: torch.Tensor, key_states: torch.Tensor,
                value_states: torch.Tensor, cache_position=None, first_key=None,
                kv_cache: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                ) -> Tuple[torch.Tensor, None]:
        """``(attn_output [B, Lq, H * D], None)``, as ElasticSparseAttention
        returns them.

        Without ``cache_position`` row r is position r.  With it (``[Lq]``, or
        ``[B, Lq]`` where every sequence has its own place; consecutive rows)
        the rows attend over the caches k and v.  ``first_key`` (int ``[B]``):
        each sequence's first key in a left-padded batch.

        A layer with ``rotary`` takes q, k, v as the projections leave them
        and norms and rotates q and k first; with ``kv_cache`` (the pair of
        caches ``[B, Hkv, Lmax, D]``) k and v are the new rows, which go into
        the caches at ``cache_position`` before the rows attend over them."""
        q, k, v = query_states, key_states, value_states
        _check_qkv(q, k, v)
        self._check_heads(q, k)
        if self.rotary is not None:
            first_key = _first_keys(first_key, q.shape[0], q.device)
            if kv_cache is not None and cache_position is not None:
                # (once for the append and the attention)
                cache_position = check_cache_position(cache_position, q.shape[0], q.shape[2],
                                                      kv_cache[0].shape[2], q.device)
            q, k, v = self.rotary.attention_rows(q, k, v, cache_position, kv_cache)
        elif kv_cache is not None:
            raise ValueError("kv_cache needs a layer with `rotary`")
        positions, first_key = _checked(q, k, v, cache_position, first_key)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            o = _SinkWindowFunction.apply(q, k, v, self.window, self.num_sinks, self.scaling,
                                          positions, first_key)
        else:
            o = _fwd(q, k, v, self.window, self.num_sinks, self.scaling, positions, first_key,
                     False)[0]
        B, Lq, H, D = o.shape
        return o.view(B, Lq, H * D), None
