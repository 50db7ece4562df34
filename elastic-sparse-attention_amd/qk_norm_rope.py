"""Norm of each head's queries and keys with their position rotation, in one
pass (no counterpart in the reference, whose layer takes q and k as its caller
prepared them): what stands between a model's projections and its attention
layers.

    y = R(p) (x / sqrt(mean(x^2) + eps) * weight)        for every head's row x

R(p) turns pair i of the first ``rotary_dim`` elements by the angle
``p * inv_freq[i]``: elements (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with
``interleaved``.  Angles are formed in float64 on the device, the rest is
float32, rounded once to the inputs' type.

* :class:`QKNormRope`, the module: ``forward`` for whole sequences (with
  gradients), ``append`` for new rows of sequences that keep caches.  Both
  attention modules take one as ``rotary``.
* :func:`qk_norm_rope_fwd`, :func:`qk_norm_rope_bwd`,
  :func:`qk_norm_rope_append`, the calls on tensors.

q is ``[B, H, n, D]`` and k ``[B, Hkv, n, D]``, of any strides with a
contiguous D (views of one fused projection ``[B, n, (H + 2 Hkv) D]`` are read
in place), in bfloat16, float16 or float32; D is a multiple of 4 up to 256 and
``rotary_dim`` one of 8.  Every call goes through libesa.so's C ABI to
hand-written gfx950 kernels; CPU tensors raise.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from elastic_sparse_attention import _dtype_code, _prep, _require_gpu, _stream
from esa_native import EsaRotaryArgs, check, load

__all__ = ["QKNormRope", "qk_norm_rope_fwd", "qk_norm_rope_bwd", "qk_norm_rope_append"]


_GET_DEVICE = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(device: torch.device, what: str, fn, *args) -> None:
    """``fn(*args, stream)`` on the device's current stream, the device made
    current where it is another one (a launch goes to the current device)."""
    index = device.index
    if index is None or index == _GET_DEVICE():
        status = fn(*args, _stream(device))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _stream(device))
    if status:
        check(status, what)


def _like(t: torch.Tensor) -> torch.Tensor:
    """An empty tensor of t's shape, its heads and rows in t's order in
    memory."""
    B, H, n, D = t.shape
    if t.stride(1) < t.stride(2):
        return torch.empty(B, n, H, D, dtype=t.dtype, device=t.device).transpose(1, 2)
    return torch.empty(B, H, n, D, dtype=t.dtype, device=t.device)


def _check_qk(q: torch.Tensor, k: torch.Tensor) -> None:
    _require_gpu(q, k)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must be 4-D [B, heads, seq, head_dim]")
    qs, ks = q.shape, k.shape
    if qs[0] != ks[0] or qs[2] != ks[2] or qs[3] != ks[3]:
        raise ValueError(f"query {tuple(qs)} and key {tuple(ks)} disagree on batch, rows or "
                         "head_dim")
    if qs[1] < 1 or ks[1] < 1:
        raise ValueError("q and k need at least one head")
    if q.dtype != k.dtype:
        raise ValueError("q and k must share one dtype")
    if q.device != k.device:
        raise ValueError(f"q and k must share one device, got {q.device} and {k.device}")


def _positions_2d(positions, batch: int, rows: int, device: torch.device) -> torch.Tensor:
    """positions as int64 on ``device``: [rows] (shared) or [batch, rows]; None
    is row r at position r (formed for the call: nothing is kept that another
    stream, or a graph's memory, would have to have finished first)."""
    if positions is None:
        return torch.arange(rows, device=device)
    if not isinstance(positions, torch.Tensor):
        positions = torch.as_tensor(positions)
    pos = positions
    if pos.dtype.is_floating_point or pos.dtype.is_complex or pos.dtype == torch.bool:
        raise ValueError(f"positions must be integers, got {pos.dtype}")
    if pos.dim() == 0:
        pos = pos.reshape(1)
    if tuple(pos.shape) not in ((rows,), (batch, rows), (1, rows)):
        raise ValueError(f"positions must be [{rows}] or [{batch}, {rows}], got "
                         f"{list(pos.shape)}")
    if pos.dtype != torch.int64 or pos.device != device:
        pos = pos.to(device=device, dtype=torch.int64)
    return pos if pos.stride(-1) == 1 or rows <= 1 else pos.contiguous()


def _weights(q_weight, k_weight, D: int, device: torch.device):
    """The gains, contiguous and of one type."""
    out = []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if w.dim() != 1 or w.shape[0] != D:
                raise ValueError(f"{name} must be [{D}], got {list(w.shape)}")
            if w.device != device:
                raise ValueError(f"{name} is on {w.device}, the rows are on {device}")
            w = w.detach() if w.is_contiguous() else w.detach().contiguous()
        out.append(w)
    qw, kw = out
    if qw is not None and kw is not None and qw.dtype != kw.dtype:
        raise ValueError("q_weight and k_weight must share one dtype")
    return qw, kw


_NO_TENSOR = (None, 0, 0, 0)


def _rows_of(t: Optional[torch.Tensor]):
    """Address and (b, h, s) strides, in the order of esa_rotary_args."""
    if t is None:
        return _NO_TENSOR
    st = t.stride()
    return t.data_ptr(), st[0], st[1], st[2]


def _rotary_args(q, k, v, q_out, k_out, v_out, q_grad, k_grad, q_weight, k_weight, inv_freq, pos,
                 eps, interleaved, kv_len=0, dq_weight=None, dk_weight=None) -> EsaRotaryArgs:
    B, H, n, D = q.shape
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or inv_freq.device != q.device \
            or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous 1-D float64 tensor on the rows' device")
    code = _dtype_code(q.dtype)
    w = q_weight if q_weight is not None else k_weight
    # in the order of esa_rotary_args' fields
    return EsaRotaryArgs(
        code, code if w is None else _dtype_code(w.dtype), B, H, k.shape[1], n, D,
        2 * inv_freq.shape[0], 1 if interleaved else 0, kv_len, eps,
        None if q_weight is None else q_weight.data_ptr(),
        None if k_weight is None else k_weight.data_ptr(), inv_freq.data_ptr(), pos.data_ptr(),
        pos.stride(0) if pos.dim() == 2 and pos.shape[0] > 1 else 0,
        *_rows_of(q), *_rows_of(k), *_rows_of(v), *_rows_of(q_out), *_rows_of(k_out),
        *_rows_of(v_out), *_rows_of(q_grad), *_rows_of(k_grad),
        None if dq_weight is None else dq_weight.data_ptr(),
        None if dk_weight is None else dk_weight.data_ptr())


def _align(t: torch.Tensor) -> int:
    """Elements whose alignment lets any rotation read t's rows."""
    n = 16 // t.element_size()
    return n if t.shape[-1] % n == 0 else 4


def qk_norm_rope_fwd(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                     k_weight: Optional[torch.Tensor], inv_freq: torch.Tensor, positions,
                     eps: float = 1e-6, interleaved: bool = False
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """q and k normed and rotated: new tensors of their shapes and dtype.

    ``positions``: int64 ``[n]`` (shared by the batch) or ``[B, n]``, any
    values, or None (row r is position r); ``inv_freq``: float64 ``[rotary_dim / 2]`` on the rows' device,
    radians per position; a weight of None is 1."""
    _check_qk(q, k)
    B, _, n, D = q.shape
    pos = _positions_2d(positions, B, n, q.device)
    qw, kw = _weights(q_weight, k_weight, D, q.device)
    qo, ko = _like(q), _like(k)
    align = _align(q)
    a = _rotary_args(_prep(q, align), _prep(k, align), None, qo, ko, None, None, None, qw, kw,
                     inv_freq, pos, eps, interleaved)
    _launch(q.device, "esa_qk_norm_rope_fwd", load().esa_qk_norm_rope_fwd, ctypes.byref(a))
    return qo, ko


def qk_norm_rope_bwd(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                     k_weight: Optional[torch.Tensor], inv_freq: torch.Tensor, positions,
                     dq_out: torch.Tensor, dk_out: torch.Tensor, eps: float = 1e-6,
                     interleaved: bool = False, weight_grads: bool = True):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of :func:`qk_norm_rope_fwd`
    for the outputs' gradients ``dq_out`` and ``dk_out``; the weights' are sums
    over every row in a fixed order (None for a weight of None, or without
    ``weight_grads``)."""
    _check_qk(q, k)
    B, _, n, D = q.shape
    if dq_out.shape != q.shape or dk_out.shape != k.shape:
        raise ValueError(f"gradients {tuple(dq_out.shape)} and {tuple(dk_out.shape)} do not "
                         f"match q {tuple(q.shape)} and k {tuple(k.shape)}")
    _require_gpu(dq_out, dk_out)
    pos = _positions_2d(positions, B, n, q.device)
    qw, kw = _weights(q_weight, k_weight, D, q.device)
    dq, dk = _like(q), _like(k)
    dqw = torch.empty_like(qw) if weight_grads and qw is not None else None
    dkw = torch.empty_like(kw) if weight_grads and kw is not None else None
    if B == 0 or n == 0:  # no rows: nothing is launched
        return dq, dk, *(None if w is None else w.zero_() for w in (dqw, dkw))
    align = _align(q)
    q, k = _prep(q, align), _prep(k, align)
    gq, gk = (_prep(g.to(device=q.device, dtype=q.dtype), align) for g in (dq_out, dk_out))
    a = _rotary_args(q, k, None, dq, dk, None, gq, gk, qw, kw, inv_freq, pos, eps, interleaved, 0,
                     dqw, dkw)
    lib = load()
    ws = ctypes.c_size_t()
    check(lib.esa_qk_norm_rope_bwd_workspace_size(ctypes.byref(a), ctypes.byref(ws)),
          "esa_qk_norm_rope_bwd_workspace_size")
    work = torch.empty(max(ws.value, 16), dtype=torch.uint8, device=q.device)
    _launch(q.device, "esa_qk_norm_rope_bwd", lib.esa_qk_norm_rope_bwd, ctypes.byref(a),
            work.data_ptr(), work.numel())
    return dq, dk, dqw, dkw


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        k_cache: torch.Tensor, v_cache: torch.Tensor,
                        q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                        inv_freq: torch.Tensor, cache_position, eps: float = 1e-6,
                        interleaved: bool = False) -> torch.Tensor:
    """New rows of sequences that keep caches ``[B, Hkv, Lmax, D]``: k normed
    and rotated into ``k_cache``, v as it is into ``v_cache``, at
    ``cache_position`` (``[n]`` or ``[B, n]``); returns q normed and rotated.

    The rows of a sequence follow each other: row s sits at the sequence's
    first position + s (a negative position counts from Lmax).  A host-side
    ``cache_position`` is checked (IndexError, ValueError); a device tensor is
    used as given: a row at any other position, or outside the cache, leaves
    the caches alone and gets a NaN query.  The caches are written in place."""
    _check_qk(q, k)
    _require_gpu(v, k_cache, v_cache)
    B, _, n, D = q.shape
    Hkv = k.shape[1]
    align = _align(q)
    if v.shape != k.shape:
        raise ValueError(f"key {tuple(k.shape)} and value {tuple(v.shape)} shapes differ")
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        cs, st = c.shape, c.stride()
        if len(cs) != 4 or cs[0] != B or cs[1] != Hkv or cs[3] != D:
            raise ValueError(f"{name} must be [{B}, {Hkv}, Lmax, {D}], got {list(cs)}")
        if c.dtype != q.dtype or c.device != q.device:
            raise ValueError(f"{name} must have the rows' dtype and device")
        if 0 in st and any(x == 0 and m > 1 for x, m in zip(st, cs)):
            raise ValueError(f"{name} is an expanded view: its rows share memory")
        if st[3] != 1 or (st[0] | st[1] | st[2]) & (align - 1) or \
                c.data_ptr() % (align * c.element_size()):
            raise ValueError(f"{name} is written in place: its rows must be contiguous and "
                             f"aligned to {align * c.element_size()} bytes")
    if k_cache.shape[2] != v_cache.shape[2]:
        raise ValueError("k_cache and v_cache differ in length")
    if v.dtype != q.dtype or v.device != q.device:
        raise ValueError("v must have the rows' dtype and device")
    Lmax = k_cache.shape[2]
    pos = check_cache_position(cache_position, B, n, Lmax, q.device)
    qw, kw = _weights(q_weight, k_weight, D, q.device)
    qo = _like(q)
    if B == 0 or n == 0:
        return qo
    if Lmax == 0:
        return qo.fill_(float("nan"))
    a = _rotary_args(_prep(q, align), _prep(k, align), _prep(v, align), qo, k_cache, v_cache, None,
                     None, qw, kw, inv_freq, pos, eps, interleaved, Lmax)
    _launch(q.device, "esa_qk_norm_rope_append", load().esa_qk_norm_rope_append, ctypes.byref(a))
    return qo


def check_cache_position(cache_position, batch: int, rows: int, kv_len: int,
                         device: torch.device) -> torch.Tensor:
    """cache_position as int64 on ``device``, ``[rows]`` or ``[batch, rows]``.
    A host-side value is checked: IndexError outside the cache, ValueError
    where a sequence's rows do not follow each other."""
    if cache_position is None:
        raise ValueError("cache_position must say where the rows are")
    on_gpu = isinstance(cache_position, torch.Tensor) and cache_position.is_cuda
    if not on_gpu:
        pos = _positions_2d(cache_position, batch, rows, torch.device("cpu"))
        if bool(((pos < -kv_len) | (pos >= kv_len)).any()):
            raise IndexError(f"cache_position out of range for kv_len {kv_len}")
        at = torch.where(pos < 0, pos + kv_len, pos)
        if rows > 1 and bool((at[..., 1:] != at[..., :-1] + 1).any()):
            raise ValueError("cache_position: a sequence's rows must follow each other")
        return pos.to(device)
    return _positions_2d(cache_position, batch, rows, device)


class _QKNormRopeFunction(torch.autograd.Function):
    """``apply(q, k, q_weight, k_weight, inv_freq, positions, eps,
    interleaved) -> (q', k')``."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, inv_freq, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return qk_norm_rope_fwd(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, qw, kw, inv_freq, positions = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dqw, dkw = qk_norm_rope_bwd(q, k, qw, kw, inv_freq, positions, gq, gk, ctx.eps,
                                            ctx.interleaved, need[2] or need[3])
        return dq, dk, dqw, dkw, None, None, None, None


class QKNormRope(nn.Module):
    """Norm of each head's queries and keys with their position rotation.

    Args:
        head_dim: elements of a head.
        rotary_dim: its first elements that are rotated (all by default).
        base: the angle of pair i at position p is ``p * base ** (-2 i /
            rotary_dim)``; assign :attr:`inv_freq` (float64
            ``[rotary_dim / 2]``) for other frequencies.
        eps: added to the mean square.
        interleaved: pairs are neighbours instead of halves.

    ``q_weight`` and ``k_weight`` (``[head_dim]``, ones) are the gains.
    """

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0,
                 eps: float = 1e-6, interleaved: bool = False):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 4 or head_dim > 256 or head_dim % 4 != 0:
            raise ValueError(f"`head_dim` ({head_dim}) must be a multiple of 4 up to 256.")
        if rotary_dim < 8 or rotary_dim > head_dim or rotary_dim % 8 != 0:
            raise ValueError(f"`rotary_dim` ({rotary_dim}) must be a multiple of 8 from 8 to "
                             f"`head_dim` ({head_dim}).")
        if not base > 0.0:
            raise ValueError(f"`base` ({base}) must be positive.")
        if not eps >= 0.0:
            raise ValueError(f"`eps` ({eps}) must not be negative.")
        self.head_dim = head_dim
        self.rotary_dim = rotary_dim
        self.base = base
        self.eps = eps
        self.interleaved = interleaved
        self.q_weight = nn.Parameter(torch.ones(head_dim))
        self.k_weight = nn.Parameter(torch.ones(head_dim))
        half = rotary_dim // 2
        inv_freq = base ** (-torch.arange(half, dtype=torch.float64) / half)
        self.register_buffer("inv_freq", inv_freq, persistent=False)

    def _apply(self, fn, *args, **kwargs):
        # the frequencies stay float64 under .half(), .bfloat16() and .to(dtype):
        # they follow the module's device alone
        freq = self.inv_freq
        super()._apply(fn, *args, **kwargs)
        moved = self._buffers["inv_freq"]
        if moved.dtype != torch.float64:
            self._buffers["inv_freq"] = freq.to(moved.device)
        return self

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions=None
                ) -> Tuple[torch.Tensor, torch.Tensor]:
        """q ``[B, H, n, D]`` and k ``[B, Hkv, n, D]`` normed and rotated at
        ``positions`` (``[n]`` or ``[B, n]``; None: row r is position r)."""
        self._check_dim(q)
        positions = _positions_2d(positions, q.shape[0], q.shape[2], q.device)
        if torch.is_grad_enabled() and any(
                t.requires_grad for t in (q, k, self.q_weight, self.k_weight)):
            return _QKNormRopeFunction.apply(q, k, self.q_weight, self.k_weight, self.inv_freq,
                                             positions, self.eps, self.interleaved)
        return qk_norm_rope_fwd(q, k, self.q_weight, self.k_weight, self.inv_freq, positions,
                                self.eps, self.interleaved)

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
               v_cache: torch.Tensor, cache_position) -> torch.Tensor:
        """:func:`qk_norm_rope_append` with the module's weights: keys and
        values into the caches, queries returned.  Not differentiable."""
        self._check_dim(q)
        if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
            raise ValueError("append writes caches in place and has no gradient: call it under "
                             "torch.no_grad(), or use forward")
        return qk_norm_rope_append(q, k, v, k_cache, v_cache, self.q_weight, self.k_weight,
                                   self.inv_freq, cache_position, self.eps, self.interleaved)

    def attention_rows(self, q, k, v, cache_position, kv_cache):
        """What an attention layer with this module as its ``rotary`` attends
        over: q and k normed and rotated at their rows' places or, with
        ``kv_cache`` (the pair of caches), q and the caches after
        :meth:`append`."""
        if kv_cache is None:
            if cache_position is not None:
                raise ValueError("a layer with `rotary` takes cache_position together with "
                                 "kv_cache: its k and v are the new rows")
            q, k = self(q, k)
            return q, k, v
        if cache_position is None:
            raise ValueError("kv_cache needs cache_position")
        k_cache, v_cache = kv_cache
        return self.append(q, k, v, k_cache, v_cache, cache_position), k_cache, v_cache

    def _check_dim(self, q: torch.Tensor) -> None:
        if q.dim() != 4 or q.shape[-1] != self.head_dim:
            raise ValueError(f"expected q [B, heads, rows, {self.head_dim}], got "
                             f"{list(q.shape)}")
