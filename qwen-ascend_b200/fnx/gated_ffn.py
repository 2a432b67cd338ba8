"""The bf16 gated feed-forward block, forward and backward, on ``libfnx_b200.so``.

The reference's deployment keeps its always-on shared expert in bf16: one concatenated gate/up
GEMM, ``silu(gate) * up``, the down projection (``fnx/engine.py:1786-1790``, weights concatenated
as in ``fnx/engine.py:1223-1236``).  ``GatedFFN`` is that block beside the W4 experts of
``engine.MoELayer``: both projections, the activation and the product in one kernel, and the
gradients of its input and weights for adapting it while the quantised experts stay frozen
(the reference does not train)."""
from __future__ import annotations

import torch

from . import _lib

BF16 = torch.bfloat16


def _rows(t, n, what, like):
    """``t [.., n]`` as bf16 rows the kernels can read: ``(2-D view or copy, row stride)``."""
    shape = t.shape
    if shape[-1] != n or t.device != like.device:
        raise ValueError(f"GatedFFN: {what} rows of {n} on {like.device} expected, got {tuple(shape)} on {t.device}")
    if t.dtype is not BF16:
        t = t.to(BF16)
    if len(shape) != 2:
        t = t.reshape(-1, n)
    ld, one = t.stride()
    if t.shape[0] < 2:
        ld = n
    if (one != 1 and n > 1) or ld % 8 or ld < n or t.data_ptr() % 16:
        t, ld = t.clone(memory_format=torch.contiguous_format), n
    return t, ld


class GatedFFN:
    """``y = (silu(x Wg^T) * (x Wu^T)) Wd^T`` with ``w_gu`` bf16 ``[2I, H]`` (gate rows, then up rows)
    and ``w_down`` bf16 ``[O, I]``; H, I and O are multiples of 8.  The weights are read in place, so
    an optimiser may update them between a backward and the next forward.

    ``__call__(x)``: ``[.., H] -> [.., O]``.  ``forward_train(x)`` also returns what the backward
    needs (``x``, ``h`` and the pre-activations in fp32), ``backward(dy, saved)`` the gradients.
    ``gated(x)`` is the first half alone, ``h [.., I]``.  No call is an autograd node: ``__call__`` and
    ``gated`` refuse an ``x`` that requires a gradient while gradients are recorded."""

    def __init__(self, w_gu, w_down):
        if (w_gu.dim() != 2 or w_down.dim() != 2 or w_gu.dtype != BF16 or w_down.dtype != BF16
                or w_gu.device != w_down.device or w_gu.shape[0] != 2 * w_down.shape[1]):
            raise ValueError("GatedFFN: bf16 w_gu [2I, H] and w_down [O, I] on one device expected")
        self.H, (self.O, self.I) = w_gu.shape[1], w_down.shape
        if min(self.H, self.I, self.O) < 8 or self.H % 8 or self.I % 8 or self.O % 8:
            raise ValueError(f"GatedFFN: H={self.H}, I={self.I}, O={self.O} must be multiples of 8")
        _lib.require_cuda(w_gu)
        if not w_gu.is_contiguous() or not w_down.is_contiguous() or (w_gu.data_ptr() | w_down.data_ptr()) % 16:
            raise ValueError("GatedFFN: weights must be contiguous and 16-byte aligned")
        self.w_gu, self.w_down = w_gu, w_down
        self._lib = _lib.lib()

    def _forward(self, x, keep, down):
        """``(x as rows, h, kept pre-activations, y)``."""
        dev = self.w_gu.device
        x2, ld = _rows(x, self.H, "input", self.w_gu)
        if _lib.elsewhere(x2):
            with torch.cuda.device(dev):
                return self._forward(x, keep, down)
        M = x2.shape[0]
        h = torch.empty(M, self.I, dtype=BF16, device=dev)
        y = torch.empty(M, self.O, dtype=BF16, device=dev) if down else None
        gu = torch.empty(self._lib.fnx_gated_ffn_saved_bytes(M, self.I), dtype=torch.uint8, device=dev) if keep else None
        rc = self._lib.fnx_gated_ffn(x2.data_ptr(), ld, self.w_gu.data_ptr(), self.w_down.data_ptr() if down else None,
                                     h.data_ptr(), _lib.ptr(gu), _lib.ptr(y), M, self.H, self.I, self.O,
                                     _lib.raw_stream(dev))
        _lib.check(rc, "gated feed-forward block")
        return x2, h, gu, y

    def __call__(self, x):
        if x.requires_grad:
            _lib.no_autograd("GatedFFN", x)
        y = self._forward(x, False, True)[3]
        return y if x.dim() == 2 else y.view(*x.shape[:-1], self.O)

    def gated(self, x):
        """``h = silu(x Wg^T) * (x Wu^T)``: ``[.., H] -> [.., I]``."""
        _lib.no_autograd("GatedFFN.gated", x)
        h = self._forward(x, False, False)[1]
        return h if x.dim() == 2 else h.view(*x.shape[:-1], self.I)

    def forward_train(self, x):
        """``(y, saved)``: ``saved`` is handed to ``backward``; it holds ``x`` itself, which must not
        be overwritten before, and ``8 * I`` bytes a row of pre-activations."""
        x2, h, gu, y = self._forward(x, True, True)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], self.O), (x2, h, gu, x.shape)

    def backward(self, dy, saved, need=(True, True, True)):
        """``(dx, dw_gu, dw_down)`` in bf16, ``None`` where ``need`` is false.  May be called again
        with the same ``saved``."""
        x2, h, gu, shape = saved
        M, dev = x2.shape[0], x2.device
        if x2.shape[1] != self.H or h.shape[1] != self.I or dev != self.w_gu.device:
            raise ValueError("GatedFFN.backward: saved comes from another block's forward_train")
        dy2, ld = _rows(dy, self.O, "gradient", self.w_gu)
        if dy2.shape[0] != M:
            raise ValueError(f"GatedFFN.backward: {dy2.shape[0]} rows for a forward of {M}")
        if _lib.elsewhere(x2):
            with torch.cuda.device(dev):
                return self.backward(dy, saved, need)
        dgu = torch.empty(M, 2 * self.I, dtype=BF16, device=dev)
        dx = torch.empty(M, self.H, dtype=BF16, device=dev) if need[0] else None
        dw_gu = torch.empty_like(self.w_gu) if need[1] else None
        dw_down = torch.empty_like(self.w_down) if need[2] else None
        rc = self._lib.fnx_gated_ffn_backward(dy2.data_ptr(), ld, x2.data_ptr(), x2.stride(0) if M > 1 else self.H,
                                              self.w_gu.data_ptr(), self.w_down.data_ptr(), h.data_ptr(), gu.data_ptr(),
                                              dgu.data_ptr(), _lib.ptr(dx), _lib.ptr(dw_gu), _lib.ptr(dw_down), M,
                                              self.H, self.I, self.O, _lib.raw_stream(dev))
        _lib.check(rc, "gated feed-forward gradients")
        return None if dx is None else dx.view(shape), dw_gu, dw_down
