"""Residual injection (``fnx/native_inject.py`` of the reference): ``hyper + y * inj`` over the
hyper-connection branches with the intermediate bf16 rounding, on ``libfnx_b200.so``
(``fnx_inject_ex``; the reference's AscendC shim ``fnx_inject`` is exported too).

``inject(hyper, gate, values)`` keeps the reference's signature and its ``None``-for-unsupported
convention: ``hyper`` bf16 ``[b, 1, HC*H]``, ``gate`` bf16 ``[b, 1, HC]``, ``values`` bf16
``[b, 1, H]`` (any batch and width here; the AscendC kernel took one token at H=2560).

``inject_norm`` / ``inject_norm_backward`` run the residual step between two blocks together with
the norms on both sides of it, and its gradients (``fnx_inject_norm``, ``fnx_inject_norm_backward``).
"""
from __future__ import annotations

import torch

from . import _lib


def inject(hyper, gate, values):
    b = hyper.shape[0]
    if b < 1 or values.numel() % b or gate.numel() % b:
        return None
    H, HC = values.numel() // b, gate.numel() // b
    if hyper.numel() != b * HC * H or H % 8 or HC > 64:
        return None
    if any(t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != hyper.device
           for t in (hyper, gate, values)) or hyper.device.type != "cuda":
        return None
    output = torch.empty_like(hyper)
    rc = _lib.lib().fnx_inject_ex(hyper.data_ptr(), values.data_ptr(), gate.data_ptr(), output.data_ptr(), b, H, HC,
                                  _lib.stream(hyper.device))
    if rc:
        raise RuntimeError(f"residual injection launch rejected: {rc}")
    return output


def _inject_norm_args(hyper, gate, values, w_next, w_post):
    """Checks shared by the two directions -> ``(b, H, HC)``."""
    b = hyper.shape[0]
    H = values.shape[-1]
    if values.numel() != b * H or H < 1 or hyper.shape[-1] % H or hyper.numel() != b * hyper.shape[-1]:
        raise ValueError(f"inject_norm: hyper {tuple(hyper.shape)} and values {tuple(values.shape)} are not "
                         "[b, 1, HC*H] and [b, 1, H]")
    HC = hyper.shape[-1] // H
    if H % 8 or H > 16384 or HC > 4 or (HC + 2) * H > 56000:
        raise ValueError(f"inject_norm: H={H}, HC={HC}: H must be a multiple of 8 up to 16384, HC at most 4 and "
                         "(HC + 2) * H at most 56000")
    for name, t, n in (("gate", gate, b * HC), ("w_next", w_next, HC * H), ("w_post", w_post, H)):
        if t is not None and t.numel() != n:
            raise ValueError(f"inject_norm: {name} holds {t.numel()} values, {n} expected")
    for t in (hyper, gate, values, w_next, w_post):
        if t is not None and (t.dtype != torch.bfloat16 or t.device != hyper.device):
            raise ValueError("inject_norm: bf16 tensors on one device expected")
    _lib.require_cuda(hyper)
    return b, H, HC


@_lib.on_device
def inject_norm(hyper, gate, values, w_next=None, *, w_post=None, scale=1.0, eps=1e-6):
    """``state = hyper + scale * gate * z`` per branch with ``z = values`` (or its rms norm times
    ``1 + w_post``), and ``normed``, the rms norm of every branch of ``state`` times ``1 + w_next``
    (``None`` without ``w_next``): the residual inject after a block and the norm that opens the next
    one (``inject`` then the first step of ``engine.gated_residual``) in one pass.  ``hyper`` bf16
    ``[b, 1, HC*H]``, ``gate`` bf16 ``[b, 1, HC]`` or ``None`` (1), ``values`` bf16 ``[b, 1, H]``,
    ``w_next`` ``[HC*H]``, ``w_post`` ``[H]``; HC = 1 is an ordinary residual stream.  Returns
    ``(state, normed)`` shaped like ``hyper``.  fp32 inside, each output rounded once; ``normed``
    comes from the unrounded state, so it can differ by one rounding from a norm of ``state``."""
    b, H, HC = _inject_norm_args(hyper, gate, values, w_next, w_post)
    hyper, values = hyper.contiguous(), values.contiguous()
    gate, w_next, w_post = (None if t is None else t.contiguous() for t in (gate, w_next, w_post))
    state = torch.empty_like(hyper)
    normed = None if w_next is None else torch.empty_like(hyper)
    rc = _lib.lib().fnx_inject_norm(hyper.data_ptr(), _lib.ptr(gate), values.data_ptr(), _lib.ptr(w_post),
                                    _lib.ptr(w_next), state.data_ptr(), _lib.ptr(normed), b, H, HC, scale, eps,
                                    _lib.stream(hyper.device))
    _lib.check(rc, "residual injection with norms")
    return state, normed


@_lib.on_device
def inject_norm_backward(d_state, d_normed, state, gate, values, w_next=None, *, w_post=None, scale=1.0, eps=1e-6):
    """Gradients of ``inject_norm`` from the gradients of its outputs (either may be ``None``: zero),
    the ``state`` it returned and its inputs: ``(d_hyper, d_gate, d_values, d_w_next, d_w_post)``,
    bf16 in the inputs' shapes, ``None`` where the input was ``None``.  Deterministic."""
    b, H, HC = _inject_norm_args(state, gate, values, w_next, w_post)
    if d_state is None and d_normed is None:
        raise ValueError("inject_norm_backward: d_state or d_normed needed")
    if d_normed is not None and w_next is None:
        raise ValueError("inject_norm_backward: d_normed without w_next")
    for t in (d_state, d_normed):
        if t is not None and (t.numel() != state.numel() or t.dtype != torch.bfloat16 or t.device != state.device):
            raise ValueError("inject_norm_backward: gradients must be bf16, shaped and placed like state")
    d_state, d_normed, gate_c, w_next_c, w_post_c = (None if t is None else t.contiguous()
                                                     for t in (d_state, d_normed, gate, w_next, w_post))
    state, values_c = state.contiguous(), values.contiguous()
    d_hyper = torch.empty_like(state)
    new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)      # noqa: E731
    d_gate, d_values, d_w_next, d_w_post = new(gate), new(values), new(w_next), new(w_post)
    L = _lib.lib()
    nws = L.fnx_inject_norm_backward_workspace(b, H, HC)
    ws = torch.empty(nws, dtype=torch.uint8, device=state.device)
    rc = L.fnx_inject_norm_backward(_lib.ptr(d_state), _lib.ptr(d_normed), state.data_ptr(), _lib.ptr(gate_c),
                                    values_c.data_ptr(), _lib.ptr(w_post_c), _lib.ptr(w_next_c), d_hyper.data_ptr(),
                                    _lib.ptr(d_gate), d_values.data_ptr(), _lib.ptr(d_w_post), _lib.ptr(d_w_next),
                                    b, H, HC, scale, eps, ws.data_ptr(), nws, _lib.stream(state.device))
    _lib.check(rc, "gradient of the residual injection with norms")
    return d_hyper, d_gate, d_values, d_w_next, d_w_post
