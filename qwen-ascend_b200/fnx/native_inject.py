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

BF16 = torch.bfloat16


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


def _in_order(t, *dims):
    """Whether ``t`` holds the values of an array ``dims`` in its order: axes merged, axes of length 1
    added or the first axis split, but none exchanged."""
    inner, at = 1, {1}
    for d in dims[:0:-1]:
        inner *= d
        at.add(inner)
    at.add(inner * dims[0])
    n, cuts = 1, []
    for d in t.shape[:0:-1]:
        n *= d
        cuts.append(n)
    return all(c in at or (c % inner == 0 and (inner == 1 or inner in cuts)) for c in cuts)


def _inject_norm_args(hyper, gate, values, w_next, w_post, eps, grads=()):
    """Checks shared by the two directions -> ``(b, H, HC, whether a tensor has to be packed,
    device index)``."""
    hs, vs = hyper.shape, values.shape
    b, W, H = hs[0], hs[-1], vs[-1]
    if H < 1 or W % H or values.numel() != b * H or hyper.numel() != b * W:
        raise ValueError(f"inject_norm: hyper {tuple(hs)} and values {tuple(vs)} are not [b, 1, HC*H] and [b, 1, H]")
    HC = W // H
    if H % 8 or H > 16384 or HC > 4 or (HC + 2) * H > 56000:
        raise ValueError(f"inject_norm: H={H}, HC={HC}: H must be a multiple of 8 up to 16384, HC at most 4 and "
                         "(HC + 2) * H at most 56000")
    if not eps >= 0:
        raise ValueError(f"inject_norm: eps={eps} must not be negative")
    at = hyper.get_device()
    pack = not (hyper.is_contiguous() and values.is_contiguous())
    ok = hyper.dtype is BF16 and values.dtype is BF16 and values.get_device() == at
    for t, n, rows in ((gate, b * HC, b), (w_next, W, HC), (w_post, H, 1)):
        if t is not None:
            ok = ok and t.dtype is BF16 and t.get_device() == at and t.numel() == n and (
                t.dim() < 2 or t.shape[-1] * rows == n or _in_order(t, rows, n // max(rows, 1)))
            pack = pack or not t.is_contiguous()
    if not ok:
        raise ValueError(f"inject_norm: bf16 tensors on one device expected, a gate [{b}, 1, {HC}], w_next [{W}], "
                         f"w_post [{H}], axes in this order")
    for t in grads:
        if t is not None and (t.numel() != b * W or t.dtype is not BF16 or t.get_device() != at
                              or t.dim() > 1 and t.shape[-1] != W and not _in_order(t, b, HC, H)):
            raise ValueError("inject_norm_backward: gradients must be bf16, shaped and placed like state")
    if at < 0:
        _lib.require_cuda(hyper)
    return b, H, HC, pack, at


def _packed(*ts):
    """Contiguous, 16-byte aligned copies of what is not."""
    return [t if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0)
            else t.clone(memory_format=torch.contiguous_format) for t in ts]


def inject_norm(hyper, gate, values, w_next=None, *, w_post=None, scale=1.0, eps=1e-6):
    """``state = hyper + scale * gate * z`` per branch with ``z = values`` (or its rms norm times
    ``1 + w_post``), and ``normed``, the rms norm of every branch of ``state`` times ``1 + w_next``
    (``None`` without ``w_next``): the residual inject after a block and the norm that opens the next
    one (``inject`` then the first step of ``engine.gated_residual``) in one pass.  ``hyper`` bf16
    ``[b, 1, HC*H]``, ``gate`` bf16 ``[b, 1, HC]`` or ``None`` (1), ``values`` bf16 ``[b, 1, H]``,
    ``w_next`` ``[HC*H]``, ``w_post`` ``[H]``; HC = 1 is an ordinary residual stream.  Returns
    ``(state, normed)`` shaped like ``hyper``.  fp32 inside, each output rounded once; ``normed``
    comes from the unrounded state, so it can differ by one rounding from a norm of ``state``.  Not an
    autograd node: a ``hyper``, ``gate`` or ``values`` that requires a gradient while gradients are
    recorded is refused; ``inject_norm_backward`` gives the gradients."""
    if hyper.requires_grad or values.requires_grad or (gate is not None and gate.requires_grad):
        _lib.no_autograd("inject_norm", hyper, gate, values)
    b, H, HC, pack, at = _inject_norm_args(hyper, gate, values, w_next, w_post, eps)
    if at != torch._C._cuda_getDevice():              # (see _lib.elsewhere)
        with torch.cuda.device(at):
            return inject_norm(hyper, gate, values, w_next, w_post=w_post, scale=scale, eps=eps)
    if pack:
        hyper, gate, values, w_next, w_post = _packed(hyper, gate, values, w_next, w_post)
    state = torch.empty_like(hyper)
    normed = None if w_next is None else torch.empty_like(hyper)
    ptr = _lib.ptr
    rc = _lib.lib().fnx_inject_norm(hyper.data_ptr(), ptr(gate), values.data_ptr(), ptr(w_post), ptr(w_next),
                                    state.data_ptr(), ptr(normed), b, H, HC, scale, eps,
                                    torch._C._cuda_getCurrentRawStream(at))
    if rc == _lib.EALIGN and not pack:                # a view that starts off a 16-byte boundary
        return inject_norm(*_packed(hyper, gate, values, w_next), w_post=_packed(w_post)[0], scale=scale, eps=eps)
    _lib.check(rc, "residual injection with norms")
    return state, normed


def inject_norm_backward(d_state, d_normed, state, gate, values, w_next=None, *, w_post=None, scale=1.0, eps=1e-6):
    """Gradients of ``inject_norm`` from the gradients of its outputs (either may be ``None``: zero),
    the ``state`` it returned and its inputs: ``(d_hyper, d_gate, d_values, d_w_next, d_w_post)``,
    bf16 in the inputs' shapes, ``None`` where the input was ``None``.  Deterministic.  ``state`` is the
    rounded one, where the forward normed it before rounding: its statistics and ``d_w_next`` carry that
    rounding (2.3e-3 relative in ``d_w_next``, 3.6e-3 with a few loud channels)."""
    b, H, HC, _, _ = _inject_norm_args(state, gate, values, w_next, w_post, eps, (d_state, d_normed))
    if d_state is None and d_normed is None:
        raise ValueError("inject_norm_backward: d_state or d_normed needed")
    if d_normed is not None and w_next is None:
        raise ValueError("inject_norm_backward: d_normed without w_next")
    dev = state.device
    if _lib.elsewhere(state):
        with torch.cuda.device(dev):
            return inject_norm_backward(d_state, d_normed, state, gate, values, w_next, w_post=w_post, scale=scale,
                                        eps=eps)
    d_state, d_normed, state, values_c, gate_c, w_next_c, w_post_c = _packed(d_state, d_normed, state, values, gate,
                                                                             w_next, w_post)
    new = lambda t: None if t is None else torch.empty_like(t)                                       # noqa: E731
    d_hyper, d_gate, d_values, d_w_next, d_w_post = new(state), new(gate_c), new(values_c), new(w_next_c), new(w_post_c)
    L = _lib.lib()
    nws = L.fnx_inject_norm_backward_workspace(b, H, HC)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev)
    rc = L.fnx_inject_norm_backward(_lib.ptr(d_state), _lib.ptr(d_normed), state.data_ptr(), _lib.ptr(gate_c),
                                    values_c.data_ptr(), _lib.ptr(w_post_c), _lib.ptr(w_next_c), d_hyper.data_ptr(),
                                    _lib.ptr(d_gate), d_values.data_ptr(), _lib.ptr(d_w_post), _lib.ptr(d_w_next),
                                    b, H, HC, scale, eps, ws.data_ptr(), nws, _lib.raw_stream(dev))
    _lib.check(rc, "gradient of the residual injection with norms")
    return d_hyper, d_gate, d_values, d_w_next, d_w_post
