"""Refusals of the fused residual step: on the host, before any launch."""
import pytest
import torch

BF16 = torch.bfloat16


def t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def test_python_refusals():
    from fnx.native_inject import inject_norm, inject_norm_backward
    h, g, v, wn = t(2, 1, 256), t(2, 1, 4), t(2, 1, 64), t(256)
    for bad in ((t(2, 1, 250), g, v, wn), (h, t(2, 1, 3), v, wn), (h, g, t(3, 1, 64), wn), (h, g, v, t(64)),
                (h.float(), g, v, wn), (h, g.float(), v, wn), (t(2, 1, 5 * 64), t(2, 1, 5), v, None),
                (t(2, 1, 12), t(2, 1, 1), t(2, 1, 12), None), (t(1, 1, 16392), None, t(1, 1, 16392), None),
                (t(1, 1, 4 * 9344), None, t(1, 1, 9344), None)):
        with pytest.raises(ValueError):
            inject_norm(*bad)
    with pytest.raises(ValueError):
        inject_norm(h, g, v, wn, w_post=t(65))
    with pytest.raises(RuntimeError):                 # no CPU path
        inject_norm(h, g, v, wn)
    for bad in ((None, None, h, g, v, wn), (h, h, h, g, v), (h.float(), None, h, g, v, wn), (t(2, 1, 8), None, h, g, v, wn)):
        with pytest.raises((ValueError, RuntimeError)):
            inject_norm_backward(*bad)


def test_abi_refusals():
    import build as fnx_build
    fnx_build.build()
    from fnx import _lib
    L = _lib.lib()
    f, b = L.fnx_inject_norm, L.fnx_inject_norm_backward
    assert f(None, 16, 16, None, None, 16, None, 1, 64, 4, 1.0, 1e-6, None) == -1        # no hyper
    assert f(16, 16, 16, None, 16, 16, None, 1, 64, 4, 1.0, 1e-6, None) == -1            # w_next without normed
    assert f(16, 16, 16, None, None, 16, None, 1, 60, 4, 1.0, 1e-6, None) == -2          # H % 8
    assert f(16, 16, 16, None, None, 16, None, 1, 64, 5, 1.0, 1e-6, None) == -2          # HC
    assert f(16, 16, 16, None, None, 16, None, -1, 64, 4, 1.0, 1e-6, None) == -2         # batch
    assert f(16, 16, 16, None, None, 16, None, 1, 9344, 4, 1.0, 1e-6, None) == -2        # (HC + 2) * H
    assert f(18, 16, 16, None, None, 16, None, 1, 64, 4, 1.0, 1e-6, None) == -3          # alignment
    assert f(16, 16, 16, 24, None, 16, None, 1, 64, 4, 1.0, 1e-6, None) == -3
    assert f(None, None, None, None, None, None, None, 0, 64, 4, 1.0, 1e-6, None) == 0   # nothing to do
    need = L.fnx_inject_norm_backward_workspace(5, 64, 4)
    assert need == 5 * 5 * 64 * 4 and L.fnx_inject_norm_backward_workspace(5, 60, 4) == 0
    ok = [16] * 12
    assert b(*ok, 5, 64, 4, 1.0, 1e-6, 16, need - 1, None) == -5
    assert b(None, None, *ok[2:], 5, 64, 4, 1.0, 1e-6, 16, need, None) == -1
    assert b(16, 16, 16, 16, 16, None, *ok[6:], 5, 64, 4, 1.0, 1e-6, 16, need, None) == -1    # d_w_post, no w_post
    assert b(16, 16, 16, None, *ok[4:], 5, 64, 4, 1.0, 1e-6, 16, need, None) == -1            # d_gate, no gate
    assert b(*ok, 5, 60, 4, 1.0, 1e-6, 16, need, None) == -2
    assert b(8, *ok[1:], 5, 64, 4, 1.0, 1e-6, 16, need, None) == -3
