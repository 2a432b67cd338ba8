"""Refusals of the dense 4-bit projection: on the host, before any launch."""
import pytest
import torch

BF16 = torch.bfloat16


def test_python_refusals():
    from fnx.engine import DenseW4
    w, s = torch.zeros(64, 4, dtype=torch.int32), torch.zeros(2, 32, dtype=BF16)
    for bad in ((w.float(), s, 32), (w[0], s, 32), (w, s.float(), 32), (w, s, 24), (w, s, 0), (w, s, 16), (w, s[:1], 32),
                (w, s[:, :16], 32), (w[:60], s, 32), (w, s, -32),
                (w, s[:1], 2 ** 32 + 128)):
        with pytest.raises(ValueError):
            DenseW4(*bad)
    with pytest.raises(RuntimeError):                       # no CPU path
        DenseW4(w, s, 32)
    with pytest.raises(ValueError):
        DenseW4.merge([])


def test_abi_refusals():
    import build as fnx_build
    fnx_build.build()
    from fnx import _lib
    f = _lib.lib().fnx_w4a16_gemv
    ok = (64, 64, 64, 64, 64, 1, 64, 64, 32, None)

    def call(**kw):
        names = ("x", "ld", "w", "s", "y", "M", "K", "N", "gs", "st")
        return f(*[kw.get(n, v) for n, v in zip(names, ok)])
    assert call(M=-1) == -1 and call(K=0) == -1 and call(gs=8) == -1 and call(gs=40) == -1 and call(ld=56) == -1
    assert call(K=60) == -2 and call(N=60) == -2
    assert call(x=None) == -1 and call(y=None) == -1 and call(w=None) == -1 and call(s=None) == -1
    assert call(x=72) == -3 and call(w=68) == -3 and call(s=72) == -3 and call(y=72) == -3 and call(ld=66) == -3
    assert call(M=0, x=None, y=None) == 0
