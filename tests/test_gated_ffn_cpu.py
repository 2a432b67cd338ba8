"""Refusals of the gated feed-forward block: on the host, before any launch."""
import pytest
import torch

BF16 = torch.bfloat16


def test_python_refusals():
    from fnx.gated_ffn import GatedFFN
    w, d = torch.zeros(64, 16, dtype=BF16), torch.zeros(24, 32, dtype=BF16)
    for bad in ((w.float(), d), (w, d.float()), (w[0], d), (w, d[:, :24]), (w[:, :12], d), (w[:60], d), (w, d[:20]),
                (torch.zeros(0, 16, dtype=BF16), torch.zeros(24, 0, dtype=BF16))):
        with pytest.raises(ValueError):
            GatedFFN(*bad)
    with pytest.raises(RuntimeError):                       # no CPU path
        GatedFFN(w, d)


def test_backward_refuses_what_another_block_kept():
    from fnx.gated_ffn import GatedFFN
    blk = GatedFFN.__new__(GatedFFN)                        # (its own checks want a GPU)
    blk.H, blk.I, blk.O, blk.w_gu = 16, 32, 24, torch.zeros(64, 16, dtype=BF16)
    dy, x, h = (torch.zeros(4, n, dtype=BF16) for n in (24, 16, 32))
    gu = torch.zeros(8, dtype=torch.uint8)
    for x2, h2 in ((x[:, :8], h), (x, h[:, :24]), (x.to("meta"), h)):
        with pytest.raises(ValueError, match="another block"):
            blk.backward(dy, (x2, h2, gu, x2.shape))
    with pytest.raises(ValueError, match="3 rows"):
        blk.backward(dy[:3], (x, h, gu, x.shape))


def test_abi_refusals():
    import build as fnx_build
    fnx_build.build()
    from fnx import _lib
    L = _lib.lib()
    f, b = L.fnx_gated_ffn, L.fnx_gated_ffn_backward
    names = ("x", "ld", "wgu", "wd", "h", "saved", "y", "M", "H", "I", "O")

    def call(**kw):
        ok = dict(x=64, ld=64, wgu=64, wd=64, h=64, saved=None, y=64, M=4, H=64, I=32, O=64)
        ok.update(kw)
        return f(*[ok[n] for n in names], None)
    assert call(M=-1) == -1 and call(H=0) == -1 and call(I=0) == -1 and call(ld=56) == -1
    assert call(H=60, ld=64) == -2 and call(I=36) == -2 and call(O=12) == -2
    assert call(x=None) == -1 and call(h=None) == -1 and call(wgu=None) == -1
    assert call(wd=None) == -1 and call(y=None) == -1       # both or neither
    assert call(x=72) == -3 and call(ld=68) == -3 and call(h=72) == -3 and call(y=72) == -3 and call(saved=72) == -3
    assert call(M=0, x=None, h=None, y=None) == 0
    assert L.fnx_gated_ffn_saved_bytes(1, 32) == 128 * 64 * 4 and L.fnx_gated_ffn_saved_bytes(129, 32) == 256 * 64 * 4
    assert L.fnx_gated_ffn_saved_bytes(4, 12) == 0
    bn = ("dy", "ld_dy", "x", "ld_x", "wgu", "wd", "h", "saved", "dgu", "dx", "dwgu", "dwd", "M", "H", "I", "O")

    def back(**kw):
        ok = dict(zip(bn, (64, 64, 64, 64) + (64,) * 8 + (4, 64, 32, 64)))
        ok.update(kw)
        return b(*[ok[n] for n in bn], None)
    assert back(dy=None) == -1 and back(saved=None) == -1 and back(dgu=None) == -1 and back(wd=None) == -1
    assert back(wgu=None) == -1 and back(x=None) == -1 and back(h=None) == -1      # needed by dx, dw_gu, dw_down
    assert back(ld_dy=56) == -1 and back(ld_x=60) == -1 and back(ld_dy=68) == -3 and back(dx=72) == -3
    assert back(H=60) == -2 and back(M=-2) == -1
    assert back(M=0, dwgu=None, dwd=None) == 0
