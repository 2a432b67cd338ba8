"""The dense operators are plain functions: a result never leads back to its inputs.  An input that
carries an autograd graph into one of them would lose its gradient without a word, so it is refused
where no gradient is made by hand either."""
import pytest
import torch

BF16 = torch.bfloat16


def t(*shape, grad=False):
    return torch.zeros(shape, dtype=BF16, requires_grad=grad)


def ffn():
    from fnx.gated_ffn import GatedFFN
    f = GatedFFN.__new__(GatedFFN)                           # (its own checks want a GPU)
    f.H, f.I, f.O, f.w_gu, f.w_down = 16, 32, 24, t(64, 16, grad=True), t(24, 32, grad=True)
    f._forward = lambda x, keep, down: (x.detach(), t(len(x), 32), None, t(len(x), 24))
    return f


def w4():
    from fnx.engine import DenseW4
    d = DenseW4.__new__(DenseW4)
    d.K, d.N, d.gs, d.w4 = 16, 24, 16, torch.zeros(16, 3, dtype=torch.int32)
    return d


def test_inputs_with_a_graph_are_refused():
    from fnx.native_inject import inject_norm
    x = t(3, 16, grad=True)
    for call in (ffn(), ffn().gated, w4()):
        with pytest.raises(ValueError, match="gradient"):
            call(x)
    for i in range(3):
        args = [t(2, 1, 64, grad=i == 0), t(2, 1, 4, grad=i == 1), t(2, 1, 16, grad=i == 2)]
        with pytest.raises(ValueError, match="gradient"):
            inject_norm(*args, t(64))


def test_without_grad_mode_and_for_a_gradient_by_hand_they_are_taken():
    from fnx.native_inject import inject_norm
    f, x = ffn(), t(3, 16, grad=True)
    with torch.no_grad():
        assert f(x).shape == (3, 24) and f.gated(x).shape == (3, 32)
        with pytest.raises(RuntimeError, match="CUDA"):      # the check for a GPU comes last
            inject_norm(t(2, 1, 64, grad=True), None, t(2, 1, 16), t(64))
    assert f.forward_train(x)[0].shape == (3, 24)            # its gradient is what backward() makes
    assert f(x.detach()).shape == (3, 24)                    # weights may be parameters
    with pytest.raises(RuntimeError, match="CUDA"):
        inject_norm(t(2, 1, 64), None, t(2, 1, 16), t(64, grad=True))
