"""What ``inject_norm`` and its gradients answer on the host, before any launch."""
import pytest
import torch


def lib():
    import build as fnx_build
    fnx_build.build()
    from fnx import _lib
    return _lib.lib()


@pytest.mark.parametrize("H,HC", [(512, 1), (4096, 1), (4104, 1), (1864, 2), (2048, 2), (2560, 2), (1536, 3), (2048, 3),
                                  (1288, 4), (2048, 4), (4104, 4)])
def test_the_backward_launches_no_more_blocks_than_fit(H, HC):
    """Its blocks are persistent: one that does not fit waits for another to end and then starts its copies
    anew, and each writes its own partial sums.  The kernels' launch bounds (512 threads, one block an SM;
    two for one branch of H <= 4096) let the compiler take 65536 / 512 = 128 registers a thread, or 64."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    blocks, rest = divmod(lib().fnx_inject_norm_backward_workspace(1 << 20, H, HC), (HC + 1) * H * 4)
    threads = (H // 8 + 31) // 32 * 32 if H <= 4096 else 512
    registers = 64 if HC == 1 and H <= 4096 else 128
    assert rest == 0 and blocks % sms == 0
    assert 1 <= blocks // sms <= max(1, 65536 // (registers * threads))


def t(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


HYPER, GATE, VALUES, W_NEXT, W_POST = t(8, 1, 4 * 64), t(8, 1, 4), t(8, 1, 64), t(256), t(64)


@pytest.mark.parametrize("gate", [t(4, 8), t(1, 4, 8), t(4, 8, 1), t(2, 16)])
def test_a_gate_in_another_order_is_refused(gate):
    from fnx.native_inject import inject_norm, inject_norm_backward
    with pytest.raises(ValueError):
        inject_norm(HYPER, gate, VALUES, W_NEXT)
    with pytest.raises(ValueError):
        inject_norm_backward(HYPER, HYPER, HYPER, gate, VALUES, W_NEXT)


@pytest.mark.parametrize("w_next,w_post", [(t(64, 4), None), (t(2, 128), None), (W_NEXT, t(8, 8)), (W_NEXT, t(2, 32))])
def test_weights_in_another_order_are_refused(w_next, w_post):
    from fnx.native_inject import inject_norm
    with pytest.raises(ValueError):
        inject_norm(HYPER, GATE, VALUES, w_next, w_post=w_post)


@pytest.mark.parametrize("grad", [t(4, 8, 64), t(256, 8), t(256, 1, 8), t(8, 64, 4), t(4, 512)])
def test_gradients_in_another_order_are_refused(grad):
    from fnx.native_inject import inject_norm_backward
    for pair in ((grad, None), (None, grad), (HYPER, grad)):
        with pytest.raises(ValueError):
            inject_norm_backward(*pair, HYPER, GATE, VALUES, W_NEXT)


def test_every_row_major_form_of_the_same_values_is_taken():
    """(as far as the check that there is a GPU, which comes last)"""
    from fnx.native_inject import inject_norm, inject_norm_backward
    for gate in (GATE, t(8, 4), t(8, 4, 1), t(32), t(2, 4, 4), None):
        for w_next, w_post in ((W_NEXT, W_POST), (t(4, 64), t(1, 64)), (t(1, 256), t(64, 1)), (t(256, 1), None), (t(1, 256, 1), None)):
            with pytest.raises(RuntimeError, match="CUDA"):
                inject_norm(HYPER, gate, VALUES, w_next, w_post=w_post)
    for grad in (HYPER, t(8, 256), t(8, 4, 64), t(32, 64), t(2, 4, 256), t(8 * 256)):
        with pytest.raises(RuntimeError, match="CUDA"):
            inject_norm_backward(grad, grad, HYPER, GATE, VALUES, W_NEXT)
    one, gate = t(8, 1, 64), t(8, 1, 1)                      # a single branch: any shape of b values
    for g in (gate, t(8), t(2, 4), t(1, 8)):
        with pytest.raises(RuntimeError, match="CUDA"):
            inject_norm(one, g, one, t(64))
    first = t(1, 1, 256)                                     # a single token
    for g in (t(4), t(1, 4), t(4, 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            inject_norm(first, g, t(1, 64), W_NEXT)
    with pytest.raises(RuntimeError, match="CUDA"):
        inject_norm(t(1, 1, 64), t(), t(1, 64), t(64))
    with pytest.raises(RuntimeError, match="CUDA"):
        inject_norm(t(0, 1, 256), t(0, 1, 4), t(0, 1, 64), W_NEXT)


@pytest.mark.parametrize("eps", [-1e-6, float("nan")])
def test_an_eps_that_is_no_bound_is_refused(eps):
    from fnx.native_inject import inject_norm, inject_norm_backward
    with pytest.raises(ValueError, match="eps"):
        inject_norm(HYPER, GATE, VALUES, W_NEXT, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        inject_norm_backward(HYPER, HYPER, HYPER, GATE, VALUES, W_NEXT, eps=eps)
    L = lib()
    assert L.fnx_inject_norm(16, 16, 16, None, None, 16, None, 0, 64, 4, 1.0, eps, None) == -1
    assert L.fnx_inject_norm_backward(*[16] * 12, 0, 64, 4, 1.0, eps, 16, 0, None) == -1
