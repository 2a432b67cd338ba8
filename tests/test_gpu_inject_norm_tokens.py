"""The gradients of ``inject_norm`` where a block of the backward takes many tokens: its refilled stages,
the sums that it keeps over them, and the column sums behind it, which start while it still runs."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"

# five tokens a block and more on 148 SMs, in the narrow kernel (H <= 4096) for each count of branches
# and in the wide one; the last round of tokens is ragged
MANY = [(6001, 512, 1), (3000, 512, 4), (2500, 2048, 2), (1501, 1096, 3), (1600, 4104, 2), (901, 8192, 4)]


def inputs(T, H, HC, seed):
    """hyper, gate, values, w_next, w_post, d_state, d_normed"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(*s, generator=g, device=DEV).to(BF16) for s in
            ((T, 1, HC * H), (T, 1, HC), (T, 1, H), (HC * H,), (H,), (T, 1, HC * H), (T, 1, HC * H))]


def step(hyper, gate, values, w_next, w_post, d_state, d_normed, scale=0.75):
    from fnx.native_inject import inject_norm, inject_norm_backward
    state, normed = inject_norm(hyper, gate, values, w_next, w_post=w_post, scale=scale)
    return (state, normed) + inject_norm_backward(d_state, d_normed, state, gate, values, w_next, w_post=w_post,
                                                  scale=scale)


@pytest.mark.parametrize("T,H,HC", MANY)
def test_inputs_written_right_before_and_overwritten_right_after(T, H, HC):
    """Two sets of inputs take turns in the same buffers, so whatever is read too early, or partial sums of
    the call before that are still in the recycled workspace, shows as other bits."""
    sets = [inputs(T, H, HC, s) for s in (1, 2)]
    want = []
    for s in sets:
        want.append([t.clone() for t in step(*s)])
        torch.cuda.synchronize()
    held = [torch.empty_like(t) for t in sets[0]]
    wrong = torch.zeros((), dtype=torch.int64, device=DEV)
    for i in range(12):
        for b, t in zip(held, sets[i % 2]):
            b.copy_(t)
        got = step(*held)
        for b in held:
            b.fill_(float("nan"))
        for x, w in zip(got, want[i % 2]):
            wrong += (x != w).sum()
    assert int(wrong) == 0
