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


def formulas(state, gate, values, w_next, w_post, d_state, d_normed, scale=0.75, eps=1e-6):
    """The gradients in 64 bits from what the backward is handed: the stored state, not the unrounded one."""
    T, H = values.shape[0], values.shape[-1]
    HC = state.shape[-1] // H
    s, y, wn, wp = state.double().view(T, HC, H), values.double().view(T, 1, H), w_next.double().view(HC, H), w_post.double()
    D, e = d_state.double().view(T, HC, H), d_normed.double().view(T, HC, H)
    g = scale * gate.double().view(T, HC, 1)
    rs = ((s * s).mean(-1, keepdim=True) + eps) ** -0.5
    rv = ((y * y).mean(-1, keepdim=True) + eps) ** -0.5
    z = y * rv * (1 + wp)
    d = D + rs * (e * (1 + wn) - s * rs ** 2 * (e * (1 + wn) * s).mean(-1, keepdim=True))
    dz = (g * d).sum(1, keepdim=True)
    dp = dz * (1 + wp)
    dy = rv * (dp - y * rv ** 2 * (dp * y).mean(-1, keepdim=True))
    return (d.reshape(state.shape), scale * (d * z).sum(-1).view(gate.shape), dy.reshape(values.shape),
            (e * s * rs).sum(0).reshape(-1), (dz * y * rv).sum((0, 1)))


@pytest.mark.parametrize("T,H,HC", MANY)
def test_gradients_summed_over_many_tokens(T, H, HC):
    """Against the formulas from the same stored state, so that only fp32 arithmetic and the last rounding
    are between the two.  The rounding: 2^-8 of the value.  The arithmetic, relative to the largest value of
    a gradient: a sum over T <= 6001 tokens has terms of at most sqrt(T) = 78 times its largest value in
    sum (Cauchy, the largest of many columns being at least the root of its squared terms); it is made of
    fewer than 41 tokens a block, 74 blocks a row group and 8 groups, 123 additions of 2^-24 each, and its
    terms are good to 2^-20: 78 * (123 * 2^-24 + 2^-20) < 2^-10.  The others are good to 2^-20 of sums whose
    terms exceed their largest value less than that.  One token left out of a sum, or counted twice, changes
    it by a term of about 1 in 2^-10 of at most 400."""
    hyper, gate, values, w_next, w_post, d_state, d_normed = a = inputs(T, H, HC, T)
    got = step(*a)
    want = formulas(got[0], gate, values, w_next, w_post, d_state, d_normed)
    for name, x, w in zip(("d_hyper", "d_gate", "d_values", "d_w_next", "d_w_post"), got[2:], want):
        assert x.dtype == BF16 and x.shape == w.shape
        lim = 2 ** -8 * w.abs() + 2 ** -10 * w.abs().max()
        err = (x.double() - w).abs()
        assert bool((err <= lim).all()), (name, float((err / lim).max()))
    again = step(*a)
    for x, w in zip(again, got):
        assert torch.equal(x, w)
