"""``inject_norm`` and its gradients against their definitions in 64 bits.

Tolerances: an output is one rounding of an fp32 value, so at most 2^-8 of its size off; the fp32
arithmetic behind it (sums of at most 16384 products, a handful of multiplications) adds less than
2^-14 of the row's scale.  A value that is a small difference of large ones carries the large ones'
fp32 error, hence the absolute part, 2^-14 of the output's largest value.  The gradients start from
the stored (rounded) state where the definition has the exact one: its 2^-9 relative error (half a
step at most, 2^-8 of an element) reaches d_normed's products, bounded by 2^-8 of the largest value,
so gradients get 2^-8 relative and 2^-7 of the largest value absolute."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"
EPS = 1e-6


def rms64(v, w):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * (1 + w)


def definition(hyper, gate, values, w_next, w_post, scale):
    b, H = hyper.shape[0], values.shape[-1]
    HC = hyper.shape[-1] // H
    z = values.view(b, 1, H)
    if w_post is not None:
        z = rms64(z, w_post)
    g = scale if gate is None else scale * gate.view(b, HC, 1)
    state = hyper.view(b, HC, H) + g * z
    normed = None if w_next is None else rms64(state, w_next.view(HC, H)).reshape(hyper.shape)
    return state.reshape(hyper.shape), normed


def inputs(b, H, HC, seed, post=True, gate=True, nxt=True):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF16).to(DEV)                       # noqa: E731
    return (rnd(b, 1, HC * H), rnd(b, 1, HC) if gate else None, rnd(b, 1, H), rnd(HC * H) if nxt else None,
            rnd(H) if post else None)


def close(got, want, rel=2 ** -8, floor=2 ** -14):
    assert got.dtype == BF16 and got.shape == want.shape
    err = (got.double() - want).abs()
    lim = rel * want.abs() + floor * want.abs().max().clamp(min=1e-30)
    assert bool((err <= lim).all()), float((err / lim).max())


CASES = [(1, 8, 1), (1, 2560, 4), (2, 264, 3), (3, 4096, 4), (7, 4104, 2), (5, 8192, 4), (2, 9328, 4), (3, 16384, 1),
         (149, 640, 4), (301, 2048, 2), (1025, 512, 1)]


@pytest.mark.parametrize("b,H,HC", CASES)
@pytest.mark.parametrize("post", [False, True])
def test_forward(b, H, HC, post):
    from fnx.native_inject import inject_norm
    a = inputs(b, H, HC, b + H + HC, post)
    for kw in (dict(scale=1.0), dict(scale=-0.37)):
        state, normed = inject_norm(a[0], a[1], a[2], a[3], w_post=a[4], **kw)
        ws, wn = definition(*(None if t is None else t.double() for t in a), kw["scale"])
        close(state, ws)
        close(normed, wn)


def test_forward_without_gate_or_norms_is_a_residual_add():
    from fnx.native_inject import inject, inject_norm
    h, g, v, _, _ = inputs(9, 256, 1, 3)
    state, normed = inject_norm(h, None, v)
    assert normed is None and torch.equal(state, (h.float() + v.float()).to(BF16))
    # one rounding against inject's two: never further from the exact value
    h, g, v, _, _ = inputs(9, 256, 4, 4)
    state, _ = inject_norm(h, g, v)
    exact, _ = definition(h.double(), g.double(), v.double(), None, None, 1.0)
    assert bool(((state.double() - exact).abs() <= (inject(h, g, v).double() - exact).abs() + 1e-12).all())


def test_strided_and_two_dimensional_inputs():
    from fnx.native_inject import inject_norm, inject_norm_backward
    h, g, v, wn, wp = inputs(6, 128, 4, 5)
    wide = torch.randn(6, 1, 2 * 512, device=DEV).to(BF16)
    wide[..., ::2] = h
    want = inject_norm(h, g, v, wn, w_post=wp)
    got = inject_norm(wide[..., ::2], g, v, wn, w_post=wp)
    flat = inject_norm(h.view(6, -1), g.view(6, -1), v.view(6, -1), wn, w_post=wp)
    for w, x, y in zip(want, got, flat):
        assert torch.equal(w, x) and torch.equal(w.view(6, -1), y)
    off = torch.empty(6 * 512 + 3, dtype=BF16, device=DEV)[3:]     # contiguous, off a 16-byte boundary
    off.copy_(h.view(-1))
    odd = inject_norm(off.view(6, 1, 512), g, v, wn, w_post=wp)
    assert torch.equal(odd[0], want[0]) and torch.equal(odd[1], want[1])
    grads = inject_norm_backward(h, h, want[0], g, v, wn, w_post=wp)
    for a, c in zip(grads, inject_norm_backward(off.view(6, 1, 512), h, want[0], g, v, wn, w_post=wp)):
        assert torch.equal(a, c)


def test_empty_batch():
    from fnx.native_inject import inject_norm, inject_norm_backward
    h, g, v, wn, wp = inputs(0, 64, 4, 6)
    state, normed = inject_norm(h, g, v, wn, w_post=wp)
    assert state.shape == normed.shape == h.shape
    grads = inject_norm_backward(state, normed, state, g, v, wn, w_post=wp)
    assert not grads[3].any() and not grads[4].any() and grads[3].shape == wn.shape


def test_values_that_are_not_finite_stay_in_their_token():
    from fnx.native_inject import inject_norm
    h, g, v, wn, wp = inputs(4, 512, 4, 7)
    want = inject_norm(h, g, v, wn, w_post=wp)
    v[1, 0, 17] = float("nan")
    h[2, 0, 5] = float("inf")
    got = inject_norm(h, g, v, wn, w_post=wp)
    for w, x in zip(want, got):
        assert torch.equal(w[0], x[0]) and torch.equal(w[3], x[3])
    assert got[0][1].isnan().all() and got[0][2, 0, 5].isinf() and got[1][2, 0, :512].isnan().any()
    assert torch.equal(got[1][2, 0, 512:], want[1][2, 0, 512:])              # the other branches of that token


@pytest.mark.parametrize("b,H,HC", CASES)
@pytest.mark.parametrize("post", [False, True])
def test_backward(b, H, HC, post):
    from fnx.native_inject import inject_norm, inject_norm_backward
    a = inputs(b, H, HC, 2 * b + H + HC, post)
    scale = 0.75
    state, normed = inject_norm(a[0], a[1], a[2], a[3], w_post=a[4], scale=scale)
    ds, dn = inputs(b, H, HC, 99)[0], inputs(b, H, HC, 100)[0]
    leaves = [None if t is None else t.double().requires_grad_() for t in a]
    outs = definition(*leaves, scale)
    for gs, gn in ((ds, dn), (None, dn), (ds, None)):
        kept = [(o, w) for o, w in zip(outs, (gs, gn)) if w is not None]
        some = [t for t in leaves if t is not None]
        want = torch.autograd.grad([o for o, _ in kept], some, [w.double() for _, w in kept], retain_graph=True,
                                   allow_unused=True)
        want = [torch.zeros_like(t) if w is None else w for w, t in zip(want, some)]
        got = inject_norm_backward(gs, gn, state, a[1], a[2], a[3], w_post=a[4], scale=scale)
        got = [t for t in got if t is not None]
        assert len(got) == len(want)
        for x, w in zip(got, want):
            close(x, w, 2 ** -8, 2 ** -7)


def test_backward_against_differences():
    """d(sum of outputs * weights) along a direction of every input, by central differences in 64 bits."""
    from fnx.native_inject import inject_norm, inject_norm_backward
    a = inputs(5, 96, 4, 11)
    state, _ = inject_norm(a[0], a[1], a[2], a[3], w_post=a[4])
    ds, dn = inputs(5, 96, 4, 12)[0], inputs(5, 96, 4, 13)[0]
    got = inject_norm_backward(ds, dn, state, a[1], a[2], a[3], w_post=a[4])
    order = (got[0], got[1], got[2], got[3], got[4])
    at = [t.double() for t in a]

    def value(args):
        s, n = definition(*args, 1.0)
        return float((s * ds.double()).sum() + (n * dn.double()).sum())
    for i, grad in enumerate(order):
        d = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(i)).double().to(DEV)
        h = 1e-5
        up, down = ([t + (h * d if j == i else 0) * s for j, t in enumerate(at)] for s in (1, -1))
        slope = (value(up) - value(down)) / (2 * h)
        # every gradient element is within 2^-8 of itself and 2^-7 of the largest: their weighted sum,
        # over independent errors, within four times its standard deviation
        g = grad.double().view(d.shape)
        dev = ((2 ** -8 * g.abs() + 2 ** -7 * g.abs().max()) * d.abs()).norm()
        assert abs(float((g * d).sum()) - slope) <= 4 * float(dev)


def test_backward_is_deterministic_and_replays_from_a_graph():
    from fnx.native_inject import inject_norm, inject_norm_backward
    a = inputs(700, 512, 4, 21)
    ds, dn = inputs(700, 512, 4, 22)[0], inputs(700, 512, 4, 23)[0]

    def step():
        state, normed = inject_norm(a[0], a[1], a[2], a[3], w_post=a[4])
        return (state, normed) + inject_norm_backward(ds, dn, state, a[1], a[2], a[3], w_post=a[4])
    want = step()
    for w, x in zip(want, step()):
        assert torch.equal(w, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    a[0].mul_(0.5)
    graph.replay()
    for w, x in zip(step(), held):
        assert torch.equal(w, x)


def test_offsets_past_32_bits():
    from fnx.native_inject import inject_norm, inject_norm_backward
    H, HC = 2048, 4
    T = 2 ** 18 + 5
    few = inputs(3, H, HC, 41)
    where = torch.tensor([0, T // 2, T - 1], device=DEV)
    big = []
    for t in few[:3]:
        b = torch.zeros(T, *t.shape[1:], dtype=BF16, device=DEV)
        b[where] = t
        big.append(b)
    assert big[0].numel() > 2 ** 31
    state, normed = inject_norm(big[0], big[1], big[2], few[3], w_post=few[4])
    want = inject_norm(few[0], few[1], few[2], few[3], w_post=few[4])
    assert torch.equal(state[where], want[0]) and torch.equal(normed[where], want[1])
    got = inject_norm_backward(state, None, state, big[1], big[2], few[3], w_post=few[4])
    want = inject_norm_backward(want[0], None, want[0], few[1], few[2], few[3], w_post=few[4])
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a[where], b)


def test_state_feeds_the_next_mix():
    """The fused step in the place of inject + the norm that opens gated_residual."""
    from fnx.engine import gated_residual
    from fnx.native_inject import inject, inject_norm
    H, hc, r = 256, 4, 64
    h, g, v, wn, _ = inputs(33, H, hc, 31)
    gen = torch.Generator().manual_seed(32)
    down = (torch.randn(r + hc, hc * H, generator=gen) / 32).to(BF16).to(DEV)
    up = (torch.randn(hc * H, r, generator=gen) / 8).to(BF16).to(DEV)
    state, normed = inject_norm(h, g, v, wn)
    want = gated_residual(inject(h, g, v), wn, down, up, n_inj=hc)
    got = gated_residual(state, wn, down, up, n_inj=hc, normed=normed)
    for w, x in zip(want, got):                       # two roundings apart at the input of two GEMMs
        assert float((w.float() - x.float()).norm() / w.float().norm()) < 2 ** -6
