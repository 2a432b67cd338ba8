"""``GatedFFN`` and its gradients against their definitions in 64 bits.

Tolerances.  u = 2^-8, the relative error of one rounding to bf16.  Every product accumulates in fp32:
K steps each off by at most 2^-22 of the sum of the magnitudes, written a(.) below.  The activation
uses exponentials and reciprocals good to 2^-20.  With mag = the same expression with absolute values:
  h        u |h| + 2^-12 mag          (K <= 4096: K * 2^-22 is at most 2^-10 of mag only if every step
                                       erred the same way; independent errors grow with sqrt(K): 2^-16)
  y        u |y| + u (|h| |Wd|^T)/ sqrt(3 I) * 6: the roundings of h are independent and at most u each,
           uniform (variance u^2 / 3 of each product's square): six standard deviations of their sum
  likewise dx (roundings of dgu), dw_gu (of dgu), dw_down (of h)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"
U = 2.0 ** -8


def make(M, H, I, O, seed=0):
    from fnx.gated_ffn import GatedFFN
    g = torch.Generator().manual_seed(seed + M + H + I)
    rnd = lambda s, *n: (torch.randn(*n, generator=g) * s).to(BF16).to(DEV)               # noqa: E731
    w_gu, w_down = rnd(H ** -0.5, 2 * I, H), rnd(I ** -0.5, O, I)
    return GatedFFN(w_gu, w_down), rnd(1, M, H), rnd(1, M, O)


def definition(f, x, dy=None):
    """64-bit outputs, and the standard deviation of what rounding the inner operands does to them."""
    x, wgu, wd = x.double(), f.w_gu.double(), f.w_down.double()
    g, u = x @ wgu[:f.I].t(), x @ wgu[f.I:].t()
    s = torch.sigmoid(g)
    h = g * s * u
    y = h @ wd.t()
    sd = lambda a, b: U / 3 ** 0.5 * ((a * a) @ (b * b)).sqrt()                            # noqa: E731
    out = {"h": (h, torch.zeros_like(h)), "y": (y, sd(h, wd.t()))}
    if dy is not None:
        dy = dy.double()
        dh = dy @ wd
        dgu = torch.cat([dh * u * s * (1 + g * (1 - s)), dh * g * s], 1)
        out["dx"] = (dgu @ wgu, sd(dgu, wgu))
        out["dw_gu"] = (dgu.t() @ x, sd(dgu.t(), x))
        out["dw_down"] = (dy.t() @ h, sd(dy.t(), h))
    return out


def close(got, want, what=""):
    v, sd = want
    assert got.dtype == BF16 and got.shape == v.shape
    lim = U * v.abs() + 6 * sd + 2 ** -12 * v.abs().max()
    err = (got.double() - v).abs()
    assert bool((err <= lim).all()), (what, float((err / lim.clamp(min=1e-300)).max()))


SHAPES = [(1, 2560, 640, 2560), (2, 8, 8, 8), (5, 64, 136, 24), (16, 1000, 328, 520), (17, 256, 128, 256),
          (33, 512, 1032, 264), (64, 2048, 512, 2048), (127, 136, 72, 128), (129, 320, 200, 640), (255, 64, 1288, 72),
          (257, 1032, 256, 1032), (511, 2560, 640, 2560), (1030, 712, 2056, 712)]


@pytest.mark.parametrize("M,H,I,O", SHAPES)
def test_forward(M, H, I, O):
    f, x, _ = make(M, H, I, O)
    want = definition(f, x)
    close(f.gated(x), want["h"], "h")
    close(f(x), want["y"], "y")


@pytest.mark.parametrize("M,H,I,O", SHAPES)
def test_backward(M, H, I, O):
    f, x, dy = make(M, H, I, O, 1)
    y, saved = f.forward_train(x)
    want = definition(f, x, dy)
    close(y, want["y"], "y")
    for name, got in zip(("dx", "dw_gu", "dw_down"), f.backward(dy, saved)):
        close(got, want[name], name)


# tiles of 160 and 192 columns, a last tile of few rows and few columns, all on CTA pairs
@pytest.mark.parametrize("M,H,I", [(4096, 2560, 640), (2047, 4096, 4104), (3000, 1032, 1096), (1153, 2568, 1288)])
def test_large(M, H, I):
    f, x, dy = make(M, H, I, H, 2)
    y, saved = f.forward_train(x)
    assert torch.equal(y, f(x))
    want = definition(f, x, dy)
    close(y, want["y"], "y")
    for name, got in zip(("dx", "dw_gu", "dw_down"), f.backward(dy, saved)):
        close(got, want[name], name)


def test_gradients_against_differences():
    """sum(y * dy) along a direction of every input, by central differences of the 64-bit block."""
    f, x, dy = make(24, 128, 64, 96, 3)
    _, saved = f.forward_train(x)
    grads = f.backward(dy, saved)
    at = [x.double(), f.w_gu.double(), f.w_down.double()]

    def value(a, wgu, wd):
        g, u = a @ wgu[:64].t(), a @ wgu[64:].t()
        return float(((g * torch.sigmoid(g) * u) @ wd.t() * dy.double()).sum())
    sds = definition(f, x, dy)
    for i, (name, grad) in enumerate(zip(("dx", "dw_gu", "dw_down"), grads)):
        d = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(i)).double().to(DEV)
        step = 1e-5
        up, down = ([t + (s * step * d if j == i else 0) for j, t in enumerate(at)] for s in (1, -1))
        slope = (value(*up) - value(*down)) / (2 * step)
        dev = ((U * sds[name][0].abs() + sds[name][1]) * d.abs()).norm()
        assert abs(float((grad.double() * d).sum()) - slope) <= 6 * float(dev)


def test_extreme_gates():
    """Gates far from zero: the sigmoid saturates without an overflow, and no NaN appears."""
    from fnx.gated_ffn import GatedFFN
    I = 64
    w_gu = torch.zeros(2 * I, 8, dtype=BF16, device=DEV)
    w_gu[:I, 0] = 1
    w_gu[I:, 1] = 1
    f = GatedFFN(w_gu, torch.eye(I, device=DEV).to(BF16))
    gates = torch.tensor([-1e4, -200., -88.8, -1., 0., 1., 88.8, 200., 1e4])
    x = torch.zeros(len(gates), 8)
    x[:, 0], x[:, 1] = gates, 2
    x = x.to(BF16).to(DEV)
    y, saved = f.forward_train(x)
    g = x[:, :1].double()
    want = 2 * g * torch.sigmoid(g)
    assert bool(((y.double() - want).abs() <= U * want.abs() + 1e-30).all())
    for t in f.backward(torch.ones_like(y), saved):
        assert bool(t.isfinite().all())


def test_rows_that_are_not_finite_stay_in_their_rows():
    f, x, dy = make(300, 64, 128, 64, 4)
    want = f(x)
    x[7, 3] = float("nan")
    x[290, 0] = float("inf")
    got = f(x)
    keep = torch.ones(300, dtype=torch.bool)
    keep[[7, 290]] = False
    assert torch.equal(got[keep], want[keep]) and bool(got[7].isnan().all())


def test_shapes_strides_and_empty():
    f, x, dy = make(6, 128, 64, 96, 5)
    y = f(x)
    assert torch.equal(f(x.view(2, 3, 128)).view(6, 96), y) and torch.equal(f(x.float()), y)
    wide = torch.zeros(6, 304, dtype=BF16, device=DEV)
    for off in (8, 3):
        wide[:, off:off + 128] = x
        assert torch.equal(f(wide[:, off:off + 128]), y)
    assert torch.equal(f(x.t().contiguous().t()), y)
    assert f(x[:0]).shape == (0, 96)
    y3, saved = f.forward_train(x.view(3, 2, 128))
    dx, dwg, dwd = f.backward(dy.view(3, 2, 96), saved)
    assert y3.shape == (3, 2, 96) and dx.shape == (3, 2, 128)
    only = f.backward(dy, saved, need=(False, True, False))
    assert only[0] is None and only[2] is None and torch.equal(only[1], dwg)
    y0, saved0 = f.forward_train(x[:0])
    dx0, dwg0, dwd0 = f.backward(y0, saved0)
    assert dx0.shape == (0, 128) and not dwg0.any() and not dwd0.any()


def test_nothing_behind_the_last_row_is_written():
    """The library writes M rows into a larger buffer and leaves the rest as it was."""
    from fnx import _lib
    f, x, _ = make(37, 64, 72, 40, 6)
    h = torch.full((64, 72), 7.0, dtype=BF16, device=DEV)
    y = torch.full((64, 40), 7.0, dtype=BF16, device=DEV)
    rc = _lib.lib().fnx_gated_ffn(x.data_ptr(), 64, f.w_gu.data_ptr(), f.w_down.data_ptr(), h.data_ptr(), None,
                                  y.data_ptr(), 37, 64, 72, 40, _lib.stream(x.device))
    assert rc == 0 and bool((h[37:] == 7).all()) and bool((y[37:] == 7).all()) and torch.equal(y[:37], f(x))


def test_deterministic_on_other_streams_and_in_graphs():
    f, x, dy = make(200, 256, 136, 256, 7)

    def step():
        y, saved = f.forward_train(x)
        return (y,) + f.backward(dy, saved)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    for a, b, c, d in zip(want, other, held, step()):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)
    x.mul_(0.5)
    graph.replay()
    for a, b in zip(held, step()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("M,H,I", [(1, 512, 256), (40, 1024, 512), (300, 512, 256), (2048, 1024, 1024)])
def test_inputs_and_weights_written_just_before_and_just_after_a_call(M, H, I):
    """Launches overlap the ends of the kernels before them: a step must see weights and rows that the
    kernel just before it wrote, and the kernel behind it must not overwrite what it still reads."""
    from fnx.gated_ffn import GatedFFN
    two = [make(M, H, I, H, 8 + i) for i in range(2)]

    def step(f, x, dy):
        y, saved = f.forward_train(x)
        return (y, f(x)) + f.backward(dy, saved)
    want = [step(*t) for t in two]
    f = GatedFFN(torch.empty_like(two[0][0].w_gu), torch.empty_like(two[0][0].w_down))
    x, dy = torch.empty_like(two[0][1]), torch.empty_like(two[0][2])
    for i in range(12):
        src = two[i % 2]
        for dst, s in ((x, src[1]), (dy, src[2]), (f.w_gu, src[0].w_gu), (f.w_down, src[0].w_down)):
            dst.copy_(s)
        got = step(f, x, dy)
        for dst in (f.w_down, f.w_gu, x, dy):
            dst.fill_(float("nan"))
        for a, b in zip(got, want[i % 2]):
            assert torch.equal(a, b)
    f.w_gu.copy_(two[0][0].w_gu)
    for i in range(12):                               # the down weights last, right before a forward
        f.w_down.copy_(two[0][0].w_down)
        y = f(two[0][1])
        f.w_down.fill_(float("nan"))
        assert torch.equal(y, want[0][1])


def test_offsets_past_32_bits():
    """More than 2^31 elements of output, of kept pre-activations and of their gradients."""
    f, _, _ = make(1, 64, 2056, 1032, 9)
    M = 2 ** 20 + 77
    x = torch.zeros(M, 64, dtype=BF16, device=DEV)
    dy = torch.zeros(M, 1032, dtype=BF16, device=DEV)
    g = torch.Generator().manual_seed(9)
    for at in (0, M // 2, M - 200):
        x[at:at + 200] = torch.randn(200, 64, generator=g).to(BF16).to(DEV)
        dy[at:at + 200] = torch.randn(200, 1032, generator=g).to(BF16).to(DEV)
    h = f.gated(x)
    assert h.numel() > 2 ** 31
    for at in (0, M // 2, M - 200):
        close(h[at:at + 200], definition(f, x[at:at + 200])["h"], "h")
    del h
    y, saved = f.forward_train(x)
    dx = f.backward(dy, saved, need=(True, False, False))[0]
    for at in (0, M // 2, M - 200):
        want = definition(f, x[at:at + 200], dy[at:at + 200])
        close(y[at:at + 200], want["y"], "y")
        close(dx[at:at + 200], want["dx"], "dx")


def test_no_device_error_was_recorded():
    from fnx import _lib
    assert _lib.device_errors() == 0
