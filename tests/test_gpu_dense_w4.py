"""``DenseW4`` against its definition in 64 bits.

Tolerance per element: one rounding to bf16 (2^-8 relative) of a sum that was accumulated in fp32:
at most K/16 tensor-core steps, G group sums and 64 parts are added one after another, each step off
by at most 2^-22 of the sum of the magnitudes so far (2^-23 for a truncated fp32 addition, twice that
for the products added within one step)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"


def layer(K, N, gs, seed=0):
    from fnx.engine import DenseW4
    g = torch.Generator().manual_seed(seed + K + N + gs)
    w = torch.randint(-2 ** 31, 2 ** 31, (K, N // 8), generator=g, dtype=torch.int64).to(torch.int32)
    s = (torch.randn(-(-K // gs), N, generator=g).abs() * 0.02).to(BF16)
    return DenseW4(w.to(DEV), s.to(DEV), gs), w, s


def values64(w, s, gs):
    """From the words by arithmetic, in 64 bits on the CPU."""
    u = w.long() & 0xFFFFFFFF
    q = torch.stack([(u >> (4 * t)) & 15 for t in range(8)], -1).reshape(w.shape[0], -1)
    q = torch.where(q > 7, q - 16, q).double()
    return q * s.double()[torch.arange(w.shape[0]) // gs]


def check(lay, w, s, gs, x):
    K = w.shape[0]
    W = values64(w, s, gs).to(DEV)
    y = lay(x)
    xd = x.double().reshape(-1, K)
    want, mag = xd @ W, xd.abs() @ W.abs()
    lim = 2 ** -8 * want.abs() + (K / 16 + s.shape[0] + 64) * 2 ** -22 * mag
    err = (y.double().reshape(want.shape) - want).abs()
    assert y.dtype == BF16 and y.shape == x.shape[:-1] + (want.shape[1],)
    assert bool((err <= lim).all()), float((err / lim.clamp(min=1e-30)).max())


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 40])
@pytest.mark.parametrize("K,N,gs", [(8, 8, 16), (2048, 5120, 128), (2504, 1288, 64), (520, 24, 32), (640, 2560, 64),
                                    (1032, 4104, 1040)])
def test_matches_the_definition(M, K, N, gs):
    lay, w, s = layer(K, N, gs)
    g = torch.Generator().manual_seed(M)
    check(lay, w, s, gs, torch.randn(M, K, generator=g).to(BF16).to(DEV))


# from 2^24 weights on they come through the ring of copies: ragged K, every N mod 32, groups that end
# inside a stage
@pytest.mark.parametrize("M,K,N,gs", [(9, 5000, 4128, 48), (1, 4104, 4128, 16), (5, 8200, 2080, 4096), (17, 4096, 4104, 32),
                                      (3, 4200, 4112, 64), (12, 4104, 4120, 128), (2, 8408, 2008, 256),
                                      (1, 8192, 28672, 128), (16, 4096, 14336, 32), (3, 2560, 151936, 64)])
def test_wide(M, K, N, gs):
    lay, w, s = layer(K, N, gs)
    check(lay, w, s, gs, torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(BF16).to(DEV))


# fewer rows than a stage holds, by far, and as many columns as bring them to the ring
@pytest.mark.parametrize("M,K,N,gs", [(2, 8, 2097160, 16), (9, 16, 1048608, 128), (1, 24, 699064, 32)])
def test_few_rows_of_many_columns(M, K, N, gs):
    lay, w, s = layer(K, N, gs)
    check(lay, w, s, gs, torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(BF16).to(DEV))


def test_activations_with_a_mean_and_outliers():
    """Values that are all positive, some a thousand times the others: nothing is taken from a large
    sum that the result does not hold itself."""
    lay, w, s = layer(1024, 512, 64)
    x = torch.rand(5, 1024, generator=torch.Generator().manual_seed(2)) + 1
    x[:, ::97] *= 1000
    check(lay, w, s, 64, x.to(BF16).to(DEV))


def test_scales_of_zero_and_extreme_values():
    lay, w, s = layer(256, 256, 32)
    lay.sc[:, 3] = 0
    y = lay(torch.full((2, 256), 1.0, device=DEV, dtype=BF16))
    assert not y[:, 3].any()
    big = torch.zeros(1, 256, device=DEV, dtype=BF16)
    big[0, 9] = 2.0 ** 120                                   # 8 * 2^120 * s stays finite
    want = values64(w, s, 32)[9] * 2.0 ** 120
    got = lay(big)[0].double().cpu()
    keep = torch.arange(256) != 3
    assert bool(((got - want).abs()[keep] <= 2 ** -8 * want.abs()[keep]).all())


def test_shapes_strides_types_and_merge():
    from fnx.engine import DenseW4
    a, wa, sa = layer(512, 128, 64, 1)
    b, wb, sb = layer(512, 264, 64, 2)
    x = torch.randn(2, 3, 512, generator=torch.Generator().manual_seed(3)).to(BF16).to(DEV)
    y = a(x)
    assert y.shape == (2, 3, 128) and torch.equal(y.view(6, 128), a(x.view(6, 512)))
    assert torch.equal(a(x[0].float()), a(x[0]))
    wide = torch.zeros(3, 1032, device=DEV, dtype=BF16)
    wide[:, 8:520] = x[0]
    assert torch.equal(a(wide[:, 8:520]), a(x[0]))
    wide[:, 3:515] = x[0]                                    # rows that start off a 16-byte boundary
    assert torch.equal(a(wide[:, 3:515]), a(x[0]))
    assert torch.equal(a(x[0].t().contiguous().t()), a(x[0]))
    assert a(x[0][:0]).shape == (0, 128)
    m = DenseW4.merge([a, b])
    assert torch.equal(m(x[0]), torch.cat([a(x[0]), b(x[0])], 1))
    assert torch.equal(a.deq_w().double().cpu(), values64(wa, sa, 64).t())


def test_rows_do_not_depend_on_their_batch_and_replay():
    lay, w, s = layer(2048, 1024, 128)
    x = torch.randn(8, 2048, generator=torch.Generator().manual_seed(5)).to(BF16).to(DEV)
    y = lay(x)
    assert torch.equal(y, lay(x))
    for m in range(8):
        assert torch.equal(lay(x[m:m + 1])[0], y[m])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = lay(x)
    x.neg_()
    graph.replay()
    assert torch.equal(held, -y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = lay(x)
    side.synchronize()
    assert torch.equal(z, held)


@pytest.mark.parametrize("K,N", [(512, 256), (4096, 8192)])
def test_inputs_written_just_before_and_just_after_a_call(K, N):
    """A call may start while the kernel before it ends: it must see what that one writes, and the one
    behind it must not overwrite what it still reads."""
    lay, w, s = layer(K, N, 64)
    a, b = (torch.randn(4, K, generator=torch.Generator().manual_seed(i)).to(BF16).to(DEV) for i in (1, 2))
    ya, yb = lay(a), lay(b)
    x = torch.empty_like(a)
    outs = []
    for i in range(40):
        x.copy_(a if i % 2 else b)
        outs.append(lay(x))
        x.fill_(float("nan"))
    for i, y in enumerate(outs):
        assert torch.equal(y, ya if i % 2 else yb)


def test_offsets_past_32_bits():
    """2^31 words and more: the last rows and columns are the ones that a 32-bit offset would miss."""
    from fnx.engine import DenseW4
    K, N, gs = 65536, 263168, 4096
    w = torch.empty(K, N // 8, dtype=torch.int32, device=DEV).random_(-2 ** 31, 2 ** 31 - 1)
    s = torch.full((K // gs, N), 0.01, dtype=BF16, device=DEV)
    x = torch.randn(1, K, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    y = DenseW4(w, s, gs)(x)
    for j in (0, 1, N // 16, N // 8 - 2, N // 8 - 1):
        W = values64(w[:, j:j + 1].cpu(), s[:, 8 * j:8 * j + 8].cpu(), gs).to(DEV)
        want, mag = x.double() @ W, x.double().abs() @ W.abs()
        lim = 2 ** -8 * want.abs() + (K / 16 + K // gs + 64) * 2 ** -22 * mag
        assert bool(((y[:, 8 * j:8 * j + 8].double() - want).abs() <= lim).all())


def test_agrees_with_the_expert_gemm():
    """The same words as one expert of ExpW4, whose weights are rounded to bf16 first (2^-9 each on
    average): the two agree within the layer contract's relative L2 of 5e-3."""
    from fnx.engine import ExpW4
    lay, w, s = layer(2048, 1024, 128)
    e = ExpW4.from_scales(lay.w4[None], lay.sc[None], 128)
    x = torch.randn(16, 2048, generator=torch.Generator().manual_seed(6)).to(BF16).to(DEV)
    a, b = lay(x).float(), e.apply(x, [0]).float()
    assert float((a - b).norm() / b.norm()) < 5e-3
