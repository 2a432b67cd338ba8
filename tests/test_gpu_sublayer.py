"""The dense operators together, as a feed-forward sublayer uses them: residual and norms, the gated
block, the residual again, forwards and backwards, against the same chain in 64 bits; and the decode form
of it with 4-bit projections.

Tolerance: relative L2.  A rounding to bf16 is off by at most 2^-8 of a value and, uniform over the
binade, 2^-8 / sqrt(3) in the mean square; the operators are norms, sums with random signs and smooth
gates, which hand a relative error on about as large as it came.  A result behind n roundings is then
within n * 2^-8 / sqrt(3)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"
STEP = 2 ** -8 / 3 ** 0.5


def rms64(v, w, eps=1e-6):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * (1 + w)


def near(got, want, roundings):
    assert got.shape == want.shape and got.dtype == BF16
    assert float((got.double() - want).norm() / want.norm()) <= roundings * STEP


def tensors(seed, *specs):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*shape, generator=g) * std).to(BF16).to(DEV) for std, shape in specs]


@pytest.mark.parametrize("b,H,I", [(3, 256, 136), (65, 512, 264), (500, 1024, 512)])
@pytest.mark.parametrize("captured", [False, True])
def test_training_step(b, H, I, captured):
    from fnx.gated_ffn import GatedFFN
    from fnx.native_inject import inject_norm, inject_norm_backward
    hyper, gate, values, w_next, w_post, w_gu, w_down, d_out = tensors(
        b, (1, (b, 1, H)), (1, (b, 1, 1)), (1, (b, 1, H)), (.1, (H,)), (.1, (H,)), (H ** -.5, (2 * I, H)),
        (I ** -.5, (H, I)), (.1, (b, 1, H)))
    ffn = GatedFFN(w_gu, w_down)

    def step():
        state, normed = inject_norm(hyper, gate, values, w_next, w_post=w_post, scale=0.5)
        y, saved = ffn.forward_train(normed)
        out, _ = inject_norm(state, None, y)
        d_state, _, dy, _, _ = inject_norm_backward(d_out, None, out, None, y)
        dx, dw_gu, dw_down = ffn.backward(dy, saved)
        d_hyper, d_gate, d_values, d_w_next, d_w_post = inject_norm_backward(
            d_state, dx, state, gate, values, w_next, w_post=w_post, scale=0.5)
        return out, d_hyper, d_gate, d_values, d_w_next, d_w_post, dw_gu, dw_down
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for t in got:
            t.zero_()
        graph.replay()
    else:
        got = step()
    leaves = [t.double().requires_grad_() for t in (hyper, gate, values, w_next, w_post, w_gu, w_down)]
    h, g, v, wn, wp, wgu, wd = leaves
    state = h + 0.5 * g * rms64(v, wp)
    a, u = (rms64(state, wn) @ wgu.t()).split(I, -1)
    out = state + (a * torch.sigmoid(a) * u) @ wd.t()
    want = (out.detach(),) + torch.autograd.grad(out, leaves, d_out.double())
    # roundings: out normed, h, y, state, itself; gradients those and dy, [dg du], dx, the state's, their own
    near(got[0], want[0], 5)
    for x, w in zip(got[1:], want[1:]):
        near(x, w, 10)


@pytest.mark.parametrize("b", [1, 5, 16])
def test_decode_step_in_four_bits(b):
    from fnx.engine import DenseW4
    from fnx.native_inject import inject_norm
    H, I, gs = 512, 384, 64
    g = torch.Generator().manual_seed(b)

    def dense(K, N):
        w = torch.randint(-2 ** 31, 2 ** 31, (K, N // 8), generator=g, dtype=torch.int64).to(torch.int32)
        s = (torch.rand(K // gs, N, generator=g) * 0.5 * K ** -0.5).to(BF16)
        return DenseW4(w.to(DEV), s.to(DEV), gs)
    gate_up = DenseW4.merge([dense(H, I), dense(H, I)])
    down = dense(I, H)
    hyper, values, w_next, w_after = tensors(b, (1, (b, 1, H)), (1, (b, 1, H)), (.1, (H,)), (.1, (H,)))
    state, normed = inject_norm(hyper, None, values, w_next)
    a, u = gate_up(normed).split(I, -1)
    act = (torch.nn.functional.silu(a.float()) * u.float()).to(BF16)
    out, nxt = inject_norm(state, None, down(act), w_after)
    st = hyper.double() + values.double()
    a, u = (rms64(st, w_next.double()) @ gate_up.deq_w().double().t()).split(I, -1)
    want = st + (a * torch.sigmoid(a) * u) @ down.deq_w().double().t()
    near(out, want, 7)                                # state, normed, gate, up, act, down, itself
    near(nxt, rms64(want, w_after.double()), 7)


FIRST_CALLS = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from fnx.engine import DenseW4
from fnx.gated_ffn import GatedFFN
from fnx.native_inject import inject_norm, inject_norm_backward
r = lambda *s: (torch.randn(*s, device="cuda") * .1).bfloat16()
ring = DenseW4(torch.randint(-2 ** 31, 2 ** 31, (4096, 512), device="cuda").int(), r(64, 4096), 64)
short = DenseW4(torch.randint(-2 ** 31, 2 ** 31, (256, 32), device="cuda").int(), r(4, 256), 64)
ffn, x, wide, wn = GatedFFN(r(512, 256), r(256, 256)), r(300, 256), r(3, 4096), r(256)

def step():
    state, normed = inject_norm(x, None, x, wn)
    y, saved = ffn.forward_train(normed)
    return (ring(wide), short(normed[:3]), state, y, *ffn.backward(y, saved),
            *[t for t in inject_norm_backward(y, None, state, None, x, wn) if t is not None])

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture():
    """What a first call sets up (shared-memory limits, occupancy) may be asked for while a stream captures."""
    import subprocess
    import sys
    from pathlib import Path

    import fnx
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS, str(Path(fnx.__file__).parents[1])], capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stderr[-2000:]
