"""The dense half of a feed-forward sublayer, measured: 4-bit matrix-vector products
(``fnx.engine.DenseW4``), the bf16 gated feed-forward block with its gradients
(``fnx.gated_ffn.GatedFFN``) and the gated residual with the norms around it
(``fnx.native_inject.inject_norm``).

Every case runs in two forms: plainly, in elementary torch operations in fp32 rounded once at the
end (``own = False``), or through this repository's kernels (``own = True``)."""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
PKG = Path("qwen-ascend_b200").resolve()


def _package():
    if str(PKG) not in sys.path:
        sys.path.insert(0, str(PKG))
    from fnx import engine, gated_ffn, native_inject
    return engine, gated_ffn, native_inject


def listed():
    return [
        # one decoded token through the concatenated qkv + z projection, in 4 bits
        dict(name="w4 one token", op="w4", M=1, K=2048, N=5120, gs=128),
        # a few tokens, a ragged last scale group and a width that fills no tile
        dict(name="w4 ragged", op="w4", M=3, K=2504, N=1288, gs=64),
        # the largest decode batch through a wide projection with fine scale groups
        dict(name="w4 wide batch", op="w4", M=16, K=4096, N=28672, gs=32),
        # one decoded token through an always-on expert of the production width
        dict(name="ffn one token", op="ffn", M=1, H=2560, I=640),
        # a decode batch through a wide dense block: every weight is read for 16 tokens
        dict(name="ffn decode batch", op="ffn", M=16, H=4096, I=11008),
        # a prefill chunk through the always-on expert
        dict(name="ffn prefill shared", op="ffn", M=4096, H=2560, I=640),
        # a long ragged prefill through a wide dense block
        dict(name="ffn prefill wide", op="ffn", M=8191, H=4096, I=8192),
        # a short ragged training batch: forward, then all gradients
        dict(name="ffn train short", op="ffn_train", M=509, H=2048, I=512),
        # a training step of a wide block
        dict(name="ffn train wide", op="ffn_train", M=4096, H=4096, I=8192),
        # one decoded token's residual and the next block's norm
        dict(name="inject one token", op="inject", T=1, H=2560, HC=4, post=False),
        # a prefill chunk, with a norm behind the block as well
        dict(name="inject prefill", op="inject", T=8192, H=2560, HC=4, post=True),
        # a training step of the same, ragged
        dict(name="inject train", op="inject_train", T=4095, H=2048, HC=4, post=True),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["w4", "w4", "ffn", "ffn", "ffn_train", "inject", "inject_train"])
    if op == "w4":
        gs = rng.choice([32, 64, 128])
        return dict(op=op, M=_log(rng, 1, 16), K=_log(rng, 512, 8192, 8), N=_log(rng, 512, 28672, 8), gs=gs)
    if op == "ffn":
        return dict(op=op, M=_log(rng, 1, 8192), H=_log(rng, 512, 4096, 8), I=_log(rng, 256, 11008, 8))
    if op == "ffn_train":
        return dict(op=op, M=_log(rng, 64, 4096), H=_log(rng, 512, 4096, 8), I=_log(rng, 256, 8192, 8))
    return dict(op=op, T=_log(rng, 1, 8192) if op == "inject" else _log(rng, 64, 4096), H=_log(rng, 512, 4096, 8),
                HC=rng.choice([1, 2, 4]), post=rng.random() < 0.5)


def _normal(g, shape, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(BF16)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    s = dict(case)
    if op == "w4":
        M, K, N, gs = case["M"], case["K"], case["N"], case["gs"]
        words = torch.randint(-2 ** 31, 2 ** 31, (K, N // 8), generator=g, device=DEV, dtype=torch.int64)
        s["w4"] = words.to(torch.int32)                    # eight uniform int4 values a word
        s["scales"] = (torch.randn((-(-K // gs), N), generator=g, device=DEV).abs() * 0.02).to(BF16)
        s["x"] = _normal(g, (M, K))
        if own:
            s["layer"] = _package()[0].DenseW4(s["w4"], s["scales"], gs)
    elif op in ("ffn", "ffn_train"):
        M, H, I = case["M"], case["H"], case["I"]
        s["x"] = _normal(g, (M, H))
        s["w_gu"] = _normal(g, (2 * I, H), H ** -0.5)      # gate rows, then up rows
        s["w_down"] = _normal(g, (H, I), I ** -0.5)
        if op == "ffn_train":
            s["dy"] = _normal(g, (M, H), 0.01)
        if own:
            s["layer"] = _package()[1].GatedFFN(s["w_gu"], s["w_down"])
    else:
        T, H, HC = case["T"], case["H"], case["HC"]
        loud = 1.0 + 15.0 * (torch.rand((HC * H,), generator=g, device=DEV) < 0.005)   # a few loud channels
        s["hyper"] = (torch.randn((T, 1, HC * H), generator=g, device=DEV) * loud).to(BF16)
        s["gate"] = (2 * torch.sigmoid(torch.randn((T, 1, HC), generator=g, device=DEV))).to(BF16)
        s["values"] = _normal(g, (T, 1, H))
        s["w_next"] = _normal(g, (HC * H,), 0.1)
        s["w_post"] = _normal(g, (H,), 0.1) if case["post"] else None
        s["scale"] = 0.5 if case["post"] else 1.0
        if op == "inject_train":
            s["d_state"] = _normal(g, (T, 1, HC * H), 0.01)
            s["d_normed"] = _normal(g, (T, 1, HC * H), 0.01)
        if own:
            s["ops"] = _package()[2]
    return s


EPS = 1e-6


# ------------------------------------------------------------------ plain forms
def _int4(words):
    """int4pack words [K, N/8] -> int32 values [K, N] (nibble t of a word is column 8j + t)."""
    t = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    v = torch.bitwise_right_shift(words[:, :, None], t) & 15
    return ((v + 8) % 16 - 8).reshape(words.shape[0], -1)


def _plain_w4(s):
    w = _int4(s["w4"]).float() * s["scales"].float().repeat_interleave(s["gs"], 0)[:s["K"]]
    return {"y": (s["x"].float() @ w).to(BF16)}


def _plain_ffn(s):
    x, wd = s["x"].float(), s["w_down"].float()
    wgu = s["w_gu"].float()
    gu = x @ wgu.t()
    gate, up = gu[:, :s["I"]], gu[:, s["I"]:]
    sig = 1 / (1 + torch.exp(-gate))
    h = gate * sig * up
    y = h @ wd.t()
    if s["op"] == "ffn":
        return {"y": y.to(BF16)}
    dy = s["dy"].float()
    dh = dy @ wd
    dgu = torch.cat([dh * up * sig * (1 + gate * (1 - sig)), dh * gate * sig], 1)
    return {"y": y.to(BF16), "dx": (dgu @ wgu).to(BF16), "dw_gu": (dgu.t() @ x).to(BF16),
            "dw_down": (dy.t() @ h).to(BF16)}


def _plain_inject(s):
    T, H, HC = s["T"], s["H"], s["HC"]
    v = s["values"].float().view(T, 1, H)
    gate = s["gate"].float().view(T, HC, 1) * s["scale"]
    wn = 1 + s["w_next"].float().view(HC, H)
    z = v
    if s["post"]:
        wp = 1 + s["w_post"].float()
        rv = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
        z = v * rv * wp
    state = s["hyper"].float().view(T, HC, H) + gate * z
    rs = torch.rsqrt((state * state).mean(-1, keepdim=True) + EPS)
    unit = state * rs
    out = {"state": state.view(T, 1, -1).to(BF16), "normed": (unit * wn).view(T, 1, -1).to(BF16)}
    if s["op"] == "inject":
        return out
    dn = s["d_normed"].float().view(T, HC, H)
    dw = dn * wn
    d = s["d_state"].float().view(T, HC, H) + rs * (dw - unit * (dw * unit).mean(-1, keepdim=True))
    dz = (gate * d).sum(1, keepdim=True)
    out["d_hyper"] = d.view(T, 1, -1).to(BF16)
    out["d_gate"] = ((d * z).sum(-1) * s["scale"]).view(T, 1, HC).to(BF16)
    out["d_w_next"] = (dn * unit).sum(0).view(-1).to(BF16)
    if s["post"]:
        uv = v * rv
        du = dz * wp
        out["d_values"] = (rv * (du - uv * (du * uv).mean(-1, keepdim=True))).to(BF16)
        out["d_w_post"] = (dz * uv).sum((0, 1)).to(BF16)
    else:
        out["d_values"] = dz.to(BF16)
    return out


# ------------------------------------------------------------------ this repository's kernels
def _own_inject(s):
    ops = s["ops"]
    state, normed = ops.inject_norm(s["hyper"], s["gate"], s["values"], s["w_next"], w_post=s["w_post"],
                                    scale=s["scale"], eps=EPS)
    out = {"state": state, "normed": normed}
    if s["op"] == "inject_train":
        g = ops.inject_norm_backward(s["d_state"], s["d_normed"], state, s["gate"], s["values"], s["w_next"],
                                     w_post=s["w_post"], scale=s["scale"], eps=EPS)
        out["d_hyper"], out["d_gate"], out["d_values"], out["d_w_next"] = g[:4]
        if s["post"]:
            out["d_w_post"] = g[4]
    return out


def run(state):
    op = state["op"]
    if not own:
        return _plain_w4(state) if op == "w4" else _plain_ffn(state) if op.startswith("ffn") else _plain_inject(state)
    if op == "w4":
        return {"y": state["layer"](state["x"])}
    if op == "ffn":
        return {"y": state["layer"](state["x"])}
    if op == "ffn_train":
        y, saved = state["layer"].forward_train(state["x"])
        dx, dw_gu, dw_down = state["layer"].backward(state["dy"], saved)
        return {"y": y, "dx": dx, "dw_gu": dw_gu, "dw_down": dw_down}
    return _own_inject(state)


def work(case):
    op = case["op"]
    if op == "w4":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": K * N // 2 + -(-K // case["gs"]) * N * 2 + 2 * M * (K + N), "flops": 2 * M * K * N}
    if op.startswith("ffn"):
        M, H, I = case["M"], case["H"], case["I"]
        if op == "ffn":
            return {"bytes": 6 * I * H + 4 * M * H, "flops": 6 * M * I * H}
        return {"bytes": 12 * I * H + 8 * M * H, "flops": 18 * M * I * H}
    T, H, HC = case["T"], case["H"], case["HC"]
    post = H if case["post"] else 0
    fwd = 2 * (T * H * (3 * HC + 1) + T * HC + HC * H + post)
    if op == "inject":
        return {"bytes": fwd, "flops": T * H * (8 * HC + 4)}
    return {"bytes": fwd + 2 * (T * H * (3 * HC + 1) + T * HC + HC * H + post), "flops": T * H * (30 * HC + 12)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _rms64(v, w):
    n = v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / v.shape[-1] + EPS)
    return n * (w + 1.0)


def exact(case, seed):
    s = prepare(case, seed)
    f = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    op = case["op"]
    if op == "w4":
        K, N, gs = case["K"], case["N"], case["gs"]
        y = torch.zeros(case["M"], N, device=DEV, dtype=torch.float64)
        u = s["w4"].to(torch.int64) & 0xFFFFFFFF
        for t in range(8):                                 # column 8j + t: nibble t, two's complement
            q = (u >> (4 * t)) & 15
            q = torch.where(q > 7, q - 16, q).double()
            for a in range(0, K, gs):
                y[:, t::8] += (f["x"][:, a:a + gs] @ q[a:a + gs]) * f["scales"][a // gs, t::8]
        return {"y": y}
    if op.startswith("ffn"):
        I = case["I"]
        leaves = [f[k].requires_grad_(op == "ffn_train") for k in ("x", "w_gu", "w_down")]
        a = torch.matmul(leaves[0], leaves[1][:I].T)
        h = a / (1.0 + torch.exp(-a)) * torch.matmul(leaves[0], leaves[1][I:].T)
        y = torch.matmul(h, leaves[2].T)
        if op == "ffn":
            return {"y": y}
        dx, dgu, dd = torch.autograd.grad(y, leaves, f["dy"])
        return {"y": y.detach(), "dx": dx, "dw_gu": dgu, "dw_down": dd}
    T, H, HC = case["T"], case["H"], case["HC"]
    names = ["hyper", "gate", "values", "w_next"] + (["w_post"] if case["post"] else [])
    leaves = {k: f[k].requires_grad_(op == "inject_train") for k in names}
    z = leaves["values"]
    if case["post"]:
        z = _rms64(z, leaves["w_post"])
    parts = [leaves["hyper"][..., b * H:(b + 1) * H] + s["scale"] * leaves["gate"][..., b:b + 1] * z for b in range(HC)]
    normed = [_rms64(p, leaves["w_next"][b * H:(b + 1) * H]) for b, p in enumerate(parts)]
    out = {"state": torch.cat(parts, -1), "normed": torch.cat(normed, -1)}
    if op == "inject_train":
        grads = torch.autograd.grad([out["state"], out["normed"]], [leaves[k] for k in names],
                                    [f["d_state"], f["d_normed"]])
        out = {k: v.detach() for k, v in out.items()}
        out.update({"d_" + k: v for k, v in zip(names, grads)})
    return out
