"""The 4-bit dense feed-forward block, the 4-bit matrix products and the rotary positions,
as cases to be timed and compared.

`run` computes each operator in elementary torch operations in 32 bits, or, with `own`,
through this package's entry points:

  ffn     y = (act(x Wg^T) * (x Wu^T)) Wd^T, Wg / Wu [I, H] and Wd [H, I] in 4 bits with
          scales and biases per group; with `grad` also the gradients of a training step
          through the frozen weights: dx, and those of the two projections' outputs.
  matmul  y = x W^T (`transpose`), or y = x W (the gradient's direction), W in 4 bits.
  rope    rotary positions over the first `dims` channels of each head; `inverse` is the
          transposed rotation, the gradient's.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one token's attention output projection in a decoder of hidden size 2048
        dict(name="matmul_1", op="matmul", M=1, N=2048, K=2048, group=32, dtype="bf16", biases=True, transpose=True),
        # one token's vocabulary logits
        dict(name="matmul_1_head", op="matmul", M=1, N=32768, K=2048, group=128, dtype="bf16", biases=True, transpose=True),
        # a ragged decode batch, an odd number of outputs, symmetric weights without biases
        dict(name="matmul_21_odd", op="matmul", M=21, N=1001, K=1408, group=64, dtype="f16", biases=False, transpose=True),
        # the input's gradient of a projection over a short training batch
        dict(name="matmul_512_back", op="matmul", M=512, N=2048, K=5632, group=32, dtype="bf16", biases=True, transpose=False),
        # a dense layer, one decode token (hidden 2048, intermediate 5632)
        dict(name="ffn_1", op="ffn", T=1, H=2048, I=5632, group=64, dtype="bf16", act="silu", grad=False),
        # a small dense layer with the GELU activation, a decode batch of 8
        dict(name="ffn_8_gelu", op="ffn", T=8, H=2048, I=1792, group=32, dtype="f16", act="gelu", grad=False),
        # a dense layer over a 512-token prompt
        dict(name="ffn_512", op="ffn", T=512, H=2048, I=5632, group=64, dtype="bf16", act="silu", grad=False),
        # training step of adapters around a small dense layer, ragged number of tokens
        dict(name="ffn_333_grad", op="ffn", T=333, H=2048, I=768, group=128, dtype="f16", act="gelu", grad=True),
        # the same around a full dense layer, 4096 tokens
        dict(name="ffn_4096_grad", op="ffn", T=4096, H=2048, I=5632, group=64, dtype="bf16", act="silu", grad=True),
        # 64 sequences at positions of their own, one new token each, long-context frequencies
        dict(name="rope_decode_64", op="rope", B=64, L=1, heads=36, D=128, dims=128, dtype="bf16", interleaved=False,
             scale=1.0, mscale=1.25, far=1000000, freqs=True, inverse=False),
        # a 4096-token prompt: query and key heads read out of the fused projection
        dict(name="rope_4096", op="rope", B=1, L=4096, heads=36, D=128, dims=128, dtype="bf16", interleaved=False,
             scale=1.0, mscale=1.0, far=0, freqs=False, inverse=False),
        # gradient of a partial, interleaved rotation with interpolated positions
        dict(name="rope_1023_back", op="rope", B=2, L=1023, heads=16, D=80, dims=64, dtype="f32", interleaved=True,
             scale=0.25, mscale=1.0, far=5000, freqs=False, inverse=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["matmul", "matmul", "ffn", "ffn", "ffn", "rope"])
    group = rng.choice([32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "matmul":
        M, N, K = _log(rng, 1, 2048), _log(rng, 40, 32768), group * _log(rng, 2, 8192 // group)
        transpose = rng.random() < 0.7
        if dtype == "bf16" and transpose and group == 64:
            group = 32  # that form is the package's earlier operator
        if not transpose:
            N = group * max(1, N // group)
        while M * N * K > 4096 * 2048 * 5632:
            M = max(1, M // 2)
        return dict(op=op, M=M, N=N, K=K, group=group, dtype=dtype, biases=rng.random() < 0.8, transpose=transpose)
    if op == "ffn":
        T = _log(rng, 1, 4096)
        H, I = group * _log(rng, 2, 4096 // group), group * _log(rng, 2, 8192 // group)
        while T * H * I > 4096 * 2048 * 5632:
            T = max(1, T // 2)
        return dict(op=op, T=T, H=H, I=I, group=group, dtype=dtype, act=rng.choice(["silu", "gelu"]),
                    grad=rng.random() < 0.4)
    D = 2 * rng.randint(16, 128)
    dims = D if rng.random() < 0.6 else 2 * rng.randint(8, D // 2)
    B, heads = _log(rng, 1, 64), _log(rng, 1, 48)
    L = _log(rng, 1, max(1, min(8192, 4096 * 48 // (B * heads))))
    return dict(op="rope", B=B, L=L, heads=heads, D=D, dims=dims, dtype=rng.choice(["bf16", "f16", "f32"]),
                interleaved=rng.random() < 0.4, scale=rng.choice([1.0, 0.25, 0.125]), mscale=rng.choice([1.0, 1.25]),
                far=rng.choice([0, 5000, 1000000]), freqs=rng.random() < 0.5, inverse=rng.random() < 0.3)


class _Linear:
    """One 4-bit matrix [rows, cols]: words of 8 fields, lowest bits first, scale and bias per group."""

    def __init__(self, gen, rows, cols, group, dtype, biases=True):
        self.group = group
        self.w = torch.randint(-2 ** 31, 2 ** 31, (rows, cols // 8), dtype=torch.int32, device="cuda", generator=gen)
        scales = (torch.randn(rows, cols // group, device="cuda", generator=gen) * 0.02).abs()
        self.scales = scales.to(DTYPES[dtype])
        # zero points between 7 and 9, as fitted weights have them
        zero = 7.0 + 2.0 * torch.rand(rows, cols // group, device="cuda", generator=gen)
        self.biases = (-zero * self.scales.float()).to(DTYPES[dtype]) if biases else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    s = dict(case=case)
    if case["op"] == "matmul":
        rows, cols = (case["N"], case["K"]) if case["transpose"] else (case["K"], case["N"])
        s["W"] = _Linear(gen, rows, cols, case["group"], case["dtype"], case["biases"])
        s["x"] = normal(case["M"], case["K"])
    elif case["op"] == "ffn":
        H, I, g = case["H"], case["I"], case["group"]
        s["gate"], s["up"] = (_Linear(gen, I, H, g, case["dtype"]) for _ in range(2))
        s["down"] = _Linear(gen, H, I, g, case["dtype"])
        s["x"] = normal(case["T"], H)
        if case["grad"]:
            s["dy"] = normal(case["T"], H)
        if own:
            from mlx_rs_b200.block import DenseMlp
            from mlx_rs_b200.synth import QWeight
            q = [QWeight(l.w, l.scales, l.biases) for l in (s["gate"], s["up"], s["down"])]
            s["mlp"] = DenseMlp(*q, activation=case["act"], group_size=g)
    else:
        B, L, h, D = case["B"], case["L"], case["heads"], case["D"]
        # query and key heads lie in front of the value heads in each token's fused projection
        s["x"] = normal(B, L, (h + (h + 7) // 8) * D)
        s["offset"] = torch.randint(0, case["far"] + 1, (B,), dtype=torch.int32, device="cuda", generator=gen)
        s["freqs"] = None
        if case["freqs"]:  # wavelengths stretched from the middle of the head on
            i = torch.arange(0, case["dims"], 2, dtype=torch.float64, device="cuda")
            f = 500000.0 ** (i / case["dims"])
            s["freqs"] = (f * (1.0 + 7.0 * (f / f.max()).sqrt())).float()
    return s


def _dense(l, cols):
    """The matrix in 32 bits."""
    shift = torch.arange(0, 32, 4, dtype=torch.int32, device=l.w.device)
    q = ((l.w[:, :, None] >> shift) & 15).reshape(l.w.shape[0], cols // l.group, l.group).float()
    w = q * l.scales.float()[:, :, None]
    if l.biases is not None:
        w = w + l.biases.float()[:, :, None]
    return w.reshape(l.w.shape[0], cols)


GELU_C = math.sqrt(2.0 / math.pi)


def _act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1.0 + g * (1.0 - s))
    t = torch.tanh(GELU_C * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * GELU_C * (1.0 + 0.134145 * g * g)


def _plain_ffn(s, case):
    dt, H, I = s["x"].dtype, case["H"], case["I"]
    wg, wu, wd = _dense(s["gate"], H), _dense(s["up"], H), _dense(s["down"], I)
    x = s["x"].float()
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, case["act"])
    out = {"out": ((a * u) @ wd.T).to(dt)}
    if case["grad"]:
        dh = s["dy"].float() @ wd
        dg, du = dh * u * da, dh * a
        out |= {"dx": (dg @ wg + du @ wu).to(dt), "dgate": dg.to(dt), "dup": du.to(dt)}
    return out


def _heads(s, case):
    B, L, h, D = case["B"], case["L"], case["heads"], case["D"]
    return s["x"].view(B, L, -1, D)[:, :, :h].transpose(1, 2)  # [B, heads, L, D]


def _plain_rope(s, case):
    x, L, dims = _heads(s, case), case["L"], case["dims"]
    # angles in 64 bits: far positions lose whole turns' worth of digits in 32
    pos = (s["offset"].double()[:, None] + torch.arange(L, device=x.device)) * case["scale"]
    i = torch.arange(0, dims, 2, dtype=torch.float64, device=x.device)
    inv = 1.0 / s["freqs"].double() if s["freqs"] is not None else 10000.0 ** (-i / dims)
    ang = pos[:, None, :, None] * inv
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    if case["inverse"]:
        sin = -sin
    v = x[..., :dims].float()
    if case["interleaved"]:
        a, b = v[..., 0::2], v[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = v[..., :dims // 2], v[..., dims // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([(r * case["mscale"]).to(x.dtype), x[..., dims:]], -1)


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "matmul":
            W, x = state["W"], state["x"].float()
            w = _dense(W, case["K"] if case["transpose"] else case["N"])
            return (x @ (w.T if case["transpose"] else w)).to(state["x"].dtype)
        return _plain_ffn(state, case) if case["op"] == "ffn" else _plain_rope(state, case)
    from mlx_rs_b200 import ops
    if case["op"] == "matmul":
        W = state["W"]
        return ops.quantized_matmul(state["x"], W.w, W.scales, W.biases, transpose=case["transpose"],
                                    group_size=case["group"])
    if case["op"] == "ffn":
        if not case["grad"]:
            return {"out": state["mlp"](state["x"])}
        out, saved = state["mlp"].forward_saved(state["x"])
        dx, dgate, dup = state["mlp"].vjp(saved, state["dy"])
        return {"out": out, "dx": dx, "dgate": dgate, "dup": dup}
    return ops.fast_rope(_heads(state, case), case["dims"], traditional=case["interleaved"], base=10000.0,
                         scale=case["scale"], offset=state["offset"], freqs=state["freqs"], mscale=case["mscale"],
                         inverse=case["inverse"])


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "rope":
        n = case["B"] * case["L"] * case["heads"]
        return {"bytes": 2 * n * case["D"] * e, "flops": 3 * n * case["dims"]}
    if case["op"] == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        per = 0.5 + (4 if case["biases"] else 2) / case["group"]
        return {"bytes": N * K * per + M * (N + K) * e, "flops": 2 * M * N * K}
    T, H, I = case["T"], case["H"], case["I"]
    weights = 3 * H * I * (0.5 + 4 / case["group"])
    if case["grad"]:  # x and dy in; out, dx and the two projections' gradients out
        return {"bytes": weights + (4 * T * H + 2 * T * I) * e, "flops": 12 * T * H * I}
    return {"bytes": weights + 2 * T * H * e, "flops": 6 * T * H * I}


def _exact_matrix(l):
    """The matrix in 64 bits, from its bytes: the low half of a byte is the earlier element."""
    b = l.w.contiguous().view(torch.uint8)
    q = torch.stack([b % 16, b // 16], -1).reshape(l.w.shape[0], -1).double()
    w = q * l.scales.double().repeat_interleave(l.group, 1)
    return w if l.biases is None else w + l.biases.double().repeat_interleave(l.group, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "matmul":
        w = _exact_matrix(s["W"])
        return torch.matmul(s["x"].double(), w.t() if case["transpose"] else w)
    if case["op"] == "ffn":
        wg, wu, wd = (_exact_matrix(s[k]) for k in ("gate", "up", "down"))
        x = s["x"].double()
        g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
        if case["act"] == "silu":
            sig = 1.0 / (1.0 + torch.exp(-g))
            a, slope = g * sig, sig + g * sig * (1.0 - sig)
        else:  # 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z))
            z2 = 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)
            sig = 1.0 / (1.0 + torch.exp(-z2))
            a = g * sig
            slope = sig + g * sig * (1.0 - sig) * 2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * g ** 2)
        out = {"out": torch.matmul(a * u, wd.t())}
        if case["grad"]:
            dh = torch.matmul(s["dy"].double(), wd)
            out["dgate"], out["dup"] = dh * u * slope, dh * a
            out["dx"] = torch.matmul(out["dgate"], wg) + torch.matmul(out["dup"], wu)
        return out
    x, dims, L = _heads(s, case).double(), case["dims"], case["L"]
    k = torch.arange(dims // 2, dtype=torch.float64, device=x.device)
    rate = torch.exp(-2.0 * k / dims * math.log(10000.0)) if s["freqs"] is None else 1.0 / s["freqs"].double()
    at = s["offset"].double().reshape(-1, 1, 1) + torch.arange(L, device=x.device, dtype=torch.float64).reshape(1, L, 1)
    turn = torch.polar(torch.full((), case["mscale"], dtype=torch.float64, device=x.device).expand(case["B"], L, dims // 2),
                       (at * case["scale"] * rate) * (-1.0 if case["inverse"] else 1.0))[:, None]
    if case["interleaved"]:
        z = torch.view_as_complex(x[..., :dims].contiguous().unflatten(-1, (dims // 2, 2)))
        r = torch.view_as_real(z * turn).flatten(-2)
    else:
        z = torch.complex(x[..., :dims // 2].contiguous(), x[..., dims // 2:dims].contiguous()) * turn
        r = torch.cat([z.real, z.imag], -1)
    return torch.cat([r, x[..., dims:]], -1)
