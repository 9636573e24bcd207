"""The feed-forward operators of a language model as this library offers them, as cases that can be timed and checked:
matrix products in 8-bit integers with a scale for each token and each channel (with the quantisation of the tokens),
and gated feed-forward projections in bf16 (forward and backward) and in int8.

``run`` computes a case in its plain form, elementary torch operations in 32 bits, or, where ``own`` is true, with the
library's entry points.  ``exact`` computes it in 64 bits.  All tensors are dense; weights are stored one output
channel per row ([N, K], [F, K])."""
import math

import torch

own = False

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}  # the library's EXO_B200_ACT_* values


def listed():
    return [
        # one token of a decoding step through a square projection: nothing but latency
        {"name": "linear_token", "op": "linear", "M": 1, "N": 4096, "K": 4096, "type": "bf16", "bias": False},
        # a handful of sequences decoded together, every size odd, float activations
        {"name": "linear_ragged_f32", "op": "linear", "M": 17, "N": 4099, "K": 513, "type": "f32", "bias": True},
        # a prompt of 2048 tokens through an up projection
        {"name": "linear_prompt", "op": "linear", "M": 2048, "N": 8192, "K": 4096, "type": "bf16", "bias": True},
        # tokens that were quantised before (shared by several projections), a pitch that is not a multiple of 16 bytes
        {"name": "product_1000_f32", "op": "product", "M": 1000, "N": 1000, "K": 1000, "type": "f32", "bias": True},
        # the largest product: a long batch of prompts
        {"name": "product_8192", "op": "product", "M": 8192, "N": 8192, "K": 8192, "type": "bf16", "bias": False},
        # one token through the gated projections of a large block: the weights cross the memory bus once
        {"name": "gated_token", "op": "gated", "M": 1, "F": 16384, "K": 4096, "act": "silu", "keep": False},
        # a ragged fine-tuning batch, pre-activations kept for the backward pass
        {"name": "gated_ragged", "op": "gated", "M": 1000, "F": 4099, "K": 513, "act": "gelu", "keep": True},
        # a training step's forward pass
        {"name": "gated_train", "op": "gated", "M": 8192, "F": 8192, "K": 4096, "act": "silu", "keep": True},
        # the backward pass of a small block, as in fine-tuning on short sequences
        {"name": "gated_back_small", "op": "gated_back", "M": 512, "F": 4096, "K": 1024, "act": "gelu_tanh"},
        # a training step's backward pass
        {"name": "gated_back_train", "op": "gated_back", "M": 8192, "F": 8192, "K": 4096, "act": "silu"},
        # sixteen sequences decoded together on int8 weights
        {"name": "gated_i8_decode", "op": "gated_i8", "M": 16, "F": 16384, "K": 4096, "act": "silu"},
        # a prompt of 4096 tokens on int8 weights
        {"name": "gated_i8_prompt", "op": "gated_i8", "M": 4096, "F": 8192, "K": 4096, "act": "gelu_tanh"},
    ]


_MOST_FLOPS = 2.3e12  # what the largest listed case computes
_MOST_BYTES = 1.3e9   # and the most that one of them has to move


def draw(rng):
    def size(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        step = rng.choice((1, 1, 8, 64, 128))  # odd sizes, whole vectors, whole tiles
        return min(hi, max(lo, n // step * step))

    while True:
        op = rng.choice(("linear", "product", "gated", "gated_back", "gated_i8"))
        case = {"op": op, "M": size(1, 8192), "N" if op in ("linear", "product") else "F": size(64, 16384),
                "K": size(64, 8192)}
        if op in ("linear", "product"):
            case["type"] = rng.choice(("bf16", "f32"))
            case["bias"] = rng.random() < 0.5
        else:
            case["act"] = rng.choice(tuple(ACTIVATIONS))
        if op == "gated":
            case["keep"] = rng.random() < 0.5
        w = work(case)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return case


def work(case):
    op, M, K = case["op"], case["M"], case["K"]
    if op in ("linear", "product"):
        N, e = case["N"], 2 if case["type"] == "bf16" else 4
        moved = N * K + 4 * N * (2 if case["bias"] else 1) + 4 * M + M * N * e
        moved += M * K * (e if op == "linear" else 1)
        return {"bytes": moved, "flops": 2 * M * N * K}
    F = case["F"]
    if op == "gated":
        return {"bytes": 2 * (M * K + 2 * F * K + M * F * (3 if case["keep"] else 1)), "flops": 4 * M * F * K}
    if op == "gated_i8":
        return {"bytes": M * K + 2 * F * K + 4 * M + 8 * F + 2 * M * F, "flops": 4 * M * F * K}
    # reads X, both weights, both pre-activations and dH; writes dG, dU, dX and both weight gradients
    return {"bytes": 2 * (2 * M * K + 4 * F * K + 5 * M * F), "flops": 8 * M * F * K}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    def tokens(rows, width):
        # activations: each token at its own level, a few channels louder than the rest
        loud = 1.0 + 7.0 * (torch.rand(width, generator=g, device="cuda") < 0.01)
        return normal(rows, width) * torch.exp(0.5 * normal(rows, 1)) * loud

    def int8_rows(x):
        top = x.abs().amax(1).clamp_min(1e-30)
        return torch.round(x * (127.0 / top)[:, None]).to(torch.int8), top / 127.0

    op, M, K = case["op"], case["M"], case["K"]
    s = {"case": dict(case)}
    if op in ("linear", "product"):
        N, dtype = case["N"], torch.bfloat16 if case["type"] == "bf16" else torch.float32
        s["weight"], s["channel"] = int8_rows(normal(N, K, std=0.02))
        s["bias"] = normal(N, std=0.1) if case["bias"] else None
        if op == "linear":
            s["x"] = tokens(M, K).to(dtype)
            # the quantised tokens and their scales: buffers that a serving loop keeps from step to step
            s["q"], s["token"] = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
        else:
            s["q"], s["token"] = int8_rows(tokens(M, K))
        s["y"] = torch.empty(M, N, dtype=dtype, device="cuda")
        return s
    F, half = case["F"], torch.bfloat16
    if op == "gated_i8":
        s["q"], s["token"] = int8_rows(tokens(M, K))
        s["gate"], s["gate_channel"] = int8_rows(normal(F, K, std=0.02))
        s["up"], s["up_channel"] = int8_rows(normal(F, K, std=0.02))
        s["h"] = torch.empty(M, F, dtype=half, device="cuda")
        return s
    s["x"] = tokens(M, K).to(half)
    s["gate"], s["up"] = normal(F, K, std=0.02).to(half), normal(F, K, std=0.02).to(half)
    kept = ("h", "g", "u") if op == "gated" and case["keep"] else ("h",) if op == "gated" else ("dg", "du")
    if op == "gated_back":
        s["g"], s["u"] = normal(M, F).to(half), normal(M, F).to(half)
        s["dh"] = normal(M, F, std=0.01).to(half)
        s["dx"] = torch.empty(M, K, dtype=half, device="cuda")
        s["dgate"], s["dup"] = (torch.empty(F, K, dtype=half, device="cuda") for _ in range(2))
    for k in kept:
        s[k] = torch.empty(M, F, dtype=half, device="cuda")
    return s


def run(s):
    return run_own(s) if own else run_plain(s)


def run_own(s):
    import exo_b200

    lib, c = exo_b200.library(), s["case"]
    op, M, K = c["op"], c["M"], c["K"]
    if op == "linear":
        call = lib.linear_i8_bf16_exo if c["type"] == "bf16" else lib.linear_i8_f32_exo
        call(None, M, c["N"], K, s["x"], s["weight"], s["channel"], s["bias"], s["q"], s["token"], s["y"])
        return {"y": s["y"], "token_scale": s["token"]}
    if op == "product":
        call = lib.gemm_i8_scaled_bf16_exo if c["type"] == "bf16" else lib.gemm_i8_scaled_f32_exo
        call(None, M, c["N"], K, s["q"], s["weight"], s["token"], s["channel"], s["bias"], s["y"])
        return {"y": s["y"]}
    F, act = c["F"], ACTIVATIONS[c["act"]]
    if op == "gated_i8":
        lib.gated_i8_bf16_exo(None, act, M, F, K, s["q"], s["gate"], s["up"], s["token"], s["gate_channel"],
                              s["up_channel"], s["h"])
        return {"h": s["h"]}
    if op == "gated":
        lib.gated_bf16_exo(None, act, M, F, K, s["x"], s["gate"], s["up"], s["h"], s.get("g"), s.get("u"))
        return {k: s[k] for k in ("h", "g", "u") if k in s}
    lib.gated_bf16_backward_exo(None, act, M, F, K, s["x"], s["gate"], s["up"], s["g"], s["u"], s["dh"],
                                s["dg"], s["du"], s["dx"], s["dgate"], s["dup"])
    return {k: s[k] for k in ("dx", "dgate", "dup", "dg", "du")}


# ------------------------------------------------------------------ the plain form
_ROOT_HALF = math.sqrt(0.5)
_ROOT_2_PI = math.sqrt(2.0 / math.pi)


def _activation(g, name):
    """The activation of g and its derivative."""
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p))
    if name == "gelu":
        p = 0.5 * (1.0 + torch.erf(g * _ROOT_HALF))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (0.5 * _ROOT_2_PI)
    t = torch.tanh(_ROOT_2_PI * (g + 0.044715 * g * g * g))
    slope = _ROOT_2_PI * (1.0 + 3.0 * 0.044715 * g * g)
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * slope


def run_plain(s):
    c = s["case"]
    op = c["op"]
    if op in ("linear", "product"):
        if op == "linear":
            x = s["x"].float()
            top = x.abs().amax(1)
            full = torch.full_like(top, 127.0)
            scale, inverse = top / full, full / top
            # the nearest whole number to the exact product, ties to even
            q = torch.round(x.double() * inverse.double()[:, None]).float()
        else:
            q, scale = s["q"].float(), s["token"]
        y = (q @ s["weight"].float().T) * scale[:, None] * s["channel"]
        if s["bias"] is not None:
            y = y + s["bias"]
        out = {"y": y.to(s["y"].dtype)}
        return out | {"token_scale": scale} if op == "linear" else out
    half = torch.bfloat16
    if op == "gated_i8":
        q = s["q"].float()
        g = (q @ s["gate"].float().T) * s["token"][:, None] * s["gate_channel"]
        u = (q @ s["up"].float().T) * s["token"][:, None] * s["up_channel"]
        return {"h": (_activation(g, c["act"])[0] * u).to(half)}
    x, gate, up = s["x"].float(), s["gate"].float(), s["up"].float()
    if op == "gated":
        g, u = x @ gate.T, x @ up.T
        out = {"h": (_activation(g, c["act"])[0] * u).to(half)}
        return out | {"g": g.to(half), "u": u.to(half)} if c["keep"] else out
    a, slope = _activation(s["g"].float(), c["act"])
    dh = s["dh"].float()
    dg, du = dh * s["u"].float() * slope, dh * a
    return {"dx": (dg @ gate + du @ up).to(half), "dgate": (dg.T @ x).to(half), "dup": (du.T @ x).to(half),
            "dg": dg.to(half), "du": du.to(half)}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    op = case["op"]
    if op in ("linear", "product"):
        if op == "linear":
            largest = s["x"].abs().max(dim=1, keepdim=True).values
            step = largest / 127
            # the inverse step is a 32-bit number by definition: it decides which way a value next to a border goes
            q = torch.round(s["x"] * (127 / largest).float().double())
        else:
            step, q = s["token"].unsqueeze(1), s["q"]
        y = torch.matmul(q, s["weight"].t()) * step * s["channel"].unsqueeze(0)
        y = y if s["bias"] is None else y + s["bias"].unsqueeze(0)
        return {"y": y, "token_scale": step.squeeze(1)} if op == "linear" else {"y": y}

    def gate_of(g):
        if case["act"] == "silu":
            return g * torch.sigmoid(g)
        if case["act"] == "gelu":
            return g * torch.special.ndtr(g)
        return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))  # (1 + tanh z) / 2 = sigmoid(2 z)

    if op in ("gated", "gated_i8"):
        rows = s["x"] if op == "gated" else s["q"] * s["token"].unsqueeze(1)
        wg = s["gate"] if op == "gated" else s["gate"] * s["gate_channel"].unsqueeze(1)
        wu = s["up"] if op == "gated" else s["up"] * s["up_channel"].unsqueeze(1)
        g, u = torch.matmul(rows, wg.t()), torch.matmul(rows, wu.t())
        h = {"h": gate_of(g) * u}
        return {**h, "g": g, "u": u} if case.get("keep") else h
    g = s["g"].requires_grad_(True)
    a = gate_of(g)
    (slope,) = torch.autograd.grad(a.sum(), g)
    dg, du = s["dh"] * s["u"] * slope, s["dh"] * a.detach()
    return {"dx": torch.addmm(torch.matmul(dg, s["gate"]), du, s["up"]), "dgate": torch.matmul(dg.t(), s["x"]),
            "dup": torch.matmul(du.t(), s["x"]), "dg": dg, "du": du}
