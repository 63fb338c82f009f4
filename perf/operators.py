"""Cases of the language-model operators that train a decoder in little memory:

- the gated feed-forward product ``act(x Wg^T + bg) * (x Wu^T + bu)``, its backward
  pass, and its form for single tokens (``gated_linear``);
- the softmax cross entropy of a language-model head in pieces of the vocabulary,
  without keeping the logits, with its gradient (``streamed_cross_entropy``);
- activation checkpoints in 8 bits and the weight gradient that reads them
  (``act8_pack``, ``act8_unpack``, ``act8_weight_grad``; ``gated_linear`` with
  ``checkpoint_8bit``).

Each operator stands here in three forms: its plain form (elementary torch
operations in 32 bits), the framework's call (``own``), and its definition in 64
bits (``exact``).
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token of a decoder that answers: the weights are read once, latency counts
        {"name": "gated_token", "op": "gated", "mode": "forward", "dtype": "bf16", "act": "silu", "bias": False,
         "M": 1, "D": 1024, "F": 4096},
        # a batch of answers of different users, one token each, odd width
        {"name": "gated_batch_fp16", "op": "gated", "mode": "forward", "dtype": "fp16", "act": "gelu", "bias": True,
         "M": 37, "D": 2048, "F": 5461},
        # the repository's language model, 32 sequences of 512 (width 256, feed-forward 1024), a training step's part
        {"name": "gated_lm_train", "op": "gated", "mode": "train", "dtype": "bf16", "act": "silu", "bias": False,
         "M": 16384, "D": 256, "F": 1024},
        # a wide block's training step
        {"name": "gated_wide_train", "op": "gated", "mode": "train", "dtype": "bf16", "act": "silu", "bias": False,
         "M": 8192, "D": 2048, "F": 8192},
        # the same with the input kept in 8 bits and nothing else: ragged rows, odd hidden width, biases
        {"name": "gated_ckpt8_ragged", "op": "gated", "mode": "train8", "dtype": "bf16", "act": "gelu", "bias": True,
         "M": 4095, "D": 1000, "F": 2731},
        # scoring one token against the repository's vocabulary
        {"name": "xent_token", "op": "xent", "mode": "forward", "dtype": "bf16", "reduction": "none",
         "M": 1, "D": 256, "V": 33278, "ignored": 0.0},
        # the repository's language model: 32 x 511 scored positions, its vocabulary
        {"name": "xent_lm_train", "op": "xent", "mode": "train", "dtype": "bf16", "reduction": "mean",
         "M": 16352, "D": 256, "V": 33278, "ignored": 0.0},
        # a wide model over a large vocabulary, padded sequences
        {"name": "xent_wide_train", "op": "xent", "mode": "train", "dtype": "bf16", "reduction": "mean",
         "M": 4096, "D": 2048, "V": 128000, "ignored": 0.1},
        # odd rows and vocabulary, half the positions masked (prompts), summed, fp16
        {"name": "xent_ragged_fp16", "op": "xent", "mode": "train", "dtype": "fp16", "reduction": "sum",
         "M": 1021, "D": 776, "V": 50021, "ignored": 0.5},
        # an activation saved and restored, odd rows, 1000 columns (a short last block)
        {"name": "act8_round_trip", "op": "act8", "mode": "round_trip", "dtype": "fp32", "M": 4099, "D": 1000, "N": 0},
        # the input of the repository's second feed-forward layer, kept in 8 bits, and that layer's weight gradient
        {"name": "act8_lm_grad", "op": "act8", "mode": "weight_grad", "dtype": "bf16", "M": 16384, "D": 1024, "N": 256},
        # a wide layer's
        {"name": "act8_wide_grad", "op": "act8", "mode": "weight_grad", "dtype": "bf16", "M": 8192, "D": 4096, "N": 4096},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: a multiple of 64 half of the time, of 8 mostly else, odd at times."""
    n, r = _log(rng, lo, hi), rng.random()
    if r < 0.5:
        return max(64, n // 64 * 64)
    if r < 0.8:
        return max(8, n // 8 * 8)
    return n | 1


def draw(rng):
    op = rng.choice(["gated", "gated", "xent", "xent", "act8"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "gated":
        mode = rng.choice(["forward", "train", "train8"])
        M = _log(rng, 1, 64) if mode == "forward" and rng.random() < 0.5 else _log(rng, 1, 16384)
        D, F = _width(rng, 64, 4096), _width(rng, 64, 16384)
        while M * D * F > 8192 * 2048 * 8192:
            M = max(1, M // 2)
        return {"op": op, "mode": mode, "dtype": dtype, "act": rng.choice(["silu", "gelu"]),
                "bias": rng.random() < 0.5, "M": M, "D": D, "F": F}
    if op == "xent":
        M, D, V = _log(rng, 1, 16384), _width(rng, 64, 4096), _log(rng, 500, 131072)
        while M * D * V > 4096 * 2048 * 128000:
            M = max(1, M // 2)
        return {"op": op, "mode": rng.choice(["forward", "train", "train"]), "dtype": dtype,
                "reduction": rng.choice(["mean", "sum", "none"]), "M": M, "D": D, "V": V,
                "ignored": rng.choice([0.0, 0.1, 0.5])}
    mode = rng.choice(["round_trip", "weight_grad"])
    if mode == "round_trip":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
    return {"op": op, "mode": mode, "dtype": dtype, "M": _log(rng, 1, 16384), "D": _width(rng, 64, 4096),
            "N": _width(rng, 64, 4096) if mode == "weight_grad" else 0}


# ------------------------------------------------------------------ the inputs
def _activation(g, M, D):
    """Normalised activations: unit variance, a few outlying channels, tokens of different size."""
    x = torch.randn(M, D, device="cuda", generator=g)
    x *= 0.5 + torch.rand(M, 1, device="cuda", generator=g)
    loud = torch.rand(D, device="cuda", generator=g) < 0.01
    return torch.where(loud, x * 8, x)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * std

    s = dict(case)
    M, D = case["M"], case["D"]
    train = case["mode"] in ("train", "train8")
    if case["op"] == "gated":
        F = case["F"]
        s["x"] = _activation(g, M, D).to(dt)
        s["wg"] = normal(F, D, std=D ** -0.5).to(dt)
        s["wu"] = normal(F, D, std=D ** -0.5).to(dt)
        s["bg"] = normal(F, std=0.2).to(dt) if case["bias"] else None
        s["bu"] = normal(F, std=0.2).to(dt) if case["bias"] else None
        if train:
            s["dh"] = normal(M, F).to(dt)
            s["leaves"] = [t.requires_grad_(True) for t in (s["x"], s["wg"], s["wu"], s["bg"], s["bu"]) if t is not None]
    elif case["op"] == "xent":
        V = case["V"]
        s["h"] = _activation(g, M, D).to(dt)
        s["w"] = normal(V, D, std=2.0 * D ** -0.5).to(dt)
        t = torch.randint(0, V, (M,), device="cuda", generator=g)
        if case["ignored"]:
            t[torch.rand(M, device="cuda", generator=g) < case["ignored"]] = IGNORE
            t[0] = 0  # a mean over no row has no value
        s["t"] = t
        if train:
            # the loss's own gradient: one value, or one of each row (weighted sequences); a mean's in fp16 is
            # scaled, as such training scales its loss to keep the gradients inside the type's range
            s["dloss"] = (torch.rand(M, device="cuda", generator=g) if case["reduction"] == "none"
                          else torch.full((), 4096.0 if (case["dtype"], case["reduction"]) == ("fp16", "mean") else 1.0,
                                          device="cuda"))
            s["h"].requires_grad_(True)
            s["w"].requires_grad_(True)
    else:
        s["x"] = _activation(g, M, D).to(dt)
        if case["mode"] == "weight_grad":
            s["dy"] = normal(M, case["N"]).to(dt)
    return s


# ------------------------------------------------------------------ the plain forms
def _act(g, name):
    """The activation and its derivative."""
    if name == "silu":
        sg = 1 / (1 + torch.exp(-g))
        return g * sg, sg * (1 + g * (1 - sg))
    cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


# exponents of a block's scale (powers of two) for which the stored values fit the type that they come back in;
# in the largest one the values end at 240, as 256 times the scale would be past that type
_EXPONENTS = {torch.float32: (-110, 120), torch.bfloat16: (-110, 120), torch.float16: (-15, 8)}


def _eight_bits(x):
    """x [M, D] as its 8-bit form (e4m3 with a power of two for each row's block of 128 columns) holds it, in 32 bits."""
    M, D = x.shape
    lo, hi = _EXPONENTS[x.dtype]
    nb = (D + 127) // 128
    p = torch.zeros(M, nb * 128, device=x.device)
    p[:, :D] = x.float()
    p = p.view(M, nb, 128)
    frac, e = torch.frexp(p.abs().amax(-1, keepdim=True))
    e = torch.where(frac <= 0.875, e - 9, e - 8).clamp(lo, hi)  # 0.875 * 2^9 = 448, the largest value of e4m3
    e = torch.where(frac == 0, torch.full_like(e, lo), e)
    v = torch.ldexp(p, -e)
    v = torch.where(e == hi, v.clamp(-240, 240), v)
    return torch.ldexp(v.to(torch.float8_e4m3fn).float(), e).view(M, -1)[:, :D]


def _plain_gated(s):
    dt = s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()

    def pre(x):
        g, u = x @ wg.T, x @ wu.T
        return (g, u) if s["bg"] is None else (g + s["bg"].float(), u + s["bu"].float())

    g, u = pre(x)
    a, da = _act(g, s["act"])
    h = (a * u).to(dt)
    if s["mode"] == "forward":
        return h
    if s["mode"] == "train8":  # the backward pass sees the 8-bit form of x
        x = _eight_bits(s["x"])
        g, u = pre(x)
        a, da = _act(g, s["act"])
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    grads = [dg @ wg + du @ wu, dg.T @ x, du.T @ x]
    if s["bg"] is not None:
        grads += [dg.sum(0), du.sum(0)]
    return [h] + [v.to(dt) for v in grads]


def _plain_xent(s):
    dt = s["h"].dtype
    w, t, M, V = s["w"].float(), s["t"], s["M"], s["V"]
    counted = t != IGNORE
    scale = counted.float()
    if s["reduction"] == "mean":
        scale = scale / counted.sum().float()
    train = s["mode"] == "train"
    losses, dh = [], []
    dw = torch.zeros_like(w) if train else None
    rows = max(1, min(M, (1 << 28) // V))
    for i in range(0, M, rows):
        h, c = s["h"][i:i + rows].float(), counted[i:i + rows]
        at = torch.where(c, t[i:i + rows], 0)[:, None]
        z = h @ w.T
        top = z.amax(1, keepdim=True)
        picked = z.gather(1, at)
        z = torch.exp(z - top)
        total = z.sum(1, keepdim=True)
        losses.append(torch.where(c, (top + torch.log(total) - picked)[:, 0], 0.0))
        if train:
            up = scale[i:i + rows] * (s["dloss"][i:i + rows] if s["reduction"] == "none" else s["dloss"])
            z /= total
            z.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
            z *= up[:, None]
            dh.append(z @ w)
            dw += z.T @ h
    loss = torch.cat(losses)
    if s["reduction"] != "none":
        loss = (loss * scale).sum()
    return [loss, torch.cat(dh).to(dt), dw.to(dt)] if train else loss


def _plain_act8(s):
    x = _eight_bits(s["x"])
    if s["mode"] == "round_trip":
        return x.to(s["x"].dtype)
    return s["dy"].float().T @ x


# ------------------------------------------------------------------ the framework's calls
def _own_gated(s):
    from paper_01_anti_decoy_pnfirtau_b200 import gated_linear

    if s["mode"] == "forward":
        with torch.no_grad():
            return gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=s["act"])
    h = gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=s["act"],
                     checkpoint_8bit=s["mode"] == "train8")
    return [h.detach(), *torch.autograd.grad(h, s["leaves"], s["dh"])]


def _own_xent(s):
    from paper_01_anti_decoy_pnfirtau_b200 import streamed_cross_entropy

    if s["mode"] == "forward":
        with torch.no_grad():
            return streamed_cross_entropy(s["h"], s["w"], s["t"], IGNORE, reduction=s["reduction"])
    loss = streamed_cross_entropy(s["h"], s["w"], s["t"], IGNORE, reduction=s["reduction"])
    return [loss.detach(), *torch.autograd.grad(loss, (s["h"], s["w"]), s["dloss"])]


def _own_act8(s):
    from paper_01_anti_decoy_pnfirtau_b200 import act8_pack, act8_unpack, act8_weight_grad

    saved = act8_pack(s["x"])
    if s["mode"] == "round_trip":
        return act8_unpack(saved)
    return act8_weight_grad(s["dy"], saved)


def run(state):
    if own:
        return {"gated": _own_gated, "xent": _own_xent, "act8": _own_act8}[state["op"]](state)
    with torch.no_grad():
        return {"gated": _plain_gated, "xent": _plain_xent, "act8": _plain_act8}[state["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    M, D = case["M"], case["D"]
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["mode"] in ("train", "train8")
    if case["op"] == "gated":
        F, b = case["F"], 2 * case["F"] if case["bias"] else 0
        # read x, the weights (and biases); write h. Training: read dh, write the gradients of all that was read
        n = M * D + 2 * F * D + b + M * F
        if train:
            n += M * F + M * D + 2 * F * D + b
        return {"bytes": n * size, "flops": (12 if train else 4) * M * D * F}
    if case["op"] == "xent":
        V = case["V"]
        n = (M * D + V * D) * size + 8 * M + (4 * M if case["reduction"] == "none" else 4)
        if train:
            n += (M * D + V * D) * size + (4 * M if case["reduction"] == "none" else 4)
        return {"bytes": n, "flops": (6 if train else 2) * M * D * V}
    if case["mode"] == "round_trip":
        # x read, the 8-bit form and its exponents written and read again, the values written
        return {"bytes": 2 * M * D * size + 2 * (M * D + M * ((D + 127) // 128)), "flops": 4 * M * D}
    N = case["N"]
    return {"bytes": M * D * size + 2 * (M * D + M * ((D + 127) // 128)) + M * N * size + 4 * N * D,
            "flops": 2 * M * D * N}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_eight_bits(x):
    """x as 8 bits hold it: every value goes to the nearest of e4m3's, ties to the even one, with 3 bits behind the
    leading one and no step below 2^-9, after its block of 128 was divided by the least power of two that brings
    the block's largest magnitude to 448 or less."""
    lo, hi = {torch.float16: (-15, 8)}.get(x.dtype, (-110, 120))
    out = x.double().clone()
    for c in range(0, x.shape[1], 128):
        b = out[:, c:c + 128]
        top = b.abs().amax(1, keepdim=True)
        e = torch.full_like(top, float(lo))
        some = top > 0
        e[some] = torch.ceil(torch.log2(top[some] / 448)).clamp(lo, hi)
        e += (some & (top > 448 * torch.exp2(e)) & (e < hi)).double()  # log2 next to a whole number
        e -= (some & (top <= 224 * torch.exp2(e)) & (e > lo)).double()
        v = b / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        v = torch.round(v / step) * step
        v = torch.where(e == hi, v.clamp(-240, 240), v)
        out[:, c:c + 128] = v * torch.exp2(e)
    return out


def _exact_gated(s):
    def forward(x, wg, wu, bg, bu):
        g, u = torch.nn.functional.linear(x, wg, bg), torch.nn.functional.linear(x, wu, bu)
        if s["act"] == "silu":
            return torch.sigmoid(g) * g * u
        return torch.special.ndtr(g) * g * u

    ops = [None if s[k] is None else s[k].detach().double() for k in ("x", "wg", "wu", "bg", "bu")]
    if s["mode"] == "forward":
        return forward(*ops)
    h = forward(*ops)
    if s["mode"] == "train8":
        ops[0] = _exact_eight_bits(s["x"].detach())
    ops = [None if t is None else t.requires_grad_(True) for t in ops]
    with torch.enable_grad():
        out = forward(*ops)
    return [h, *torch.autograd.grad(out, [t for t in ops if t is not None], s["dh"].double())]


def _exact_xent(s):
    w, t, M, V = s["w"].detach().double(), s["t"], s["M"], s["V"]
    n = int((t != IGNORE).sum())
    weight = 1.0 / n if s["reduction"] == "mean" else 1.0
    train = s["mode"] == "train"
    loss = torch.zeros(M, dtype=torch.float64, device=w.device)
    dh, dw = torch.zeros_like(s["h"], dtype=torch.float64), torch.zeros_like(w)
    rows = max(1, (1 << 27) // V)
    for i in range(0, M, rows):
        live = (t[i:i + rows] != IGNORE).nonzero()[:, 0] + i
        if not live.numel():
            continue
        h = s["h"].detach()[live].double()
        logp = torch.log_softmax(h @ w.T, 1)
        loss[live] = -logp[torch.arange(len(live)), t[live]]
        if train:
            p = logp.exp()
            p[torch.arange(len(live)), t[live]] -= 1
            p *= weight * (s["dloss"].double()[live, None] if s["reduction"] == "none" else float(s["dloss"]))
            dh[live] = p @ w
            dw += p.T @ h
    if s["reduction"] != "none":
        loss = loss.sum() * weight
    return [loss, dh, dw] if train else loss


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "gated":
            return _exact_gated(s)
        if case["op"] == "xent":
            return _exact_xent(s)
        x = _exact_eight_bits(s["x"])
        return x if case["mode"] == "round_trip" else s["dy"].double().T @ x
