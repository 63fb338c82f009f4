"""The operators of lm_lean_ops (gated product, streamed cross entropy, 8-bit
activations) against their formulas in 64 bits.

Tolerances: u is half a step of the 16-bit type (bf16 2^-8, fp16 2^-11); a sum of n
products of 16-bit numbers in fp32, whatever its order and even if every addition
truncates, is off by at most n 2^-23 times the sum of the products' magnitudes; the
fast exponential and quotient cost a few 2^-22. Every value that the kernels round to
16 bits on the way adds u times its magnitude, carried through the next product by the
magnitudes of the other factor. The bounds below add these up element by element."""
import math

import pytest
import torch

from conftest import rel_l2
from paper_01_anti_decoy_pnfirtau_b200 import (act8_pack, act8_unpack, act8_weight_grad, check_device_status, gated_linear,
                                               gated_mlp, streamed_cross_entropy)

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SUM = 2.0 ** -23


def u(dt):
    return torch.finfo(dt).eps / 2


def act(g, name):
    """The activation, its derivative, and a bound of the second derivative."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = torch.special.ndtr(g)
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


SECOND = 0.8  # both activations: |act''| <= 2 phi(0) = 0.798 (GELU), 0.5 (SiLU); |act'| <= 1.13


def gated_oracle(x, wg, wu, bg, bu, dh, name, dt, kept):
    """(value, bound) of h, dx, dwg, dwu, dbg, dbu; `kept`: the backward reads g and u rounded to dt."""
    x, wg, wu, dh = (t.detach().double() for t in (x, wg, wu, dh))
    e, D, F, M = u(dt), x.shape[1], wg.shape[0], x.shape[0]
    g, up = x @ wg.T, x @ wu.T
    eg, eu = D * SUM * (x.abs() @ wg.abs().T), D * SUM * (x.abs() @ wu.abs().T)
    if bg is not None:
        g, eg = g + bg.double(), eg + SUM * (g.abs() + bg.double().abs())
    if bu is not None:
        up, eu = up + bu.double(), eu + SUM * (up.abs() + bu.double().abs())
    fast = 2.0 ** -18
    a, da = act(g, name)
    h = a * up
    ea = 1.13 * eg + fast * g.abs()
    eh = ea * up.abs() + (a.abs() + ea) * eu + e * h.abs() + torch.finfo(dt).tiny * 2 ** -8
    if kept:
        eg, eu = eg + e * (g.abs() + eg), eu + e * (up.abs() + eu)
    ea = 1.13 * eg + fast * g.abs()
    eda = SECOND * eg + fast * (1 + g.abs())
    dg, du = dh * up * da, dh * a
    edg = dh.abs() * (eu * da.abs() + (up.abs() + eu) * eda)
    edg = edg + e * (dg.abs() + edg) + torch.finfo(dt).tiny * 2 ** -8
    edu = dh.abs() * ea
    edu = edu + e * (du.abs() + edu) + torch.finfo(dt).tiny * 2 ** -8
    out = [(h, eh)]
    dx = dg @ wg + du @ wu
    edx = edg @ wg.abs() + edu @ wu.abs() + 2 * F * SUM * ((dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs())
    out.append((dx, edx + e * (dx.abs() + edx) + 2.0 ** -25))
    for d, ed in ((dg, edg), (du, edu)):
        v = d.T @ x
        ev = ed.T @ x.abs() + M * SUM * ((d.abs() + ed).T @ x.abs())
        out.append((v, ev + e * (v.abs() + ev) + 2.0 ** -25))
    for d, ed in ((dg, edg), (du, edu)):
        v, ev = d.sum(0), ed.sum(0) + M * SUM * (d.abs() + ed).sum(0)
        out.append((v, ev + e * (v.abs() + ev) + 2.0 ** -25))
    return out


def check(name, got, want):
    value, bound = want
    assert got.shape == value.shape, name
    err = (got.double() - value).abs()
    assert torch.isfinite(got).all(), name
    worst = (err - bound).max() if err.numel() else torch.tensor(-1.0)
    assert float(worst) <= 0, f"{name}: error {float(err.max()):.3e} past its bound by {float(worst):.3e}"


def gated_inputs(M, D, F, dt, bias, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, device=device, generator=g) * std).to(dt)  # noqa: E731
    x, wg, wu = r(M, D), r(F, D, std=D ** -0.5), r(F, D, std=D ** -0.5)
    bg, bu = (r(F, std=0.3), r(F, std=0.3)) if bias else (None, None)
    return x, wg, wu, bg, bu, r(M, F)


# (M, D, F): one token; a few; a tile's edges on each side; K tails; odd widths; one column; wide;
# products whose last round of tiles is split along K
GATED = [(1, 64, 128), (3, 256, 1024), (17, 100, 77), (127, 64, 129), (128, 128, 128), (129, 72, 127), (300, 1, 5),
         (5, 1001, 1), (33, 520, 2731), (1000, 256, 1024), (257, 2048, 640), (4200, 1300, 1800)]


@pytest.mark.parametrize("shape", GATED)
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("name,bias", [("silu", False), ("gelu", True)])
def test_gated_linear(cuda, shape, dt, name, bias):
    M, D, F = shape
    x, wg, wu, bg, bu, dh = gated_inputs(M, D, F, dt, bias, M * 31 + D + F, cuda)
    want = gated_oracle(x, wg, wu, bg, bu, dh, name, dt, kept=True)
    with torch.no_grad():
        check("h without gradient", gated_linear(x, wg, wu, bg, bu, activation=name), want[0])
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, bg, bu) if t is not None]
    h = gated_linear(x, wg, wu, bg, bu, activation=name)
    grads = torch.autograd.grad(h, leaves, dh)
    check_device_status(cuda)
    for n, got, w in zip(("h", "dx", "dwg", "dwu", "dbg", "dbu"), (h.detach(), *grads), want):
        assert got.dtype == dt
        check(n, got, w)
        if got.numel() > 1000:
            assert rel_l2(got, w[0]) < 4 * u(dt), n


@pytest.mark.parametrize("shape", [(1, 64, 128), (17, 100, 77), (129, 1000, 127), (1000, 256, 1024)])
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("name,bias", [("silu", True), ("gelu", False)])
def test_gated_linear_with_8bit_checkpoint(cuda, shape, dt, name, bias):
    M, D, F = shape
    x, wg, wu, bg, bu, dh = gated_inputs(M, D, F, dt, bias, M + D * 3 + F, cuda)
    forward = gated_oracle(x, wg, wu, bg, bu, dh, name, dt, kept=False)[0]
    x8 = eight_bits(x)
    want = [forward] + gated_oracle(x8, wg, wu, bg, bu, dh, name, dt, kept=False)[1:]
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, bg, bu) if t is not None]
    h = gated_linear(x, wg, wu, bg, bu, activation=name, checkpoint_8bit=True)
    grads = torch.autograd.grad(h, leaves, dh)
    check_device_status(cuda)
    for n, got, w in zip(("h", "dx", "dwg", "dwu", "dbg", "dbu"), (h.detach(), *grads), want):
        check(n, got, w)


# ---------------------------------------------------------------- 8-bit activations
def eight_bits(x):
    """x's values in 8 bits, from the definition, in 64 bits."""
    lo, hi = (-15, 8) if x.dtype == FP16 else (-110, 120)
    out = x.detach().double().clone()
    for c in range(0, x.shape[1], 128):
        b = out[:, c:c + 128]
        fine = torch.isfinite(b)
        top = torch.where(fine, b.abs(), 0.0).amax(1, keepdim=True)
        e = torch.full_like(top, float(lo))
        for k in range(lo, hi):  # the least exponent that brings the largest magnitude to 448
            e = torch.where(top > 448 * 2.0 ** k, float(k + 1), e)
        v = b / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        v = torch.round(v / step) * step
        v = torch.where(e == hi, v.clamp(-240, 240), v)
        out[:, c:c + 128] = torch.where(fine, v * torch.exp2(e), float("nan"))
    return out


def same(got, want):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.double(), nan=0.0), torch.nan_to_num(want, nan=0.0))


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,D", [(1, 1), (1, 128), (3, 129), (70, 1000), (257, 256), (5, 127)])
def test_act8_values(cuda, dt, M, D):
    g = torch.Generator(device=cuda).manual_seed(M * 1000 + D)
    x = torch.randn(M, D, device=cuda, generator=g) * torch.exp(3 * torch.randn(M, 1, device=cuda, generator=g))
    x = x.to(dt)
    x[0, 0] = 448.0
    if M >= 3:
        x[1] = 0
        x[2, 0] = 449 if dt != BF16 else 452
    p = act8_pack(x)
    y = act8_unpack(p)
    assert y.dtype == dt and y.shape == x.shape
    same(y, eight_bits(x))  # values past fp16's range are infinities here, NaN in 8 bits


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
def test_act8_extremes(cuda, dt):
    x = torch.zeros(9, 256, device=cuda, dtype=dt)
    x[0] = torch.finfo(dt).max
    x[1, ::2], x[1, 1::2] = torch.finfo(dt).tiny, -torch.finfo(dt).tiny
    x[2, 5], x[2, 6], x[2, 7], x[2, 8] = float("nan"), float("inf"), float("-inf"), 3.0
    x[3, :128] = float("nan")  # a block without a finite value, and one beside it
    x[3, 128:] = 1.5
    x[4, 0] = torch.finfo(dt).smallest_normal / 4  # subnormal
    x[5, 0], x[5, 1] = torch.finfo(dt).max, 1.0
    x[6] = -torch.finfo(dt).max
    x[7] = torch.linspace(-500, 500, 256).to(dt)
    same(act8_unpack(act8_pack(x)), eight_bits(x))


def test_act8_strides_and_shape(cuda):
    base = torch.randn(6, 40, 300, device=cuda).to(BF16)
    for x in (base[:, ::3, 7:200], base.transpose(0, 1), base[:, :, ::2], base[0, 0], base[:0]):
        y = act8_unpack(act8_pack(x))
        assert y.shape == x.shape
        assert torch.equal(y.reshape(-1, x.shape[-1]).double(), eight_bits(x.reshape(-1, x.shape[-1])))
    p = act8_pack(base)
    assert p.nbytes < 0.6 * base.numel() * 2


@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("M,N,D", [(1, 8, 128), (5, 3, 1), (64, 256, 1024), (1000, 129, 257), (4099, 256, 1000), (0, 16, 24), (4001, 2500, 2309)])
def test_act8_weight_grad(cuda, dt, M, N, D):
    g = torch.Generator(device=cuda).manual_seed(M + N + D)
    x = torch.randn(M, D, device=cuda, generator=g).to(dt)
    dy = torch.randn(M, N, device=cuda, generator=g).to(dt)
    got = act8_weight_grad(dy, act8_pack(x))
    x8 = eight_bits(x)
    want, mags = dy.double().T @ x8, dy.double().abs().T @ x8.abs()
    assert got.dtype == FP32
    check("dw", got, (want, M * SUM * mags + 2.0 ** -100))


# ---------------------------------------------------------------- streamed cross entropy
def xent_oracle(h, w, t, up, dt, ignore=-100):
    """(value, bound) of the rows' losses, dh and dW for the rows' upstream factors `up`."""
    h, w = h.detach().double(), w.detach().double()
    live = t != ignore
    at = torch.where(live, t, 0)[:, None]
    h = torch.where(live[:, None], h, 0.0)
    z = h @ w.T
    D, V, e = h.shape[1], w.shape[0], u(dt)
    ez = (D * SUM * (h.abs() @ w.abs().T)).amax(1)
    lse = torch.logsumexp(z, 1)
    loss = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    size = z.abs().amax(1)
    # the sums: V additions in fp32; log2 e times z, the maximum and the logarithm in fp32
    el = 2 * ez + V * SUM + 2.0 ** -20 * (1 + size + lse.abs())
    p = torch.exp(z - lse[:, None])
    s = torch.where(live, up.double(), 0.0)[:, None]
    dz = p * s
    edz = dz.abs() * (torch.expm1(el + ez) + 2.0 ** -20)[:, None]
    dz.scatter_add_(1, at, -s)
    # a 16-bit value of up to 1 (bf16) or 2^14 (fp16) times the largest factor
    top = s.abs().max()
    edz = edz + e * (dz.abs() + edz) + top * (2.0 ** -133 if dt == BF16 else 2.0 ** -38)
    dh, dw = dz @ w, dz.T @ h
    edh = edz @ w.abs() + V * SUM * ((dz.abs() + edz) @ w.abs())
    edw = edz.T @ h.abs() + h.shape[0] * SUM * ((dz.abs() + edz).T @ h.abs())
    tiny = torch.finfo(dt).smallest_normal * 2 * e
    return (loss, torch.where(live, el, 0.0)), (dh, edh + e * (dh.abs() + edh) + tiny), (dw, edw + e * (dw.abs() + edw) + tiny)


# (M, V, D): one token; a tile's edges; a vocabulary of one; odd widths; several pieces;
# a dW whose last round of tiles is split along K
XENT = [(1, 1000, 64), (1, 33278, 256), (5, 1, 8), (7, 257, 72), (128, 256, 128), (129, 255, 1), (300, 1025, 1001),
        (1000, 5000, 256), (64, 50021, 776), (2100, 40000, 64), (4000, 20001, 300)]


@pytest.mark.parametrize("shape", XENT)
@pytest.mark.parametrize("dt", [BF16, FP16])
@pytest.mark.parametrize("reduction,ignored", [("mean", 0.0), ("sum", 0.4), ("none", 0.2)])
def test_streamed_cross_entropy(cuda, shape, dt, reduction, ignored):
    M, V, D = shape
    g = torch.Generator(device=cuda).manual_seed(M + V + D)
    h = torch.randn(M, D, device=cuda, generator=g).to(dt).requires_grad_(True)
    w = (torch.randn(V, D, device=cuda, generator=g) * 2 / D ** 0.5).to(dt).requires_grad_(True)
    t = torch.randint(0, V, (M,), device=cuda, generator=g)
    t[-1] = V - 1
    if ignored and M > 1:
        t[:-1][torch.rand(M - 1, device=cuda, generator=g) < ignored] = -100
    n = int((t != -100).sum())
    if reduction == "none":
        dloss = torch.randn(M, device=cuda, generator=g)
        up = dloss
    else:
        dloss = torch.tensor(3.0 if dt == BF16 else 512.0, device=cuda)
        up = (dloss / (n if reduction == "mean" else 1)).expand(M)
    (loss, el), dh, dw = xent_oracle(h, w, t, up, dt)
    with torch.no_grad():
        alone = streamed_cross_entropy(h, w, t, reduction=reduction)
    got = streamed_cross_entropy(h, w, t, reduction=reduction)
    assert got.dtype == FP32
    gh, gw = torch.autograd.grad(got, (h, w), dloss)
    check_device_status(cuda)
    if reduction != "none":
        k = n if reduction == "mean" else 1
        loss, el = loss.sum() / k, el.sum() / k + 2.0 ** -23 * loss.sum() / k
    check("loss", got.detach(), (loss, el))
    check("loss without gradient", alone, (loss, el))  # few rows: a kernel of its own
    check("dh", gh, dh)
    check("dw", gw, dw)
    assert torch.all(gh[t == -100] == 0)
    if M * D > 1000:
        assert rel_l2(gh, dh[0]) < 4 * u(dt) and rel_l2(gw, dw[0]) < 4 * u(dt)
