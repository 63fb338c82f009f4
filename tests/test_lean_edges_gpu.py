"""Calls that the lean training-step operators allow beside the ordinary ones: views and
strides, empty inputs, masked rows that hold NaN, targets outside the vocabulary, extreme
logits, autocast with fp32 parameters, parameter copies, partial gradients, other streams,
CUDA graphs, repeated runs, differences. And the calls that they refuse."""
import pytest
import torch
import torch.nn.functional as F

from conftest import rel_l2
from paper_01_anti_decoy_pnfirtau_b200 import (Act8, act8_pack, act8_unpack, act8_weight_grad, check_device_status,
                                               gated_linear, streamed_cross_entropy)
from paper_01_anti_decoy_pnfirtau_b200.lm_ops import Bf16Casts

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, dt=BF16, std=1.0, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed + sum(shape))
    return (torch.randn(*shape, device=device, generator=g) * std).to(dt)


def gated_all(x, wg, wu, bg=None, bu=None, dh=None, **kw):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, wg, wu, bg, bu)]
    h = gated_linear(*leaves, **kw)
    grads = torch.autograd.grad(h, [t for t in leaves if t is not None], torch.ones_like(h) if dh is None else dh)
    return [h.detach(), *grads]


def xent_all(h, w, t, dloss=None, **kw):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = streamed_cross_entropy(h, w, t, **kw)
    return [loss.detach(), *torch.autograd.grad(loss, (h, w), torch.ones_like(loss) if dloss is None else dloss)]


def same(a, b):
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and torch.equal(x, y)


# ------------------------------------------------------------------ layouts
@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("D", [72, 1000])
def test_gated_views_equal_their_copies(cuda, M, D):
    wide = rand(M, D + 24, seed=1)
    w2 = rand(2 * 160, D, std=D ** -0.5, seed=2)
    dh = rand(M, 160, seed=3)
    want = gated_all(wide[:, :D].contiguous(), w2[:160].clone(), w2[160:].clone(), dh=dh)
    same(gated_all(wide[:, :D], w2[:160], w2[160:], dh=dh), want)
    odd = torch.empty(M, D + 3, device=cuda, dtype=BF16)[:, 1:D + 1].copy_(wide[:, :D])  # 2-byte aligned rows
    same(gated_all(odd, w2[:160], w2[160:], dh=dh), want)
    cols = wide[:, :D].t().contiguous().t()  # column-major x and weights
    wt = w2[:160].t().contiguous().t()
    same(gated_all(cols, wt, w2[160:], dh=dh), want)
    bigger = torch.zeros(M, 200, device=cuda, dtype=BF16)
    bigger[:, 7:167] = dh
    same(gated_all(wide[:, :D], w2[:160], w2[160:], dh=bigger[:, 7:167]), want)
    h3 = gated_linear(wide[:, :D].contiguous().view(1, M, 1, D), w2[:160], w2[160:])
    assert h3.shape == (1, M, 1, 160)


def test_gated_expanded_gradient_and_input(cuda):
    x, wg, wu = rand(1, 64).expand(130, 64), rand(96, 64, std=0.1, seed=1), rand(96, 64, std=0.1, seed=2)
    one = gated_all(x.contiguous(), wg, wu, dh=rand(1, 96).expand(130, 96).contiguous())
    same(gated_all(x, wg, wu, dh=rand(1, 96).expand(130, 96)), one)
    leaves = [t.clone().requires_grad_(True) for t in (x.contiguous(), wg, wu)]
    gated_linear(*leaves).sum().backward()  # the gradient of a sum has no strides of its own
    same([t.grad for t in leaves], gated_all(x.contiguous(), wg, wu)[1:])


def test_gated_empty_and_one(cuda):
    wg, wu, b = rand(24, 16), rand(24, 16, seed=1), rand(24, seed=2)
    h, dx, dwg, dwu, dbg, dbu = gated_all(torch.empty(0, 16, device=cuda, dtype=BF16), wg, wu, b, b)
    assert h.shape == (0, 24) and dx.shape == (0, 16)
    assert all(torch.all(t == 0) for t in (dwg, dwu, dbg, dbu))
    assert gated_linear(torch.empty(2, 0, 16, device=cuda, dtype=BF16), wg, wu).shape == (2, 0, 24)
    h8 = gated_all(torch.empty(0, 16, device=cuda, dtype=BF16), wg, wu, checkpoint_8bit=True)
    assert h8[0].shape == (0, 24)
    assert gated_linear(rand(16), wg, wu).shape == (24,)


@pytest.mark.parametrize("lead", [(2, 3), (7,), ()])
def test_xent_shapes_views_and_target_types(cuda, lead):
    h, w = rand(*lead, 40), rand(300, 40, std=0.3, seed=1)
    t = torch.randint(0, 300, lead, device=cuda)
    rows = streamed_cross_entropy(h, w, t, reduction="none")
    assert rows.shape == t.shape and rows.dtype == FP32
    ref = F.cross_entropy(h.float().reshape(-1, 40) @ w.float().T, t.reshape(-1), reduction="none")
    assert torch.allclose(rows.reshape(-1), ref, rtol=1e-5, atol=1e-5)
    assert torch.equal(streamed_cross_entropy(h, w, t.int(), reduction="none"), rows)
    seq = rand(3, 9, 40, seed=5)
    tt = torch.randint(0, 300, (3, 8), device=cuda)
    same(xent_all(seq[:, :-1].contiguous(), w, tt), [*xent_all(seq, w, F.pad(tt, (0, 1), value=-100))[:1],
                                                     xent_all(seq, w, F.pad(tt, (0, 1), value=-100))[1][:, :-1],
                                                     xent_all(seq, w, F.pad(tt, (0, 1), value=-100))[2]])


# ------------------------------------------------------------------ masks, bad values
@pytest.mark.parametrize("M", [5, 700])
def test_xent_masked_rows_may_hold_anything(cuda, M):
    h, w = rand(M, 64), rand(1000, 64, std=0.2, seed=1)
    t = torch.randint(0, 1000, (M,), device=cuda)
    t[1::3] = -100
    clean = xent_all(h, w, t)
    dirty = h.clone()
    dirty[1::3] = float("nan")
    dirty[1] = float("inf")
    same(xent_all(dirty, w, t), clean)
    with torch.no_grad():
        assert torch.equal(streamed_cross_entropy(dirty, w, t), streamed_cross_entropy(h, w, t))
    keep = t != -100
    want = xent_all(h[keep], w, t[keep])  # the rows alone
    assert torch.equal(clean[0], want[0]) and torch.equal(clean[1][keep], want[1]) and torch.all(clean[1][~keep] == 0)
    assert rel_l2(clean[2], want[2]) < 2.0 ** -8


def test_xent_no_row_counts(cuda):
    h, w = rand(9, 64), rand(100, 64, seed=1)
    t = torch.full((9,), -100, device=cuda)
    for red in ("mean", "sum", "none"):
        loss, dh, dw = xent_all(h, w, t, reduction=red)
        assert torch.isnan(loss) if red == "mean" else torch.all(loss == 0)
        assert torch.all(dh == 0) and torch.all(dw == 0)
        with torch.no_grad():
            alone = streamed_cross_entropy(h, w, t, reduction=red)
        assert torch.isnan(alone) if red == "mean" else torch.all(alone == 0)
    for red in ("mean", "sum", "none"):  # and none at all
        loss, dh, dw = xent_all(h[:0], w, t[:0], reduction=red)
        assert dh.shape == (0, 64) and dw.shape == w.shape and (red != "mean" or torch.isnan(loss))


@pytest.mark.parametrize("grad", [True, False])
def test_xent_bad_target_is_reported(cuda, grad):
    h, w = rand(40, 64), rand(100, 64, seed=1)
    t = torch.randint(0, 100, (40,), device=cuda)
    t[3], t[7] = 100, -5
    h.requires_grad_(grad)
    rows = streamed_cross_entropy(h if grad else h[:10], w, t if grad else t[:10], reduction="none").detach()
    with pytest.raises(RuntimeError, match="outside"):
        check_device_status(cuda)
    bad = torch.isnan(rows)
    assert bad[3] and bad[7] and int(bad.sum()) == 2
    t[3] = t[7] = 0
    streamed_cross_entropy(h, w, t)
    check_device_status(cuda)  # the word was cleared


def test_xent_ignore_index_inside_the_vocabulary(cuda):
    h, w = rand(50, 64), rand(30, 64, seed=1)
    t = torch.randint(0, 30, (50,), device=cuda)
    loss, dh, _ = xent_all(h, w, t, ignore_index=7)
    ref = F.cross_entropy(h.float() @ w.float().T, t, ignore_index=7)
    assert abs(float(loss) - float(ref)) < 1e-5 * float(ref)
    assert torch.all(dh[t == 7] == 0)


@pytest.mark.parametrize("M", [4, 100])
def test_xent_large_and_infinite_logits(cuda, M):
    h, w = rand(M, 64, std=100.0), rand(500, 64, std=10.0, seed=1)
    t = torch.randint(0, 500, (M,), device=cuda)
    z = h.double() @ w.double().T
    ref = F.cross_entropy(z, t, reduction="none")
    rows, dh, dw = xent_all(h, w, t, reduction="none")
    # fp32 keeps a logit of magnitude |z| to 2^-24 |z|, its sum over 64 products to 64 2^-23 of their magnitudes
    bound = 2 * 64 * 2.0 ** -23 * (h.double().abs() @ w.double().abs().T).amax(1) + 2.0 ** -20 * z.abs().amax(1) + 1e-6
    assert torch.all((rows - ref).abs() <= bound)
    assert torch.isfinite(dh).all() and torch.isfinite(dw).all()
    with torch.no_grad():
        assert torch.all((streamed_cross_entropy(h, w, t, reduction="none") - ref).abs() <= bound)
    w2 = w.clone()
    w2[11] = float("inf")  # as F.cross_entropy: NaN
    assert torch.isnan(streamed_cross_entropy(h.abs(), w2, t, reduction="none")).all()
    h2 = h.clone()
    h2[2] = float("nan")
    bad = torch.isnan(streamed_cross_entropy(h2, w, t, reduction="none"))
    assert bad[2] and int(bad.sum()) == 1


@pytest.mark.parametrize("dt", [BF16, FP16])
def test_gated_extreme_preactivations(cuda, dt):
    """Saturated activations: exact limits, no NaN from 0 times infinity inside the range."""
    x = torch.tensor([[60.0], [-60.0], [0.0], [1e-3]], device=cuda, dtype=dt)
    wg, wu = torch.full((8, 1), 4.0, device=cuda, dtype=dt), torch.full((8, 1), 0.5, device=cuda, dtype=dt)
    for name, fn in (("silu", F.silu), ("gelu", F.gelu)):
        for kw in ({}, {"checkpoint_8bit": True}):
            got = gated_all(x, wg, wu, activation=name, **kw)
            xs = x.double() if not kw else act8_unpack(act8_pack(x)).double()
            leaves = [t.requires_grad_(True) for t in (xs, wg.double(), wu.double())]
            out = fn(leaves[0] @ leaves[1].T) * (leaves[0] @ leaves[2].T)
            grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
            if not kw:
                assert torch.allclose(got[0].double(), out.detach(), rtol=2 * torch.finfo(dt).eps, atol=1e-6)
            for a, b in zip(got[1:], grads):
                assert torch.allclose(a.double(), b, rtol=4 * torch.finfo(dt).eps, atol=1e-4), (name, a, b)


# ------------------------------------------------------------------ types, autocast, copies
@pytest.mark.parametrize("dt", [BF16, FP16])
def test_autocast_with_fp32_parameters(cuda, dt):
    x, wg, wu, b = rand(70, 48, dt=FP32), rand(56, 48, dt=FP32, std=0.2, seed=1), rand(56, 48, dt=FP32, std=0.2, seed=2), rand(56, dt=FP32, seed=3)
    with torch.autocast("cuda", dtype=dt):
        got = gated_all(x, wg, wu, b, b, dh=rand(70, 56, dt=dt, seed=4))
    want = gated_all(x.to(dt), wg.to(dt), wu.to(dt), b, b, dh=rand(70, 56, dt=dt, seed=4))
    assert got[0].dtype == dt and all(t.dtype == FP32 for t in got[1:])
    assert torch.equal(got[0], want[0])
    for a, c in zip(got[1:], want[1:]):
        assert torch.equal(a.to(c.dtype), c)  # the same sums, rounded later
    h, w, t = rand(90, 48, dt=FP32), rand(200, 48, dt=FP32, seed=1), torch.randint(0, 200, (90,), device=cuda)
    with torch.autocast("cuda", dtype=dt):
        got = xent_all(h, w, t)
    want = xent_all(h.to(dt), w.to(dt), t)
    assert got[1].dtype == got[2].dtype == FP32 and torch.equal(got[0], want[0])
    assert torch.equal(got[1].to(dt), want[1]) and torch.equal(got[2].to(dt), want[2])


def test_parameter_copies_are_used_while_current(cuda):
    wg, wu, w = (torch.nn.Parameter(rand(64, 32, dt=FP32, seed=i)) for i in range(3))
    casts = Bf16Casts([wg, wu, w], padded={id(w): 128})
    casts.refresh()
    x, t = rand(40, 32), torch.randint(0, 64, (40,), device=cuda)
    with torch.autocast("cuda", dtype=BF16):
        a = gated_linear(x, wg, wu, casts=casts)
        assert torch.equal(a, gated_linear(x, wg, wu))
        b = streamed_cross_entropy(x, w, t, casts=casts)
        assert torch.equal(b, streamed_cross_entropy(x, w, t))
        with torch.no_grad():
            wg.mul_(2), w.mul_(2)  # stale copies are not used
        assert torch.equal(gated_linear(x, wg, wu, casts=casts), gated_linear(x, wg, wu))
        assert torch.equal(streamed_cross_entropy(x, w, t, casts=casts), streamed_cross_entropy(x, w, t))


def test_gradients_of_a_part_of_the_inputs(cuda):
    x, wg, wu, b = rand(70, 64), rand(96, 64, std=0.1, seed=1), rand(96, 64, std=0.1, seed=2), rand(96, seed=3)
    full = gated_all(x, wg, wu, b, b)
    for i in range(5):
        leaves = [t.detach().clone() for t in (x, wg, wu, b, b)]
        leaves[i].requires_grad_(True)
        g, = torch.autograd.grad(gated_linear(*leaves), [leaves[i]], torch.ones(70, 96, device=cuda, dtype=BF16))
        assert torch.equal(g, full[1 + i]), i
    only = gated_all(x, wg, wu, b, None)
    assert torch.equal(only[4], gated_all(x, wg, wu, b, torch.zeros_like(b))[4])
    h, w, t = rand(70, 64), rand(300, 64, seed=1), torch.randint(0, 300, (70,), device=cuda)
    _, dh, dw = xent_all(h, w, t)
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(streamed_cross_entropy(hh, w, t), hh)[0], dh)
    assert torch.equal(torch.autograd.grad(streamed_cross_entropy(h, ww, t), ww)[0], dw)


def test_one_gradient_of_a_product_with_a_split_last_round(cuda):
    x, wg, wu, dh = rand(4200, 1300), rand(1800, 1300, std=0.03, seed=1), rand(1800, 1300, std=0.03, seed=2), rand(4200, 1800, seed=3)
    full = gated_all(x, wg, wu, dh=dh)
    for i in range(3):
        leaves = [t.detach().clone() for t in (x, wg, wu)]
        leaves[i].requires_grad_(True)
        assert torch.equal(torch.autograd.grad(gated_linear(*leaves), leaves[i], dh)[0], full[1 + i]), i


def test_xent_zero_and_huge_upstream_gradients(cuda):
    h, w, t = rand(70, 64), rand(300, 64, std=0.2, seed=1), torch.randint(0, 300, (70,), device=cuda)
    for dt in (BF16, FP16):
        hh, ww = h.to(dt), w.to(dt)
        _, dh, dw = xent_all(hh, ww, t, reduction="none", dloss=torch.zeros(70, device=cuda))
        assert torch.all(dh == 0) and torch.all(dw == 0)
        up = torch.zeros(70, device=cuda)
        up[5] = 3.0
        _, dh, _ = xent_all(hh, ww, t, reduction="none", dloss=up)
        assert torch.all(dh[:5] == 0) and torch.all(dh[6:] == 0) and torch.any(dh[5] != 0)
        # the upstream factor enters after the sums, in fp32: a power of two changes no bit of a normal number
        one, scaled = xent_all(hh, ww, t), xent_all(hh, ww, t, dloss=torch.tensor(2.0 ** 10, device=cuda))
        for a, b in zip(one[1:], scaled[1:]):
            normal = a.abs() >= torch.finfo(dt).smallest_normal
            assert torch.any(normal) and torch.equal(a[normal].float() * 2.0 ** 10, b[normal].float())


# ------------------------------------------------------------------ streams, graphs, reruns, differences
@pytest.mark.parametrize("D", [64, 320])
def test_xent_infinite_upstream_gradient_of_one_row(cuda, D):
    h, w = rand(70, D, seed=8), rand(300, D, std=D ** -0.5, seed=9)
    t = torch.arange(70, device=cuda)
    dloss = torch.ones(70, device=cuda)
    want = xent_all(h, w, t, dloss=dloss, reduction="none")[1]
    for bad in (float("inf"), float("nan")):
        dloss[33] = bad
        dh = xent_all(h, w, t, dloss=dloss, reduction="none")[1]
        rest = torch.arange(70, device=cuda) != 33
        assert not torch.isfinite(dh[33]).any()
        assert torch.equal(dh[rest], want[rest])


def test_calls_on_another_stream(cuda):
    x, wg, wu, t, w = rand(500, 256), rand(384, 256, std=0.05, seed=1), rand(384, 256, std=0.05, seed=2), torch.randint(0, 999, (500,), device=cuda), rand(999, 256, std=0.1, seed=3)
    want = gated_all(x, wg, wu), xent_all(x, w, t), act8_weight_grad(x, act8_pack(x))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gated_all(x, wg, wu), xent_all(x, w, t), act8_weight_grad(x, act8_pack(x))
    s.synchronize()
    same(got[0], want[0]), same(got[1], want[1])
    assert torch.equal(got[2], want[2])


def test_two_streams_at_once(cuda):
    """Calls that share no buffer run side by side."""
    xs = [rand(700, 256, seed=i) for i in range(2)]
    w, t = rand(5000, 256, std=0.1, seed=9), torch.randint(0, 5000, (700,), device=cuda)
    want = [xent_all(x, w, t) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(xent_all(x, w, t))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        same(a, b)


def test_offsets_past_32_bits(cuda):
    """The far end of tensors of more than 2^31 elements. bf16 results of two summation orders
    of fp32 sums differ by one rounding each at most: 2^-8 relative in all."""
    far = slice(-300, None)
    M, D, F_ = 66_000, 64, 33_000  # h, dh, and dg beside du
    x, wg, wu = rand(M, D), rand(F_, D, std=D ** -0.5, seed=1), rand(F_, D, std=D ** -0.5, seed=2)
    dh = rand(1, F_, seed=3).expand(M, F_).contiguous()
    xa = x.detach().requires_grad_(True)
    h = gated_linear(xa, wg, wu)
    dx, = torch.autograd.grad(h, xa, dh)
    xb = x[far].detach().requires_grad_(True)
    hb = gated_linear(xb, wg, wu)
    assert torch.equal(h[far], hb)
    assert rel_l2(dx[far], torch.autograd.grad(hb, xb, dh[far])[0]) < 2 ** -8
    del h, dh, dx
    M, D = 2_100_000, 1032
    x = rand(4096, D).repeat(M // 4096 + 1, 1)[:M]
    assert torch.equal(act8_unpack(act8_pack(x))[far], act8_unpack(act8_pack(x[far])))
    del x
    V, D, M = 2_200_000, 1000, 64
    w, h = rand(V, D, std=D ** -0.5), rand(M, D, seed=5)
    t = V - 1 - torch.arange(M, device=cuda)
    loss, gh, gw = xent_all(h, w, t, reduction="sum")
    z = torch.cat([h.float() @ c.float().t() for c in w.split(550_000)], 1)
    p = torch.softmax(z, 1)
    assert abs(loss.item() - F.cross_entropy(z, t, reduction="sum").item()) < 1e-4 * loss.item()
    p[torch.arange(M), t] -= 1
    # two roundings to bf16, of dz and of the result, and TF32 or fp32 sums in the plain form
    assert rel_l2(gw[-300:], p[:, -300:].t() @ h.float()) < 2 ** -8 + 2 ** -9


@pytest.mark.parametrize("M", [8, 600])
def test_forward_captured_and_replayed_on_new_inputs(cuda, M):
    x, w, t = rand(M, 128), rand(2000, 128, std=0.1, seed=1), torch.randint(0, 2000, (M,), device=cuda)
    wg, wu = rand(256, 128, std=0.1, seed=2), rand(256, 128, std=0.1, seed=3)

    def step():
        with torch.no_grad():
            return (gated_linear(x, wg, wu), streamed_cross_entropy(x, w, t, reduction="none"),
                    act8_unpack(act8_pack(x)), act8_weight_grad(x, act8_pack(x)))

    step()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for seed in (5, 6):
        x.copy_(rand(M, 128, seed=seed))
        t.copy_(torch.randint(0, 2000, (M,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)))
        t[seed % M] = -100
        for g, out in graphs:
            g.replay()
        want = step()
        for _, out in graphs:
            same(out, want)


def test_backward_captured_and_replayed_on_new_inputs(cuda):
    """The number of rows that count is data: a replay follows it."""
    h, w = rand(600, 128).requires_grad_(True), rand(3000, 128, std=0.1, seed=1).requires_grad_(True)
    t = torch.randint(0, 3000, (600,), device=cuda)

    def step():
        loss = streamed_cross_entropy(h, w, t)
        return [loss, *torch.autograd.grad(loss, (h, w))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for ignored in (0, 130, 599):
        with torch.no_grad():
            h.copy_(rand(600, 128, seed=ignored))
        t.copy_(torch.randint(0, 3000, (600,), device=cuda))
        t[:ignored] = -100
        g.replay()
        same([o.detach() for o in out], xent_all(h, w, t))


@pytest.mark.parametrize("D", [72, 1000])
def test_a_graph_is_differentiated_twice_and_checks_its_tensors(cuda, D):
    """retain_graph, another upstream gradient for each pass; an input changed in place since raises."""
    x, wg, wu = (rand(*s, std=D ** -0.5, seed=i).requires_grad_(True) for i, s in enumerate([(200, D), (130, D), (130, D)]))
    w, t = rand(1000, 130, seed=9).requires_grad_(True), torch.arange(200, device=cuda)
    for in8 in (False, True):
        h = gated_linear(x, wg, wu, checkpoint_8bit=in8)
        loss = streamed_cross_entropy(h, w, t, reduction="none")
        up = rand(200, dt=FP32, seed=3)
        a = torch.autograd.grad(loss, (x, wg, wu, w), up, retain_graph=True)
        b = torch.autograd.grad(loss, (x, wg, wu, w), torch.zeros_like(up), retain_graph=True)
        assert all(not torch.any(g) for g in b)
        same(torch.autograd.grad(loss, (x, wg, wu, w), up), a)
    h = gated_linear(x, wg, wu)
    with torch.no_grad():
        wg.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h.sum(), x)


def test_reruns_are_bitwise_equal(cuda):
    x, wg, wu, b = rand(1500, 700), rand(1030, 700, std=0.04, seed=1), rand(1030, 700, std=0.04, seed=2), rand(1030, seed=3)
    w, t = rand(7001, 700, std=0.1, seed=4), torch.randint(0, 7001, (1500,), device=cuda)
    t[::5] = -100
    a = gated_all(x, wg, wu, b, b), gated_all(x, wg, wu, b, b, checkpoint_8bit=True), xent_all(x, w, t)
    for _ in range(3):
        c = gated_all(x, wg, wu, b, b), gated_all(x, wg, wu, b, b, checkpoint_8bit=True), xent_all(x, w, t)
        for p, q in zip(a, c):
            same(p, q)


def test_gradients_against_differences(cuda):
    """Directional differences of the fp32 loss: streamed cross entropy of a gated product's rows."""
    wg, wu, w = rand(64, 48, std=0.2, seed=1), rand(64, 48, std=0.2, seed=2), rand(400, 64, std=0.3, seed=3)
    x, t = rand(50, 48, seed=4), torch.randint(0, 400, (50,), device=cuda)

    def loss(x, w):
        return streamed_cross_entropy(gated_linear(x, wg, wu), w, t)

    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(loss(xs, ws), (xs, ws))
    dx, dw = dx.double(), dw.double()
    # A step along the weight's gradient: the head is linear in w, inputs stay exact bf16 numbers when the step is
    # taken in whole bf16 steps of w; the difference's curvature and the 2^-24 of the loss stay below 3 percent.
    for leaf, g, f in ((w, dw, lambda v: loss(x, v)), (x, dx, lambda v: loss(v, w))):
        step = (g.sign() * leaf.abs().double() * 2.0 ** -5).to(BF16)
        up, down = (leaf + step), (leaf - step)
        with torch.no_grad():
            diff = float(f(up).double() - f(down).double())
        expect = float((g * (up.double() - down.double())).sum())
        # the gated product rounds h to bf16 in both evaluations: x's differences see 2^-8 of |h| per row, averaged
        assert abs(diff - expect) < 0.05 * abs(expect) + 2e-3, (diff, expect)


# ------------------------------------------------------------------ refusals
def test_refusals(cuda):
    x, w = rand(10, 64), rand(96, 64)
    t = torch.zeros(10, dtype=torch.int64, device=cuda)
    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        gated_linear(x.float(), w.float(), w.float())
    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        streamed_cross_entropy(x.float(), w, t)
    with pytest.raises(ValueError, match="activation"):
        gated_linear(x, w, w, activation="relu")
    with pytest.raises(ValueError, match="reduction"):
        streamed_cross_entropy(x, w, t, reduction="max")
    for args in ((x[:, :32], w, w), (x, w, w[:50]), (x, w[0], w[0]), (x[0, 0], w, w), (x, w[:, :0], w[:, :0])):
        with pytest.raises(RuntimeError):
            gated_linear(*args)
    with pytest.raises(RuntimeError, match="bias"):
        gated_linear(x, w, w, rand(95))
    with pytest.raises(RuntimeError, match="one dtype"):
        gated_linear(x, w, w.float())
    with pytest.raises(RuntimeError, match="one dtype"):
        gated_linear(x, w, w, rand(96), rand(96, dt=FP32))
    with pytest.raises(RuntimeError, match="dtype|float"):
        gated_linear(x, w.double(), w.double())
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_linear(x, w.cpu(), w)
    for bad in (t[:9], t.float(), t.bool()):
        with pytest.raises(RuntimeError, match="targets"):
            streamed_cross_entropy(x, w, bad)
    with pytest.raises(RuntimeError):
        streamed_cross_entropy(x, w[:, :32], t)
    with pytest.raises(RuntimeError, match="CUDA"):
        streamed_cross_entropy(x, w, t.cpu())
    with pytest.raises(RuntimeError):
        act8_pack(x.double())
    with pytest.raises(RuntimeError):
        act8_pack(x[:, :0])
    p = act8_pack(x)
    assert isinstance(p, Act8) and p.width == 64
    with pytest.raises(RuntimeError, match="rows"):
        act8_weight_grad(x[:9], p)
    with pytest.raises(RuntimeError):
        act8_weight_grad(x.float(), p)
    with pytest.raises(RuntimeError, match="float16"):
        act8_weight_grad(x.half(), p)


def test_twice_differentiating_raises(cuda):
    x, w = rand(10, 64).requires_grad_(True), rand(96, 64)
    h = gated_linear(x, w, w)
    g, = torch.autograd.grad(h.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
    loss = streamed_cross_entropy(x, w, torch.zeros(10, dtype=torch.int64, device=cuda))
    g, = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
