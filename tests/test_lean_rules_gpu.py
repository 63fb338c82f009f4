"""Calls of the lean training-step operators at the edges of what they allow."""
import pytest
import torch

from paper_01_anti_decoy_pnfirtau_b200 import (act8_pack, act8_unpack, act8_weight_grad, check_device_status, gated_linear,
                                               streamed_cross_entropy)
from paper_01_anti_decoy_pnfirtau_b200 import lm_lean_ops as lean
from paper_01_anti_decoy_pnfirtau_b200 import lm_ops
from paper_01_anti_decoy_pnfirtau_b200.lm_ops import Bf16Casts, Linear, mlp_gelu

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, dt=BF16, std=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dt)


# ------------------------------------------------------------------ parameter copies
def copied_calls():
    """An input, and (call, parameters) of every operator that takes parameter copies."""
    x = rand(40, 32).requires_grad_(True)
    a, b, w = (torch.nn.Parameter(rand(64, 32, dt=FP32, std=0.3, seed=i)) for i in range(3))
    t = torch.arange(40, device="cuda")
    lin = Linear(32, 64).to("cuda")
    fc1, fc2 = torch.nn.Linear(32, 64).to("cuda"), torch.nn.Linear(64, 32).to("cuda")

    def linear(casts):
        lin.casts = casts
        return lin(x)

    return x, {
        "gated": (lambda casts: gated_linear(x, a, b, casts=casts), [a, b]),
        "gated8": (lambda casts: gated_linear(x, a, b, checkpoint_8bit=True, casts=casts), [a, b]),
        "xent": (lambda casts: streamed_cross_entropy(x, w, t, casts=casts), [w]),
        "linear": (linear, list(lin.parameters())),
        "mlp": (lambda casts: mlp_gelu(x, fc1, fc2, casts), [*fc1.parameters(), *fc2.parameters()]),
    }


@pytest.mark.parametrize("name", ["gated", "gated8", "xent", "linear", "mlp"])
def test_a_graph_on_parameter_copies_refreshed_since(cuda, name):
    """Copies refreshed from parameters that changed raise in the backward of a graph made before, as an in-place
    change of the parameters themselves does; refreshed from the same parameters they do not."""
    x, calls = copied_calls()
    call, params = calls[name]
    casts = Bf16Casts(params)
    casts.refresh()
    with torch.autocast("cuda", dtype=BF16):
        first, want = call(casts), call(None)
        casts.refresh()  # another forward in between, say of the next micro-batch
        second = call(casts)
    for out in (first, second):
        got = torch.autograd.grad(out.float().sum(), [x, *params], retain_graph=True)
        for g, r in zip(got, torch.autograd.grad(want.float().sum(), [x, *params], retain_graph=True)):
            assert torch.equal(g, r)
    with torch.no_grad():
        params[0].mul_(2)
    casts.refresh()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(first.float().sum(), x)


# ------------------------------------------------------------------ forward mode, tracing
def raw_calls():
    x, w, t = rand(40, 64), rand(96, 64, std=0.1, seed=1), torch.arange(40, device="cuda")
    bias, p = rand(96, seed=2), act8_pack(x)
    return {
        "gated x": (lambda v: gated_linear(v, w, w), x),
        "gated weight": (lambda v: gated_linear(x, w, v), w),
        "gated bias": (lambda v: gated_linear(x, w, w, v), bias),
        "xent h": (lambda v: streamed_cross_entropy(v, w, t), x),
        "xent weight": (lambda v: streamed_cross_entropy(x, v, t), w),
        "pack": (lambda v: act8_unpack(act8_pack(v)), x),
        "weight grad": (lambda v: act8_weight_grad(v, p), x),
    }


@pytest.mark.parametrize("name", ["gated x", "gated weight", "gated bias", "xent h", "xent weight", "pack", "weight grad"])
def test_forward_mode_and_tracing_are_refused(cuda, name):
    """A tangent would be lost and a trace would hold no operator; without tangents a dual level changes nothing."""
    import torch.autograd.forward_ad as fwAD

    call, v = raw_calls()[name]
    want = call(v)
    with fwAD.dual_level():
        assert torch.equal(call(v), want)
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(fwAD.make_dual(v, torch.ones_like(v)))
    with pytest.raises(RuntimeError, match="trac"):
        torch.jit.trace(call, (v,))
    from torch.fx.experimental.proxy_tensor import make_fx

    with pytest.raises(RuntimeError, match="trac"):
        make_fx(call)(v)
    assert torch.equal(call(v), want)


def test_act8_results_require_no_gradient(cuda):
    x, dy = rand(20, 64).requires_grad_(True), rand(20, 32, seed=1).requires_grad_(True)
    p = act8_pack(x)
    assert not act8_unpack(p).requires_grad and not act8_weight_grad(dy, p).requires_grad


# ------------------------------------------------------------------ evaluation
def test_linear_packs_its_input_for_a_backward_alone(cuda, monkeypatch):
    """With checkpoint_8bit set a call that no backward follows packs nothing, and takes any type as before."""
    torch.manual_seed(0)
    lin, x = Linear(100, 77).to(cuda), rand(33, 100)
    with torch.no_grad():
        want, want32 = lin(x), lin(x.float())
    lin.checkpoint_8bit = True
    packed = []
    monkeypatch.setattr(lm_ops, "act8_pack", lambda t: packed.append(t.shape) or act8_pack(t))
    for context in (torch.no_grad, torch.inference_mode):
        with context():
            assert torch.equal(lin(x), want) and torch.equal(lin(x.float()), want32)
    assert not packed
    assert torch.equal(lin(x).detach(), want) and packed == [(33, 100)]


# ------------------------------------------------------------------ few rows
@pytest.mark.parametrize("M", [24, 25, 31, 32, 33])
@pytest.mark.parametrize("dt", [BF16, FP16])
def test_gated_few_rows_take_rows_as_they_are(cuda, M, dt, monkeypatch):
    """Without a gradient, up to 32 rows of an odd width are read in place; 2-byte aligned views equal their copies."""
    from test_lean_ops_gpu import check, gated_inputs, gated_oracle

    copied = []
    monkeypatch.setattr(lean, "_rows16", lambda t, d, f=lean._rows16: copied.append(t.shape) or f(t, d))
    for D in (77, 1001):
        x, wg, wu, bg, bu, dh = gated_inputs(M, D, 61, dt, True, M + D, cuda)
        want = gated_oracle(x, wg, wu, bg, bu, dh, "gelu", dt, kept=False)[0]
        check("h", gated_linear(x, wg, wu, bg, bu, "gelu"), want)
    assert (not copied) == (M <= 32)
    base = rand(200, 66, dt=dt)
    for cols in (slice(1, 65), slice(1, 64)):
        x, w = base[:M, cols], base[100:, cols]
        assert torch.equal(gated_linear(x, w, w), gated_linear(x.contiguous(), w.contiguous(), w.contiguous()))


# ------------------------------------------------------------------ saved tensors
@pytest.mark.parametrize("D", [64, 77, 1001])
def test_saved_tensors_that_were_moved_come_back(cuda, D):
    """A backward whose saved tensors were kept on the host, and one that computes its forward again."""
    from torch.utils.checkpoint import checkpoint

    x, wg, wu, w = (rand(n, D, std=D ** -0.5, seed=i).requires_grad_(True) for i, n in enumerate((50, 130, 130, 300)))
    t = torch.arange(50, device=cuda)
    lin = Linear(D, 40).to(cuda).bfloat16()
    lin.checkpoint_8bit = True
    calls = {
        "gated": (lambda: gated_linear(x, wg, wu), (x, wg, wu)),
        "gated8": (lambda: gated_linear(x, wg, wu, checkpoint_8bit=True), (x, wg, wu)),
        "xent": (lambda: streamed_cross_entropy(x, w, t), (x, w)),
        "linear8": (lambda: lin(x), (x, lin.weight)),
    }
    for name, (call, leaves) in calls.items():
        want = torch.autograd.grad(call().float().sum(), leaves)
        for pinned in (False, True):
            with torch.autograd.graph.save_on_cpu(pin_memory=pinned):
                out = call()
            for g, r in zip(torch.autograd.grad(out.float().sum(), leaves), want):
                assert torch.equal(g, r), name
        for g, r in zip(torch.autograd.grad(checkpoint(call, use_reentrant=False).float().sum(), leaves), want):
            assert torch.equal(g, r), name
    check_device_status(cuda)


# ------------------------------------------------------------------ masked rows
@pytest.mark.parametrize("D", [64, 320])
@pytest.mark.parametrize("up", [float("inf"), float("nan")])
def test_ignored_rows_have_no_gradient_whatever_the_loss_s_own(cuda, D, up):
    """As F.cross_entropy: an upstream gradient that is not finite reaches the rows that count alone."""
    h, w = rand(300, D).requires_grad_(True), rand(500, D, std=D ** -0.5, seed=1)
    t = torch.arange(300, device=cuda)
    t[::3] = -100
    for reduction in ("mean", "sum"):
        loss = streamed_cross_entropy(h, w, t, reduction=reduction)
        dh, = torch.autograd.grad(loss, h, torch.tensor(up, device=cuda))
        ref, = torch.autograd.grad(torch.nn.functional.cross_entropy(h.float() @ w.float().T, t, reduction=reduction), h,
                                   torch.tensor(up, device=cuda))
        assert torch.all(ref[::3] == 0) and torch.all(dh[::3] == 0)
        counted = t != -100
        assert not torch.isfinite(dh[counted]).any()


# ------------------------------------------------------------------ precision of what is kept and summed in fp32
@pytest.mark.parametrize("D", [520, 1000])
@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_backward_sees_preactivations_of_at_least_24_bits(cuda, D, name):
    """Bias gradients of one row are dg and du themselves, in fp32. g and u are multiples of 2^-8 below 2^7, exact
    in the sums; kept with 24 bits (width 1000) they lose less than 2^-15 of their size, computed again nothing.
    |act'| <= 1.13, |act''| <= 0.8; the fast exponential and quotient cost 2^-18."""
    from test_lean_ops_gpu import act

    g0 = torch.Generator(device=cuda).manual_seed(D)
    Fh = 2000
    x = torch.randint(-3, 4, (1, D), device=cuda, generator=g0).float()
    wg, wu = (torch.randint(-8, 9, (Fh, D), device=cuda, generator=g0) / 256.0 for _ in range(2))
    bg, bu = (torch.zeros(Fh, device=cuda).requires_grad_(True) for _ in range(2))
    dh = rand(1, Fh, seed=1)
    with torch.autocast("cuda", dtype=BF16):
        h = gated_linear(x, wg, wu, bg, bu, name)
    dg, du = (t.double() for t in torch.autograd.grad(h, (bg, bu), dh))
    g, u = (x.double() @ w.double().T for w in (wg, wu))
    assert float(g.abs().max()) < 128 and float(u.abs().max()) < 128
    a, da = act(g, name)
    d, lost, fast = dh.double(), 2.0 ** -15 if D == 1000 else 0.0, 2.0 ** -18
    eg, eu = lost * g.abs(), lost * u.abs()
    want_g, want_u = (d * u * da)[0], (d * a)[0]
    bound_g = (d.abs() * (eu * 1.13 + (u.abs() + eu) * (0.8 * eg + fast * (1 + g.abs()))))[0] + 1e-30
    bound_u = (d.abs() * (1.13 * eg + fast * g.abs()))[0] + 1e-30
    assert torch.all((dg - want_g).abs() <= bound_g) and torch.all((du - want_u).abs() <= bound_u)
    # and pre-activations rounded to 16 bits would be seen here
    r = u.to(BF16).double()
    assert float(((d * r * da)[0] - want_g).abs().sub(bound_g).max()) > 0


def test_fp32_weight_gradient_of_many_rows(cuda):
    """Products of positive numbers over 65536 rows, one tile after the other without splits. The tensor core adds 16
    products at a time and loses at most two steps (2^-22) of the running sum each time; it sums 2048 rows (128 times,
    so 64.5 2^-22 of the piece's sum; half more, as numbers from 1/16 to 16 make its rows unlike), and 32 pieces are
    added in fp32. Over so many octaves the products have more bits than the sum, so that every addition loses some."""
    M, N, D = 65536, 2048, 2048
    g = torch.Generator(device=cuda).manual_seed(1)
    x, dy = (torch.exp2(8 * torch.rand(M, n, device=cuda, generator=g) - 4).to(BF16) for n in (D, N))
    p = act8_pack(x)
    got = act8_weight_grad(dy, p)
    x8, want = act8_unpack(p), torch.zeros(N, D, dtype=torch.float64, device=cuda)
    for i in range(0, M, 8192):
        want += dy[i:i + 8192].double().T @ x8[i:i + 8192].double()
    worst = float(((got.double() - want) / want).abs().max())
    assert worst <= 1.5 * 64.5 * 2.0 ** -22 + 32 * 2.0 ** -24, worst


@pytest.mark.parametrize("M,grad", [(200, True), (200, False), (20, False)])
def test_fp32_loss_of_a_wide_model(cuda, M, grad):
    """Logits that are sums of 32768 positive products, against a target whose logit is 0: the loss has the logits' own
    relative error. Sums of the tensor core as above, in pieces of 1024 (64 additions; few rows 512 and 32), which are
    added in fp32; the logarithm and its base cost 2^-20."""
    D, V = 32768, 300
    g = torch.Generator(device=cuda).manual_seed(2)
    h = (torch.rand(M, D, device=cuda, generator=g) + 0.5).to(BF16).requires_grad_(grad)
    w = ((torch.rand(V, D, device=cuda, generator=g) + 0.5) * (30.0 / D)).to(BF16)
    w[0] = 0
    rows = streamed_cross_entropy(h, w, torch.zeros(M, dtype=torch.int64, device=cuda), reduction="none").detach()
    z = h.detach().double() @ w.double().T
    want = torch.logsumexp(z, 1) - z[:, 0]
    piece, adds = (16.5, 64) if M <= 24 and not grad else (32.5, 32)
    bound = 1.1 * piece * 2.0 ** -22 + adds * 2.0 ** -24 + 2.0 ** -20
    worst = float(((rows.double() - want) / want).abs().max())
    assert worst <= bound, (worst, bound)


# ------------------------------------------------------------------ threads, whole steps
def test_two_threads_at_once(cuda):
    """Calls from two threads, each on its own stream, with backward passes."""
    import threading

    w, wg, wu = rand(3000, 256, std=0.1, seed=9), rand(512, 256, std=0.06, seed=1), rand(512, 256, std=0.06, seed=2)
    t = torch.arange(300, device=cuda)
    xs = [rand(300, 256, seed=20 + i) for i in range(2)]

    def step(x):
        leaves = [v.clone().requires_grad_(True) for v in (x, wg, wu, w)]
        h = gated_linear(*leaves[:3], checkpoint_8bit=True)
        loss = streamed_cross_entropy(h[:, :256], leaves[3], t)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    out, failed = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    out[i] = step(xs[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed
    for a, b in zip(out, want):
        for p, q in zip(a, b):
            assert torch.equal(p, q)
    check_device_status(cuda)


def test_lean_lm_step_replayed_bit_for_bit(cuda):
    """With the attention's ordered backward the captured step and eager ones agree in every bit, and so do the
    parameters after three steps (deterministic mode also fills uninitialised memory with NaN)."""
    from paper_01_anti_decoy_pnfirtau_b200.lm import GraphedTrainStep, LMConfig, PnFirLM, make_optimizer, train_step

    was, warn = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled()
    torch.use_deterministic_algorithms(True, warn_only=True)
    try:
        models = []
        for _ in range(2):
            torch.manual_seed(0)
            cfg = LMConfig(vocab=1003, d_model=128, n_heads=2, n_layers=2, d_ff=344, max_seq=128, ffn="swiglu")
            models.append(PnFirLM(cfg, streamed_loss=True, checkpoint_8bit=True).to(cuda))
        a, b = models
        gen = torch.Generator(device=cuda).manual_seed(2)
        batches = [torch.randint(0, 1003, (4, 64), device=cuda, generator=gen) for _ in range(3)]
        oa, ob = make_optimizer(a, capturable=True), make_optimizer(b, capturable=True)
        step = GraphedTrainStep(b, ob, batches[0])
        start = [p.detach().clone() for p in b.parameters()]
        for idx in batches:
            assert torch.equal(train_step(a, oa, idx), step.step(idx))
        step.close()
        for (n, p), (_, q), s in zip(a.named_parameters(), b.named_parameters(), start):
            assert torch.equal(p, q) and not torch.equal(q, s), n
    finally:
        torch.use_deterministic_algorithms(was, warn_only=warn)
    check_device_status(cuda)


def test_calls_captured_behind_copies_and_other_streams(cuda):
    """In a capture the first kernel of a call may follow a copy, a fill, or work of another stream."""
    x, wg, wu, w = rand(600, 128), rand(256, 128, std=0.1, seed=1), rand(256, 128, std=0.1, seed=2), rand(2000, 128, std=0.1, seed=3)
    t, source = torch.arange(600, device=cuda), rand(600, 128, seed=4)
    xs = [torch.empty_like(x) for _ in range(3)]
    side = torch.cuda.Stream()

    def calls(v):
        return gated_linear(v, wg, wu), streamed_cross_entropy(v, w, t, reduction="none"), act8_unpack(act8_pack(v))

    def step():
        out = []
        xs[0].copy_(source)
        out.append(calls(xs[0]))
        xs[1].zero_()
        out.append(calls(xs[1]))
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            xs[2].copy_(source)
            a = calls(xs[2])
        b = calls(x)
        here.wait_stream(side)
        out += [a, b, calls(xs[2])]
        return out

    with torch.no_grad():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for seed in (7, 8):
            source.copy_(rand(600, 128, seed=seed))
            x.copy_(rand(600, 128, seed=seed + 10))
            graph.replay()
            torch.cuda.synchronize()
            for a, v in zip(got, (source, torch.zeros_like(x), source, x, source)):
                for p, q in zip(a, calls(v)):
                    assert torch.equal(p, q)
    check_device_status(cuda)
