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
