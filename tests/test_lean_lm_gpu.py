"""The lean training-step operators where the LM uses them: gated feed-forward, streamed
loss and 8-bit checkpoints in PnFirLM against plain compositions of the same model, the
whole step in a CUDA graph, and 8-bit checkpoints in Linear."""
import pytest
import torch
import torch.nn.functional as F

from conftest import rel_l2
from paper_01_anti_decoy_pnfirtau_b200 import lm
from paper_01_anti_decoy_pnfirtau_b200 import act8_pack, act8_unpack, check_device_status, gated_linear, gated_mlp
from paper_01_anti_decoy_pnfirtau_b200.lm import GatedFFN, GraphedTrainStep, LMConfig, PnFirLM, lm_loss, make_optimizer, train_step
from paper_01_anti_decoy_pnfirtau_b200.lm_ops import Linear

pytestmark = pytest.mark.gpu

CFG = dict(vocab=1003, d_model=128, n_heads=2, n_layers=2, d_ff=344, max_seq=128)


def model(device, seed=0, **kw):
    torch.manual_seed(seed)
    cfg = LMConfig(**CFG, ffn=kw.pop("ffn", "swiglu"))
    return PnFirLM(cfg, **kw).to(device)


def grads(m, loss):
    loss.backward()
    out = {n: p.grad.detach().clone() for n, p in m.named_parameters()}
    m.zero_grad(set_to_none=True)
    return float(loss.detach()), out


class PlainLinear8(torch.autograd.Function):
    """A Linear layer in bf16 whose weight gradient sees its input in 8 bits."""

    @staticmethod
    def forward(ctx, x, w, b):
        xb, wb = x.bfloat16(), w.bfloat16()
        ctx.save_for_backward(xb, wb)
        return F.linear(xb, wb, None if b is None else b.bfloat16())

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        x8 = act8_unpack(act8_pack(x)).float().reshape(-1, x.shape[-1])
        d = dy.bfloat16().float().reshape(-1, dy.shape[-1])
        return (d @ w.float()).view(x.shape), d.T @ x8, d.sum(0) if ctx.needs_input_grad[2] else None


class PlainGated8(torch.autograd.Function):
    """The gated product in fp32 on bf16 operands, its gradient taken at x in 8 bits."""

    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act):
        ctx.act = act
        ctx.save_for_backward(x, wg, wu, bg, bu)
        with torch.autocast("cuda", enabled=False):
            return PlainGated8.product(x.float(), *(t.bfloat16().float() for t in (wg, wu)), bg, bu, act).bfloat16()

    @staticmethod
    def product(x, wg, wu, bg, bu, act):
        return act(x @ wg.T + bg) * (x @ wu.T + bu)

    @staticmethod
    def backward(ctx, dh):
        x, *ws = ctx.saved_tensors
        with torch.enable_grad(), torch.autocast("cuda", enabled=False):
            ops = [act8_unpack(act8_pack(x)).float()] + [t.bfloat16().float() for t in ws[:2]] + [t.detach() for t in ws[2:]]
            ops = [t.requires_grad_(True) for t in ops]
            out = PlainGated8.product(*ops, ctx.act)
        return (*torch.autograd.grad(out, ops, dh.float()), None)


# Both sides of the comparisons below run the same attention, norms and residuals on the same
# bf16 operands; they differ in sums' order and in 16-bit roundings of single products'
# operands (the logits' gradient, the hidden layer's gradients) and results: at most 12 on a
# gradient's way through two blocks, each at most 2^-8 of its tensor in L2.
TOL = 12 * 2.0 ** -8


@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
def test_lm_streamed_loss_against_fp32_logits(cuda, ffn):
    idx = torch.randint(0, CFG["vocab"], (5, 97), device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    m = model(cuda, ffn=ffn, streamed_loss=True)
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        l1, g1 = grads(m, lm_loss(m, idx))
        casts = m._step_casts(idx.device)
        h = m._trunk_fused(m.embed(idx) + m.pos(torch.arange(97, device=cuda)), casts)
    logits = h[:, :-1].bfloat16().float() @ m.head.weight.bfloat16().float().T
    l0, g0 = grads(m, F.cross_entropy(logits.reshape(-1, CFG["vocab"]), idx[:, 1:].reshape(-1)))
    check_device_status(cuda)
    assert abs(l0 - l1) < 1e-5 * abs(l0)
    for n, g in g0.items():
        assert rel_l2(g1[n], g) < TOL, (n, rel_l2(g1[n], g))


@pytest.mark.parametrize("ffn", ["swiglu", "geglu"])
def test_lm_8bit_checkpoints_against_plain_layers(cuda, ffn, monkeypatch):
    idx = torch.randint(0, CFG["vocab"], (5, 97), device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    m = model(cuda, ffn=ffn, streamed_loss=True, checkpoint_8bit=True)
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        l1, g1 = grads(m, lm_loss(m, idx))
    check_device_status(cuda)
    act = F.silu if ffn == "swiglu" else F.gelu
    monkeypatch.setattr(Linear, "forward", lambda self, x: PlainLinear8.apply(x, self.weight, self.bias))
    monkeypatch.setattr(lm, "gated_mlp", lambda x, g, u, d, name, **kw: d(
        PlainGated8.apply(x, g.weight, u.weight, g.bias, u.bias, act)))
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        l0, g0 = grads(m, lm_loss(m, idx))
    assert abs(l0 - l1) < 1e-3 * abs(l0)
    for n, g in g0.items():
        assert rel_l2(g1[n], g) < TOL, (n, rel_l2(g1[n], g))


def test_lm_8bit_checkpoints_leave_the_forward_alone(cuda):
    idx = torch.randint(0, CFG["vocab"], (3, 40), device=cuda, generator=torch.Generator(device=cuda).manual_seed(5))
    a, b = model(cuda, streamed_loss=True), model(cuda, streamed_loss=True, checkpoint_8bit=True)
    b.load_state_dict(a.state_dict())
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        la, lb = lm_loss(a, idx), lm_loss(b, idx)
    assert torch.equal(la, lb)


def test_lean_lm_step_captured_and_replayed(cuda):
    """The step with every lean option in one CUDA graph, replayed on new ids, equals eager steps bit for bit."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    batches = [torch.randint(0, CFG["vocab"], (4, 64), device=cuda, generator=gen) for _ in range(3)]
    a = model(cuda, streamed_loss=True, checkpoint_8bit=True)
    b = model(cuda, streamed_loss=True, checkpoint_8bit=True)
    b.load_state_dict(a.state_dict())
    oa, ob = make_optimizer(a, capturable=True), make_optimizer(b, capturable=True)
    step = GraphedTrainStep(b, ob, batches[0])
    for idx in batches:
        la = train_step(a, oa, idx)
        lb = step.step(idx)
        assert abs(float(la) - float(lb)) <= 1e-3 * abs(float(la))
    step.close()
    check_device_status(cuda)
    for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert rel_l2(q, p) < 1e-3, n


def test_lean_lm_step_keeps_less(cuda):
    """Memory that the forward keeps for the backward, at a size where activations dominate."""
    cfg = LMConfig(vocab=8192, d_model=256, n_heads=4, n_layers=4, d_ff=1024, max_seq=512, ffn="swiglu")
    idx = torch.randint(0, 8192, (16, 512), device=cuda)
    kept = {}
    for name, kw in (("plain", {}), ("lean", dict(streamed_loss=True, checkpoint_8bit=True))):
        torch.manual_seed(0)
        m = PnFirLM(cfg, **kw).to(cuda)
        for _ in range(2):
            before = torch.cuda.memory_allocated()
            with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
                loss = lm_loss(m, idx)
            kept[name] = torch.cuda.memory_allocated() - before
            loss.backward()
            m.zero_grad(set_to_none=True)
        del m, loss
    logits = 16 * 511 * 8192 * 2
    assert kept["plain"] - kept["lean"] > logits  # the logits and more


@pytest.mark.parametrize("bias", [True, False])
def test_linear_with_8bit_checkpoint(cuda, bias):
    torch.manual_seed(3)
    lin = Linear(100, 77, bias=bias).to(cuda)
    x = torch.randn(3, 33, 100, device=cuda).bfloat16().requires_grad_(True)
    dy = torch.randn(3, 33, 77, device=cuda).bfloat16()
    y = lin(x)
    plain = torch.autograd.grad(y, [x, *lin.parameters()], dy)
    lin.checkpoint_8bit = True
    y8 = lin(x)
    packed = torch.autograd.grad(y8, [x, *lin.parameters()], dy)
    assert torch.equal(y, y8) and torch.equal(plain[0], packed[0])
    if bias:
        assert torch.equal(plain[2], packed[2])
    x8 = act8_unpack(act8_pack(x.detach().reshape(-1, 100))).double()
    d = dy.reshape(-1, 77).double()
    # products of bf16 numbers summed over 99 rows in fp32
    err = (packed[1].double() - d.T @ x8).abs()
    assert torch.all(err <= 99 * 2.0 ** -23 * (d.abs().T @ x8.abs()))
    with pytest.raises(RuntimeError, match="bfloat16"):
        lin(x.float())


def test_gated_mlp_is_its_three_layers(cuda):
    torch.manual_seed(4)
    ffn = GatedFFN(96, 200, "geglu").to(cuda).bfloat16()
    x = torch.randn(2, 50, 96, device=cuda).bfloat16()
    y = ffn(x)
    h = gated_linear(x, ffn.gate.weight, ffn.up.weight, ffn.gate.bias, ffn.up.bias, "gelu")
    assert torch.equal(y, ffn.down(h)) and torch.equal(y, gated_mlp(x, ffn.gate, ffn.up, ffn.down, "gelu"))
    ref = F.linear(F.gelu(F.linear(x.float(), ffn.gate.weight.float(), ffn.gate.bias.float()))
                   * F.linear(x.float(), ffn.up.weight.float(), ffn.up.bias.float()),
                   ffn.down.weight.float(), ffn.down.bias.float())
    assert rel_l2(y, ref) < 1e-2


def test_lean_options_are_refused_where_they_cannot_run(cuda):
    with pytest.raises(ValueError, match="fused_step_ops"):
        PnFirLM(LMConfig(**CFG), fused_step_ops=False, streamed_loss=True)
    with pytest.raises(ValueError, match="ffn"):
        PnFirLM(LMConfig(**CFG, ffn="relu"))
    m = model(cuda, streamed_loss=True)
    with pytest.raises(RuntimeError, match="bfloat16"):
        m(torch.zeros(1, 8, dtype=torch.int64, device=cuda), targets=torch.zeros(1, 7, dtype=torch.int64, device=cuda))
